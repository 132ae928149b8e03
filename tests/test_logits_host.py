"""CPU: the float64 restatement against numerical differences, and what the entry points over wide rows of logits refuse."""
import math

import numpy as np
import pytest
import torch

from oracle import logits as ol


def _differences(f, z, h=1e-5):
    g = np.zeros_like(z)
    for i in np.ndindex(z.shape):
        a, b = z.copy(), z.copy()
        a[i] += h
        b[i] -= h
        g[i] = (f(a) - f(b)) / (2 * h)
    return g


@pytest.mark.parametrize("tau", [1.0, 2.5])
def test_token_logprobs_gradient_is_the_derivative(tau):
    g = np.random.default_rng(3)
    z = g.standard_normal((3, 7)) * 2
    tokens = np.array([2, -100, 6])
    ids = ol.top_ids(z, 3)
    gl, ge, gs, gt = (g.standard_normal(s) for s in (3, 3, 3, (3, 3)))

    def f(x):
        r = ol.token_logprobs(x, tokens, 0, tau)
        lp, _, _ = ol.log_softmax(x, tau)
        return (gl * r["logp"]).sum() + (ge * r["entropy"]).sum() + (gs * r["lse"]).sum() + (gt * np.take_along_axis(lp, ids, 1)).sum()

    got, bound = ol.token_logprobs_grad(z, tokens, ids, tau, gl, ge, gs, gt)
    np.testing.assert_allclose(got, _differences(f, z), atol=1e-8, rtol=1e-6)    # h^2 f''' / 6 ~ 1e-10, rounding 1e-16 / h = 1e-11 of sums near 10
    assert (bound >= 0).all()


@pytest.mark.parametrize("tail", [False, True])
def test_distill_gradient_is_the_derivative(tail):
    g = np.random.default_rng(5)
    z = g.standard_normal((4, 9)) * 2
    ids = np.array([[1, 4, 7], [3, 3, 0], [5, -1, -1], [-1, -1, -1]])     # a token twice, empty slots, an empty list
    t = np.log(np.array([[0.5, 0.2, 0.1]] * 4))
    w = np.array([0.5, 0.25, 1.0, 2.0])
    for tau in (1.0, 3.0):
        f = lambda x: (ol.distill(x, ids, t, tau, tail, w)[0] * w).sum()   # noqa: E731
        np.testing.assert_allclose(ol.distill(z, ids, t, tau, tail, w)[1], _differences(f, z), atol=2e-8, rtol=1e-6)


def test_distill_by_hand():
    z = np.log(np.array([[0.1, 0.2, 0.3, 0.4]]))
    ids, t = np.array([[3, 1]]), np.log(np.array([[0.6, 0.2]]))
    w = np.ones(1)
    want = 0.75 * math.log(0.75 / 0.4) + 0.25 * math.log(0.25 / 0.2)
    np.testing.assert_allclose(ol.distill(z, ids, t, 1.0, False, w)[0], [want], rtol=1e-12)
    want = 0.6 * math.log(0.6 / 0.4) + 0.2 * math.log(0.2 / 0.2) + 0.2 * math.log(0.2 / 0.4)
    np.testing.assert_allclose(ol.distill(z, ids, t, 1.0, True, w)[0], [want], rtol=1e-12)


def _call(fn, **kw):
    from autognothi_amd import ops
    z = torch.zeros(3, 11)
    if fn == "token_logprobs":
        return ops.token_logprobs(**{**dict(logits=z, tokens=torch.zeros(3, dtype=torch.int64)), **kw})
    if fn == "token_logprobs_bwd":
        fwd = ops.TokenLogprobs(None, torch.zeros(3), torch.zeros(3), None, None, torch.zeros(5, 3), 1.0)
        return ops.token_logprobs_bwd(**{**dict(logits=z, fwd=fwd, tokens=torch.zeros(3, dtype=torch.int64), d_logp=torch.zeros(3)), **kw})
    base = dict(logits=z, teacher_ids=torch.zeros(3, 2, dtype=torch.int64), teacher_logp=torch.zeros(3, 2))
    if fn == "topk_distill_bwd":
        base["fwd"] = ops.TopkDistill(None, None, None, torch.zeros(3, 4))
    if isinstance(kw.get("fwd"), tuple):
        kw = {**kw, "fwd": ops.TopkDistill(*kw["fwd"])}
    return getattr(ops, fn)(**{**base, **kw})


ALL = ["token_logprobs", "token_logprobs_bwd", "topk_distill", "topk_distill_bwd"]


@pytest.mark.parametrize("fn", ALL)
def test_no_cpu_fallback(fn):
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        _call(fn)


@pytest.mark.parametrize("fn", ALL)
@pytest.mark.parametrize("logits,exc,text", [
    (torch.zeros(3, 11, dtype=torch.float16), TypeError, "fp32 or bf16"), (torch.zeros(3, 11, dtype=torch.float64), TypeError, "fp32 or bf16"),
    (torch.zeros(11), ValueError, "rows, vocabulary"), (torch.zeros(1, 3, 11), ValueError, "rows, vocabulary"),
    (torch.zeros(3, 0), ValueError, "rows of 0 logits"), (torch.zeros(3, 1).expand(3, 524289), ValueError, "rows of 524289 logits")])
def test_refused_logits(fn, logits, exc, text):
    with pytest.raises(exc, match=text):
        _call(fn, logits=logits)


@pytest.mark.parametrize("fn,kw,exc,text", [
    ("token_logprobs", dict(tokens=torch.zeros(3, dtype=torch.int32)), TypeError, "tokens must be torch.int64"),
    ("token_logprobs", dict(tokens=torch.zeros(4, dtype=torch.int64)), ValueError, "tokens must be"),
    ("token_logprobs", dict(top_k=-1), ValueError, "top_k"), ("token_logprobs", dict(top_k=12), ValueError, "top_k"),
    ("token_logprobs", dict(logits=torch.zeros(3, 500), top_k=129), ValueError, "top_k"),
    ("token_logprobs", dict(temperature=0.0), ValueError, "temperature"), ("token_logprobs", dict(temperature=-1.0), ValueError, "temperature"),
    ("token_logprobs", dict(temperature=1e-7), ValueError, "temperature"), ("topk_distill", dict(temperature=2e6), ValueError, "temperature"),
    ("token_logprobs", dict(temperature=float("nan")), ValueError, "temperature"), ("topk_distill", dict(temperature=float("inf")), ValueError, "temperature"),
    ("token_logprobs_bwd", dict(tokens=None), ValueError, "without tokens"),
    ("token_logprobs_bwd", dict(d_top_logp=torch.zeros(3, 2)), ValueError, "without alternatives"),
    ("token_logprobs_bwd", dict(d_logp=torch.zeros(3, dtype=torch.float64)), TypeError, "d_logp must be"),
    ("token_logprobs_bwd", dict(d_entropy=torch.zeros(2)), ValueError, "d_entropy must be"),
    ("topk_distill", dict(teacher_ids=torch.zeros(3, 0, dtype=torch.int64)), ValueError, "teacher_ids must be"),
    ("topk_distill", dict(teacher_ids=torch.zeros(3, 129, dtype=torch.int64)), ValueError, "teacher_ids must be"),
    ("topk_distill", dict(teacher_ids=torch.zeros(2, 2, dtype=torch.int64)), ValueError, "teacher_ids must be"),
    ("topk_distill", dict(teacher_ids=torch.zeros(3, 2)), TypeError, "teacher_ids must be"),
    ("topk_distill", dict(teacher_logp=torch.zeros(3, 2, dtype=torch.float16)), TypeError, "teacher_logp must be"),
    ("topk_distill", dict(teacher_logp=torch.zeros(3, 3)), ValueError, "teacher_logp must be"),
    ("topk_distill", dict(weights=torch.zeros(3, 1)), ValueError, "weights must be"),
    ("topk_distill", dict(logits=torch.zeros(0, 11), teacher_ids=torch.zeros(0, 2, dtype=torch.int64), teacher_logp=torch.zeros(0, 2)), ValueError, "no rows"),
    ("topk_distill_bwd", dict(fwd=(None, None, None, None)), ValueError, "has computed the gradient"),
    ("topk_distill_bwd", dict(d_loss=torch.zeros(3)), ValueError, "d_loss must be"),
    ("topk_distill_bwd", dict(d_row_loss=torch.zeros(2)), ValueError, "d_row_loss must be")])
def test_refused_arguments(fn, kw, exc, text):
    with pytest.raises(exc, match=text):
        _call(fn, **kw)


def test_c_entries_refuse_bad_arguments_before_any_launch():
    from autognothi_amd import _lib as L
    lib = L.lib()
    x = 0x1000    # never read: every call below is refused on the host

    def tl(n=1, v=8, dtype=0, ld=8, tau=1.0, k=0, z=x, ent=x, ids=None, ws=None, have=0):
        return lib.ag_token_logprobs(z, ld, n, v, dtype, tau, None, k, None, ent, x, x, ids, ids, ws, have, None)

    def bw(ldd=8, st=x, g=None):
        return lib.ag_token_logprobs_bwd(x, 8, 1, 8, 0, 1.0, st, x, None, g, None, None, 0, None, None, x, ldd, None)

    def di(n=1, k=1, ids=x, tdt=0, ldd=8, dz=x, loss=x, tau=1.0):
        return lib.ag_topk_distill(x, 8, n, 8, 0, tau, ids, x, tdt, k, None, 0, x, loss, x, dz, ldd, None)

    def db(n=1, k=1, st=x, ldd=8, dz=x):
        return lib.ag_topk_distill_bwd(x, 8, n, 8, 0, 1.0, x, x, 0, k, None, 0, st, None, None, dz, ldd, None)

    for rc in (tl(n=-1), tl(v=0), tl(v=524289), tl(dtype=2), tl(ld=-1), tl(tau=0.0), tl(tau=float("nan")), tl(k=9), tl(k=-1), tl(z=None), tl(ent=None),
               tl(k=2, ids=None),
               tl(v=200000, ld=200000, ws=x, have=lib.ag_token_logprobs_workspace_bytes(1, 200000, 0, 0) - 1), tl(ws=x + 4), bw(ldd=7), bw(st=None), bw(g=x), di(n=0), di(k=0), di(k=129), di(ids=None), di(tdt=5), di(ldd=7), di(loss=None),
               di(tau=-1.0), db(n=0), db(k=0), db(st=None), db(ldd=7), db(dz=None)):
        assert rc < 0 and lib.ag_last_error()
    assert tl(n=0) == 0    # no rows: nothing to do


@pytest.mark.parametrize("fn", ALL)
def test_more_rows_than_a_launch_holds_are_refused(fn):
    z = torch.zeros(1, 11)
    with pytest.raises(ValueError, match="rows in one call"):
        _call(fn, logits=z.expand(1 << 28, 11))
    with pytest.raises(ValueError, match="rows in one call"):
        _call(fn, logits=z.expand((1 << 32) + 3, 11))


@pytest.mark.parametrize("dtype,v,n", [(0, 64, 1 << 28), (0, 65, 1 << 26), (1, 2567, 1 << 26), (0, 1284, 1 << 24), (0, 8195, 1 << 24), (0, 8196, 1 << 22),
                                       (1, 16391, 1 << 24), (1, 524288, 1 << 22)])
def test_c_entries_refuse_more_rows_than_a_launch_holds(dtype, v, n):
    from autognothi_amd import _lib as L
    lib = L.lib()
    x = 0x1000    # never read: every call below is refused on the host
    for rc in (lib.ag_token_logprobs(x, 0, n, v, dtype, 1.0, None, 0, None, x, x, x, None, None, None, 0, None),
               lib.ag_token_logprobs_bwd(x, 0, n, v, dtype, 1.0, x, x, None, None, None, None, 0, None, None, x, v, None),
               lib.ag_topk_distill(x, 0, n, v, dtype, 1.0, x, x, 0, 1, None, 0, x, x, x, x, v, None),
               lib.ag_topk_distill_bwd(x, 0, n, v, dtype, 1.0, x, x, 0, 1, None, 0, x, None, None, x, v, None)):
        assert rc < 0 and b"rows of" in lib.ag_last_error()
