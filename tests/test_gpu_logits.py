"""GPU: the operators over wide rows of logits against their float64 restatement (oracle/logits.py).  Tolerances are that module's first-order
bounds on an fp32 evaluation; a bf16 gradient may be off by half a step more (2^-8 of its value)."""
import numpy as np
import pytest
import torch

from oracle import logits as ol

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
INF, LOWEST = float("inf"), {F32: torch.finfo(F32).min, BF16: torch.finfo(BF16).min}


def _logits(g, n, v, dtype, dev, sigma=3.0, pad=0, lead=0):
    """fp32 / bf16 [n, v] on the device, as a view into rows of v + pad (+ lead elements in front) when asked for, and as float64"""
    buf = torch.from_numpy((g.standard_normal((n, v + pad)) * sigma).astype(np.float32)).to(dtype)
    flat = torch.cat([torch.zeros(lead, dtype=dtype), buf.reshape(-1)]).to(dev)
    z = flat[lead:].view(n, v + pad)[:, :v]
    return z, buf[:, :v].double().numpy()


def _near(got, want, bound, what, rounded=False):
    got, want = got.double().cpu().numpy(), np.asarray(want, dtype=np.float64)
    assert got.shape == want.shape, what
    fin = np.isfinite(want)
    np.testing.assert_array_equal(np.isfinite(got), fin, err_msg=what)
    np.testing.assert_array_equal(got[~fin], want[~fin], err_msg=what)
    bound = np.broadcast_to(bound, want.shape)
    # bf16: half a step of the value, and of the smallest normal number below it
    tol = bound[fin] + (2.0 ** -8 * (np.abs(want[fin]) + bound[fin]) + 2.0 ** -134 if rounded else 2.0 ** -126)
    off = np.abs(got[fin] - want[fin])
    worst = np.argmax(off - tol) if off.size else 0
    assert off.size == 0 or (off <= tol).all(), f"{what}: {(off > tol).sum()} of {off.size} off, worst {off[worst]:.3g} against {tol[worst]:.3g}"


def _check_forward(z, z64, tokens, k, tau):
    from autognothi_amd import ops
    r = ops.token_logprobs(z, None if tokens is None else torch.from_numpy(tokens).to(z.device), k, tau)
    want = ol.token_logprobs(z64, tokens, k, tau)
    for name in ("logp", "entropy", "lse", "top_logp"):
        if name in want:
            _near(getattr(r, name), want[name], want["err_" + name], name)
    if k:
        np.testing.assert_array_equal(r.top_ids.cpu().numpy(), want["top_ids"])
    else:
        assert r.top_ids is None and r.top_logp is None
    return r


def _check_backward(z, z64, r, tokens, tau, g, with_top=True):
    from autognothi_amd import ops
    n = z.shape[0]
    gl, ge, gs = (g.standard_normal(n).astype(np.float32) for _ in range(3))
    k = 0 if r.top_ids is None or not with_top else r.top_ids.shape[1]
    gt = g.standard_normal((n, k)).astype(np.float32) if k else None
    dev = z.device
    t = lambda a: None if a is None else torch.from_numpy(a).to(dev)   # noqa: E731
    dz = ops.token_logprobs_bwd(z, r, t(tokens), None if tokens is None else t(gl), t(ge), t(gs), t(gt))
    assert dz.dtype == z.dtype and dz.is_contiguous()
    want, bound = ol.token_logprobs_grad(z64, tokens, r.top_ids.cpu().numpy() if k else None, tau, None if tokens is None else gl, ge, gs, gt)
    _near(dz, want, bound, "dlogits", rounded=z.dtype == BF16)


SHAPES = [(1, 1), (3, 2), (5, 3), (2, 7), (4, 8), (3, 10), (7, 63), (2, 64), (3, 65), (2, 100), (3, 127), (2, 128), (5, 257), (3, 511), (2, 512), (3, 1000),
          (2, 1025), (3, 2047), (2, 2049), (3, 4099), (2, 8191), (2, 16385), (3, 30522), (2, 50001), (2, 65537), (1, 131072), (2, 200003), (1, 262145),
          (1, 524288)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", SHAPES)
def test_token_logprobs(cuda_device, dtype, n, v):
    g = np.random.default_rng(1000 * n + v)
    tau = [1.0, 2.0, 0.7][v % 3]
    z, z64 = _logits(g, n, v, dtype, cuda_device)
    tokens = g.integers(0, v, n)
    tokens[n // 2] = -100
    for k in sorted({0, 1, min(v, 5), min(v, 128)}):
        r = _check_forward(z, z64, tokens, k, tau)
        _check_backward(z, z64, r, tokens, tau, g)
    _check_forward(z, z64, None, min(v, 3), tau)
    _check_backward(z, z64, r, None, tau, g, with_top=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [5, 1000, 30522])
@pytest.mark.parametrize("pad,lead", [(1, 0), (3, 1), (0, 1), (0, 3), (64, 7)])
def test_token_logprobs_any_stride_and_alignment(cuda_device, dtype, v, pad, lead):
    g = np.random.default_rng(v + 10 * pad + lead)
    z, z64 = _logits(g, 5, v, dtype, cuda_device, pad=pad, lead=lead)
    tokens = g.integers(0, v, 5)
    r = _check_forward(z, z64, tokens, min(5, v), 1.0)
    _check_backward(z, z64, r, tokens, 1.0, g)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_broadcast_and_transposed_rows(cuda_device, dtype):
    from autognothi_amd import ops
    g = np.random.default_rng(8)
    one, one64 = _logits(g, 1, 777, dtype, cuda_device)
    _check_forward(one.expand(6, 777), np.repeat(one64, 6, axis=0), g.integers(0, 777, 6), 4, 1.0)
    z, z64 = _logits(g, 300, 40, dtype, cuda_device)
    r = _check_forward(z.t(), z64.T, g.integers(0, 300, 40), 6, 1.5)
    _check_backward(z.t(), z64.T, r, g.integers(0, 300, 40), 1.5, g)
    r = ops.token_logprobs(z[:0], torch.zeros(0, dtype=torch.int64, device=cuda_device), 3)
    assert r.logp.shape == (0,) and r.top_ids.shape == (0, 3)
    assert ops.token_logprobs_bwd(z[:0], r, None, d_entropy=r.entropy).shape == (0, 40)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [12, 700, 3000, 40000, 140000, 263000])
def test_ties_go_to_the_lowest_index(cuda_device, dtype, v):
    g = np.random.default_rng(v)
    rows = np.stack([np.zeros(v), np.where(g.random(v) < 0.5, 0.0, -0.0), g.integers(-3, 4, v) * 0.5, np.round(g.standard_normal(v) * 2) / 2,
                     -np.arange(v) // 7 * 0.25, np.arange(v) // 3 * 0.125, np.where(np.arange(v) % 97 == 5, 4.0, -1.0)])
    z = torch.from_numpy(rows.astype(np.float32)).to(dtype)
    z64 = z.double().numpy()
    for k in sorted({1, min(v, 12), min(v, 100), min(v, 128)}):
        _check_forward(z.to(cuda_device), z64, g.integers(0, v, len(rows)), k, 1.0)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [6, 300, 2500, 33333, 270000])
def test_masked_and_degenerate_rows(cuda_device, dtype, v):
    """-inf among the logits, rows of nothing but -inf, masks of the type's lowest value, one survivor, far apart values"""
    g = np.random.default_rng(v + 1)
    low = LOWEST[dtype]
    n = 9
    z, _ = _logits(g, n, v, dtype, cuda_device)
    z = z.clone()
    z[0] = -INF
    z[1] = low
    z[2, v // 2:] = -INF
    z[3, v // 2:] = low
    z[4] = -INF
    z[4, v - 1] = 3.0
    z[5] = low
    z[5, 0] = 3.0
    z[6, : v // 3] = 60000.0        # a distribution over a third of the row, the rest nowhere
    z[7] = low / 2
    z[7, v // 2] = low / 4
    z[8, ::2] = -INF
    z[8, 1::4] = low
    z64 = z.double().cpu().numpy()
    tokens = np.full(n, v - 1)
    tokens[6] = 0
    for k in (0, min(v, 4), min(v, 128)):
        r = _check_forward(z, z64, tokens, k, 1.0)
        _check_backward(z, z64, r, tokens, 1.0, g)
    want = np.full(n, 0.0)
    tokens = np.full(n, -1)
    r = _check_forward(z, z64, tokens, 0, 2.0)
    assert np.array_equal(r.logp.cpu().numpy(), want)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [9, 400, 5000, 70000, 300000])
def test_nan_and_inf_stay_in_their_row(cuda_device, dtype, v):
    from autognothi_amd import ops
    g = np.random.default_rng(v + 2)
    z, z64 = _logits(g, 5, v, dtype, cuda_device)
    z[1, v // 2] = float("nan")
    z[3, 0] = INF
    z64 = z.double().cpu().numpy()
    tokens = torch.full((5,), v - 1, device=cuda_device)
    k = min(v, 7)
    r = ops.token_logprobs(z, tokens, k)
    bad = np.array([False, True, False, True, False])
    for t in (r.logp, r.entropy, r.lse):
        np.testing.assert_array_equal(np.isnan(t.cpu().numpy()), bad)
    np.testing.assert_array_equal(r.top_ids.cpu().numpy(), ol.top_ids(z64, k))
    ok = ~bad
    want = ol.token_logprobs(z64[ok], np.full(3, v - 1), k, 1.0)
    for name in ("logp", "entropy", "lse", "top_logp"):
        _near(getattr(r, name)[torch.from_numpy(ok)], want[name], want["err_" + name], name)
    dz = ops.token_logprobs_bwd(z, r, tokens, d_logp=torch.ones(5, device=cuda_device)).float().cpu().numpy()
    assert np.isnan(dz[bad]).any(axis=1).all() and np.isfinite(dz[ok]).all()


@pytest.mark.parametrize("tau", [1e-6, 1e-2, 100.0, 1e6])
def test_temperatures_far_from_one(cuda_device, tau):
    """x = z / tau reaches 1e7, where a product m / tau rounds to units and more, and 1e-5, where every row is nearly uniform"""
    g = np.random.default_rng(17)
    for n, v in ((4, 40), (3, 900), (3, 5000), (2, 40000)):
        z, z64 = _logits(g, n, v, F32, cuda_device)
        tokens = z64.argmax(axis=1)                       # (at 1e-6 every other token's probability is 0)
        tau32 = float(np.float32(tau))
        r = _check_forward(z, z64, tokens, 3, tau32)
        _check_backward(z, z64, r, tokens, tau32, g)
        if tau > 1e-3:
            ids, lp, lp64 = _teacher(g, n, v, 5, 0.8, False, F32)
            _check_distill(z, z64, ids, lp, lp64, tau32, True, None)


def test_tokens_outside_the_row_are_nan_and_read_nothing(cuda_device):
    from autognothi_amd import ops
    z = torch.randn(4, 50, device=cuda_device)
    tokens = torch.tensor([50, 1 << 40, -(1 << 40), 49], device=cuda_device)
    r = ops.token_logprobs(z, tokens)
    assert torch.isnan(r.logp[:2]).all() and r.logp[2] == 0 and torch.isfinite(r.logp[3])
    assert torch.isfinite(r.lse).all() and torch.isfinite(r.entropy).all()
    dz = ops.token_logprobs_bwd(z, r, tokens, d_logp=torch.ones(4, device=cuda_device))
    assert torch.isnan(dz[:2]).all() and (dz[2] == 0).all() and torch.isfinite(dz[3]).all()


# ------------------------------------------------------------------------------------------------ distillation
def _teacher(g, n, v, k, mass, ragged, dtype, dup=False):
    ids = np.stack([g.choice(v, k, replace=False) for _ in range(n)]).astype(np.int64)
    if dup and k > 1:
        ids[0, -1] = ids[0, 0]
        ids[n - 1, :] = ids[n - 1, 0]
    t = g.standard_normal((n, k)) * 2
    lp = t - np.log(np.exp(t).sum(axis=1, keepdims=True)) + np.log(mass)
    if ragged:
        ids[np.arange(k)[None, :] >= g.integers(1, k + 1, n)[:, None]] = -1
    lp = torch.from_numpy(lp.astype(np.float32)).to(dtype)
    return ids, lp, lp.double().numpy()


def _check_distill(z, z64, ids, lp, lp64, tau, tail, w):
    from autognothi_amd import ops
    dev = z.device
    n = z.shape[0]
    w64 = np.full(n, np.float32(1.0 / n), dtype=np.float64) if w is None else w.astype(np.float64)
    r = ops.topk_distill(z, torch.from_numpy(ids).to(dev), lp.to(dev), None if w is None else torch.from_numpy(w).to(dev), tau, tail)
    row, grad, e_row, e_grad = ol.distill(z64, ids, lp64, tau, tail, w64)
    _near(r.row_loss, row, e_row, "row_loss")
    part = w64 != 0
    _near(r.loss, [np.sum(row[part] * w64[part])], np.sum(e_row[part] * np.abs(w64[part])) + 2 * ol.U * np.abs(row[part] * w64[part]).sum(), "loss")
    _near(r.dlogits, grad, e_grad, "dlogits", rounded=z.dtype == BF16)
    only = ops.topk_distill(z, torch.from_numpy(ids).to(dev), lp.to(dev), None if w is None else torch.from_numpy(w).to(dev), tau, tail, want_grad=False)
    assert only.dlogits is None
    _near(only.row_loss, row, e_row, "row_loss (no gradient asked for)")
    g_loss, g_row = torch.tensor([1.5], device=dev), torch.linspace(-1, 1, n, device=dev)
    dz = ops.topk_distill_bwd(z, only, torch.from_numpy(ids).to(dev), lp.to(dev), None if w is None else torch.from_numpy(w).to(dev), tau, tail, g_loss, g_row)
    eff = np.where(part, 1.5 * w64 + g_row.double().cpu().numpy(), 0.0)
    at = np.where(part, 1.0, 0.0)
    _, unit, _, e_unit = ol.distill(z64, ids, lp64, tau, tail, at)
    _near(dz, unit * eff[:, None], e_unit * (np.abs(1.5 * w64) + 1.0)[:, None] * (1 + 4 * ol.U), "dlogits of the separate backward", rounded=z.dtype == BF16)
    return r


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("n,v", [s for s in SHAPES if s[1] > 1])
def test_topk_distill(cuda_device, dtype, tail, n, v):
    g = np.random.default_rng(77 * n + v + tail)
    tau = [1.0, 2.0, 0.7][v % 3]
    z, z64 = _logits(g, n, v, dtype, cuda_device)
    for k in sorted({1, min(v, 6), min(v, 128)}):
        for ragged, dup, tdt in ((False, False, F32), (True, True, BF16)):
            ids, lp, lp64 = _teacher(g, n, v, k, 0.8, ragged, tdt, dup)
            w = g.random(n).astype(np.float32) + 0.1
            w[n // 3] = 0.0 if n > 1 else w[n // 3]
            _check_distill(z, z64, ids, lp, lp64, tau, tail, w if ragged else None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("v,pad,lead", [(5, 3, 1), (999, 2, 0), (1000, 0, 1), (30522, 5, 3)])
def test_topk_distill_any_stride_and_alignment(cuda_device, dtype, tail, v, pad, lead):
    g = np.random.default_rng(v + pad)
    z, z64 = _logits(g, 4, v, dtype, cuda_device, pad=pad, lead=lead)
    ids, lp, lp64 = _teacher(g, 4, v, min(v, 20), 0.9, False, F32)
    _check_distill(z, z64, ids, lp, lp64, 1.0, tail, None)


@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("v", [4, 700, 20000])
def test_distill_edges(cuda_device, tail, v):
    """an empty list, the list of the whole vocabulary, masses of 0 and of 1, a student sure of itself, -inf and the lowest value in the student"""
    g = np.random.default_rng(v)
    k = 4
    n = 9
    z, _ = _logits(g, n, v, F32, cuda_device, sigma=2.0)
    ids, lp, _ = _teacher(g, n, v, k, 0.7, False, F32)
    lp = lp.clone()
    ids[0] = -1                                           # nothing listed
    lp[1] = -INF                                          # listed, of no mass
    lp[2] = torch.tensor([0.0, -INF, -INF, -INF])         # all the mass on one token
    lp[3] = torch.tensor([-1e-6, -15.0, -20.0, -30.0])    # a rest of about 7e-7
    z[4, int(ids[4, 0])] = 40.0                           # the student leaves e^-40 for everything else
    z[5, int(ids[5, 1])] = LOWEST[F32]                    # ... gives a listed token nothing
    lp[5, 1] = -INF
    z[6] = LOWEST[F32]                                    # ... is uniform
    off = np.setdiff1d(np.arange(v), ids[7])
    z[7, torch.from_numpy(off[: len(off) // 2]).to(z.device)] = -INF     # part of what is off the list is ruled out
    z[8] = -200.0
    z[8, int(ids[8, 0])] = 0.0                            # further apart than fp32 holds as a ratio
    _check_distill(z, z.double().cpu().numpy(), ids, lp, lp.double().numpy(), 1.0, tail, None)


@pytest.mark.parametrize("tail", [False, True])
def test_distill_infinite_rows(cuda_device, tail):
    """a student that rules out what the teacher has mass on: an infinite loss and no NaN in the gradient; rows of weight 0 may hold anything"""
    from autognothi_amd import ops
    v = 1500
    z = torch.randn(5, v, device=cuda_device)
    ids = torch.arange(8, device=cuda_device).repeat(5, 1) * 100
    lp = torch.log_softmax(torch.randn(5, 8, device=cuda_device), 1) + np.log(0.9)
    z[0, 100] = -INF
    z[1] = -INF
    z[2] = float("nan")
    w = torch.tensor([1.0, 1.0, 0.0, 1.0, 1.0], device=cuda_device)
    ids[2, 0] = v + 5
    ids[4, 3] = v
    r = ops.topk_distill(z, ids, lp, w, tail=tail)
    row = r.row_loss.cpu().numpy()
    assert row[0] == INF and row[1] == INF and row[2] == 0 and np.isfinite(row[3]) and np.isnan(row[4])
    d = r.dlogits.cpu().numpy()
    assert np.isfinite(d[:4]).all() and (d[1] == 0).all() and (d[2] == 0).all() and np.isnan(d[4]).all()
    assert d[0, 100] < 0


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_against_differences_of_the_kernels_own_loss(cuda_device, dtype):
    """<dL/dz, u> against (L(z + h u) - L(z - h u)) / 2h for a row u of +-1: the remainder is h^2 / 6 times a third cumulant of u, |.| <= 1 in all
    directions of one distribution and at most 2 here (p and the share off the list), the rounding of two losses about 1e-6 / 2h"""
    from autognothi_amd import ops
    g = np.random.default_rng(4)
    n, v, k, h = 4, 3001, 32, 2.0 ** -6
    z = torch.from_numpy((g.integers(-64, 64, (n, v)) / 16.0).astype(np.float32)).to(cuda_device)      # exact in bf16, and z +- h in fp32
    ids, lp, _ = _teacher(g, n, v, k, 0.8, False, F32)
    ids, lp = torch.from_numpy(ids).to(cuda_device), lp.to(cuda_device)
    u = torch.from_numpy(g.choice([-1.0, 1.0], (n, v)).astype(np.float32)).to(cuda_device)
    w = torch.ones(n, device=cuda_device)
    for tail in (False, True):
        f = lambda x: ops.topk_distill(x, ids, lp, w, 1.0, tail, want_grad=False).row_loss.double()   # noqa: E731
        got = (ops.topk_distill(z.to(dtype), ids, lp, w, 1.0, tail).dlogits.double() * u.double()).sum(dim=1)
        want = (f(z + h * u) - f(z - h * u)) / (2 * h)
        # (a bf16 gradient: half a step of every element, at worst all of one sign; sum |g| <= 2)
        assert float((got - want).abs().max()) <= 2 * h * h / 6 + 1e-6 * 8 / h + (2 * 2.0 ** -8 if dtype == BF16 else 0.0)
    tok = torch.from_numpy(g.integers(0, v, n)).to(cuda_device)
    fwd = ops.token_logprobs(z.to(dtype), tok)
    got = (ops.token_logprobs_bwd(z.to(dtype), fwd, tok, d_logp=w, d_entropy=0.5 * w).double() * u.double()).sum(dim=1)
    f = lambda x: (lambda r: r.logp.double() + 0.5 * r.entropy.double())(ops.token_logprobs(x, tok))   # noqa: E731
    want = (f(z + h * u) - f(z - h * u)) / (2 * h)
    # (the entropy's third derivative: cumulants weighted with |ln p| <= 16 here)
    assert float((got - want).abs().max()) <= 20 * h * h / 6 + 1e-6 * 16 / h + (8 * 2.0 ** -8 if dtype == BF16 else 0.0)


# ------------------------------------------------------------------------------------------------ as they are used together
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_record_a_teacher_and_train_on_the_record(cuda_device, dtype):
    """a student equal to its teacher has no loss and no gradient left; another student's loss and gradient are the full distributions' when the
    whole vocabulary is recorded"""
    from autognothi_amd import ops
    from autognothi_amd.models import distill
    g = np.random.default_rng(21)
    b, t, v, k, tau = 2, 5, 5000, 64, 2.0
    teacher = torch.from_numpy((g.standard_normal((b, t, v)) * 3).astype(np.float32)).to(dtype).to(cuda_device)
    rec = distill.token_logprobs(teacher, top_k=k, temperature=tau)
    assert rec.logp is None and rec.top_ids.shape == (b, t, k)
    same = teacher.clone().requires_grad_(True)
    loss, row = distill.loss_topk_distillation(same, rec.top_ids, rec.top_logp, temperature=tau, tail=True)
    loss.backward()
    assert row.shape == (b, t) and same.grad.shape == same.shape and same.grad.dtype == dtype
    z64 = teacher.double().cpu().numpy().reshape(b * t, v)
    ids, lp = rec.top_ids.cpu().numpy().reshape(-1, k), rec.top_logp.double().cpu().numpy().reshape(-1, k)
    w = np.full(b * t, np.float32(1.0 / (b * t)), dtype=np.float64)
    _, _, e_row, e_grad = ol.distill(z64, ids, lp, tau, True, w)
    # the record itself is fp32: its error enters the loss through q (ln q - ln p), of first order zero at q = p, and the gradient through q
    err = ol.token_logprobs(z64, None, k, tau)["err_top_logp"].max()
    assert float(row.detach().abs().max()) <= float(e_row.max()) + tau ** 2 * 2 * err
    extra = tau * w[0] * 4 * err
    assert float((same.grad.double().cpu().numpy().reshape(b * t, v).__abs__() - e_grad).max()) <= extra
    # whole vocabulary
    v = 100
    teacher, student = (torch.randn(6, v, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(s)) for s in (1, 2))
    rec = ops.token_logprobs(teacher, top_k=v)
    for tail in (False, True):
        r = ops.topk_distill(student, rec.top_ids, rec.top_logp, tail=tail)
        p, lq = torch.log_softmax(teacher.double(), 1).exp(), torch.log_softmax(teacher.double(), 1)
        kl = (p * (lq - torch.log_softmax(student.double(), 1))).sum(dim=1)
        np.testing.assert_allclose(r.row_loss.cpu().numpy(), kl.cpu().numpy(), atol=200 * 8 * ol.U)    # 100 terms of size <= 1, 8 roundings each
        want = (torch.softmax(student.double(), 1) - p) / 6
        np.testing.assert_allclose(r.dlogits.cpu().numpy(), want.cpu().numpy(), atol=200 * ol.U)


def test_autograd_of_the_log_probabilities(cuda_device):
    from autognothi_amd.models import distill
    g = np.random.default_rng(31)
    z, z64 = _logits(g, 6, 2222, F32, cuda_device)
    z = z.clone().requires_grad_(True)
    tokens = torch.from_numpy(g.integers(0, 2222, 6)).to(cuda_device)
    r = distill.token_logprobs(z.view(2, 3, 2222), tokens.view(2, 3), top_k=3, temperature=1.5)
    assert r.logp.shape == (2, 3) and not r.top_ids.requires_grad
    (-r.logp.mean() + 0.1 * r.entropy.sum() + 0.01 * (r.lse ** 2).sum() + r.top_logp[..., 1].sum()).backward()
    gt = np.zeros((6, 3))
    gt[:, 1] = 1.0
    lse = r.lse.detach().double().cpu().numpy().reshape(-1)
    want, bound = ol.token_logprobs_grad(z64, tokens.cpu().numpy(), r.top_ids.cpu().numpy().reshape(6, 3), 1.5, np.full(6, -1 / 6), np.full(6, 0.1), 0.02 * lse, gt)
    _near(z.grad, want, bound + 8 * ol.U * np.abs(want), "z.grad")
    z.grad = None
    distill.token_logprobs(z, tokens).logp.sum().backward()                  # one output used
    want, bound = ol.token_logprobs_grad(z64, tokens.cpu().numpy(), None, 1.0, np.ones(6))
    _near(z.grad, want, bound, "z.grad")
    with torch.no_grad():
        assert not distill.token_logprobs(z, tokens).logp.requires_grad


@pytest.mark.parametrize("v", [40, 1500, 30522, 270000])
def test_captured_replayed_and_repeated(cuda_device, v):
    """one graph of record -> distil -> gradient, replayed on new contents with eager work between; two graphs on two streams; the same bits"""
    from autognothi_amd import ops
    n, k = 37, 16
    gen = torch.Generator(cuda_device).manual_seed(v)
    zt, zs = (torch.randn(n, v, device=cuda_device, generator=gen) for _ in range(2))
    tokens = torch.randint(0, v, (n,), device=cuda_device, generator=gen)

    def step(a, b):
        rec = ops.token_logprobs(a, tokens, k)
        d = ops.topk_distill(b, rec.top_ids, rec.top_logp, tail=True)
        f = ops.token_logprobs(b, tokens)
        return rec.logp, rec.top_ids, d.loss, d.row_loss, d.dlogits, ops.token_logprobs_bwd(b, f, tokens, d_logp=rec.logp, d_entropy=rec.entropy)

    step(zt, zs)
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        a, b = zt.clone(), zs.clone()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(a, b)
        graphs.append((g, a, b, out))
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for it in range(4):
        news = [[torch.randn(n, v, device=cuda_device, generator=gen) for _ in range(2)] for _ in graphs]
        want = [[t.clone() for t in step(*new)] for new in news]
        for (g, a, b, _), new in zip(graphs, news):
            a.copy_(new[0])
            b.copy_(new[1])
        torch.cuda.synchronize()
        for (g, *_), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), w in zip(graphs, want):
            for x, y in zip(out, w):
                assert torch.equal(x, y)


def test_captured_autograd(cuda_device):
    """loss and gradient of the autograd forms in one graph, replayed on new logits with eager work between"""
    from autognothi_amd import ops
    from autognothi_amd.models import distill
    n, v, k = 9, 5000, 12
    gen = torch.Generator(cuda_device).manual_seed(1)
    z = torch.randn(n, v, device=cuda_device, generator=gen).requires_grad_(True)
    tokens = torch.randint(0, v, (n,), device=cuda_device, generator=gen)
    rec = ops.token_logprobs(torch.randn(n, v, device=cuda_device, generator=gen), top_k=k)

    def step(x):
        loss, _ = distill.loss_topk_distillation(x, rec.top_ids, rec.top_logp, tail=True)
        total = loss - 0.1 * distill.token_logprobs(x, tokens).logp.mean()
        return total.detach(), torch.autograd.grad(total, x)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(z)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(z)
    for _ in range(3):
        new = torch.randn(n, v, device=cuda_device, generator=gen)
        want = [t.clone() for t in step(new.clone().requires_grad_(True))]
        with torch.no_grad():
            z.copy_(new)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        for x, y in zip(out, want):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [20, 1000, 9000])
def test_c_entries_write_their_rows_alone(cuda_device, dtype, v):
    """gradient rows further apart than they are long, and results one row short of their buffers: nothing else is touched"""
    from autognothi_amd import _lib as L, ops
    lib, n, k, ldd = L.lib(), 5, 4, v + 9
    T = L.AG_F32 if dtype == F32 else L.AG_BF16
    z = torch.randn(n, v, device=cuda_device).to(dtype)
    tok = torch.zeros(n, dtype=torch.int64, device=cuda_device)
    r = ops.token_logprobs(z, tok, k)
    ids = torch.full(((n + 1) * k,), 77, dtype=torch.int64, device=cuda_device)
    top, st = torch.full(((n + 1) * k,), 7.0, device=cuda_device), torch.full((5 * n + 1,), 7.0, device=cuda_device)
    a, s = st.data_ptr(), L.stream()
    L.check(lib.ag_token_logprobs(z.data_ptr(), v, n, v, T, 1.0, tok.data_ptr(), k, a, a + 4 * n, a + 8 * n, a + 12 * n, ids.data_ptr(), top.data_ptr(), None, 0, s))
    assert torch.equal(st[: 5 * n].view(5, n), r.stats) and st[-1] == 7 and (ids[n * k:] == 77).all() and (top[n * k:] == 7).all()
    want = ops.token_logprobs_bwd(z, r, tok, d_logp=torch.ones(n, device=cuda_device))
    g = torch.ones(n, device=cuda_device)
    d = torch.full((n, ldd), 7.0, device=cuda_device).to(dtype)
    L.check(lib.ag_token_logprobs_bwd(z.data_ptr(), v, n, v, T, 1.0, a + 12 * n, a + 4 * n, tok.data_ptr(), g.data_ptr(), None, None, 0, None, None,
                                      d.data_ptr(), ldd, s))
    assert torch.equal(d[:, :v], want) and (d[:, v:] == 7).all()
    lp = torch.log_softmax(torch.randn(n, k, device=cuda_device), 1)
    w = torch.tensor([1.0, 0.0, 0.5, 1.0, 0.0], device=cuda_device)
    row, loss = torch.full((n + 1,), 7.0, device=cuda_device), torch.full((2,), 7.0, device=cuda_device)
    for tail in (0, 1):
        want = ops.topk_distill(z, r.top_ids, lp, w, tail=bool(tail))
        d.fill_(7.0)
        L.check(lib.ag_topk_distill(z.data_ptr(), v, n, v, T, 1.0, r.top_ids.data_ptr(), lp.data_ptr(), 0, k, w.data_ptr(), tail, row.data_ptr(),
                                    loss.data_ptr(), None, d.data_ptr(), ldd, s))
        assert torch.equal(d[:, :v], want.dlogits) and (d[:, v:] == 7).all()
        assert torch.equal(row[:n], want.row_loss) and row[n] == 7 and torch.equal(loss[:1], want.loss) and loss[1] == 7


def test_other_streams_and_repeats_give_the_same_bits(cuda_device):
    from autognothi_amd import ops
    gen = torch.Generator(cuda_device).manual_seed(5)
    z = torch.randn(300, 20011, device=cuda_device, generator=gen).to(BF16)
    rec = ops.token_logprobs(z, top_k=50)
    rec.top_ids[::3, 20:30] = rec.top_ids[::3, 40:50]      # (tokens listed twice)
    base = ops.topk_distill(z, rec.top_ids, rec.top_logp, tail=True)
    torch.cuda.synchronize()
    for _ in range(3):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            again, rep = ops.topk_distill(z, rec.top_ids, rec.top_logp, tail=True), ops.token_logprobs(z, top_k=50)
            rep.top_ids[::3, 20:30] = rep.top_ids[::3, 40:50]
        s.synchronize()
        for x, y in zip((*again[:3], rep.top_ids, rep.top_logp, rep.lse), (*base[:3], rec.top_ids, rec.top_logp, rec.lse)):
            assert torch.equal(x, y)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_rows_beyond_32_bit_offsets(cuda_device, dtype):
    """rows 2^30 elements apart: the last one starts beyond 2^32 elements"""
    from autognothi_amd import ops
    n, v, ld = 6, 1001, 1 << 30
    buf = torch.empty((n - 1) * ld + v, dtype=dtype, device=cuda_device)
    z = torch.as_strided(buf, (n, v), (ld, 1))
    g = np.random.default_rng(0)
    src, z64 = _logits(g, n, v, dtype, cuda_device)
    z.copy_(src)
    tokens = g.integers(0, v, n)
    r = _check_forward(z, z64, tokens, 5, 1.0)
    _check_backward(z, z64, r, tokens, 1.0, g)
    ids, lp, lp64 = _teacher(g, n, v, 10, 0.8, False, F32)
    _check_distill(z, z64, ids, lp, lp64, 1.0, True, None)
    del buf, z


def test_gradient_offsets_beyond_32_bits(cuda_device):
    """more than 2^32 bytes of gradient: the last rows are those of a small call"""
    from autognothi_amd import ops
    n, v, k = 16500, 140000, 3
    z = torch.zeros((n, v), dtype=BF16, device=cuda_device)
    z[-2:] = torch.randn(2, v, device=cuda_device, generator=torch.Generator(cuda_device).manual_seed(3)).to(BF16)
    ids = torch.arange(k, device=cuda_device).repeat(n, 1) * 40000
    lp = torch.full((n, k), -1.5, device=cuda_device)
    w = torch.ones(n, device=cuda_device)
    big = ops.topk_distill(z, ids, lp, w, tail=True)
    small = ops.topk_distill(z[-2:], ids[-2:], lp[-2:], w[-2:], tail=True)
    assert torch.equal(big.dlogits[-2:], small.dlogits) and torch.equal(big.row_loss[-2:], small.row_loss)
    assert torch.equal(big.dlogits[0], big.dlogits[n // 2])
    f = ops.token_logprobs(z, ids[:, 1].contiguous(), 2)
    fs = ops.token_logprobs(z[-2:], ids[-2:, 1].contiguous(), 2)
    assert torch.equal(f.top_ids[-2:], fs.top_ids) and torch.equal(f.logp[-2:], fs.logp)


def test_refused_across_devices(cuda_device):
    from autognothi_amd import ops
    z = torch.zeros(2, 5, device=cuda_device)
    with pytest.raises(RuntimeError, match="the logits are on"):
        ops.token_logprobs(z, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="the logits are on"):
        ops.topk_distill(z, torch.zeros(2, 2, dtype=torch.int64, device=cuda_device), torch.zeros(2, 2))


# Calls of many rows take other threads per row than calls of few: some rows of each against the oracle, the others by the sums they enter.
MANY = [(4500, 40), (1100, 300), (1100, 700), (1100, 1500), (1100, 2040), (1100, 3000), (1100, 9000), (600, 3000), (300, 1000), (300, 3000), (300, 9000), (300, 20000),
        (200, 20000), (100, 40000), (128, 33000), (1300, 16000), (400, 33000)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,chunks", MANY)
def test_many_rows(cuda_device, dtype, n, chunks):
    from autognothi_amd import ops
    v = chunks * (4 if dtype == F32 else 8) + 3
    gen = torch.Generator(cuda_device).manual_seed(n + chunks)
    z = (torch.randn(n, v + 5, device=cuda_device, generator=gen) * 3.0).to(dtype)[:, :v]
    g = np.random.default_rng(n * chunks)
    pick = np.unique(np.concatenate([[0, n - 1], g.integers(0, n, 6)]))
    at = torch.from_numpy(pick).to(cuda_device)
    z64 = z[at].double().cpu().numpy()
    tokens = g.integers(0, v, n)
    tok = torch.from_numpy(tokens).to(cuda_device)
    tau = [1.0, 2.0, 0.7][chunks % 3]
    for k in (0, 7, 32, 128):
        r = ops.token_logprobs(z, tok, k, tau)
        want = ol.token_logprobs(z64, tokens[pick], k, tau)
        for name in ("logp", "entropy", "lse", "top_logp"):
            if name in want:
                _near(getattr(r, name)[at], want[name], want["err_" + name], name)
        assert torch.isfinite(r.lse).all() and torch.isfinite(r.entropy).all()
        if k:
            np.testing.assert_array_equal(r.top_ids[at].cpu().numpy(), want["top_ids"])
            assert (r.top_logp[:, 1:] <= r.top_logp[:, :-1]).all() and torch.equal(z.gather(1, r.top_ids).float().amax(1), z.float().amax(1))
    gl, ge = g.standard_normal(n).astype(np.float32), g.standard_normal(n).astype(np.float32)
    dz = ops.token_logprobs_bwd(z, r, tok, torch.from_numpy(gl).to(cuda_device), torch.from_numpy(ge).to(cuda_device))
    want, bound = ol.token_logprobs_grad(z64, tokens[pick], None, tau, gl[pick], ge[pick], None, None)
    _near(dz[at], want, bound, "dlogits", rounded=dtype == BF16)
    assert torch.isfinite(dz).all()
    k = [5, 50, 128][chunks % 3]
    ids, lp, lp64 = _teacher(g, n, v, k, 0.8, True, F32)
    w = g.random(n).astype(np.float32) / n
    w[g.integers(0, n, n // 5)] = 0.0
    args = (torch.from_numpy(ids).to(cuda_device), lp.to(cuda_device), torch.from_numpy(w).to(cuda_device), tau)
    for tail in (False, True):
        row, grad, e_row, e_grad = ol.distill(z64, ids[pick], lp64[pick], tau, tail, w[pick].astype(np.float64))
        r = ops.topk_distill(z, *args, tail)
        only = ops.topk_distill(z, *args, tail, want_grad=False)
        apart = ops.topk_distill_bwd(z, only, *args, tail)
        for a in (r, only):
            _near(a.row_loss[at], row, e_row, "row_loss")
            assert torch.isfinite(a.row_loss).all() and (a.row_loss[args[2] == 0] == 0).all()
            total = (a.row_loss.double() * args[2].double()).sum()
            assert abs(a.loss.double() - total) <= 2 ** -23 * total.abs()
        for d in (r.dlogits, apart):
            _near(d[at], grad, e_grad * (1 + 4 * ol.U), "dlogits", rounded=dtype == BF16)
            assert torch.isfinite(d).all() and not d[args[2] == 0].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("v", [9, 100, 1000])
def test_gradients_of_very_many_short_rows(cuda_device, dtype, v):
    """more logits than the chip's caches hold: the same bits as a call of the last rows alone"""
    from autognothi_amd import ops
    for mb in (200, 340):
        n = mb * 1000000 // (v * (4 if dtype == F32 else 2))
        gen = torch.Generator(cuda_device).manual_seed(v)
        z = torch.randn(n, v, device=cuda_device, generator=gen).to(dtype)
        tok = torch.randint(0, v, (n,), device=cuda_device, generator=gen)
        g = torch.randn(n, device=cuda_device, generator=gen)
        ids = torch.randint(0, v, (n, 4), device=cuda_device, generator=gen)
        lp = torch.log_softmax(torch.randn(n, 4, device=cuda_device, generator=gen), 1) - 0.3
        for sl in (slice(None), slice(n - 7, n)):
            f = ops.token_logprobs(z[sl], tok[sl])
            d = ops.token_logprobs_bwd(z[sl], f, tok[sl], g[sl], g[sl])
            t = ops.topk_distill(z[sl], ids[sl], lp[sl], g[sl], tail=True, want_grad=False)
            e = ops.topk_distill_bwd(z[sl], t, ids[sl], lp[sl], g[sl], tail=True)
            if sl.start is None:
                all_ = (f.logp[-7:], f.entropy[-7:], d[-7:], t.row_loss[-7:], e[-7:])
                assert torch.isfinite(d).all() and torch.isfinite(e).all()
            else:
                for a, b in zip(all_, (f.logp, f.entropy, d, t.row_loss, e)):
                    assert torch.equal(a, b)


@pytest.mark.parametrize("n,v", [(2, 300000), (40, 30522), (1500, 3000)])
def test_two_threads_on_two_streams(cuda_device, n, v):
    """calls at the same time share nothing: each thread's results are those of its calls alone"""
    import threading
    from autognothi_amd import ops
    made = []
    for seed in range(2):
        gen = torch.Generator(cuda_device).manual_seed(seed)
        z = torch.randn(n, v, device=cuda_device, generator=gen)
        ids = torch.randint(0, v, (n, 6), device=cuda_device, generator=gen)
        lp = torch.log_softmax(torch.randn(n, 6, device=cuda_device, generator=gen), 1) - 0.2
        made.append((z, ids, lp))

    def calls(z, ids, lp):
        f = ops.token_logprobs(z, ids[:, 0].contiguous(), 8)
        d = ops.topk_distill(z, ids, lp, tail=True)
        return [t.clone() for t in (f.logp, f.entropy, f.lse, f.top_ids, f.top_logp, ops.token_logprobs_bwd(z, f, ids[:, 0].contiguous(), f.lse, f.entropy),
                                    d.loss, d.row_loss, d.dlogits)]

    alone = [calls(*m) for m in made]
    torch.cuda.synchronize()
    failed = []

    def run(i):
        try:
            stream = torch.cuda.Stream(cuda_device)
            with torch.cuda.stream(stream):
                for _ in range(8):
                    got = calls(*made[i])
                    stream.synchronize()
                    for a, b in zip(got, alone[i]):
                        assert torch.equal(a, b)
        except BaseException as e:      # noqa: BLE001 (reported by the main thread)
            failed.append((i, e))

    threads = [threading.Thread(target=run, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed, failed
