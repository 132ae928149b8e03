"""GPU: calls over rows of logits that the documentation allows and that no size or mask of the other tests makes: lists longer than the row, rows that all
take no part, one token, the widest rows among many, an edited list of alternatives."""
import numpy as np
import pytest
import torch

from oracle import logits as ol

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16


def _near(got, want, bound, what, half=0.0):
    off = (got.double().cpu().numpy() - want)
    assert (np.abs(off) <= bound + half * (np.abs(want) + bound) + 2.0 ** -126).all(), (what, np.abs(off).max())


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("tail", [False, True])
@pytest.mark.parametrize("v", [1, 2, 3, 17, 64, 65, 100, 127])
def test_lists_longer_than_the_row(cuda_device, dtype, tail, v):
    """128 slots for v tokens: most of them listed several times, some slots empty; in one row every slot names the same token"""
    from autognothi_amd import ops
    g = np.random.default_rng(v)
    n, k = 7, 128
    z = torch.from_numpy((g.standard_normal((n, v)) * 2).astype(np.float32)).to(dtype).to(cuda_device)
    ids = g.integers(0, v, (n, k))
    ids[g.random((n, k)) < 0.2] = -1
    ids[3] = v - 1
    ids[4, 1:] = -1
    t = g.standard_normal((n, k))
    lp = (t - np.log(np.exp(t).sum(axis=1, keepdims=True)) + np.log(0.7)).astype(np.float32)
    w = (g.random(n) + 0.1).astype(np.float32)
    dev = lambda a: torch.from_numpy(a).to(cuda_device)   # noqa: E731
    row, grad, e_row, e_grad = ol.distill(z.double().cpu().numpy(), ids, lp.astype(np.float64), 1.5, tail, w.astype(np.float64))
    one = ops.topk_distill(z, dev(ids), dev(lp), dev(w), 1.5, tail)
    apart = ops.topk_distill(z, dev(ids), dev(lp), dev(w), 1.5, tail, want_grad=False)
    d = ops.topk_distill_bwd(z, apart, dev(ids), dev(lp), dev(w), 1.5, tail)
    half = 2.0 ** -8 if dtype == BF16 else 0.0
    # (a token's mass is a sum over its slots: each of them to (2 k + 32) roundings)
    for a in (one, apart):
        _near(a.row_loss, row, e_row + 2.25 * 2 * k * ol.U, "row loss")
    scale = (1.5 * w)[:, None]
    for a in (one.dlogits, d):
        _near(a, grad, e_grad + scale * 2 * k * ol.U, "gradient", half)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(5, 40), (5, 1000), (700, 3001), (4, 270000)])
def test_no_row_takes_part(cuda_device, dtype, n, v):
    """weights that are all 0: loss 0, gradient 0, whatever the rows hold"""
    from autognothi_amd import ops
    z = torch.full((n, v), float("nan"), dtype=dtype, device=cuda_device)
    ids = torch.full((n, 3), v + 1, device=cuda_device)
    lp, w = torch.full((n, 3), float("nan"), device=cuda_device), torch.zeros(n, device=cuda_device)
    w[1] = -0.0
    for tail in (False, True):
        one = ops.topk_distill(z, ids, lp, w, tail=tail)
        apart = ops.topk_distill(z, ids, lp, w, tail=tail, want_grad=False)
        d = ops.topk_distill_bwd(z, apart, ids, lp, w, tail=tail, d_row_loss=torch.ones(n, device=cuda_device))
        for t in (one.loss, one.row_loss, one.dlogits, apart.loss, apart.row_loss, d):
            assert not t.any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_token(cuda_device, dtype):
    """V = 1: p = 1 whatever the logit"""
    from autognothi_amd import ops
    z = torch.tensor([[0.0], [-3.0], [60000.0], [-torch.inf]], device=cuda_device).to(dtype)
    tokens = torch.tensor([0, 0, -1, 0], device=cuda_device)
    r = ops.token_logprobs(z, tokens, 1, 2.0)
    assert r.logp.tolist() == [0.0, 0.0, 0.0, -np.inf] and r.entropy.tolist() == [0.0] * 4 and not r.top_ids.any()
    assert r.top_logp[:, 0].tolist() == [0.0, 0.0, 0.0, -np.inf]
    g = torch.ones(4, device=cuda_device)
    # (1 - p) (g_t + g_1) / 2: two products of size 1, p an exponential and its inverse reference, a handful of roundings of 2^-24 each
    assert ops.token_logprobs_bwd(z, r, tokens, g, g, None, g[:, None]).abs().max() <= 8 * 2.0 ** -24
    d = ops.topk_distill(z[:3], torch.zeros(3, 1, dtype=torch.int64, device=cuda_device), torch.full((3, 1), -0.5, device=cuda_device), tail=True)
    assert torch.isfinite(d.row_loss).all() and d.dlogits.abs().max() <= 8 * 2.0 ** -24      # (q (p - 1) / 3)


@pytest.mark.parametrize("n,v", [(6, 700), (600, 20000)])
def test_alternatives_taken_out_of_the_list_pass_no_gradient_through_it(cuda_device, n, v):
    """top_ids belongs to the caller and is what the backward reads: a slot set to -1 (or beyond the row) adds nothing to its token"""
    from autognothi_amd import ops
    gen = torch.Generator(cuda_device).manual_seed(0)
    z = torch.randn(n, v, device=cuda_device, generator=gen) * 3.0
    r = ops.token_logprobs(z, top_k=4)
    ids = r.top_ids.clone()
    gt = torch.ones(n, 4, device=cuda_device)
    full = ops.token_logprobs_bwd(z, r, d_top_logp=gt)
    r.top_ids[:, 2] = -1
    r.top_ids[:, 3] = v
    cut = ops.token_logprobs_bwd(z, r, d_top_logp=gt)
    assert torch.isfinite(cut).all()
    rows = torch.arange(n, device=cuda_device)
    for j in (0, 1):
        assert torch.equal(cut[rows, ids[:, j]], full[rows, ids[:, j]])
    for j in (2, 3):      # (one() of them lost: the gradient of the normaliser alone, 4 p below 0)
        assert (cut[rows, ids[:, j]] < 0).all() and (full[rows, ids[:, j]] - cut[rows, ids[:, j]] - 1.0).abs().max() <= 8 * 2.0 ** -24
