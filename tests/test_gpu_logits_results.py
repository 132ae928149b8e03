"""GPU: what the operators over wide rows of logits hand out belongs to the caller: editing a result in place changes no gradient and no other
result, here as with elementary torch operations; and the results keep the signs that the definitions give them."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def _made(dev, n, v, seed=0):
    gen = torch.Generator(dev).manual_seed(seed)
    z = torch.randn(n, v, device=dev, generator=gen) * 3.0
    tokens = torch.randint(0, v, (n,), device=dev, generator=gen)
    return z, tokens, torch.randn(n, device=dev, generator=gen)


# (16 lanes a row, one wave, a workgroup, several workgroups a row)
SIZES = [(6, 40), (6, 700), (600, 20000), (3, 270000)]


@pytest.mark.parametrize("n,v", SIZES)
@pytest.mark.parametrize("edited", ["logp", "entropy", "lse", "top_logp"])
def test_a_result_edited_before_the_backward_changes_no_gradient(cuda_device, n, v, edited):
    from autognothi_amd import ops
    z, tokens, g = _made(cuda_device, n, v)
    r = ops.token_logprobs(z, tokens, 3)
    gt = torch.ones(n, 3, device=cuda_device)
    want = ops.token_logprobs_bwd(z, r, tokens, g, g, g, gt)
    others = {f: getattr(r, f).clone() for f in ("logp", "entropy", "lse", "top_ids", "top_logp") if f != edited}
    getattr(r, edited).mul_(-0.25).add_(7.0)
    assert torch.equal(ops.token_logprobs_bwd(z, r, tokens, g, g, g, gt), want)
    for f, t in others.items():
        assert torch.equal(getattr(r, f), t), f


@pytest.mark.parametrize("n,v", SIZES)
def test_stats_hold_what_the_results_do(cuda_device, n, v):
    from autognothi_amd import ops
    z, tokens, _ = _made(cuda_device, n, v)
    r = ops.token_logprobs(z, tokens, 2)
    assert r.stats.shape == (5, n)
    for row, t in zip(r.stats, (r.logp, r.entropy, r.lse)):
        assert torch.equal(row, t)
    none = ops.token_logprobs(z, top_k=2)
    assert none.logp is None and torch.equal(none.stats[1:], r.stats[1:])


@pytest.mark.parametrize("n,v", SIZES)
def test_c_entry_with_a_saved_entropy_writes_its_rows_alone(cuda_device, n, v):
    """the results of ag_token_logprobs, the entropy twice, and nothing behind any of them"""
    from autognothi_amd import _lib as L, ops
    z, tokens, g = _made(cuda_device, n, v)
    k = 3
    r = ops.token_logprobs(z, tokens, k)
    logp, entropy, lse, saved = (torch.full((n + 1,), 7.0, device=cuda_device) for _ in range(4))
    stats, top = torch.full((2 * n + 1,), 7.0, device=cuda_device), torch.full((n * k + 1,), 7.0, device=cuda_device)
    ids = torch.full((n * k + 1,), 77, dtype=torch.int64, device=cuda_device)
    need = L.lib().ag_token_logprobs_workspace_bytes(n, v, L.AG_F32, k)
    ws = torch.empty(max(need, 1), dtype=torch.uint8, device=cuda_device)
    L.check(L.lib().ag_token_logprobs_saved(z.data_ptr(), v, n, v, L.AG_F32, 1.0, tokens.data_ptr(), k, logp.data_ptr(), entropy.data_ptr(), lse.data_ptr(),
                                            stats.data_ptr(), saved.data_ptr(), ids.data_ptr(), top.data_ptr(), ws.data_ptr() if need else None, need, L.stream()))
    for got, want in ((logp, r.logp), (entropy, r.entropy), (lse, r.lse), (saved, r.entropy), (stats, r.stats[3:].reshape(-1)), (top, r.top_logp.reshape(-1)),
                      (ids, r.top_ids.reshape(-1))):
        assert torch.equal(got[:-1], want) and float(got[-1]) in (7.0, 77.0)


def _edit(t):
    t.mul_(2.0)
    t += 1.0


def _same(t):
    return t * 2.0 + 1.0


@pytest.mark.parametrize("shape", [(6, 700), (2, 3, 700)])
@pytest.mark.parametrize("which", ["logp", "entropy", "lse", "top_logp"])
def test_autograd_outputs_can_be_edited_in_place(cuda_device, shape, which):
    """out.mul_(w) of any output: the gradient of the edited graph, and of the other outputs what it was"""
    from autognothi_amd.models import distill
    z, tokens, _ = _made(cuda_device, 6, 700)
    z, tokens = z.view(shape), tokens.view(shape[:-1])
    grads = []
    for edit in (False, True):
        x = z.clone().requires_grad_(True)
        r = distill.token_logprobs(x, tokens, top_k=3)
        out = getattr(r, which)
        if edit:
            _edit(out)
        else:
            out = _same(out)
        total = (out ** 2).sum() + sum(getattr(r, f).sum() for f in ("logp", "entropy", "lse", "top_logp") if f != which)
        grads.append((total.detach(), *torch.autograd.grad(total, x)))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("which", ["logp", "entropy", "lse", "top_logp"])
def test_autograd_outputs_edited_behind_the_graph(cuda_device, which):
    """an edit through detach() leaves the gradients as they were, and the other outputs usable"""
    from autognothi_amd.models import distill
    z, tokens, _ = _made(cuda_device, 6, 700)
    x = z.clone().requires_grad_(True)
    grads = []
    for edit in (False, True):
        r = distill.token_logprobs(x, tokens, top_k=3)
        if edit:
            getattr(r, which).detach().mul_(-3.0)
        grads.append(torch.autograd.grad(sum(getattr(r, f).sum() for f in ("logp", "entropy", "lse", "top_logp")), x)[0])
    assert torch.equal(*grads)


@pytest.mark.parametrize("shape", [(6, 700), (2, 3, 700)])
def test_autograd_loss_can_be_edited_in_place(cuda_device, shape):
    """loss += ..., loss.div_(steps) and row.mul_(...): as with any loss"""
    from autognothi_amd import ops
    from autognothi_amd.models import distill
    z, _, _ = _made(cuda_device, 6, 700)
    rec = ops.token_logprobs(_made(cuda_device, 6, 700, seed=1)[0], top_k=5)
    ids, lp = rec.top_ids.view(*shape[:-1], 5), rec.top_logp.view(*shape[:-1], 5)
    grads = []
    for edit in (False, True):
        x = z.view(shape).clone().requires_grad_(True)
        loss, row = distill.loss_topk_distillation(x, ids, lp, tail=True)
        assert loss.shape == () and row.shape == shape[:-1]
        if edit:
            loss += row.sum()
            loss.div_(4.0)
            _edit(row)
        else:
            loss = (loss + row.sum()) / 4.0
            row = _same(row)
        total = loss + (row ** 2).sum()
        grads.append((total.detach(), *torch.autograd.grad(total, x)))
    for a, b in zip(*grads):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_one_row_without_leading_dimensions(cuda_device, dtype):
    """logits [V]: the numbers of the call with one row, in forward and backward"""
    from autognothi_amd.models import distill
    z, tokens, _ = _made(cuda_device, 1, 1234)
    z = z.to(dtype)
    got = []
    for shape in ((1234,), (1, 1234)):
        x = z.view(shape).clone().requires_grad_(True)
        r = distill.token_logprobs(x, tokens.view(shape[:-1]), top_k=4, temperature=2.0)
        assert r.logp.shape == r.entropy.shape == r.lse.shape == shape[:-1] and r.top_ids.shape == r.top_logp.shape == (*shape[:-1], 4)
        loss, row = distill.loss_topk_distillation(x, r.top_ids, r.top_logp.detach() - 0.25, torch.ones(shape[:-1], device=cuda_device), tail=True)
        assert loss.shape == () and row.shape == shape[:-1]
        total = loss + row.sum() + r.logp.sum() + r.entropy.sum() + r.lse.sum() + r.top_logp.sum()
        got.append([t.detach().reshape(-1) for t in (r.logp, r.entropy, r.lse, r.top_ids, r.top_logp, loss, row, *torch.autograd.grad(total, x))])
    for a, b in zip(*got):
        assert torch.equal(a, b)
    assert distill.token_logprobs(z[0]).lse.shape == ()


# ------------------------------------------------------------------------------------------------ signs
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("n,v", [(4000, 40), (4000, 100), (4000, 700), (4000, 5000), (1500, 30522), (600, 70000), (100, 140000)])
def test_no_probability_above_one_and_no_entropy_below_zero(cuda_device, dtype, n, v):
    """rows that are sure of one token: ln p <= 0 and H >= 0 in every bit, and within the bounds of the sums' rounding"""
    from autognothi_amd import ops
    gen = torch.Generator(cuda_device).manual_seed(v)
    z = (torch.randn(n, v, device=cuda_device, generator=gen) * 3.0).to(dtype)
    at = torch.randint(0, v, (n, 1), device=cuda_device, generator=gen)
    z.scatter_(1, at, (torch.rand(n, 1, device=cuda_device, generator=gen) * 200.0 + 30.0).to(dtype))
    for tau in (1.0, 0.7):
        for k in (0, 3):
            r = ops.token_logprobs(z, at[:, 0].contiguous(), k, tau)
            assert (r.logp <= 0).all() and (r.entropy >= 0).all()
            # the token stands at least 10 / 0.7 above the others: s is 1 + v e^-10 at most and every further number a few roundings of it
            x = z.double() / float(np.float32(tau))
            lse = torch.logsumexp(x, 1)
            logp = x.gather(1, at)[:, 0] - lse
            p = (x - lse[:, None]).exp()
            ent = -(p * (x - lse[:, None])).sum(1)
            # (the sums' relative error: chains of at most 32 chunks a lane and the joins; with |y| <= 400 for every term but the largest)
            rel = (128 + 800 * (1 - p.amax(1))) * U
            assert ((r.logp.double() - logp).abs() <= rel).all()
            assert ((r.entropy.double() - ent).abs() <= 8 * rel + 512 * U * ent).all()
            if k:
                assert (r.top_logp <= 0).all() and torch.equal(r.top_ids[:, 0], at[:, 0]) and torch.equal(r.top_logp[:, 0], r.logp)
