"""CPU: leading dimensions of the autograd forms over wide rows of logits, the workspace query for calls that are refused, and the sizes at which a
call takes a workspace: the header's on both sides."""
import os
import re
import subprocess
import sys

import pytest
import torch


def _int(*shape):
    return torch.zeros(shape, dtype=torch.int64)


@pytest.mark.parametrize("logits,tokens", [((2, 3, 11), (3, 2)), ((2, 3, 11), (5,)), ((6, 11), (2, 3)), ((6, 11), (6, 1)), ((6, 11), (5,)), ((11,), (11,)),
                                           ((1, 11), ())])
def test_tokens_of_other_leading_dimensions_are_refused(logits, tokens):
    """[3, 2] tokens for [2, 3, V] logits are as many, but not the same ones"""
    from autognothi_amd.models import distill
    with pytest.raises(ValueError, match="token_logprobs: tokens must be"):
        distill.token_logprobs(torch.zeros(logits), _int(*tokens))


@pytest.mark.parametrize("flat", [False, True])
def test_one_dimension_for_all_rows_reaches_the_operator(flat):
    from autognothi_amd.models import distill
    lead = (6,) if flat else (2, 3)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        distill.token_logprobs(torch.zeros(2, 3, 11), _int(*lead))
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        distill.loss_topk_distillation(torch.zeros(2, 3, 11), _int(*lead, 4), torch.zeros(*lead, 4), torch.zeros(lead))


@pytest.mark.parametrize("logits,ids,logp,weights,what", [
    ((2, 3, 11), (3, 2, 4), (2, 3, 4), None, "teacher_ids"), ((2, 3, 11), (5, 4), (6, 4), None, "teacher_ids"), ((6, 11), (2, 3, 4), (2, 3, 4), None, "teacher_ids"),
    ((2, 3, 11), (2, 3, 4), (3, 2, 4), None, "teacher_logp"), ((2, 3, 11), (2, 3, 4), (2, 3, 5), None, "teacher_logp"), ((2, 3, 11), (2, 3, 4), (2, 3, 4), (3, 2), "weights"),
    ((2, 3, 11), (2, 3, 4), (2, 3, 4), (5,), "weights"), ((6, 11), (6, 4), (6, 4), (6, 1), "weights"), ((11,), (2, 4), (2, 4), None, "teacher_ids"),
    ((11,), (4,), (4,), (2,), "weights"), ((6, 11), (), (6, 4), None, "teacher_ids")])
def test_a_record_of_other_leading_dimensions_is_refused(logits, ids, logp, weights, what):
    from autognothi_amd.models import distill
    with pytest.raises(ValueError, match=f"{what} must be"):
        distill.loss_topk_distillation(torch.zeros(logits), _int(*ids), torch.zeros(logp), None if weights is None else torch.zeros(weights))


def test_a_number_is_no_row_of_logits():
    from autognothi_amd.models import distill
    with pytest.raises(ValueError, match="logits must be"):
        distill.token_logprobs(torch.zeros(()))
    with pytest.raises(ValueError, match="logits must be"):
        distill.loss_topk_distillation(torch.zeros(()), _int(4), torch.zeros(4))


@pytest.mark.parametrize("lead", [(), (1,), (6,), (2, 3), (0,), (2, 0)])
def test_leading_dimensions_as_documented_reach_the_operator(lead):
    """[..., V] with any leading dimensions, none among them (an operator on the CPU: the refusal comes from there)"""
    from autognothi_amd.models import distill
    z = torch.zeros(*lead, 11)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        distill.token_logprobs(z, _int(*lead), top_k=2)
    with pytest.raises(RuntimeError, match="no CPU fallback") if 0 not in lead else pytest.raises(ValueError, match="no rows"):
        distill.loss_topk_distillation(z, _int(*lead, 4), torch.zeros(*lead, 4), torch.zeros(lead))
    if 0 not in lead:
        with pytest.raises(ValueError, match="teacher_ids must be"):
            distill.loss_topk_distillation(z, _int(*lead, 0), torch.zeros(*lead, 0))


def test_results_get_the_leading_dimensions_back(monkeypatch):
    from autognothi_amd import ops
    from autognothi_amd.models import distill

    def forward(logits, tokens, top_k, temperature, no_views):
        assert logits.dim() == 2 and tokens.shape == logits.shape[:1]
        n = logits.shape[0]
        return ops.TokenLogprobs(*(torch.zeros(n) for _ in range(3)), _int(n, top_k), torch.zeros(n, top_k), torch.zeros(5, n), temperature)

    monkeypatch.setattr(ops, "_token_logprobs", forward)
    for lead in ((), (1,), (6,), (2, 3), (2, 1, 3)):
        r = distill.token_logprobs(torch.zeros(*lead, 11), _int(*lead), top_k=2)
        assert r.logp.shape == r.entropy.shape == r.lse.shape == lead and r.top_ids.shape == r.top_logp.shape == (*lead, 2)


def test_workspace_of_a_refused_call_is_nothing():
    """(in a process of its own: a division by zero at a C entry ends it)"""
    code = """
from autognothi_amd import _lib as L
f = L.lib().ag_token_logprobs_workspace_bytes
assert f(1, 200000, 0, 4) > 0
for n in (-5, 0, 1, 100, 2 ** 31 - 1):
    for v in (-2 ** 31, -1, 0, 1, 200000, L.AG_LOGITS_MAX_V + 1, 2 ** 31 - 1):
        for k in (-2 ** 31, -1000, -257, -2, -1, 0, 1, 129, 2 ** 31 - 1):
            for dtype in (L.AG_F32, L.AG_BF16, 2, -1):
                if n < 0 or not 1 <= v <= L.AG_LOGITS_MAX_V or not 0 <= k <= min(v, L.AG_LOGITS_MAX_TOP) or dtype not in (L.AG_F32, L.AG_BF16):
                    assert f(n, v, dtype, k) == 0, (n, v, dtype, k)
"""
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, (r.returncode, r.stderr[-2000:])


def test_sizes_of_the_header_and_of_the_binding_agree():
    from autognothi_amd import _lib as L
    header = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "autognothi_hip.h")
    found = dict(re.findall(r"^#define (AG_LOGITS_\w+) (\d+)$", open(header).read(), flags=re.M))
    assert len(found) == 6
    for name, value in found.items():
        assert getattr(L, name) == int(value), name


def test_no_workspace_below_the_sizes_at_which_it_is_asked_for():
    from autognothi_amd import _lib as L, ops
    f = L.lib().ag_token_logprobs_workspace_bytes
    for dtype, e in ((L.AG_F32, 4), (L.AG_BF16, 8)):
        least = L.AG_LOGITS_SHARED_PIECES * e
        for k in (0, 1, 32):
            assert f(1, least, dtype, k) > 0 and f(L.AG_LOGITS_SHARED_ROWS, least, dtype, k) > 0
            assert f(1, least - 1, dtype, k) == 0 and f(L.AG_LOGITS_SHARED_ROWS + 1, least, dtype, k) == 0
        assert ops._pieces(least, dtype) == L.AG_LOGITS_SHARED_PIECES == ops._pieces(least - 1, dtype) + 1


def test_c_entry_with_a_saved_entropy_refuses_before_any_launch():
    from autognothi_amd import _lib as L
    lib = L.lib()
    x = 0x1000    # never read: every call below is refused on the host

    def call(n=1, v=8, dtype=0, k=0, z=x, ent=x, stats=x, saved=x, ws=None, have=0):
        return lib.ag_token_logprobs_saved(z, 8, n, v, dtype, 1.0, None, k, None, ent, x, stats, saved, None, None, ws, have, None)

    for rc in (call(saved=None), call(stats=None), call(ent=None), call(z=None), call(n=-1), call(v=0), call(dtype=2), call(k=2), call(k=9), call(ws=x + 4)):
        assert rc < 0 and b"ag_token_logprobs_saved" in lib.ag_last_error()
    assert call(n=0, saved=None) == 0
