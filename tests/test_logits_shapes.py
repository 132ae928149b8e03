"""CPU: leading dimensions of the autograd forms over wide rows of logits."""
import pytest
import torch


def _int(*shape):
    return torch.zeros(shape, dtype=torch.int64)


@pytest.mark.parametrize("lead", [(), (1,), (6,), (2, 3), (0,), (2, 0)])
def test_leading_dimensions_as_documented_reach_the_operator(lead):
    """[..., V] with any leading dimensions, none among them (an operator on the CPU: the refusal comes from there)"""
    from autognothi_amd.models import distill
    z = torch.zeros(*lead, 11)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        distill.token_logprobs(z, _int(*lead), top_k=2)
    with pytest.raises(RuntimeError, match="no CPU fallback") if 0 not in lead else pytest.raises(ValueError, match="no rows"):
        distill.loss_topk_distillation(z, _int(*lead, 4), torch.zeros(*lead, 4), torch.zeros(lead))


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
