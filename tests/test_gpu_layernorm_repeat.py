"""GPU: LayerNorm's weight gradients are sums in a fixed order: the same bits on every call."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h", [192, 768, 1024])
@pytest.mark.parametrize("rows", [1, 7, 197, 1576])
def test_layernorm_backward_repeats_bit_for_bit(cuda_device, rows, h):
    from autognothi_amd import ops
    gen = torch.Generator(cuda_device).manual_seed(rows + h)
    x, dy = (torch.randn(rows, h, device=cuda_device, generator=gen) for _ in range(2))
    gamma = torch.randn(h, device=cuda_device, generator=gen)
    first = None
    for _ in range(12):
        dg, db = torch.zeros(h, device=cuda_device), torch.zeros(h, device=cuda_device)
        dx = ops.layernorm_bwd(x, gamma, dy, 1e-12, dg, db)
        if first is None:
            first = (dx, dg, db)
            xh = torch.nn.functional.layer_norm(x.double(), (h,), eps=1e-12)
            # (a sum of `rows` products: each term a few roundings of 2^-24, the sum at most one more for every term)
            for got, terms in ((dg, dy.double() * xh), (db, dy.double())):
                assert ((got.double() - terms.sum(0)).abs() <= (rows + 16) * 2.0 ** -24 * terms.abs().sum(0) + (rows + 16) * 2.0 ** -24 * dy.double().abs().sum(0)).all()
        for a, b in zip(first, (dx, dg, db)):
            assert torch.equal(a, b)
