"""GPU: LayerNorm's weight gradients repeat bit for bit at every width, those included whose rows are not held in registers."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("h", [1, 33, 96, 384, 512, 1000, 1536, 4096])
@pytest.mark.parametrize("rows", [1, 2, 7, 197, 1576, 9001])
@pytest.mark.parametrize("plain", [False, True])
def test_layernorm_backward_of_any_width_repeats(cuda_device, rows, h, plain):
    """plain: no gamma, no added gradient.  Against the formula in 64 bits, every sum to one rounding per term"""
    from autognothi_amd import ops
    gen = torch.Generator(cuda_device).manual_seed(rows + h)
    x, dy, add = (torch.randn(rows, h, device=cuda_device, generator=gen) for _ in range(3))
    gamma = None if plain else torch.randn(h, device=cuda_device, generator=gen)
    add = None if plain else add
    eps, u = 1e-5, 2.0 ** -24
    first = None
    for _ in range(8):
        dg, db = torch.zeros(h, device=cuda_device), torch.zeros(h, device=cuda_device)
        dx = ops.layernorm_bwd(x, gamma, dy, eps, dg, db, add=add)
        if first is None:
            first = (dx, dg, db)
            x64, dy64 = x.double(), dy.double()
            mean, var = x64.mean(1, keepdim=True), x64.var(1, unbiased=False, keepdim=True)
            rstd = (var + eps).rsqrt()
            xh = (x64 - mean) * rstd
            # x - mean is off by the rounding of a mean of numbers of size |x|, the rest by a few roundings each
            xh_err = (h / 64 + 24) * u * ((x64.abs().mean(1, keepdim=True) + x64.abs()) * rstd + xh.abs())
            for got, terms, err in ((dg, dy64 * xh, dy64.abs() * xh_err), (db, dy64, 0.0 * dy64)):
                assert ((got.double() - terms.sum(0)).abs() <= (rows + 16) * u * terms.abs().sum(0) + err.sum(0) + 1e-30).all()
            dyg = dy64 if gamma is None else dy64 * gamma.double()
            want = rstd * (dyg - dyg.mean(1, keepdim=True) - xh * (dyg * xh).mean(1, keepdim=True)) + (0.0 if add is None else add.double())
            size = rstd * (dyg.abs() + dyg.abs().mean(1, keepdim=True) + (xh.abs() + 1) * (dyg * xh).abs().mean(1, keepdim=True)) + want.abs()
            err = (h / 64 + 32) * u * 4 * size + 4 * rstd * (xh_err * (dyg * xh).abs().mean(1, keepdim=True) + xh.abs() * (dyg.abs() * xh_err).mean(1, keepdim=True))
            assert ((dx.double() - want).abs() <= err).all()
        for a, b in zip(first, (dx, dg, db)):
            assert torch.equal(a, b)
