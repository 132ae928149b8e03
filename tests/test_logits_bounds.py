"""CPU: the bounds that the kernels over wide rows of logits are held to are tight enough to notice logits that a sum leaves out."""
import numpy as np
import pytest

from oracle import logits as ol


@pytest.mark.parametrize("v", [3001, 30522, 131072, 524288])
@pytest.mark.parametrize("sigma", [1.0, 3.0])
def test_a_wave_of_lost_pieces_is_noticed(v, sigma):
    """64 pieces of 16 bytes (one load of a wave) from anywhere in a row of random logits"""
    g = np.random.default_rng(v)
    z = g.standard_normal((4, v)) * sigma
    whole = ol.token_logprobs(z, np.zeros(4, dtype=np.int64), 0, 1.0)
    for at in g.integers(1, v - 256, 8):
        lost = z.copy()
        lost[:, at: at + 256] = -np.inf
        part = ol.token_logprobs(lost, np.zeros(4, dtype=np.int64), 0, 1.0)
        for name in ("lse", "logp"):
            assert (np.abs(part[name] - whole[name]) > whole["err_" + name]).all(), name


def test_the_bounds_are_those_of_the_longest_chain():
    """a lane's additions one after another under the launch rules: 64 lanes up to 2048 pieces, 256 threads or more beyond"""
    for v in [*range(65, 9000, 13), 32768, 131072, 524288]:
        for per_piece in (4, 8):
            pieces = v / per_piece
            assert ol.chain(v) >= min(pieces / (64 if pieces <= 2048 else 256), 32 if pieces <= 2048 else np.inf) - 1e-9
