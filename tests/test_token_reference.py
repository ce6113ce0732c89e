"""The definitions over whole arrays, which large batches are checked with, against those that go through the tokens one by one."""
import numpy as np
import pytest

import token_reference as R


def _logits(rng, shape, how):
    x = rng.standard_normal(shape) * 3
    if how == "ties":
        x = np.round(x).clip(-1, 1)
        x[rng.random(shape) < 0.3] = -0.0
    if how == "masked":
        x[rng.random(shape) < 0.5] = -np.inf
        x[rng.random(shape) < 0.1] = np.nan
        x[:, 1], x[0, 2, 1:] = -np.inf, np.nan
    if how == "infinite":
        x[0, 0, ::3], x[-1, -1, -1] = np.inf, np.inf
    return x.astype(np.float32)


@pytest.mark.parametrize("normalise", [True, False])
@pytest.mark.parametrize("how", ["normal", "ties", "masked", "infinite"])
@pytest.mark.parametrize("npes,tokens,experts,topk", [(2, 9, 12, 3), (3, 5, 4, 4), (1, 7, 1, 1), (2, 6, 40, 8)])
def test_router(npes, tokens, experts, topk, how, normalise):
    rng = np.random.default_rng(experts)
    x = _logits(rng, (npes, tokens, experts), how)
    one, many = R.route(x, topk, normalise, 1.5), R.route_many(x, topk, normalise, 1.5)
    assert np.array_equal(one[0], many[0]) and np.array_equal(one[2], many[2])
    for a, b in zip((one[1], one[3], one[4]), (many[1], many[3], many[4])):
        np.testing.assert_allclose(b, a, rtol=1e-13, atol=1e-300)
    dgate, dloss = rng.standard_normal(one[1].shape).astype(np.float32), np.arange(1.0, npes + 1)
    for balance in (None, np.broadcast_to(one[4], (npes, experts))):
        a = R.route_grad(x, one[0], dgate, balance, dloss, normalise, 1.5)
        b = R.route_grad_many(x, one[0], dgate, balance, dloss, normalise, 1.5)
        # the same sums in 64 bits in another order
        np.testing.assert_allclose(b[1], a[1], rtol=1e-13, atol=1e-300)
        assert (np.abs(b[0] - a[0]) <= 1e-14 * a[1]).all()
