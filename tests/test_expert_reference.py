"""The gradients that the experts' reference gives are those of its forward pass, by differences."""
import pytest
import torch

import expert_reference as R


@pytest.mark.parametrize("n,dim,hidden", [(1, 1, 1), (3, 5, 4), (7, 4, 6)])
def test_gradients_against_differences(n, dim, hidden):
    g = torch.Generator().manual_seed(n * 100 + dim)
    x, dout = (torch.randn(n, dim, generator=g, dtype=torch.float64) for _ in range(2))
    w_in = torch.randn(2 * hidden, dim, generator=g, dtype=torch.float64)
    w_out = torch.randn(dim, hidden, generator=g, dtype=torch.float64)

    def value(x, w_in, w_out):
        return (R.forward(x, w_in, w_out, "float")[2] * dout).sum()

    pre = R.forward(x, w_in, w_out, "float")[0]
    grads = [v for v, _ in R.backward(dout, x, pre, w_in, w_out, "float")]
    step = 1e-5
    for at, grad in enumerate(grads):
        operands = [x, w_in, w_out]
        for i in range(operands[at].numel()):
            moved = []
            for sign in (1, -1):
                changed = [o.clone() for o in operands]
                changed[at].view(-1)[i] += sign * step
                moved.append(value(*changed))
            difference = (moved[0] - moved[1]) / (2 * step)
            # the third derivatives are of the size of the values: step^2, and 2^-52 of the value over the step
            assert abs(difference - grad.reshape(-1)[i]) <= 1e-7 * (1 + grad.abs().max())


def test_ranges_are_cut():
    assert R.ranges([-3, 4, 2, 99, 100], 50) == [(0, 4), (4, 4), (2, 50), (50, 50)]
