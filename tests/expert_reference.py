"""The experts' block in 64 bits, from its definition, with bounds for what the kernels may be off by.

Of every sum of n products in fp32 the bounds take n + 2 steps of 2^-23 of the sum of their magnitudes (a matrix core may round each of
its additions by up to a whole step), of sigmoid and what is multiplied with it 16 half steps, and half a step of the type for each
rounding to it."""
import numpy as np
import torch

from token_util import EPS, TINY

STEP = 2.0 ** -24
FEW = 16 * STEP


def f64(a):
    return torch.from_numpy(np.ascontiguousarray(a)).double()


def ranges(expert_row, cap):
    """[first, end) of every expert of a PE, cut to the rows that exist."""
    r = [min(max(int(v), 0), cap) for v in expert_row]
    return [(a, max(a, b)) for a, b in zip(r, r[1:])]


def gamma(n):
    return (n + 2) * 2 * STEP


def rounding(v, kind):
    return v.abs() * (EPS[kind] / 2) * 1.01 + TINY[kind]


def product(a, da, b, n):
    """a b^T where a is known to da: the value and what it may be off by."""
    value = a @ b.T
    return value, da @ b.abs().T + gamma(n) * ((a.abs() + da) @ b.abs().T)


def silu_parts(gate):
    s = torch.sigmoid(gate)
    return s, gate * s


def forward(x, w_in, w_out, kind):
    """pre, its bound, out, its bound"""
    hidden = w_out.shape[1]
    pre, dpre = product(x, torch.zeros_like(x), w_in, x.shape[1])
    gate, up, dgate, dup = pre[:, :hidden], pre[:, hidden:], dpre[:, :hidden], dpre[:, hidden:]
    _, silu = silu_parts(gate)
    h = silu * up
    dsilu = 1.1 * dgate + FEW * silu.abs()          # (the derivative of silu is at most 1.1)
    dh = (silu.abs() + dsilu) * (up.abs() + dup) - silu.abs() * up.abs() + STEP * h.abs()
    dh = dh + (h.abs() + dh) * (EPS[kind] / 2) * 1.01 + TINY[kind]
    out, dout = product(h, dh, w_out, hidden)
    return pre, dpre + rounding(pre, kind), out, dout + rounding(out, kind)


def backward(dout, x, pre, w_in, w_out, kind):
    """(drows, bound), (dw_in, bound), (dw_out, bound)"""
    hidden, n = w_out.shape[1], x.shape[0]
    gate, up = pre[:, :hidden], pre[:, hidden:]
    s, silu = silu_parts(gate)
    dh, ddh = product(dout, torch.zeros_like(dout), w_out.T, x.shape[1])
    slope, slope_size = s + silu * (1 - s), s + silu.abs() * (1 - s)
    dup, dgate = dh * silu, dh * up * slope
    ddup = ddh * silu.abs() * 1.01 + FEW * dup.abs()
    ddgate = (ddh * slope.abs() + FEW * (dh.abs() + ddh) * slope_size) * up.abs() * 1.01
    dpre, ddpre = torch.cat([dgate, dup], 1), torch.cat([ddgate, ddup], 1)
    ddpre = ddpre + (dpre.abs() + ddpre) * (EPS[kind] / 2) * 1.01 + TINY[kind]
    h = silu * up
    dh_own = FEW * h.abs() + rounding(h, kind)
    drows, ddrows = product(dpre, ddpre, w_in.T, 2 * hidden)
    dw_in, ddw_in = product(dpre.T, ddpre.T, x.T, n)
    dw_out, ddw_out = product(h.T, dh_own.T, dout.T, n)
    return ((drows, ddrows + rounding(drows, kind)), (dw_in, ddw_in + rounding(dw_in, kind)),
            (dw_out.T, ddw_out.T + rounding(dw_out.T, kind)))


def four_bits(packed, scale, k, group):
    """[n, k] values of packed weights: element 2 i in the low half of byte i, 8 stands for 0."""
    packed = torch.from_numpy(np.ascontiguousarray(packed)).long()
    q = torch.stack([packed % 16, packed // 16], 2).reshape(packed.shape[0], -1)[:, :k].double()
    return (q - 8) * f64(scale)[:, torch.arange(k) // group]


def forward_four_bits(x, w_in, s_in, w_out, s_out, kind):
    """forward() where a sum goes over 16 + q and takes 24 back: its magnitudes are those of 55 times the scales `s`, expanded like the
    weights.  That are 2 n additions; those of an fp32 element's second and third part are of 2^-8 of the first's magnitude.  (Sums over
    another power of two plus q are of larger magnitudes; they are held to this all the same.)"""
    hidden = w_out.shape[1]

    def product4(a, da, w, s):
        n = 2.1 * a.shape[1]
        return a @ w.T, da @ w.abs().T + gamma(n) * ((a.abs() + da) @ (55 * s.abs()).T)

    pre, dpre = product4(x, torch.zeros_like(x), w_in, s_in)
    gate, up, dgate, dup = pre[:, :hidden], pre[:, hidden:], dpre[:, :hidden], dpre[:, hidden:]
    _, silu = silu_parts(gate)
    h = silu * up
    dsilu = 1.1 * dgate + FEW * silu.abs()
    dh = (silu.abs() + dsilu) * (up.abs() + dup) - silu.abs() * up.abs() + STEP * h.abs()
    dh = dh + (h.abs() + dh) * (EPS[kind] / 2) * 1.01 + TINY[kind]
    out, dout = product4(h, dh, w_out, s_out)
    return out, dout + rounding(out, kind)
