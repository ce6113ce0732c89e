"""The experts' block with weights of 4 bits, called on whole numbers q of 0 to 15."""
import numpy as np

from gpu_util import note

ROWS = [1, 16, 17, 33, 64, 65, 130]  # of the experts of one PE: on both sides of all limits
TABLE = np.concatenate([[0], np.cumsum(ROWS)])[None]


def packed(q):
    """Two values a byte, the low half first."""
    q = np.asarray(q, np.uint8)
    if q.shape[-1] % 2:
        q = np.concatenate([q, np.zeros(q.shape[:-1] + (1,), np.uint8)], -1)
    return q[..., 0::2] | q[..., 1::2] << 4


def values(q, scale, group):
    """What q (.., n, k) and the scales (.., n, groups) stand for, in 64 bits."""
    k = q.shape[-1]
    return (q.astype(np.float64) - 8) * scale.astype(np.float64)[..., np.arange(k) // group]


def call(rt, new, kind, x, q_in, s_in, q_out, s_out, expert_row, group, shift=0):
    """out of moe_experts_w4 for x [npes, cap, dim] and weights [npes, mine, .., ..]; rows that no expert has have to be left alone."""
    npes, cap, dim = x.shape
    mine, hidden = q_in.shape[1], q_out.shape[3]
    w_in, w_out = packed(q_in), packed(q_out)
    arrays = [new(kind, (cap, dim), x, shift), new("byte", w_in.shape[1:], w_in, shift), new(kind, s_in.shape[1:], s_in, shift),
              new("byte", w_out.shape[1:], w_out, shift), new(kind, s_out.shape[1:], s_out, shift),
              new("int64", (mine + 1,), expert_row)]
    out, ws = new(kind, (cap, dim), None, shift), new.workspace("moe_experts", cap, mine * npes, dim, hidden)
    untouched = out.get()
    note("moe_experts_w4", kind, npes, mine, cap, dim, hidden, group, np.asarray(expert_row).tolist())
    rt.moe_experts_w4(kind, out.address, ws.address, *[a.address for a in arrays], cap, mine * npes, dim, hidden, group)
    rt.sync()
    ws.get()
    got = out.get()
    for pe in range(npes):
        idle = np.ones(cap, bool)
        for a, b in zip(expert_row[pe], expert_row[pe][1:]):
            idle[max(int(a), 0):max(int(b), 0)] = False
        assert np.array_equal(got[pe][idle], untouched[pe][idle])
    return got
