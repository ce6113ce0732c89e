"""The weighted sum of a token's copies and its gradients, against 64 bits."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from nvshmem_amd import hip
from token_util import Arrays, EPS, TINY, close, rounded

pytestmark = pytest.mark.gpu


def _tables(rng, npes, tokens, topk, cap, dropped=0.15):
    """Distinct rows for all copies, some of them dropped in one of the ways that an entry can say it."""
    places = rng.permutation(npes * cap)[:npes * tokens * topk].reshape(npes, tokens, topk)
    dest_pe, dest_row = (places // cap).astype(np.int32), places % cap
    for pe, row in ((-1, -1), (npes, 0), (0, cap), (0, -1), (1 << 30, 3), (0, 1 << 40)):
        at = rng.random(places.shape) < dropped / 6
        dest_pe[at], dest_row[at] = pe, row
    return dest_pe, dest_row


SIZES = [  # npes, tokens, topk, dim, shift of the rows' buffers in elements
    (8, 20, 8, 512, 0), (4, 33, 3, 1029, 1), (4, 7, 1, 1, 0), (16, 5, 6, 7168, 0), (2, 65, 9, 63, 3), (3, 10, 17, 2050, 2),
    (1, 12, 4, 129, 0), (8, 1, 2, 8192, 0), (2, 9, 5, 600, 1), (4, 6, 7, 100, 0), (2, 5, 4, 5, 3), (2, 150, 2, 2053, 1)]


@pytest.mark.parametrize("npes,tokens,topk,dim,shift", SIZES)
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_sum(kind, npes, tokens, topk, dim, shift):
    rng = np.random.default_rng(dim)
    cap = tokens * topk + 5
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        recv_values = rounded(rng.standard_normal((npes, cap, dim)), kind)
        pe_values, row_values = _tables(rng, npes, tokens, topk, cap)
        pe_values[0, 0] = -1      # a token without a copy
        gate_values = rng.random((npes, tokens, topk)).astype(np.float32)
        recv, gate = new(kind, (cap, dim), recv_values, shift), new("float", (tokens, topk), gate_values)
        dest_pe, dest_row = new("int32", (tokens, topk), pe_values), new("int64", (tokens, topk), row_values)
        for weights in (gate, None):
            out = new(kind, (tokens, dim), shift=shift)
            note("moe_combine_sum", kind, npes, tokens, topk, dim, weights is not None)
            rt.moe_combine_sum(kind, out.address, recv.address, cap, weights and weights.address, dest_pe.address,
                               dest_row.address, tokens, topk, dim)
            rt.sync()
            want, size = R.combine_sum(recv_values, weights and gate_values, pe_values, row_values)
            # a product and a sum per copy in fp32, one rounding to the type
            close(out.get(), want, 2 * topk * R.STEP * size + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "out")


@pytest.mark.parametrize("npes,tokens,dim,shift", [(8, 700, 509, 1), (3, 1367, 256, 0), (8, 4099, 72, 2), (16, 4097, 20, 0),
                                                   (4, 99, 5000, 1), (1, 4096, 257, 0)])
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_sum_of_one_copy_of_many_tokens(kind, npes, tokens, dim, shift):
    rng = np.random.default_rng(dim)
    cap = tokens + 5
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        recv_values = rounded(rng.standard_normal((npes, cap, dim)), kind)
        pe_values, row_values = _tables(rng, npes, tokens, 1, cap, 0.5)
        gate_values = rng.random((npes, tokens, 1)).astype(np.float32)
        gate_values[~R.kept(pe_values, row_values, npes, cap)] = np.nan
        recv, gate = new(kind, (cap, dim), recv_values, shift), new("float", (tokens, 1), gate_values)
        dest_pe, dest_row = new("int32", (tokens, 1), pe_values), new("int64", (tokens, 1), row_values)
        for weights in (gate, None):
            out = new(kind, (tokens, dim), shift=shift)
            note("moe_combine_sum", kind, npes, tokens, dim, weights is not None)
            rt.moe_combine_sum(kind, out.address, recv.address, cap, weights and weights.address, dest_pe.address,
                               dest_row.address, tokens, 1, dim)
            rt.sync()
            want, size = R.combine_sum(recv_values, weights and np.nan_to_num(gate_values), pe_values, row_values)
            close(out.get(), want, 2 * R.STEP * size + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "out")


@pytest.mark.parametrize("in_place", [False, True])
@pytest.mark.parametrize("npes,tokens,topk,dim,shift", SIZES)
@pytest.mark.parametrize("kind", ["float", "half", "bfloat16"])
def test_gradient(kind, npes, tokens, topk, dim, shift, in_place):
    rng = np.random.default_rng(dim + 1)
    cap = tokens * topk + 5
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        recv_values = rounded(rng.standard_normal((npes, cap, dim)), kind)
        dout_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        pe_values, row_values = _tables(rng, npes, tokens, topk, cap)
        gate_values = rng.random((npes, tokens, topk)).astype(np.float32)
        recv, gate = new(kind, (cap, dim), recv_values, shift), new("float", (tokens, topk), gate_values)
        dout = new(kind, (tokens, dim), dout_values, shift)
        dest_pe, dest_row = new("int32", (tokens, topk), pe_values), new("int64", (tokens, topk), row_values)
        before = recv_values if in_place else np.full((npes, cap, dim), 3.0, np.float32)
        drecv = recv if in_place else new(kind, (cap, dim), before, shift)
        dgate = new("float", (tokens, topk))
        note("moe_combine_grad", kind, npes, tokens, topk, dim, in_place)
        rt.moe_combine_grad(kind, drecv.address, dgate.address, dout.address, recv.address, cap, gate.address, dest_pe.address,
                            dest_row.address, tokens, topk, dim)
        rt.sync()
        want, want_gate, size = R.combine_grad(before, dout_values, recv_values, gate_values, pe_values, row_values)
        ok = R.kept(pe_values, row_values, npes, cap)
        named = np.zeros((npes, cap), bool)
        named[pe_values[ok], row_values[ok]] = True
        tolerance = np.where(named[..., None], (R.STEP + EPS[kind] / 2) * 1.01 * np.abs(want) + TINY[kind], 0.0)
        close(drecv.get(), want, tolerance, "drecv")
        # dim products added up in fp32, in whatever order
        close(dgate.get(), want_gate, (dim + 1) * R.STEP * size, "dgate")
        assert (dgate.get()[~ok] == 0).all()


def test_long_rows_are_added_up_in_parts():
    """Sums of 14336-byte rows stay far below the bound of one long chain: every lane adds up its own part first."""
    rng = np.random.default_rng(2)
    npes, tokens, topk, dim = 2, 4, 8, 7168
    cap = tokens * topk
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        recv_values, dout_values = (rounded(rng.random((npes, n, dim)), "bfloat16") for n in (cap, tokens))
        pe_values, row_values = _tables(rng, npes, tokens, topk, cap, 0)
        recv, dout = new("bfloat16", (cap, dim), recv_values), new("bfloat16", (tokens, dim), dout_values)
        gate = new("float", (tokens, topk), np.float32(1))
        dest_pe, dest_row = new("int32", (tokens, topk), pe_values), new("int64", (tokens, topk), row_values)
        drecv, dgate = new("bfloat16", (cap, dim)), new("float", (tokens, topk))
        rt.moe_combine_grad("bfloat16", drecv.address, dgate.address, dout.address, recv.address, cap, gate.address,
                            dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.sync()
        _, want, size = R.combine_grad(recv_values, dout_values, recv_values, np.ones((npes, tokens, topk)), pe_values, row_values)
        # 7168 elements over 64 lanes or more, at most 128 in each, then at most 10 steps
        close(dgate.get(), want, (128 + 10 + 1) * R.STEP * size, "dgate")


@pytest.mark.parametrize("topk", [1, 3, 8, 11])
@pytest.mark.parametrize("kind,dim", [("float", 3), ("bfloat16", 100), ("half", 520)])
def test_a_dropped_copy_s_gate_adds_nothing(kind, dim, topk):
    rng = np.random.default_rng(dim + topk)
    npes, tokens, cap = 2, 9, 9 * topk
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        recv_values = rounded(np.abs(rng.standard_normal((npes, cap, dim))) + 0.5, kind)
        pe_values, row_values = _tables(rng, npes, tokens, topk, cap, 0.9)
        pe_values[0, 0], pe_values[1, 0, 0] = -1, npes
        ok = R.kept(pe_values, row_values, npes, cap)
        gate_values = rng.random((npes, tokens, topk)).astype(np.float32)
        gate_values[~ok] = rng.choice([np.nan, np.inf, -np.inf], np.count_nonzero(~ok))
        pe_values[1, 1, -1], row_values[1, 1, -1] = 0, 0
        gate_values[1, 1, -1], ok[1, 1, -1] = np.inf, True         # one that counts, and is a token's last
        recv, gate = new(kind, (cap, dim), recv_values), new("float", (tokens, topk), gate_values)
        dest_pe, dest_row = new("int32", (tokens, topk), pe_values), new("int64", (tokens, topk), row_values)
        out = new(kind, (tokens, dim))
        note("moe_combine_sum", kind, npes, tokens, topk, dim)
        rt.moe_combine_sum(kind, out.address, recv.address, cap, gate.address, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.sync()
        gate_values[~ok], gate_values[1, 1, -1] = 0, 1
        want, size = R.combine_sum(recv_values, gate_values, pe_values, row_values)
        got = out.get()
        assert (got[1, 1] == np.inf).all()
        got[1, 1] = want[1, 1]
        close(got, want, 2 * topk * R.STEP * size + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "out")


@pytest.mark.parametrize("kind,dim", [("float", 1029), ("bfloat16", 101), ("half", 9), ("bfloat16", 512), ("float", 3)])
def test_an_infinite_gradient_is_counted_once(kind, dim):
    npes, tokens, cap = 2, dim, dim
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        pe_values = np.repeat(np.arange(npes, dtype=np.int32)[:, None, None], tokens, 1)
        row_values = np.broadcast_to(np.arange(tokens)[None, :, None], (npes, tokens, 1))
        dout_values = np.ones((npes, tokens, dim), np.float32)
        dout_values[0, np.arange(dim), np.arange(dim)] = np.inf       # another element of each token
        recv = new(kind, (cap, dim), np.full((npes, cap, dim), 0.5, np.float32))
        dout, gate = new(kind, (tokens, dim), dout_values), new("float", (tokens, 1), np.ones((npes, tokens, 1)))
        dest_pe, dest_row = new("int32", (tokens, 1), pe_values), new("int64", (tokens, 1), row_values)
        drecv, dgate = new(kind, (cap, dim)), new("float", (tokens, 1))
        note("moe_combine_grad", kind, npes, tokens, dim)
        rt.moe_combine_grad(kind, drecv.address, dgate.address, dout.address, recv.address, cap, gate.address, dest_pe.address,
                            dest_row.address, tokens, 1, dim)
        rt.sync()
        got = dgate.get()
        assert (got[0] == np.inf).all() and (got[1] == dim / 2).all()
        assert np.array_equal(drecv.get(), dout_values)


def test_infinities_and_nan_stay_with_their_token():
    with runtime(2, 16 << 20) as rt, Arrays(rt) as new:
        tokens, topk, dim = 6, 2, 40
        cap = 20
        rng = np.random.default_rng(3)
        pe_values, row_values = _tables(rng, 2, tokens, topk, cap, 0)
        recv_values = np.ones((2, cap, dim), np.float32)
        recv_values[pe_values[0, 1, 0], row_values[0, 1, 0], 3] = np.nan
        recv_values[pe_values[1, 2, 1], row_values[1, 2, 1], 4] = np.inf
        unused = np.ones((2, cap), bool)
        unused[pe_values, row_values] = False
        recv_values[unused] = np.nan                     # rows that no copy names, and one that is dropped
        recv_values[pe_values[0, 5, 0], row_values[0, 5, 0]] = np.nan
        pe_values[0, 5, 0] = -1
        recv, gate = new("half", (cap, dim), recv_values), new("float", (tokens, topk), np.float32(0.5))
        dest_pe, dest_row = new("int32", (tokens, topk), pe_values), new("int64", (tokens, topk), row_values)
        out = new("half", (tokens, dim))
        rt.moe_combine_sum("half", out.address, recv.address, cap, gate.address, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.sync()
        want = np.ones((2, tokens, dim))
        want[0, 1, 3], want[1, 2, 4], want[0, 5] = np.nan, np.inf, 0.5
        assert np.array_equal(out.get(), want, equal_nan=True)


def test_no_tokens_and_no_rows():
    with runtime(4, 16 << 20) as rt, Arrays(rt) as new:
        rt.moe_combine_sum("float", None, None, 0, None, None, None, 0, 2, 5)
        rt.moe_combine_grad("float", None, None, None, None, 0, None, None, None, 0, 2, 5)
        dest_pe, dest_row = new("int32", (3, 2), 0), new("int64", (3, 2), 0)      # nothing is received: all copies are dropped
        out, dgate = new("float", (3, 5)), new("float", (3, 2))
        gate, dout = new("float", (3, 2), np.float32(1)), new("float", (3, 5), np.float32(1))
        rt.moe_combine_sum("float", out.address, None, 0, gate.address, dest_pe.address, dest_row.address, 3, 2, 5)
        rt.moe_combine_grad("float", None, dgate.address, dout.address, None, 0, gate.address, dest_pe.address, dest_row.address,
                            3, 2, 5)
        rt.sync()
        assert (out.get() == 0).all() and (dgate.get() == 0).all()


def test_in_a_graph():
    rng = np.random.default_rng(4)
    npes, tokens, topk, dim, cap = 4, 30, 4, 300, 150
    with runtime(npes, 32 << 20) as rt, Arrays(rt) as new:
        recv, gate = new("float", (cap, dim)), new("float", (tokens, topk))
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        out, drecv, dgate = new("float", (tokens, dim)), new("float", (cap, dim)), new("float", (tokens, topk))
        stream = hip.Stream()
        with hip.Graph(stream) as graph:
            rt.moe_combine_sum("float", out.address, recv.address, cap, gate.address, dest_pe.address, dest_row.address, tokens,
                               topk, dim, stream=stream)
            rt.moe_combine_grad("float", drecv.address, dgate.address, out.address, recv.address, cap, gate.address,
                                dest_pe.address, dest_row.address, tokens, topk, dim, stream=stream)
        for _ in range(3):
            pe_values, row_values = _tables(rng, npes, tokens, topk, cap)
            recv_values = rng.integers(-4, 5, (npes, cap, dim)).astype(np.float32)    # sums that fp32 holds exactly
            gate_values = rng.integers(1, 5, (npes, tokens, topk)).astype(np.float32)
            for array, values in ((recv, recv_values), (gate, gate_values), (dest_pe, pe_values), (dest_row, row_values),
                                  (drecv, np.float32(0))):
                array.put(values)
            hip.synchronize()
            graph.launch()
            stream.synchronize()
            want, _ = R.combine_sum(recv_values, gate_values, pe_values, row_values)
            assert np.array_equal(out.get(), want)
            want_rows, want_gate, _ = R.combine_grad(np.zeros((npes, cap, dim)), want, recv_values, gate_values, pe_values, row_values)
            assert np.array_equal(drecv.get(), want_rows) and np.array_equal(dgate.get(), want_gate)
        graph.destroy()
        stream.destroy()
