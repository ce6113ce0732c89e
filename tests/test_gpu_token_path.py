"""The operators as a model with experts uses them: lookup, router, tables, the shuffle, combine - and back through all of them."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from token_util import Arrays, EPS, close, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float", "bfloat16"])
def test_forward_and_backward(kind):
    """Expert e doubles its rows e % 3 times.  What a step rounds is taken from the kernels for the next, so that each is
    held to its own bounds."""
    npes, tokens, experts, topk, dim, vocab = 8, 45, 32, 4, 264, 777
    cap = tokens * topk * 2
    rng = np.random.default_rng(11)
    size = 4 if kind == "float" else 2
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        perf = rt.perftest()
        rows = -(-vocab // npes)
        table_values = rounded(rng.standard_normal((npes, rows, dim)), kind)
        ids_values = rng.integers(0, vocab, (npes, tokens))
        ids_values[:, -3:] = -1
        table, ids, x = new(kind, (rows, dim), table_values), new("int64", (tokens,), ids_values), new(kind, (tokens, dim))
        note("lookup")
        rt.embedding(kind, x.address, table.address, ids.address, tokens, vocab, dim, 1.0)
        # the router's product is not this library's: logits as if it had made them, padding masked
        l = rounded(rng.standard_normal((npes, tokens, experts)) * 2, kind)
        l[:, -3:] = -np.inf
        logits = new(kind, (tokens, experts), l)
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance, ws = new("float", (1,)), new("float", (experts,)), new.workspace("moe_route", tokens, experts)
        note("route and place")
        rt.moe_route(kind, expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                     loss.address, balance.address)
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (experts // npes + 1,))
        place_ws = new.workspace("moe_place", tokens, topk, experts)
        rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, place_ws.address, expert.address,
                     counts.address, tokens, topk, experts, cap)
        recv, sig = new(kind, (cap, dim), np.float32(0)), new("int64", (npes,), 0)

        def dispatch(to, rows_of):
            sig.put(0)
            assert perf.nvshmem_perftest_moe_dispatch_pieces(to.address, cap, rows_of.address, dest_pe.address, dest_row.address,
                                                             expected.address, sig.address, tokens, topk, dim * size, 1024, 256,
                                                             None) == 0
            rt.sync()
            assert rt.lib.nvshmemx_amd_timeout_count() == 0

        note("dispatch")
        dispatch(recv, x)
        want_expert, _, want_counts, want_loss, b = R.route(l, topk, True, 1.0)
        assert np.array_equal(expert.get(), want_expert) and np.array_equal(counts.get(), want_counts)
        want_pe, want_row, want_expected, want_expert_row = R.place(want_expert, experts, cap)
        assert np.array_equal(dest_pe.get(), want_pe) and np.array_equal(dest_row.get(), want_row)
        assert np.array_equal(expected.get(), want_expected) and np.array_equal(sig.get(), want_expected)
        ok = ids_values >= 0
        x_values = np.where(ok[..., None], table_values.reshape(-1, dim)[np.where(ok, ids_values, 0)], 0)
        assert np.array_equal(x.get(), x_values)
        got_rows, kept = R.copies(recv.get(), want_pe, want_row)
        assert np.array_equal(got_rows, np.where(kept[..., None], x_values[:, :, None], 0))

        # the experts' own work, on the rows that expert_row says are theirs
        factor = np.zeros((npes, cap, 1), np.float32)
        for pe in range(npes):
            for i in range(experts // npes):
                factor[pe, want_expert_row[pe, i]:want_expert_row[pe, i + 1]] = 2.0 ** ((pe * (experts // npes) + i) % 3)
        y_values = recv.get() * factor
        y, out = new(kind, (cap, dim), y_values), new(kind, (tokens, dim))
        gate_values = gate.get()
        note("combine")
        rt.moe_combine_sum(kind, out.address, y.address, cap, gate.address, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.sync()
        want, magnitude = R.combine_sum(y_values, gate_values, want_pe, want_row)
        close(out.get(), want, 2 * topk * R.STEP * magnitude + EPS[kind] / 2 * np.abs(want) * 1.01, "out")

        note("backward")
        dout_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        dout, dy, dgate = new(kind, (tokens, dim), dout_values), new(kind, (cap, dim), np.float32(0)), new("float", (tokens, topk))
        rt.moe_combine_grad(kind, dy.address, dgate.address, dout.address, y.address, cap, gate.address, dest_pe.address,
                            dest_row.address, tokens, topk, dim)
        rt.sync()
        want_rows, want_dgate, magnitude = R.combine_grad(np.zeros((npes, cap, dim)), dout_values, y_values, gate_values, want_pe, want_row)
        close(dy.get(), want_rows, (R.STEP + EPS[kind] / 2) * 1.01 * np.abs(want_rows), "dy")
        close(dgate.get(), want_dgate, (dim + 1) * R.STEP * magnitude, "dgate")
        drecv_values = dy.get() * factor
        drecv, dx = new(kind, (cap, dim), drecv_values), new(kind, (tokens, dim))
        rt.moe_combine_sum(kind, dx.address, drecv.address, cap, None, dest_pe.address, dest_row.address, tokens, topk, dim)
        dloss, dlogits = new("float", (1,), np.float32(0.1)), new(kind, (tokens, experts))
        rt.moe_route_grad(kind, dlogits.address, logits.address, expert.address, dgate.address, tokens, experts, topk,
                          balance.address, dloss.address)
        dtable, grad_ws = new(kind, (rows, dim), np.float32(0)), new.workspace("embedding_grad", tokens, vocab, dim)
        rt.embedding_grad(kind, dtable.address, dx.address, ids.address, grad_ws.address, tokens, vocab, dim, 1.0)
        rt.sync()
        want, magnitude = R.combine_sum(drecv_values, None, want_pe, want_row)
        close(dx.get(), want, 2 * topk * R.STEP * magnitude + EPS[kind] / 2 * np.abs(want) * 1.01, "dx")
        want, magnitude = R.route_grad(l, want_expert, dgate.get(), balance.get(), np.full(npes, 0.1, np.float32), True, 1.0)
        span = l[np.isfinite(l)].max() - l[np.isfinite(l)].min()
        close(dlogits.get(), want, (3 * (2 * (3 * span + 4) + 28) + 52) * R.STEP * magnitude + EPS[kind] / 2 * np.abs(want) * 1.01, "dlogits")
        want, magnitude, n = R.embedding_grad(np.zeros((npes, rows, dim)), dx.get(), ids_values, vocab, 1.0)
        close(dtable.get(), want, (n[..., None] + 1) * R.STEP * magnitude * 1.01 + EPS[kind] / 2 * np.abs(want) * 1.01, "dtable")
