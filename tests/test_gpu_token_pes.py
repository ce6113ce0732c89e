"""The operators on rows of tokens on more PEs than a kernel looks at together, up to the most that there can be."""
import numpy as np
import pytest

import token_reference as R
from gpu_util import note, runtime
from test_gpu_token_combine import _tables
from test_gpu_token_router import _exp_tolerance, _logits
from token_util import Arrays, EPS, TINY, close, rounded

pytestmark = pytest.mark.gpu

PES = [17, 24, 48, 64]


@pytest.mark.parametrize("tokens", [5, 90])
@pytest.mark.parametrize("npes", PES)
def test_router_and_tables(npes, tokens):
    experts, topk, kind = 3 * npes, 4, "float"
    cap = tokens * topk * 9 // 10
    rng = np.random.default_rng(npes)
    x = _logits(rng, kind, (npes, tokens, experts), "masked")
    tol = _exp_tolerance(x)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        logits, dlogits = new(kind, (tokens, experts), x), new(kind, (tokens, experts))
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        loss, balance = new("float", (1,)), new("float", (experts,))
        up = np.linspace(-1, 1, npes).astype(np.float32)
        dloss = new("float", (1,), up[:, None])
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (experts // npes + 1,))
        ws, ws2 = new.workspace("moe_route", tokens, experts), new.workspace("moe_place", tokens, topk, experts)
        for normalise, with_loss in ((True, True), (False, True), (True, False)):
            note("moe_route", npes, tokens, experts, normalise, with_loss)
            rt.moe_route(kind, expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk,
                         loss.address if with_loss else None, balance.address if with_loss else None, normalise)
            rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, ws2.address, expert.address,
                         counts.address, tokens, topk, experts, cap)
            rt.moe_route_grad(kind, dlogits.address, logits.address, expert.address, gate.address, tokens, experts, topk,
                              balance.address if with_loss else None, dloss.address if with_loss else None, normalise)
            rt.sync()
            want_expert, want_gate, want_counts, want_loss, b = R.route_many(x, topk, normalise, 1.0)
            assert np.array_equal(expert.get(), want_expert) and np.array_equal(counts.get(), want_counts)
            close(gate.get(), want_gate, tol * R.STEP * want_gate + 1e-37, "gate")
            if with_loss:
                close(balance.get(), np.broadcast_to(b, (npes, experts)), 1.01 * R.STEP * b, "balance")
                close(loss.get(), np.full((npes, 1), want_loss), (tol + 82) * R.STEP * want_loss, "loss")
            want, size = R.route_grad_many(x, want_expert, gate.get(), balance.get() if with_loss else None, up, normalise, 1.0)
            close(dlogits.get(), want, (3 * tol + 52) * R.STEP * size + (EPS[kind] / 2) * np.abs(want) * 1.01 + 1e-36, "dlogits")
            for got, want in zip((dest_pe, dest_row, expected, expert_row), R.place(want_expert, experts, cap)):
                assert np.array_equal(got.get(), want)
            ws.get()
            ws2.get()


@pytest.mark.parametrize("kind,dim", [("float", 70), ("bfloat16", 520)])
@pytest.mark.parametrize("npes", PES)
def test_rows(npes, kind, dim):
    tokens, topk, vocab = 11, 3, 5 * npes - 3
    cap, rows = tokens * topk + 5, 5
    rng = np.random.default_rng(npes + dim)
    with runtime(npes, 16 << 20) as rt, Arrays(rt) as new:
        table_values = rounded(rng.standard_normal((npes, rows, dim)), kind)
        ids_values = rng.integers(-1, vocab + 1, (npes, tokens))
        table, ids, x = new(kind, (rows, dim), table_values), new("int64", (tokens,), ids_values), new(kind, (tokens, dim))
        note("embedding", npes, kind, dim)
        rt.embedding(kind, x.address, table.address, ids.address, tokens, vocab, dim, 1.0)
        dtable, ws = new(kind, (rows, dim), np.float32(1)), new.workspace("embedding_grad", tokens, vocab, dim)
        rt.embedding_grad(kind, dtable.address, x.address, ids.address, ws.address, tokens, vocab, dim, 1.0)
        rt.sync()
        ok = (ids_values >= 0) & (ids_values < vocab)
        x_values = np.where(ok[..., None], table_values.reshape(-1, dim)[np.where(ok, ids_values, 0)], np.float32(0))
        assert np.array_equal(x.get(), x_values)
        want, size, n = R.embedding_grad(np.ones((npes, rows, dim)), x_values, ids_values, vocab, 1.0)
        close(dtable.get(), want, (n[..., None] + 1) * R.STEP * size * 1.01 + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "dtable")
        ws.get()

        recv_values = rounded(rng.standard_normal((npes, cap, dim)), kind)
        pe_values, row_values = _tables(rng, npes, tokens, topk, cap)
        gate_values = rng.random((npes, tokens, topk)).astype(np.float32)
        recv, gate, out = new(kind, (cap, dim), recv_values), new("float", (tokens, topk), gate_values), new(kind, (tokens, dim))
        dest_pe, dest_row = new("int32", (tokens, topk), pe_values), new("int64", (tokens, topk), row_values)
        drecv, dgate = new(kind, (cap, dim), np.float32(3)), new("float", (tokens, topk))
        note("moe_combine", npes, kind, dim)
        rt.moe_combine_sum(kind, out.address, recv.address, cap, gate.address, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.moe_combine_grad(kind, drecv.address, dgate.address, x.address, recv.address, cap, gate.address, dest_pe.address,
                            dest_row.address, tokens, topk, dim)
        rt.sync()
        want, size = R.combine_sum(recv_values, gate_values, pe_values, row_values)
        close(out.get(), want, 2 * topk * R.STEP * size + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "out")
        want, want_gate, size = R.combine_grad(np.full((npes, cap, dim), 3.0), x_values, recv_values, gate_values, pe_values, row_values)
        close(drecv.get(), want, (R.STEP + EPS[kind] / 2) * 1.01 * np.abs(want) + TINY[kind], "drecv")
        close(dgate.get(), want_gate, (dim + 1) * R.STEP * size, "dgate")
