"""The experts' block where it is used: between dispatch and combine, on streams and in graphs, and far into large buffers."""
import numpy as np
import pytest

import expert_reference as R
import token_reference as T
from dropout_reference import kept
from gpu_util import note, runtime
from nvshmem_amd import hip
from test_gpu_experts import Case, starts
from token_util import EPS, TINY, Arrays, close, rounded

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["float", "bfloat16"])
def test_forward_and_backward(kind):
    """Router, tables, dispatch, experts, combine, dropout onto the residual - and back.  What a step rounds is taken from the kernels for
    the next, so that each is held to its own bounds."""
    npes, tokens, experts, topk, dim, hidden, p = 8, 45, 32, 4, 264, 72, 0.2
    cap, mine, size = tokens * topk * 2, experts // npes, 4 if kind == "float" else 2
    limit, seed_values = int(np.rint(np.float64(np.float32(p)) * 65536)), [1234567890123, 42]
    rng = np.random.default_rng(3)
    with runtime(npes, 64 << 20) as rt, Arrays(rt) as new:
        perf = rt.perftest()
        x_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        l = rounded(rng.standard_normal((npes, tokens, experts)) * 2, kind)
        l[:, -3:] = -np.inf                                                      # padding
        x, logits = new(kind, (tokens, dim), x_values), new(kind, (tokens, experts), l)
        expert, gate, counts = new("int32", (tokens, topk)), new("float", (tokens, topk)), new("int64", (experts,))
        ws = new.workspace("moe_route", tokens, experts)
        note("route and place")
        rt.moe_route(kind, expert.address, gate.address, counts.address, ws.address, logits.address, tokens, experts, topk)
        dest_pe, dest_row = new("int32", (tokens, topk)), new("int64", (tokens, topk))
        expected, expert_row = new("int64", (npes,)), new("int64", (mine + 1,))
        place_ws = new.workspace("moe_place", tokens, topk, experts)
        rt.moe_place(dest_pe.address, dest_row.address, expected.address, expert_row.address, place_ws.address, expert.address,
                     counts.address, tokens, topk, experts, cap)
        recv, sig = new(kind, (cap, dim), np.float32(np.nan)), new("int64", (npes,), 0)
        note("dispatch")
        assert perf.nvshmem_perftest_moe_dispatch_pieces(recv.address, cap, x.address, dest_pe.address, dest_row.address, expected.address,
                                                         sig.address, tokens, topk, dim * size, 1024, 256, None) == 0
        rt.sync()
        assert rt.lib.nvshmemx_amd_timeout_count() == 0
        pe_values, row_values, er = dest_pe.get(), dest_row.get(), expert_row.get()
        w_in_values = rounded(rng.standard_normal((npes, mine, 2 * hidden, dim)) / np.sqrt(dim), kind)
        w_out_values = rounded(rng.standard_normal((npes, mine, dim, hidden)) / np.sqrt(hidden), kind)
        w_in, w_out = new(kind, (mine, 2 * hidden, dim), w_in_values), new(kind, (mine, dim, hidden), w_out_values)
        y, pre = new(kind, (cap, dim), np.float32(0)), new(kind, (cap, 2 * hidden), np.float32(0))
        ews = new.workspace("moe_experts", cap, experts, dim, hidden)
        note("experts")
        rt.moe_experts(kind, y.address, ews.address, recv.address, w_in.address, w_out.address, expert_row.address, cap, experts, dim,
                       hidden, pre=pre.address)
        out, z, seed = new(kind, (tokens, dim)), new(kind, (tokens, dim)), new("int64", (2,), np.array(seed_values))
        note("combine and dropout")
        rt.moe_combine_sum(kind, out.address, y.address, cap, gate.address, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.dropout(kind, z.address, out.address, seed.address, tokens, dim, p, residual=x.address)
        rt.sync()
        recv_values, y_values, pre_values, out_values, gate_values = recv.get(), y.get(), pre.get(), out.get(), gate.get()
        ranges = [(pe, i, a, b) for pe in range(npes) for i, (a, b) in enumerate(R.ranges(er[pe], cap))]
        assert sum(b - a for _, _, a, b in ranges) == npes * (tokens - 3) * topk
        for pe, i, a, b in ranges:
            want_pre, pre_bound, want, bound = R.forward(R.f64(recv_values[pe, a:b]), R.f64(w_in_values[pe, i]), R.f64(w_out_values[pe, i]), kind)
            close(pre_values[pe, a:b], want_pre, pre_bound, "pre")
            close(y_values[pe, a:b], want, bound, "y")
        want, magnitude = T.combine_sum(y_values, gate_values, pe_values, row_values)
        close(out_values, want, 2 * topk * T.STEP * magnitude + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "out")
        keep = np.stack([kept(tokens * dim, pe, seed_values, limit).reshape(tokens, dim) for pe in range(npes)])
        scale = 65536.0 / (65536 - limit)
        want = np.where(keep, out_values.astype(np.float64) * scale, 0) + x_values
        close(z.get(), want, 3 * T.STEP * (np.abs(want) + np.abs(x_values)) + EPS[kind] / 2 * 1.01 * np.abs(want) + TINY[kind], "z")

        note("backward")
        dz_values = rounded(rng.standard_normal((npes, tokens, dim)), kind)
        dz, dout = new(kind, (tokens, dim), dz_values), new(kind, (tokens, dim))
        rt.dropout(kind, dout.address, dz.address, seed.address, tokens, dim, p)
        dy, dgate = new(kind, (cap, dim), np.float32(np.nan)), new("float", (tokens, topk))
        rt.moe_combine_grad(kind, dy.address, dgate.address, dout.address, y.address, cap, gate.address, dest_pe.address,
                            dest_row.address, tokens, topk, dim)
        drecv = new(kind, (cap, dim), np.float32(0))
        dw_in, dw_out = new(kind, (mine, 2 * hidden, dim)), new(kind, (mine, dim, hidden))
        gws = new.workspace("moe_experts_grad", cap, experts, dim, hidden)
        rt.moe_experts_grad(kind, drecv.address, dw_in.address, dw_out.address, gws.address, dy.address, recv.address, pre.address,
                            w_in.address, w_out.address, expert_row.address, cap, experts, dim, hidden)
        dx = new(kind, (tokens, dim))
        rt.moe_combine_sum(kind, dx.address, drecv.address, cap, None, dest_pe.address, dest_row.address, tokens, topk, dim)
        rt.sync()
        dout_values = dout.get()
        want = np.where(keep, dz_values.astype(np.float64) * scale, 0)
        close(dout_values, want, (3 * T.STEP + EPS[kind] / 2 * 1.01) * np.abs(want) + TINY[kind], "dout")
        dy_values, drecv_values, got_in, got_out = dy.get(), drecv.get(), dw_in.get(), dw_out.get()
        for pe, i, a, b in ranges:
            grads = R.backward(R.f64(dy_values[pe, a:b]), R.f64(recv_values[pe, a:b]), R.f64(pre_values[pe, a:b]),
                               R.f64(w_in_values[pe, i]), R.f64(w_out_values[pe, i]), kind)
            for name, got, (want, bound) in zip(("drows", "dw_in", "dw_out"), (drecv_values[pe, a:b], got_in[pe, i], got_out[pe, i]), grads):
                close(got, want, bound, name)
        want, magnitude = T.combine_sum(drecv_values, None, pe_values, row_values)
        close(dx.get(), want, 2 * topk * T.STEP * magnitude + EPS[kind] / 2 * np.abs(want) * 1.01 + TINY[kind], "dx")


def test_in_graphs_and_on_other_streams():
    """Two graphs with workspaces of their own, replayed side by side with new inputs, and with eager calls in between."""
    npes, mine, cap, dim, hidden, group = 4, 3, 500, 256, 192, 64
    rng = np.random.default_rng(8)
    with runtime(npes, 128 << 20) as rt, Arrays(rt) as new:
        c = Case(new, rng, "half", npes, mine, cap, dim, hidden, starts(npes, mine, cap, [200, 20, 100], rng))
        n = mine * npes
        q_in = new("byte", (mine, 2 * hidden, dim // 2), rng.integers(0, 256, (npes, mine, 2 * hidden, dim // 2)))
        q_out = new("byte", (mine, dim, hidden // 2), rng.integers(0, 256, (npes, mine, dim, hidden // 2)))
        s_in = new("half", (mine, 2 * hidden, dim // group), rng.uniform(0.01, 0.02, (npes, mine, 2 * hidden, dim // group)))
        s_out = new("half", (mine, dim, hidden // group), rng.uniform(0.01, 0.02, (npes, mine, dim, hidden // group)))
        seed = new("int64", (2,), np.array([5, 6]))

        def outputs():
            return dict(out=new("half", (cap, dim)), pre=new("half", (cap, 2 * hidden)), drows=new("half", (cap, dim)),
                        dw_in=new("half", (mine, 2 * hidden, dim)), dw_out=new("half", (mine, dim, hidden)), four=new("half", (cap, dim)),
                        dropped=new("half", (cap, dim)), ws=new.workspace("moe_experts_grad", cap, n, dim, hidden))

        def calls(o, stream):
            size = (c.er.address, cap, n, dim, hidden)
            rt.moe_experts("half", o["out"].address, o["ws"].address, c.x.address, c.w_in.address, c.w_out.address, *size,
                           pre=o["pre"].address, stream=stream)
            rt.dropout("half", o["dropped"].address, o["out"].address, seed.address, cap, dim, 0.4, stream=stream)
            rt.moe_experts_grad("half", o["drows"].address, o["dw_in"].address, o["dw_out"].address, o["ws"].address,
                                o["dropped"].address, c.x.address, o["pre"].address, c.w_in.address, c.w_out.address, *size, stream=stream)
            rt.moe_experts_w4("half", o["four"].address, o["ws"].address, c.x.address, q_in.address, s_in.address, q_out.address,
                              s_out.address, *size, group, stream=stream)

        sets = [outputs() for _ in range(3)]
        streams = [hip.Stream(), hip.Stream()]
        graphs = []
        for o, stream in zip(sets, streams):
            note("capture")
            with hip.Graph(stream) as graph:
                calls(o, stream)
            graphs.append(graph)
        names = [k for k in sets[0] if k != "ws"]
        for replay in range(3):
            c.x.put(rounded(rng.standard_normal((npes, cap, dim)), "half"))
            c.er.put(starts(npes, mine, cap, [[200, 20, 100], [1, 0, 40], [0, 0, 0]][replay], rng, replay))
            seed.put(np.array([5, replay]))
            for o in sets:
                for k in names:
                    o[k].put(np.float32(1))
            note("replay", replay)
            for graph in graphs:
                graph.launch()
            for stream in streams:
                stream.synchronize()
            calls(sets[2], None)
            rt.sync()
            for k in names:
                want = sets[2][k].raw()
                for o in sets[:2]:
                    got = o[k].raw()
                    assert np.array_equal(got, want), (replay, k)
        for graph in graphs:
            graph.destroy()
        for stream in streams:
            stream.destroy()


@pytest.mark.parametrize("kind", ["bfloat16"])
def test_rows_and_weights_beyond_4_gib(kind):
    """The last rows of buffers of more than 4 GiB, and the last expert of weights of more than that."""
    cap, dim, hidden, experts = 310_000, 7168, 64, 2500 // 4
    n, first = 70, 309_900
    rng = np.random.default_rng(2)
    size = 2
    with runtime(1, 24 << 30) as rt:
        note("beyond 4 GiB")
        rows, out, drows = (rt.malloc(cap * dim * size) for _ in range(3))
        pre, ws = rt.malloc(cap * 2 * hidden * size), rt.malloc(rt.workspace_bytes("moe_experts_grad", cap, experts, dim, hidden))
        w_in, w_out = rt.malloc(experts * 2 * hidden * dim * size), rt.malloc(experts * dim * hidden * size)
        er = rt.malloc((experts + 1) * 8)
        table = np.full(experts + 1, first, np.int64)
        table[-1] = first + n
        rt.upload(er, 0, table)

        def put(at, values, elements):
            import torch
            bits = torch.from_numpy(values).to(torch.bfloat16).view(torch.int16).numpy()
            rt.upload(at, 0, bits, elements * size)

        def get(at, shape, elements):
            import torch
            return torch.from_numpy(rt.download(at, 0, shape, np.int16, elements * size)).view(torch.bfloat16).float().numpy()

        x = rounded(rng.standard_normal((n, dim)), kind)
        wi, wo = rounded(rng.standard_normal((2 * hidden, dim)) / 85, kind), rounded(rng.standard_normal((dim, hidden)) / 8, kind)
        last = experts - 1
        put(rows, x, first * dim)
        put(w_in, wi, last * 2 * hidden * dim)
        put(w_out, wo, last * dim * hidden)
        rt.moe_experts(kind, out, ws, rows, w_in, w_out, er, cap, experts, dim, hidden, pre=pre)
        rt.sync()
        want_pre, pre_bound, want, bound = R.forward(R.f64(x), R.f64(wi), R.f64(wo), kind)
        got_pre = get(pre, (n, 2 * hidden), first * 2 * hidden)
        close(got_pre, want_pre, pre_bound, "pre")
        close(get(out, (n, dim), first * dim), want, bound, "out")
        dw_in, dw_out = rt.malloc(experts * 2 * hidden * dim * size), rt.malloc(experts * dim * hidden * size)
        rt.moe_experts_grad(kind, drows, dw_in, dw_out, ws, out, rows, pre, w_in, w_out, er, cap, experts, dim, hidden)
        rt.sync()
        (want, bound), (want_in, bound_in), (want_out, bound_out) = R.backward(R.f64(get(out, (n, dim), first * dim)), R.f64(x), R.f64(got_pre),
                                                                               R.f64(wi), R.f64(wo), kind)
        close(get(drows, (n, dim), first * dim), want, bound, "drows")
        close(get(dw_in, (2 * hidden, dim), last * 2 * hidden * dim), want_in, bound_in, "dw_in")
        close(get(dw_out, (dim, hidden), last * dim * hidden), want_out, bound_out, "dw_out")
        assert not get(dw_in, (2 * hidden, dim), 0).any()


def test_wide_rows_of_experts():
    """dim and hidden at their most, one after the other."""
    npes, mine, cap = 1, 1, 40
    rng = np.random.default_rng(4)
    for dim, hidden in ((65536, 8), (8, 65536)):
        with runtime(npes, 512 << 20) as rt, Arrays(rt) as new:
            c = Case(new, rng, "bfloat16", npes, mine, cap, dim, hidden, np.array([[3, 38]]))
            from test_gpu_experts import check_backward, check_forward
            check_forward(rt, new, c, True)
            check_backward(rt, new, c)
