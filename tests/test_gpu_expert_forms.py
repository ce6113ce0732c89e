"""Every form of the experts' products, against 64 bits: the calls of expert_forms.py with their values compared."""
import numpy as np
import pytest

import expert_bounds as B
import expert_forms as F
from gpu_util import note, runtime
from test_gpu_experts import Case
from token_util import Arrays

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", F.KINDS)
@pytest.mark.parametrize("name,rows,dim,hidden", F.CALLS, ids=[c[0] for c in F.CALLS])
def test_forward_and_gradients(kind, name, rows, dim, hidden):
    npes, mine, cap = F.NPES, F.MINE, rows * F.MINE
    n = mine * npes
    rng = np.random.default_rng(rows * dim)
    with runtime(npes, 1 << 30) as rt, Arrays(rt) as new:
        c = Case(new, rng, kind, npes, mine, cap, dim, hidden, F.table(rng, npes, mine, cap, F.ROWS + F.MORE))
        out, pre = new(kind, (cap, dim)), new(kind, (cap, 2 * hidden))
        ws = new.workspace("moe_experts", cap, n, dim, hidden)
        untouched = out.get()
        note("moe_experts", kind, name)
        rt.moe_experts(kind, out.address, ws.address, c.x.address, c.w_in.address, c.w_out.address, c.er.address, cap, n, dim, hidden,
                       pre=pre.address)
        rt.sync()
        ws.get()
        got, got_pre = out.get(), pre.get()
        assert np.array_equal(got[~c.busy], untouched[~c.busy])
        assert np.array_equal(got_pre[~c.busy][:, :dim], np.broadcast_to(untouched[0, :1, :1], got_pre[~c.busy][:, :dim].shape))
        weights = {}
        for pe, i, a, b in c.each():
            if a == b:
                continue
            weights[pe, i] = B.f64(c.w_in_values[pe, i]), B.f64(c.w_out_values[pe, i])
            (want_pre, pre_bound), (want, bound) = B.forward(B.f64(c.x_values[pe, a:b]), *weights[pe, i], kind)
            what = " of expert %d of PE %d, %d rows" % (i, pe, b - a)
            B.hold(got_pre[pe, a:b], want_pre, pre_bound, kind, "pre" + what)
            B.hold(got[pe, a:b], want, bound, kind, "out" + what)

        dout_values, dout = c.rows(dim, 0.5)
        pre_values, pre = c.rows(2 * hidden, 1.5)
        drows, dw_in, dw_out = new(kind, (cap, dim)), new(kind, (mine, 2 * hidden, dim)), new(kind, (mine, dim, hidden))
        ws = new.workspace("moe_experts_grad", cap, n, dim, hidden)
        note("moe_experts_grad", kind, name)
        rt.moe_experts_grad(kind, drows.address, dw_in.address, dw_out.address, ws.address, dout.address, c.x.address, pre.address,
                            c.w_in.address, c.w_out.address, c.er.address, cap, n, dim, hidden)
        rt.sync()
        ws.get()
        got, got_in, got_out = drows.get(), dw_in.get(), dw_out.get()
        assert np.array_equal(got[~c.busy], untouched[~c.busy])
        for pe, i, a, b in c.each():
            if a == b:
                assert not got_in[pe, i].any() and not got_out[pe, i].any()
                continue
            grads = B.backward(B.f64(dout_values[pe, a:b]), B.f64(c.x_values[pe, a:b]), B.f64(pre_values[pe, a:b]), *weights[pe, i], kind)
            what = " of expert %d of PE %d, %d rows" % (i, pe, b - a)
            for part, result, (want, bound) in zip(("drows", "dw_in", "dw_out"), (got[pe, a:b], got_in[pe, i], got_out[pe, i]), grads):
                B.hold(result, want, bound, kind, part + what)
