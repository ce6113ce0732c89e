"""The measured work of the operators around the token shuffle: rows of tokens on their way through a model with experts.

  embed, embed_grad      a token's row out of a table that is cut by rows over the PEs, and the table's gradient
  route, route_grad      top-k of the experts with gates, counts and the balance loss, then the shuffle's tables; and the
                         gradient of the gates and of the loss
  combine, combine_grad  a token's copies summed up with its gates, and the gradients of the copies and of the gates

A pass is what a program that keeps its tensors in the symmetric heap calls; every tensor here is [npes, ...], every
PE's copy.  `own` chooses between the library's calls and their plain form in torch.  Where it is false nothing of the
library is loaded, and the tensors are ordinary ones: that is all that prepare() decides by it.
"""
import ctypes as C
import math

import torch

own = False

HEAP_BYTES = 96 << 30  # of all PEs together
TYPES = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
STORAGE = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.int32: "<i4", torch.int64: "<i8",
           torch.uint8: "|u1"}


def listed():
    return [
        # a step of 64 sequences on every PE: top-8 of 256 experts, no loss
        {"name": "route_decode", "op": "route", "npes": 8, "type": "bfloat16", "tokens": 64, "experts": 256, "topk": 8,
         "normalise": True, "loss": False},
        # a training step's router: logits in fp32, counts and the balance loss
        {"name": "route_train", "op": "route", "npes": 8, "type": "float", "tokens": 8192, "experts": 256, "topk": 8,
         "normalise": True, "loss": True},
        # its backward pass; and that of a ragged batch on more PEs
        {"name": "route_grad_train", "op": "route_grad", "npes": 8, "type": "float", "tokens": 8192, "experts": 256,
         "topk": 8, "normalise": True},
        {"name": "route_grad_ragged", "op": "route_grad", "npes": 16, "type": "half", "tokens": 333, "experts": 176,
         "topk": 6, "normalise": False},
        # behind the shuffle's decode and prefill: rows of 7168 bf16, 8 copies a token
        {"name": "combine_decode", "op": "combine", "npes": 8, "type": "bfloat16", "tokens": 64, "experts": 256, "topk": 8,
         "dim": 7168},
        {"name": "combine_prefill", "op": "combine", "npes": 8, "type": "bfloat16", "tokens": 4096, "experts": 256,
         "topk": 8, "dim": 7168},
        # the backward pass of a micro-batch; and of rows that no vector divides
        {"name": "combine_grad_train", "op": "combine_grad", "npes": 8, "type": "bfloat16", "tokens": 2048, "experts": 256,
         "topk": 8, "dim": 7168},
        {"name": "combine_grad_odd", "op": "combine_grad", "npes": 4, "type": "half", "tokens": 501, "experts": 64, "topk": 2,
         "dim": 1029},
        # the rows of a step's tokens; of a prompt's
        {"name": "embed_decode", "op": "embed", "npes": 8, "type": "bfloat16", "tokens": 64, "vocab": 100003, "dim": 7168},
        {"name": "embed_prefill", "op": "embed", "npes": 8, "type": "bfloat16", "tokens": 4096, "vocab": 100003,
         "dim": 7168},
        # a training step's gradient: every row of the table is written; and fine-tuning with a small table in fp32
        {"name": "embed_grad_train", "op": "embed_grad", "npes": 8, "type": "bfloat16", "tokens": 4096, "vocab": 100003,
         "dim": 7168},
        {"name": "embed_grad_small", "op": "embed_grad", "npes": 4, "type": "float", "tokens": 152, "vocab": 32003,
         "dim": 515},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["route", "route", "route_grad", "combine", "combine_grad", "embed", "embed_grad"])
    npes, kind = rng.choice([4, 8, 8, 16]), rng.choice(["float", "half", "bfloat16", "bfloat16"])
    size = 4 if kind == "float" else 2
    tokens = _spread(rng, 1, 65536 // npes)
    case = {"op": op, "npes": npes, "type": kind}
    if op.startswith("embed"):
        dim = _ragged(rng, _spread(rng, 64, 8000))
        # 64 Ki tokens, or what 470 MB of rows hold; a table of at most 1.4 GB
        tokens = max(1, min(tokens, 470_000_000 // (npes * dim * size)))
        vocab = _spread(rng, 1000, min(150_000, 1_400_000_000 // (dim * size)))
        return dict(case, tokens=tokens, vocab=vocab, dim=dim)
    experts = npes * _spread(rng, 1, 512 // npes)
    topk = min(experts, rng.choice([1, 2, 4, 6, 8, 8]))
    case = dict(case, tokens=tokens, experts=experts, topk=topk)
    if op.startswith("route"):
        case["tokens"] = max(1, min(tokens, (1 << 24) // (npes * experts)))
        case["normalise"] = rng.random() < 0.5
        return dict(case, loss=rng.random() < 0.5) if op == "route" else case
    dim = _ragged(rng, _spread(rng, 64, 8000))
    budget = 1_800_000_000 if op == "combine_grad" else 3_600_000_000
    return dict(case, tokens=max(1, min(tokens, budget // (npes * topk * dim * size))), dim=dim)


def _ragged(rng, n):
    """Every second size is rounded up to a multiple of 64 elements, the others stay as they fell."""
    return n if rng.random() < 0.5 else (n + 63) // 64 * 64


# ------------------------------------------------------------------------------------------------------------
# The symmetric heap, as tensors
# ------------------------------------------------------------------------------------------------------------
_live = 0  # objects that hold memory of the current heap


def _library(npes):
    """The library, initialised for npes PEs: a heap that nothing holds memory of makes room for one of another PE count."""
    from nvshmem_amd import _lib
    lib = _lib.load()
    if lib.nvshmem_n_pes() != npes or not lib.nvshmemx_init_status():
        if _live:
            raise RuntimeError("symmetric memory of %d PEs is still in use" % lib.nvshmem_n_pes())
        torch.cuda.synchronize()
        lib.nvshmem_finalize()
        rc = lib.nvshmemx_amd_init(npes, HEAP_BYTES // npes)
        if rc != 0:
            raise RuntimeError("nvshmemx_amd_init: %s" % lib.nvshmemx_amd_last_error().decode())
    return lib


class _Memory:
    """One symmetric allocation; a tensor over it keeps this object."""

    def __init__(self, lib, nbytes):
        global _live
        self.lib, self.address = lib, lib.nvshmem_malloc(max(nbytes, 16))
        if not self.address:
            raise MemoryError("out of memory: %d bytes per PE" % nbytes)
        _live += 1
        self.stride = lib.nvshmem_ptr(self.address, 1) - lib.nvshmem_ptr(self.address, 0)

    def __del__(self):
        global _live
        if getattr(self, "address", None):
            self.lib.nvshmem_free(self.address)
            self.address = None
            _live -= 1


def _tensor(npes, shape, dtype):
    """A [npes, *shape] tensor: symmetric memory, or ordinary memory for the plain form."""
    if not own:
        return torch.zeros((npes,) + tuple(shape), dtype=dtype, device="cuda")
    count = math.prod(shape)
    memory = _Memory(_library(npes), count * dtype.itemsize)
    strides, step = [], dtype.itemsize
    for extent in reversed(shape):
        strides.insert(0, step)
        step *= extent
    memory.__cuda_array_interface__ = {"shape": (npes,) + tuple(shape), "typestr": STORAGE[dtype], "version": 3,
                                       "strides": (memory.stride,) + tuple(strides), "data": (memory.address, False)}
    return torch.as_tensor(memory, device="cuda").view(dtype).zero_()


# ------------------------------------------------------------------------------------------------------------
# prepare
# ------------------------------------------------------------------------------------------------------------
class _State:
    """What a program keeps: its tensors by name, and the sizes."""

    def __init__(self, case):
        self.case, self.t = case, {}


def _logits(case, g):
    """Router logits with some experts more popular than others; the last 1/16 of a batch is padding, masked as a whole."""
    npes, tokens, experts = case["npes"], case["tokens"], case["experts"]
    x = torch.randn(npes, tokens, experts, device="cuda", generator=g)
    x += 0.5 * torch.randn(experts, device="cuda", generator=g)
    x[:, tokens - tokens // 16:] = -math.inf
    return x.to(TYPES[case["type"]])


def _capacity(case):
    """Receive rows of a PE: a quarter more than its share of the copies, and a few for small batches."""
    return case["tokens"] * case["topk"] * 5 // 4 + 64


def _experts(case, g):
    """Distinct experts of every token, the r-th most popular one with probability ~ 1/r, the popular ones dealt out over
    the PEs."""
    npes, tokens, experts, topk = case["npes"], case["tokens"], case["experts"], case["topk"]
    weight = -torch.arange(1, experts + 1, device="cuda", dtype=torch.float32).log_()
    noise = torch.empty(npes, tokens, experts, device="cuda").exponential_(generator=g).log_().neg_()
    rank = (weight + noise).topk(topk, dim=2).indices
    return (rank % npes) * (experts // npes) + rank // npes


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = _State(case)
    t, npes, tokens, dtype = state.t, case["npes"], case["tokens"], TYPES[case["type"]]
    op = case["op"]

    def put(name, value):
        t[name] = _tensor(npes, value.shape[1:], value.dtype)
        t[name].copy_(value)

    def make(name, shape, dt):
        t[name] = _tensor(npes, shape, dt)

    if op in ("route", "route_grad"):
        experts, topk = case["experts"], case["topk"]
        put("logits", _logits(case, g))
        if op == "route":
            make("expert", (tokens, topk), torch.int32)
            make("gate", (tokens, topk), torch.float32)
            make("counts", (experts,), torch.int64)
            make("loss", (1,), torch.float32)
            make("balance", (experts,), torch.float32)
            make("dest_pe", (tokens, topk), torch.int32)
            make("dest_row", (tokens, topk), torch.int64)
            make("expected", (npes,), torch.int64)
            make("expert_row", (experts // npes + 1,), torch.int64)
        else:
            forward = _plain_route(t["logits"], topk, case["normalise"], 1.0)
            put("expert", forward["expert"])
            put("balance", forward["balance"])
            put("dgate", torch.randn(npes, tokens, topk, device="cuda", generator=g))
            put("dloss", torch.full((npes, 1), 0.01, device="cuda"))
            make("dlogits", (tokens, experts), dtype)
    elif op in ("combine", "combine_grad"):
        topk, dim, cap = case["topk"], case["dim"], _capacity(case)
        expert = _experts(case, g)
        place = _plain_place(expert, case["experts"], cap)
        put("dest_pe", place["dest_pe"])
        put("dest_row", place["dest_row"])
        put("gate", torch.rand(npes, tokens, topk, device="cuda", generator=g).add_(0.1).div_(topk))
        make("recv", (cap, dim), dtype)
        for pe in range(npes):
            t["recv"][pe].normal_(generator=g)
        if op == "combine":
            make("out", (tokens, dim), dtype)
        else:
            put("dout", torch.randn(npes, tokens, dim, device="cuda", generator=g).to(dtype))
            make("drecv", (cap, dim), dtype)  # rows that nothing was sent to stay as they are
            make("dgate", (tokens, topk), torch.float32)
    else:
        vocab, dim = case["vocab"], case["dim"]
        # ids by a Zipf distribution over a shuffled vocabulary; the last 1/16 of a batch is padding
        rank = torch.rand(npes, tokens, device="cuda", generator=g, dtype=torch.float64).mul_(math.log(vocab)).exp_().long() - 1
        ids = torch.randperm(vocab, device="cuda", generator=g)[rank.clamp_(0, vocab - 1)]
        ids[:, tokens - tokens // 16:] = -1
        put("ids", ids)
        rows = -(-vocab // npes)
        state.scale = math.sqrt(dim)
        if op == "embed":
            make("table", (rows, dim), dtype)
            for pe in range(npes):
                t["table"][pe].normal_(0, 0.02, generator=g)
            make("out", (tokens, dim), dtype)
        else:
            put("dout", torch.randn(npes, tokens, dim, device="cuda", generator=g).to(dtype))
            make("dtable", (rows, dim), dtype)
    if own:
        _bind(state)
    return state


# ------------------------------------------------------------------------------------------------------------
# The library's calls
# ------------------------------------------------------------------------------------------------------------
def _bind(state):
    """Addresses, workspaces and entry points, as a program keeps them."""
    from nvshmem_amd import _lib
    case, lib = state.case, _lib.load()
    state.error = lib.nvshmemx_amd_last_error
    a = {name: lib.nvshmem_ptr(tensor.data_ptr(), 0) for name, tensor in state.t.items()}
    size, dim, topk, experts = C.c_size_t, case.get("dim"), case.get("topk"), case.get("experts")
    tokens, npes = case["tokens"], case["npes"]

    def entry(name):
        return getattr(lib, "nvshmemx_amd_%s_%s_on_stream" % (case["type"], name))

    def workspace(nbytes):
        state.t["workspace"] = _tensor(npes, (nbytes,), torch.uint8)
        return state.t["workspace"].data_ptr()

    op = case["op"]
    if op == "route":
        need = max(lib.nvshmemx_amd_moe_route_workspace(tokens, experts), lib.nvshmemx_amd_moe_place_workspace(tokens, topk, experts))
        ws = workspace(need)
        loss, balance = (a["loss"], a["balance"]) if case["loss"] else (None, None)
        state.calls = [
            (entry("moe_route"), (a["expert"], a["gate"], a["counts"], loss, balance, ws, a["logits"], size(tokens), experts,
                                  topk, int(case["normalise"]), 1.0)),
            (lib.nvshmemx_amd_moe_place_on_stream, (a["dest_pe"], a["dest_row"], a["expected"], a["expert_row"], ws, a["expert"],
                                                    a["counts"], size(tokens), topk, experts, size(_capacity(case))))]
    elif op == "route_grad":
        state.calls = [(entry("moe_route_grad"), (a["dlogits"], a["logits"], a["expert"], a["dgate"], a["balance"], a["dloss"],
                                                  size(tokens), experts, topk, int(case["normalise"]), 1.0))]
    elif op == "combine":
        state.calls = [(entry("moe_combine_sum"), (a["out"], a["recv"], size(_capacity(case)), a["gate"], a["dest_pe"],
                                                   a["dest_row"], size(tokens), topk, size(dim)))]
    elif op == "combine_grad":
        state.calls = [(entry("moe_combine_grad"), (a["drecv"], a["dgate"], a["dout"], a["recv"], size(_capacity(case)), a["gate"],
                                                    a["dest_pe"], a["dest_row"], size(tokens), topk, size(dim)))]
    elif op == "embed":
        state.calls = [(entry("embedding"), (a["out"], a["table"], a["ids"], size(tokens), size(case["vocab"]), size(dim),
                                             state.scale))]
    else:
        ws = workspace(lib.nvshmemx_amd_embedding_grad_workspace(tokens, case["vocab"], dim))
        state.calls = [(entry("embedding_grad"), (a["dtable"], a["dout"], a["ids"], ws, size(tokens), size(case["vocab"]),
                                                  size(dim), state.scale))]


def _outputs(case):
    return {"route": ["expert", "gate", "counts", "dest_pe", "dest_row", "expected", "expert_row"]
            + (["loss", "balance"] if case.get("loss") else []),
            "route_grad": ["dlogits"], "combine": ["out"], "combine_grad": ["drecv", "dgate"], "embed": ["out"],
            "embed_grad": ["dtable"]}[case["op"]]


def run(state):
    if own:
        stream = torch.cuda.current_stream().cuda_stream or None
        for fn, args in state.calls:
            if fn(*args, stream):
                raise RuntimeError(state.error().decode())
        return {name: state.t[name] for name in _outputs(state.case)}
    case, t = state.case, state.t
    op = case["op"]
    if op == "route":
        out = _plain_route(t["logits"], case["topk"], case["normalise"], 1.0)
        out |= _plain_place(out["expert"], case["experts"], _capacity(case))
    elif op == "route_grad":
        out = {"dlogits": _plain_route_grad(t, case["normalise"], 1.0)}
    elif op == "combine":
        out = {"out": _plain_combine(t)}
    elif op == "combine_grad":
        out = _plain_combine_grad(t)
    elif op == "embed":
        out = {"out": _plain_embed(t, case["vocab"], state.scale)}
    else:
        out = {"dtable": _plain_embed_grad(t, case["vocab"], state.scale)}
    return {name: out[name] for name in _outputs(case)}


# ------------------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------------------
def _probabilities(logits):
    """softmax over the experts that are not masked (a masked one has -inf), 0 for the others."""
    x = logits.float()
    x = torch.where(x > -math.inf, x, -math.inf)
    some = (x > -math.inf).any(2, keepdim=True)
    e = torch.exp(x - torch.where(some, x.amax(2, keepdim=True), 0.0))
    return x, torch.where(some, e / e.sum(2, keepdim=True), 0.0), some


def _plain_route(logits, topk, normalise, scale):
    x, p, some = _probabilities(logits)
    npes, _, experts = x.shape
    value, index = (v[:, :, :topk] for v in torch.sort(x, dim=2, descending=True, stable=True))
    chosen = value > -math.inf
    gate = torch.where(chosen, p.gather(2, index), 0.0)
    if normalise:
        gate = torch.where(chosen, gate / gate.sum(2, keepdim=True), 0.0)
    counts = torch.zeros(npes, experts + 1, dtype=torch.int64, device=x.device)
    slot = torch.where(chosen, index, experts).reshape(npes, -1)
    counts = counts.scatter_add_(1, slot, torch.ones_like(slot))[:, :experts]
    c = counts.sum(0).double()
    balance = experts * c / (c.sum() * some.sum()).clamp(min=1)
    loss = (balance * p.double().sum((0, 1))).sum()
    return {"expert": torch.where(chosen, index, -1).int(), "gate": gate * scale, "counts": counts,
            "loss": loss.float().expand(npes, 1), "balance": balance.float().expand(npes, experts)}


def _plain_place(expert, experts, cap):
    npes, tokens, topk = expert.shape
    per_pe = experts // npes
    e = expert.reshape(npes, -1).long()
    source = torch.arange(npes, device=e.device).unsqueeze(1).expand_as(e)
    key = torch.where(e >= 0, e * npes + source, experts * npes).reshape(-1)
    rows = torch.bincount(key, minlength=experts * npes + 1)
    first = rows.cumsum(0) - rows
    order = torch.sort(key, stable=True).indices
    rank = torch.empty_like(order)
    rank[order] = torch.arange(order.numel(), device=e.device)
    pe = key // (npes * per_pe)
    row = rank - first[pe.clamp(max=npes - 1) * per_pe * npes]
    kept = (key < experts * npes) & (row < cap)
    flow = torch.where(kept, pe * npes + source.reshape(-1), npes * npes)
    expected = torch.bincount(flow, minlength=npes * npes + 1)[:npes * npes].reshape(npes, npes)
    edges = torch.cat([first[:experts * npes:npes], first[-1:]])
    at = torch.arange(npes, device=e.device).unsqueeze(1) * per_pe + torch.arange(per_pe + 1, device=e.device)
    expert_row = (edges[at] - edges[at[:, :1]]).clamp(max=cap)
    shape = (npes, tokens, topk)
    return {"dest_pe": torch.where(kept, pe, -1).int().reshape(shape), "dest_row": torch.where(kept, row, -1).reshape(shape),
            "expected": expected, "expert_row": expert_row}


def _plain_route_grad(t, normalise, scale):
    logits, expert, dgate = t["logits"], t["expert"].long(), t["dgate"]
    _, p, _ = _probabilities(logits)
    index = expert.clamp(min=0)
    g = torch.where(expert >= 0, dgate * scale, 0.0)
    q = (t["dloss"] * t["balance"]).unsqueeze(1).expand_as(p)
    if not normalise:
        q = q.scatter_add(2, index, g)
    d = p * (q - (q * p).sum(2, keepdim=True))
    if normalise:
        w = torch.where(expert >= 0, p.gather(2, index), 0.0)
        w = w / w.sum(2, keepdim=True).clamp(min=1e-30)
        d = d.scatter_add(2, index, w * (g - (g * w).sum(2, keepdim=True)))
    return d.to(logits.dtype)


def _rows(t):
    """Every copy's row in fp32, zeros where it was dropped."""
    pe, row = t["dest_pe"].long(), t["dest_row"]
    kept = (pe >= 0).unsqueeze(3)
    return torch.where(kept, t["recv"][pe.clamp(min=0), row.clamp(min=0)].float(), 0.0), kept


def _plain_combine(t):
    rows, _ = _rows(t)
    return (rows * t["gate"].unsqueeze(3)).sum(2).to(t["recv"].dtype)


def _plain_combine_grad(t):
    rows, kept = _rows(t)
    dout = t["dout"].float().unsqueeze(2)
    dgate = (rows * dout).sum(3)
    d = (t["gate"].unsqueeze(3) * dout).to(t["recv"].dtype)
    kept = kept.squeeze(3)
    drecv = t["drecv"].clone()
    drecv[t["dest_pe"].long()[kept], t["dest_row"][kept]] = d[kept]
    return {"drecv": drecv, "dgate": dgate}


def _plain_embed(t, vocab, scale):
    ids, table = t["ids"], t["table"]
    some = (ids >= 0) & (ids < vocab)
    at = torch.where(some, ids, 0)
    rows = table[at // table.shape[1], at % table.shape[1]].float() * scale
    return torch.where(some.unsqueeze(2), rows, 0.0).to(table.dtype)


def _plain_embed_grad(t, vocab, scale):
    ids, dout, dtable = t["ids"].reshape(-1), t["dout"], t["dtable"]
    npes, rows, dim = dtable.shape
    some = (ids >= 0) & (ids < vocab)
    total = torch.zeros(npes * rows + 1, dim, device=ids.device)
    total.index_add_(0, torch.where(some, ids, npes * rows), dout.reshape(-1, dim).float())
    out = (total[:npes * rows] * scale).to(dtable.dtype)
    out[vocab:] = dtable.reshape(-1, dim)[vocab:]
    return out.reshape(npes, rows, dim)


# ------------------------------------------------------------------------------------------------------------
# In 64 bits, from the definitions
# ------------------------------------------------------------------------------------------------------------
def exact(case, seed):
    global own
    was, own = own, False
    try:
        state = prepare(case, seed)
    finally:
        own = was
    t, npes, op = state.t, case["npes"], case["op"]
    if op in ("route", "route_grad"):
        live = torch.isfinite(t["logits"]).any(2)
        x = t["logits"].double()
        p = torch.zeros_like(x)
        p[live] = torch.softmax(x[live], dim=1)
        if op == "route":
            top, at = torch.topk(p, case["topk"], dim=2)
            gate = torch.zeros_like(top)
            gate[live] = top[live] / top[live].sum(1, keepdim=True) if case["normalise"] else top[live]
            counts = t["logits"].new_zeros(case["experts"], dtype=torch.float64)
            # (equal logits at the edge of the top-k go to the lowest experts, which topk does not promise)
            at = torch.sort(x, dim=2, descending=True, stable=True).indices[:, :, :case["topk"]]
            counts.index_add_(0, at[live].reshape(-1), torch.ones(at[live].numel(), dtype=torch.float64, device=x.device))
            share = counts / counts.sum().clamp(min=1)
            mean = p.sum((0, 1)) / live.sum().clamp(min=1)
            values = {"gate": gate, "loss": (case["experts"] * (share * mean).sum()).expand(npes, 1),
                      "balance": (case["experts"] * share / live.sum().clamp(min=1)).expand(npes, case["experts"])}
            return {name: values.get(name) for name in _outputs(case)}
        # the gradient of <gate, dgate> + dloss * <balance, sum of p>, by differentiating it
        x = torch.where(torch.isfinite(x), x, -1e300).masked_fill(~live.unsqueeze(2), 0.0).requires_grad_()
        p = torch.softmax(x, dim=2)
        e = t["expert"].long()
        gate = p.gather(2, e.clamp(min=0)) * (e >= 0)
        if case["normalise"]:
            gate = gate / gate.sum(2, keepdim=True).clamp(min=1e-300)
        value = (gate * t["dgate"].double()).sum(2) + (p * (t["balance"].double() * t["dloss"].double()).unsqueeze(1)).sum(2)
        return {"dlogits": torch.autograd.grad((value * live).sum(), x)[0]}
    if op in ("combine", "combine_grad"):
        keep = t["dest_pe"] >= 0
        at = torch.where(keep, t["dest_pe"].long() * _capacity(case) + t["dest_row"], 0)
        rows = t["recv"].reshape(-1, case["dim"])[at].double() * keep.unsqueeze(3)
        gate = t["gate"].double()
        if op == "combine":
            return {"out": torch.matmul(gate.unsqueeze(2), rows).squeeze(2)}
        dout = t["dout"].double()
        drecv = t["drecv"].double().reshape(-1, case["dim"])
        token = torch.arange(npes * case["tokens"], device=at.device).reshape(npes, -1, 1).expand_as(at)
        drecv[at[keep]] = gate[keep].unsqueeze(1) * dout.reshape(-1, case["dim"])[token[keep]]
        return {"drecv": drecv.reshape(npes, -1, case["dim"]), "dgate": torch.matmul(rows, dout.unsqueeze(3)).squeeze(3)}
    ids, vocab, dim = t["ids"], case["vocab"], case["dim"]
    if op == "embed":
        table = torch.cat([t["table"].reshape(-1, dim)[:vocab], t["table"].new_zeros(1, dim)])
        return {"out": table[ids].double() * math.sqrt(dim)}  # (padding, -1, finds the row of zeros)
    total = torch.zeros(t["dtable"].shape[1] * npes, dim, dtype=torch.float64, device=ids.device)
    some = ids >= 0
    total.index_add_(0, ids[some], t["dout"][some].double())
    return {"dtable": (total * math.sqrt(dim)).reshape(npes, -1, dim)}


# ------------------------------------------------------------------------------------------------------------
def work(case):
    """What a pass cannot do without: every input read once, every output written once."""
    npes, tokens, size = case["npes"], case["npes"] * case["tokens"], TYPES[case["type"]].itemsize
    op = case["op"]
    if op.startswith("route"):
        values, copies = tokens * case["experts"], tokens * case["topk"]
        if op == "route":
            tables = 12 * copies + 8 * npes * (2 * case["experts"] + npes)
            return {"bytes": values * size + 8 * copies + tables, "flops": 6 * values}
        return {"bytes": 2 * values * size + 8 * copies, "flops": 8 * values}
    if op.startswith("combine"):
        copies, row = tokens * case["topk"], case["dim"] * size
        if op == "combine":
            return {"bytes": (copies + tokens) * row + 16 * copies, "flops": 2 * copies * case["dim"]}
        return {"bytes": (2 * copies + tokens) * row + 20 * copies, "flops": 3 * copies * case["dim"]}
    row, vocab = case["dim"] * size, case["vocab"]
    # a Zipf distribution's distinct ids among n draws: the sum over ranks of the chance to come up at all
    if op == "embed":
        distinct = sum(1.0 - math.exp(-tokens / (r * math.log(vocab))) for r in range(1, vocab + 1))
        return {"bytes": (min(distinct, tokens) + tokens) * row + 8 * tokens, "flops": tokens * case["dim"]}
    return {"bytes": (tokens + vocab) * row + 8 * tokens, "flops": tokens * case["dim"]}
