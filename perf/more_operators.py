"""The measured work of what stands between the token shuffle's two halves, and of dropout on rows of tokens.

  experts, experts_grad  the experts' gated feed-forward block on the rows that were dispatched to them, and its gradients
  experts_w4             the same block with weights of 4 bits and a scale per group of them
  dropout                rows of tokens with elements dropped by a counter-based generator, added to a residual

A pass is what a program that keeps its tensors in the symmetric heap calls; every tensor here is [npes, ...], every
PE's copy.  `own` chooses between the library's calls and their plain form in torch.  Where it is false nothing of the
library is loaded, and the tensors are ordinary ones: that is all that prepare() decides by it.
"""
import ctypes as C
import math

import torch

own = False

HEAP_BYTES = 128 << 30  # of all PEs together
TYPES = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
STORAGE = {torch.float32: "<f4", torch.float16: "<f2", torch.bfloat16: "<i2", torch.int32: "<i4", torch.int64: "<i8",
           torch.uint8: "|u1"}


def listed():
    return [
        # one token on every PE of a model with rows of 7168: top-8 of 64 experts, so that most experts have a row or none
        {"name": "experts_token", "op": "experts", "npes": 8, "type": "bfloat16", "tokens": 1, "experts": 64, "topk": 8,
         "dim": 7168, "hidden": 2048, "train": False},
        # a step of a small model, where latency counts
        {"name": "experts_small", "op": "experts", "npes": 4, "type": "half", "tokens": 16, "experts": 16, "topk": 2,
         "dim": 1024, "hidden": 512, "train": False},
        # prompts of 2048 tokens a PE
        {"name": "experts_prefill", "op": "experts", "npes": 8, "type": "bfloat16", "tokens": 2048, "experts": 64, "topk": 8,
         "dim": 7168, "hidden": 2048, "train": False},
        # a ragged batch in training, whose projections are kept; rows that no vector divides
        {"name": "experts_odd", "op": "experts", "npes": 4, "type": "float", "tokens": 501, "experts": 12, "topk": 2,
         "dim": 1029, "hidden": 515, "train": True},
        # the backward pass of a micro-batch; of fine-tuning with rows of a medium size; of a ragged batch in fp32
        {"name": "grad_train", "op": "experts_grad", "npes": 8, "type": "bfloat16", "tokens": 1024, "experts": 32, "topk": 8,
         "dim": 7168, "hidden": 2048},
        {"name": "grad_medium", "op": "experts_grad", "npes": 8, "type": "half", "tokens": 152, "experts": 64, "topk": 4,
         "dim": 2048, "hidden": 1408},
        {"name": "grad_odd", "op": "experts_grad", "npes": 4, "type": "float", "tokens": 152, "experts": 16, "topk": 2,
         "dim": 515, "hidden": 333},
        # one token on every PE, 256 experts in 4 bits; a step of 64 sequences on every PE; and prompts
        {"name": "w4_token", "op": "experts_w4", "npes": 8, "type": "bfloat16", "tokens": 1, "experts": 256, "topk": 8,
         "dim": 7168, "hidden": 2048, "group": 128},
        {"name": "w4_decode", "op": "experts_w4", "npes": 8, "type": "half", "tokens": 64, "experts": 256, "topk": 8,
         "dim": 7168, "hidden": 2048, "group": 64},
        {"name": "w4_prefill", "op": "experts_w4", "npes": 8, "type": "bfloat16", "tokens": 512, "experts": 64, "topk": 8,
         "dim": 7168, "hidden": 2048, "group": 32},
        # behind the combine of a training step, on to the residual; and a ragged batch alone, as its gradient is
        {"name": "dropout_train", "op": "dropout", "npes": 8, "type": "bfloat16", "tokens": 4096, "dim": 7168, "p": 0.1,
         "residual": True},
        {"name": "dropout_odd", "op": "dropout", "npes": 4, "type": "float", "tokens": 501, "dim": 1029, "p": 0.3,
         "residual": False},
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, spread over its logarithm."""
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _ragged(rng, n):
    """Every second size is rounded up to a multiple of 64 elements, the others stay as they fell."""
    return n if rng.random() < 0.5 else (n + 63) // 64 * 64


def draw(rng):
    op = rng.choice(["experts", "experts", "experts_grad", "experts_w4", "dropout"])
    npes, kind = rng.choice([4, 8, 8, 16]), rng.choice(["float", "half", "bfloat16", "bfloat16"])
    size = 4 if kind == "float" else 2
    dim, tokens = _ragged(rng, _spread(rng, 64, 8000)), _spread(rng, 1, 65536 // npes)
    case = {"op": op, "npes": npes, "type": kind, "dim": dim}
    if op == "dropout":
        tokens = max(1, min(tokens, 470_000_000 // (npes * dim * size)))
        return dict(case, tokens=tokens, p=round(rng.uniform(0.02, 0.6), 3), residual=rng.random() < 0.5)
    hidden = _ragged(rng, _spread(rng, 64, 4096))
    expert = 3 * dim * hidden * (0.5 if op == "experts_w4" else size)  # bytes of one's weights
    most = {"experts": 5_000_000_000, "experts_grad": 2_500_000_000, "experts_w4": 5_000_000_000}[op]
    experts = npes * max(1, min(_spread(rng, 1, 256 // npes), int(most / expert) // npes))
    topk = min(experts, rng.choice([1, 2, 4, 6, 8, 8]))
    # at most the work of the largest listed ones; fp32 products run at a tenth of the rate of the others
    work = {"experts": 11e12, "experts_grad": 11e12, "experts_w4": 2.8e12}[op] / (8 if size == 4 else 1)
    flops = npes * topk * dim * hidden * (12 if op == "experts_grad" else 6)
    tokens = max(1, min(tokens, int(work / flops), 2_200_000_000 // (npes * topk * (dim + hidden) * size)))
    case = dict(case, tokens=tokens, experts=experts, topk=topk, hidden=hidden)
    if op == "experts_w4":
        case["group"] = rng.choice([32, 64, 128, 128])
    if op == "experts":
        case["train"] = rng.random() < 0.5
    return case


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
    """What a program keeps: its tensors by name, the sizes, and for the plain form which rows are whose."""

    def __init__(self, case):
        self.case, self.t, self.rows_of = case, {}, []


def _capacity(case):
    """Receive rows of a PE: a quarter more than its share of the copies, and a few for small batches."""
    return case["tokens"] * case["topk"] * 5 // 4 + 64


def _expert_rows(case, g):
    """Where each expert's rows begin on its PE, and the last one's end: a batch whose tokens choose their top-k of logits
    that favour some experts, as after the shuffle's tables."""
    npes, experts = case["npes"], case["experts"]
    logits = torch.randn(npes * case["tokens"], experts, device="cuda", generator=g)
    logits += 0.5 * torch.randn(experts, device="cuda", generator=g)
    counts = torch.bincount(logits.topk(case["topk"], dim=1).indices.reshape(-1), minlength=experts).reshape(npes, -1)
    rows = torch.zeros(npes, experts // npes + 1, dtype=torch.int64, device="cuda")
    rows[:, 1:] = counts.cumsum(1)
    return rows.clamp_(max=_capacity(case))


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    state = _State(case)
    t, npes, tokens, dtype, dim = state.t, case["npes"], case["tokens"], TYPES[case["type"]], case["dim"]
    op = case["op"]

    def make(name, shape, dt):
        t[name] = _tensor(npes, shape, dt)
        return t[name]

    def normal(name, shape, scale):
        for part in make(name, shape, dtype).unbind(0):
            part.normal_(0, scale, generator=g)

    if op == "dropout":
        normal("rows", (tokens, dim), 1.0)
        if case["residual"]:
            normal("residual", (tokens, dim), 1.0)
        # a seed for all PEs, and the number of the step
        make("seed", (2,), torch.int64)[:] = torch.randint(0, 1 << 62, (2,), device="cuda", generator=g)
        make("out", (tokens, dim), dtype)
        if own:
            _bind(state)
        return state
    hidden, cap, mine = case["hidden"], _capacity(case), case["experts"] // npes
    rows = _expert_rows(case, g)
    make("expert_row", (mine + 1,), torch.int64).copy_(rows)
    state.rows_of = [(pe, i, r[i], r[i + 1]) for pe, r in enumerate(rows.tolist()) for i in range(mine) if r[i + 1] > r[i]]
    # rows that no expert has are zeros in all of these
    ends = rows[:, -1].tolist()

    def fill(name, width, scale):
        make(name, (cap, width), dtype)
        for pe in range(npes):
            t[name][pe, :ends[pe]].normal_(0, scale, generator=g)

    fill("rows", dim, 1.0)
    if op == "experts_w4":
        for name, n, k in (("w_in", 2 * hidden, dim), ("w_out", dim, hidden)):
            groups = -(-k // case["group"])
            for part in make(name, (mine, n, (k + 1) // 2), torch.uint8).unbind(0):
                # two values of 0 to 15 a byte, most of them near 8
                q = torch.empty(2, mine, n, (k + 1) // 2, dtype=torch.float16, device="cuda").normal_(8, 2.5, generator=g)
                q = q.round_().clamp_(0, 15).to(torch.uint8)
                part.copy_(q[0] | q[1] << 4)
            for part in make(name + "_scale", (mine, n, groups), dtype).unbind(0):
                part.uniform_(0.2 / math.sqrt(k), 0.6 / math.sqrt(k), generator=g)
        make("out", (cap, dim), dtype)
    else:
        normal("w_in", (mine, 2 * hidden, dim), 1 / math.sqrt(dim))
        normal("w_out", (mine, dim, hidden), 1 / math.sqrt(hidden))
        if op == "experts":
            make("out", (cap, dim), dtype)
            if case["train"]:
                make("pre", (cap, 2 * hidden), dtype)
        else:
            fill("pre", 2 * hidden, 1.0)
            fill("dout", dim, 0.1)
            make("drows", (cap, dim), dtype)
            make("dw_in", (mine, 2 * hidden, dim), dtype)
            make("dw_out", (mine, dim, hidden), dtype)
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
    size, op, npes = C.c_size_t, case["op"], case["npes"]

    def entry(name):
        return getattr(lib, "nvshmemx_amd_%s_%s_on_stream" % (case["type"], name))

    if op == "dropout":
        state.call = entry("dropout"), (a["out"], a["rows"], a.get("residual"), a["seed"], size(case["tokens"]),
                                        size(case["dim"]), case["p"])
        return
    cap, experts, dim, hidden = size(_capacity(case)), case["experts"], size(case["dim"]), size(case["hidden"])
    need = getattr(lib, "nvshmemx_amd_moe_%s_workspace" % ("experts_grad" if op == "experts_grad" else "experts"))
    state.t["workspace"] = _tensor(npes, (need(cap, experts, dim, hidden),), torch.uint8)
    ws = state.t["workspace"].data_ptr()
    if op == "experts":
        state.call = entry("moe_experts"), (a["out"], a.get("pre"), ws, a["rows"], a["w_in"], a["w_out"], a["expert_row"], cap,
                                            experts, dim, hidden)
    elif op == "experts_w4":
        state.call = entry("moe_experts_w4"), (a["out"], ws, a["rows"], a["w_in"], a["w_in_scale"], a["w_out"], a["w_out_scale"],
                                               a["expert_row"], cap, experts, dim, hidden, case["group"])
    else:
        state.call = entry("moe_experts_grad"), (a["drows"], a["dw_in"], a["dw_out"], ws, a["dout"], a["rows"], a["pre"],
                                                 a["w_in"], a["w_out"], a["expert_row"], cap, experts, dim, hidden)


def _outputs(case):
    return {"experts": ["out", "pre"] if case.get("train") else ["out"], "experts_w4": ["out"], "dropout": ["out"],
            "experts_grad": ["drows", "dw_in", "dw_out"]}[case["op"]]


def run(state):
    names = _outputs(state.case)
    if own:
        fn, args = state.call
        if fn(*args, torch.cuda.current_stream().cuda_stream or None):
            raise RuntimeError(state.error().decode())
    else:
        {"experts": _plain_experts, "experts_w4": _plain_experts, "experts_grad": _plain_experts_grad,
         "dropout": _plain_dropout}[state.case["op"]](state)
    return {name: state.t[name] for name in names}


# ------------------------------------------------------------------------------------------------------------
# The plain forms
# ------------------------------------------------------------------------------------------------------------
def _dequantised(packed, scale, k, group):
    """[n, k] values of 4-bit weights: element 2 i in the low half of byte i, 8 stands for 0."""
    q = torch.stack([packed & 15, packed >> 4], 2).reshape(packed.shape[0], -1)[:, :k]
    return (q.float() - 8.0) * scale.float().repeat_interleave(group, 1)[:, :k]


def _weights(state, pe, i):
    """Expert i of PE pe: both input projections below each other, and the output projection, in fp32."""
    t, case = state.t, state.case
    if case["op"] != "experts_w4":
        return t["w_in"][pe, i].float(), t["w_out"][pe, i].float()
    return (_dequantised(t["w_in"][pe, i], t["w_in_scale"][pe, i], case["dim"], case["group"]),
            _dequantised(t["w_out"][pe, i], t["w_out_scale"][pe, i], case["hidden"], case["group"]))


def _plain_experts(state):
    t, hidden = state.t, state.case["hidden"]
    for pe, i, first, end in state.rows_of:
        w_in, w_out = _weights(state, pe, i)
        pre = t["rows"][pe, first:end].float() @ w_in.t()
        gate, up = pre[:, :hidden], pre[:, hidden:]
        h = gate / (1.0 + torch.exp(-gate)) * up
        t["out"][pe, first:end] = (h @ w_out.t()).to(t["out"].dtype)
        if "pre" in t:
            t["pre"][pe, first:end] = pre.to(t["pre"].dtype)


def _plain_experts_grad(state):
    t, hidden, dtype = state.t, state.case["hidden"], state.t["rows"].dtype
    busy = set()
    for pe, i, first, end in state.rows_of:
        busy.add((pe, i))
        w_in, w_out = _weights(state, pe, i)
        x, dout, pre = (t[name][pe, first:end].float() for name in ("rows", "dout", "pre"))
        gate, up = pre[:, :hidden], pre[:, hidden:]
        s = 1.0 / (1.0 + torch.exp(-gate))
        silu = gate * s
        dh = dout @ w_out
        dpre = torch.cat([dh * up * s * (1.0 + gate * (1.0 - s)), dh * silu], 1)
        t["drows"][pe, first:end] = (dpre @ w_in).to(dtype)
        t["dw_in"][pe, i] = (dpre.t() @ x).to(dtype)
        t["dw_out"][pe, i] = (dout.t() @ (silu * up)).to(dtype)
    for pe in range(state.case["npes"]):
        for i in range(t["dw_in"].shape[1]):
            if (pe, i) not in busy:
                t["dw_in"][pe, i].zero_()
                t["dw_out"][pe, i].zero_()


MULTIPLIERS, KEY_STEPS, ROUNDS = (0xD2511F53, 0xCD9E8D57), (0x9E3779B9, 0xBB67AE85), 10


def _philox(counter, key):
    """Philox4x32-10 (Salmon, Moraes, Dror and Shaw, 2011): four words of 32 bits for each counter of four, as int64."""
    low = 0xFFFFFFFF
    c, k = list(counter), list(key)
    for _ in range(ROUNDS):
        products = [c[0] * MULTIPLIERS[0], c[2] * MULTIPLIERS[1]]  # (modulo 2^64, which keeps all bits)
        high = [p >> 32 & low for p in products]
        c = [high[1] ^ c[1] ^ k[0], products[1] & low, high[0] ^ c[3] ^ k[1], products[0] & low]
        k = [(v + step) & low for v, step in zip(k, KEY_STEPS)]
    return c


def _kept(case, seed, pe):
    """Which elements of PE pe's rows stay, as [tokens, dim]: element e has 16 bits of the block e / 8, e % 8 of it in
    ascending order, and is dropped where they are less than p * 2^16, rounded."""
    n = case["tokens"] * case["dim"]
    block = torch.arange(-(-n // 8), device="cuda", dtype=torch.int64)
    word = torch.zeros_like(block)
    low = 0xFFFFFFFF
    words = _philox([block & low, (block >> 32) + (pe << 16), word + (seed[1] & low), word + (seed[1] >> 32 & low)],
                    [seed[0] & low, seed[0] >> 32 & low])
    words = torch.stack(words, 1)
    bits = torch.stack([words & 0xFFFF, words >> 16], 2).reshape(-1)[:n]
    return (bits >= int(round(case["p"] * 65536))).reshape(case["tokens"], case["dim"])


def _plain_dropout(state):
    t, case = state.t, state.case
    scale = 1.0 / (1.0 - int(round(case["p"] * 65536)) / 65536)
    for pe in range(case["npes"]):
        y = torch.where(_kept(case, t["seed"][pe], pe), t["rows"][pe].float() * scale, 0.0)
        if case["residual"]:
            y += t["residual"][pe].float()
        t["out"][pe] = y.to(t["out"].dtype)


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
    t, op, npes = state.t, case["op"], case["npes"]
    if op == "dropout":
        out = []
        limit = math.floor(case["p"] * 65536 + 0.5)
        for pe in range(npes):
            keep = _kept(case, t["seed"][pe], pe).double()  # (which elements stay is the generator's definition)
            y = t["rows"][pe].double() * keep * (65536.0 / (65536 - limit))
            out.append(y + t["residual"][pe].double() if case["residual"] else y)
        return {"out": torch.stack(out)}
    hidden, double = case["hidden"], torch.float64
    values = {name: torch.zeros(t[name].shape, dtype=double, device="cuda") for name in _outputs(case)}

    def four_bits(name, pe, i, k):
        n, group = t[name].shape[2], case["group"]
        w = torch.empty(n, t[name].shape[3] * 2, dtype=double, device="cuda")
        w[:, 0::2] = t[name][pe, i] % 16
        w[:, 1::2] = t[name][pe, i] // 16
        column = torch.arange(k, device="cuda") // group
        return (w[:, :k] - 8) * t[name + "_scale"][pe, i].double()[:, column]

    for pe, i, first, end in state.rows_of:
        if op == "experts_w4":
            w_in, w_out = four_bits("w_in", pe, i, case["dim"]), four_bits("w_out", pe, i, hidden)
        else:
            w_in, w_out = t["w_in"][pe, i].double(), t["w_out"][pe, i].double()
        x = t["rows"][pe, first:end].double()
        if op != "experts_grad":
            gate, up = torch.mm(x, w_in[:hidden].T), torch.mm(x, w_in[hidden:].T)
            values["out"][pe, first:end] = torch.mm(gate * torch.sigmoid(gate) * up, w_out.T)
            if "pre" in values:
                values["pre"][pe, first:end, :hidden] = gate
                values["pre"][pe, first:end, hidden:] = up
            continue
        # <dout, out> differentiated, once the projections are known
        pre = t["pre"][pe, first:end].double().requires_grad_()
        h = torch.nn.functional.silu(pre[:, :hidden]) * pre[:, hidden:]
        dout = t["dout"][pe, first:end].double()
        dpre = torch.autograd.grad(h, pre, torch.mm(dout, w_out))[0]
        values["drows"][pe, first:end] = torch.mm(dpre, w_in)
        values["dw_in"][pe, i] = torch.mm(dpre.T.contiguous(), x)
        values["dw_out"][pe, i] = torch.mm(dout.T.contiguous(), h.detach())
    return values


# ------------------------------------------------------------------------------------------------------------
def work(case):
    """What a pass cannot do without: every input read once, every output written once.  Of the weights, those of the
    experts that tokens chose, when each chooses among all of them alike."""
    npes, dim, size = case["npes"], case["dim"], TYPES[case["type"]].itemsize
    tokens = npes * case["tokens"]
    if case["op"] == "dropout":
        return {"bytes": tokens * dim * size * (3 if case["residual"] else 2), "flops": 2 * tokens * dim}
    hidden, rows, experts = case["hidden"], tokens * case["topk"], case["experts"]
    busy = experts * (1.0 - (1.0 - case["topk"] / experts) ** tokens)
    weights = 3 * dim * hidden * size
    product = 2 * rows * dim * hidden
    if case["op"] == "experts":
        return {"bytes": busy * weights + rows * (2 * dim + (2 * hidden if case["train"] else 0)) * size, "flops": 3 * product}
    if case["op"] == "experts_w4":
        group = case["group"]
        scales = (2 * hidden * -(-dim // group) + dim * -(-hidden // group)) * size
        return {"bytes": busy * (3 * dim * hidden / 2 + scales) + 2 * rows * dim * size, "flops": 3 * product}
    return {"bytes": (busy + experts) * weights + rows * (3 * dim + 2 * hidden) * size, "flops": 6 * product}
