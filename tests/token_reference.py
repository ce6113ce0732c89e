"""The operators on rows of tokens in 64 bits, straight from their definitions, over [npes, ...] arrays."""
import numpy as np

STEP = 2.0 ** -24   # half a step of fp32, relative: what one rounding is off by at most


def live(logits):
    return logits > -np.inf      # (a NaN is not)


def softmax(logits):
    ok = live(logits)
    with np.errstate(invalid="ignore", over="ignore"):
        x = np.where(ok, logits.astype(np.float64), -np.inf)
        m = x.max(-1, keepdims=True)
        e = np.where(ok, np.exp(np.where(x == m, 0.0, x - m)), 0.0)
    z = e.sum(-1, keepdims=True)
    return np.where(z > 0, e / np.where(z > 0, z, 1.0), 0.0)


def route(logits, topk, normalise, scale):
    """expert, gate, counts, loss, balance"""
    npes, tokens, experts = logits.shape
    ok, p = live(logits), softmax(logits)
    expert = np.full((npes, tokens, topk), -1, np.int32)
    gate = np.zeros((npes, tokens, topk))
    for pe in range(npes):
        for t in range(tokens):
            x = logits[pe, t].astype(np.float64)
            order = sorted((e for e in range(experts) if ok[pe, t, e]), key=lambda e: (-x[e], e))[:topk]
            expert[pe, t, :len(order)] = order
            if order:
                if normalise:    # against the largest, whose weight is 1
                    with np.errstate(invalid="ignore"):
                        w = np.exp(np.where(x[order] == x[order[0]], 0.0, x[order] - x[order[0]]))
                    gate[pe, t, :len(order)] = scale * w / w.sum()
                else:
                    gate[pe, t, :len(order)] = scale * p[pe, t, order]
    counts = np.stack([np.bincount(expert[pe][expert[pe] >= 0], minlength=experts) for pe in range(npes)]).astype(np.int64)
    c, n = counts.sum(0).astype(np.float64), ok.any(-1).sum()
    balance = experts * c / (c.sum() * n) if n else np.zeros(experts)
    return expert, gate, counts, float((balance * p.sum((0, 1))).sum()), balance


def route_value(logits, expert, dgate, balance, dloss, normalise, scale):
    """The number whose gradient by the logits route_grad gives."""
    p = softmax(logits)
    some = expert >= 0
    w = np.where(some, np.take_along_axis(p, np.maximum(expert, 0).astype(np.int64), 2), 0.0)
    if normalise:
        s = w.sum(2, keepdims=True)
        w = np.where(some, w / np.where(s > 0, s, 1.0), 0.0)
    value = scale * (w * dgate).sum()
    if balance is not None:
        value += (dloss * (balance[:, None] * p).sum((1, 2))).sum()
    return value


def route_grad(logits, expert, dgate, balance, dloss, normalise, scale):
    """dlogits, and the sum of the magnitudes that it is made of."""
    npes, tokens, experts = logits.shape
    p = softmax(logits)
    ok = live(logits)
    q = np.zeros(logits.shape) if balance is None else np.broadcast_to((dloss[:, None] * balance)[:, None, :], logits.shape).copy()
    d, size = np.zeros(logits.shape), np.zeros(logits.shape)
    for pe in range(npes):
        for t in range(tokens):
            chosen = [(k, e) for k, e in enumerate(expert[pe, t]) if e >= 0 and ok[pe, t, e]]
            qt, extra, extra_size = q[pe, t].copy(), np.zeros(experts), np.zeros(experts)
            if chosen:
                k, e = (np.array(v) for v in zip(*chosen))
                g = scale * dgate[pe, t, k].astype(np.float64)
                if normalise:
                    x = logits[pe, t, e].astype(np.float64)
                    with np.errstate(invalid="ignore"):
                        w = np.exp(np.where(x == x.max(), 0.0, x - x.max()))
                    w /= w.sum()
                    extra[e] = w * (g - (w * g).sum())
                    extra_size[e] = w * (np.abs(g) + (w * np.abs(g)).sum())
                else:
                    qt[e] += g
            d[pe, t] = p[pe, t] * (qt - (qt * p[pe, t]).sum()) + extra
            size[pe, t] = p[pe, t] * (np.abs(qt) + (np.abs(qt) * p[pe, t]).sum()) + extra_size
    return d, size


def place(expert, experts, cap):
    """dest_pe, dest_row, expected, expert_row"""
    npes, tokens, topk = expert.shape
    per_pe = experts // npes
    dest_pe = np.full(expert.shape, -1, np.int32)
    dest_row = np.full(expert.shape, -1, np.int64)
    expected = np.zeros((npes, npes), np.int64)
    expert_row = np.zeros((npes, per_pe + 1), np.int64)
    for pe in range(npes):
        row = 0
        for i in range(per_pe):
            expert_row[pe, i] = min(row, cap)
            for src in range(npes):
                for t, k in zip(*np.nonzero(expert[src] == pe * per_pe + i)):
                    if row < cap:
                        dest_pe[src, t, k], dest_row[src, t, k] = pe, row
                        expected[pe, src] += 1
                    row += 1
        expert_row[pe, per_pe] = min(row, cap)
    return dest_pe, dest_row, expected, expert_row


def kept(dest_pe, dest_row, npes, cap):
    return (dest_pe >= 0) & (dest_pe < npes) & (dest_row >= 0) & (dest_row < cap)


def copies(recv, dest_pe, dest_row):
    """Every copy's row, zeros where it was skipped."""
    ok = kept(dest_pe, dest_row, *recv.shape[:2])
    return np.where(ok[..., None], recv[np.where(ok, dest_pe, 0), np.where(ok, dest_row, 0)].astype(np.float64), 0.0), ok


def combine_sum(recv, gate, dest_pe, dest_row):
    """out, and the sum of the magnitudes that it is made of."""
    rows, ok = copies(recv, dest_pe, dest_row)
    w = np.where(ok, 1.0 if gate is None else gate.astype(np.float64), 0.0)[..., None]
    return (w * rows).sum(2), np.abs(w * rows).sum(2)


def combine_grad(drecv, dout, recv, gate, dest_pe, dest_row):
    """drecv with the named rows replaced, dgate, and the sum of magnitudes of dgate."""
    rows, ok = copies(recv, dest_pe, dest_row)
    product = rows * dout.astype(np.float64)[:, :, None, :]
    drecv = drecv.astype(np.float64).copy()
    for pe, t, k in zip(*np.nonzero(ok)):
        drecv[dest_pe[pe, t, k], dest_row[pe, t, k]] = gate[pe, t, k].astype(np.float64) * dout[pe, t]
    return drecv, product.sum(-1), np.abs(product).sum(-1)


def embedding_grad(dtable, dout, ids, vocab, scale):
    """dtable with the vocabulary's rows replaced, the sum of magnitudes, and how many tokens name each row."""
    npes, rows, dim = dtable.shape
    flat = dtable.astype(np.float64).reshape(-1, dim).copy()
    size, n = np.zeros_like(flat), np.zeros(npes * rows, np.int64)
    flat[:vocab] = 0.0
    ok = (ids >= 0) & (ids < vocab)
    np.add.at(flat, ids[ok], scale * dout[ok].astype(np.float64))
    np.add.at(size, ids[ok], abs(scale) * np.abs(dout[ok].astype(np.float64)))
    np.add.at(n, ids[ok], 1)
    return flat.reshape(dtable.shape), size.reshape(dtable.shape), n.reshape(npes, rows)


# ---- the same for batches that are too large to go through token by token ----

def route_many(logits, topk, normalise, scale):
    """route(), over whole arrays."""
    npes, tokens, experts = logits.shape
    ok, p = live(logits), softmax(logits)
    x = np.where(ok, logits.astype(np.float64), -np.inf)
    order = np.argsort(-x, axis=2, kind="stable")[..., :topk]
    chosen = np.take_along_axis(ok, order, 2)
    if normalise:
        l = np.take_along_axis(x, order, 2)
        with np.errstate(invalid="ignore"):
            w = np.where(chosen, np.exp(np.where(l == l[..., :1], 0.0, l - l[..., :1])), 0.0)
        w /= np.maximum(w.sum(2, keepdims=True), 1.0)
    else:
        w = np.where(chosen, np.take_along_axis(p, order, 2), 0.0)
    expert = np.where(chosen, order, -1).astype(np.int32)
    counts = np.stack([np.bincount(e[e >= 0], minlength=experts) for e in expert]).astype(np.int64)
    c, n = counts.sum(0).astype(np.float64), ok.any(-1).sum()
    balance = experts * c / (c.sum() * n) if n else np.zeros(experts)
    return expert, scale * w, counts, float((balance * p.sum((0, 1))).sum()), balance


def route_grad_many(logits, expert, dgate, balance, dloss, normalise, scale):
    """route_grad(), over whole arrays."""
    ok, p, experts = live(logits), softmax(logits), logits.shape[2]
    at = np.maximum(expert, 0).astype(np.int64)
    chosen = (expert >= 0) & np.take_along_axis(ok, at, 2)
    g = np.where(chosen, scale * dgate.astype(np.float64), 0.0)

    def spread(values):             # from a token's chosen ones to all of its experts, and those behind the last for none
        out = np.zeros(logits.shape[:2] + (experts + 1,))
        np.put_along_axis(out, np.where(chosen, at, experts), np.where(chosen, values, 0.0), 2)
        return out[..., :experts]

    q = np.zeros((1, 1, 1)) if balance is None else (dloss[:, None] * balance)[:, None, :]
    extra = extra_size = 0.0
    if normalise:
        l = np.where(chosen, np.take_along_axis(logits, at, 2).astype(np.float64), -np.inf)
        m = l.max(2, keepdims=True)
        with np.errstate(invalid="ignore"):
            w = np.where(chosen, np.exp(np.where(l == m, 0.0, l - m)), 0.0)
        w /= np.maximum(w.sum(2, keepdims=True), 1.0)
        extra = spread(w * (g - (w * g).sum(2, keepdims=True)))
        extra_size = spread(w * (np.abs(g) + (w * np.abs(g)).sum(2, keepdims=True)))
    else:
        q = q + spread(g)
    d = p * (q - (q * p).sum(2, keepdims=True)) + extra
    return d, p * (np.abs(q) + (np.abs(q) * p).sum(2, keepdims=True)) + extra_size
