"""Symmetric arrays of the token operators' types, with guard bytes around them."""
import numpy as np
import torch

TORCH = {"float": torch.float32, "half": torch.float16, "bfloat16": torch.bfloat16}
EPS = {t: torch.finfo(d).eps for t, d in TORCH.items()}
TINY = {"float": 2.0 ** -150, "half": 2.0 ** -25, "bfloat16": 2.0 ** -134}   # half of the smallest number
SIZE = {"float": 4, "half": 2, "bfloat16": 2, "int32": 4, "int64": 8, "byte": 1}
NUMPY = {"int32": np.int32, "int64": np.int64, "byte": np.uint8}
GUARD, SENTINEL = 256, 0xA5


def rounded(values, kind):
    """The values as `kind` holds them, in fp32."""
    return torch.from_numpy(np.ascontiguousarray(values, np.float32)).to(TORCH[kind]).float().numpy()


class Sym:
    """A symmetric array, `shift` elements behind a boundary of 256 bytes, in front of and behind it guard bytes."""

    def __init__(self, rt, kind, shape, values=None, shift=0):
        self.rt, self.kind, self.shape = rt, kind, tuple(shape)
        self.first = GUARD + shift * SIZE[kind]
        self.bytes = int(np.prod(self.shape, dtype=np.int64)) * SIZE[kind]
        self.total = self.first + self.bytes + GUARD
        self.base = rt.malloc(self.total)
        self.address = self.base + self.first
        rt.fill(self.base, SENTINEL, self.total)
        if values is not None:
            self.put(values)

    def put(self, values):
        values = np.broadcast_to(values, (self.rt.npes,) + self.shape)
        if self.bytes == 0:
            return
        for pe in range(self.rt.npes):
            if self.kind in TORCH:
                data = torch.from_numpy(np.array(values[pe], np.float32)).to(TORCH[self.kind])
                data = data.view(torch.int32 if self.kind == "float" else torch.int16).numpy()
            else:
                data = np.ascontiguousarray(values[pe], NUMPY[self.kind])
            self.rt.upload(self.base, pe, data, self.first)

    def raw(self):
        return self.rt.download_all(self.base, (self.total,), np.uint8)

    def get(self):
        """[npes, *shape] values; the bytes around them have to be as they were."""
        raw = self.raw()
        assert (raw[:, :self.first] == SENTINEL).all() and (raw[:, self.first + self.bytes:] == SENTINEL).all(), "guard"
        data = np.ascontiguousarray(raw[:, self.first:self.first + self.bytes])
        if self.kind in TORCH:
            out = torch.from_numpy(data).view(TORCH[self.kind]).float().numpy()
        else:
            out = data.view(NUMPY[self.kind])
        return out.reshape((self.rt.npes,) + self.shape)

    def free(self):
        self.rt.free(self.base)


class Arrays:
    """Makes arrays and frees them together."""

    def __init__(self, rt):
        self.rt, self.all = rt, []

    def __enter__(self):
        return self

    def __call__(self, kind, shape, values=None, shift=0):
        self.all.append(Sym(self.rt, kind, shape, values, shift))
        return self.all[-1]

    def workspace(self, *sizes):
        return self("byte", (self.rt.workspace_bytes(*sizes),))

    def __exit__(self, *exc):
        for a in self.all:
            a.free()


def close(got, want, tolerance, what=""):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    tolerance = np.broadcast_to(tolerance, want.shape)
    bad = ~(np.abs(got - want) <= tolerance)
    bad &= ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if bad.any():
        at = tuple(np.argwhere(bad)[0])
        raise AssertionError("%s: %d of %d are off, first at %s: %r instead of %r, tolerance %r"
                             % (what, bad.sum(), bad.size, at, got[at], want[at], tolerance[at]))
