"""References in 64 bits and device buffers for the dense operators' tests."""

from __future__ import annotations

import numpy as np

from darknet_zig_amd import gpu

F32, BF16 = gpu.F32, gpu.BF16
LOGISTIC, RELU, LINEAR, TANH, LEAKY, ELU, SELU = 0, 1, 3, 5, 7, 8, 13
# Half a step of a stored value, relative to it.
HALF = {F32: 2.0**-24, BF16: 2.0**-8}


def to_bf16(a: np.ndarray) -> np.ndarray:
    """fp32 to bf16 bits, to nearest even; a NaN stays one."""
    u = np.ascontiguousarray(a, np.float32).view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> np.uint64(16)) & np.uint64(1))) >> np.uint64(16)).astype(np.uint16)
    return np.where(np.isnan(a), np.uint16(0x7FC0), r).reshape(np.shape(a))


def from_bf16(b: np.ndarray) -> np.ndarray:
    return (b.astype(np.uint32) << np.uint32(16)).view(np.float32)


def rounded(a, kind: int) -> np.ndarray:
    """fp32 values that `kind` holds exactly."""
    a = np.asarray(a, np.float32)
    return from_bf16(to_bf16(a)) if kind == BF16 else a


class Dev:
    """A device array of `kind` (or fp32 / int32 for kind None), between guard bytes; `shift` elements off its alignment."""

    GUARD = 64

    def __init__(self, values=None, kind=None, n: int = 0, shift: int = 0):
        if values is not None:
            v = np.ascontiguousarray(values)
            raw = to_bf16(v) if kind == BF16 else v if v.dtype == np.int32 else v.astype(np.float32)
            self.shape, self.dtype = v.shape, raw.dtype
        else:
            self.shape, self.dtype = (n,) if np.isscalar(n) else tuple(n), np.dtype(np.uint16 if kind == BF16 else np.float32)
            raw = np.full(self.shape, 0x5A5A5A5A & (0xFFFF if kind == BF16 else 0xFFFFFFFF),
                          np.uint16 if kind == BF16 else np.uint32).view(self.dtype)
        self.kind, self.nbytes = kind, raw.nbytes
        self.at = self.GUARD + shift * raw.dtype.itemsize
        total = (self.at + raw.nbytes + self.GUARD + 3) // 4 * 4
        self.host = np.full(total, 0xA5, np.uint8)
        self.host[self.at : self.at + raw.nbytes] = np.frombuffer(raw.tobytes(), np.uint8)
        self.base = gpu.make(self.host.view(np.int32))
        self.buf = gpu.Buf(self.base.ptr + self.at, (raw.nbytes + 3) // 4)

    def raw(self) -> np.ndarray:
        """The array's elements; the bytes around them have to be as they were."""
        back = np.empty_like(self.host)
        gpu.pull(self.base, back.view(np.int32))
        lo, hi = self.at, self.at + self.nbytes
        assert (back[:lo] == 0xA5).all() and (back[hi:] == 0xA5).all(), "written outside the tensor"
        return np.frombuffer(back[lo:hi].tobytes(), self.dtype).reshape(self.shape)

    def get(self) -> np.ndarray:
        r = self.raw()
        return from_bf16(r) if self.kind == BF16 else r

    def free(self) -> None:
        gpu.free(self.base)


class Pool:
    """Frees what a test made."""

    def __init__(self):
        self.made = []

    def __call__(self, *a, **k) -> Dev:
        self.made.append(Dev(*a, **k))
        return self.made[-1]

    def work(self, nbytes: int):
        """A workspace of exactly `nbytes` (rounded up to 4) and its guard."""
        return self(n=(nbytes + 3) // 4) if nbytes else None

    def free(self):
        for d in self.made:
            d.free()


def buf(d):
    return None if d is None else d.buf


# ---- draws ----


def _hash(x: np.ndarray) -> np.ndarray:
    x = x.astype(np.uint32)
    x = (x ^ (x >> np.uint32(16))) * np.uint32(0x7FEB352D)
    x = (x ^ (x >> np.uint32(15))) * np.uint32(0x846CA68B)
    return x ^ (x >> np.uint32(16))


def dropped(n: int, prob: float, seed: int, first: int) -> np.ndarray:
    j = np.arange(n, dtype=np.uint64) + np.uint64(first)
    high = ((j >> np.uint64(32)) * np.uint64(0x9E3779B9)).astype(np.uint32)
    u = _hash(np.uint32(seed) ^ _hash(j.astype(np.uint32)) ^ _hash(high))
    return (u >> np.uint32(8)).astype(np.float32) * np.float32(2.0**-24) < np.float32(prob)


# ---- activations, in 64 bits ----


def activate(act: int, z: np.ndarray) -> np.ndarray:
    with np.errstate(over="ignore"):
        return {
            LOGISTIC: lambda: 1 / (1 + np.exp(-z)),
            RELU: lambda: np.where(z > 0, z, 0.0),
            LINEAR: lambda: z,
            TANH: lambda: np.tanh(z),
            LEAKY: lambda: np.where(z > 0, z, float(np.float32(0.1)) * z),
            ELU: lambda: np.where(z >= 0, z, np.expm1(np.minimum(z, 0))),
            SELU: lambda: np.where(z >= 0, float(np.float32(1.0507)) * z, float(np.float32(1.75803124)) * np.expm1(np.minimum(z, 0))),
        }[act]()


def gradient(act: int, y: np.ndarray) -> np.ndarray:
    return {
        LOGISTIC: lambda: (1 - y) * y,
        RELU: lambda: np.where(y > 0, 1.0, 0.0),
        LINEAR: lambda: np.ones_like(y),
        TANH: lambda: 1 - y * y,
        LEAKY: lambda: np.where(y > 0, 1.0, float(np.float32(0.1))),
        ELU: lambda: np.where(y >= 0, 1.0, y + 1),
        SELU: lambda: np.where(y >= 0, float(np.float32(1.0507)), y + float(np.float32(1.75803124))),
    }[act]()


# Largest slope of an activation, and the rounding errors of its fp32 evaluation relative to 1 + |value|
# (an exponential, a division and a few sums: at most eight roundings).
SLOPE = {LOGISTIC: 0.25, RELU: 1, LINEAR: 1, TANH: 1, LEAKY: 1, ELU: 1, SELU: 1.7581}
ACT_ROUNDINGS = 8


def assert_within(got, want, bound, what: str):
    got, want = np.asarray(got, np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape, (what, got.shape, want.shape)
    bad = ~(np.abs(got - want) <= bound) & ~((got == want) | (np.isnan(got) & np.isnan(want)))
    if bad.any():
        i = np.argwhere(bad)[:5]
        b = np.broadcast_to(bound, got.shape)
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.size} outside; first " + ", ".join(
            f"{tuple(int(x) for x in p)}: {got[tuple(p)]!r} for {want[tuple(p)]!r} +- {b[tuple(p)]!r}" for p in i))


def product_error(a: np.ndarray, b: np.ndarray) -> np.ndarray:
    """Bound on an fp32 evaluation of a @ b: each of the k products and sums rounds by 2^-24 of a partial sum,
    which is at most the sum of magnitudes (bf16 products are exact; the split fp32 ones are within 2^-24 of it)."""
    k = a.shape[1]
    return (k + 2) * 2.0**-24 * (np.abs(a) @ np.abs(b))
