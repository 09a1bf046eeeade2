"""More rows' parts than a launch has workgroups (2^20), and rows past 2^32 elements: what follows logits, on the GPU."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from . import lm_ref as lm
from .dense_ref import BF16, F32, Pool, assert_within, buf
from .test_gpu_lm_distillation import evaluate, teacher
from .test_gpu_lm_log_probs import make

pytestmark = pytest.mark.gpu

PERIOD = 16  # rows after which everything repeats, and results have to


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


class Rows:
    """`rows` rows of a period's `values` [PERIOD, n], of 16-byte rows so that every period is read alike."""

    def __init__(self, values, kind, rows):
        raw = np.ascontiguousarray(ref.to_bf16(values) if kind == BF16 else values.astype(np.float32)).view(np.int32)
        self.kind, self.words, self.values = kind, raw.shape[1], values
        assert self.words % 4 == 0
        self.buf = gpu.alloc(rows * self.words)
        gpu.push(self.buf.offset(0), raw.ravel())
        done = PERIOD
        while done < rows:
            n = min(done, rows - done, (1 << 30) // self.words // PERIOD * PERIOD)
            gpu.copy(n * self.words, self.buf, self.buf.offset(done * self.words))
            done += n

    def pull(self, first, n=PERIOD):
        back = np.empty((n, self.words), np.int32)
        gpu.pull(self.buf.offset(first * self.words), back)
        return ref.from_bf16(back.view(np.uint16)) if self.kind == BF16 else back.view(np.float32)


def repeats(values):
    """Whether every period's values are the first one's, bit for bit."""
    v = np.ascontiguousarray(values).view(np.uint32).reshape(len(values), -1)
    whole = len(v) // PERIOD * PERIOD
    return (v[:whole].reshape(-1, PERIOD, v.shape[1]) == v[:PERIOD]).all() and (v[whole:] == v[: len(v) - whole]).all()


def check_windows(z, rows, want, err):
    for first in (0, rows // 2 // PERIOD * PERIOD, (rows - PERIOD) // PERIOD * PERIOD):
        got = z.pull(first)
        assert_within(got, want, err + lm.rounding(z.kind) * (np.abs(want) + err), f"rows from {first}")


# Rows in 17 parts, 1048900 of them; of 8.1 or 4.0 G elements.
@pytest.mark.parametrize("kind,rows,classes", [(F32, 61700, 65540), (BF16, 61700, 131080)])
def test_distillation_of_more_parts_than_workgroups(pool, kind, rows, classes):
    z = Rows(make(kind, PERIOD, classes, classes), kind, rows)
    try:
        t, l = teacher(PERIOD, 70, classes)
        every = -(-rows // PERIOD)
        dt, dl, loss = pool(np.tile(t, (every, 1))[:rows]), pool(np.tile(l, (every, 1))[:rows]), pool(n=rows)
        ws = pool.work(gpu.distillationWorkspace(kind, rows, classes))
        want, err, d, d_err = evaluate(z.values, classes, 1.5, t, l, np.full(PERIOD, np.float32(0.5)))
        for delta in (None, z.buf):
            gpu.distillation(kind, rows, classes, classes, z.buf, 1.5, 70, dt.buf, dl.buf, None, 0.5, loss.buf, delta, buf(ws))
            got = loss.get()
            assert_within(got[:PERIOD], want, err, "loss")
            assert repeats(got)
        check_windows(z, rows, d, d_err)
    finally:
        gpu.free(z.buf)
