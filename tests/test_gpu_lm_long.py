"""More rows' parts than a launch has workgroups (2^20), and rows past 2^32 elements: what follows logits, on the GPU."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from . import lm_ref as lm
from .dense_ref import BF16, F32, Pool, assert_within, buf
from .test_gpu_lm_distillation import check as check_distillation
from .test_gpu_lm_distillation import evaluate, teacher
from .test_gpu_lm_log_probs import make, run_backward

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


MORE = (1 << 20) + 21  # rows of a group each


@pytest.mark.parametrize("kind", [F32, BF16])
def test_short_rows_of_more_than_workgroups(pool, kind):
    classes = 3
    z = make(kind, MORE, classes, classes)
    t, l = teacher(MORE, 2, classes)
    check_distillation(pool, kind, z, classes, 1.0, t, l)
    check_distillation(pool, kind, z, classes, 1.0, t, l, want_delta=False)
    run_backward(pool, kind, z, classes, 1.0, np.arange(2 * MORE, dtype=np.int32).reshape(MORE, 2) % 4, True)


# A workgroup a row, of 1.2 or 2.3 G elements; and 17 parts a row.
@pytest.mark.parametrize("kind,rows,classes", [(F32, MORE, 1100), (BF16, MORE, 2200), (F32, 61700, 65540), (BF16, 61700, 131080)])
def test_long_rows_of_more_than_workgroups(pool, kind, rows, classes):
    """Distillation, log probabilities with alternatives, and their delta with the entropy's onto the logits."""
    z = Rows(make(kind, PERIOD, classes, classes), kind, rows)
    try:
        every = -(-rows // PERIOD)
        one = np.arange(PERIOD, dtype=np.int32)[:, None] * 7 + np.array([[0, 5]], np.int32)
        tokens = pool(np.tile(one, (every, 1))[:rows])
        lp, h, stats = pool(n=(rows, 2)), pool(n=rows), pool(n=(rows, 2))
        tt, tl = pool(np.zeros((rows, 3), np.int32)), pool(n=(rows, 3))
        ws = pool.work(gpu.tokenLogProbsWorkspace(kind, rows, classes, 3))
        gpu.tokenLogProbs(kind, rows, classes, classes, z.buf, 1.5, 2, tokens.buf, 3, lp.buf, h.buf, stats.buf, tt.buf, tl.buf, buf(ws))
        s = lm.Softmax(z.values, 1.5)
        at = np.arange(PERIOD)[:, None]
        assert_within(lp.get()[:PERIOD], *s.log_prob(at, one), "log_probs")
        assert_within(h.get()[:PERIOD], s.h, s.h_err, "entropy")
        assert (tt.get()[:PERIOD] == np.stack([lm.best(v, 3) for v in z.values])).all()
        assert all(repeats(x.get()) for x in (lp, h, stats, tt, tl))

        if rows == MORE:  # held rows (those in parts are above)
            t, l = teacher(PERIOD, 70, classes)
            dt, dl, loss = pool(np.tile(t, (every, 1))[:rows]), pool(np.tile(l, (every, 1))[:rows]), pool(n=rows)
            want, err, _, _ = evaluate(z.values, classes, 1.5, t, l, np.ones(PERIOD, np.float32))
            gpu.distillation(kind, rows, classes, classes, z.buf, 1.5, 70, dt.buf, dl.buf, None, 1.0, loss.buf, None, None)
            got = loss.get()
            assert_within(got[:PERIOD], want, err, "loss")
            assert repeats(got)

        a, e = np.float32(0.75), np.float32(-0.5)
        da, de = pool(np.full((rows, 2), a, np.float32)), pool(np.full(rows, e, np.float32))
        gpu.tokenLogProbsBackward(kind, rows, classes, classes, z.buf, 1.5, 2, tokens.buf, stats.buf, h.buf, da.buf, de.buf, 0.0, z.buf)
        q = 2 * a + e * (s.lp + s.h[:, None])
        d = -s.p * q
        d[at, one] += a
        # As in run_backward, and the forward's l and h are off by their own errors.
        off = s.l_err[:, None]
        q_err = np.abs(e) * (lm.U * (6 * np.abs(s.y) + 8 * np.abs(s.lp) + 6 * np.abs(s.h)[:, None]) + off + s.h_err[:, None]) + 8 * lm.U
        d_err = s.p * (np.abs(q) * (lm.probability_error(s.y, s.l) + off + 4 * lm.U) + q_err) + 8 * lm.U * np.abs(d) + 2.0**-110
        check_windows(z, rows, d / 1.5, d_err / 1.5)
    finally:
        gpu.free(z.buf)


@pytest.mark.parametrize("kind,classes", [(F32, 1100), (BF16, 2200)])
def test_deltas_of_held_rows_of_more_than_workgroups(pool, kind, classes):
    z = Rows(make(kind, PERIOD, classes, classes), kind, MORE)
    try:
        t, l = teacher(PERIOD, 70, classes)
        every = -(-MORE // PERIOD)
        dt, dl, loss = pool(np.tile(t, (every, 1))[:MORE]), pool(np.tile(l, (every, 1))[:MORE]), pool(n=MORE)
        _, _, d, d_err = evaluate(z.values, classes, 0.75, t, l, np.full(PERIOD, np.float32(2)))
        gpu.distillation(kind, MORE, classes, classes, z.buf, 0.75, 70, dt.buf, dl.buf, None, 2.0, loss.buf, z.buf, None)
        assert repeats(loss.get())
        check_windows(z, MORE, d, d_err)
    finally:
        gpu.free(z.buf)
