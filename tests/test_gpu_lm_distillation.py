"""Distillation from a teacher's top logits (dkz_distillation) on the GPU, against its formulas in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from . import lm_cases as cases
from . import lm_ref as lm
from .dense_ref import BF16, F32, Pool, assert_within, buf
from .test_gpu_lm_log_probs import make

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


def teacher(rows, top, classes, seed=5):
    """Entries, some of them none, some classes twice; the third row has no entry."""
    r = np.random.default_rng(seed + top)
    t = r.integers(0, classes, (rows, top)).astype(np.int32)
    t.ravel()[2::9] = -1
    t.ravel()[4::13] = classes
    if top > 4:
        t[:, 3] = t[:, 0]
    if rows > 2:
        t[2] = -1
    return t, (r.normal(size=(rows, top)) * 2).astype(np.float32)


def evaluate(z, classes, temperature, tokens, logits, scales):
    """loss, delta and bounds of theirs, in 64 bits."""
    s = lm.Softmax(z[:, :classes], temperature)
    rows, top = tokens.shape
    t = s.t
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        has = (tokens >= 0) & (tokens < classes)
        w = np.where(has, logits.astype(np.float64), -np.inf)
        m = w.max(1, initial=-np.inf, keepdims=True)
        y = (w - np.where(np.isneginf(m), 0.0, m)) / t
        e = np.exp(y)
        total = e.sum(1, keepdims=True)
        p = e / np.where(total == 0, 1.0, total)
        lp = y - np.log(total)
        on = p > 0
        row = np.broadcast_to(np.arange(rows)[:, None], tokens.shape)
        lq, lq_err = s.log_prob(row, np.where(has, tokens, 0)) if classes else (np.zeros(tokens.shape), np.zeros(tokens.shape))
        terms = np.where(on, p * (lp - lq), 0.0)
        loss = t * t * terms.sum(1)
        # p: its exponent has three roundings, the sum at most eight and a tree's, the quotient one; log p as much.
        p_rel = lm.U * (4 * np.where(on, np.abs(y), 0.0) + 30)
        lp_err = lm.U * (4 * np.abs(y) + 30 + 4 * np.abs(np.log(total)) + np.abs(lp))
        size = np.where(on, p * (np.abs(lp) + np.abs(lq)), 0.0)
        loss_err = t * t * (np.where(on, p * (lp_err + lq_err), 0.0) + (p_rel + 20 * lm.U) * size).sum(1)
        factor = scales.astype(np.float64) * t
        hot, hot_err = np.zeros((rows, classes)), np.zeros((rows, classes))
        rr, jj = np.nonzero(has)
        np.add.at(hot, (rr, tokens[rr, jj]), p[rr, jj])
        np.add.at(hot_err, (rr, tokens[rr, jj]), (p_rel * p)[rr, jj] + (top + 4) * lm.U * p[rr, jj])
        q = s.p
        # q: as a probability from l, which is off by l_err itself.
        q_err = q * (lm.probability_error(np.where(q > 0, s.y, 0), np.where(np.isfinite(s.l), s.l, 0)) + s.l_err[:, None] + 4 * lm.U) + 2.0**-120
        none = (total[:, 0] == 0) | (factor == 0) | np.isneginf(s.l)
        delta = np.where(none[:, None], 0.0, factor[:, None] * (hot - q))
        delta_err = np.where(none[:, None], 0.0, np.abs(factor)[:, None] * (hot_err + q_err + 3 * lm.U * hot))
    return loss, loss_err, delta, delta_err


def check(pool, kind, z, classes, temperature, tokens, logits, scales=None, scale=1.0, shift=0, shift_out=None, onto=False, want_delta=True):
    rows, pitch = z.shape
    top = tokens.shape[1]
    dz = pool(z, kind, shift=shift)
    out = None if not want_delta else dz if onto else pool(kind=kind, n=(rows, pitch), shift=shift if shift_out is None else shift_out)
    before = out.raw().copy() if want_delta else None
    dt, dl, ds = pool(tokens), pool(logits), pool(scales) if scales is not None else None
    loss = pool(n=rows)
    ws = pool.work(gpu.distillationWorkspace(kind, rows, classes))
    gpu.distillation(kind, rows, classes, pitch, dz.buf, temperature, top, dt.buf, dl.buf, buf(ds), scale, loss.buf, buf(out), buf(ws))
    if ws is not None:
        ws.raw()
    full = np.full(rows, np.float32(scale)) * (scales if scales is not None else np.float32(1))
    l, l_err, d, d_err = evaluate(z, classes, temperature, tokens, logits, full)
    assert_within(loss.get(), l, l_err, "loss")
    if want_delta:
        assert out.raw()[:, classes:].tobytes() == before[:, classes:].tobytes(), "written between the rows"
        assert_within(out.get()[:, :classes], d, d_err + lm.rounding(kind) * (np.abs(d) + d_err), "logits_delta")
    return loss.get()


SHAPES = [(1, 1, 0, 1), (3, 2, 0, 2), (5, 7, 1, 5), (4, 64, 0, 64), (2, 65, 3, 256), (9, 1000, 24, 20), (3, 1025, 0, 1), (3, 2041, 7, 8),
          (2, 2049, 0, 64), (5, 8192, 0, 5), (1, 8193, 0, 256), (600, 4100, 0, 3), (513, 2100, 1, 64), (2, 50001, 47, 100), (1, 131072, 0, 64)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes,gap,top", SHAPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_shapes_and_alignments(pool, kind, rows, classes, gap, top, shift):
    z = make(kind, rows, classes, classes + gap)
    t, l = teacher(rows, top, classes)
    check(pool, kind, z, classes, 1.0, t, l, scale=1.0 / rows, shift=shift)
    r = np.random.default_rng(9).normal(size=rows).astype(np.float32)
    r[0] = 0
    check(pool, kind, z, classes, 2.0, t, l, scales=r, shift=shift, shift_out=1 - shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", cases.ROWS)
def test_every_kernel(pool, kind, rows, classes):
    t, l = teacher(rows, 130, classes)
    check(pool, kind, make(kind, rows, classes, classes + 1), classes, 1.0, t, l, scale=0.5)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", [(4, 900), (3, 20000), (600, 4000), (3, 70000)])
@pytest.mark.parametrize("temperature", [0.5, 3.0])
def test_onto_the_logits_and_without_a_delta(pool, kind, rows, classes, temperature):
    z = make(kind, rows, classes, classes + 5)
    t, l = teacher(rows, 200, 50)  # every class several times
    a = check(pool, kind, z, classes, temperature, t, l, onto=True)
    b = check(pool, kind, z, classes, temperature, t, l, want_delta=False)
    assert (a == b).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [40, 3001, 40000])
def test_masks(pool, kind, classes):
    z = make(kind, 7, classes, classes)
    t, l = teacher(7, 12, classes)
    t[:, 0] = 1
    z[0] = -np.inf  # no class left: the loss is infinite
    z[1, 1] = -np.inf  # a masked class that the teacher has
    z[3, 5:] = -np.inf
    t[3] = [0, 1, 2, 3, 4, 4, 0, 1, -1, -1, 2, 2]
    l[4] = -np.inf  # entries without probability
    l[5, :8] = -np.inf
    t[6, 1:] = -1  # one entry: the cross-entropy of a class
    t[2] = -1
    l[2] = np.nan  # no entry's logit is looked at
    loss = check(pool, kind, z, classes, 1.5, t, l)
    assert np.isposinf(loss[:2]).all() and loss[2] == 0 and loss[4] == 0


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [300, 30000])
def test_specials_stay_in_their_rows(pool, kind, classes):
    z = make(kind, 6, classes, classes)
    t, l = teacher(6, 9, classes)
    t[:] = np.arange(9) * 3
    z[1, classes - 1], z[2, 0], l[4, 2], l[5, 3] = np.nan, np.inf, np.nan, np.inf
    dz, dt, dl, loss, out = pool(z, kind), pool(t), pool(l), pool(n=6), pool(kind=kind, n=(6, classes))
    ws = pool.work(gpu.distillationWorkspace(kind, 6, classes))
    gpu.distillation(kind, 6, classes, classes, dz.buf, 1.0, 9, dt.buf, dl.buf, None, 1.0, loss.buf, out.buf, buf(ws))
    got, d = loss.get(), out.get()
    assert np.isnan(got[[1, 2, 4, 5]]).all() and np.isfinite(got[[0, 3]]).all() and np.isfinite(d[[0, 3]]).all()
    assert np.isnan(d[[1, 2]]).all()
    other = np.ones(classes, bool)
    other[t[4]] = False
    assert np.isnan(d[4][t[4][2]]) and np.isnan(d[5][t[5][3]]) and np.isfinite(d[4:][:, other]).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [300, 30000, 140000])
@pytest.mark.parametrize("special", [np.nan, np.inf])
def test_a_teacher_s_special_is_in_all_of_its_entries(pool, kind, classes, special):
    """No entry of such a row has a probability: the deltas of all their classes are NaN, those of the others as without."""
    rows, top = 4, 70
    z = make(kind, rows, classes, classes)
    t = np.tile(np.arange(top, dtype=np.int32) * 3, (rows, 1))
    l = np.random.default_rng(3).normal(size=(rows, top)).astype(np.float32)
    t[1:, 5], t[1:, 68] = -1, classes  # no entries
    l[2, 66] = l[3, 0] = special
    l[3, 1], l[3, 2], l[1, 5], l[1, 68] = -np.inf, special, special, special
    l[3, 4] = -1000.0
    dz, dt, dl, loss, out = pool(z, kind), pool(t), pool(l), pool(n=rows), pool(kind=kind, n=(rows, classes))
    ws = pool.work(gpu.distillationWorkspace(kind, rows, classes))
    gpu.distillation(kind, rows, classes, classes, dz.buf, 1.0, top, dt.buf, dl.buf, None, 1.0, loss.buf, out.buf, buf(ws))
    got, d = loss.get(), out.get()
    assert np.isfinite(got[:2]).all() and np.isfinite(d[:2]).all() and np.isnan(got[2:]).all()
    want = np.zeros((2, classes), bool)
    for i in (0, 1):
        want[i, t[2 + i][(t[2 + i] >= 0) & (t[2 + i] < classes)]] = True
    assert (np.isnan(d[2:]) == want).all()
    q = lm.Softmax(z, 1.0).p[2:]
    assert_within(d[2:][~want], -q[~want], 2.0**-7 * q[~want] + 2.0**-120, "the others")


@pytest.mark.parametrize("kind", [F32, BF16])
def test_one_class_left_that_the_teacher_has_is_no_loss(pool, kind):
    rows, classes = 2000, 40
    r = np.random.default_rng(4)
    z = np.full((rows, classes), -np.inf, np.float32)
    at = r.integers(0, classes, rows)
    z[np.arange(rows), at] = ref.rounded(r.normal(size=rows) * 8, kind)
    loss = check(pool, kind, z, classes, 0.7, at[:, None].astype(np.int32), np.ones((rows, 1), np.float32))
    assert (loss == 0).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [500, 20000, 70000])
@pytest.mark.parametrize("temperature", [2.0**-60, 0.3, 0.7, 1.0])
def test_masks_of_the_type_s_lowest_value(pool, kind, classes, temperature):
    """A loss is finite where its formula's value is."""
    lowest = -np.finfo(np.float32).max if kind == F32 else -float.fromhex("0x1.fep127")
    z = make(kind, 5, classes, classes)
    z[1, ::3] = z[3, 1:] = z[4] = lowest
    t, l = teacher(5, 9, classes)
    t[:, 0], t[3, 1] = 0, classes - 1
    loss = check(pool, kind, z, classes, temperature, t, l)  # at most the temperature times 2^128
    assert np.isfinite(loss).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [500, 20000, 70000])
def test_logits_far_from_zero(pool, kind, classes):
    """Rows whose logits are all large: only their distances matter."""
    r = np.random.default_rng(2)
    far = [0.0, 300.0, -300.0, 1e5, -1e5, 1e8, -1e8, 1e11, -1e11, 1e20, 1e30, -1e30]
    z = np.stack([ref.rounded(f + np.maximum(3, abs(f) * 2.0**-7) * r.integers(-2, 3, classes), kind) for f in far])
    tokens, logits = teacher(len(far), 5, classes)
    for temperature in (1.0, 0.7):
        check(pool, kind, z, classes, temperature, tokens, logits)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_no_classes_and_no_rows(pool, kind):
    t, l = np.zeros((3, 2), np.int32), np.zeros((3, 2), np.float32)
    dt, dl, loss = pool(t), pool(l), pool(n=3)
    gpu.distillation(kind, 3, 0, 0, gpu.Buf(), 1.0, 2, dt.buf, dl.buf, None, 1.0, loss.buf, None, None)
    assert (loss.get() == 0).all()
    gpu.distillation(kind, 0, 5, 5, gpu.Buf(), 1.0, 2, gpu.Buf(), gpu.Buf(), None, 1.0, gpu.Buf(), None, None)


def test_delta_is_the_derivative():
    """The formula of the tests above, by central differences in 64 bits."""
    r = np.random.default_rng(2)
    z = r.normal(size=(3, 40)) * 2
    t, l = teacher(3, 8, 40)
    t[2, 3:] = [1, 1, 2, 5, 9]
    temperature, scales = 1.25, np.array([0.5, 1.0, 2.0], np.float32)
    delta = evaluate(z, 40, temperature, t, l, scales)[2]
    for _ in range(5):
        v = r.normal(size=z.shape)
        up, down = ((scales * evaluate(z + h * v, 40, temperature, t, l, scales)[0]).sum() for h in (1e-5, -1e-5))
        assert abs((up - down) / 2e-5 + (delta * v).sum()) < 1e-7 * np.abs(delta * v).sum()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", [(1, 65536), (300, 9001), (1000, 700)])
def test_same_call_same_bits(pool, kind, rows, classes):
    z = make(kind, rows, classes, classes)
    t, l = teacher(rows, 100, classes)
    dz, dt, dl, loss, out = pool(z, kind), pool(t), pool(l), pool(n=rows), pool(kind=kind, n=(rows, classes))
    ws = pool.work(gpu.distillationWorkspace(kind, rows, classes))
    first = None
    for _ in range(4):
        gpu.distillation(kind, rows, classes, classes, dz.buf, 1.3, 100, dt.buf, dl.buf, None, 1.0, loss.buf, out.buf, buf(ws))
        got = (loss.raw().tobytes(), out.raw().tobytes())
        assert first is None or got == first
        first = got
