"""Log probabilities of tokens, entropies and alternatives (dkz_token_log_probs, _backward) on the GPU, in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from . import lm_cases as cases
from . import lm_ref as lm
from .dense_ref import BF16, F32, Pool, assert_within, buf

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


def make(kind, rows, classes, pitch, seed=0, std=3.0):
    """Logits in rows of `pitch`, NaN in what lies between the rows."""
    r = np.random.default_rng(seed + rows * 31 + classes)
    z = np.full((rows, pitch), np.nan, np.float32)
    z[:, :classes] = ref.rounded(r.normal(size=(rows, classes)) * std, kind)
    return z


def tokens_of(rows, given, classes, seed=3):
    r = np.random.default_rng(seed)
    t = r.integers(0, max(classes, 1), (rows, given)).astype(np.int32)
    t.ravel()[::7] = -1
    t.ravel()[3::11] = classes  # past the last
    if given > 2:
        t[:, 2] = t[:, 0]  # the same twice
    return t


def run(pool, kind, z, classes, temperature=1.0, tokens=None, top=0, entropy=True, shift=0):
    rows, pitch = z.shape
    given = 0 if tokens is None else tokens.shape[1]
    dz = pool(z, kind, shift=shift)
    dt = pool(tokens) if given else None
    lp, h = pool(n=(rows, given)) if given else None, pool(n=rows) if entropy else None
    stats = pool(n=(rows, 2))
    tt, tl = (pool(np.full((rows, top), 77, np.int32)), pool(n=(rows, top))) if top else (None, None)
    ws = pool.work(gpu.tokenLogProbsWorkspace(kind, rows, classes, top))
    gpu.tokenLogProbs(kind, rows, classes, pitch, dz.buf, temperature, given, buf(dt), top, buf(lp), buf(h), stats.buf, buf(tt), buf(tl), buf(ws))
    if ws is not None:
        ws.raw()
    dz.raw()
    return [None if d is None else d.get() for d in (lp, h, stats, tt, tl)]


def check(pool, kind, z, classes, temperature=1.0, tokens=None, top=0, entropy=True, shift=0):
    rows = z.shape[0]
    lp, h, stats, tt, tl = run(pool, kind, z, classes, temperature, tokens, top, entropy, shift)
    x = z[:, :classes]
    s = lm.Softmax(x, temperature)
    assert (stats[:, 0] == s.m).all()
    assert_within(stats[:, 1], s.l, s.l_err, "log sums")
    if entropy:
        assert_within(h, s.h, s.h_err, "entropy")
    row = np.arange(rows)[:, None]
    if tokens is not None:
        is_class = (tokens >= 0) & (tokens < classes)
        want, err = s.log_prob(np.broadcast_to(row, tokens.shape), np.where(is_class, tokens, 0)) if classes else (0.0, 0.0)
        assert_within(lp, np.where(is_class, want, 0.0), np.where(is_class, err, 0.0), "log_probs")
    if top:
        want = np.stack([lm.best(v, top) for v in x]) if classes else np.full((rows, top), -1)
        assert (tt == want).all(), np.argwhere(tt != want)[:5]
        if classes:
            v, err = s.log_prob(np.broadcast_to(row, want.shape), np.maximum(want, 0))
            assert_within(tl, np.where(want >= 0, v, -np.inf), np.where(want >= 0, err, 0.0), "top_log_probs")
        else:
            assert np.isneginf(tl).all()
    return stats


SHAPES = [(1, 1, 0, 1), (3, 2, 0, 2), (5, 7, 1, 5), (4, 63, 0, 64), (7, 64, 0, 3), (2, 65, 3, 64), (9, 1000, 24, 20), (3, 1023, 0, 1),
          (2, 1025, 0, 5), (3, 2041, 7, 8), (2, 2049, 0, 64), (1, 4096, 0, 20), (5, 8192, 0, 5), (1, 8193, 0, 64), (600, 4100, 0, 3),
          (513, 2100, 1, 64), (2, 50001, 47, 20), (1, 131072, 0, 64), (1, 300000, 0, 10)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes,gap,top", SHAPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_shapes_and_alignments(pool, kind, rows, classes, gap, top, shift):
    z = make(kind, rows, classes, classes + gap)
    check(pool, kind, z, classes, 1.0, tokens_of(rows, 3, classes), top, True, shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", cases.ROWS)
@pytest.mark.parametrize("entropy", [False, True])
def test_every_kernel(pool, kind, rows, classes, entropy):
    z = make(kind, rows, classes, classes + 1)
    check(pool, kind, z, classes, 1.0, tokens_of(rows, 2, classes), 5 if entropy else 0, entropy)
    run_backward(pool, kind, z, classes, 1.0, tokens_of(rows, 2, classes), entropy, beta=0.5)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("temperature", [0.3, 0.7, 1.0, 2.0, 100.0])
@pytest.mark.parametrize("parts", [(0, 0, True), (0, 5, False), (4, 0, False), (256, 64, True)], ids=str)
def test_temperatures_and_what_is_asked_for(pool, kind, temperature, parts):
    given, top, entropy = parts
    z = make(kind, 6, 9001, 9008)
    check(pool, kind, z, 9001, temperature, tokens_of(6, given, 9001) if given else None, top, entropy)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", [(3, 500), (2, 5000), (1, 70000), (700, 5000)])
def test_orders_and_ties(pool, kind, rows, classes):
    """Rows in the order that offers every element as an alternative, in the other, all equal, of two values, and of zeros of
    both signs."""
    up = np.linspace(-4, 4, classes)
    kinds = [up, up[::-1], np.full(classes, 1.5), np.where(np.arange(classes) % 3 == 1, 2.0, -1.0), np.where(np.arange(classes) % 2, 0.0, -0.0)]
    for i, v in enumerate(kinds):
        z = np.broadcast_to(ref.rounded(v, kind), (rows, classes)).copy()
        for top in (1, 20, 64):
            check(pool, kind, z, classes, 1.0, None, top)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [40, 3001, 40000])
def test_masks(pool, kind, classes):
    z = make(kind, 6, classes, classes)
    r = np.random.default_rng(1)
    z[0, :] = -np.inf  # no class left
    z[1, r.random(classes) < 0.9] = -np.inf
    z[2, :] = -np.inf
    z[2, classes // 2] = 3.0  # one
    z[3, :] = ref.rounded(np.finfo(np.float32).min if kind == F32 else -3.3e38, kind)  # the type's lowest, all of it
    z[4, 1:] = ref.rounded(-3.3e38, kind)
    z[5, : classes - 3] = -np.inf
    t = tokens_of(6, 5, classes)
    t[:, 1], t[2, 3] = 0, classes // 2
    check(pool, kind, z, classes, 1.0, t, min(64, classes))
    stats = check(pool, kind, z[[0, 1, 2, 5]], classes, 0.7, t[[0, 1, 2, 5]], 20)
    assert np.isneginf(stats[0]).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [300, 30000])
@pytest.mark.parametrize("bad", [np.nan, np.inf])
def test_specials_stay_in_their_rows(pool, kind, classes, bad):
    z = make(kind, 5, classes, classes)
    z[1, classes - 2] = bad
    z[3, 0] = bad
    t = np.tile(np.array([[0, classes - 2, -1]], np.int32), (5, 1))
    lp, h, stats, tt, tl = run(pool, kind, z, classes, 1.0, t, 4)
    for row in (1, 3):
        assert np.isnan(stats[row, 1]) and np.isnan(h[row]) and np.isnan(lp[row, :2]).all() and lp[row, 2] == 0 and np.isnan(tl[row]).all()
        assert (tt[row] == -1).all()
    good = [0, 2, 4]
    s = lm.Softmax(z[good], 1.0)
    assert_within(stats[good, 1], s.l, s.l_err, "log sums")
    assert_within(h[good], s.h, s.h_err, "entropy")


@pytest.mark.parametrize("kind", [F32, BF16])
def test_extreme_temperatures(pool, kind):
    """A tiny one leaves the largest logit alone (log p 0 and -infinity), a large one makes all alike."""
    z = make(kind, 2, 5000, 5000)
    z[0, 17] = z[1, 4999] = 60.0
    t = np.array([[17, 3], [4999, 0]], np.int32)
    lp, h, stats, tt, _ = run(pool, kind, z, 5000, 2.0**-64, t, 1)
    assert (tt[:, 0] == [17, 4999]).all() and (lp[:, 0] == 0).all() and (lp[:, 1] < -1e20).all() and (h == 0).all() and (stats[:, 1] == 0).all()
    check(pool, kind, z, 5000, 2.0**64, t, 5)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("classes", [500, 20000])
def test_logits_far_from_zero(pool, kind, entropy, classes):
    """Rows whose logits are all large: only their distances matter."""
    r = np.random.default_rng(2)
    far = [0.0, 300.0, -300.0, 1e5, -1e5, 1e8, -1e8, 1e11, -1e11, 1e20, 1e30, -1e30, 1e37, -1e37]
    z = np.stack([ref.rounded(f + np.maximum(3, abs(f) * 2.0**-7) * r.integers(-2, 3, classes), kind) for f in far])
    for temperature in (1.0, 0.7):
        check(pool, kind, z, classes, temperature, tokens_of(len(far), 2, classes), 3, entropy)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_no_rows_and_no_classes(pool, kind):
    check(pool, kind, np.zeros((4, 0), np.float32), 0, 1.0, np.zeros((4, 2), np.int32), 3)
    gpu.tokenLogProbs(kind, 0, 10, 10, gpu.Buf(), 1.0, 1, None, 1, None, None, gpu.Buf(), None, None, None)


def test_more_rows_than_workgroups(pool):
    rows, classes = (1 << 20) + 5, 3
    z = make(F32, rows, classes, classes)
    lp, h, stats, tt, tl = run(pool, F32, z, classes, 1.0, np.zeros((rows, 1), np.int32), 1)
    s = lm.Softmax(z, 1.0)
    assert_within(stats[:, 1], s.l, s.l_err, "log sums")
    assert_within(h, s.h, s.h_err, "entropy")
    assert (tt[:, 0] == z.argmax(1)).all()
    want, err = s.log_prob(np.arange(rows), np.zeros(rows, int))
    assert_within(lp[:, 0], want, err, "log_probs")


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", [(2000, 12), (1000, 900), (600, 5000), (3, 70000)])
@pytest.mark.parametrize("entropy", [False, True])
@pytest.mark.parametrize("temperature", [1.0, 0.7])
def test_no_probability_is_above_1(pool, kind, rows, classes, entropy, temperature):
    """Rows with one class left, or one far above the others: log probabilities are at most 0, entropies and log sums at least 0."""
    r = np.random.default_rng(rows + classes)
    for others in (-np.inf, -200.0, -30.0):
        z = np.full((rows, classes), np.nan, np.float32)
        m = ref.rounded(r.normal(size=(rows, 1)) * 8, kind)
        z[:] = ref.rounded(m + others, kind)
        at = r.integers(0, classes, rows)
        z[np.arange(rows), at] = m[:, 0]
        lp, h, stats, tt, tl = run(pool, kind, z, classes, temperature, at[:, None].astype(np.int32), 2, entropy)
        assert (lp <= 0).all() and (stats[:, 1] >= 0).all() and (tl <= 0).all() and (tt[:, 0] == at).all()
        assert h is None or (h >= 0).all()
        s = lm.Softmax(z, temperature)
        assert_within(stats[:, 1], s.l, s.l_err, "log sums")
        if entropy:
            assert_within(h, s.h, s.h_err, "entropy")


def test_offsets_past_32_bits(pool):
    """Rows whose elements lie past 2^32 bytes and 2^31 elements: 33000 x 65600 bf16. (65001 classes: the sums are within
    U (34 + 6 (65001 / 4096 + 110)) = 5e-5, see lm_ref.Softmax.)"""
    rows, classes, pitch = 33000, 65001, 65600
    z = gpu.alloc(rows * pitch // 2)
    try:
        last = make(BF16, 3, pitch, pitch)
        tail = np.ascontiguousarray(ref.to_bf16(last)).view(np.int32).ravel()
        gpu.push(z.offset((rows - 3) * pitch // 2), tail)
        tokens = np.full((rows, 1), 64000, np.int32)
        dt, lp, stats, tt, tl = pool(tokens), pool(n=rows), pool(n=(rows, 2)), pool(np.zeros((rows, 2), np.int32)), pool(n=(rows, 2))
        ws = pool.work(gpu.tokenLogProbsWorkspace(BF16, rows, classes, 2))
        gpu.tokenLogProbs(BF16, rows, classes, pitch, z, 1.0, 1, dt.buf, 2, lp.buf, None, stats.buf, tt.buf, tl.buf, buf(ws))
        s = lm.Softmax(last[:, :classes], 1.0)
        assert_within(stats.get()[-3:, 1], s.l, s.l_err, "log sums")
        assert (tt.get()[-3:] == np.stack([lm.best(v, 2) for v in last[:, :classes]])).all()
        assert (tt.get()[:-3] == [0, 1]).all()
        assert_within(lp.get()[:-3], np.full(rows - 3, -np.log(classes)), 1e-4, "uniform rows")
        # The way back, onto the logits.
        a = pool(np.ones(rows, np.float32))
        gpu.tokenLogProbsBackward(BF16, rows, classes, pitch, z, 1.0, 1, dt.buf, stats.buf, None, a.buf, None, 0.0, z)
        back = np.empty_like(tail)
        gpu.pull(z.offset((rows - 3) * pitch // 2), back)
        got = ref.from_bf16(back.view(np.uint16)).reshape(3, pitch)
        want = -s.p
        want[:, 64000] += 1
        assert (got[:, classes:] == last[:, classes:]).all()
        assert_within(got[:, :classes], want, 2.0**-8 * np.abs(want) + 1e-4 * s.p, "delta")
    finally:
        gpu.free(z)


# ---- backward ----


def run_backward(pool, kind, z, classes, temperature, tokens, entropy, beta=0.0, shift=0, shift_out=None, onto=False, stats=None, wild=False):
    rows, pitch = z.shape
    r = np.random.default_rng(rows + classes)
    given = 0 if tokens is None else tokens.shape[1]
    s = lm.Softmax(z[:, :classes], temperature)
    with np.errstate(invalid="ignore"):
        st = np.stack([s.m, s.l], 1).astype(np.float32)
    h = s.h.astype(np.float32)
    a = r.normal(size=(rows, given)).astype(np.float32)
    e = r.normal(size=rows).astype(np.float32) if entropy else None
    old = ref.rounded(r.normal(size=(rows, pitch)), kind) if beta else np.full((rows, pitch), np.nan, np.float32)
    shift_out = shift if shift_out is None else shift_out
    dz = pool(z, kind, shift=shift)
    do = dz if onto else pool(old, kind, shift=shift_out)
    before = do.raw().copy()
    dt, da = (pool(tokens), pool(a)) if given else (None, None)
    dst, dh, de = pool(st), pool(h) if entropy else None, pool(e) if entropy else None
    gpu.tokenLogProbsBackward(kind, rows, classes, pitch, dz.buf, temperature, given, buf(dt), dst.buf, buf(dh), buf(da), buf(de), beta, do.buf)
    assert do.raw()[:, classes:].tobytes() == before[:, classes:].tobytes(), "written between the rows"
    got = do.get()[:, :classes]
    with np.errstate(invalid="ignore", over="ignore"):
        t = s.t
        l64, h64 = st[:, 1].astype(np.float64), h.astype(np.float64)
        none = np.isneginf(s.m) & np.isneginf(l64)
        y = np.maximum(s.y, -300 * np.log(2))
        p = np.exp(s.y - l64[:, None])
        is_class = np.zeros((rows, given), bool) if given == 0 else (tokens >= 0) & (tokens < classes)
        aa = np.where(is_class, a, 0.0).astype(np.float64)
        q = aa.sum(1)[:, None] + (e[:, None] * (y - l64[:, None] + h64[:, None]) if entropy else 0.0)
        d = -p * q
        hot, hot_abs = np.zeros_like(d), np.zeros_like(d)
        rr, jj = np.nonzero(is_class)
        if given:
            np.add.at(hot, (rr, tokens[rr, jj]), aa[rr, jj])
            np.add.at(hot_abs, (rr, tokens[rr, jj]), np.abs(aa[rr, jj]))
        d = np.where(none[:, None], 0.0, (d + hot) / t)
        size = np.abs(aa).sum(1)[:, None]
        q_err = U(given) * size
        if entropy:
            q_err = q_err + np.abs(e)[:, None] * lm.U * (6 * np.abs(y) + 3 * np.abs(l64)[:, None] + 4 * np.abs(y - l64[:, None]) + 3 * np.abs(h64)[:, None])
        err = p * (np.abs(q) * (lm.probability_error(np.where(p > 0, s.y, 0), l64) + 4 * lm.U) + q_err) + 2.0**-120 * (1 + np.abs(q))
        err = np.where(none[:, None], 0.0, (err + U(given) * hot_abs) / t)
        if beta:
            d = d + beta * old[:, :classes]
            err = err + 4 * lm.U * np.abs(beta * old[:, :classes]) + lm.U * np.abs(d)
    assert_within(got, d, err + lm.rounding(kind) * (np.abs(d) + err), "logits_delta")


def U(given):
    """Of a sum of `given` terms and a product or two."""
    return (given + 4) * lm.U


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes,gap,top", SHAPES)
@pytest.mark.parametrize("shift", [0, 1])
def test_backward_shapes_and_alignments(pool, kind, rows, classes, gap, top, shift):
    z = make(kind, rows, classes, classes + gap)
    run_backward(pool, kind, z, classes, 1.0, tokens_of(rows, 3, classes), True, shift=shift)
    run_backward(pool, kind, z, classes, 0.7, tokens_of(rows, 1, classes), False, beta=0.5, shift=shift, shift_out=1 - shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [100, 9001])
@pytest.mark.parametrize("given,entropy,beta", [(0, True, 0.0), (0, False, 1.0), (256, True, 0.0), (256, False, -2.0), (16, True, 1.0)])
def test_backward_of_what_there_is(pool, kind, classes, given, entropy, beta):
    z = make(kind, 5, classes, classes + 3)
    run_backward(pool, kind, z, classes, 2.0, tokens_of(5, given, classes) if given else None, entropy, beta=beta)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", [(4, 900), (3, 20000), (600, 4000)])
def test_backward_onto_the_logits(pool, kind, rows, classes):
    z = make(kind, rows, classes, classes + 5)
    t = np.zeros((rows, 256), np.int32) + np.arange(256, dtype=np.int32) % 40  # every class several times
    run_backward(pool, kind, z, classes, 1.0, t, True, onto=True)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [100, 9001])
def test_backward_of_masks(pool, kind, classes):
    z = make(kind, 5, classes, classes)
    z[0] = -np.inf
    z[1, ::2] = -np.inf
    z[2, 1:] = -np.inf
    z[3] = ref.rounded(-3.3e38, kind)
    t = np.tile(np.array([[0, 1, -1]], np.int32), (5, 1))
    for beta in (0.0, 1.0):
        run_backward(pool, kind, z, classes, 1.0, t, True, beta=beta)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_of_a_row_with_a_nan_is_nan(pool, kind):
    z = make(kind, 3, 700, 700)
    z[1, 5] = np.nan
    t = np.array([[1], [2], [3]], np.int32)
    lp, h, stats, _, _ = run(pool, kind, z, 700, 1.0, t)
    dz, dt, ds, dh, out = pool(z, kind), pool(t), pool(stats), pool(h), pool(kind=kind, n=(3, 700))
    a, e = pool(np.ones(3, np.float32)), pool(np.ones(3, np.float32))
    gpu.tokenLogProbsBackward(kind, 3, 700, 700, dz.buf, 1.0, 1, dt.buf, ds.buf, dh.buf, a.buf, e.buf, 0.0, out.buf)
    got = out.get()
    assert np.isnan(got[1]).all() and np.isfinite(got[[0, 2]]).all()


def test_backward_is_the_derivative():
    """The formula of the tests above, by central differences in 64 bits: of sum a * log p + e * H along random directions.
    Steps of 1e-5 leave 1e-10 of the third derivative and 1e-11 of rounding."""
    r = np.random.default_rng(4)
    z, tok, t = r.normal(size=(3, 50)) * 2, np.array([[4, 9, 4], [0, 1, 2], [49, 49, 7]]), 0.75
    a, e = r.normal(size=(3, 3)), r.normal(size=3)

    def value(v):
        s = lm.Softmax(v, t)
        return sum((a[i, j] * s.lp[i, tok[i, j]]) for i in range(3) for j in range(3)) + (e * s.h).sum()

    s = lm.Softmax(z, t)
    d = -s.p * (a.sum(1)[:, None] + e[:, None] * (s.lp + s.h[:, None]))
    np.add.at(d, (np.repeat(np.arange(3), 3), tok.ravel()), a.ravel())
    d /= t
    for _ in range(5):
        v = r.normal(size=z.shape)
        num = (value(z + 1e-5 * v) - value(z - 1e-5 * v)) / 2e-5
        assert abs(num - (d * v).sum()) < 1e-7 * np.abs(d * v).sum()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows,classes", [(1, 65536), (300, 9001), (1000, 700)])
def test_same_call_same_bits(pool, kind, rows, classes):
    z, t = make(kind, rows, classes, classes), tokens_of(rows, 2, classes)
    first = None
    for _ in range(4):
        got = [x.tobytes() for x in run(pool, kind, z, classes, 0.9, t, 20)]
        assert first is None or got == first
        first = got
