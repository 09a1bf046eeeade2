"""Softmax cross-entropy of a linear layer without its logits, on the GPU, against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from .dense_ref import BF16, F32, HALF, Pool, assert_within, buf

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


def make(kind, rows, inputs, classes, bias=True, spread=2.5):
    r = np.random.default_rng(rows * 7 + inputs * 1009 + classes)
    x = ref.rounded(r.normal(size=(rows, inputs)), kind)
    w = ref.rounded(r.normal(size=(classes, inputs)) * spread / np.sqrt(max(inputs, 1)), kind)
    b = r.normal(size=classes).astype(np.float32) if bias else None
    t = r.integers(0, classes, rows).astype(np.int32) if classes else np.full(rows, -1, np.int32)
    t[r.random(rows) < 0.2] = -1
    if rows > 2:
        t[1] = classes  # past the last class: none
    return x, w, b, t


def reference(x, w, b, t):
    """(logits, bound of an fp32 logit's error, lse, loss)."""
    x, w = x.astype(np.float64), w.astype(np.float64)
    z, err = x @ w.T, ref.product_error(x, w.T)
    if b is not None:
        z = z + b
        err = err + 2.0**-24 * np.abs(np.where(np.isfinite(z), z, 0))
    classes = z.shape[1]
    m = z.max(1, initial=-np.inf)
    base = np.where(np.isneginf(m), 0, m)
    with np.errstate(divide="ignore"):
        lse = base + np.log(np.exp(z - base[:, None]).sum(1))
    has = (t >= 0) & (t < classes)
    at = z[np.arange(len(t)), np.where(has, t, 0)] if classes else np.zeros(len(t))
    with np.errstate(invalid="ignore"):
        loss = np.where(has, np.where(np.isneginf(lse), np.inf, lse - at), 0.0)
    return z, err, lse, loss


def exp_error(z, lse):
    """Relative error of the fp32 exp(z - lse): its argument's difference and scaling round by 2^-24 of |z|, |lse| and
    |z - lse|, the exponential itself by a step."""
    d = np.where(np.isfinite(z), np.abs(z) + np.abs(lse)[:, None] + 2 * np.abs(z - lse[:, None]), 0)
    return 2.0**-24 * (d + 4)


def lse_error(z, err, lse):
    """Sums of exponentials, each off by exp_error and its logit's error, in fp32 parts of at most 64 merged pairwise;
    the logarithm and the sum with the maximum."""
    top = np.where(np.isfinite(z), err, 0).max(1, initial=0)
    e = exp_error(z, np.where(np.isfinite(lse), lse, 0)).max(1, initial=0)
    return top + e + (64 + 32) * 2.0**-24 + 3 * 2.0**-24 * np.abs(np.where(np.isfinite(lse), lse, 0))


def run(pool, kind, x, w, b, t, beta=0.0, row_scales=None, scale=1.0, least=False, shift=0, want=(1, 1, 1), backward=True):
    rows, inputs = x.shape
    classes = w.shape[0]
    dx, dw = pool(x, kind, shift=shift), pool(w, kind, shift=shift)
    db, dt = pool(b) if b is not None else None, pool(t)
    loss, lse = pool(n=rows), pool(n=rows)
    sizes = gpu.linearCrossEntropyForwardWorkspace(kind, rows, inputs, classes)
    ws = pool.work(sizes[0 if least else 1])
    gpu.linearCrossEntropyForward(kind, rows, inputs, classes, dx.buf, dw.buf, buf(db), dt.buf, loss.buf, lse.buf, buf(ws))
    if ws is not None:
        ws.raw()
    z, err, l64, loss64 = reference(x, w, b, t)
    l_err = lse_error(z, err, l64)
    assert_within(lse.get(), l64, l_err, "lse")
    assert_within(loss.get(), loss64, l_err + np.where(np.isfinite(z), err, 0).max(1, initial=0) + 2.0**-24 * np.where(np.isfinite(loss64), np.abs(loss64), 0), "loss")
    if not backward:
        return loss, lse
    r = np.random.default_rng(3)
    bu, wu = r.normal(size=classes).astype(np.float32), ref.rounded(r.normal(size=(classes, inputs)), kind)
    if beta == 0:
        bu, wu = np.full_like(bu, np.nan), np.full_like(wu, np.nan)
    gb, gw = pool(bu) if want[0] else None, pool(wu, kind, shift=shift) if want[1] else None
    gx = pool(kind=kind, n=(rows, inputs), shift=shift) if want[2] else None
    ds = pool(row_scales) if row_scales is not None else None
    sizes = gpu.linearCrossEntropyBackwardWorkspace(kind, rows, inputs, classes)
    ws = pool.work(sizes[0 if least else 1])
    gpu.linearCrossEntropyBackward(kind, rows, inputs, classes, dx.buf, dw.buf, buf(db), dt.buf, lse.buf, buf(ds), scale, beta, buf(gb),
                                   buf(gw), buf(gx), buf(ws))
    if ws is not None:
        ws.raw()
    has = (t >= 0) & (t < classes) & ~np.isneginf(l64)
    safe = np.where(np.isfinite(l64), l64, 0)
    p = np.where(has[:, None], np.exp(z - safe[:, None]), 0)
    hot = np.zeros_like(p)
    hot[np.nonzero(has)[0], t[has]] = 1
    s = scale * (row_scales.astype(np.float64) if row_scales is not None else np.ones(rows))
    s = np.where(has, s, 0)[:, None]
    d = s * (hot - p)
    d_err = np.abs(s) * (p * (exp_error(z, safe) + np.where(np.isfinite(err), err, 0) + l_err[:, None]) * 1.01) + 3 * 2.0**-24 * np.abs(d)
    # Below 2^-126 there is no normal fp32 number: a probability, a product or a sum there may become 0.
    d_err = d_err + 2.0**-126 * (1 + np.abs(s))
    p_err = d_err + (HALF[BF16] * np.abs(d) * (1 + 2.0**-8) if kind == BF16 else 0)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    if gb is not None:
        base = beta * bu.astype(np.float64) if beta else 0.0
        total = base + d.sum(0)
        e = d_err.sum(0) + 130 * 2.0**-24 * np.abs(d).sum(0) + 3 * 2.0**-24 * (np.abs(total) + np.abs(base))
        assert_within(gb.get(), total, e, "bias_updates")
    for got, a, m, e, base, name in ((gw, d.T, x64, p_err.T, beta * wu.astype(np.float64) if beta else 0.0, "weight_updates"),
                                     (gx, d, w64, p_err, 0.0, "input_delta")):
        if got is None:
            continue
        y = a @ m + base
        bound = ref.product_error(a, m) * 1.01 + (a.shape[1] + 1) * 2.0**-126 + e @ np.abs(m) + 3 * 2.0**-24 * (np.abs(y) + np.abs(base))
        assert_within(got.get(), y, bound + HALF[kind] * (np.abs(y) + bound), name)
    return gb, gw, gx


SHAPES = [(1, 1, 1), (1, 8, 2), (2, 64, 1000), (3, 7, 9), (5, 33, 257), (64, 128, 512), (130, 72, 1001), (129, 65, 130), (17, 1030, 700),
          (1, 256, 5003)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("bias,shift", [(False, 0), (True, 1)])
def test_shapes_and_alignments(pool, kind, shape, bias, shift):
    run(pool, kind, *make(kind, *shape, bias=bias), scale=0.25, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("classes", [255, 256, 257, 700, 1024])
def test_pieces_of_the_classes(pool, kind, classes):
    """The least workspace: pieces of 256 classes, the last one of any size."""
    run(pool, kind, *make(kind, 37, 40, classes), least=True, beta=0.5)
    run(pool, kind, *make(kind, 150, 41, classes), least=True)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_row_scales_and_accumulation(pool, kind):
    x, w, b, t = make(kind, 50, 48, 300)
    s = np.random.default_rng(1).uniform(0, 1, 50).astype(np.float32)
    s[7] = 0
    run(pool, kind, x, w, b, t, row_scales=s, scale=-0.5, beta=1.0)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1)])
def test_backward_computes_what_is_asked_for(pool, kind, want):
    run(pool, kind, *make(kind, 40, 48, 300), want=want)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_masked_classes(pool, kind):
    """Classes whose bias is -infinity have probability 0; a target among them has loss +infinity and a gradient."""
    x, w, b, t = make(kind, 20, 24, 600)
    b[::2] = -np.inf
    b[300:590] = -np.inf
    t[:4] = [0, 2, 301, 599]
    run(pool, kind, x, w, b, t, least=True)
    run(pool, kind, x, w, b, t)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_no_class_left(pool, kind):
    x, w, b, t = make(kind, 6, 16, 400)
    b[:] = -np.inf
    t[:] = [0, 5, 399, -1, 7, 400]
    loss, lse = run(pool, kind, x, w, b, t, backward=False)
    assert np.isneginf(lse.get()).all() and (loss.get() == [np.inf, np.inf, np.inf, 0, np.inf, 0]).all()
    gb, gw, gx = run(pool, kind, x, w, b, t)
    assert not gb.get().any() and not gw.get().any() and not gx.get().any()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_the_lowest_bias_is_a_number(pool, kind):
    x, w, b, t = make(kind, 6, 16, 400)
    b[1:] = np.finfo(np.float32).min
    t[:] = [0, 0, -1, 0, 0, 0]
    loss, lse = pool(n=6), pool(n=6)
    dx, dw, db, dt = pool(x, kind), pool(w, kind), pool(b), pool(t)
    ws = pool.work(gpu.linearCrossEntropyForwardWorkspace(kind, 6, 16, 400)[1])
    gpu.linearCrossEntropyForward(kind, 6, 16, 400, dx.buf, dw.buf, db.buf, dt.buf, loss.buf, lse.buf, ws.buf)
    z0 = x.astype(np.float64) @ w[0].astype(np.float64) + b[0]
    assert_within(lse.get(), z0, 20 * 2.0**-24 * (np.abs(x) @ np.abs(w[0]) + abs(b[0])) + 2.0**-23, "lse")
    assert (loss.get() == 0).all()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_nan_stays_in_its_row(pool, kind):
    x, w, b, t = make(kind, 140, 64, 300)
    x[3, 5] = np.nan
    t[3], t[4] = 7, 8
    dx, dw, db, dt = pool(x, kind), pool(w, kind), pool(b), pool(t)
    loss, lse = pool(n=140), pool(n=140)
    ws = pool.work(max(gpu.linearCrossEntropyForwardWorkspace(kind, 140, 64, 300)[1], gpu.linearCrossEntropyBackwardWorkspace(kind, 140, 64, 300)[1]))
    gpu.linearCrossEntropyForward(kind, 140, 64, 300, dx.buf, dw.buf, db.buf, dt.buf, loss.buf, lse.buf, ws.buf)
    other = np.arange(140) != 3
    assert np.isnan(lse.get()[3]) and np.isnan(loss.get()[3]) and np.isfinite(lse.get()[other]).all() and np.isfinite(loss.get()[other]).all()
    gx = pool(kind=kind, n=(140, 64))
    gpu.linearCrossEntropyBackward(kind, 140, 64, 300, dx.buf, dw.buf, db.buf, dt.buf, lse.buf, None, 1.0, 0.0, None, None, gx.buf, ws.buf)
    assert np.isnan(gx.get()[3]).all() and np.isfinite(gx.get()[other]).all()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_large_logits_do_not_overflow(pool, kind):
    x, w, b, t = make(kind, 9, 32, 500, spread=400.0)
    run(pool, kind, x, w, b, t, scale=0.1)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_empty_sizes(pool, kind):
    x, w, b, t = make(kind, 4, 0, 30)
    run(pool, kind, x, w, b, t)  # logits are the biases
    x, w, b, t = make(kind, 4, 8, 0, bias=False)
    loss, lse = run(pool, kind, x, w, b, t, backward=False)
    assert np.isneginf(lse.get()).all() and not loss.get().any()
    gx = pool(kind=kind, n=(4, 8))
    gpu.linearCrossEntropyBackward(kind, 4, 8, 0, None, None, None, None, None, None, 1.0, 0.0, None, None, gx.buf, None)
    assert not gx.get().any()
    gb, gw = pool(np.arange(30, dtype=np.float32)), pool(np.ones((30, 8), np.float32), kind)
    ws = pool.work(gpu.linearCrossEntropyBackwardWorkspace(kind, 0, 8, 30)[1])
    gpu.linearCrossEntropyBackward(kind, 0, 8, 30, None, None, None, None, None, None, 1.0, 2.0, gb.buf, gw.buf, None, buf(ws))
    assert (gb.get() == 2 * np.arange(30)).all() and (gw.get() == 2).all()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_gradient_by_differences(pool, kind):
    """Central differences of the 64-bit loss, whose negative the deltas are."""
    x, w, b, t = make(kind, 7, 6, 12)
    t[:] = [0, 3, 11, -1, 5, 5, 2]
    gb, gw, gx = run(pool, kind, x, w, b, t)
    h = 1e-4
    x64, w64, b64 = x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)

    def loss(x, w, b):
        return reference(x, w, b, t)[3].sum()

    for got, base, which in ((gb.get(), b64, 2), (gw.get(), w64, 1), (gx.get(), x64, 0)):
        num = np.empty_like(base)
        for i in np.ndindex(base.shape):
            args = [x64, w64, b64]
            up, down = base.copy(), base.copy()
            up[i] += h
            down[i] -= h
            num[i] = (loss(*args[:which], up, *args[which + 1 :]) - loss(*args[:which], down, *args[which + 1 :])) / (2 * h)
        mags = {2: np.full(12, 7.0), 1: np.abs(x64).sum(0)[None, :] * np.ones((12, 1)), 0: np.abs(w64).sum(0)[None, :] * np.ones((7, 1))}[which]
        # d and the result are rounded to the type; truncation of the differences is below h^2 of the magnitudes.
        assert_within(got, -num, (2.5 * HALF[kind] + 2e-6) * mags, ("input", "weights", "biases")[which])


@pytest.mark.parametrize("kind", [F32, BF16])
def test_same_call_same_bits(pool, kind):
    x, w, b, t = make(kind, 200, 136, 900)
    first = [d.raw().copy() for d in run(pool, kind, x, w, b, t)]
    again = [d.raw().copy() for d in run(pool, kind, x, w, b, t)]
    for p, q in zip(first, again):
        assert (p.view(np.uint8) == q.view(np.uint8)).all()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_more_rows_than_workgroups(pool, kind):
    """Kernels that take a row a workgroup take several beyond 2^18 rows."""
    run(pool, kind, *make(kind, (1 << 18) + 77, 2, 3), backward=False)
