"""Dropout without a stored mask (dkz_seeded_dropout) on the GPU."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from .dense_ref import BF16, F32, Pool, buf

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


def want(x, residual, prob, scale, seed, first, y_type):
    """The fp32 arithmetic of the definition, rounded once."""
    with np.errstate(invalid="ignore", over="ignore"):
        y = np.where(ref.dropped(x.size, prob, seed, first), np.float32(0), x * np.float32(scale))
        if residual is not None:
            y = y + residual
    return ref.to_bf16(y) if y_type == BF16 else y.astype(np.float32)


def assert_same(got, expect):
    as_f = ref.from_bf16 if expect.dtype == np.uint16 else lambda a: a
    g, w = as_f(got), as_f(expect)
    nan = np.isnan(w)
    assert (np.isnan(g) == nan).all()
    assert (got[~nan] == expect[~nan]).all() and (np.signbit(g[~nan]) == np.signbit(w[~nan])).all()


@pytest.mark.parametrize("n", [1, 3, 255, 1024, 4097, 100003])
def test_fp32_is_rand_uniform_then_dropout(pool, n):
    r = np.random.default_rng(n)
    x = r.normal(size=n).astype(np.float32)
    a, draws, b = pool(x), pool(n=n), pool(n=n)
    gpu.randUniform(n, draws.buf, 77)
    gpu.dropout(a.buf, n, draws.buf, 0.3, 1 / 0.7)
    xs = pool(x)
    gpu.seededDropout(n, F32, xs.buf, None, 0.3, 1 / 0.7, 77, 0, F32, b.buf)
    assert (a.raw().view(np.uint32) == b.raw().view(np.uint32)).all()


@pytest.mark.parametrize("x_type", [F32, BF16])
@pytest.mark.parametrize("y_type", [F32, BF16])
@pytest.mark.parametrize("n,shift,prob,first", [(1, 0, 0.5, 0), (7, 1, 0.0, 5), (2048, 0, 0.1, 2**32 - 1000), (5000, 3, 0.9, 2**40 + 3),
                                                (65536 + 9, 1, 0.5, 2**32 - 60000), (300001, 0, 1.0, 1)])
@pytest.mark.parametrize("residual", [False, True])
def test_types_alignments_and_counters(pool, x_type, y_type, n, shift, prob, first, residual):
    r = np.random.default_rng(n)
    x, b = ref.rounded(r.normal(size=n), x_type), ref.rounded(r.normal(size=n), y_type)
    dx, db = pool(x, x_type, shift=shift), pool(b, y_type, shift=shift) if residual else None
    dy = pool(kind=y_type, n=n, shift=shift)
    gpu.seededDropout(n, x_type, dx.buf, buf(db), prob, 1.25, 0xDEADBEEF, first, y_type, dy.buf)
    assert_same(dy.raw(), want(x, b if residual else None, prob, 1.25, 0xDEADBEEF, first, y_type))


@pytest.mark.parametrize("shifts", [(0, 1, 0), (1, 0, 0), (0, 0, 2), (1, 2, 3)])
def test_mixed_alignments(pool, shifts):
    n = 3001
    r = np.random.default_rng(5)
    x, b = ref.rounded(r.normal(size=n), BF16), r.normal(size=n).astype(np.float32)
    dx, db, dy = pool(x, BF16, shift=shifts[0]), pool(b, F32, shift=shifts[1]), pool(kind=F32, n=n, shift=shifts[2])
    gpu.seededDropout(n, BF16, dx.buf, db.buf, 0.25, 4 / 3, 9, 0, F32, dy.buf)
    assert_same(dy.raw(), want(x, b, 0.25, 4 / 3, 9, 0, F32))


@pytest.mark.parametrize("kind", [F32, BF16])
def test_in_place_and_onto_the_residual(pool, kind):
    n = 4099
    r = np.random.default_rng(8)
    x, b = ref.rounded(r.normal(size=n), kind), ref.rounded(r.normal(size=n), kind)
    d = pool(x, kind)
    gpu.seededDropout(n, kind, d.buf, None, 0.5, 2.0, 3, 11, kind, d.buf)
    assert_same(d.raw(), want(x, None, 0.5, 2.0, 3, 11, kind))
    dx, db = pool(x, kind), pool(b, kind)
    gpu.seededDropout(n, kind, dx.buf, db.buf, 0.5, 2.0, 3, 11, kind, db.buf)
    assert_same(db.raw(), want(x, b, 0.5, 2.0, 3, 11, kind))


def test_conversion_rounds_to_nearest_even_and_keeps_specials(pool):
    u = np.arange(0, 2**32, 65537 * 7 + 2, dtype=np.uint64).astype(np.uint32)  # every exponent, ties among them
    ties = (np.arange(0x3F80, 0x3FA0, dtype=np.uint32) << np.uint32(16)) + np.uint32(0x8000)
    x = np.concatenate([u, ties]).view(np.float32)
    x = np.concatenate([x, np.array([0.0, -0.0, np.inf, -np.inf, np.nan, 3.4e38, 1e-45], np.float32)])
    dx, dy = pool(x), pool(kind=BF16, n=x.size)
    gpu.seededDropout(x.size, F32, dx.buf, None, 0.0, 1.0, 0, 0, BF16, dy.buf)
    assert_same(dy.raw(), want(x, None, 0.0, 1.0, 0, 0, BF16))


def test_dropped_specials_are_zero(pool):
    n = 1000
    x = np.full(n, np.nan, np.float32)
    x[::3] = np.inf
    dx, dy = pool(x), pool(kind=F32, n=n)
    gpu.seededDropout(n, F32, dx.buf, None, 0.5, 2.0, 1, 0, F32, dy.buf)
    out = ref.dropped(n, 0.5, 1, 0)
    assert out.any() and (dy.get()[out] == 0).all() and not np.isfinite(dy.get()[~out]).any()


def test_backward_drops_what_the_forward_dropped(pool):
    n = 10007
    ones = np.ones(n, np.float32)
    x, y, d = pool(ones), pool(kind=F32, n=n), pool(kind=BF16, n=n)
    gpu.seededDropout(n, F32, x.buf, None, 0.4, 1.0, 42, 123456789012, F32, y.buf)
    gpu.seededDropout(n, F32, x.buf, None, 0.4, 1.0, 42, 123456789012, BF16, d.buf)
    assert (y.get() == d.get()).all()
    # 10007 draws at 0.4: the share is within five standard deviations of it.
    assert abs((y.get() == 0).mean() - 0.4) < 5 * np.sqrt(0.4 * 0.6 / n)
