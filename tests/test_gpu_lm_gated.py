"""Gated feed-forward blocks (dkz_gated_forward, dkz_gated_backward) on the GPU, against their formulas in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from . import lm_cases as cases
from . import lm_ref as lm
from .dense_ref import BF16, F32, HALF, Pool, assert_within, buf
from .lm_ref import GATES, GELU, LINEAR, LOGISTIC, RELU, SILU, U

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


def run_forward(pool, kind, rows, inputs, hidden, act, bias=True, keep=True, shift=0, x=None, w=None):
    r = np.random.default_rng(rows * 7919 + inputs * 31 + hidden)
    x = ref.rounded(r.normal(size=(rows, inputs)), kind) if x is None else x
    w = ref.rounded(r.normal(size=(2 * hidden, inputs)) / np.sqrt(max(inputs, 1)), kind) if w is None else w
    b = r.normal(size=2 * hidden).astype(np.float32) if bias else None
    dx, dw, db = pool(x, kind, shift=shift), pool(w, kind, shift=shift), pool(b) if bias else None
    out, kept = pool(kind=kind, n=(rows, hidden), shift=shift), pool(kind=kind, n=(rows, 2 * hidden), shift=shift) if keep else None
    ws = pool.work(gpu.gatedForwardWorkspace(kind, rows, inputs, hidden))
    gpu.gatedForward(kind, rows, inputs, hidden, act, dx.buf, dw.buf, buf(db), buf(kept), out.buf, buf(ws))
    for d in (ws, dx, dw):
        if d is not None:
            d.raw()
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    s = x64 @ w64.T
    err = ref.product_error(x64, w64.T)
    if bias:
        s = s + b
        err = err + U * np.abs(s)
    if keep:
        assert_within(kept.get(), s, err + HALF[kind] * (np.abs(s) + err), "sums")
    g, up, g_err, up_err = s[:, :hidden], s[:, hidden:], err[:, :hidden], err[:, hidden:]
    a, a_err = lm.gate(act, g), lm.STEEPEST * g_err + lm.gate_error(act, g)
    y = a * up
    y_err = np.abs(a) * up_err + a_err * (np.abs(up) + up_err) + U * np.abs(y)
    assert_within(out.get(), y, y_err + HALF[kind] * (np.abs(y) + y_err), "output")
    return out


SHAPES = [(1, 1, 1), (1, 64, 5), (2, 8, 8), (3, 7, 9), (16, 65, 33), (31, 129, 130), (33, 40, 31), (128, 128, 128), (129, 200, 257), (1, 1000, 1003),
          (5, 4096, 40), (300, 72, 264), (64, 1032, 520)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_forward_shapes_and_alignments(pool, kind, shape, shift):
    run_forward(pool, kind, *shape, SILU, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", GATES)
@pytest.mark.parametrize("extras", [(False, False), (True, True), (False, True), (True, False)], ids=str)
def test_forward_gates_and_what_there_is(pool, kind, act, extras):
    run_forward(pool, kind, 70, 96, 132, act, *extras)
    run_forward(pool, kind, 4, 96, 130, act, *extras)


@pytest.mark.parametrize("case", cases.FORWARD, ids=str)
def test_forward_of_every_kernel(pool, case):
    kind, rows, inputs, hidden, act, shift = case
    run_forward(pool, kind, rows, inputs, hidden, act, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_forward_without_inputs_is_the_bias(pool, kind):
    run_forward(pool, kind, 5, 0, 12, GELU)
    run_forward(pool, kind, 40, 0, 7, LINEAR, bias=False)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", GATES)
def test_gates_over_the_range(pool, kind, act):
    """Gates from far below 0 to far above, and the values where a logistic is 0 or 1. A row an input, the other projection 1."""
    g = np.concatenate([np.linspace(-30, 30, 241), [-1e4, -200, -104, -89, 89, 104, 200, 1e4, 0.0, -0.0, 1e-30, -1e-30]])
    x = ref.rounded(np.stack([g, np.ones_like(g)], 1), kind)
    run_forward(pool, kind, len(g), 2, 1, act, False, True, x=x, w=np.eye(2, dtype=np.float32))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows", [3, 140])
def test_forward_specials_stay_in_their_rows_and_units(pool, kind, rows):
    inputs, hidden = 150, 136
    r = np.random.default_rng(6)
    x, w = ref.rounded(r.normal(size=(rows, inputs)), kind), ref.rounded(r.normal(size=(2 * hidden, inputs)), kind)
    x[1, 149], w[100, 3], w[hidden + 20, 0] = np.nan, np.nan, np.inf
    dx, dw, out = pool(x, kind), pool(w, kind), pool(kind=kind, n=(rows, hidden))
    ws = pool.work(gpu.gatedForwardWorkspace(kind, rows, inputs, hidden))
    gpu.gatedForward(kind, rows, inputs, hidden, SILU, dx.buf, dw.buf, None, None, out.buf, buf(ws))
    bad = np.zeros((rows, hidden), bool)
    bad[1], bad[:, 100], bad[:, 20] = True, True, True
    assert (np.isfinite(out.get()) == ~bad).all()


# ---- backward ----


def run_backward(pool, kind, rows, inputs, hidden, act, add=True, beta=0.0, shift=0, want=(1, 1, 1), onto=False):
    r = np.random.default_rng(rows * 104729 + inputs * 17 + hidden)
    x = ref.rounded(r.normal(size=(rows, inputs)), kind)
    w = ref.rounded(r.normal(size=(2 * hidden, inputs)), kind)
    s = ref.rounded(r.normal(size=(rows, 2 * hidden)) * 2, kind)
    delta = ref.rounded(r.normal(size=(rows, hidden)), kind)
    res = ref.rounded(r.normal(size=(rows, inputs)), kind) if add else None
    bu, wu = r.normal(size=2 * hidden).astype(np.float32), ref.rounded(r.normal(size=(2 * hidden, inputs)), kind)
    if beta == 0:
        bu, wu = np.full_like(bu, np.nan), np.full_like(wu, np.nan)  # not read
    dx, dw, ds, dd = (pool(v, kind, shift=shift) for v in (x, w, s, delta))
    dres = pool(res, kind, shift=shift) if add else None
    out_b, out_w = pool(bu) if want[0] else None, pool(wu, kind, shift=shift) if want[1] else None
    out_x = (dres if onto else pool(kind=kind, n=(rows, inputs), shift=shift)) if want[2] else None
    ws = pool.work(gpu.gatedBackwardWorkspace(kind, rows, inputs, hidden))
    gpu.gatedBackward(kind, rows, inputs, hidden, act, dx.buf, dw.buf, ds.buf, dd.buf, buf(dres), beta, buf(out_b), buf(out_w), buf(out_x), buf(ws))
    if ws is not None:
        ws.raw()
    g, up, dl = s[:, :hidden].astype(np.float64), s[:, hidden:].astype(np.float64), delta.astype(np.float64)
    a, slope = lm.gate(act, g), lm.gate_slope(act, g)
    d = np.concatenate([dl * up * slope, dl * a], 1)
    d_err = np.concatenate([np.abs(dl * up) * lm.slope_error(act, g), np.abs(dl) * lm.gate_error(act, g)], 1) + 3 * U * np.abs(d)
    p_err = d_err + (HALF[BF16] * (np.abs(d) + d_err) if kind == BF16 else 0)  # rounded once more for the products
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    if out_b is not None:
        base = beta * bu.astype(np.float64) if beta else 0.0
        total = base + d.sum(0)
        # sums of at most 64 rows in fp32, then 64 bits, then two roundings
        assert_within(out_b.get(), total, d_err.sum(0) + 64 * U * (np.abs(d) + d_err).sum(0) + 3 * U * (np.abs(total) + np.abs(base)), "bias_updates")
    for got, p, q, e, base, name in (
        (out_w, d.T, x64, p_err.T, beta * wu.astype(np.float64) if beta else 0.0, "weight_updates"),
        (out_x, d, w64, p_err, res.astype(np.float64) if add else 0.0, "input_delta"),
    ):
        if got is None:
            continue
        y = p @ q + base
        err = ref.product_error(p, q) * 1.01 + e @ np.abs(q) + 3 * U * (np.abs(y) + np.abs(base))
        assert_within(got.get(), y, err + HALF[kind] * (np.abs(y) + err), name)
    for t in (dx, dw, ds, dd):
        t.raw()


BACK_SHAPES = [(1, 1, 1), (1, 8, 5), (3, 7, 9), (16, 64, 32), (65, 33, 130), (128, 128, 128), (200, 129, 77), (257, 264, 72), (1, 1003, 300),
               (700, 40, 24)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", BACK_SHAPES, ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_backward_shapes_and_alignments(pool, kind, shape, shift):
    run_backward(pool, kind, *shape, SILU, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", GATES)
@pytest.mark.parametrize("beta", [0.0, 0.5])
def test_backward_gates(pool, kind, act, beta):
    run_backward(pool, kind, 70, 72, 45, act, False, beta=beta)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)])
def test_backward_computes_what_is_asked_for(pool, kind, want):
    run_backward(pool, kind, 40, 48, 28, GELU, True, want=want)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_adds_onto_the_input_delta(pool, kind):
    run_backward(pool, kind, 37, 41, 43, LOGISTIC, True, onto=True)


@pytest.mark.parametrize("case", cases.BACKWARD, ids=str)
def test_backward_of_every_kernel(pool, case):
    kind, rows, inputs, hidden, act, shift = case
    run_backward(pool, kind, rows, inputs, hidden, act, shift=shift, beta=0.5)


@pytest.mark.parametrize("case,want", cases.BACKWARD_PARTS, ids=str)
def test_backward_of_some_results(pool, case, want):
    kind, rows, inputs, hidden, act, shift = case
    run_backward(pool, kind, rows, inputs, hidden, act, shift=shift, beta=0.5, want=want)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_without_rows_or_inputs(pool, kind):
    b, w = np.arange(12, dtype=np.float32), ref.rounded(np.arange(48).reshape(12, 4), kind)
    db, dw = pool(b), pool(w, kind)
    gpu.gatedBackward(kind, 0, 4, 6, SILU, gpu.Buf(), gpu.Buf(), gpu.Buf(), gpu.Buf(), None, 0.5, db.buf, dw.buf, None, None)
    assert (db.get() == 0.5 * b).all() and (dw.get() == 0.5 * w).all()
    run_backward(pool, kind, 5, 0, 6, RELU, False, want=(1, 0, 0))


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("rows", [3, 300])
@pytest.mark.parametrize("shift", [0, 1])
def test_backward_without_units_or_inputs(pool, kind, rows, shift):
    """No units: the input's delta is the residual, or 0. No inputs: there are bias sums alone."""
    for inputs in (1, 13, 264):
        res = ref.rounded(np.random.default_rng(rows + inputs).normal(size=(rows, inputs)), kind)
        dres, dx, out = (pool(res, kind, shift=shift) for _ in range(3))
        ws = pool.work(gpu.gatedBackwardWorkspace(kind, rows, inputs, 0))
        none = gpu.Buf()
        gpu.gatedBackward(kind, rows, inputs, 0, SILU, dx.buf, none, none, none, dres.buf, 0.0, none, none, out.buf, buf(ws))
        assert (out.get() == res).all()
        gpu.gatedBackward(kind, rows, inputs, 0, SILU, dx.buf, none, none, none, dres.buf, 0.5, none, none, dres.buf, buf(ws))
        assert (dres.get() == res).all() and (dx.get() == res).all()
        gpu.gatedBackward(kind, rows, inputs, 0, SILU, dx.buf, none, none, none, None, 0.0, none, none, out.buf, buf(ws))
        assert (out.get() == 0).all()
    run_backward(pool, kind, rows, 0, 24, GELU, True, beta=0.5, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", GATES)
def test_backward_over_the_range(pool, kind, act):
    """The two parts of d by themselves (identity weights): gates far from 0 give no NaN and the slopes of their limits."""
    g = np.concatenate([np.linspace(-30, 30, 122), [-1e4, -200, -104, -89, 89, 104, 200, 1e4, 0.0, 1e-30]])
    if act == RELU:
        g = g[g != 0]
    rows = len(g)
    s, one = ref.rounded(np.stack([g, np.full(rows, 2.0)], 1), kind), np.ones((rows, 1), np.float32)
    eye = np.eye(2, dtype=np.float32)
    ds, dd, dw, out = pool(s, kind), pool(one, kind), pool(eye, kind), pool(kind=kind, n=(rows, 2))
    ws = pool.work(gpu.gatedBackwardWorkspace(kind, rows, 2, 1))
    gpu.gatedBackward(kind, rows, 2, 1, act, dd.buf, dw.buf, ds.buf, dd.buf, None, 0.0, None, None, out.buf, buf(ws))
    v = s[:, 0].astype(np.float64)
    want = np.stack([2 * lm.gate_slope(act, v), lm.gate(act, v)], 1)
    err = np.stack([2 * lm.slope_error(act, v) + 0 * v, lm.gate_error(act, v) + 0 * v], 1) + 6 * U * np.abs(want)
    assert_within(out.get(), want, err + 2 * HALF[kind] * (np.abs(want) + err), "d")


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", [(4096, 1024, 2048), (333, 1001, 1503), (20, 4096, 1000)], ids=str)
def test_same_call_same_bits(pool, kind, shape):
    rows, inputs, hidden = shape
    r = np.random.default_rng(9)
    x, w, delta = (pool(r.standard_normal(s, np.float32), kind) for s in ((rows, inputs), (2 * hidden, inputs), (rows, hidden)))
    y, s, gb = pool(kind=kind, n=(rows, hidden)), pool(kind=kind, n=(rows, 2 * hidden)), pool(n=2 * hidden)
    gw, gx = pool(kind=kind, n=(2 * hidden, inputs)), pool(kind=kind, n=(rows, inputs))
    ws = pool.work(max(f(kind, rows, inputs, hidden) for f in (gpu.gatedForwardWorkspace, gpu.gatedBackwardWorkspace)))
    first = None
    for _ in range(4):
        gpu.gatedForward(kind, rows, inputs, hidden, SILU, x.buf, w.buf, None, s.buf, y.buf, ws.buf)
        gpu.gatedBackward(kind, rows, inputs, hidden, SILU, x.buf, w.buf, s.buf, delta.buf, None, 0.0, gb.buf, gw.buf, gx.buf, ws.buf)
        got = [d.raw().tobytes() for d in (y, s, gb, gw, gx)]
        assert first is None or got == first
        first = got
