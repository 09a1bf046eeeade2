"""Linear layers with their epilogue (dkz_linear_forward, dkz_linear_backward) on the GPU,
against their formulas in 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from .dense_ref import BF16, ELU, F32, HALF, LEAKY, LINEAR, LOGISTIC, RELU, SELU, TANH, Pool, assert_within, buf

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


def run_forward(pool, kind, rows, inputs, outputs, act, prob, residual, bias, keep, shift=0, seed=1, first=0, x=None, w=None):
    r = np.random.default_rng(rows * 7919 + inputs * 31 + outputs)
    x = ref.rounded(r.normal(size=(rows, inputs)), kind) if x is None else x
    w = ref.rounded(r.normal(size=(outputs, inputs)) / np.sqrt(max(inputs, 1)), kind) if w is None else w
    b = r.normal(size=outputs).astype(np.float32) if bias else None
    res = ref.rounded(r.normal(size=(rows, outputs)), kind) if residual else None
    scale = 1.0 / (1.0 - prob)
    dx, dw = pool(x, kind, shift=shift), pool(w, kind, shift=shift)
    db, dres = pool(b) if bias else None, pool(res, kind, shift=shift) if residual else None
    out = pool(kind=kind, n=(rows, outputs), shift=shift)
    kept = pool(kind=kind, n=(rows, outputs), shift=shift) if keep else None
    ws = pool.work(gpu.linearForwardWorkspace(kind, rows, inputs, outputs))
    gpu.linearForward(kind, rows, inputs, outputs, act, prob, scale, seed, first, dx.buf, dw.buf, buf(db), buf(dres), buf(kept),
                      out.buf, buf(ws))
    if ws is not None:
        ws.raw()
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    z = x64 @ w64.T
    z_err = ref.product_error(x64, w64.T)
    if bias:
        z = z + b
        z_err = z_err + 2.0**-24 * np.abs(z)
    a = ref.activate(act, z)
    a_err = ref.SLOPE[act] * z_err + (ref.ACT_ROUNDINGS * 2.0**-24 * (1 + np.abs(a)) if act != LINEAR else 0)
    if keep:
        assert_within(kept.get(), a, a_err + HALF[kind] * (np.abs(a) + a_err), "activated")
    drop = ref.dropped(rows * outputs, prob, seed, first).reshape(rows, outputs)
    s = float(np.float32(scale))
    y, y_err = np.where(drop, 0.0, a * s), np.where(drop, 0.0, (a_err + 2.0**-24 * np.abs(a)) * s)
    if residual:
        y = y + res
        y_err = y_err + 2.0**-24 * np.abs(y)
    assert_within(out.get(), y, y_err + HALF[kind] * (np.abs(y) + y_err), "output")
    for d in (dx, dw, db, dres):
        if d is not None:
            d.raw()
    return out


SHAPES = [(1, 1, 1), (1, 64, 5), (2, 8, 8), (3, 7, 9), (16, 65, 33), (31, 129, 130), (128, 128, 128), (129, 200, 257), (1, 1000, 1003),
          (5, 4096, 40), (300, 72, 264), (64, 1032, 520)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_forward_shapes_and_alignments(pool, kind, shape, shift):
    run_forward(pool, kind, *shape, LEAKY, 0.25, True, True, True, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 70, 8192), (16, 129, 8190), (3, 8200, 9000), (17, 64, 5001), (32, 200, 4097)], ids=str)
def test_forward_few_rows_of_many_outputs(pool, kind, shape):
    run_forward(pool, kind, *shape, RELU, 0.2, True, True, True)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", [LOGISTIC, RELU, LINEAR, TANH, LEAKY, ELU, SELU])
@pytest.mark.parametrize("extras", [(0.0, False, False, False), (0.5, False, True, True), (0.0, True, False, True)], ids=str)
def test_forward_activations_and_operands(pool, kind, act, extras):
    prob, residual, bias, keep = extras
    run_forward(pool, kind, 70, 96, 132, act, prob, residual, bias, keep, first=2**32 - 4000)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_forward_every_activation_is_the_framework_s(pool, kind):
    """fp32: the bits of activate_array on the product. bf16: its value rounded once, but for the exponentials, whose
    formulas of at most six fp32 roundings (an exponential and a reciprocal within a step each, 1.76 the largest factor)
    are within 2^-21 of the larger of 1 and the value before that rounding."""
    r = np.random.default_rng(3)
    rows, n = 40, 36
    x = ref.rounded(r.normal(size=(rows, n)) * 3, kind)
    w = np.eye(n, dtype=np.float32)  # the product is the input, exactly
    for act in range(14):
        dx, dw, out = pool(x, kind), pool(w, kind), pool(kind=kind, n=(rows, n))
        ws = pool.work(gpu.linearForwardWorkspace(kind, rows, n, n))
        gpu.linearForward(kind, rows, n, n, act, 0.0, 1.0, 0, 0, dx.buf, dw.buf, None, None, None, out.buf, buf(ws))
        want = pool(x)
        gpu.activateArray(want.buf, x.size, act)
        expect, got = want.get(), out.get()
        if kind == BF16 and act in (LOGISTIC, TANH, ELU, SELU, 9):
            assert_within(got, expect, 2.0**-21 * np.maximum(1, np.abs(expect)) + HALF[BF16] * np.abs(expect), f"activation {act}")
        else:
            assert (got == ref.rounded(expect, kind)).all(), (act, np.argwhere(got != ref.rounded(expect, kind))[:4])


def test_forward_bf16_exponentials_saturate(pool):
    x = np.array([[-200.0, -89, -50, -20, 0, 20, 45, 89, 200, np.inf, -np.inf, np.nan]], np.float32).T
    one = np.ones((1, 1), np.float32)
    with np.errstate(over="ignore"):
        want = {LOGISTIC: 1 / (1 + np.exp(-x)), TANH: np.tanh(x), ELU: np.where(x >= 0, x, np.expm1(np.minimum(x, 0)))}
    dx, dw, out = pool(x, BF16), pool(one, BF16), pool(kind=BF16, n=(12, 1))
    for act, w in want.items():
        gpu.linearForward(BF16, 12, 1, 1, act, 0.0, 1.0, 0, 0, dx.buf, dw.buf, None, None, None, out.buf, None)
        got = out.get()
        assert np.isnan(got[11]) and (got[:11][np.isinf(w[:11])] == w[:11][np.isinf(w[:11])]).all()
        fine = np.isfinite(w)
        assert_within(got[fine], w[fine], 2.0**-21 + HALF[BF16] * np.abs(w[fine]), f"activation {act}")


@pytest.mark.parametrize("kind", [F32, BF16])
def test_forward_without_inputs_is_the_bias(pool, kind):
    run_forward(pool, kind, 5, 0, 12, RELU, 0.0, True, True, False)
    run_forward(pool, kind, 3, 0, 7, LINEAR, 0.0, False, False, False)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_forward_output_onto_the_residual(pool, kind):
    rows, k, n = 33, 40, 50
    r = np.random.default_rng(2)
    x, w = ref.rounded(r.normal(size=(rows, k)), kind), ref.rounded(r.normal(size=(n, k)), kind)
    res = ref.rounded(r.normal(size=(rows, n)), kind)
    a, b, c = pool(x, kind), pool(w, kind), pool(res, kind)
    apart, out = pool(res, kind), pool(kind=kind, n=(rows, n))
    ws = pool.work(gpu.linearForwardWorkspace(kind, rows, k, n))
    gpu.linearForward(kind, rows, k, n, TANH, 0.3, 1.5, 4, 0, a.buf, b.buf, None, apart.buf, None, out.buf, buf(ws))
    gpu.linearForward(kind, rows, k, n, TANH, 0.3, 1.5, 4, 0, a.buf, b.buf, None, c.buf, None, c.buf, buf(ws))
    assert (c.raw() == out.raw()).all()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_forward_specials_stay_in_their_rows_and_columns(pool, kind):
    rows, k, n = 140, 150, 136
    r = np.random.default_rng(6)
    x, w = r.normal(size=(rows, k)), r.normal(size=(n, k))
    x[5, 149], x[77, 0], w[100, 3] = np.nan, np.inf, -np.inf
    x, w = ref.rounded(x, kind), ref.rounded(w, kind)
    dx, dw, out = pool(x, kind), pool(w, kind), pool(kind=kind, n=(rows, n))
    ws = pool.work(gpu.linearForwardWorkspace(kind, rows, k, n))
    gpu.linearForward(kind, rows, k, n, LINEAR, 0.0, 1.0, 0, 0, dx.buf, dw.buf, None, None, None, out.buf, buf(ws))
    got = out.get()
    with np.errstate(invalid="ignore"):
        z = x.astype(np.float64) @ w.astype(np.float64).T
    assert (np.isnan(got) == np.isnan(z)).all() and (np.isinf(got) == np.isinf(z)).all()
    assert (np.sign(got[np.isinf(z)]) == np.sign(z[np.isinf(z)])).all()
    fine = np.isfinite(z)
    xf, wf = np.where(np.isfinite(x), x, 0).astype(np.float64), np.where(np.isfinite(w), w, 0).astype(np.float64)
    bound = ref.product_error(xf, wf.T) + HALF[kind] * np.abs(z)
    assert_within(np.where(fine, got, 0), np.where(fine, z, 0), np.where(fine, bound, 0), "finite part")


# ---- backward ----


def run_backward(pool, kind, rows, inputs, outputs, act, prob, add, beta=0.0, shift=0, seed=5, first=0, want=(1, 1, 1), onto=False):
    r = np.random.default_rng(rows * 104729 + inputs * 17 + outputs)
    x = ref.rounded(r.normal(size=(rows, inputs)), kind)
    w = ref.rounded(r.normal(size=(outputs, inputs)), kind)
    act_out = ref.rounded(ref.activate(act, r.normal(size=(rows, outputs))), kind)
    delta = ref.rounded(r.normal(size=(rows, outputs)), kind)
    res = ref.rounded(r.normal(size=(rows, inputs)), kind) if add else None
    bu, wu = r.normal(size=outputs).astype(np.float32), ref.rounded(r.normal(size=(outputs, inputs)), kind)
    if beta == 0:
        bu, wu = np.full_like(bu, np.nan), np.full_like(wu, np.nan)  # not read
    scale = 1.0 / (1.0 - prob)
    dx, dw, dd = pool(x, kind, shift=shift), pool(w, kind, shift=shift), pool(delta, kind, shift=shift)
    da = pool(act_out, kind, shift=shift) if act != LINEAR else None
    dres = pool(res, kind, shift=shift) if add else None
    out_b, out_w = pool(bu) if want[0] else None, pool(wu, kind, shift=shift) if want[1] else None
    out_x = (dres if onto else pool(kind=kind, n=(rows, inputs), shift=shift)) if want[2] else None
    ws = pool.work(gpu.linearBackwardWorkspace(kind, rows, inputs, outputs))
    gpu.linearBackward(kind, rows, inputs, outputs, act, prob, scale, seed, first, dx.buf, dw.buf, buf(da), dd.buf, buf(dres), beta,
                       buf(out_b), buf(out_w), buf(out_x), buf(ws))
    if ws is not None:
        ws.raw()
    drop = ref.dropped(rows * outputs, prob, seed, first).reshape(rows, outputs)
    a64 = act_out.astype(np.float64)
    d = np.where(drop, 0.0, delta.astype(np.float64) * float(np.float32(scale))) * ref.gradient(act, a64)
    # fp32: a product and a gradient of up to three roundings; bf16: rounded once more for the products.
    d_err = 5 * 2.0**-24 * np.abs(delta) * scale * (1 + a64 * a64)
    p_err = d_err + (HALF[BF16] * np.abs(d) * (1 + 2.0**-8) if kind == BF16 else 0)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    if out_b is not None:
        base = beta * bu.astype(np.float64) if beta else 0.0
        total = base + d.sum(0)
        # sums of at most 64 rows in fp32, then 64 bits, then two roundings
        err = d_err.sum(0) + 64 * 2.0**-24 * np.abs(d).sum(0) + 3 * 2.0**-24 * (np.abs(total) + np.abs(base))
        assert_within(out_b.get(), total, err, "bias_updates")
    for got, a, b, e, base, name in (
        (out_w, d.T, x64, p_err.T, beta * wu.astype(np.float64) if beta else 0.0, "weight_updates"),
        (out_x, d, w64, p_err, res.astype(np.float64) if add else 0.0, "input_delta"),
    ):
        if got is None:
            continue
        y = a @ b + base
        err = ref.product_error(a, b) * 1.01 + e @ np.abs(b) + 3 * 2.0**-24 * (np.abs(y) + np.abs(base))
        assert_within(got.get(), y, err + HALF[kind] * (np.abs(y) + err), name)
    for t in (dx, dw, dd, da):
        if t is not None:
            t.raw()


BACK_SHAPES = [(1, 1, 1), (1, 8, 5), (3, 7, 9), (16, 64, 32), (65, 33, 130), (128, 128, 128), (200, 129, 77), (257, 264, 72), (1, 1003, 300),
               (700, 40, 24)]


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", BACK_SHAPES, ids=str)
@pytest.mark.parametrize("shift", [0, 1])
def test_backward_shapes_and_alignments(pool, kind, shape, shift):
    run_backward(pool, kind, *shape, LEAKY, 0.25, True, shift=shift)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", [(1024, 1000, 1024), (100, 8, 32768), (4096, 16, 512), (64, 24, 40), (129, 30, 33)], ids=str)
def test_backward_many_and_few_rows(pool, kind, shape):
    """Bias sums in one launch and in two, eight columns a thread and one, both products in one launch."""
    run_backward(pool, kind, *shape, RELU, 0.5, False, beta=0.5)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("act", [LOGISTIC, RELU, LINEAR, TANH, ELU, SELU])
@pytest.mark.parametrize("prob", [0.0, 0.5])
def test_backward_activations(pool, kind, act, prob):
    run_backward(pool, kind, 70, 72, 90, act, prob, False, first=2**32 - 1000)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("beta", [1.0, 0.5])
def test_backward_adds_to_the_updates(pool, kind, beta):
    run_backward(pool, kind, 40, 48, 56, RELU, 0.0, False, beta=beta)
    run_backward(pool, kind, 33, 17, 21, LINEAR, 0.0, False, beta=beta)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("want", [(1, 0, 0), (0, 1, 0), (0, 0, 1), (0, 1, 1)])
def test_backward_computes_what_is_asked_for(pool, kind, want):
    run_backward(pool, kind, 40, 48, 56, TANH, 0.1, True, want=want)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_adds_onto_the_input_delta(pool, kind):
    run_backward(pool, kind, 37, 41, 43, RELU, 0.0, True, onto=True)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_without_rows_keeps_beta_of_the_updates(pool, kind):
    b, w = np.arange(6, dtype=np.float32), ref.rounded(np.arange(24).reshape(6, 4), kind)
    db, dw = pool(b), pool(w, kind)
    gpu.linearBackward(kind, 0, 4, 6, LINEAR, 0.0, 1.0, 0, 0, None, None, None, None, None, 0.5, db.buf, dw.buf, None, None)
    assert (db.get() == 0.5 * b).all() and (dw.get() == 0.5 * w).all()


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("outputs", [6, 8])
def test_backward_without_inputs_touches_no_delta_unless_for_the_bias(pool, kind, outputs):
    """No inputs: weights and input gradients are empty, whatever their pointers, and delta is read for the bias alone."""
    rows, some = 5, pool(np.zeros(8, np.float32))
    ws = pool.work(gpu.linearBackwardWorkspace(kind, rows, 0, outputs))
    gpu.linearBackward(kind, rows, 0, outputs, RELU, 0.5, 2.0, 0, 0, None, None, None, None, None, 0.0, None, some.buf, some.buf, buf(ws))
    assert (some.get() == 0).all()
    run_backward(pool, kind, rows, 0, outputs, RELU, 0.5, False, want=(1, 0, 0))


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_is_the_forward_s_derivative(pool, kind):
    """Differences: the gradients of L = sum(g * output) by weights, biases and input, against central differences of
    the 64-bit forward with the GPU's own draws."""
    rows, k, n, prob, seed = 9, 11, 13, 0.3, 21
    r = np.random.default_rng(4)
    x, w = ref.rounded(r.normal(size=(rows, k)), kind), ref.rounded(r.normal(size=(n, k)) * 0.3, kind)
    b, g = r.normal(size=n).astype(np.float32), ref.rounded(r.normal(size=(rows, n)), kind)
    scale = 1 / (1 - prob)
    drop = ref.dropped(rows * n, prob, seed, 0).reshape(rows, n)

    def loss(x, w, b):
        return (np.where(drop, 0, np.tanh(x @ w.T + b) * scale) * g).sum()

    dx, dw, db, dg = pool(x, kind), pool(w, kind), pool(b), pool(g, kind)
    act, out = pool(kind=kind, n=(rows, n)), pool(kind=kind, n=(rows, n))
    ws = pool.work(max(4, gpu.linearForwardWorkspace(kind, rows, k, n), gpu.linearBackwardWorkspace(kind, rows, k, n)))
    gpu.linearForward(kind, rows, k, n, TANH, prob, scale, seed, 0, dx.buf, dw.buf, db.buf, None, act.buf, out.buf, ws.buf)
    gb, gw, gx = pool(n=n), pool(kind=kind, n=(n, k)), pool(kind=kind, n=(rows, k))
    gpu.linearBackward(kind, rows, k, n, TANH, prob, scale, seed, 0, dx.buf, dw.buf, act.buf, dg.buf, None, 0.0, gb.buf, gw.buf, gx.buf,
                       ws.buf)
    h = 1e-4  # truncation h^2/6 * third derivative (below 2 * magnitudes): 1e-8 of them; rounding 1e-16/h
    x64, w64, b64 = x.astype(np.float64), w.astype(np.float64), b.astype(np.float64)
    # The kernel's activation is rounded to its type: the slope 1 - a^2 is off by 2|a| half steps, d and the result by one each.
    tol = 4 * HALF[kind] + 1e-6
    for got, base, which in ((gb.get(), b64, 2), (gw.get(), w64, 1), (gx.get(), x64, 0)):
        num, size = np.empty_like(base), np.abs(g).sum() * scale
        for i in np.ndindex(base.shape):
            args = [x64, w64, b64]
            up, down = base.copy(), base.copy()
            up[i] += h
            down[i] -= h
            num[i] = (loss(*args[:which], up, *args[which + 1 :]) - loss(*args[:which], down, *args[which + 1 :])) / (2 * h)
        mags = {2: np.abs(g).sum(0), 1: np.abs(g).T @ np.abs(x64), 0: np.abs(g) @ np.abs(w64)}[which] * scale
        assert_within(got, num, tol * mags + 1e-7 * size, ("input", "weights", "biases")[which])


@pytest.mark.parametrize("kind", [F32, BF16])
def test_more_rows_than_a_grid_side(pool, kind):
    """Workgroups of 64 rows: 65537 of them and more. Values -1, 0 and 1: every sum is a whole number below 2^24, exact in
    fp32, so that only the rounding to the result's type is left."""
    rows, k, n = 4194304 + 65, 2, 3
    r = np.random.default_rng(1)
    x, w, d = (r.integers(-1, 2, s).astype(np.float32) for s in ((rows, k), (n, k), (rows, n)))
    dx, dw, dd = pool(x, kind), pool(w, kind), pool(d, kind)
    y, gx, gb, gw = pool(kind=kind, n=(rows, n)), pool(kind=kind, n=(rows, k)), pool(n=n), pool(kind=kind, n=(n, k))
    ws = pool.work(max(gpu.linearForwardWorkspace(kind, rows, k, n), gpu.linearBackwardWorkspace(kind, rows, k, n)))
    gpu.linearForward(kind, rows, k, n, LINEAR, 0.0, 1.0, 0, 0, dx.buf, dw.buf, None, None, None, y.buf, buf(ws))
    gpu.linearBackward(kind, rows, k, n, LINEAR, 0.0, 1.0, 0, 0, dx.buf, dw.buf, None, dd.buf, None, 0.0, gb.buf, gw.buf, gx.buf, buf(ws))
    x64, w64, d64 = x.astype(np.float64), w.astype(np.float64), d.astype(np.float64)
    assert (y.get() == ref.rounded(x64 @ w64.T, kind)).all()
    assert (gx.get() == ref.rounded(d64 @ w64, kind)).all()
    assert (gb.get() == d64.sum(0)).all()
    assert (gw.get() == ref.rounded(d64.T @ x64, kind)).all()
