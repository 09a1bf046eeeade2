"""Every kernel of the dense operators, on the GPU: shapes that take large tiles and small ones, cut products and
their joins, operands straight to LDS and through registers, few rows, pairs, streamed tiles (dense_cases.py), against
64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_cases as cases
from . import dense_ref as ref
from . import test_gpu_dense_cross_entropy as cross_entropy
from . import test_gpu_dense_linear as linear
from .dense_ref import BF16, F32, Pool

pytestmark = pytest.mark.gpu


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


@pytest.mark.parametrize("case", cases.FORWARD, ids=str)
def test_forward(pool, case):
    kind, rows, inputs, outputs, act, shift = case
    linear.run_forward(pool, kind, rows, inputs, outputs, act, 0.25, True, True, True, shift=shift)


@pytest.mark.parametrize("case", cases.BACKWARD, ids=str)
def test_backward(pool, case):
    kind, rows, inputs, outputs, act, shift = case
    linear.run_backward(pool, kind, rows, inputs, outputs, act, 0.25, True, beta=0.5, shift=shift)


@pytest.mark.parametrize("act", [ref.LINEAR, ref.RELU])
@pytest.mark.parametrize("shape,prob", [((300, 136, 200), 0.1), ((70, 41, 53), 0.3), ((3400, 72, 264), 0.1), ((64, 64, 64), 0.0)], ids=str)
def test_backward_rounds_no_delta_that_is_kept_or_dropped(pool, act, shape, prob):
    """Where the gradient is 0 or 1, d is the scale times a bf16 delta or 0: the products take it unrounded, and their results
    are off by their own rounding alone."""
    rows, inputs, outputs = shape
    r = np.random.default_rng(rows + inputs)
    x, w, delta, a = (ref.rounded(r.normal(size=s), BF16) for s in ((rows, inputs), (outputs, inputs), (rows, outputs), (rows, outputs)))
    scale, seed = 1 / (1 - prob) if prob else 1.7, 11
    dx, dw, dd, da = (pool(v, BF16) for v in (x, w, delta, a))
    gb, gw, gx = pool(n=outputs), pool(kind=BF16, n=(outputs, inputs)), pool(kind=BF16, n=(rows, inputs))
    ws = pool.work(gpu.linearBackwardWorkspace(BF16, rows, inputs, outputs))
    gpu.linearBackward(BF16, rows, inputs, outputs, act, prob, scale, seed, 0, dx.buf, dw.buf, da.buf if act != ref.LINEAR else None, dd.buf, None,
                       0.0, gb.buf, gw.buf, gx.buf, ws.buf)
    drop = ref.dropped(rows * outputs, prob, seed, 0).reshape(rows, outputs)
    d = np.where(drop, 0.0, delta.astype(np.float64) * float(np.float32(scale))) * ref.gradient(act, a.astype(np.float64))
    for got, p, q, what in ((gw, d.T, x, "weight_updates"), (gx, d, w, "input_delta")):
        q = q.astype(np.float64)
        y, err = p @ q, ref.product_error(p, q) * 1.01
        err = err + 2.0**-24 * np.abs(y)  # the scale
        ref.assert_within(got.get(), y, err + ref.HALF[BF16] * (np.abs(y) + err), what)
    total = d.sum(0)  # 64 rows in fp32, each element off by its scaling's rounding at most, then 64 bits and two roundings
    ref.assert_within(gb.get(), total, (65 * np.abs(d).sum(0) + 3 * np.abs(total)) * 2.0**-24, "bias_updates")


@pytest.mark.parametrize("kind", [F32, BF16])
def test_backward_of_everything_dropped(pool, kind):
    """prob 1: the scale 1 / (1 - prob) is infinite and no element is kept, so every d is 0, and no gradient a NaN."""
    rows, inputs, outputs = 70, 40, 48
    x, w, d = (pool(np.ones(s, np.float32), kind) for s in ((rows, inputs), (outputs, inputs), (rows, outputs)))
    gb, gw, gx = pool(n=outputs), pool(kind=kind, n=(outputs, inputs)), pool(kind=kind, n=(rows, inputs))
    ws = pool.work(gpu.linearBackwardWorkspace(kind, rows, inputs, outputs))
    gpu.linearBackward(kind, rows, inputs, outputs, ref.LINEAR, 1.0, float("inf"), 1, 0, x.buf, w.buf, None, d.buf, None, 0.0, gb.buf, gw.buf,
                       gx.buf, ws.buf)
    assert not gb.get().any() and not gw.get().any() and not gx.get().any()


@pytest.mark.parametrize("scale", [2.0**-100, 2.0**100])
def test_backward_with_an_extreme_scale(pool, scale):
    """Sums that only the scale keeps in fp32's range: deltas and weights of 2^66, or 2^-66, whose products are 2^132, or 2^-132.
    All values are powers of two and the sums exact."""
    rows, inputs, outputs, v = 48, 40, 64, 2.0**66 if scale < 1 else 2.0**-66
    x, w, d = (pool(np.full(s, v, np.float32), BF16) for s in ((rows, inputs), (outputs, inputs), (rows, outputs)))
    gw, gx = pool(kind=BF16, n=(outputs, inputs)), pool(kind=BF16, n=(rows, inputs))
    ws = pool.work(gpu.linearBackwardWorkspace(BF16, rows, inputs, outputs))
    gpu.linearBackward(BF16, rows, inputs, outputs, ref.LINEAR, 0.0, scale, 1, 0, x.buf, w.buf, None, d.buf, None, 0.0, None, gw.buf, gx.buf, ws.buf)
    assert (gw.get() == rows * v * v * scale).all() and (gx.get() == outputs * v * v * scale).all()


def many_classes(plain, kind, classes):
    """lse_error where a row is more than a few parts. Pairs are merged in at most five roundings, fp32 logits added in at
    most ten for every eight; all terms are positive. bf16: parts of at least 16 classes, a thread merging every 256th, then 9 among
    the workgroup's. fp32: a thread takes eight logits of every 4096, then 13 merges, and one for each piece of at least 256."""
    more = 5 * (-(-classes // 4096) + 9) if kind == BF16 else 10 * -(-classes // 4096) + 5 * (13 + -(-classes // 256))
    return lambda z, err, lse: plain(z, err, lse) + more * 2.0**-24


@pytest.mark.parametrize("case", cases.LOSS, ids=str)
def test_loss_and_gradients(pool, monkeypatch, case):
    kind, rows, inputs, classes, least, shift = case
    monkeypatch.setattr(cross_entropy, "lse_error", many_classes(cross_entropy.lse_error, kind, classes))
    cross_entropy.run(pool, kind, *cross_entropy.make(kind, rows, inputs, classes), scale=0.25, least=least, shift=shift)


@pytest.mark.parametrize("case", cases.PIECES, ids=str)
def test_some_pieces(pool, monkeypatch, case):
    some = cases.between(gpu.linearCrossEntropyBackwardWorkspace(BF16, *case))
    monkeypatch.setattr(gpu, "linearCrossEntropyBackwardWorkspace", lambda *a: (some, some))
    monkeypatch.setattr(cross_entropy, "lse_error", many_classes(cross_entropy.lse_error, BF16, case[2]))
    cross_entropy.run(pool, BF16, *cross_entropy.make(BF16, *case), beta=0.5)


def repeated(outputs, call, times=4):
    """The same bits in every one of some calls, the outputs wiped between them."""
    first = None
    for _ in range(times):
        for d in outputs:
            gpu.push(d.base, d.host.view(np.int32))
        call()
        got = [d.raw().tobytes() for d in outputs]
        assert first is None or got == first
        first = got


@pytest.mark.parametrize("kind,rows,inputs,outputs", [(BF16, 4096, 4096, 4096), (BF16, 8200, 2056, 4104), (BF16, 2000, 1001, 1503),
                                                      (BF16, 3400, 3368, 264), (F32, 1568, 1000, 1000)])
def test_same_call_same_bits_of_large_layers(pool, kind, rows, inputs, outputs):
    r = np.random.default_rng(9)
    x, w, delta, act = (pool(r.standard_normal(s, np.float32), kind) for s in ((rows, inputs), (outputs, inputs), (rows, outputs), (rows, outputs)))
    y, kept, gb = pool(kind=kind, n=(rows, outputs)), pool(kind=kind, n=(rows, outputs)), pool(n=outputs)
    gw, gx = pool(kind=kind, n=(outputs, inputs)), pool(kind=kind, n=(rows, inputs))
    ws = pool.work(max(gpu.linearForwardWorkspace(kind, rows, inputs, outputs), gpu.linearBackwardWorkspace(kind, rows, inputs, outputs)))
    repeated((y, kept), lambda: gpu.linearForward(kind, rows, inputs, outputs, ref.LEAKY, 0.5, 2.0, 7, 0, x.buf, w.buf, None, None, kept.buf,
                                                  y.buf, ws.buf))
    repeated((gb, gw, gx), lambda: gpu.linearBackward(kind, rows, inputs, outputs, ref.LEAKY, 0.5, 2.0, 7, 0, x.buf, w.buf, act.buf,
                                                      delta.buf, None, 0.0, gb.buf, gw.buf, gx.buf, ws.buf))


@pytest.mark.parametrize("kind,rows,inputs,classes", [(BF16, 4096, 1024, 16384), (BF16, 4000, 264, 9001), (F32, 333, 1030, 9001)])
def test_same_call_same_bits_of_large_losses(pool, kind, rows, inputs, classes):
    x, w, b, t = cross_entropy.make(kind, rows, inputs, classes)
    dx, dw, db, dt = pool(x, kind), pool(w, kind), pool(b), pool(t)
    loss, lse, gb = pool(n=rows), pool(n=rows), pool(n=classes)
    gw, gx = pool(kind=kind, n=(classes, inputs)), pool(kind=kind, n=(rows, inputs))
    ws = pool.work(max(f(kind, rows, inputs, classes)[1]
                       for f in (gpu.linearCrossEntropyForwardWorkspace, gpu.linearCrossEntropyBackwardWorkspace)))
    repeated((loss, lse), lambda: gpu.linearCrossEntropyForward(kind, rows, inputs, classes, dx.buf, dw.buf, db.buf, dt.buf, loss.buf,
                                                                lse.buf, ws.buf))
    repeated((gb, gw, gx), lambda: gpu.linearCrossEntropyBackward(kind, rows, inputs, classes, dx.buf, dw.buf, db.buf, dt.buf, lse.buf, None,
                                                                  1.0 / rows, 0.0, gb.buf, gw.buf, gx.buf, ws.buf))
