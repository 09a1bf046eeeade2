"""The dense operators at their largest sizes, on the GPU."""

from __future__ import annotations

import numpy as np
import pytest

from darknet_zig_amd import gpu

from . import dense_ref as ref
from .dense_ref import BF16, assert_within

pytestmark = pytest.mark.gpu


def fill(b: gpu.Buf, value: float) -> None:
    for at in range(0, b.len, 1 << 30):
        part = b.offset(at)
        gpu.fill(part, min(part.len, 1 << 30), value)


def test_the_most_logits(dev):
    """2^38 logits through registers (the inputs lie off a 16-byte boundary): a product of 2^24 workgroups, whose threads are too
    many for one launch. Every row has a class of its own with weights, the other classes' are 0."""
    rows, inputs, classes = 4096, 8, 1 << 26
    r = np.random.default_rng(38)
    at = np.sort(r.choice(classes, rows, replace=False)).astype(np.int32)
    at[0], at[-1] = 0, classes - 1
    t = r.permutation(at).astype(np.int32)
    x, w = ref.rounded(r.normal(size=(rows, inputs)), BF16), ref.rounded(r.normal(size=(rows, inputs)) * 2, BF16)
    dx, dt, loss, lse = ref.Dev(x, BF16, shift=1), ref.Dev(t), ref.Dev(n=rows), ref.Dev(n=rows)
    weights = gpu.alloc(classes * inputs // 2)
    ws = gpu.alloc(gpu.linearCrossEntropyForwardWorkspace(BF16, rows, inputs, classes)[0] // 4)
    try:
        fill(ws, 1e30)  # a part that is not written would be the row's largest
        for c, row in zip(at, ref.to_bf16(w)):
            gpu.push(weights.offset(int(c) * inputs // 2), row.view(np.int32))
        gpu.linearCrossEntropyForward(BF16, rows, inputs, classes, dx.buf, weights, None, dt.buf, loss.buf, lse.buf, ws)
        got_loss, got_lse = loss.get(), lse.get()
    finally:
        for b in (weights, ws, dx.base, dt.base, loss.base, lse.base):
            gpu.free(b)
    x64, w64 = x.astype(np.float64), w.astype(np.float64)
    z = x64 @ w64.T
    want = np.log(np.exp(z).sum(1) + (classes - rows))
    # A thread of the row's merges 2^20 / 256 pairs one by one, then 6 + 3 among the workgroup's; a merge is two exponentials
    # within a step, two products and a sum: five roundings at most of all positive terms. Before them a wave's sums of 64 exponentials,
    # each off by its argument's roundings (2^-24 of |z|, the maximum and their difference) and a step; at last the logarithm.
    parts = 2.0**-24 * (5 * (4096 + 9) + 64 + 4 * np.abs(z).max() + 4)
    err = parts + 2.0**-23 * np.abs(want) + ref.product_error(x64, w64.T).max()
    assert_within(got_lse, want, err, "lse")
    target = z[np.arange(rows), np.searchsorted(at, t)]
    assert_within(got_loss, want - target, err + 2.0**-23 * (np.abs(want) + np.abs(target)), "loss")
