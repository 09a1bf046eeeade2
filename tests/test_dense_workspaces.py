"""What the workspaces of the cross-entropy hold, by size, on the CPU."""

from __future__ import annotations

import pytest

from darknet_zig_amd import gpu

F32, BF16 = gpu.F32, gpu.BF16
SHAPES = [(1, 8, 5), (32, 4096, 65536), (33, 40, 1000), (4096, 4096, 65536), (1 << 19, 16, 5000), (1 << 20, 8, 257), (1 << 22, 8, 1000),
          (1 << 24, 8, 300), (1 << 26, 8, 4096), (1 << 26, 31, 100)]


def padded(n: int) -> int:
    return -(-n // 256) * 256


def pieces(size: int, rows: int, classes: int) -> int:
    """Bytes of a piece's logits or deltas at most: half a gigabyte, but at least 256 classes, or all."""
    return padded(max(min(1 << 29, size * rows * (classes + 63)), size * rows * min(256, classes + 63)))


@pytest.mark.parametrize("rows,inputs,classes", SHAPES)
@pytest.mark.parametrize("type", [F32, BF16])
def test_backward(type, rows, inputs, classes):
    """A piece's deltas; their sums for the biases (one for every 16 rows at least, or for each of few rows); bf16: the input's gradient
    in fp32 where the classes are several pieces, copies of operands whose rows are no whole eights, partial sums of at
    most 1024 tiles; fp32: partial sums of at most 64 MiB."""
    size = 4 if type == F32 else 2
    d = pieces(size, rows, classes)
    sums = padded(d // size * 4 // (16 if rows > 32 else 1) + 4 * classes + 4 * 64 * classes)
    rest = 1 << 26 if type == F32 else (padded(4 * rows * inputs) + (0 if inputs % 8 == 0 else padded(2 * (rows + classes) * (inputs + 8)) + 512)
                                       + 1024 * 256 * 256 * 4)
    least, best = gpu.linearCrossEntropyBackwardWorkspace(type, rows, inputs, classes)
    assert 0 < least <= best <= d + sums + rest


@pytest.mark.parametrize("rows,inputs,classes", SHAPES)
def test_forward_of_fp32_takes_the_classes_in_pieces(rows, inputs, classes):
    """A piece's logits, the rows' pairs and their targets' logits, partial sums of at most 64 MiB."""
    least, best = gpu.linearCrossEntropyForwardWorkspace(F32, rows, inputs, classes)
    assert 0 < least <= best <= pieces(4, rows, classes) + padded(8 * rows) + padded(4 * rows) + (1 << 26)


@pytest.mark.parametrize("rows,inputs,classes", SHAPES)
def test_forward_of_bf16_takes_all_classes_at_once(rows, inputs, classes):
    """A pair for every 16 to 128 classes of a row, its target's logit, copies of operands whose rows are no whole eights."""
    least, best = gpu.linearCrossEntropyForwardWorkspace(BF16, rows, inputs, classes)
    assert least == best
    copies = 0 if inputs % 8 == 0 or rows <= 32 else 2 * (rows + classes) * (-(-inputs // 8) * 8)
    assert rows * (8 * -(-classes // 128) + 4) + copies <= best <= padded(8 * rows * (classes // 16 + 8)) + padded(4 * rows) + copies + 512
