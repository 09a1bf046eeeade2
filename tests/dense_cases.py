"""Shapes of the dense operators that together run every kernel of libdkz_dense.so: the
GPU tests take them, and a CPU test looks which kernels they launch.

A linear layer: (type, rows, inputs, outputs, activation, elements off a 16-byte
boundary). A loss with its gradients: (type, rows, inputs, classes, whether in the
least workspace, elements off a 16-byte boundary)."""

from __future__ import annotations

F32, BF16 = 0, 1
TANH, LEAKY = 5, 7  # with an exponential and without: kernels of their own

FORWARD = [
    (F32, 3, 161, 40, TANH, 0), (F32, 3, 161, 40, LEAKY, 0), (F32, 3, 2067, 40, LEAKY, 1), (F32, 3, 2072, 40, TANH, 0),
    (F32, 33, 456, 11755, LEAKY, 0), (F32, 67, 24663, 1, TANH, 0), (F32, 67, 25446, 1, LEAKY, 1), (F32, 93, 972, 10896, LEAKY, 0),
    (F32, 96, 976, 11008, TANH, 1), (F32, 203, 68, 24849, LEAKY, 0), (F32, 688, 5632, 65, TANH, 1), (F32, 793, 293, 5135, TANH, 0),
    (F32, 2048, 400, 2049, LEAKY, 0), (F32, 2822, 2721, 66, TANH, 1), (BF16, 3, 68, 37, TANH, 1), (BF16, 3, 68, 4131, LEAKY, 1),
    (BF16, 3, 69, 37, LEAKY, 1), (BF16, 3, 69, 4165, TANH, 1), (BF16, 3, 70, 37, TANH, 0), (BF16, 3, 70, 4238, LEAKY, 0),
    (BF16, 3, 70, 4276, TANH, 0), (BF16, 3, 72, 37, LEAKY, 0), (BF16, 17, 71, 37, TANH, 0), (BF16, 17, 76, 4168, LEAKY, 1),
    (BF16, 17, 79, 37, LEAKY, 0), (BF16, 18, 68, 37, LEAKY, 0), (BF16, 18, 74, 37, TANH, 0), (BF16, 18, 76, 4308, LEAKY, 0),
    (BF16, 19, 69, 4133, TANH, 0), (BF16, 20, 72, 4171, TANH, 0), (BF16, 33, 1079, 38, TANH, 0), (BF16, 38, 72, 37, LEAKY, 1),
    (BF16, 40, 72, 37, TANH, 1), (BF16, 66, 264, 25511, TANH, 1), (BF16, 68, 72, 8243, TANH, 0), (BF16, 68, 74, 8403, LEAKY, 0),
    (BF16, 72, 72, 24994, LEAKY, 1), (BF16, 130, 4100, 200, LEAKY, 0), (BF16, 385, 203, 28301, TANH, 0),
    (BF16, 390, 200, 28300, LEAKY, 0), (BF16, 777, 1000, 2500, TANH, 1), (BF16, 777, 1001, 2503, LEAKY, 0),
    (BF16, 3397, 1130, 1, LEAKY, 0), (BF16, 3500, 136, 3400, TANH, 0), (BF16, 3549, 1100, 2, TANH, 1),
]

BACKWARD = [
    (F32, 3, 69, 161, TANH, 1), (F32, 3, 72, 163, TANH, 0), (F32, 3, 72, 32640, LEAKY, 1), (F32, 3, 195, 24705, TANH, 0),
    (F32, 3, 19688, 129, TANH, 0), (F32, 96, 10968, 967, LEAKY, 0), (F32, 133, 19875, 13, TANH, 1), (F32, 133, 26209, 296, TANH, 0),
    (F32, 161, 72, 37, TANH, 0), (F32, 170, 68, 37, LEAKY, 1), (F32, 199, 24922, 13, LEAKY, 1), (F32, 293, 26240, 138, LEAKY, 1),
    (F32, 312, 22008, 162, TANH, 0), (F32, 2110, 69, 37, TANH, 0), (F32, 8170, 68, 8, LEAKY, 0), (BF16, 3, 76, 32528, TANH, 1),
    (BF16, 3, 395, 25129, TANH, 1), (BF16, 3, 26176, 67, TANH, 1), (BF16, 72, 26040, 37, LEAKY, 1), (BF16, 130, 3400, 3500, LEAKY, 0),
    (BF16, 2000, 1000, 1500, LEAKY, 0), (BF16, 2000, 1000, 1500, LEAKY, 1), (BF16, 3368, 3615, 37, LEAKY, 1),
    (BF16, 3476, 855, 131, TANH, 1), (BF16, 3500, 300, 3400, LEAKY, 0), (BF16, 3500, 3400, 100, LEAKY, 0),
]

LOSS = [
    (F32, 3, 72, 2065, False, 0), (F32, 3, 193, 24926, False, 1), (F32, 3, 2059, 40, True, 1), (F32, 3, 20504, 129, True, 0),
    (F32, 34, 458, 10972, False, 1), (F32, 96, 1032, 10976, False, 1), (F32, 100, 25288, 1, True, 0), (F32, 305, 6808, 584, False, 0),
    (F32, 308, 297, 13085, False, 1), (F32, 1000, 400, 2101, False, 0), (F32, 1070, 10954, 87, True, 0), (F32, 5474, 1382, 65, True, 0),
    (BF16, 3, 68, 4216, True, 0), (BF16, 3, 69, 4105, False, 0), (BF16, 3, 72, 326, True, 1), (BF16, 3, 72, 25024, False, 1),
    (BF16, 3, 80, 4232, False, 1), (BF16, 3, 388, 24786, False, 0), (BF16, 17, 72, 4300, False, 1), (BF16, 17, 76, 37, False, 0),
    (BF16, 17, 80, 37, True, 1), (BF16, 18, 72, 4216, False, 0), (BF16, 74, 24688, 37, True, 1), (BF16, 129, 73, 24588, False, 1),
    (BF16, 1500, 200, 4100, False, 0), (BF16, 1500, 200, 4100, False, 1), (BF16, 3500, 200, 3601, False, 0),
    (BF16, 5149, 2328, 1744, True, 0), (BF16, 5608, 134, 460, True, 1), (BF16, 6368, 464, 944, True, 1),
    (BF16, 7020, 1699, 37, False, 1), (BF16, 7064, 400, 732, True, 0), (BF16, 7136, 392, 129, False, 0),
]

# bf16 losses in a workspace between the least and the best: some pieces, whose products are cut along the classes.
PIECES = [(5, 72, 5000), (129, 265, 5001), (257, 520, 6000), (300, 400, 4100)]


def between(sizes: tuple[int, int]) -> int:
    """A workspace's bytes for PIECES."""
    least, best = sizes
    return (least + (best - least) // 10 * 9) // 4 * 4
