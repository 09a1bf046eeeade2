"""Shapes of gated blocks that together run every kernel of libdkz_lm.so's: the GPU tests take them, and a CPU test looks
which kernels they launch. (type, rows, inputs, hidden, activation, elements off a 16-byte boundary)."""

from __future__ import annotations

F32, BF16 = 0, 1
RELU, SILU = 1, 14  # without an exponential and with: kernels of their own

FORWARD = [
    (F32, 1, 664, 1, RELU, 0), (F32, 3, 132, 1, RELU, 0), (F32, 17, 2959, 1, SILU, 0), (F32, 17, 4136, 14, SILU, 0), (F32, 17, 5768,
    13720, RELU, 1), (F32, 20, 2720, 500, RELU, 0), (F32, 232, 5911, 968, SILU, 0), (F32, 312, 78, 6064, RELU, 0), (F32, 3155, 5864,
    161, SILU, 1), (F32, 4241, 3360, 20, RELU, 0), (BF16, 1, 80, 2472, RELU, 0), (BF16, 1, 4824, 3904, SILU, 0), (BF16, 3, 500, 385,
    SILU, 0), (BF16, 3, 1123, 12303, RELU, 0), (BF16, 8, 102, 6824, SILU, 1), (BF16, 8, 2367, 3049, RELU, 0), (BF16, 8, 3843, 37, SILU,
    0), (BF16, 16, 2166, 272, RELU, 0), (BF16, 17, 184, 7714, RELU, 0), (BF16, 17, 248, 53, SILU, 1), (BF16, 17, 545, 2051, RELU, 0),
    (BF16, 17, 2343, 2163, SILU, 0), (BF16, 17, 5512, 408, SILU, 0), (BF16, 20, 574, 5194, SILU, 0), (BF16, 23, 72, 197, RELU, 0),
    (BF16, 32, 535, 296, RELU, 1), (BF16, 48, 512, 5, RELU, 1), (BF16, 59, 361, 240, SILU, 0), (BF16, 60, 2424, 717, RELU, 0), (BF16,
    128, 2832, 1552, SILU, 1), (BF16, 224, 2840, 24, SILU, 0), (BF16, 460, 205, 8616, RELU, 1), (BF16, 872, 952, 3632, RELU, 0), (BF16,
    1064, 265, 5784, SILU, 0), (BF16, 1334, 112, 10000, RELU, 0), (BF16, 1741, 264, 936, SILU, 0), (BF16, 1830, 69, 16, RELU, 0), (BF16,
    1830, 128, 7308, SILU, 1), (BF16, 3720, 5690, 30, RELU, 0), (BF16, 4267, 242, 2679, SILU, 0), (BF16, 4608, 96, 695, RELU, 1),
    (F32, 48, 2768, 9464, SILU, 0), (F32, 88, 238, 3, SILU, 0), (F32, 3848, 13, 670, SILU, 0),
]

BACKWARD = [
    (F32, 3, 132, 1, RELU, 0), (F32, 3, 152, 7696, SILU, 0), (F32, 17, 4136, 14, SILU, 0), (F32, 20, 485, 4248, SILU, 0), (F32, 20,
    1626, 13224, RELU, 0), (F32, 20, 2720, 500, RELU, 0), (F32, 37, 3453, 2392, SILU, 1), (F32, 232, 5911, 968, SILU, 0), (F32, 322,
    288, 11416, RELU, 0), (F32, 1021, 744, 2, SILU, 1), (F32, 1060, 2720, 1378, SILU, 1), (F32, 1168, 1749, 1029, SILU, 0), (F32, 1552,
    122, 11128, SILU, 0), (F32, 1714, 5664, 192, SILU, 0), (F32, 2976, 152, 1, RELU, 0), (F32, 3056, 784, 5, SILU, 1), (F32, 4241, 3360,
    20, RELU, 0), (BF16, 1, 80, 2472, RELU, 0), (BF16, 8, 2367, 3049, RELU, 0), (BF16, 17, 248, 53, SILU, 1), (BF16, 17, 4064, 892,
    RELU, 1), (BF16, 59, 361, 240, SILU, 0), (BF16, 460, 205, 8616, RELU, 1), (BF16, 872, 952, 3632, RELU, 0), (BF16, 1741, 264, 936,
    SILU, 0), (BF16, 1886, 3304, 5, SILU, 1), (BF16, 4267, 242, 2679, SILU, 0), (BF16, 5832, 2652, 77, SILU, 1),
    (F32, 5, 9, 36272, SILU, 1), (F32, 7, 8, 38488, RELU, 0), (BF16, 7, 16, 39224, SILU, 1), (BF16, 100, 16, 33800, RELU, 0),
    (BF16, 857, 46, 5, RELU, 0), (BF16, 2863, 2712, 584, SILU, 0),
    (BF16, 8896, 73, 16, SILU, 0), (BF16, 6776, 8, 1104, RELU, 0), (BF16, 3808, 8, 2232, SILU, 0), (F32, 1636, 8, 6320, RELU, 0), (F32, 2104,
    12, 16, SILU, 0),
]

# The same with some results alone (bias, weights, input).
BACKWARD_PARTS = [((BF16, 16, 8, 21, SILU, 0), (1, 1, 0)), ((BF16, 16, 8, 21, SILU, 0), (1, 0, 1)), ((BF16, 16, 1560, 3877, RELU, 0), (1, 1, 0)),
                  ((BF16, 333, 1001, 1503, SILU, 0), (0, 1, 1)), ((BF16, 333, 1001, 1503, SILU, 0), (1, 1, 0)), ((BF16, 333, 1001, 1503, SILU, 0), (1, 0, 1)),
                  ((BF16, 300, 768, 1024, SILU, 0), (0, 1, 1)), ((BF16, 300, 768, 1024, RELU, 0), (1, 0, 0))]

# Rows and classes of logits: a wave a row, a workgroup, several; held in registers by groups of several sizes, read twice.
ROWS = [(5, 40), (70, 4000), (66, 8001), (600, 9001), (65, 16001), (70, 32000), (66, 65003), (65, 131000), (65, 140001), (2, 65536), (3, 140001)]
