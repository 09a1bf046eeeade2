"""References in 64 bits for a token model's operators, with bounds on what fp32 arithmetic may be off by."""

from __future__ import annotations

import numpy as np

from darknet_zig_amd import gpu

from .dense_ref import F32

U = 2.0**-24  # half a step of fp32
LOGISTIC, RELU, LINEAR, SILU, GELU = 0, 1, 3, gpu.SILU, gpu.GELU
GATES = (LOGISTIC, RELU, LINEAR, SILU, GELU)
C_GELU = np.sqrt(2 / np.pi)


# ---- gates ----


def sigmoid(x):
    with np.errstate(over="ignore"):
        return 1 / (1 + np.exp(-x))


def gate(act, g):
    if act == GELU:  # (1 + tanh(x)) / 2 is the logistic of 2 x, and cancels nothing
        return g * sigmoid(2 * C_GELU * (g + 0.044715 * g**3))
    return {LOGISTIC: lambda: sigmoid(g), RELU: lambda: np.where(g > 0, g, 0.0), LINEAR: lambda: g, SILU: lambda: g * sigmoid(g)}[act]()


def gate_slope(act, g):
    if act == GELU:
        u = 2 * C_GELU * (g + 0.044715 * g**3)
        return sigmoid(u) + g * sigmoid(u) * sigmoid(-u) * 2 * C_GELU * (1 + 3 * 0.044715 * g * g)
    p, rest = sigmoid(g), sigmoid(-g)
    return {LOGISTIC: lambda: p * rest, RELU: lambda: np.where(g > 0, 1.0, 0.0), LINEAR: lambda: np.ones_like(g),
            SILU: lambda: p + g * p * rest}[act]()


def inner(act, g):
    """The magnitude of the logistic's argument."""
    return np.abs(2 * C_GELU * (g + 0.044715 * g**3)) if act == GELU else np.abs(g)


STEEPEST = 1.13  # of the slopes above: gelu's


def gate_error(act, g):
    """Of evaluating a gate in fp32 at g. The logistic's argument has at most five roundings and its exponential's argument
    two more, so that exp is off by 7 |u| U and its own two U, 1 / (1 + exp) by that and three, the product by one. (fp32
    values below 2^-126 may be lost.)"""
    if act in (RELU, LINEAR):
        return 0.0
    return (8 * inner(act, g) + 8) * U * np.abs(gate(act, g)) + 2.0**-126 * (1 + np.abs(g))


def slope_error(act, g):
    """The same of the slope, p + g * (p (1 - p)) * u': p and 1 - p are off as above, u' by four roundings."""
    if act in (RELU, LINEAR):
        return 0.0
    u = 2 * C_GELU * (g + 0.044715 * g**3) if act == GELU else g
    p, rest = sigmoid(u), sigmoid(-u)
    du = 2 * C_GELU * (1 + 3 * 0.044715 * g * g) if act == GELU else 1.0
    return (16 * inner(act, g) + 24) * U * (p + np.abs(g) * p * rest * du) + 2.0**-126 * (1 + np.abs(g) * du)


# ---- softmax of rows ----


class Softmax:
    """Rows of logits [rows, classes]: y = (z - m) / T, probabilities, and error bounds of their fp32 evaluation.

    exp: y has at most five roundings (the difference, 1 / T, log2(e) / T and two products), so exp is off by 5 |y| U, and by
    two U of its own. A sum of positive terms is off by U for every addition in the longest chain: a thread's 32 of a tile, and
    merges, where exp(shift) is as above (|shift| exp(-|shift|) is below 0.37), with a multiplication and an addition: six U.
    Merges: one a tile of 4096 elements at least, 6 in a wave, 16 waves, and 3 + 16 + 64 of parts."""

    def __init__(self, z, temperature):
        z = np.asarray(z, np.float64)
        self.t = float(np.float32(temperature))
        rows, n = z.shape
        with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
            self.m = z.max(1, initial=-np.inf)
            base = np.where(np.isneginf(self.m), 0.0, self.m)
            self.y = (z - base[:, None]) / self.t
            e = np.exp(self.y)
            s = e.sum(1)
            self.l = np.log(s)
            p = e / np.where(s == 0, 1.0, s)[:, None]
            yy = np.where(p > 0, self.y, 0.0)
            py = p * np.abs(yy)
            self.p, self.lp = p, self.y - self.l[:, None]
            self.moment = py.sum(1)
            self.h = np.where(s == 0, 0.0, self.l + self.moment)
            merges = n // 4096 + 110
            s_err = U * (5 * py.sum(1) + 34 + 6 * merges)
            self.l_err = s_err + 4 * U * np.abs(self.l)  # logf: within two steps
            t_err = U * ((5 * np.abs(yy) + 12) * py).sum(1) + U * (34 + 8 * merges) * self.moment
            self.h_err = self.l_err + t_err + (s_err + 4 * U) * self.moment + U * np.abs(self.h)

    def log_prob(self, rows, classes):
        """Values and bounds at (rows, classes)."""
        y, l = self.y[rows, classes], self.l[rows]
        with np.errstate(invalid="ignore"):
            v = np.where(np.isneginf(l), -np.inf, y - l)
            return v, 3 * U * np.abs(y) + self.l_err[rows] + U * np.abs(v)


def probability_error(y, l):
    """Relative, of exp(y - l) from a given l: y as above, l's product with log2(e) and the difference a rounding each."""
    return U * (5 * np.abs(y) + 2 * np.abs(l)[:, None] + np.abs(y - l[:, None]) + 4)


def best(z, top):
    """The classes of the `top` largest of a row, equal ones by class, -1 past the last that is not masked."""
    order = np.lexsort((np.arange(z.size), -z))
    order = order[~np.isneginf(z[order])][:top]
    return np.concatenate([order, np.full(top - order.size, -1)]).astype(np.int64)


def rounding(kind):
    return U if kind == F32 else 2.0**-8
