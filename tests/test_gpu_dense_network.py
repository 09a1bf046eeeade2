"""The dense operators together, as a network's end runs them: two connected layers with activation, dropout and a
residual, a classifier's loss over them, and the way back; eagerly, on two streams at once and in captured graphs."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from darknet_zig_amd import _lib, gpu

from . import dense_ref as ref
from .dense_ref import BF16, F32, LEAKY, TANH, Pool
from .test_gpu_streams_graphs import Hip

pytestmark = pytest.mark.gpu

PROB, SCALE = 0.2, 1.25


class Net:
    """input -> tanh layer with dropout -> leaky layer onto a residual (the input) -> loss over `classes`."""

    def __init__(self, pool, kind, rows, width, hidden, classes, seed):
        r = np.random.default_rng(seed)
        self.kind, self.rows, self.width, self.hidden, self.classes, self.seed = kind, rows, width, hidden, classes, seed
        h = {
            "x": r.normal(size=(rows, width)), "w1": r.normal(size=(hidden, width)) / np.sqrt(width),
            "w2": r.normal(size=(width, hidden)) / np.sqrt(hidden), "w3": r.normal(size=(classes, width)) * 2 / np.sqrt(width),
        }
        self.h = {k: ref.rounded(v, kind) for k, v in h.items()}
        self.h |= {k: (r.normal(size=n) * 0.1).astype(np.float32) for k, n in (("b1", hidden), ("b2", width), ("b3", classes))}
        self.h["t"] = r.integers(0, classes, rows).astype(np.int32)
        self.h["t"][::7] = -1
        self.d = {k: pool(v, kind if k[0] in "xw" else None) for k, v in self.h.items()}
        for k, shape in (("a1", (rows, hidden)), ("y1", (rows, hidden)), ("a2", (rows, width)), ("y2", (rows, width)), ("dy2", (rows, width)),
                         ("dy1", (rows, hidden)), ("dx", (rows, width)), ("dw1", (hidden, width)), ("dw2", (width, hidden)),
                         ("dw3", (classes, width))):
            self.d[k] = pool(kind=kind, n=shape)
        for k, n in (("db1", hidden), ("db2", width), ("db3", classes), ("loss", rows), ("lse", rows)):
            self.d[k] = pool(n=n)
        need = max(gpu.linearForwardWorkspace(kind, rows, width, hidden), gpu.linearForwardWorkspace(kind, rows, hidden, width),
                   gpu.linearBackwardWorkspace(kind, rows, width, hidden), gpu.linearBackwardWorkspace(kind, rows, hidden, width),
                   gpu.linearCrossEntropyForwardWorkspace(kind, rows, width, classes)[1],
                   gpu.linearCrossEntropyBackwardWorkspace(kind, rows, width, classes)[0])
        self.d["ws"] = pool(n=(need + 3) // 4)

    def step(self):
        k, m, w, h, c, s = self.kind, self.rows, self.width, self.hidden, self.classes, self.seed
        b = {n: v.buf for n, v in self.d.items()}
        gpu.linearForward(k, m, w, h, TANH, PROB, SCALE, s, 0, b["x"], b["w1"], b["b1"], None, b["a1"], b["y1"], b["ws"])
        gpu.linearForward(k, m, h, w, LEAKY, 0.0, 1.0, 0, 0, b["y1"], b["w2"], b["b2"], b["x"], b["a2"], b["y2"], b["ws"])
        gpu.linearCrossEntropyForward(k, m, w, c, b["y2"], b["w3"], b["b3"], b["t"], b["loss"], b["lse"], b["ws"])
        gpu.linearCrossEntropyBackward(k, m, w, c, b["y2"], b["w3"], b["b3"], b["t"], b["lse"], None, 1.0 / m, 0.0, b["db3"], b["dw3"],
                                       b["dy2"], b["ws"])
        gpu.linearBackward(k, m, h, w, LEAKY, 0.0, 1.0, 0, 0, b["y1"], b["w2"], b["a2"], b["dy2"], None, 0.0, b["db2"], b["dw2"], b["dy1"],
                           b["ws"])
        gpu.linearBackward(k, m, w, h, TANH, PROB, SCALE, s, 0, b["x"], b["w1"], b["a1"], b["dy1"], b["dy2"], 0.0, b["db1"], b["dw1"],
                           b["dx"], b["ws"])

    OUT = ("loss", "lse", "y2", "dx", "dw1", "dw2", "dw3", "db1", "db2", "db3")

    def results(self):
        return {k: self.d[k].raw().copy() for k in self.OUT}

    def wipe(self):
        for k in self.OUT + ("a1", "y1", "a2", "dy1", "dy2"):
            gpu.push(self.d[k].base, self.d[k].host.view(np.int32))

    def loss64(self, p):
        drop = ref.dropped(self.rows * self.hidden, PROB, self.seed, 0).reshape(self.rows, self.hidden)
        y1 = np.where(drop, 0, np.tanh(p["x"] @ p["w1"].T + p["b1"]) * SCALE)
        y2 = ref.activate(LEAKY, y1 @ p["w2"].T + p["b2"]) + p["x"]
        z = y2 @ p["w3"].T + p["b3"]
        m = z.max(1)
        lse = m + np.log(np.exp(z - m[:, None]).sum(1))
        t = self.h["t"]
        return np.where(t >= 0, lse - z[np.arange(len(t)), np.maximum(t, 0)], 0).sum() / self.rows


def same(a, b):
    return {k: (a[k].view(np.uint8) == b[k].view(np.uint8)).all() for k in a}


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


@pytest.fixture
def quiet(dev):
    """No waiting after launches (not allowed in a capture); the null stream again afterwards."""
    gpu.setSyncAfterLaunch(False)
    yield Hip()
    _lib.load().dkz_set_stream(None)
    gpu.setSyncAfterLaunch(True)


@pytest.mark.parametrize("shape", [(50, 24, 40, 90), (33, 21, 35, 301), (200, 64, 136, 520)], ids=str)
def test_whole_step_is_the_loss_s_derivative(pool, shape):
    """fp32: the derivative of the mean loss along random directions of every parameter, by central differences in 64 bits.
    The gradients' roundings are below 1e-5 of sum |gradient * direction| (sums of at most 520 products of 2^-24 each, through three
    layers); the leaky layer's kinks, where a difference of step 1e-6 may cross one, move it by less than 1e-4 of that."""
    net = Net(pool, F32, *shape, seed=11)
    net.step()
    p = {k: v.astype(np.float64) for k, v in net.h.items() if k != "t"}
    got = net.results()
    assert abs(got["loss"].astype(np.float64).sum() / shape[0] - net.loss64(p)) < 1e-5 * (1 + net.loss64(p))
    r = np.random.default_rng(5)
    for name, grad in (("x", "dx"), ("w1", "dw1"), ("w2", "dw2"), ("w3", "dw3"), ("b1", "db1"), ("b2", "db2"), ("b3", "db3")):
        g = net.d[grad].get().astype(np.float64)
        for _ in range(3):
            v = r.normal(size=g.shape)
            h = 1e-6
            num = (net.loss64(p | {name: p[name] + h * v}) - net.loss64(p | {name: p[name] - h * v})) / (2 * h)
            # deltas are the negative gradient
            assert abs(num + (g * v).sum()) < 1e-4 * np.abs(g * v).sum() + 1e-8, (name, num, -(g * v).sum())


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", [(40, 64, 72, 600), (257, 200, 129, 1001), (5, 40, 33, 300)], ids=str)
def test_captured_step_replays_the_eager_one(pool, quiet, kind, shape):
    net = Net(pool, kind, *shape, seed=3)
    net.step()
    gpu.sync()
    want = net.results()
    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert quiet.hipStreamCreate(C.byref(stream)) == 0
    _lib.load().dkz_set_stream(stream)
    assert quiet.hipStreamBeginCapture(stream, 2) == 0  # relaxed
    net.step()
    assert quiet.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert quiet.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    for replay in range(3):
        net.wipe()
        gpu.sync()
        assert quiet.hipGraphLaunch(exe, stream) == 0
        assert quiet.hipStreamSynchronize(stream) == 0
        got = same(net.results(), want)
        assert all(got.values()), (replay, got)
        net.step()  # eager work of the same buffers between the replays
        gpu.sync()
        assert all(same(net.results(), want).values()), replay
    _lib.load().dkz_set_stream(None)
    assert quiet.hipGraphExecDestroy(exe) == 0 and quiet.hipGraphDestroy(graph) == 0 and quiet.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("kind", [F32, BF16])
def test_two_streams_with_their_own_workspaces(pool, quiet, kind):
    nets = [Net(pool, kind, 300, 160, 264, 900, seed=s) for s in (1, 2)]
    want = []
    for net in nets:
        net.step()
        gpu.sync()
        want.append(net.results())
        net.wipe()
    gpu.sync()
    streams = [C.c_void_p(), C.c_void_p()]
    for s in streams:
        assert quiet.hipStreamCreate(C.byref(s)) == 0
    for _ in range(5):
        for net, s in zip(nets, streams):
            _lib.load().dkz_set_stream(s)
            net.step()
    for s in streams:
        assert quiet.hipStreamSynchronize(s) == 0
    _lib.load().dkz_set_stream(None)
    for net, w in zip(nets, want):
        assert all(same(net.results(), w).values())
    for s in streams:
        assert quiet.hipStreamDestroy(s) == 0


@pytest.mark.parametrize("kind", [F32, BF16])
def test_two_graphs_replayed_at_once(pool, quiet, kind):
    nets = [Net(pool, kind, 300, 160, 264, 900, seed=s) for s in (4, 5)]
    runs, want = [], []
    for net in nets:
        net.step()
        gpu.sync()
        want.append(net.results())
        net.wipe()
        stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
        assert quiet.hipStreamCreate(C.byref(stream)) == 0
        _lib.load().dkz_set_stream(stream)
        assert quiet.hipStreamBeginCapture(stream, 2) == 0
        net.step()
        assert quiet.hipStreamEndCapture(stream, C.byref(graph)) == 0
        assert quiet.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
        runs.append((stream, graph, exe))
        _lib.load().dkz_set_stream(None)
    gpu.sync()
    for _ in range(4):
        for stream, _, exe in runs:
            assert quiet.hipGraphLaunch(exe, stream) == 0
    for stream, graph, exe in runs:
        assert quiet.hipStreamSynchronize(stream) == 0
    for net, w in zip(nets, want):
        assert all(same(net.results(), w).values())
    for stream, graph, exe in runs:
        assert quiet.hipGraphExecDestroy(exe) == 0 and quiet.hipGraphDestroy(graph) == 0 and quiet.hipStreamDestroy(stream) == 0
