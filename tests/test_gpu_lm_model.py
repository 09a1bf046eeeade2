"""A token model's operators together with the dense ones, as a training step runs them: a gated block with its last layer onto
the residual, logits, a teacher's divergence and the tokens' log probabilities with an entropy bonus, and the way back; eagerly,
on two streams at once and in captured graphs. And a decoding step for single tokens."""

from __future__ import annotations

import ctypes as C

import numpy as np
import pytest

from darknet_zig_amd import _lib, gpu

from . import dense_ref as ref
from . import lm_ref as lm
from .dense_ref import BF16, F32, LINEAR, Pool
from .test_gpu_dense_network import quiet, same  # noqa: F401
from .test_gpu_lm_distillation import evaluate

pytestmark = pytest.mark.gpu

T = 1.5
TOP = 6


@pytest.fixture
def pool(dev):
    p = Pool()
    yield p
    p.free()


class Model:
    """x -> gated(hidden) -> linear + x -> logits; loss = sum distill / rows - sum a log p - sum e H, over tokens and rows."""

    def __init__(self, pool, kind, rows, width, hidden, classes, seed, act=lm.SILU):
        r = np.random.default_rng(seed)
        self.kind, self.rows, self.width, self.hidden, self.classes, self.act = kind, rows, width, hidden, classes, act
        h = {"x": r.normal(size=(rows, width)), "wg": r.normal(size=(2 * hidden, width)) / np.sqrt(width),
             "wd": r.normal(size=(width, hidden)) / np.sqrt(hidden), "wl": r.normal(size=(classes, width)) * 2 / np.sqrt(width)}
        self.h = {k: ref.rounded(v, kind) for k, v in h.items()}
        self.h |= {k: (r.normal(size=n) * 0.1).astype(np.float32) for k, n in (("bg", 2 * hidden), ("bd", width), ("bl", classes))}
        self.h["tokens"] = r.integers(-1, classes, (rows, 2)).astype(np.int32)
        self.h["teacher"] = r.integers(-1, classes, (rows, TOP)).astype(np.int32)
        self.h["tlogits"] = (r.normal(size=(rows, TOP)) * 2).astype(np.float32)
        self.h["a"], self.h["e"] = (r.normal(size=(rows, 2)) / rows).astype(np.float32), np.full(rows, 0.05 / rows, np.float32)
        self.d = {k: pool(v, kind if k in h else None) for k, v in self.h.items()}
        for k, shape in (("s", (rows, 2 * hidden)), ("y", (rows, hidden)), ("o", (rows, width)), ("z", (rows, classes)), ("dz", (rows, classes)),
                         ("do", (rows, width)), ("dy", (rows, hidden)), ("dx", (rows, width)), ("dwg", (2 * hidden, width)),
                         ("dwd", (width, hidden)), ("dwl", (classes, width))):
            self.d[k] = pool(kind=kind, n=shape)
        for k, shape in (("dbg", 2 * hidden), ("dbd", width), ("dbl", classes), ("loss", rows), ("lp", (rows, 2)), ("ent", rows), ("stats", (rows, 2)),
                         ("tl", (rows, 4))):
            self.d[k] = pool(n=shape)
        self.d["tt"] = pool(np.zeros((rows, 4), np.int32))
        need = max(gpu.gatedForwardWorkspace(kind, rows, width, hidden), gpu.gatedBackwardWorkspace(kind, rows, width, hidden),
                   gpu.linearForwardWorkspace(kind, rows, hidden, width), gpu.linearBackwardWorkspace(kind, rows, hidden, width),
                   gpu.linearForwardWorkspace(kind, rows, width, classes), gpu.linearBackwardWorkspace(kind, rows, width, classes),
                   gpu.tokenLogProbsWorkspace(kind, rows, classes, 4), gpu.distillationWorkspace(kind, rows, classes))
        self.d["ws"] = pool(n=(need + 3) // 4)

    def forward(self):
        k, m, w, h, c = self.kind, self.rows, self.width, self.hidden, self.classes
        b = {n: v.buf for n, v in self.d.items()}
        gpu.gatedForward(k, m, w, h, self.act, b["x"], b["wg"], b["bg"], b["s"], b["y"], b["ws"])
        gpu.linearForward(k, m, h, w, LINEAR, 0.0, 1.0, 0, 0, b["y"], b["wd"], b["bd"], b["x"], None, b["o"], b["ws"])
        gpu.linearForward(k, m, w, c, LINEAR, 0.0, 1.0, 0, 0, b["o"], b["wl"], b["bl"], None, None, b["z"], b["ws"])
        gpu.tokenLogProbs(k, m, c, c, b["z"], T, 2, b["tokens"], 4, b["lp"], b["ent"], b["stats"], b["tt"], b["tl"], b["ws"])

    def step(self):
        self.forward()
        k, m, w, h, c = self.kind, self.rows, self.width, self.hidden, self.classes
        b = {n: v.buf for n, v in self.d.items()}
        gpu.distillation(k, m, c, c, b["z"], T, TOP, b["teacher"], b["tlogits"], None, 1.0 / m, b["loss"], b["dz"], b["ws"])
        gpu.tokenLogProbsBackward(k, m, c, c, b["z"], T, 2, b["tokens"], b["stats"], b["ent"], b["a"], b["e"], 1.0, b["dz"])
        gpu.linearBackward(k, m, w, c, LINEAR, 0.0, 1.0, 0, 0, b["o"], b["wl"], None, b["dz"], None, 0.0, b["dbl"], b["dwl"], b["do"], b["ws"])
        gpu.linearBackward(k, m, h, w, LINEAR, 0.0, 1.0, 0, 0, b["y"], b["wd"], None, b["do"], None, 0.0, b["dbd"], b["dwd"], b["dy"], b["ws"])
        gpu.gatedBackward(k, m, w, h, self.act, b["x"], b["wg"], b["s"], b["dy"], b["do"], 0.0, b["dbg"], b["dwg"], b["dx"], b["ws"])

    OUT = ("y", "o", "z", "lp", "ent", "stats", "tt", "tl", "loss", "dz", "dx", "dwg", "dwd", "dwl", "dbg", "dbd", "dbl")

    def results(self):
        return {k: self.d[k].raw().copy() for k in self.OUT}

    def wipe(self):
        for k in self.OUT + ("s", "do", "dy"):
            gpu.push(self.d[k].base, self.d[k].host.view(np.int32))

    def logits64(self, p):
        s = p["x"] @ p["wg"].T + p["bg"]
        y = lm.gate(self.act, s[:, : self.hidden]) * s[:, self.hidden :]
        return (p["x"] + y @ p["wd"].T + p["bd"]) @ p["wl"].T + p["bl"]

    def loss64(self, p):
        """What the step's deltas are the negative gradient of."""
        z = self.logits64(p)
        s = lm.Softmax(z, T)
        t = self.h["tokens"]
        lp = np.where(t >= 0, s.lp[np.arange(self.rows)[:, None], np.maximum(t, 0)], 0)
        distilled = evaluate(z, self.classes, T, self.h["teacher"], self.h["tlogits"], np.ones(self.rows, np.float32))[0]
        return distilled.sum() / self.rows - (self.h["a"] * lp).sum() - (self.h["e"] * s.h).sum()


@pytest.mark.parametrize("shape,act", [((50, 24, 40, 90), lm.SILU), ((33, 21, 35, 301), lm.GELU), ((120, 64, 136, 2500), lm.LOGISTIC)], ids=str)
def test_whole_step_is_the_loss_s_derivative(pool, shape, act):
    """fp32: the derivative along random directions of every parameter, by central differences in 64 bits. The gradients'
    roundings, of sums of at most 2500 products through three layers, are below 1e-5 of sum |gradient * direction|; a difference of
    step 1e-5 is off by 1e-10 of third derivatives that are as large as the magnitudes, and by 1e-11 of rounding: 1e-4 covers them."""
    net = Model(pool, F32, *shape, seed=11, act=act)
    net.step()
    p = {k: v.astype(np.float64) for k, v in net.h.items() if k in ("x", "wg", "wd", "wl", "bg", "bd", "bl")}
    z = net.d["z"].get()
    s = lm.Softmax(z, T)
    ref.assert_within(net.d["ent"].get(), s.h, s.h_err, "entropy")
    r = np.random.default_rng(5)
    for name, grad in (("x", "dx"), ("wg", "dwg"), ("wd", "dwd"), ("wl", "dwl"), ("bg", "dbg"), ("bd", "dbd"), ("bl", "dbl")):
        g = net.d[grad].get().astype(np.float64)
        for _ in range(3):
            v, h = r.normal(size=g.shape), 1e-5
            num = (net.loss64(p | {name: p[name] + h * v}) - net.loss64(p | {name: p[name] - h * v})) / (2 * h)
            assert abs(num + (g * v).sum()) < 1e-4 * np.abs(g * v).sum() + 1e-8, (name, num, -(g * v).sum())


def capture(hip, net, call):
    """A stream and a captured graph of call()."""
    stream, graph, exe = C.c_void_p(), C.c_void_p(), C.c_void_p()
    assert hip.hipStreamCreate(C.byref(stream)) == 0
    _lib.load().dkz_set_stream(stream)
    assert hip.hipStreamBeginCapture(stream, 2) == 0  # relaxed
    call()
    assert hip.hipStreamEndCapture(stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(exe), graph, None, None, 0) == 0
    return stream, graph, exe


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("shape", [(40, 64, 72, 600), (257, 200, 129, 3001), (1, 64, 128, 40000), (5, 40, 33, 20001)], ids=str)
def test_captured_step_replays_the_eager_one(pool, quiet, kind, shape):  # noqa: F811
    net = Model(pool, kind, *shape, seed=3)
    net.step()
    gpu.sync()
    want = net.results()
    stream, graph, exe = capture(quiet, net, net.step)
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
@pytest.mark.parametrize("shape", [(300, 160, 264, 900), (2, 160, 264, 30000)], ids=str)
def test_two_streams_and_two_graphs_at_once(pool, quiet, kind, shape):  # noqa: F811
    nets, want, runs = [Model(pool, kind, *shape, seed=s) for s in (1, 2)], [], []
    for net in nets:
        net.step()
        gpu.sync()
        want.append(net.results())
        net.wipe()
    gpu.sync()
    for net in nets:
        runs.append(capture(quiet, net, net.step))
    for _ in range(4):
        for net, (stream, _, _) in zip(nets, runs):
            _lib.load().dkz_set_stream(stream)
            net.step()
    for net, (stream, _, _), w in zip(nets, runs, want):
        assert quiet.hipStreamSynchronize(stream) == 0
        assert all(same(net.results(), w).values())
        net.wipe()
    _lib.load().dkz_set_stream(None)
    gpu.sync()
    for _ in range(4):
        for stream, _, exe in runs:
            assert quiet.hipGraphLaunch(exe, stream) == 0
    for net, (stream, graph, exe), w in zip(nets, runs, want):
        assert quiet.hipStreamSynchronize(stream) == 0
        assert all(same(net.results(), w).values())
        assert quiet.hipGraphExecDestroy(exe) == 0 and quiet.hipGraphDestroy(graph) == 0 and quiet.hipStreamDestroy(stream) == 0


@pytest.mark.parametrize("kind", [F32, BF16])
def test_a_decoding_step_is_the_batch_s_row(pool, kind):
    """Single tokens and a batch of them: the same alternatives, log probabilities as near as the logits' roundings let them be."""
    rows, width, hidden, classes = 5, 128, 320, 9001
    many = Model(pool, kind, rows, width, hidden, classes, seed=8)
    many.forward()
    for i in range(rows):
        one = Model(pool, kind, 1, width, hidden, classes, seed=8)
        for k in ("x", "wg", "wd", "wl", "bg", "bd", "bl", "tokens"):
            v = many.h[k][i : i + 1] if k in ("x", "tokens") else many.h[k]
            one.d[k] = pool(v, kind if k in ("x", "wg", "wd", "wl") else None)
        one.forward()
        za, zb = many.d["z"].get()[i].astype(np.float64), one.d["z"].get()[0].astype(np.float64)
        gap = np.abs(za - zb).max()  # a log probability moves by at most twice the logits' largest change
        tokens = many.h["tokens"][i]
        assert (np.abs(many.d["lp"].get()[i] - one.d["lp"].get()[0]) <= np.where(tokens >= 0, 2 * gap / T + 1e-4, 0)).all()
        assert (one.d["tt"].get()[0] == lm.best(one.d["z"].get()[0], 4)).all()
