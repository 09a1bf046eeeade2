"""Operators of a network's dense end, as a program calls them through `darknet_zig_amd.gpu`.

  dropout  dropout whose draws come from a counter (seed and element index), so no mask is kept: forward, and
           backward on the gradient; with the residual that is added after it; between the element types
  linear   a connected layer with its bias, activation, dropout and residual in the product's epilogue
  back     its backward pass: bias, weight and input gradients, the draws made again
  loss     softmax cross-entropy of a linear layer over many classes, without keeping the logits
  train    the same with its gradients: loss forward, then the gradients of input, weights and biases

Tensors are fp32 or bf16; biases, losses and bias gradients are fp32. Deltas are the framework's: the negative
gradient, truth - probability.
"""

from __future__ import annotations

import math

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
ACTS = {"logistic": 0, "relu": 1, "linear": 3, "tanh": 5, "leaky": 7}  # the framework's activation codes
# Caps on a drawn case, below the largest listed ones.
MAX_BYTES = 8.0e8
MAX_FLOPS = {"f32": 4.0e11, "bf16": 2.0e12}


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # One token's row of a serving loop joins the residual stream: the smallest call, a launch.
        dict(name="dropout_row", kind="dropout", x="bf16", y="bf16", n=4096, prob=0.1, residual=True, first=0),
        # An odd-sized fp32 tensor whose element counter passes 2^32, as a long run's does.
        dict(name="dropout_ragged_f32", kind="dropout", x="f32", y="f32", n=5000011, prob=0.5, residual=False,
             first=4294967296 - 1234567),
        # A training batch's bf16 block output into the fp32 residual stream: pure memory traffic.
        dict(name="dropout_large", kind="dropout", x="bf16", y="f32", n=67108864, prob=0.1, residual=True, first=0),
        # One token through a wide layer: every weight is read for one row.
        dict(name="linear_token", kind="linear", type="bf16", rows=1, inputs=4096, outputs=16384, act="relu", prob=0.0,
             residual=False, bias=True),
        # A classifier's connected layer in fp32 with its activation and dropout, a training batch.
        dict(name="linear_f32", kind="linear", type="f32", rows=256, inputs=4096, outputs=4096, act="leaky", prob=0.5,
             residual=False, bias=True),
        # Odd sizes, none a multiple of eight: rows start at any alignment.
        dict(name="linear_ragged", kind="linear", type="bf16", rows=777, inputs=1001, outputs=2503, act="logistic",
             prob=0.0, residual=True, bias=True),
        # The widening layer of a large training batch: the largest single product.
        dict(name="linear_large", kind="linear", type="bf16", rows=8192, inputs=4096, outputs=16384, act="leaky", prob=0.1,
             residual=False, bias=True),
        # The repository's connected layer before 1000 classes, backward, small batch.
        dict(name="back_small", kind="back", type="bf16", rows=128, inputs=4096, outputs=1000, act="linear", prob=0.0,
             residual=False, bias=True),
        # Backward of a square layer with activation, dropout and a residual's gradient at a large batch.
        dict(name="back_large", kind="back", type="bf16", rows=8192, inputs=4096, outputs=4096, act="leaky", prob=0.1,
             residual=True, bias=True),
        # Scoring a few rows against a large vocabulary: the weights are read once.
        dict(name="loss_rows", kind="loss", type="bf16", rows=4, inputs=4096, classes=32768, bias=False),
        # A many-class fp32 classifier with odd sizes: loss and gradients.
        dict(name="train_f32", kind="train", type="f32", rows=333, inputs=1030, classes=9001, bias=True),
        # A training batch over a large vocabulary: the largest case.
        dict(name="train_large", kind="train", type="bf16", rows=4096, inputs=4096, classes=65536, bias=False),
    ]


def _log(rng, lo, hi):
    """An integer of [lo, hi], spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _size(rng, lo, hi):
    """A size of [lo, hi], often a multiple of 8 or 64, as layers' are."""
    n = _log(rng, lo, hi)
    m = rng.choice([1, 8, 64])
    return max(lo, n // m * m)


def _draw(rng):
    kind = rng.choice(["dropout", "linear", "back", "loss", "train"])
    if kind == "dropout":
        return dict(kind=kind, x=rng.choice(["f32", "bf16"]), y=rng.choice(["f32", "bf16"]), n=_log(rng, 1000, 60000000),
                    prob=rng.choice([0.0, 0.1, 0.3, 0.5]), residual=rng.random() < 0.5,
                    first=rng.choice([0, rng.randrange(1 << 20), 4294967296 - 500, rng.randrange(1 << 40)]))
    case = dict(kind=kind, type=rng.choice(["bf16", "bf16", "f32"]), rows=_log(rng, 1, 8192), inputs=_size(rng, 32, 8192))
    if kind in ("linear", "back"):
        case.update(outputs=_size(rng, 10, 16384), act=rng.choice(sorted(ACTS)), prob=rng.choice([0.0, 0.1, 0.5]),
                    residual=rng.random() < 0.5)
    else:
        case.update(classes=_size(rng, 200, 65536))
    case["bias"] = rng.random() < 0.7
    return case


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS[case.get("type", "bf16")]:
            return case


def _item(name):
    return 4 if name == "f32" else 2


def work(case):
    kind = case["kind"]
    if kind == "dropout":  # x and the residual in, y out
        n = case["n"]
        return {"bytes": n * (_item(case["x"]) + _item(case["y"]) * (2 if case["residual"] else 1)), "flops": 0.0}
    size, rows, k = _item(case["type"]), case["rows"], case["inputs"]
    n = case.get("outputs") or case.get("classes")
    x, w, y, product = rows * k, n * k, rows * n, 2.0 * rows * n * k
    if kind == "linear":  # input, weights, biases and residual in; output and, where the backward needs it, activation out
        total = x + w + y * (1 + (1 if case["residual"] else 0) + (1 if _keeps(case) else 0))
        return {"bytes": size * total + 4 * n * case["bias"], "flops": product}
    if kind == "back":  # input, weights, activation, delta and the residual's delta in; both gradients and the biases' out
        total = x * (2 + (1 if case["residual"] else 0)) + 2 * w + y * (1 if case["act"] == "linear" else 2)
        return {"bytes": size * total + 4 * n * case["bias"], "flops": 2 * product}
    if kind == "loss":  # input, weights, biases and targets in; loss and log-sum out
        return {"bytes": size * (x + w) + 4 * (n * case["bias"] + 3 * rows), "flops": product}
    # Logits that are not kept are computed twice: four products.
    return {"bytes": size * 2 * (x + w) + 4 * (2 * n * case["bias"] + 3 * rows), "flops": 4 * product}


def _keeps(case):
    """Whether a linear layer's training forward writes its activation apart from its output."""
    return case["act"] != "linear" and (case["residual"] or case["prob"] > 0)


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def _activate(act, z):
    if act == "logistic":
        return 1 / (1 + torch.exp(-z))
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "tanh":
        e = torch.exp(2 * z)
        return (e - 1) / (e + 1)
    return torch.where(z > 0, z, z * 0.1) if act == "leaky" else z


def _scale(case):
    return 1.0 / (1.0 - case["prob"])


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)

    kind, s = case["kind"], {"case": case, "seed": (seed * 2654435761 + 12345) & 0xFFFFFFFF}
    if kind == "dropout":
        s["x"] = normal(case["n"], dtype=TYPES[case["x"]])
        s["residual"] = normal(case["n"], dtype=TYPES[case["y"]]) if case["residual"] else None
        s["output"] = torch.empty(case["n"], dtype=TYPES[case["y"]], device="cuda")
        return s
    dtype, rows, k = TYPES[case["type"]], case["rows"], case["inputs"]
    n = case.get("outputs") or case.get("classes")
    s["input"] = normal(rows, k, dtype=dtype)
    # Layers start at unit gain; a trained classifier's logits are wider.
    s["weights"] = normal(n, k, std=(math.sqrt(2.0 / k) if "outputs" in case else 2.5 / math.sqrt(k)), dtype=dtype)
    s["biases"] = normal(n, std=0.1) if case["bias"] else None

    def empty(*shape, dtype=dtype):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    if kind == "linear":
        s["residual"] = normal(rows, n, dtype=dtype) if case["residual"] else None
        s["output"], s["activated"] = empty(rows, n), empty(rows, n) if _keeps(case) else None
    elif kind == "back":
        s["activated"] = _activate(case["act"], normal(rows, n)).to(dtype) if case["act"] != "linear" else None
        s["delta"] = normal(rows, n, std=0.05, dtype=dtype)
        s["input_residual"] = normal(rows, k, std=0.05, dtype=dtype) if case["residual"] else None
    else:
        # One row in sixteen has no class, as padding has none.
        t = torch.randint(0, n, (rows,), generator=g, device="cuda", dtype=torch.int32)
        s["targets"] = torch.where(torch.rand(rows, generator=g, device="cuda") < 1 / 16, torch.full_like(t, -1), t)
        s["loss"], s["lse"] = empty(rows, dtype=torch.float32), empty(rows, dtype=torch.float32)
    if kind in ("back", "train"):
        s["input_delta"], s["weight_updates"] = torch.empty_like(s["input"]), torch.empty_like(s["weights"])
        s["bias_updates"] = empty(n, dtype=torch.float32) if case["bias"] else None
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _mix(x):
    """The framework's 32-bit hash, on int64 tensors that hold unsigned 32-bit values."""
    x = ((x ^ (x >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    x = ((x ^ (x >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _dropped(seed, first, n, prob):
    """Which of n elements fall out: draw(seed, first + i) < prob, with draw = hash(seed ^ hash(low) ^ hash(high * c)) / 2^32."""
    i = torch.arange(first, first + n, device="cuda")
    h = _mix(_mix(i & 0xFFFFFFFF) ^ _mix(((i >> 32) * 0x9E3779B9) & 0xFFFFFFFF) ^ seed)
    return (h >> 8).float() * 2.0**-24 < torch.tensor(prob, dtype=torch.float32, device="cuda")


def _drop(v, seed, first, prob, scale):
    if prob == 0:
        return v * scale if scale != 1 else v
    return torch.where(_dropped(seed, first, v.numel(), prob).view_as(v), torch.zeros_like(v), v * scale)


def _gradient(act, y):
    if act == "logistic":
        return (1 - y) * y
    if act == "tanh":
        return 1 - y * y
    if act == "linear":
        return torch.ones_like(y)
    return torch.where(y > 0, torch.ones_like(y), torch.full_like(y, 0.0 if act == "relu" else 0.1))


def _logits(s):
    z = s["input"].float() @ s["weights"].float().T
    return z + s["biases"] if s["biases"] is not None else z


def _plain_loss(s):
    z, t = _logits(s), s["targets"].long()
    m = z.amax(1)
    lse = m + torch.log(torch.exp(z - m[:, None]).sum(1))
    at = z.gather(1, t.clamp(min=0)[:, None])[:, 0]
    return torch.where(t >= 0, lse - at, torch.zeros_like(lse)), lse


def _plain(s):
    case = s["case"]
    kind = case["kind"]
    if kind == "dropout":
        y = _drop(s["x"].float(), s["seed"], case["first"], case["prob"], _scale(case))
        return {"output": (y if s["residual"] is None else y + s["residual"].float()).to(s["output"].dtype)}
    dtype = TYPES[case["type"]]
    if kind == "linear":
        a = _activate(case["act"], _logits(s))
        y = _drop(a, s["seed"], 0, case["prob"], _scale(case))
        y = y if s["residual"] is None else y + s["residual"].float()
        return {"output": y.to(dtype), **({"activated": a.to(dtype)} if _keeps(case) else {})}
    if kind == "back":
        d = _drop(s["delta"].float(), s["seed"], 0, case["prob"], _scale(case))
        if s["activated"] is not None:
            d = d * _gradient(case["act"], s["activated"].float())
        x, out = s["input"].float(), {}
    else:
        loss, lse = _plain_loss(s)
        out = {"loss": loss, "lse": lse}
        if kind == "loss":
            return out
        t = s["targets"].long()
        p = torch.exp(_logits(s) - lse[:, None])
        d = -p
        d[torch.arange(case["rows"], device="cuda"), t.clamp(min=0)] += 1
        d = d * (torch.where(t >= 0, 1.0, 0.0) / case["rows"])[:, None]
        x = s["input"].float()
    dx = d @ s["weights"].float()
    if s.get("input_residual") is not None:
        dx = dx + s["input_residual"].float()
    out.update(input_delta=dx.to(dtype), weight_updates=(d.T @ x).to(dtype))
    if s["bias_updates"] is not None:
        out["bias_updates"] = d.sum(0)
    return out


# ---------------------------------------------------------------------------
# the framework's calls
# ---------------------------------------------------------------------------


def _handles(s):
    """The buffers and workspace that a program keeps for the layer, made on its first pass."""
    from darknet_zig_amd import gpu

    if not gpu.active():
        gpu.init(0)
    case = s["case"]
    b = {name: gpu.Buf(t.data_ptr(), (t.numel() * t.element_size() + 3) // 4) for name, t in s.items()
         if isinstance(t, torch.Tensor)}
    kind = case["kind"]
    code = {"f32": gpu.F32, "bf16": gpu.BF16}
    if kind == "dropout":
        return gpu, b, code
    kt, rows, k, n = code[case["type"]], case["rows"], case["inputs"], case.get("outputs") or case.get("classes")
    if kind == "linear":
        need = gpu.linearForwardWorkspace(kt, rows, k, n)
    elif kind == "back":
        need = gpu.linearBackwardWorkspace(kt, rows, k, n)
    else:
        need = gpu.linearCrossEntropyForwardWorkspace(kt, rows, k, n)[1]
        if kind == "train":
            need = max(need, gpu.linearCrossEntropyBackwardWorkspace(kt, rows, k, n)[1])
    s["workspace"] = torch.empty(max(4, (need + 3) // 4), dtype=torch.int32, device="cuda")
    b["workspace"] = gpu.Buf(s["workspace"].data_ptr(), s["workspace"].numel())
    return gpu, b, code


def _own(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    gpu, b, code = s["handles"]
    case, at = s["case"], b.get
    kind = case["kind"]
    if kind == "dropout":
        gpu.seededDropout(case["n"], code[case["x"]], b["x"], at("residual"), case["prob"], _scale(case), s["seed"],
                          case["first"], code[case["y"]], b["output"])
        return {"output": s["output"]}
    kt, rows, k = code[case["type"]], case["rows"], case["inputs"]
    if kind == "linear":
        gpu.linearForward(kt, rows, k, case["outputs"], ACTS[case["act"]], case["prob"], _scale(case), s["seed"], 0,
                          b["input"], b["weights"], at("biases"), at("residual"), at("activated"), b["output"],
                          b["workspace"])
        return {"output": s["output"], **({"activated": s["activated"]} if _keeps(case) else {})}
    out = {}
    if kind == "back":
        gpu.linearBackward(kt, rows, k, case["outputs"], ACTS[case["act"]], case["prob"], _scale(case), s["seed"], 0,
                           b["input"], b["weights"], at("activated"), b["delta"], at("input_residual"), 0.0,
                           at("bias_updates"), b["weight_updates"], b["input_delta"], b["workspace"])
    else:
        gpu.linearCrossEntropyForward(kt, rows, k, case["classes"], b["input"], b["weights"], at("biases"), b["targets"],
                                      b["loss"], b["lse"], b["workspace"])
        out = {"loss": s["loss"], "lse": s["lse"]}
        if kind == "loss":
            return out
        gpu.linearCrossEntropyBackward(kt, rows, k, case["classes"], b["input"], b["weights"], at("biases"),
                                       b["targets"], b["lse"], None, 1.0 / rows, 0.0, at("bias_updates"),
                                       b["weight_updates"], b["input_delta"], b["workspace"])
    out.update(input_delta=s["input_delta"], weight_updates=s["weight_updates"])
    if s["bias_updates"] is not None:
        out["bias_updates"] = s["bias_updates"]
    return out


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------


def _keep64(seed, first, n, prob, scale):
    """scale where an element is kept, 0 where it falls out, from the generator's definition on unsigned 32-bit words."""
    i = np.arange(n, dtype=np.uint64) + np.uint64(first)
    low, high = i.astype(np.uint32), (i >> np.uint64(32)).astype(np.uint32) * np.uint32(0x9E3779B9)

    def scramble(v):
        for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
            v = (v ^ (v >> np.uint32(shift))) * np.uint32(factor)
        return v ^ (v >> np.uint32(16))

    u = scramble(np.uint32(seed) ^ scramble(low) ^ scramble(high)) >> np.uint32(8)
    kept = u.astype(np.float64) / 16777216.0 >= float(np.float32(prob))
    return torch.from_numpy(np.where(kept, float(np.float32(scale)), 0.0)).cuda()


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "dropout":
        y = s["x"].double() * _keep64(s["seed"], case["first"], case["n"], case["prob"], _scale(case))
        return {"output": y if s["residual"] is None else y.add_(s["residual"])}
    x, w = s["input"].double(), s["weights"].double()
    rows, n = case["rows"], w.shape[0]
    keep = None
    if kind in ("linear", "back"):
        keep = _keep64(s["seed"], 0, rows * n, case["prob"], _scale(case)).view(rows, n)
    if kind != "back":
        z = torch.mm(x, w.t())
        if s["biases"] is not None:
            z += s["biases"].double()
    if kind == "linear":
        act = case["act"]
        if act == "logistic":
            z = torch.sigmoid(z)
        elif act == "tanh":
            z = torch.tanh(z)
        elif act == "relu":
            z = z.clamp(min=0)
        elif act == "leaky":
            z = torch.maximum(z, float(np.float32(0.1)) * z)
        y = keep * z
        if s["residual"] is not None:
            y += s["residual"].double()
        return {"output": y, **({"activated": z} if _keeps(case) else {})}
    out = {}
    if kind == "back":
        d = keep.mul_(s["delta"].double())
        if s["activated"] is not None:
            a = s["activated"].double()
            d = d * {"logistic": lambda: a - a * a, "tanh": lambda: 1 - a**2, "relu": lambda: (a > 0).double(),
                     "leaky": lambda: 1 - (1 - float(np.float32(0.1))) * (a <= 0).double()}[case["act"]]()
    else:
        lse = torch.logsumexp(z, 1)
        has = s["targets"] >= 0
        at = torch.nonzero(has)[:, 0]
        label = s["targets"][at].long()
        loss = torch.zeros_like(lse)
        loss[at] = lse[at] - z[at, label]
        out = {"loss": loss, "lse": lse}
        if kind == "loss":
            return out
        d = -torch.exp(z.sub_(lse[:, None]))
        d[at, label] += 1.0
        d *= has.double()[:, None] / rows
    dx = torch.mm(d, w)
    if s.get("input_residual") is not None:
        dx += s["input_residual"].double()
    out.update(input_delta=dx, weight_updates=torch.mm(d.t(), x))
    if s["bias_updates"] is not None:
        out["bias_updates"] = d.sum(0)
    return out
