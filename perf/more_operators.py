"""Operators of a token model beside the dense end: the gated feed-forward block before its last layers and what
follows its logits, as a program calls them through `darknet_zig_amd.gpu`.

  gated      a gated block's two projections, the gate's activation and the product of the two
  back       its backward pass: bias, weight and input gradients from the projections that the forward kept
  logp       log probabilities of given tokens from logits, the entropy and the top alternatives
  logp_back  the gradient of the logits from the deltas of those log probabilities and of the entropy
  distill    the divergence from a teacher's top logits, with the gradient of the logits

Tensors are fp32 or bf16; biases, log probabilities, entropies, losses, teachers' logits and bias gradients are fp32.
Deltas are the framework's: the negative gradient.
"""

from __future__ import annotations

import math

import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
GATES = {"logistic": 0, "relu": 1, "linear": 3, "silu": 14, "gelu": 15}  # the activation codes
# Caps on a drawn case, below the largest listed ones.
MAX_BYTES = 8.0e8
MAX_FLOPS = {"f32": 2.0e11, "bf16": 1.0e12}
GELU = 2.0 * math.sqrt(2.0 / math.pi)


# ---------------------------------------------------------------------------
# the cases
# ---------------------------------------------------------------------------


def listed():
    return [
        # One token through a block while serving: every weight is read for one row.
        dict(name="gated_token", kind="gated", type="bf16", rows=1, inputs=4096, hidden=8192, gate="silu", bias=False, keep=False),
        # An fp32 block with odd sizes in training: rows start at any alignment.
        dict(name="gated_ragged_f32", kind="gated", type="f32", rows=333, inputs=1001, hidden=1503, gate="gelu", bias=True, keep=True),
        # The block of a large training batch, its projections kept for the backward pass.
        dict(name="gated_large", kind="gated", type="bf16", rows=8192, inputs=4096, hidden=8192, gate="silu", bias=False, keep=True),
        # Backward of a small block with odd sizes.
        dict(name="back_ragged", kind="back", type="bf16", rows=333, inputs=1001, hidden=1503, gate="gelu", bias=True, residual=False),
        # Backward of a training batch, joined to the residual stream's delta: the largest case.
        dict(name="back_large", kind="back", type="bf16", rows=4096, inputs=4096, hidden=8192, gate="silu", bias=False, residual=True),
        # One step of a decoding loop: the token's log probability and twenty alternatives.
        dict(name="logp_token", kind="logp", type="f32", rows=1, classes=65536, pitch=65536, temperature=0.7, given=1, top=20,
             entropy=True, masked=False),
        # A serving batch with a vocabulary of odd size in padded rows, a few candidates scored for each.
        dict(name="logp_rows", kind="logp", type="bf16", rows=48, classes=50001, pitch=50048, temperature=1.0, given=4, top=5,
             entropy=True, masked=True),
        # The tokens of a training batch with their entropies: logits read once.
        dict(name="logp_large", kind="logp", type="bf16", rows=4096, classes=65536, pitch=65536, temperature=1.0, given=1, top=0,
             entropy=True, masked=False),
        # The way back of a policy's log probabilities and entropies.
        dict(name="logp_back", kind="logp_back", type="f32", rows=1024, classes=50001, pitch=50048, temperature=1.0, given=1,
             entropy=True, masked=True),
        # A small classifier taught by a larger one.
        dict(name="distill_small", kind="distill", type="f32", rows=16, classes=1000, pitch=1000, temperature=2.0, top=16),
        # Rows of odd length without gaps, so that each starts at another alignment.
        dict(name="distill_ragged", kind="distill", type="bf16", rows=500, classes=9001, pitch=9001, temperature=1.5, top=50),
        # A training batch over a large vocabulary.
        dict(name="distill_large", kind="distill", type="bf16", rows=4096, classes=65536, pitch=65536, temperature=1.0, top=64),
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
    kind = rng.choice(["gated", "back", "logp", "logp_back", "distill"])
    case = dict(kind=kind, type=rng.choice(["bf16", "bf16", "f32"]), rows=_log(rng, 1, 8192))
    if kind in ("gated", "back"):
        case.update(inputs=_size(rng, 32, 8192), hidden=_size(rng, 32, 16384), gate=rng.choice(sorted(GATES)), bias=rng.random() < 0.4)
        case["keep" if kind == "gated" else "residual"] = rng.random() < 0.5
        return case
    classes = _size(rng, 300, 131072)
    case.update(classes=classes, pitch=classes if rng.random() < 0.6 else (classes + 63) // 64 * 64, temperature=rng.choice([1.0, 1.0, 0.7, 2.0]))
    if kind == "distill":
        case["top"] = _log(rng, 1, 128)
        return case
    case.update(given=rng.choice([1, 1, 1, 3, 16]), entropy=rng.random() < 0.7, masked=rng.random() < 0.3)
    if kind == "logp":
        case["top"] = rng.choice([0, 1, 5, 20, 64])
    return case


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= MAX_BYTES and w["flops"] <= MAX_FLOPS[case["type"]]:
            return case


def work(case):
    kind, size, rows = case["kind"], 4 if case["type"] == "f32" else 2, case["rows"]
    if kind in ("gated", "back"):
        k, n = case["inputs"], case["hidden"]
        x, w, s, y, product = rows * k, 2 * n * k, 2 * rows * n, rows * n, 4.0 * rows * n * k
        if kind == "gated":  # input, weights and biases in; output and, for training, both projections out
            return {"bytes": size * (x + w + y + (s if case["keep"] else 0)) + 8 * n * case["bias"], "flops": product}
        # input, weights, projections, delta and the residual's delta in; the gradients out
        return {"bytes": size * (2 * x + 2 * w + s + y + (x if case["residual"] else 0)) + 8 * n * case["bias"], "flops": 2 * product}
    z = size * rows * case["classes"]
    if kind == "logp":  # logits in; two numbers a token and an alternative, and three a row
        return {"bytes": z + rows * (8 * case["given"] + 8 * case["top"] + 12), "flops": 0.0}
    if kind == "logp_back":  # logits in, their delta out
        return {"bytes": z * 2 + rows * (8 * case["given"] + 16), "flops": 0.0}
    return {"bytes": 2 * z + rows * (8 * case["top"] + 8), "flops": 0.0}  # logits in, their delta out


# ---------------------------------------------------------------------------
# inputs
# ---------------------------------------------------------------------------


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return torch.randn(*shape, generator=g, device="cuda").mul_(std).to(dtype)

    def uniform(*shape):
        return torch.rand(*shape, generator=g, device="cuda")

    def integers(hi, *shape):
        return torch.randint(0, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    def empty(*shape, dtype=torch.float32):
        return torch.empty(*shape, dtype=dtype, device="cuda")

    kind, dtype, rows, s = case["kind"], TYPES[case["type"]], case["rows"], {"case": case}
    if kind in ("gated", "back"):
        k, n = case["inputs"], case["hidden"]
        s["input"] = normal(rows, k, dtype=dtype)
        s["weights"] = normal(2 * n, k, std=1.0 / math.sqrt(k), dtype=dtype)
        if kind == "gated":
            s["biases"] = normal(2 * n, std=0.1) if case["bias"] else None
            s["sums"], s["output"] = empty(rows, 2 * n, dtype=dtype) if case["keep"] else None, empty(rows, n, dtype=dtype)
            return s
        s["sums"], s["delta"] = normal(rows, 2 * n, dtype=dtype), normal(rows, n, std=0.05, dtype=dtype)
        s["input_residual"] = normal(rows, k, std=0.05, dtype=dtype) if case["residual"] else None
        s["input_delta"], s["weight_updates"] = torch.empty_like(s["input"]), torch.empty_like(s["weights"])
        s["bias_updates"] = empty(2 * n) if case["bias"] else None
        return s
    classes, pitch = case["classes"], case["pitch"]
    # A trained model's logits are wide. The end of a padded row holds anything.
    s["logits"] = normal(rows, pitch, std=2.5, dtype=dtype)
    allowed = classes
    if case.get("masked"):  # classes that no token has
        allowed = classes - classes // 50
        s["logits"][:, allowed:classes] = -math.inf
    if kind == "distill":
        top = case["top"]
        # The teacher's tokens lie all over the vocabulary and are likely ones for the student too. One row in sixteen is
        # padding, without any; some rows have fewer.
        at = (integers(classes, rows, 1).long() + torch.arange(top, device="cuda") * (classes // top)) % classes
        s["teacher_logits"] = normal(rows, top, std=2.0).sort(1, descending=True).values + 6.0
        s["logits"][:, :classes] = s["logits"][:, :classes].scatter_add(1, at, (0.7 * s["teacher_logits"]).to(dtype))
        count = torch.where(uniform(rows, 1) < 1 / 16, 0, torch.where(uniform(rows, 1) < 0.25, (top + 1) // 2, top))
        s["teacher_tokens"] = torch.where(torch.arange(top, device="cuda") < count, at, -1).to(torch.int32)
        s["loss"], s["logits_delta"] = empty(rows), torch.zeros_like(s["logits"])
        return s
    given = case["given"]
    t = integers(allowed, rows, given)
    # One in sixteen is no token, as padding is.
    s["tokens"] = torch.where(uniform(rows, given) < 1 / 16, torch.full_like(t, -1), t)
    if kind == "logp":
        s["log_probs"], s["stats"] = empty(rows, given), empty(rows, 2)
        s["entropy"] = empty(rows) if case["entropy"] else None
        s["top_tokens"] = empty(rows, case["top"], dtype=torch.int32) if case["top"] else None
        s["top_log_probs"] = empty(rows, case["top"]) if case["top"] else None
        return s
    # What the forward pass left behind, and the deltas of what it gave.
    m, total, moment = _row_sums(s["logits"][:, :classes], case["temperature"])
    s["stats"], s["entropy"] = torch.stack([m, torch.log(total)], 1), torch.log(total) - moment / total
    s["log_prob_deltas"] = normal(rows, given, std=1.0 / rows)
    s["entropy_deltas"] = torch.full((rows,), 0.01 / rows, device="cuda") if case["entropy"] else None
    s["logits_delta"] = torch.zeros_like(s["logits"])
    return s


# ---------------------------------------------------------------------------
# the plain forms
# ---------------------------------------------------------------------------


def _gate(gate, g):
    """The gate's activation and its derivative."""
    if gate == "relu":
        on = (g > 0).float()
        return g * on, on
    if gate == "linear":
        return g, torch.ones_like(g)
    u = g if gate != "gelu" else GELU * (g + 0.044715 * g * g * g)
    p = 1 / (1 + torch.exp(-u))
    if gate == "logistic":
        return p, p * (1 - p)
    slope = 1.0 if gate == "silu" else GELU * (1 + 3 * 0.044715 * g * g)
    return g * p, p + g * p * (1 - p) * slope


def _row_sums(z, temperature):
    """Of every row: the maximum, and the sums of e = exp(y) and of e * y, y being (z - maximum) / temperature."""
    z = z.float()
    m = z.amax(1)
    y = (z - m[:, None]) / temperature
    e = torch.exp(y)
    return m, e.sum(1), torch.where(e > 0, e * y, torch.zeros_like(e)).sum(1)


def _top(z, top):
    """The `top` largest of every row, equal ones by their index: keys of the value's order and the index's complement."""
    bits = (z.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits >= 0, bits, -0x80000000 - bits)
    key = order * (1 << 32) + (0xFFFFFFFF - torch.arange(z.shape[1], device=z.device))
    return 0xFFFFFFFF - (torch.topk(key, top, dim=1).values & 0xFFFFFFFF)


def _plain(s):
    case = s["case"]
    kind, dtype = case["kind"], TYPES[case["type"]]
    if kind == "gated":
        z = s["input"].float() @ s["weights"].float().T
        if s["biases"] is not None:
            z = z + s["biases"]
        n = case["hidden"]
        out = {"output": (_gate(case["gate"], z[:, :n])[0] * z[:, n:]).to(dtype)}
        return {**out, "sums": z.to(dtype)} if case["keep"] else out
    if kind == "back":
        n, z, d = case["hidden"], s["sums"].float(), s["delta"].float()
        a, slope = _gate(case["gate"], z[:, :n])
        ds = torch.cat([d * z[:, n:] * slope, d * a], 1)
        dx = ds @ s["weights"].float()
        if s["input_residual"] is not None:
            dx = dx + s["input_residual"].float()
        out = {"input_delta": dx.to(dtype), "weight_updates": (ds.T @ s["input"].float()).to(dtype)}
        return {**out, "bias_updates": ds.sum(0)} if s["bias_updates"] is not None else out
    classes, t = case["classes"], case["temperature"]
    z = s["logits"][:, :classes]
    if kind == "logp":
        m, total, moment = _row_sums(z, t)
        log_sum = torch.log(total)

        def log_prob(at):
            return (z.gather(1, at).float() - m[:, None]) / t - log_sum[:, None]

        token = s["tokens"].long()
        at = log_prob(token.clamp(min=0))
        out = {"log_probs": torch.where(token >= 0, at, torch.zeros_like(at)), "stats": torch.stack([m, log_sum], 1)}
        if case["entropy"]:
            out["entropy"] = log_sum - moment / total
        if case["top"]:
            best = _top(z, case["top"])
            out.update(top_tokens=best.int(), top_log_probs=log_prob(best))
        return out
    if kind == "logp_back":
        m, log_sum = s["stats"][:, :1], s["stats"][:, 1:]
        token = s["tokens"].long()
        a = torch.where(token >= 0, s["log_prob_deltas"], torch.zeros_like(s["log_prob_deltas"]))
        lp = (z.float() - m) / t - log_sum
        p = torch.exp(lp)
        factor = a.sum(1)[:, None]
        if case["entropy"]:
            factor = factor + s["entropy_deltas"][:, None] * torch.where(p > 0, lp + s["entropy"][:, None], torch.zeros_like(lp))
        d = ((-p * factor).scatter_add(1, token.clamp(min=0), a)) / t
        return {"logits_delta": d.to(dtype)}
    token = s["teacher_tokens"].long()
    has = token >= 0
    w = torch.where(has, s["teacher_logits"] / t, torch.full_like(s["teacher_logits"], -math.inf))
    any_ = has.any(1, keepdim=True)
    w = torch.where(any_, w - w.amax(1, keepdim=True), torch.full_like(w, -math.inf))
    e = torch.exp(w)
    norm = e.sum(1, keepdim=True).clamp(min=1e-30)
    p, log_p = e / norm, w - torch.log(norm)
    m, total, _ = _row_sums(z, t)
    log_q = (z.gather(1, token.clamp(min=0)).float() - m[:, None]) / t - torch.log(total)[:, None]
    loss = t * t * torch.where(has, p * (log_p - log_q), torch.zeros_like(p)).sum(1)
    q = torch.exp((z.float() - m[:, None]) / t) / total[:, None]
    d = (-q).scatter_add(1, token.clamp(min=0), p) * (t / case["rows"])
    return {"loss": loss, "logits_delta": torch.where(any_, d, torch.zeros_like(d)).to(dtype)}


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
    kind, kt, rows, need = case["kind"], {"f32": gpu.F32, "bf16": gpu.BF16}[case["type"]], case["rows"], 0
    if kind == "gated":
        need = gpu.gatedForwardWorkspace(kt, rows, case["inputs"], case["hidden"])
    elif kind == "back":
        need = gpu.gatedBackwardWorkspace(kt, rows, case["inputs"], case["hidden"])
    elif kind == "logp":
        need = gpu.tokenLogProbsWorkspace(kt, rows, case["classes"], case["top"])
    elif kind == "distill":
        need = gpu.distillationWorkspace(kt, rows, case["classes"])
    s["workspace"] = torch.empty(max(4, (need + 3) // 4), dtype=torch.int32, device="cuda")
    b["workspace"] = gpu.Buf(s["workspace"].data_ptr(), s["workspace"].numel())
    return gpu, b, kt


def _own(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    gpu, b, kt = s["handles"]
    case, at = s["case"], b.get
    kind, rows = case["kind"], case["rows"]
    if kind == "gated":
        gpu.gatedForward(kt, rows, case["inputs"], case["hidden"], GATES[case["gate"]], b["input"], b["weights"], at("biases"),
                         at("sums"), b["output"], b["workspace"])
        return {"output": s["output"], **({"sums": s["sums"]} if case["keep"] else {})}
    if kind == "back":
        gpu.gatedBackward(kt, rows, case["inputs"], case["hidden"], GATES[case["gate"]], b["input"], b["weights"], b["sums"],
                          b["delta"], at("input_residual"), 0.0, at("bias_updates"), b["weight_updates"], b["input_delta"],
                          b["workspace"])
        out = {"input_delta": s["input_delta"], "weight_updates": s["weight_updates"]}
        return {**out, "bias_updates": s["bias_updates"]} if case["bias"] else out
    classes, pitch, t = case["classes"], case["pitch"], case["temperature"]
    if kind == "logp":
        gpu.tokenLogProbs(kt, rows, classes, pitch, b["logits"], t, case["given"], b["tokens"], case["top"], b["log_probs"],
                          at("entropy"), b["stats"], at("top_tokens"), at("top_log_probs"), b["workspace"])
        return {name: s[name] for name in ("log_probs", "stats", "entropy", "top_tokens", "top_log_probs") if s[name] is not None}
    if kind == "logp_back":
        gpu.tokenLogProbsBackward(kt, rows, classes, pitch, b["logits"], t, case["given"], b["tokens"], b["stats"], b["entropy"],
                                  b["log_prob_deltas"], at("entropy_deltas"), 0.0, b["logits_delta"])
        return {"logits_delta": s["logits_delta"][:, :classes]}
    gpu.distillation(kt, rows, classes, pitch, b["logits"], t, case["top"], b["teacher_tokens"], b["teacher_logits"], None,
                     1.0 / rows, b["loss"], b["logits_delta"], b["workspace"])
    return {"loss": s["loss"], "logits_delta": s["logits_delta"][:, :classes]}


def run(state):
    return _own(state) if own else _plain(state)


# ---------------------------------------------------------------------------
# the definition, in 64 bits
# ---------------------------------------------------------------------------


def _activation64(gate, g):
    return {"logistic": lambda: torch.sigmoid(g), "relu": lambda: g.clamp(min=0), "linear": lambda: g, "silu": lambda: g * torch.sigmoid(g),
            "gelu": lambda: 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)))}[gate]()


def _slope64(gate, g):
    if gate == "relu":
        return (g > 0).double()
    if gate == "linear":
        return torch.ones_like(g)
    if gate == "gelu":
        c = math.sqrt(2 / math.pi)
        th = torch.tanh(c * (g + 0.044715 * g**3))
        return 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * c * (1 + 0.134145 * g * g)
    p = torch.sigmoid(g)
    return p * torch.sigmoid(-g) * (1.0 if gate == "logistic" else g) + (0.0 if gate == "logistic" else p)


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind in ("gated", "back"):
        n, x, w = case["hidden"], s["input"].double(), s["weights"].double()
        if kind == "gated":
            z = torch.mm(x, w.t())
            if s["biases"] is not None:
                z += s["biases"].double()
            out = {"output": _activation64(case["gate"], z[:, :n]) * z[:, n:]}
            return {**out, "sums": z} if case["keep"] else out
        gate, up, d = s["sums"][:, :n].double(), s["sums"][:, n:].double(), s["delta"].double()
        ds = torch.empty(case["rows"], 2 * n, dtype=torch.float64, device="cuda")
        ds[:, :n] = _slope64(case["gate"], gate) * up * d
        ds[:, n:] = _activation64(case["gate"], gate) * d
        dx = torch.mm(ds, w)
        if s["input_residual"] is not None:
            dx += s["input_residual"].double()
        out = {"input_delta": dx, "weight_updates": torch.mm(ds.t(), x)}
        return {**out, "bias_updates": ds.sum(0)} if s["bias_updates"] is not None else out
    classes, rows = case["classes"], case["rows"]
    t = float(torch.tensor(case["temperature"], dtype=torch.float32))
    z = s["logits"][:, :classes].double() / t
    lse = torch.logsumexp(z, 1)
    if kind == "logp":
        lp = z - lse[:, None]
        token = s["tokens"].long()
        at = torch.nonzero(token >= 0, as_tuple=True)
        log_probs = torch.zeros(token.shape, dtype=torch.float64, device="cuda")
        log_probs[at] = lp[at[0], token[at]]
        m = s["logits"][:, :classes].amax(1).double()
        out = {"log_probs": log_probs, "stats": torch.stack([m, lse - m / t], 1)}
        if case["entropy"]:
            out["entropy"] = -(torch.exp(lp) * lp.clamp(min=-1e6)).sum(1)
        if case["top"]:
            order = torch.sort(lp, dim=1, descending=True, stable=True)
            out["top_tokens"] = order.indices[:, : case["top"]].int()
            out["top_log_probs"] = order.values[:, : case["top"]]
        return out
    if kind == "logp_back":
        lp = z - lse[:, None]
        p = torch.exp(lp)
        token = s["tokens"].long()
        a = s["log_prob_deltas"].double() * (token >= 0)
        d = -p * a.sum(1)[:, None]
        if case["entropy"]:
            lp = lp.clamp(min=-1e6)
            h = -(p * lp).sum(1)
            d -= s["entropy_deltas"].double()[:, None] * p * (lp + h[:, None])
        d.scatter_add_(1, token.clamp(min=0), a)
        d /= t
        return {"logits_delta": d}
    token = s["teacher_tokens"].long()
    has = token >= 0
    w = torch.where(has, s["teacher_logits"].double() / t, torch.full((), -math.inf, dtype=torch.float64, device="cuda"))
    any_ = has.any(1)
    log_p = torch.nan_to_num(w - torch.logsumexp(w, 1, keepdim=True), nan=-math.inf)
    p = torch.exp(log_p)
    q_at = z.gather(1, token.clamp(min=0)) - lse[:, None]
    loss = t * t * torch.where(has, p * (log_p.clamp(min=-1e6) - q_at), torch.zeros_like(p)).sum(1)
    d = torch.exp(z.sub_(lse[:, None])).neg_()
    d.scatter_add_(1, token.clamp(min=0), p)
    d *= any_.double()[:, None] * (t / rows)
    return {"loss": loss, "logits_delta": d}
