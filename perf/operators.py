"""The operators of a language model's training step, as cases that can be timed and checked.

* ``loss``: softmax cross entropy of ``hidden @ weight.T`` against target tokens over a whole vocabulary, with the
  gradients of both factors (``train``) or the losses alone (evaluation).
* ``linear``: ``act(x @ weight.T + bias) + residual``, with the gradients of all its inputs (``train``) or alone
  (serving).
* ``adamw``: one AdamW step over all tensors of a model, with states in 32 bits or in 8.  Tensor ``i`` lies at a
  multiple of 256 elements of flat buffers, in the order of the list; gradients are views of such a buffer too, as
  those of a bucketed data-parallel job are.

A state of 8 bits is kept in blocks of 256 elements, each with a scale that is a power of two: ``exp_avg`` and the
square root of the second moment are ``float8_e4m3fn`` times that scale.  They are rounded to 3 bits of mantissa at
random: 16 random bits, from a hash of the element's place in the flat buffers and of a number that the step is given,
are added below the mantissa's end before it is cut off.
"""
import math
import random

import torch

own = False

_TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
_BYTES = {"fp32": 4, "bf16": 2, "fp16": 2}
_ACTS = ("none", "gelu", "gelu_tanh", "silu", "relu")
_IGNORE = -100
_BLOCK = 256
_LR, _BETAS, _EPS, _WD, _SEED = 3e-4, (0.9, 0.95), 1e-8, 0.1, 20


def listed():
    return [
        # the tiny GPT-2 of the tests (vocabulary 257, width 64), four sequences of 64 tokens: all latency
        dict(name="loss-tiny", op="loss", rows=256, vocab=257, dim=64, dtype="bf16", train=True, reduction="mean", ignored=0.0),
        # evaluation of one sequence of GPT-2 medium: a loss for each token
        dict(name="loss-eval-1k", op="loss", rows=1024, vocab=50257, dim=1024, dtype="bf16", train=False, reduction="none", ignored=0.0),
        # GPT-2 medium's micro-batch: 8 sequences of 1024 tokens
        dict(name="loss-gpt2-medium", op="loss", rows=8192, vocab=50257, dim=1024, dtype="bf16", train=True, reduction="mean", ignored=0.0),
        # a ragged batch: prompts are masked out of the loss, each token's loss has a weight of its own
        dict(name="loss-ragged", op="loss", rows=1531, vocab=32003, dim=776, dtype="fp16", train=True, reduction="none", ignored=0.3),
        # one token through the first half of GPT-2 medium's MLP (decoding)
        dict(name="linear-one-token", op="linear", rows=1, inner=1024, outer=4096, dtype="bf16", act="gelu_tanh", bias=True, residual=False, train=False),
        # both halves of GPT-2 medium's MLP in a training step of 8 sequences of 1024 tokens
        dict(name="linear-mlp-up", op="linear", rows=8192, inner=1024, outer=4096, dtype="bf16", act="gelu_tanh", bias=True, residual=False, train=True),
        dict(name="linear-mlp-down", op="linear", rows=8192, inner=4096, outer=1024, dtype="bf16", act="none", bias=True, residual=True, train=True),
        # odd sizes all round
        dict(name="linear-odd", op="linear", rows=777, inner=1001, outer=1111, dtype="fp16", act="silu", bias=True, residual=True, train=True),
        # LeNet-5: ten small tensors in 32 bits
        dict(name="adamw-lenet", op="adamw", tensors=10, numel=44426, dtype="fp32", bits=32),
        # as many parameters and tensors as ResNet-50 has, in 32 bits, states in 8
        dict(name="adamw-25M-8bit", op="adamw", tensors=161, numel=25557032, dtype="fp32", bits=8),
        # many small odd tensors of 16 bits with 32-bit weights and states behind them
        dict(name="adamw-odd-fp16", op="adamw", tensors=301, numel=7654321, dtype="fp16", bits=32),
        # GPT-2 medium in bf16, states in 8 bits
        dict(name="adamw-gpt2-8bit", op="adamw", tensors=292, numel=354823168, dtype="bf16", bits=8),
    ]


def _log_size(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["loss", "linear", "adamw"])
    half = rng.choice(["bf16", "fp16"])
    # half of the widths are whole vectors of 16 bytes, the others are what they are
    even = lambda n: max(8, n // 8 * 8) if rng.random() < 0.5 else n  # noqa: E731
    if op == "loss":
        return dict(op=op, rows=_log_size(rng, 1, 8192), vocab=_log_size(rng, 257, 50257), dim=even(_log_size(rng, 64, 1024)), dtype=half,
                    train=rng.random() < 0.7, reduction=rng.choice(["mean", "sum", "none"]), ignored=rng.choice([0.0, 0.1, 0.5]))
    if op == "linear":
        return dict(op=op, rows=_log_size(rng, 1, 8192), inner=even(_log_size(rng, 64, 4096)), outer=even(_log_size(rng, 64, 4096)), dtype=half,
                    act=rng.choice(_ACTS), bias=rng.random() < 0.7, residual=rng.random() < 0.5, train=rng.random() < 0.6)
    tensors = _log_size(rng, 2, 300)
    return dict(op=op, tensors=tensors, numel=_log_size(rng, 200 * tensors, 350_000_000), dtype=rng.choice(["fp32", "bf16", "fp16"]), bits=rng.choice([8, 32]))


def _sizes(case):
    """Sizes of the tensors: far apart, as a model's are, and the same for a case whatever the seed."""
    k, n = case["tensors"], case["numel"]
    rng = random.Random(k * 1_000_003 + n)
    share = [math.exp(rng.gauss(0.0, 2.0)) for _ in range(k)]
    got = [max(1, int(n * s / sum(share))) for s in share]
    got[got.index(max(got))] += n - sum(got)
    return got


def _starts(sizes):
    at, got = 0, []
    for n in sizes:
        got.append(at)
        at += -(-n // _BLOCK) * _BLOCK
    return got, at


def _inside(sizes, device):
    """Which elements of the flat buffers belong to a tensor."""
    starts, total = _starts(sizes)
    edge = torch.zeros(total + 1, dtype=torch.int8, device=device)
    edge[torch.tensor(starts, device=device)] += 1
    edge.index_add_(0, torch.tensor([a + n for a, n in zip(starts, sizes)], device=device),
                    torch.full((len(sizes),), -1, dtype=torch.int8, device=device))
    return torch.cumsum(edge[:total], 0, dtype=torch.int8) > 0


# ---- inputs ----------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *size: torch.randn(*size, generator=gen, device="cuda")  # noqa: E731
    state = {"case": case, "own": own}
    dtype = _TYPES[case["dtype"]]
    if case["op"] == "loss":
        rows, vocab, dim = case["rows"], case["vocab"], case["dim"]
        state["hidden"] = normal(rows, dim).to(dtype)                        # behind a norm
        state["weight"] = (normal(vocab, dim) * (2.0 / math.sqrt(dim))).to(dtype)
        targets = torch.randint(0, vocab, (rows,), generator=gen, device="cuda")
        drop = torch.rand(rows, generator=gen, device="cuda") < case["ignored"]
        drop[0] = False
        state["targets"] = torch.where(drop, _IGNORE, targets)
        if case["reduction"] == "none":
            state["grad"] = torch.rand(rows, generator=gen, device="cuda") + 0.5
        else:
            state["grad"] = torch.ones((), device="cuda")
        if case["train"]:
            state["hidden"].requires_grad_(own)
            state["weight"].requires_grad_(own)
    elif case["op"] == "linear":
        rows, inner, outer = case["rows"], case["inner"], case["outer"]
        state["x"] = normal(rows, inner).to(dtype)
        state["weight"] = (normal(outer, inner) / math.sqrt(inner)).to(dtype)
        state["bias"] = (normal(outer) * 0.1).to(dtype) if case["bias"] else None
        state["residual"] = normal(rows, outer).to(dtype) if case["residual"] else None
        state["grad"] = normal(rows, outer).to(dtype)
        if case["train"]:
            for name in ("x", "weight", "bias"):
                if state[name] is not None:
                    state[name].requires_grad_(own)
    else:
        sizes = _sizes(case)
        starts, total = _starts(sizes)
        inside = _inside(sizes, "cuda")
        flat = {"master": normal(total).mul_(0.02).mul_(inside)}
        grad = normal(total).mul_(1e-3).mul_(inside).to(dtype)
        if case["bits"] == 32:
            flat["exp_avg"] = normal(total).mul_(3e-4).mul_(inside)
            flat["exp_avg_sq"] = normal(total).mul_(1e-3).square_().mul_(inside)
        else:
            scale = lambda low, high: torch.ldexp(torch.ones((), device="cuda"), torch.randint(low, high, (total // _BLOCK,), generator=gen, device="cuda"))  # noqa: E731
            flat["exp_avg"] = normal(total).mul_(64.0).clamp_(-440, 440).mul_(inside).to(torch.float8_e4m3fn)
            flat["exp_avg_scale"] = scale(-20, -16)
            flat["exp_avg_rms"] = normal(total).abs_().mul_(64.0).clamp_(1.0, 440.0).mul_(inside).to(torch.float8_e4m3fn)
            flat["exp_avg_rms_scale"] = scale(-18, -15)
        if dtype is not torch.float32:
            flat["param"] = flat["master"].to(dtype)
        else:
            flat["param"] = flat.pop("master")
        if own:
            from comprex_b200 import AdamW
            params = []
            for a, n in zip(starts, sizes):
                p = torch.nn.Parameter(flat["param"][a:a + n])
                p.grad = grad[a:a + n]
                params.append(p)
            opt = AdamW(params, lr=_LR, betas=_BETAS, eps=_EPS, weight_decay=_WD, state_bits=case["bits"], seed=_SEED)
            mine = opt.flat_state()
            for name in mine:
                mine[name].copy_(flat[name])
            state |= {"opt": opt, "grad": grad, "param": flat["param"]}
        else:
            state |= {"flat": flat, "grad": grad, "step": 0}
    return state


# ---- plain forms ------------------------------------------------------------------------------------------------------

def _plain_loss(s):
    case, h, w, t = s["case"], s["hidden"].float(), s["weight"].float(), s["targets"]
    rows = torch.arange(t.numel(), device=t.device)
    kept = t != _IGNORE
    at = torch.where(kept, t, 0)
    logits = h @ w.T
    top = logits.amax(1)
    e = torch.exp(logits - top[:, None])
    z = e.sum(1)
    loss = torch.where(kept, torch.log(z) + top - logits[rows, at], 0.0)
    del logits
    count = kept.sum()
    total = {"none": loss, "sum": loss.sum(), "mean": loss.sum() / count}[case["reduction"]]
    if not case["train"]:
        return {"loss": total}
    g = torch.where(kept, s["grad"].expand(t.numel()), 0.0)
    if case["reduction"] == "mean":
        g = g / count
    e *= (g / z)[:, None]
    e[rows, at] -= g
    return {"loss": total, "hidden": (e @ w).to(s["hidden"].dtype), "weight": (e.T @ h).to(s["weight"].dtype)}


def _act(u, act):
    """The activation and its derivative."""
    if act == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(u * math.sqrt(0.5)))
        return u * cdf, cdf + u * torch.exp(-0.5 * u * u) * (1.0 / math.sqrt(2.0 * math.pi))
    if act == "gelu_tanh":
        k = math.sqrt(2.0 / math.pi)
        t = torch.tanh(k * (u + 0.044715 * u * u * u))
        return 0.5 * u * (1.0 + t), 0.5 * (1.0 + t) + 0.5 * u * (1.0 - t * t) * k * (1.0 + 3 * 0.044715 * u * u)
    if act == "silu":
        q = 1.0 / (1.0 + torch.exp(-u))
        return u * q, q * (1.0 + u * (1.0 - q))
    if act == "relu":
        return torch.clamp_min(u, 0.0), (u > 0).to(u.dtype)
    return u, torch.ones_like(u)


def _plain_linear(s):
    case, dtype = s["case"], s["x"].dtype
    x, w = s["x"].float(), s["weight"].float()
    u = x @ w.T
    if s["bias"] is not None:
        u = u + s["bias"].float()
    y, slope = _act(u, case["act"])
    if s["residual"] is not None:
        y = y + s["residual"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        du = s["grad"].float() * slope
        out["x"], out["weight"] = (du @ w).to(dtype), (du.T @ x).to(dtype)
        if s["bias"] is not None:
            out["bias"] = du.sum(0).to(dtype)
    return out


def _mix(v):
    """A 32-bit number from another one, in int64: two rounds of multiply and shift."""
    v = ((v ^ (v >> 16)) * 0x7FEB352D) & 0xFFFFFFFF
    v = ((v ^ (v >> 15)) * 0x846CA68B) & 0xFFFFFFFF
    return v ^ (v >> 16)


def _at_random(x, bits):
    """float8_e4m3fn of |x| < 512 with 16 random bits added below the mantissa's end."""
    raw = x.abs().view(torch.int32)
    cut = ((raw + (bits << 4).to(torch.int32)) & ~0xFFFFF).view(torch.float32)
    return torch.copysign(cut, x)


def _scale_of(exponent):
    """Power of two that brings numbers below 2 ** (exponent - 126) under 256; ``exponent`` as float32 holds it."""
    return torch.ldexp(torch.ones((), device=exponent.device), exponent.clamp_min(8) - 134)


def _plain_adamw(s):
    case, flat = s["case"], s["flat"]
    s["step"] += 1
    b1, b2 = _BETAS
    c1, c2 = 1.0 - b1 ** s["step"], 1.0 - b2 ** s["step"]
    g = s["grad"].float()
    eight = case["bits"] == 8
    blocks = lambda x: x.view(-1, _BLOCK)  # noqa: E731
    if eight:
        m = (blocks(flat["exp_avg"].float()) * flat["exp_avg_scale"][:, None]).view(-1)
        v = (blocks(flat["exp_avg_rms"].float()) * flat["exp_avg_rms_scale"][:, None]).view(-1)
        v = v * v
    else:
        m, v = flat["exp_avg"], flat["exp_avg_sq"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * (1.0 - b2)) * g
    rms = torch.sqrt(v)
    p = flat.get("master", flat["param"])
    p = p * (1.0 - _LR * _WD) - (m * (_LR / c1)) / (rms * (1.0 / math.sqrt(c2)) + _EPS)
    if "master" in flat:
        flat["master"] = p
    flat["param"] = p.to(flat["param"].dtype)
    if eight:
        place = torch.arange(m.numel(), device=m.device)
        bits = _mix((_mix(place & 0xFFFFFFFF) + _mix(torch.tensor(_SEED + s["step"], device=m.device))) & 0xFFFFFFFF)
        del place
        exponent = blocks(m.abs()).amax(1).view(torch.int32) >> 23
        flat["exp_avg_scale"] = _scale_of(exponent)
        q = (blocks(m) * (1.0 / flat["exp_avg_scale"])[:, None]).view(-1)
        flat["exp_avg"] = _at_random(q, bits & 0xFFFF).to(torch.float8_e4m3fn)
        # the square root of a number below 2 ** e is below 2 ** ceil(e / 2)
        exponent = blocks(v).amax(1).view(torch.int32) >> 23
        flat["exp_avg_rms_scale"] = _scale_of(((exponent - 127) >> 1) + 127)
        q = (blocks(rms) * (1.0 / flat["exp_avg_rms_scale"])[:, None]).view(-1)
        q = torch.where(v > 0, _at_random(q, bits >> 16).clamp_min(2.0 ** -9), 0.0)     # what is not zero stays above it
        flat["exp_avg_rms"] = q.to(torch.float8_e4m3fn)
    else:
        flat["exp_avg"], flat["exp_avg_sq"] = m, v
    return dict(flat)


# ---- one pass ---------------------------------------------------------------------------------------------------------

def run(state):
    case = state["case"]
    if not state["own"]:
        return {"loss": _plain_loss, "linear": _plain_linear, "adamw": _plain_adamw}[case["op"]](state)
    import comprex_b200 as cx
    if case["op"] == "loss":
        loss = cx.linear_cross_entropy(state["hidden"], state["weight"], state["targets"], ignore_index=_IGNORE, reduction=case["reduction"])
        if not case["train"]:
            return {"loss": loss}
        dh, dw = torch.autograd.grad(loss, (state["hidden"], state["weight"]), state["grad"])
        return {"loss": loss.detach(), "hidden": dh, "weight": dw}
    if case["op"] == "linear":
        y = cx.linear(state["x"], state["weight"], state["bias"], activation=None if case["act"] == "none" else case["act"], residual=state["residual"])
        if not case["train"]:
            return {"y": y}
        names = [n for n in ("x", "weight", "bias") if state[n] is not None]
        return {"y": y.detach(), **dict(zip(names, torch.autograd.grad(y, [state[n] for n in names], state["grad"])))}
    state["opt"].step()
    return {**state["opt"].flat_state(), "param": state["param"]}


# ---- what a pass cannot do without -----------------------------------------------------------------------------------

def work(case):
    b = _BYTES[case["dtype"]]
    if case["op"] == "loss":
        rows, vocab, dim, train = case["rows"], case["vocab"], case["dim"], case["train"]
        size = (rows + vocab) * dim * b
        return {"bytes": size * (2 if train else 1) + rows * (8 + (4 if case["reduction"] == "none" else 0) * (2 if train else 1)),
                "flops": 2 * rows * vocab * dim * (3 if train else 1)}
    if case["op"] == "linear":
        rows, inner, outer, train = case["rows"], case["inner"], case["outer"], case["train"]
        more = outer * case["bias"] + rows * outer * case["residual"]
        size = rows * inner + outer * inner + rows * outer + more
        if train:
            size += rows * outer + rows * inner + outer * inner + outer * case["bias"]
        return {"bytes": size * b, "flops": 2 * rows * inner * outer * (3 if train else 1)}
    n = case["numel"]
    each = b + 2 * 4 + (b if b < 4 else 0)                # gradient, 32-bit weights in and out, 16-bit copy
    each += 2 * (8 if case["bits"] == 32 else 2 + 8 / _BLOCK)
    return {"bytes": n * each, "flops": 14 * n}


# ---- 64 bits ----------------------------------------------------------------------------------------------------------

def exact(case, seed):
    global own
    mine, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = mine
    return {"loss": _exact_loss, "linear": _exact_linear, "adamw": _exact_adamw}[case["op"]](s)


def _exact_loss(s):
    case = s["case"]
    h, w, t = s["hidden"].double(), s["weight"].double(), s["targets"]
    keep = (t != _IGNORE).double()
    dh, dw, losses = torch.zeros_like(h), torch.zeros_like(w), []
    scale = s["grad"].double().expand(t.numel()) * keep
    if case["reduction"] == "mean":
        scale = scale / keep.sum()
    for i in range(0, t.numel(), 1024):
        part = slice(i, i + 1024)
        logp = torch.log_softmax(h[part] @ w.T, 1)
        hot = torch.zeros_like(logp).scatter_(1, t[part].clamp_min(0)[:, None], 1.0)
        losses.append(-(logp * hot).sum(1) * keep[part])
        if case["train"]:
            d = (logp.exp_() - hot) * scale[part, None]
            dh[part] = d @ w
            dw += d.T @ h[part]
    loss = torch.cat(losses)
    if case["reduction"] != "none":
        loss = loss.sum() / (keep.sum() if case["reduction"] == "mean" else 1.0)
    return {"loss": loss, "hidden": dh, "weight": dw} if case["train"] else {"loss": loss}


def _exact_linear(s):
    case = s["case"]
    x, w, b, r = (None if s[n] is None else s[n].double() for n in ("x", "weight", "bias", "residual"))
    u = (x @ w.T if b is None else torch.addmm(b, x, w.T)).requires_grad_()
    act = {"none": lambda v: v * 1.0, "gelu": torch.nn.functional.gelu, "silu": torch.nn.functional.silu, "relu": torch.relu,
           "gelu_tanh": lambda v: torch.nn.functional.gelu(v, approximate="tanh")}[case["act"]]
    y = act(u)
    out = {"y": (y if r is None else y + r).detach()}
    if case["train"]:
        du, = torch.autograd.grad(y, u, s["grad"].double())
        out |= {"x": du @ w, "weight": du.T @ x}
        if b is not None:
            out["bias"] = du.sum(0)
    return out


def _exact_adamw(s):
    case, flat, g = s["case"], s["flat"], s["grad"].double()
    eight = case["bits"] == 8
    spread = lambda name: torch.repeat_interleave(flat[name].double(), _BLOCK)  # noqa: E731
    if eight:
        m, v = flat["exp_avg"].double() * spread("exp_avg_scale"), (flat["exp_avg_rms"].double() * spread("exp_avg_rms_scale")) ** 2
    else:
        m, v = flat["exp_avg"].double(), flat["exp_avg_sq"].double()
    b1, b2 = _BETAS
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    p = flat.get("master", flat["param"]).double()
    p = (1 - _LR * _WD) * p - _LR * (m / (1 - b1)) / (torch.sqrt(v / (1 - b2)) + _EPS)
    # what is rounded at random has no value of its own
    out = {name: None for name in flat}
    if not eight:
        out |= {"exp_avg": m, "exp_avg_sq": v}
    out["param"] = p
    if "master" in out:
        out["master"] = p
    return out
