"""Operators around a quantised language model, as cases that can be timed and compared.

Kinds, by the public entry point that a pass calls:

  fake     microscale.quantize_fp4(x, format).dequantize(): a matrix rounded to 4-bit blocks and back, as calibration does
  linear   microscale.fp4_linear(x, w, bias, relu): activations quantised on the fly, product with a packed weight
  score    scoring.token_logprobs(logits, tokens, top_k): log probability, rank, entropy and the top alternatives
  distill  scoring.distillation_loss(logits, ids, teacher, ...) and its backward pass, as a training step issues them
  grad     scoring.distillation_loss_and_grad(...): the same loss and gradient from one call

Formats: "mxfp4" is blocks of 32 with a power-of-two scale 2^(floor(log2 amax) - 2); "nvfp4" is blocks of 16 with an e4m3 scale
RN(amax / (6 g)) under a power of two g per row, the smallest with 448 * 6 * g >= the row's largest magnitude. Elements are e2m1
(0, 0.5, 1, 1.5, 2, 3, 4, 6), round to nearest, ties to the even code.
"""
import math

import torch

own = False

DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
BLOCK = {"mxfp4": 32, "nvfp4": 16}


def listed():
    return [
        # a weight of the widest layer (fc1 of OPT-6.7B), as a model is converted and checked
        {"name": "fake weight nvfp4", "kind": "fake", "R": 16384, "K": 4096, "dtype": "fp32", "format": "nvfp4"},
        # activations of a small batch with a width that is no multiple of a block
        {"name": "fake ragged mxfp4", "kind": "fake", "R": 515, "K": 2050, "dtype": "bf16", "format": "mxfp4"},
        # one token through fc1 of OPT-6.7B: the smallest call, latency and the weight's bytes
        {"name": "linear 1 token", "kind": "linear", "M": 1, "K": 4096, "N": 16384, "dtype": "fp16", "format": "nvfp4", "relu": True},
        # a decode batch through fc2: deep, few output columns
        {"name": "linear 16 tokens deep", "kind": "linear", "M": 16, "K": 16384, "N": 4096, "dtype": "bf16", "format": "mxfp4", "relu": False},
        # a short prompt through an attention projection
        {"name": "linear 512 tokens", "kind": "linear", "M": 512, "K": 4096, "N": 4096, "dtype": "bf16", "format": "nvfp4", "relu": False},
        # no power of two anywhere, depth that ends inside a block
        {"name": "linear ragged", "kind": "linear", "M": 777, "K": 2090, "N": 5003, "dtype": "fp16", "format": "mxfp4", "relu": False},
        # prefill of 32 sequences of 256 tokens through fc1
        {"name": "linear prefill", "kind": "linear", "M": 8192, "K": 4096, "N": 16384, "dtype": "bf16", "format": "nvfp4", "relu": True},
        # one decoding step of 8 sequences over OPT's vocabulary, with the alternatives that an API returns
        {"name": "score decode", "kind": "score", "B": 8, "T": 1, "V": 50272, "dtype": "fp16", "top": 20},
        # evaluation of 8 sequences of 256 tokens: every position scores the token after it, the last one has none
        {"name": "score sequences", "kind": "score", "B": 8, "T": 256, "V": 50272, "dtype": "fp16", "top": 5},
        # a teacher's pass over a large odd vocabulary in float32, 64 alternatives kept for a student
        {"name": "score teacher", "kind": "score", "B": 3, "T": 211, "V": 128011, "dtype": "fp32", "top": 64},
        # a training step's loss: forward and backward over the logits of 2048 positions
        {"name": "distill step", "kind": "distill", "rows": 2048, "V": 50272, "dtype": "bf16", "top": 64, "temperature": 2.0, "tail": False},
        # a few positions over a large vocabulary, the rest of the teacher's mass as one class, loss and gradient at once
        {"name": "grad tail", "kind": "grad", "rows": 96, "V": 128011, "dtype": "fp32", "top": 16, "temperature": 1.0, "tail": True},
    ]


def _size(rng, low, high, multiple):
    """A size spread over the logarithm of [low, high]: half of the time a multiple, else any number."""
    n = int(round(low * (high / low) ** rng.random()))
    if rng.random() < 0.5:
        n = max(multiple, n // multiple * multiple)
    return max(low, min(high, n))


def draw(rng):
    kind = rng.choice(["fake", "linear", "linear", "score", "score", "distill", "grad"])
    case = {"kind": kind, "dtype": rng.choice(["fp16", "bf16", "fp32"])}
    if kind in ("fake", "linear"):
        case["format"] = rng.choice(["mxfp4", "nvfp4"])
    if kind == "fake":
        case.update(R=_size(rng, 1, 16384, 128), K=_size(rng, 64, 16384, 64))
        while case["R"] * case["K"] > 16384 * 4096:
            case["R"] = max(1, case["R"] // 2)
    elif kind == "linear":
        case.update(M=_size(rng, 1, 8192, 32), K=_size(rng, 128, 16384, 64), N=_size(rng, 256, 16384, 128), relu=rng.random() < 0.3)
        while case["M"] * case["K"] * case["N"] > 8192 * 4096 * 16384:
            case["M"] = max(1, case["M"] // 2)
    elif kind == "score":
        case.update(B=_size(rng, 1, 16, 4), T=_size(rng, 1, 512, 16), V=_size(rng, 1000, 200000, 32), top=rng.choice([0, 1, 5, 20, 64, 128]))
        while case["B"] * case["T"] * case["V"] > 8 * 256 * 50272:
            case["T"] = max(1, case["T"] // 2)
            case["B"] = case["B"] if case["T"] > 1 else max(1, case["B"] // 2)
    else:
        case.update(rows=_size(rng, 1, 4096, 32), V=_size(rng, 1000, 200000, 32), top=rng.choice([1, 8, 20, 64, 128]),
                    temperature=rng.choice([1.0, 2.0, 0.7]), tail=rng.random() < 0.5)
        while case["rows"] * case["V"] > 2048 * 50272:
            case["rows"] = max(1, case["rows"] // 2)
    return case


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def _gen(seed, salt=0):
    return torch.Generator(device="cuda").manual_seed((seed * 7919 + salt) % (1 << 62))


def _normal(shape, g, std=1.0):
    return torch.empty(shape, dtype=torch.float32, device="cuda").normal_(0.0, std, generator=g)


def _activations(rows, width, g):
    """What a LayerNorm leaves: unit normals, one channel in a hundred twenty times as large."""
    x = _normal((rows, width), g)
    hot = torch.rand(width, generator=g, device="cuda") < 0.01
    return x.mul_(1.0 + 19.0 * hot)


def _logits(rows, vocab, g):
    """Logits of a language model: most near a common level, a heavy upper tail."""
    x = _normal((rows, vocab), g, 1.5)
    return x.add_(x.abs().pow_(3).mul_(0.05))


def prepare(case, seed):
    g = _gen(seed)
    kind, dtype = case["kind"], DTYPES[case["dtype"]]
    if kind == "fake":
        return {"case": case, "x": _activations(case["R"], case["K"], g).mul_(0.02).to(dtype)}
    if kind == "linear":
        x = _activations(case["M"], case["K"], g).to(dtype)
        w = _normal((case["N"], case["K"]), g, 0.02)
        state = {"case": case, "x": x, "bias": _normal((case["N"],), g, 0.1)}
        if own:      # a model's weight is packed once, when it is loaded
            from bsipytorch_b200 import microscale
            state["w"] = microscale.quantize_fp4(w, case["format"])
        else:        # the values that the packed weight stands for
            state["w"] = _rounded(w, case["format"])
        return state
    if kind == "score":
        B, T, V = case["B"], case["T"], case["V"]
        state = {"case": case, "logits": _logits(B * (T + 1), V, g).to(dtype).view(B, T + 1, V)}
        state["ids"] = torch.randint(0, V, (B, T + 1), generator=g, device="cuda")
        state["ids"][:, -1] = state["logits"][:, -2].argmax(-1)      # some tokens are the model's own choice
        state["ids"][-1, 1::7] = -100                                # and some are not scored
        return state
    rows, V, K, T = case["rows"], case["V"], case["top"], case["temperature"]
    logits = _logits(rows, V, g)
    teacher = logits + _normal((rows, V), g, 0.5)
    if case["tail"]:     # log probabilities at the loss's temperature
        teacher = torch.log_softmax(teacher / T, -1)
    top, ids = torch.topk(teacher, K, -1)
    weights = (torch.rand(rows, generator=g, device="cuda") < 0.9).float()    # padded positions
    weights[0] = 1.0
    ids[-1, K // 2:] = -1 if rows > 1 else ids[-1, K // 2:]                    # a position with fewer alternatives
    return {"case": case, "logits": logits.to(dtype), "ids": ids, "teacher": top, "weights": weights}


# ---- the framework's calls ---------------------------------------------------------------------------------------------------

def _own(state):
    from bsipytorch_b200 import microscale, scoring
    case = state["case"]
    kind = case["kind"]
    if kind == "fake":
        return microscale.quantize_fp4(state["x"], case["format"]).dequantize()
    if kind == "linear":
        return microscale.fp4_linear(state["x"], state["w"], state["bias"], relu=case["relu"])
    if kind == "score":
        s = scoring.token_logprobs(state["logits"][:, :-1], state["ids"][:, 1:], top_k=case["top"])
        return [s.logprobs, s.ranks, s.entropy, s.top_logprobs, s.top_ids]
    more = dict(temperature=case["temperature"], tail=case["tail"], weights=state["weights"])
    if kind == "grad":
        return scoring.distillation_loss_and_grad(state["logits"], state["ids"], state["teacher"], **more)
    logits = state["logits"].detach().requires_grad_()
    loss = scoring.distillation_loss(logits, state["ids"], state["teacher"], **more)
    loss.backward()
    return loss.detach(), logits.grad


# ---- plain forms ---------------------------------------------------------------------------------------------------------------

def _e2m1(v):
    """The nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 with v's sign; ties to the even code."""
    a = v.abs()
    q = 0.5 * ((a > 0.25).float() + (a >= 0.75).float() + (a > 1.25).float() + (a >= 1.75).float())
    q = q + (a > 2.5).float() + (a >= 3.5).float() + 2.0 * (a > 5.0).float()
    return torch.where(v < 0, -q, q)


def _rounded(x, fmt):
    """The float32 values that a matrix packed as fmt stands for. Every quotient below is compared with a border of at most seven
    bits, for which float32 division is exact enough: a quotient on the wrong side would have to be nearer than half a step."""
    rows, width = x.shape
    block = BLOCK[fmt]
    pad = -width % block
    v = torch.nn.functional.pad(x.float(), (0, pad)).view(rows, -1, block)
    amax = v.abs().amax(-1, keepdim=True)
    if fmt == "mxfp4":
        _, e = torch.frexp(amax)                    # amax = m 2^e, m in [0.5, 1)
        scale = torch.ldexp(torch.ones_like(amax), (e - 3).clamp(-126, 127))
    else:
        _, e = torch.frexp(amax.amax(1, keepdim=True) / 2688.0)
        g = torch.ldexp(torch.ones_like(amax[:, :1]), e.clamp(-126, 127))
        half = g * 0.5
        g = torch.where(amax.amax(1, keepdim=True) <= half * 2688.0, half, g)       # on the border the smaller one will do
        scale = (amax / (6.0 * g)).to(torch.float8_e4m3fn).float() * g
    safe = torch.where(scale > 0, scale, 1.0)
    q = torch.where(scale > 0, _e2m1(v / safe) * scale, 0.0)
    return q.view(rows, width + pad)[:, :width].contiguous()


def _plain_score(state):
    case = state["case"]
    z = state["logits"][:, :-1].reshape(-1, case["V"]).float()
    ids = state["ids"][:, 1:].reshape(-1)
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(-1)
    lse = m.squeeze(-1) + torch.log(s)
    entropy = lse - (e * z).sum(-1) / s
    scored = ids >= 0
    zt = z.gather(1, ids.clamp(min=0)[:, None])
    index = torch.arange(case["V"], device=z.device)
    ahead = (z > zt) | ((z == zt) & (index < ids[:, None]))
    logprobs = torch.where(scored, zt.squeeze(1) - lse, 0.0)
    ranks = torch.where(scored, ahead.sum(-1), -1)
    # one whole number for each entry, larger for a larger value and, among equals, for a lower index
    bits = z.view(torch.int32).long()
    key = torch.where(bits < 0, -(bits & 0x7FFFFFFF), bits) * (1 << 20) + ((1 << 20) - 1 - index)
    top_ids = torch.topk(key, case["top"], -1).indices
    top = z.gather(1, top_ids) - lse[:, None]
    shape = (case["B"], case["T"])
    return [logprobs.view(shape), ranks.view(shape), entropy.view(shape), top.view(*shape, -1), top_ids.view(*shape, -1)]


def _plain_distill(state):
    case = state["case"]
    T = case["temperature"]
    z = state["logits"].float() / T
    ids, there = state["ids"].clamp(min=0), state["ids"] >= 0
    m = z.amax(-1, keepdim=True)
    e = torch.exp(z - m)
    s = e.sum(-1, keepdim=True)
    t = state["teacher"].float()
    if case["tail"]:
        logp = t
        p = torch.where(there, torch.exp(t), 0.0)
        rest = (1.0 - p.sum(-1, keepdim=True)).clamp(min=0.0)
    else:
        t = torch.where(there, t / T, -math.inf)
        top = t.amax(-1, keepdim=True)
        logp = t - top - torch.log(torch.exp(t - top).sum(-1, keepdim=True))
        p = torch.exp(logp)
        rest = torch.zeros_like(s)
    logq = z.gather(1, ids) - m - torch.log(s)
    loss = torch.where(p > 0, p * (logp - logq), 0.0).sum(-1)
    q = e / s
    target = torch.zeros_like(z).scatter_add_(1, ids, p)
    if case["tail"]:
        listed_ = torch.zeros_like(z).scatter_add_(1, ids, there.float()) > 0
        out = torch.where(listed_, 0.0, e).sum(-1, keepdim=True)
        logr = torch.log(out) - torch.log(s)
        loss = loss + torch.where(rest > 0, rest * (torch.log(rest) - logr), 0.0).squeeze(-1)
        grad = torch.where(listed_, q - target, q * (1.0 - rest * s / out))
    else:
        grad = q - target
    w = state["weights"] / state["weights"].sum()
    return (loss * w).sum() * T * T, (grad * (w * T)[:, None]).to(state["logits"].dtype)


def run(state):
    if own:
        return _own(state)
    case = state["case"]
    if case["kind"] == "fake":
        return _rounded(state["x"], case["format"]).to(state["x"].dtype)
    if case["kind"] == "linear":
        y = torch.matmul(_rounded(state["x"], case["format"]), state["w"].t()) + state["bias"]
        return (torch.relu(y) if case["relu"] else y).to(state["x"].dtype)
    return _plain_score(state) if case["kind"] == "score" else _plain_distill(state)


# ---- the same from the definitions, in 64 bits -----------------------------------------------------------------------------------

def _exact_rounded(x, fmt):
    grid = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64, device=x.device)
    fine = torch.tensor([i * 2.0 ** -9 for i in range(8)] + [(8 + i) * 2.0 ** (e - 3) for e in range(-6, 9) for i in range(8)][:119],
                        dtype=torch.float64, device=x.device)        # what e4m3 holds: 0 to 448

    def nearest(v, table):
        """Index of the entry that each v >= 0 rounds to: nearest, the even index on a tie, the last one beyond."""
        up = torch.searchsorted(table, v).clamp(1, table.numel() - 1)
        low = up - 1
        to_low, to_up = v - table[low], table[up] - v
        return torch.where((to_low < to_up) | ((to_low == to_up) & (low % 2 == 0)), low, up)

    parts = torch.nn.functional.pad(x.double(), (0, -x.shape[1] % BLOCK[fmt])).unflatten(1, (-1, BLOCK[fmt]))
    largest = parts.abs().amax(2)
    if fmt == "mxfp4":
        e = torch.round(torch.log2(largest.clamp(min=1e-300)))        # a logarithm may be off beside a whole number
        scale = torch.exp2(torch.where(torch.exp2(e) > largest, e - 1.0, e) - 2.0) * (largest > 0)
    else:
        most = largest.amax(1, keepdim=True).clamp(min=1e-300) / 2688.0
        e = torch.round(torch.log2(most))
        g = torch.exp2(torch.where(torch.exp2(e) < most, e + 1.0, e))
        scale = fine[nearest(largest / (6.0 * g), fine)] * g
    on = scale > 0
    units = parts.abs() / torch.where(on, scale, 1.0)[..., None]
    values = grid[nearest(units, grid)] * torch.sign(parts) * torch.where(on, scale, 0.0)[..., None]
    return values.flatten(1)[:, :x.shape[1]]


def exact(case, seed):
    kind = case["kind"]
    g = _gen(seed)
    state = prepare(case, seed)
    if kind == "fake":
        return _exact_rounded(state["x"], case["format"])
    if kind == "linear":
        _activations(case["M"], case["K"], g)                     # the generator's way to the weight
        w = _normal((case["N"], case["K"]), g, 0.02)
        y = torch.addmm(state["bias"].double(), _exact_rounded(state["x"], case["format"]), _exact_rounded(w, case["format"]).t())
        return y.clamp(min=0.0) if case["relu"] else y
    if kind == "score":
        z = state["logits"][:, :-1].double()
        ids = state["ids"][:, 1:]
        logq = torch.log_softmax(z, -1)
        chosen = torch.where(ids >= 0, logq.gather(-1, ids.clamp(min=0)[..., None])[..., 0], 0.0)
        entropy = -(torch.exp(logq) * logq).sum(-1)
        best = torch.topk(logq, case["top"], -1).values
        return [chosen, None, entropy, best, None]
    T = case["temperature"]
    logits = state["logits"].double().requires_grad_()
    logq = torch.log_softmax(logits / T, -1)
    there = state["ids"] >= 0
    ids = state["ids"].clamp(min=0)
    t = state["teacher"].double()
    if case["tail"]:
        p = torch.where(there, torch.exp(t), 0.0)
        rest = (1.0 - p.sum(-1)).clamp(min=0.0)
        outside = torch.ones_like(logq, dtype=torch.bool)
        rows, places = torch.nonzero(there, as_tuple=True)
        outside[rows, ids[rows, places]] = False
        cross = -(rest * torch.logsumexp(torch.where(outside, logq, -math.inf), -1))
        own_part = torch.xlogy(p, p).sum(-1) + torch.xlogy(rest, rest)
    else:
        p = torch.softmax(torch.where(there, t / T, -math.inf), -1)
        cross = 0.0
        own_part = torch.xlogy(p, p).sum(-1)
    each = own_part + cross - (p * logq.gather(-1, ids)).sum(-1)
    loss = T * T * (each * state["weights"].double()).sum() / state["weights"].double().sum()
    loss.backward()
    return loss.detach(), logits.grad


def work(case):
    kind = case["kind"]
    size = {"fp16": 2, "bf16": 2, "fp32": 4}[case["dtype"]]
    if kind == "fake":
        n = case["R"] * case["K"]
        return {"bytes": 2 * n * size, "flops": 4 * n}
    if kind == "linear":
        M, K, N = case["M"], case["K"], case["N"]
        packed = N * K // 2 + N * K // BLOCK[case["format"]]
        return {"bytes": M * K * size + packed + N * 4 + M * N * size, "flops": 2 * M * K * N}
    if kind == "score":
        rows, V, K = case["B"] * case["T"], case["V"], case["top"]
        return {"bytes": rows * (V * size + 8 + 16 + K * 12), "flops": 6 * rows * V}
    rows, V, K = case["rows"], case["V"], case["top"]
    return {"bytes": 2 * rows * V * size + rows * (K * 12 + 4) + 4, "flops": 10 * rows * V}
