"""Products with what stands behind them: 8-bit linear layers, the gated feed-forward block and the cross entropy of a
linear head, forward and backward, over the sizes at which a program calls them.

A case is a dict of plain values; `op` says which operator it measures.  `listed()` names twelve of them, `draw()` gives further ones
of the same ranges.  `run` computes them from elementary operations in 32 bits (products of 8-bit integers, whose sums pass 2^24, in 64), or,
where `own` is true, through tilefusion_amd.ops.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
IGNORED = -100

# Bounds of a drawn case, so that none costs more than the largest listed ones.
MAX_INT8_FLOPS = 2.0 * 4096 ** 3
MAX_FFN_FLOPS = 4.0 * 8191 * 4096 * 11264
MAX_FFN_BACKWARD_FLOPS = 8.0 * 8192 * 4096 * 11264
MAX_LOSS_FLOPS = 2.0 * 4095 * 50021 * 2048
MAX_LOSS_BACKWARD_FLOPS = 6.0 * 8192 * 131072 * 1024


def listed():
    return [
        # A linear layer over the rows of one decoding step, its weight held in 8 bits: every weight read once.
        {"name": "int8_few_rows", "op": "int8", "m": 16, "n": 4096, "k": 4096, "dtype": "bf16", "out": "bf16"},
        # The GEMM's packed tokens: a row count of no particular divisor, an fp32 result.
        {"name": "int8_ragged", "op": "int8", "m": 2999, "n": 1544, "k": 1032, "dtype": "fp16", "out": "fp32"},
        # The repository's GEMM benchmark in 8 bits.
        {"name": "int8_4096", "op": "int8", "m": 4096, "n": 4096, "k": 4096, "dtype": "fp16", "out": "fp16"},
        # One token of one conversation: the smallest call of the block, two weights read once.
        {"name": "ffn_one_token", "op": "ffn", "m": 1, "k": 4096, "f": 11264, "dtype": "bf16", "activation": "silu", "keep": False},
        # A training step's forward pass over packed tokens at widths that no tile divides.
        {"name": "ffn_ragged", "op": "ffn", "m": 2999, "k": 1032, "f": 1544, "dtype": "fp16", "activation": "gelu", "keep": True},
        # Prefill of a long prompt.
        {"name": "ffn_prefill", "op": "ffn", "m": 8191, "k": 4096, "f": 11264, "dtype": "bf16", "activation": "silu", "keep": False},
        # Fine-tuning on short batches.
        {"name": "ffn_backward_ragged", "op": "ffn_backward", "m": 1337, "k": 1032, "f": 1544, "dtype": "fp16", "activation": "gelu_tanh"},
        # A training step at full size.
        {"name": "ffn_backward_large", "op": "ffn_backward", "m": 8192, "k": 4096, "f": 11264, "dtype": "bf16", "activation": "silu"},
        # Scoring a short text against the embedding table of the scatter_nd case.
        {"name": "loss_scoring", "op": "loss", "t": 37, "k": 1024, "v": 32000, "dtype": "fp16"},
        # Evaluating a long batch over an odd vocabulary.
        {"name": "loss_odd_vocabulary", "op": "loss", "t": 4095, "k": 2048, "v": 50021, "dtype": "bf16"},
        # The head's gradient in fine-tuning: few tokens, every sequence with a mean of its own.
        {"name": "loss_backward_few", "op": "loss_backward", "t": 613, "k": 1024, "v": 32003, "dtype": "fp16", "weights": "sequence"},
        # The head's gradient of a training step, with the largest table that scatter_nd is measured on.
        {"name": "loss_backward_large", "op": "loss_backward", "t": 8192, "k": 1024, "v": 131072, "dtype": "bf16", "weights": "mean"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _width(rng, low, high):
    """A layer's width: mostly a multiple of 64, otherwise of 8, now and then of nothing."""
    x, r = _log_int(rng, low, high), rng.random()
    return max(64, x // 64 * 64) if r < 0.6 else max(8, x // 8 * 8) if r < 0.9 else x


def draw(rng):
    op = rng.choice(["int8", "ffn", "ffn_backward", "loss", "loss_backward"])
    dtype = rng.choice(["fp16", "bf16"])
    while True:
        if op == "int8":
            case = {"op": op, "m": _log_int(rng, 1, 8192), "n": _width(rng, 64, 8192), "k": _width(rng, 64, 8192), "dtype": dtype,
                    "out": rng.choice(["fp32", dtype])}
            most = MAX_INT8_FLOPS
        elif op == "ffn":
            case = {"op": op, "m": _log_int(rng, 1, 8192), "k": _width(rng, 64, 8192), "f": _width(rng, 64, 14336), "dtype": dtype,
                    "activation": rng.choice(["silu", "silu", "gelu", "gelu_tanh"]), "keep": rng.random() < 0.5}
            most = MAX_FFN_FLOPS
        elif op == "ffn_backward":
            case = {"op": op, "m": _log_int(rng, 1, 8192), "k": _width(rng, 64, 8192), "f": _width(rng, 64, 14336), "dtype": dtype,
                    "activation": rng.choice(["silu", "silu", "gelu", "gelu_tanh"])}
            most = MAX_FFN_BACKWARD_FLOPS
        elif op == "loss":
            case = {"op": op, "t": _log_int(rng, 1, 8192), "k": _width(rng, 64, 4096), "v": _log_int(rng, 1000, 131072), "dtype": dtype}
            most = MAX_LOSS_FLOPS
        else:
            case = {"op": op, "t": _log_int(rng, 1, 8192), "k": _width(rng, 64, 4096), "v": _log_int(rng, 1000, 131072), "dtype": dtype,
                    "weights": rng.choice(["mean", "sequence"])}
            most = MAX_LOSS_BACKWARD_FLOPS
        if work(case)["flops"] <= most:
            return case


def _randn(g, *shape, dtype, scale=1.0):
    x = torch.randn(*shape, device=DEVICE, dtype=dtype, generator=g)
    return x if scale == 1.0 else x.mul_(scale)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, dtype, k = case["op"], DTYPES[case["dtype"]], case["k"]
    if op == "int8":
        m, n = case["m"], case["n"]
        # a checkpoint's weight: 8-bit rows, each filling its range, and what a step of each is worth
        return {"op": op, "x": _randn(g, m, k, dtype=dtype), "w": torch.randint(-127, 128, (n, k), device=DEVICE, dtype=torch.int8, generator=g),
                "w_scale": torch.rand(n, device=DEVICE, generator=g).add_(0.5).mul_(1.0 / (74.0 * math.sqrt(k))),
                "c": torch.empty(m, n, device=DEVICE, dtype=DTYPES[case["out"]])}
    if op in ("ffn", "ffn_backward"):
        m, f = case["m"], case["f"]
        state = {"op": op, "activation": case["activation"], "x": _randn(g, m, k, dtype=dtype),
                 "w_gate": _randn(g, f, k, dtype=dtype, scale=k ** -0.5), "w_up": _randn(g, f, k, dtype=dtype, scale=k ** -0.5)}
        if op == "ffn":
            return {**state, "keep": case["keep"]}
        # gate and up as the forward pass kept them: of unit variance, as the inputs and weights above make them
        return {**state, "gate": _randn(g, m, f, dtype=dtype), "up": _randn(g, m, f, dtype=dtype), "grad_h": _randn(g, m, f, dtype=dtype)}
    t, v = case["t"], case["v"]
    hidden, weight = _randn(g, t, k, dtype=dtype), _randn(g, v, k, dtype=dtype, scale=2.0 * k ** -0.5)
    # log-uniform words; the first fifth of the tokens, a prompt, has no target
    target = (torch.pow(float(v), torch.rand(t, device=DEVICE, dtype=torch.float64, generator=g)).long() - 1).clamp_(0, v - 1)
    target[: t // 5] = IGNORED
    state = {"op": op, "hidden": hidden, "weight": weight, "target": target}
    if op == "loss":
        return state
    if case["weights"] == "mean":
        grad_loss = torch.full((t,), 1.0 / (t - t // 5), device=DEVICE)
    else:
        # sequences of 64 tokens, the weight of a token that of its sequence
        sequence = torch.rand((t + 63) // 64, device=DEVICE, generator=g).add_(0.25).div_(64.0)
        grad_loss = sequence.repeat_interleave(64)[:t].contiguous()
    if case["dtype"] == "fp16":
        grad_loss *= 4096.0   # the scale of the loss, without which gradients in fp16 vanish
    # as the forward pass returned it
    lse = torch.logsumexp(hidden.float() @ weight.float().t(), dim=-1)
    return {**state, "grad_loss": grad_loss, "lse": lse}


def _act(g, activation):
    """The activation and its derivative."""
    if activation == "silu":
        s = 1.0 / (1.0 + torch.exp(-g))
        return g * s, s * (1.0 + g * (1.0 - s))
    if activation == "gelu":
        cdf = 0.5 * (1.0 + torch.erf(g * math.sqrt(0.5)))
        return g * cdf, cdf + g * torch.exp(-0.5 * g * g) * (1.0 / math.sqrt(2.0 * math.pi))
    c = math.sqrt(2.0 / math.pi)
    th = torch.tanh(c * (g + 0.044715 * g * g * g))
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * c * (1.0 + 3 * 0.044715 * g * g)


def _plain_int8(s):
    x = s["x"].float()
    # (quotients in 64 bits: one in 32 that lies next to the middle of two whole numbers is rounded onto it)
    step = (x.abs().amax(dim=1).double() / 127.0).float().double().unsqueeze(1)
    q = torch.where(step > 0, torch.round(x.double() / step), torch.zeros_like(step))
    y = (q @ s["w"].double().t()) * step * s["w_scale"].double()
    s["c"].copy_(y)
    return s["c"]


def _plain_ffn(s):
    dtype, x = s["x"].dtype, s["x"].float()
    gate, up = x @ s["w_gate"].float().t(), x @ s["w_up"].float().t()
    h = (_act(gate, s["activation"])[0] * up).to(dtype)
    return (h, gate.to(dtype), up.to(dtype)) if s["keep"] else h


def _plain_ffn_backward(s):
    dtype = s["x"].dtype
    gate, up, grad_h = s["gate"].float(), s["up"].float(), s["grad_h"].float()
    value, slope = _act(gate, s["activation"])
    grad_gate, grad_up = grad_h * up * slope, grad_h * value
    grad_x = grad_gate @ s["w_gate"].float() + grad_up @ s["w_up"].float()
    x = s["x"].float()
    return grad_x.to(dtype), (grad_gate.t() @ x).to(dtype), (grad_up.t() @ x).to(dtype)


def _plain_loss(s):
    logits = s["hidden"].float() @ s["weight"].float().t()
    top = logits.amax(dim=1)
    lse = top + torch.log(torch.exp(logits - top.unsqueeze(1)).sum(dim=1))
    valid = s["target"] != IGNORED
    at_target = logits.gather(1, torch.where(valid, s["target"], 0).unsqueeze(1)).squeeze(1)
    return torch.where(valid, lse - at_target, torch.zeros_like(lse)), lse


def _plain_loss_backward(s):
    dtype, hidden, weight = s["hidden"].dtype, s["hidden"].float(), s["weight"].float()
    valid = s["target"] != IGNORED
    p = torch.exp(hidden @ weight.t() - s["lse"].unsqueeze(1))
    at_target = torch.where(valid, s["target"], 0).unsqueeze(1)
    p.scatter_add_(1, at_target, torch.full_like(at_target, -1, dtype=torch.float32))
    p *= torch.where(valid, s["grad_loss"], torch.zeros_like(s["grad_loss"])).unsqueeze(1)
    return (p @ weight).to(dtype), (p.t() @ hidden).to(dtype)


def _own(s):
    from tilefusion_amd import ops

    op = s["op"]
    if op == "int8":
        q, scale = ops.quantize_rows(s["x"])
        ops.gemm_int8(q, s["w"], scale, s["w_scale"], s["c"])
        return s["c"]
    if op == "ffn":
        return ops.gated_ffn(s["x"], s["w_gate"], s["w_up"], s["activation"], s["keep"])
    if op == "ffn_backward":
        return ops.gated_ffn_backward(s["grad_h"], s["x"], s["w_gate"], s["w_up"], s["gate"], s["up"], s["activation"])
    if op == "loss":
        return ops.linear_cross_entropy(s["hidden"], s["weight"], s["target"], IGNORED)
    return ops.linear_cross_entropy_backward(s["grad_loss"], s["hidden"], s["weight"], s["target"], s["lse"], IGNORED)


_PLAIN = {"int8": _plain_int8, "ffn": _plain_ffn, "ffn_backward": _plain_ffn_backward, "loss": _plain_loss,
          "loss_backward": _plain_loss_backward}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


def work(case):
    op, k = case["op"], case["k"]
    if op == "int8":
        m, n = case["m"], case["n"]
        # (x in 16 bits, the weight in 8, its scales, the result)
        return {"bytes": 2 * m * k + n * k + 4 * n + m * n * (4 if case["out"] == "fp32" else 2), "flops": 2.0 * m * n * k}
    if op == "ffn":
        m, f = case["m"], case["f"]
        return {"bytes": 2 * (m * k + 2 * f * k + m * f * (3 if case["keep"] else 1)), "flops": 4.0 * m * k * f}
    if op == "ffn_backward":
        m, f = case["m"], case["f"]
        return {"bytes": 2 * (2 * m * k + 4 * f * k + 3 * m * f), "flops": 8.0 * m * k * f}
    t, v = case["t"], case["v"]
    if op == "loss":
        return {"bytes": 2 * (t * k + v * k) + 16 * t, "flops": 2.0 * t * k * v}
    return {"bytes": 4 * (t * k + v * k) + 16 * t, "flops": 6.0 * t * k * v}


# ---- the definitions in 64 bits, in rows of at most this many values ------------------------------------------------
_BLOCK = 1 << 28


def exact(case, seed):
    s = prepare(case, seed)
    return {"int8": _exact_int8, "ffn": _exact_ffn, "ffn_backward": _exact_ffn_backward, "loss": _exact_loss,
            "loss_backward": _exact_loss_backward}[case["op"]](s)


def _exact_int8(s):
    weight = (s["w"].to(torch.float64) * s["w_scale"].to(torch.float64)[:, None]).T.contiguous()
    x = s["x"].to(torch.float64)
    # the step of a row is the 32-bit number that the operator hands on
    step = (torch.linalg.vector_norm(x, ord=math.inf, dim=1) / 127).to(torch.float32).to(torch.float64)
    whole = torch.nan_to_num(x / step[:, None]).round()
    return (whole * step[:, None]) @ weight


def _phi(g, activation):
    if activation == "silu":
        return torch.sigmoid(g)
    if activation == "gelu":
        return torch.special.ndtr(g)
    return torch.sigmoid(math.sqrt(8.0 / math.pi) * (g + 0.044715 * g ** 3))   # (1 + tanh(y)) / 2 = sigmoid(2 y)


def _phi_slope(g, activation):
    if activation == "gelu":
        return torch.exp(-g ** 2 / 2) / math.sqrt(2 * math.pi)
    p = _phi(g, activation)
    inner = 1.0 if activation == "silu" else math.sqrt(8.0 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
    return p * (1 - p) * inner


def _exact_ffn(s):
    x = s["x"].to(torch.float64)
    gate = torch.nn.functional.linear(x, s["w_gate"].to(torch.float64))
    up = torch.nn.functional.linear(x, s["w_up"].to(torch.float64))
    h = gate * _phi(gate, s["activation"]) * up
    return (h, gate, up) if s["keep"] else h


def _exact_ffn_backward(s):
    g, u, d = (s[name].to(torch.float64) for name in ("gate", "up", "grad_h"))
    p = _phi(g, s["activation"])
    d_gate = d * u * (p + g * _phi_slope(g, s["activation"]))
    d_up = d * g * p
    both = torch.cat([d_gate, d_up], dim=1)
    weights = torch.cat([s["w_gate"], s["w_up"]]).to(torch.float64)
    grad_weights = torch.mm(both.T.contiguous(), s["x"].to(torch.float64))
    f = g.shape[1]
    return torch.mm(both, weights), grad_weights[:f], grad_weights[f:]


def _exact_loss(s):
    hidden, weight = s["hidden"].to(torch.float64), s["weight"].to(torch.float64)
    target, step = s["target"], max(1, _BLOCK // weight.shape[0])
    loss, lse = [], []
    for at in range(0, hidden.shape[0], step):
        logits = torch.nn.functional.linear(hidden[at:at + step], weight)
        lse.append(torch.logsumexp(logits, dim=1))
        loss.append(torch.nn.functional.nll_loss(torch.log_softmax(logits, dim=1), target[at:at + step], ignore_index=IGNORED, reduction="none"))
    return torch.cat(loss), torch.cat(lse)


def _exact_loss_backward(s):
    hidden, weight = s["hidden"].to(torch.float64), s["weight"].to(torch.float64)
    target, step = s["target"], max(1, _BLOCK // weight.shape[0])
    grad_hidden, grad_weight = torch.zeros_like(hidden), torch.zeros_like(weight)
    for at in range(0, hidden.shape[0], step):
        rows = slice(at, at + step)
        p = torch.softmax(torch.nn.functional.linear(hidden[rows], weight), dim=1)
        has = target[rows] != IGNORED
        line = torch.nonzero(has).squeeze(1)
        p[line, target[rows][line]] -= 1.0
        p *= (s["grad_loss"][rows].to(torch.float64) * has)[:, None]
        grad_hidden[rows] = p @ weight
        grad_weight += p.T.contiguous() @ hidden[rows]
    return grad_hidden, grad_weight
