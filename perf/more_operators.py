"""Attention as a program with sequences of different lengths meets it: keys and values appended to a paged cache with the
position rotation on the way, one new token over that cache, and packed prompts, forward and backward.

A case is a dict of plain values; `op` says which operator it measures.  `listed()` names twelve of them, `draw()` gives further ones
of the same ranges.  `run` computes them from elementary operations in 32 bits, or, where `own` is true, through tilefusion_amd.ops.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}

# Bounds of a drawn case, so that none costs more than the largest listed ones.
MAX_APPEND_ROWS = 8191 * 32
MAX_CACHE_BYTES = 4.0 * 16 * 8 * 32768 * 128
MAX_PACKED_FLOPS = 4.0 * 32 * 128 * 8192 * 8193 / 2
MAX_BACKWARD_FLOPS = 10.0 * 32 * 128 * 4 * 2048 * 2049 / 2


def listed():
    return [
        # One step of 64 conversations: a new token each, latency and nothing else.
        {"name": "append_step", "op": "append", "batch": 64, "shortest": 60, "longest": 2048, "new": 1, "heads": 32, "kv_heads": 8, "d": 128,
         "rotated": 128, "interleaved": False, "page": 16, "layout": "heads", "dtype": "bf16", "keep": False},
        # Prompts of different lengths enter the cache; half of a head is rotated, in neighbouring pairs, and the keys stay for the attention.
        {"name": "append_prompts", "op": "append", "batch": 9, "shortest": 77, "longest": 2999, "new": 0, "heads": 32, "kv_heads": 8, "d": 128,
         "rotated": 64, "interleaved": True, "page": 64, "layout": "tokens", "dtype": "fp16", "keep": True},
        # One conversation: the smallest call over a cache.
        {"name": "decode_one", "op": "decode", "batch": 1, "shortest": 1999, "longest": 1999, "idle": 0, "heads": 32, "kv_heads": 8, "d": 128,
         "page": 16, "layout": "heads", "dtype": "bf16"},
        # A busy server: conversations from their start to far on, slots without any, pages with the tokens' heads side by side.
        {"name": "decode_ragged", "op": "decode", "batch": 60, "shortest": 17, "longest": 8001, "idle": 4, "heads": 24, "kv_heads": 8, "d": 64,
         "page": 16, "layout": "tokens", "dtype": "fp16"},
        # All query heads share one head of keys.
        {"name": "decode_one_kv_head", "op": "decode", "batch": 128, "shortest": 500, "longest": 5000, "idle": 0, "heads": 16, "kv_heads": 1, "d": 128,
         "page": 32, "layout": "heads", "dtype": "bf16"},
        # The lengths of the repository's decoding benchmark with grouped heads: 2 GiB of pages, the largest call.
        {"name": "decode_32768", "op": "decode", "batch": 16, "shortest": 32768, "longest": 32768, "idle": 0, "heads": 32, "kv_heads": 8, "d": 128,
         "page": 64, "layout": "heads", "dtype": "fp16"},
        # Short texts, packed without padding.
        {"name": "packed_short", "op": "packed", "batch": 37, "shortest": 1, "longest": 300, "past": 0, "causal": True, "heads": 16, "kv_heads": 4,
         "d": 64, "dtype": "fp16", "keep": False},
        # A training step's forward pass over texts of all lengths.
        {"name": "packed_ragged", "op": "packed", "batch": 14, "shortest": 64, "longest": 4001, "past": 0, "causal": True, "heads": 32, "kv_heads": 8,
         "d": 128, "dtype": "bf16", "keep": True},
        # A long prompt.
        {"name": "packed_prompt", "op": "packed", "batch": 1, "shortest": 8192, "longest": 8192, "past": 0, "causal": True, "heads": 32, "kv_heads": 8,
         "d": 128, "dtype": "bf16", "keep": False},
        # The next pieces of prompts of which much has been seen.
        {"name": "packed_chunks", "op": "packed", "batch": 4, "shortest": 100, "longest": 512, "past": 6000, "causal": True, "heads": 32, "kv_heads": 4,
         "d": 128, "dtype": "bf16", "keep": False},
        # Gradients of fine-tuning on short texts.
        {"name": "backward_ragged", "op": "backward", "batch": 11, "shortest": 30, "longest": 1001, "past": 0, "causal": True, "heads": 16, "kv_heads": 4,
         "d": 64, "dtype": "fp16"},
        # Gradients of a training step at full size.
        {"name": "backward_large", "op": "backward", "batch": 4, "shortest": 2048, "longest": 2048, "past": 0, "causal": True, "heads": 32,
         "kv_heads": 8, "d": 128, "dtype": "bf16"},
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "decode", "decode", "packed", "packed", "backward"])
    while True:
        d = rng.choice([64, 128, 128])
        kv_heads = rng.choice([1, 2, 4, 8, 8])
        heads = kv_heads * rng.choice([1, 2, 3, 4, 4, 6, 8])
        case = {"op": op, "heads": heads, "kv_heads": kv_heads, "d": d, "dtype": rng.choice(["fp16", "bf16"])}
        if op == "append":
            case.update(batch=_log_int(rng, 1, 256), rotated=rng.choice([d, d, d // 2]), interleaved=rng.random() < 0.5,
                        page=rng.choice([16, 16, 32, 64, 128]), layout=rng.choice(["heads", "tokens"]), keep=rng.random() < 0.5)
            if rng.random() < 0.5:
                case.update(new=1, shortest=_log_int(rng, 1, 100), longest=_log_int(rng, 100, 4000))
            else:
                case.update(new=0, shortest=_log_int(rng, 1, 100), longest=_log_int(rng, 100, 8000))
            new = sum(_new(case))
            if new * heads <= MAX_APPEND_ROWS and _cache_bytes(case) <= MAX_CACHE_BYTES / 2:
                return case
        elif op == "decode":
            case.update(batch=_log_int(rng, 1, 512), idle=rng.choice([0, 0, 1, 5]), shortest=_log_int(rng, 1, 1000), longest=_log_int(rng, 1000, 60000),
                        page=rng.choice([16, 16, 32, 64, 128]), layout=rng.choice(["heads", "heads", "tokens"]))
            if _cache_bytes(case) <= MAX_CACHE_BYTES:
                return case
        else:
            case.update(batch=_log_int(rng, 1, 64), shortest=_log_int(rng, 1, 500), longest=_log_int(rng, 500, 8000),
                        past=rng.choice([0, 0, 0, _log_int(rng, 1, 8000)]), causal=rng.random() < 0.75)
            if op == "packed":
                case["keep"] = rng.random() < 0.4
            # (the plain form takes all pairs of a sequence, allowed or not)
            pairs = sum(n * (n + case["past"]) for n in _lengths(case))
            per_pair = (4.0 if op == "packed" else 10.0) * heads * d
            if pairs * per_pair <= 2 * (MAX_PACKED_FLOPS if op == "packed" else MAX_BACKWARD_FLOPS) and \
                    work(case)["flops"] <= (MAX_PACKED_FLOPS if op == "packed" else MAX_BACKWARD_FLOPS):
                return case


# ---- the lengths of a case's sequences: spread over their logarithm, in no order ------------------------------------------
def _lengths(case):
    low, high = case["shortest"], case["longest"]
    spread = [(0.5 + i * 0.6180339887498949) % 1.0 for i in range(case["batch"])]
    return [min(high, max(low, int(round(low * (high / low) ** s)))) for s in spread] + [0] * case.get("idle", 0)


def _new(case):
    """New tokens of each sequence: one, or the whole prompt."""
    return [n if case["new"] == 0 else min(n, case["new"]) for n in _lengths(case)]


def _pages(case):
    return [-(-n // case["page"]) for n in _lengths(case)]


def _cache_bytes(case):
    return 4.0 * sum(_pages(case)) * case["page"] * case["kv_heads"] * case["d"]


def _offsets(lengths):
    out = [0]
    for n in lengths:
        out.append(out[-1] + n)
    return torch.tensor(out, dtype=torch.int32, device=DEVICE)


def _randn(g, *shape, dtype):
    return torch.randn(*shape, device=DEVICE, dtype=dtype, generator=g)


def _cache(case, g, dtype):
    """Keys, values [pages, page, kv_heads, d] of all sequences, their pages in no order, and some that belong to nobody."""
    pages = _pages(case)
    total, page, hkv, d = sum(pages) + 3, case["page"], case["kv_heads"], case["d"]
    if case["layout"] == "heads":
        key, value = (_randn(g, total, hkv, page, d, dtype=dtype).permute(0, 2, 1, 3) for _ in range(2))
    else:
        key, value = (_randn(g, total, page, hkv, d, dtype=dtype) for _ in range(2))
    order = torch.randperm(total, device=DEVICE, generator=g).to(torch.int32)
    table = torch.full((len(pages), max(pages)), -1, dtype=torch.int32, device=DEVICE)
    at = 0
    for i, n in enumerate(pages):
        table[i, :n] = order[at:at + n]
        at += n
    return key, value, table, torch.tensor(_lengths(case), dtype=torch.int32, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    op, dtype, h, hkv, d = case["op"], DTYPES[case["dtype"]], case["heads"], case["kv_heads"], case["d"]
    if op in ("append", "decode"):
        key, value, table, lengths = _cache(case, g, dtype)
        state = {"op": op, "key_cache": key, "value_cache": value, "table": table, "lengths": lengths, "dense": _lengths(case)}
        if op == "decode":
            return {**state, "query": _randn(g, lengths.numel(), h, d, dtype=dtype)}
        new = _new(case)
        # the tables of a model's longest text, made once
        angle = torch.arange(2 * case["longest"], device=DEVICE, dtype=torch.float64)[:, None] * \
            10000.0 ** (-torch.arange(0, case["rotated"], 2, device=DEVICE, dtype=torch.float64) / case["rotated"])
        # queries, keys and values leave one projection side by side
        qkv = _randn(g, sum(new), (h + 2 * hkv) * d, dtype=dtype)
        q, k, v = qkv.split([h * d, hkv * d, hkv * d], dim=1)
        return {**state, "new": new, "offsets": None if case["new"] == 1 else _offsets(new), "cos": angle.cos().float(), "sin": angle.sin().float(),
                "query": q.unflatten(1, (h, d)), "key": k.unflatten(1, (hkv, d)), "value": v.unflatten(1, (hkv, d)),
                "interleaved": case["interleaved"], "keep": case["keep"]}
    lq = _lengths(case)
    lkv = [n + case["past"] for n in lq]
    state = {"op": op, "causal": case["causal"], "scale": d ** -0.5, "lq": lq, "lkv": lkv, "offsets": _offsets(lq),
             "kv_offsets": _offsets(lkv) if case["past"] else None, "query": _randn(g, sum(lq), h, d, dtype=dtype),
             "key": _randn(g, sum(lkv), hkv, d, dtype=dtype), "value": _randn(g, sum(lkv), hkv, d, dtype=dtype)}
    if op == "packed":
        return {**state, "keep": case["keep"]}
    # as the forward pass returned them
    out, lse = _plain_packed({**state, "keep": True})
    return {**state, "out": out, "lse": lse, "grad_out": _randn(g, sum(lq), h, d, dtype=dtype)}


# ---- the plain forms ------------------------------------------------------------------------------------------------
def _places(s, sequence, position):
    """Page and row of tokens in the cache."""
    page = s["key_cache"].shape[1]
    return s["table"][sequence, position // page].long(), position % page


def _plain_append(s):
    new = torch.tensor(s["new"], device=DEVICE)
    sequence = torch.repeat_interleave(torch.arange(len(s["new"]), device=DEVICE), new)
    first = torch.cumsum(new, 0) - new
    position = torch.arange(sequence.numel(), device=DEVICE) - first[sequence] + (s["lengths"].long() - new)[sequence]
    cos, sin = s["cos"][position].unsqueeze(1), s["sin"][position].unsqueeze(1)
    half = cos.shape[-1]

    def rotate(x):
        out = x.float()
        a, b = (out[..., 0:2 * half:2], out[..., 1:2 * half:2]) if s["interleaved"] else (out[..., :half], out[..., half:2 * half])
        ra, rb = a * cos - b * sin, a * sin + b * cos
        rotated = torch.stack([ra, rb], dim=-1).flatten(-2) if s["interleaved"] else torch.cat([ra, rb], dim=-1)
        return torch.cat([rotated, out[..., 2 * half:]], dim=-1).to(x.dtype)

    query, key = rotate(s["query"]), rotate(s["key"])
    page, row = _places(s, sequence, position)
    s["key_cache"][page, row] = key
    s["value_cache"][page, row] = s["value"]
    return (query, s["key_cache"], s["value_cache"]) + ((key,) if s["keep"] else ())


_BLOCK = 1 << 28   # elements of a cache that are gathered at a time


def _plain_decode(s):
    q, lengths = s["query"].float(), s["lengths"].long()
    hkv, d = s["key_cache"].shape[2:]
    longest = max(s["dense"])
    step = max(1, _BLOCK // (longest * hkv * d))
    position = torch.arange(longest, device=DEVICE)
    out = torch.empty_like(s["query"])
    for at in range(0, q.shape[0], step):
        rows = slice(at, at + step)
        n = lengths[rows]
        inside = position[None, :] < n[:, None]
        sequence = torch.arange(at, at + n.numel(), device=DEVICE)[:, None].expand_as(inside)
        page, row = _places(s, sequence, position[None, :].expand_as(inside))
        page = torch.where(inside, page, torch.zeros_like(page))
        keep = inside[:, None, :, None]
        k = s["key_cache"][page, row].transpose(1, 2).float().masked_fill(~keep, 0.0)   # [b, kv_heads, longest, d]
        qg = q[rows].unflatten(1, (hkv, -1))
        score = (qg @ k.transpose(2, 3).contiguous()) * d ** -0.5
        score = score.masked_fill(~inside[:, None, None, :], -math.inf)
        top = score.amax(dim=-1, keepdim=True)
        p = torch.exp(score - torch.where(top == -math.inf, torch.zeros_like(top), top))
        del score, k
        total = p.sum(dim=-1, keepdim=True)
        v = s["value_cache"][page, row].transpose(1, 2).float().masked_fill(~keep, 0.0)
        o = (p @ v) / torch.where(total == 0, torch.ones_like(total), total)
        out[rows] = o.flatten(1, 2).to(out.dtype)
    return out


def _pieces(s, hkv):
    """Every sequence and head of keys: rows of queries, rows of keys, the head, and the pairs that are masked."""
    q0 = k0 = 0
    for lq, lkv in zip(s["lq"], s["lkv"]):
        masked = None
        if s["causal"]:
            masked = torch.arange(lkv, device=DEVICE)[None, :] > torch.arange(lq, device=DEVICE)[:, None] + (lkv - lq)
        for j in range(hkv):
            yield slice(q0, q0 + lq), slice(k0, k0 + lkv), j, masked
        q0, k0 = q0 + lq, k0 + lkv


def _plain_packed(s):
    hkv = s["key"].shape[1]
    group = s["query"].shape[1] // hkv
    out = torch.empty_like(s["query"])
    lse = torch.empty(s["query"].shape[1], s["query"].shape[0], device=DEVICE)
    for rows, keys, j, masked in _pieces(s, hkv):
        heads = slice(j * group, (j + 1) * group)
        q = s["query"][rows, heads].float().transpose(0, 1).contiguous()
        k, v = s["key"][keys, j].float(), s["value"][keys, j].float()
        score = (q @ k.t()) * s["scale"]
        if masked is not None:
            score = score.masked_fill(masked, -math.inf)
        top = score.amax(dim=-1, keepdim=True)
        p = torch.exp(score - top)
        total = p.sum(dim=-1, keepdim=True)
        out[rows, heads] = ((p @ v) / total).transpose(0, 1).to(out.dtype)
        lse[heads, rows] = (top + torch.log(total)).squeeze(-1)
    return (out, lse) if s["keep"] else out


def _plain_backward(s):
    hkv = s["key"].shape[1]
    group = s["query"].shape[1] // hkv
    grad_q, grad_k, grad_v = (torch.empty_like(s[name]) for name in ("query", "key", "value"))
    for rows, keys, j, masked in _pieces(s, hkv):
        heads = slice(j * group, (j + 1) * group)
        q, o, do = (s[name][rows, heads].float().transpose(0, 1).contiguous() for name in ("query", "out", "grad_out"))
        k, v = s["key"][keys, j].float(), s["value"][keys, j].float()
        p = torch.exp((q @ k.t()) * s["scale"] - s["lse"][heads, rows].unsqueeze(-1))
        if masked is not None:
            p = p.masked_fill(masked, 0.0)
        grad_v[keys, j] = (p.flatten(0, 1).t() @ do.flatten(0, 1)).to(grad_v.dtype)
        ds = p * (do @ v.t() - (do * o).sum(dim=-1, keepdim=True)) * s["scale"]
        del p
        grad_q[rows, heads] = (ds @ k).transpose(0, 1).to(grad_q.dtype)
        grad_k[keys, j] = (ds.flatten(0, 1).t() @ q.flatten(0, 1)).to(grad_k.dtype)
    return grad_q, grad_k, grad_v


def _own(s):
    from tilefusion_amd import ops

    op = s["op"]
    if op == "append":
        out = ops.append_paged_kv(s["query"], s["key"], s["value"], s["cos"], s["sin"], s["key_cache"], s["value_cache"], s["table"], s["lengths"],
                                  s["offsets"], s["interleaved"], s["keep"])
        query, key = out if s["keep"] else (out, None)
        return (query, s["key_cache"], s["value_cache"]) + ((key,) if s["keep"] else ())
    if op == "decode":
        return ops.flash_decode_paged(s["query"], s["key_cache"], s["value_cache"], s["table"], s["lengths"])
    if op == "packed":
        return ops.flash_attention_packed(s["query"], s["key"], s["value"], s["offsets"], s["kv_offsets"], s["scale"], s["causal"], s["keep"])
    return ops.flash_attention_packed_backward(s["grad_out"], s["query"], s["key"], s["value"], s["out"], s["lse"], s["offsets"], s["kv_offsets"],
                                               s["scale"], s["causal"])


_PLAIN = {"append": _plain_append, "decode": _plain_decode, "packed": _plain_packed, "backward": _plain_backward}


def run(state):
    if own:
        return _own(state)
    return _PLAIN[state["op"]](state)


def work(case):
    op, h, hkv, d = case["op"], case["heads"], case["kv_heads"], case["d"]
    lengths = _lengths(case)
    if op == "append":
        new = sum(_new(case))
        # queries, keys and values in, the same out, the keys twice where they stay; a position's row of the tables once
        positions = max(lengths) if case["new"] == 0 else min(len(lengths), max(lengths))
        return {"bytes": 2 * new * d * (2 * h + 4 * hkv + (hkv if case["keep"] else 0)) + 4 * case["rotated"] * positions,
                "flops": 3.0 * new * (h + hkv) * case["rotated"]}
    if op == "decode":
        # every key and value of the sequences once
        return {"bytes": 4 * d * hkv * sum(lengths) + 4 * d * h * len(lengths), "flops": 4.0 * d * h * sum(lengths)}
    past = case["past"]
    pairs = sum(n * past + n * (n + 1) // 2 for n in lengths) if case["causal"] else sum(n * (n + past) for n in lengths)
    t, u = sum(lengths), sum(n + past for n in lengths)
    if op == "packed":
        return {"bytes": 4 * d * (h * t + hkv * u) + (4 * h * t if case["keep"] else 0), "flops": 4.0 * h * d * pairs}
    return {"bytes": 2 * d * (4 * h * t + 4 * hkv * u) + 4 * h * t, "flops": 10.0 * h * d * pairs}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "decode": _exact_decode, "packed": _exact_packed, "backward": _exact_backward}[case["op"]](s)


def _turned(x, cos, sin, interleaved):
    """x [n, heads, d] as complex numbers, times cos + i sin."""
    x, r = x.to(torch.float64), 2 * cos.shape[1]
    turn = torch.complex(cos.to(torch.float64), sin.to(torch.float64))[:, None]
    if interleaved:
        z = torch.view_as_complex(x[..., :r].unflatten(-1, (-1, 2)).contiguous()) * turn
        return torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], dim=-1)
    z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * turn
    return torch.cat([z.real, z.imag, x[..., r:]], dim=-1)


def _exact_append(s):
    key_cache, value_cache = s["key_cache"].to(torch.float64), s["value_cache"].to(torch.float64)
    page, query, key, at = key_cache.shape[1], [], [], 0
    table = s["table"].tolist()
    for b, (new, length) in enumerate(zip(s["new"], s["dense"])):
        where, tokens = slice(length - new, length), slice(at, at + new)
        query.append(_turned(s["query"][tokens], s["cos"][where], s["sin"][where], s["interleaved"]))
        key.append(_turned(s["key"][tokens], s["cos"][where], s["sin"][where], s["interleaved"]))
        spot = torch.tensor([table[b][p // page] * page + p % page for p in range(length - new, length)], device=DEVICE)
        for cache, rows in ((key_cache, key[-1]), (value_cache, s["value"][tokens].to(torch.float64))):
            cache[spot // page, spot % page] = rows
        at += new
    return (torch.cat(query), key_cache, value_cache) + ((torch.cat(key),) if s["keep"] else ())


def _exact_decode(s):
    hkv, d = s["key_cache"].shape[2:]
    page, out = s["key_cache"].shape[1], []
    for b, length in enumerate(s["dense"]):
        pages = s["table"][b, :-(-length // page)].long()
        k, v = (s[name][pages].flatten(0, 1)[:length].to(torch.float64) for name in ("key_cache", "value_cache"))   # [length, kv_heads, d]
        q = s["query"][b].to(torch.float64).unflatten(0, (hkv, -1))
        p = torch.softmax(torch.matmul(q, k.permute(1, 2, 0).contiguous()) / math.sqrt(d), dim=-1)
        out.append(torch.matmul(p, v.permute(1, 0, 2).contiguous()).flatten(0, 1) if length else torch.zeros_like(s["query"][b], dtype=torch.float64))
    return torch.stack(out)


def _ranges(lengths):
    ends = torch.tensor(lengths).cumsum(0).tolist()
    return [(end - n, end) for n, end in zip(lengths, ends)]


def _exact_scores(s, q, k):
    score = torch.matmul(q, k.T.contiguous()) * s["scale"]
    if s["causal"]:
        score += torch.full(score.shape, -math.inf, dtype=torch.float64, device=DEVICE).triu(1 + k.shape[0] - q.shape[0])
    return score


def _exact_packed(s):
    out = s["query"].to(torch.float64)
    h, group = out.shape[1], out.shape[1] // s["key"].shape[1]
    lse = torch.empty(h, out.shape[0], dtype=torch.float64, device=DEVICE)
    for (qa, qb), (ka, kb) in zip(_ranges(s["lq"]), _ranges(s["lkv"])):
        for head in range(h):
            k, v = (s[name][ka:kb, head // group].to(torch.float64) for name in ("key", "value"))
            score = _exact_scores(s, out[qa:qb, head], k)
            lse[head, qa:qb] = torch.logsumexp(score, dim=1)
            out[qa:qb, head] = torch.softmax(score, dim=1) @ v
    return (out, lse) if s["keep"] else out


def _exact_backward(s):
    q, k, v, o, do = (s[name].to(torch.float64) for name in ("query", "key", "value", "out", "grad_out"))
    grads = tuple(torch.zeros_like(x) for x in (q, k, v))
    group = q.shape[1] // k.shape[1]
    for (qa, qb), (ka, kb) in zip(_ranges(s["lq"]), _ranges(s["lkv"])):
        for head in range(q.shape[1]):
            rows, keys = (slice(qa, qb), head), (slice(ka, kb), head // group)
            p = (_exact_scores(s, q[rows], k[keys]) - s["lse"][head, qa:qb].to(torch.float64)[:, None]).exp()
            slope = p * (torch.matmul(do[rows], v[keys].T.contiguous()) - torch.linalg.vecdot(do[rows], o[rows])[:, None])
            grads[0][rows] = s["scale"] * torch.matmul(slope, k[keys])
            grads[1][keys] += s["scale"] * torch.matmul(slope.T.contiguous(), q[rows])
            grads[2][keys] += torch.matmul(p.T.contiguous(), do[rows])
    return grads
