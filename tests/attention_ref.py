"""Attention from its formula in 64 bits, with bounds on what a kernel may be off, a paged cache to run it on, and the rotation of positions."""

import math

import torch

DEV = "cuda:0"


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def attend(q, k, v, scale, masked=None, weight_step=2.0 ** -15, floor=0.0):
    """q [m, D], k and v [n, D] -> out [m, D], lse [m] in 64 bits, and how far off a result in q's type and an fp32 lse may be.

    A score is a sum of D exact products in fp32, scaled: off by (D + 4) 2^-24 sum|q k| scale at most, which is the relative error of its weight.  A
    weight is off by `weight_step` more (exp2 and its argument, and the weight's own rounding where it is rounded), and by `floor` of the largest
    weight where its type has a smallest number.  Sums over n keys in fp32: n 2^-24.  The result is rounded once."""
    dtype = q.dtype
    q, k, v = q.double(), k.double(), v.double()
    m, d = q.shape
    n = k.shape[0]
    if n == 0:
        return torch.zeros_like(q), torch.full((m,), -math.inf, dtype=torch.float64, device=q.device), torch.zeros_like(q), torch.zeros(m, device=q.device)
    score = q @ k.t().contiguous() * scale
    size = q.abs() @ k.abs().t().contiguous() * abs(scale) * (d + 4) * 2.0 ** -24
    if masked is not None:
        score = score.masked_fill(masked, -math.inf)
        size = size.masked_fill(masked, 0.0)
    lse = torch.logsumexp(score, dim=1)
    p = torch.exp(score - torch.where(lse == -math.inf, torch.zeros_like(lse), lse)[:, None])
    out = p @ v
    # (the weights' relative errors, and that of their sum, which is no larger)
    relative = size.amax(dim=1, keepdim=True) + weight_step + n * 2.0 ** -24
    spread = p @ v.abs()
    largest = p.amax(dim=1, keepdim=True)
    tail = floor * largest * (n * v.abs().amax() + n * out.abs())
    bound = half_step(dtype) * out.abs() + 2.01 * relative * spread + tail + torch.finfo(dtype).tiny * half_step(dtype)
    return out, lse, bound, (relative.squeeze(1) + (1.0 + lse.abs()) * 2.0 ** -22)


def assert_within(got, want, bound, what=""):
    most = torch.finfo(got.dtype).max
    got = got.double()
    # (an infinity is right where the value may be beyond the type's range)
    same = (got == want) | (got.isnan() & want.isnan()) | (got.isinf() & (want.sign() == got.sign()) & (want.abs() + bound > most))
    off = torch.where(same, torch.zeros_like(got), (got - want).abs() - bound)
    assert (off <= 0).all(), f"{what}: {int((off > 0).sum() + off.isnan().sum())} of {off.numel()} beyond, worst by {off.max().item():.3e}"


class Cache:
    """Pages of keys and values whose unused rows hold NaN, in places drawn at random."""

    def __init__(self, lengths, page, kv_heads, d, dtype, layout="heads", extra=2, seed=0, device=DEV, width=None):
        g = torch.Generator().manual_seed(seed)
        need = [max(0, -(-n // page)) for n in lengths]
        total = sum(need) + extra
        shape = (total, kv_heads, page, d) if layout == "heads" else (total, page, kv_heads, d)
        self.key, self.value = (torch.full(shape, math.nan, dtype=dtype, device=device) for _ in range(2))
        if layout == "heads":
            self.key, self.value = self.key.permute(0, 2, 1, 3), self.value.permute(0, 2, 1, 3)
        order = torch.randperm(total, generator=g).to(torch.int32)
        table = torch.full((len(lengths), width if width is not None else max(need + [1])), -7, dtype=torch.int32)
        at = 0
        self.keys, self.values = [], []
        for b, n in enumerate(need):
            table[b, :n] = order[at:at + n]
            at += n
            k, v = (torch.randn(max(lengths[b], 0), kv_heads, d, generator=g).to(dtype).to(device) for _ in range(2))
            self.keys.append(k)
            self.values.append(v)
        self.table = table.to(device)
        self.lengths = torch.tensor(lengths, dtype=torch.int32, device=device)
        self.page = page
        for b, n in enumerate(lengths):
            if n > 0:
                pages, rows = self.places(b, 0, n)
                self.key[pages, rows] = self.keys[b]
                self.value[pages, rows] = self.values[b]

    def places(self, b, first, last):
        position = torch.arange(first, last, device=self.key.device)
        return self.table[b].long()[position // self.page], position % self.page


def decode(q, keys, values, scale=None, **kw):
    """q [sequences, heads, D] over lists of keys and values [n, kv_heads, D]."""
    scale = q.shape[-1] ** -0.5 if scale is None else scale
    out, bound = torch.zeros(q.shape, dtype=torch.float64, device=q.device), torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    for b, (k, v) in enumerate(zip(keys, values)):
        if k.shape[0] == 0:
            continue
        group = q.shape[1] // k.shape[1]
        for j in range(k.shape[1]):
            heads = slice(j * group, (j + 1) * group)
            out[b, heads], _, bound[b, heads], _ = attend(q[b, heads], k[:, j], v[:, j], scale, **kw)
    return out, bound


def rotate(x, position, cos, sin, interleaved):
    """x [tokens, heads, D] turned in 64 bits, and how far off a result in x's type may be: two products and a sum in fp32, one rounding."""
    half = cos.shape[1]
    y = x.double().clone()
    c, s = cos.double()[position][:, None], sin.double()[position][:, None]
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    xa, xb = x[..., a].double(), x[..., b].double()
    y[..., a], y[..., b] = xa * c - xb * s, xa * s + xb * c
    size = torch.zeros_like(y)
    size[..., a], size[..., b] = (xa * c).abs() + (xb * s).abs(), (xa * s).abs() + (xb * c).abs()
    return y, half_step(x.dtype) * y.abs() + 2.0 ** -22 * size + torch.finfo(x.dtype).tiny * half_step(x.dtype)


# ---- gradients without a formula of them: of a loss in 64 bits, by autograd and by differences -------------------------------
def loss(q, k, v, do, lengths, scale, causal):
    """sum(do * attention) over packed sequences, all in 64 bits."""
    total, group, a = 0.0, q.shape[1] // k.shape[1], 0
    for n in lengths:
        masked = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if causal else torch.zeros(n, n, dtype=torch.bool, device=q.device)
        for head in range(q.shape[1]):
            rows, keys = (slice(a, a + n), head), (slice(a, a + n), head // group)
            score = (q[rows] @ k[keys].t().contiguous() * scale).masked_fill(masked, -math.inf)
            total = total + ((torch.softmax(score, 1) @ v[keys]) * do[rows].double()).sum()
        a += n
    return total


def gradients(q, k, v, do, out, lse, lengths, scale, causal):
    """The gradients of `loss` in q, k and v by autograd in 64 bits, and how far off those of a kernel may be that starts from `out` and `lse` as they are
    (rounded, and with the forward pass's errors).

    Of P = exp(s - lse) the relative error is that of its score, of lse, of exp2 and its argument, and one rounding.  Of dS = P (dP - delta) it is that and a
    rounding, and P times the errors of dP and delta: sums of D products in fp32, and what do makes of the error of out.  All that is weighed with
    what it multiplies; sums in fp32 over keys or over a group's rows; one rounding of the result."""
    leaves = [x.double().requires_grad_() for x in (q, k, v)]
    grads = torch.autograd.grad(loss(*leaves, do, lengths, scale, causal), leaves)
    bounds = [torch.zeros_like(x) for x in grads]
    dtype, d, group, step, a = q.dtype, q.shape[-1], q.shape[1] // k.shape[1], half_step(q.dtype), 0
    for n in lengths:
        masked = torch.ones(n, n, dtype=torch.bool, device=q.device).triu(1) if causal else torch.zeros(n, n, dtype=torch.bool, device=q.device)
        for head in range(q.shape[1]):
            rows, keys = (slice(a, a + n), head), (slice(a, a + n), head // group)
            o, l = attend(q[rows], k[keys], v[keys], scale, masked)[:2]
            qd, kd, vd, gd = (x.double() for x in (q[rows], k[keys], v[keys], do[rows]))
            s = qd @ kd.t().contiguous() * scale
            p = torch.exp(s - l[:, None]).masked_fill(masked, 0.0)
            off_p = qd.abs() @ kd.abs().t().contiguous() * abs(scale) * (d + 8) * 2.0 ** -24 + 2.0 ** -20 + (l[:, None].abs() + s.abs()) * 2.0 ** -22
            off_p = off_p + (lse[head, a:a + n].double() - l).abs()[:, None]
            dp, delta = gd @ vd.t().contiguous(), (gd * o).sum(1, keepdim=True)
            off_d = (d + 4) * 2.0 ** -24 * (gd.abs() @ vd.abs().t().contiguous() + (gd * o).abs().sum(1, keepdim=True))
            off_d = off_d + (gd * (out[rows].double() - o)).sum(1, keepdim=True).abs()
            ds = (p * (dp - delta)).abs()
            err = p * off_d + (off_p + step) * ds
            bounds[0][rows] += abs(scale) * ((err + n * 2.0 ** -24 * ds) @ kd.abs())
            bounds[1][keys] += abs(scale) * ((err + n * group * 2.0 ** -24 * ds).t().contiguous() @ qd.abs())
            bounds[2][keys] += ((off_p + step + n * group * 2.0 ** -24) * p).t().contiguous() @ gd.abs()
        a += n
    return grads, [1.02 * e + step * x.abs() + 2 * step * torch.finfo(dtype).tiny for e, x in zip(bounds, grads)]


def assert_slopes(got, q, k, v, do, lengths, scale, causal, bounds, seed=1):
    """Each gradient against differences of `loss` along a way that goes up wherever the gradient does: nothing cancels in their product, so that what is
    allowed is a few hundredths of it, and the differences' own error (of the third order in steps of 10^-4) nothing beside it."""
    g, h = torch.Generator().manual_seed(seed), 1e-4
    inputs = [x.double() for x in (q, k, v)]
    for n, (name, grad, bound) in enumerate(zip(("grad_query", "grad_key", "grad_value"), got, bounds)):
        way = torch.randn(grad.shape, generator=g, dtype=torch.float64).abs().to(grad.device) * grad.double().sign()
        ahead, behind = ([x + (h * way if i == n else 0.0) * sign for i, x in enumerate(inputs)] for sign in (1.0, -1.0))
        slope = ((loss(*ahead, do, lengths, scale, causal) - loss(*behind, do, lengths, scale, causal)) / (2 * h)).item()
        rise, allowed = (grad.double() * way).sum().item(), (bound * way.abs()).sum().item() + 1e-5 * abs(slope)
        assert allowed < 0.1 * rise, f"{name}: {allowed} of {rise} would pass anything"
        assert abs(rise - slope) <= allowed, f"{name}: {rise}, by differences {slope}, allowed {allowed}"
