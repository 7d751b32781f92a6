"""Plain 64-bit forms of the operators whose results are more than a product, and how far a result may be from them.

Bounds are per element and come from arithmetic alone.  `half_step(t)` is the largest relative error of one rounding to type t.  A sum of n
products in fp32, in whatever order, is off by at most n * 2^-24 times the sum of the products' magnitudes (n - 1 additions, each rounded
once or less; products of 16-bit numbers are exact in fp32), which `product` gives beside the value.  FN = 2^-20 stands for the functions that
are computed in fp32 (exp, erf, division, a few multiplications: each within 4 of 2^-24, arguments of exp up to 2^4 in size)."""

import math

import torch

FN = 2.0 ** -20
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -133}   # the smallest number of a type


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def product(a, b):
    """a [M, K] @ b [N, K]^T and the bound of its fp32 error."""
    a, b = a.double(), b.double()
    return a @ b.t().contiguous(), a.shape[1] * 2.0 ** -24 * (a.abs() @ b.abs().t().contiguous())


def phi(g, activation):
    if activation == "silu":
        return torch.sigmoid(g)
    if activation == "gelu":
        return torch.special.ndtr(g)
    return torch.sigmoid(math.sqrt(8 / math.pi) * (g + 0.044715 * g ** 3))


def act(g, activation):
    return g * phi(g, activation)


def act_slope(g, activation):
    p = phi(g, activation)
    if activation == "gelu":
        return p + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    inner = 1.0 if activation == "silu" else math.sqrt(8 / math.pi) * (1 + 3 * 0.044715 * g ** 2)
    return p + g * p * (1 - p) * inner


def gated_ffn(x, w_gate, w_up, activation):
    """(h, gate, up) and their bounds for results of x's type."""
    step = half_step(x.dtype)
    gate, d_gate = product(x, w_gate)
    up, d_up = product(x, w_up)
    value = act(gate, activation)
    h = value * up
    # |act'| < 1.13 for each of the three
    d_h = 1.13 * d_gate * (up.abs() + d_up) + value.abs() * d_up + FN * (gate.abs() + d_gate) * (up.abs() + d_up)
    bounds = [d_h + step * (h.abs() + d_h), d_gate + step * (gate.abs() + d_gate), d_up + step * (up.abs() + d_up)]
    return (h, gate, up), [b + TINY[x.dtype] for b in bounds]


def gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up, activation):
    """(grad_x, grad_w_gate, grad_w_up) and their bounds: the gradients of gate and up are rounded to the type on the way."""
    step, tiny = half_step(x.dtype), TINY[x.dtype]
    d, g, u = grad_h.double(), gate.double(), up.double()
    grad_gate, grad_up = d * u * act_slope(g, activation), d * act(g, activation)
    # the slope is a sum of terms of magnitude up to 1 + |g|
    off_gate = FN * (d * u).abs() * (1 + g.abs()) + step * grad_gate.abs() + tiny
    off_up = FN * (d * g).abs() + step * grad_up.abs() + tiny
    return _products([(torch.cat([grad_gate, grad_up], 1), torch.cat([off_gate, off_up], 1), torch.cat([w_gate, w_up]).t()),
                      (grad_gate.t(), off_gate.t(), x.t()), (grad_up.t(), off_up.t(), x.t())], x.dtype)


def _products(pairs, dtype):
    """For (a, bound of a, b): a @ b^T rounded to dtype, and its bound."""
    values, bounds = [], []
    for a, off, b in pairs:
        a, off, b = a.contiguous(), off.contiguous(), b.double().contiguous()
        bt = b.t().contiguous()
        value = a @ bt
        most = (a.abs() + off) @ bt.abs()
        bound = off @ bt.abs() + a.shape[1] * 2.0 ** -24 * most
        values.append(value)
        bounds.append(bound + half_step(dtype) * (value.abs() + bound) + TINY[dtype])
    return values, bounds


def linear_cross_entropy(hidden, weight, target, ignore_index):
    """(loss, lse) and their bounds, in fp32."""
    z, off = product(hidden, weight)
    lse = torch.logsumexp(z, dim=1)
    valid = target != ignore_index
    at_target = z.gather(1, torch.where(valid, target, 0)[:, None]).squeeze(1)
    loss = torch.where(valid, lse - at_target, torch.zeros_like(lse))
    # a shift of every logit by at most `worst` shifts lse by as much; sums of exp in fp32: V terms in a tree of far less depth than 2^4 a level
    worst = off.amax(dim=1)
    d_lse = worst + FN * (1 + lse.abs())
    return (loss, lse), [torch.where(valid, d_lse + worst + 2.0 ** -24 * loss.abs(), torch.zeros_like(lse)), d_lse]


def linear_cross_entropy_backward(grad_loss, hidden, weight, target, ignore_index):
    """(grad_hidden, grad_weight) and their bounds: softmax gradients are rounded to the type, relative to the largest |grad_loss|, and so
    are the rows of hidden times what grad_loss is more than a power of two, m in (0.5, 1]."""
    dtype = hidden.dtype
    z, off = product(hidden, weight)
    lse = torch.logsumexp(z, dim=1, keepdim=True)
    p = torch.exp(z - lse)
    # the logit's error, that of lse as it was handed over (fp32, from a forward pass), and that of exp
    far = off + off.amax(dim=1, keepdim=True) + FN * (1 + lse.abs()) + FN * (1 + (z - lse).abs())
    off_p = p * far * 2
    valid = (target != ignore_index).double()[:, None]
    one = torch.nn.functional.one_hot(torch.where(target != ignore_index, target, 0), weight.shape[0]).double()
    g = grad_loss.double()[:, None] * valid
    signed = (p - one) * g
    top = g.abs().max()
    # rounded to the type; fp16 holds them times 2^14 relative to at least the largest |grad_loss|
    # (and four roundings in fp32: grad_loss divided by a number, the power of two times the softmax gradient, the factor of the row, the sum times it)
    off_p = off_p * g.abs() + (half_step(dtype) + 2.0 ** -22) * signed.abs() + (2.0 ** -38 * 2 * top if dtype == torch.float16 else 2.0 ** -120 * top)
    off_p = torch.where(valid.bool(), off_p, torch.zeros_like(off_p))
    off_w = off_p + half_step(dtype) * (signed.abs() + off_p)   # m * hidden, rounded
    values, bounds = _products([(signed, off_p, weight.t()), (signed.t(), off_w.t(), hidden.t())], dtype)
    # m * hidden below the normal numbers is off by TINY / 2; what it is multiplied by is signed / m, less than twice as much
    bounds[1] = bounds[1] + TINY[dtype] * signed.abs().sum(0)[:, None]
    return values, bounds


def assert_within(got, want, bound, what=""):
    """Returns where the result is a number: what may lie beyond the type's largest one may be that infinity, and nothing else may."""
    largest = torch.finfo(got.dtype).max
    got = got.double()
    assert got.shape == want.shape, f"{what}: shape {tuple(got.shape)}, not {tuple(want.shape)}"
    finite = torch.isfinite(got)
    beyond = want.abs() + bound > largest
    assert (finite | (beyond & (got == torch.sign(want) * float("inf")))).all(), f"{what}: not finite"
    assert (~finite | (want.abs() - bound <= largest)).all(), f"{what}: finite"
    over = torch.where(finite, (got - want).abs() - bound, torch.zeros_like(want))
    if (over > 0).any():
        at = int(over.argmax())
        raise AssertionError(f"{what}: {int((over > 0).sum())} of {got.numel()} out of bounds; element {at}: {got.flatten()[at]:.9g}, "
                             f"not {want.flatten()[at]:.9g} +- {bound.flatten()[at]:.3g}")
    return finite
