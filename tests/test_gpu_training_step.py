"""The operators as a program uses them together: a training step of the position-wise half of a layer and the head (gated_ffn, the
framework's gemm as the down projection, linear_cross_entropy, and back), and the same layer served with its down projection in 8 bits."""

import pytest
import torch

from tests import product_ref as ref
from tilefusion_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _tile(n):
    return next(t for t in (64, 32, 16, 8, 4, 2, 1) if n % t == 0)


def _linear(x, w):
    """x @ w.T through the framework's gemm."""
    out = torch.empty(x.shape[0], w.shape[0], device=x.device, dtype=x.dtype)
    ops.gemm(x, w, out, _tile(x.shape[0]), _tile(w.shape[0]), _tile(x.shape[1]), 2, 1)
    return out


def _model(dtype, t=330, k=136, f=264, v=1003, seed=0):
    g = torch.Generator(device=DEV).manual_seed(seed)
    def make(*s, scale):
        return (torch.randn(*s, device=DEV, generator=g) * scale).to(dtype)
    x = make(t, k, scale=1.0)
    w = {"gate": make(f, k, scale=k ** -0.5), "up": make(f, k, scale=k ** -0.5), "down": make(k, f, scale=2 * f ** -0.5), "head": make(v, k, scale=2 * k ** -0.5)}
    target = torch.randint(0, v, (t,), device=DEV, generator=g)
    target[: t // 5] = -100
    return x, w, target


def _step(x, w, target, scale):
    """Loss and gradients, call by call."""
    valid = (target != -100).sum()
    h, gate, up = ops.gated_ffn(x, w["gate"], w["up"], keep=True)
    y = _linear(h, w["down"])
    loss, lse = ops.linear_cross_entropy(y, w["head"], target)
    grad_loss = (scale / valid).expand(x.shape[0])
    grad_y, grad_head = ops.linear_cross_entropy_backward(grad_loss, y, w["head"], target, lse)
    grad_down = _linear(_padded(grad_y.t()), _padded(h.t()))
    grad_h = _linear(grad_y, w["down"].t().contiguous())
    grad_x, grad_gate, grad_up = ops.gated_ffn_backward(grad_h, x, w["gate"], w["up"], gate, up)
    return loss.sum() / valid, grad_x, grad_gate, grad_up, grad_down, grad_head


def _padded(a):
    """Rows completed by zeros to what gemm sums over, a multiple of 8."""
    return torch.nn.functional.pad(a, (0, -a.shape[1] % 8)).contiguous()


def _plain_step(x, w, target, scale):
    leaves = {n: a.double().requires_grad_() for n, a in {"x": x, **w}.items()}
    h = ref.act(leaves["x"] @ leaves["gate"].t(), "silu") * (leaves["x"] @ leaves["up"].t())
    loss = torch.nn.functional.cross_entropy(h @ leaves["down"].t() @ leaves["head"].t(), target)
    (loss * scale).backward()
    return loss.detach(), *(leaves[n].grad for n in ("x", "gate", "up", "down", "head"))


@pytest.mark.parametrize("dtype,scale", [(torch.float16, 1024.0), (torch.bfloat16, 1.0)])
@pytest.mark.parametrize("t", [1, 64, 330, 1025])
def test_step(dtype, scale, t):
    x, w, target = _model(dtype, t=t)
    got, want = _step(x, w, target, scale), _plain_step(x, w, target, scale)
    # Roundings to 16 bits between x and a gradient: h, y, P, grad_y, grad_h, gate, up, grad_gate or grad_up, the result: at most ten, each
    # relative to a value of which the gradient is a sum of products; a factor 4 for what differences (p - 1, the slope) enlarge.
    assert abs(got[0].double() - want[0]) <= 40 * ref.half_step(dtype) * want[0]
    for a, b in zip(got[1:], want[1:]):
        assert (a.double() - b).norm() <= 40 * ref.half_step(dtype) * b.norm()


def test_step_with_autograd_and_replayed():
    x, w, target = _model(torch.bfloat16)
    want = [a.clone() for a in _step(x, w, target, 1.0)]
    leaves = {n: a.clone().requires_grad_() for n, a in w.items()}
    h = ops.gated_ffn(x, leaves["gate"], leaves["up"])
    y = torch.nn.functional.linear(h, leaves["down"])
    loss, _ = ops.linear_cross_entropy(y, leaves["head"], target)
    (loss.sum() / (target != -100).sum()).backward()
    # (the projection between them is another kernel's: its roundings may differ)
    for n, b in zip(("gate", "up", "down", "head"), want[2:]):
        a = leaves[n].grad
        assert (a.double() - b.double()).norm() <= 8 * ref.half_step(torch.bfloat16) * b.double().norm()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = _step(x, w, target, 1.0)
    for n in range(4):
        want = [a.clone() for a in _step(x, w, target, 1.0)]
        for a in out:
            a.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), n
        for a, d in zip((w["gate"], w["up"], w["down"], w["head"]), want[2:]):
            a.sub_(d)


@pytest.mark.parametrize("t", [1, 5, 200])
def test_served_with_an_8_bit_projection(t):
    x, w, target = _model(torch.bfloat16, t=t)
    q_down, s_down = ops.quantize_rows(w["down"])
    h = ops.gated_ffn(x, w["gate"], w["up"])
    q, s = ops.quantize_rows(h)
    y = torch.empty(t, w["down"].shape[0], device=DEV, dtype=torch.bfloat16)
    ops.gemm_int8(q, q_down, s, s_down, y)
    # (whole numbers first: a sum that is zero has to be zero)
    want = (q.double() @ q_down.double().t().contiguous()) * s.double()[:, None] * s_down.double()
    assert ((y.double() - want).abs() <= want.abs() * (ref.half_step(torch.bfloat16) + 2.0 ** -21) + 2.0 ** -130).all()
    # half a step of either operand, each off by chance
    full = h.double() @ w["down"].double().t().contiguous()
    step = (s.double()[:, None] ** 2 / 12 * (w["down"].double() ** 2).sum(1) + s_down.double() ** 2 / 12 * (h.double() ** 2).sum(1)[:, None]).sqrt()
    assert (want - full).norm() <= 2 * step.norm()
    loss, lse = ops.linear_cross_entropy(y, w["head"], target)
    (want_loss, want_lse), bounds = ref.linear_cross_entropy(y, w["head"], target, -100)
    ref.assert_within(loss, want_loss, bounds[0])
    ref.assert_within(lse, want_lse, bounds[1])
