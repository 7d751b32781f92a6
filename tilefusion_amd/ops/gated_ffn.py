"""The gated feed-forward block, forward and backward (no counterpart in the reference)."""

from typing import Any, Tuple, Union

import torch

from .. import _direct
from ._autograd import not_captured, records, refuse_transforms

__all__ = ["gated_ffn", "gated_ffn_backward"]


def _rows(x: torch.Tensor, width: int, name: str, op: str) -> torch.Tensor:
    if x.dim() < 1 or x.size(-1) != width or width == 0:
        raise RuntimeError(f"{op}: {name} must be [.., {width}], got {list(x.shape)}")
    return x.reshape(-1, width).contiguous()


def _forward(
    x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str, keep: bool
) -> Tuple[torch.Tensor, ...]:
    if w_gate.dim() != 2 or w_up.dim() != 2:
        raise RuntimeError("gated_ffn: w_gate and w_up must be [F, K]")
    rows = _rows(x, w_gate.size(1), "x", "gated_ffn")
    shape = (*x.shape[:-1], w_gate.size(0))
    out = [torch.empty(rows.size(0), shape[-1], dtype=x.dtype, device=x.device) for _ in range(3 if keep else 1)]
    gate, up = (out[1], out[2]) if keep else (None, None)
    torch.ops.tilefusion.gated_ffn(rows, w_gate.contiguous(), w_up.contiguous(), activation, out[0], gate, up)
    return tuple(t.reshape(shape) for t in out)


def _backward(
    grad_h: torch.Tensor,
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    gate: torch.Tensor,
    up: torch.Tensor,
    activation: str,
    of_x: bool,
    of_weights: bool,
) -> Tuple[Any, ...]:
    """The gradients that are asked for, None in the place of the others."""
    if w_gate.dim() != 2 or w_up.dim() != 2:
        raise RuntimeError("gated_ffn_backward: w_gate and w_up must be [F, K]")
    f, k = w_gate.shape
    rows = _rows(x, k, "x", "gated_ffn_backward")
    grad_h, gate, up = (
        _rows(t, f, name, "gated_ffn_backward") for t, name in ((grad_h, "grad_h"), (gate, "gate"), (up, "up"))
    )
    grad_x = torch.empty_like(rows) if of_x else None
    grad_w = torch.empty(2 * f, k, dtype=x.dtype, device=x.device) if of_weights else None
    with torch.no_grad():
        torch.ops.tilefusion.gated_ffn_backward(
            grad_h, rows, w_gate.contiguous(), w_up.contiguous(), gate, up, activation, grad_x, grad_w
        )
    return (
        grad_x.reshape(x.shape) if grad_x is not None else None,
        *((grad_w[:f], grad_w[f:]) if grad_w is not None else (None, None)),
    )


class _GatedFfn(torch.autograd.Function):
    @staticmethod
    def forward(ctx: Any, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str) -> Tuple[torch.Tensor, ...]:
        h, gate, up = _forward(x, w_gate, w_up, activation, True)
        ctx.save_for_backward(x, w_gate, w_up, gate, up)
        ctx.activation = activation
        ctx.mark_non_differentiable(gate, up)
        return h, gate, up

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_h: torch.Tensor, *_: Any) -> Tuple[Any, ...]:
        not_captured("gated_ffn")
        of_x, of_gate, of_up, _ = ctx.needs_input_grad
        return (*_backward(grad_h, *ctx.saved_tensors, ctx.activation, of_x, of_gate or of_up), None)


def gated_ffn(
    x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu", keep: bool = False
) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor, torch.Tensor]]:
    """h = act(x @ w_gate.T) * (x @ w_up.T), both products, the activation and their product in one kernel.

    Args:
        x: [.., K] fp16 or bf16.
        w_gate, w_up: [F, K] of the same type.
        activation: "silu", "gelu" (with erf) or "gelu_tanh".
        keep: also return x @ w_gate.T and x @ w_up.T, rounded to the type, for `gated_ffn_backward`.

    Returns h [.., F], or (h, gate, up).  Everything is fp32 up to h, which is rounded once.  Under autograd h carries the backward
    pass (once: no gradient of a gradient, no forward mode), and gate and up none; neither the call nor that pass is captured into a graph.
    """
    if not torch.compiler.is_compiling():
        direct = _direct.gated_ffn(x, w_gate, w_up, activation, keep)   # (no gradient is asked for)
        if direct is not None:
            return direct if keep else direct[0]
    if records("gated_ffn", x, w_gate, w_up):
        out = _GatedFfn.apply(x, w_gate, w_up, activation)
    else:
        out = _forward(x, w_gate, w_up, activation, keep)
    return out if keep else out[0]


def gated_ffn_backward(
    grad_h: torch.Tensor,
    x: torch.Tensor,
    w_gate: torch.Tensor,
    w_up: torch.Tensor,
    gate: torch.Tensor,
    up: torch.Tensor,
    activation: str = "silu",
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Gradients of x, w_gate and w_up, from that of h [.., F] and the gate and up [.., F] that `gated_ffn` kept.

    The gradients of gate and up are rounded to the type on the way, as operands of the products that follow (in fp16 times a power of two
    where their own range is not the type's, which the products are divided by).  gate and up are taken as they were kept: an up beyond 65504,
    infinite in fp16, makes its gradients so."""
    if not torch.compiler.is_compiling():
        direct = _direct.gated_ffn_backward(grad_h, x, w_gate, w_up, gate, up, activation)
        if direct is not None:
            return direct[0], direct[1][0], direct[1][1]
    refuse_transforms("gated_ffn_backward", grad_h, x, w_gate, w_up, gate, up)
    return _backward(grad_h, x, w_gate, w_up, gate, up, activation, True, True)
