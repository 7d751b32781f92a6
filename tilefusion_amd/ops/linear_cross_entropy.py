"""Softmax cross entropy of a linear head without its logits, forward and backward (no counterpart in the reference)."""

from typing import Any, Tuple

import torch

from .. import _direct
from ._autograd import not_captured, records, refuse_transforms

__all__ = ["linear_cross_entropy", "linear_cross_entropy_backward"]


def _operands(
    hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, op: str
) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    if weight.dim() != 2 or weight.size(1) == 0:
        raise RuntimeError(f"{op}: weight must be [V, K], got {list(weight.shape)}")
    if hidden.dim() < 1 or hidden.size(-1) != weight.size(1):
        raise RuntimeError(f"{op}: hidden must be [.., {weight.size(1)}], got {list(hidden.shape)}")
    if target.shape != hidden.shape[:-1]:
        raise RuntimeError(f"{op}: target must be {list(hidden.shape[:-1])}, got {list(target.shape)}")
    return hidden.reshape(-1, hidden.size(-1)).contiguous(), weight.contiguous(), target.reshape(-1).contiguous()


def _forward(
    hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int
) -> Tuple[torch.Tensor, torch.Tensor]:
    rows, table, words = _operands(hidden, weight, target, "linear_cross_entropy")
    loss = torch.empty(rows.size(0), dtype=torch.float32, device=hidden.device)
    lse = torch.empty_like(loss)
    torch.ops.tilefusion.linear_cross_entropy(rows, table, words, ignore_index, loss, lse)
    return loss.reshape(target.shape), lse.reshape(target.shape)


def _backward(
    grad_loss: torch.Tensor,
    hidden: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    lse: torch.Tensor,
    ignore_index: int,
    of_hidden: bool,
    of_weight: bool,
) -> Tuple[Any, Any]:
    """The gradients that are asked for, None in the place of the others."""
    rows, table, words = _operands(hidden, weight, target, "linear_cross_entropy_backward")
    for name, t in (("grad_loss", grad_loss), ("lse", lse)):
        if t.shape != target.shape:
            raise RuntimeError(f"linear_cross_entropy_backward: {name} must be {list(target.shape)}, got {list(t.shape)}")
    grad_hidden = torch.empty_like(rows) if of_hidden else None
    grad_weight = torch.empty_like(table) if of_weight else None
    with torch.no_grad():
        torch.ops.tilefusion.linear_cross_entropy_backward(
            grad_loss.reshape(-1).contiguous(), rows, table, words, lse.reshape(-1).contiguous(), ignore_index, grad_hidden, grad_weight
        )
    return grad_hidden.reshape(hidden.shape) if grad_hidden is not None else None, grad_weight


class _LinearCrossEntropy(torch.autograd.Function):
    @staticmethod
    def forward(
        ctx: Any, hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int
    ) -> Tuple[torch.Tensor, torch.Tensor]:
        loss, lse = _forward(hidden, weight, target, ignore_index)
        ctx.save_for_backward(hidden, weight, target, lse)
        ctx.ignore_index = ignore_index
        ctx.mark_non_differentiable(lse)
        return loss, lse

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_loss: torch.Tensor, _: Any) -> Tuple[Any, ...]:
        not_captured("linear_cross_entropy")
        of_hidden, of_weight, _, _ = ctx.needs_input_grad
        return (*_backward(grad_loss, *ctx.saved_tensors, ctx.ignore_index, of_hidden, of_weight), None, None)


def linear_cross_entropy(
    hidden: torch.Tensor, weight: torch.Tensor, target: torch.Tensor, ignore_index: int = -100
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Cross entropy of softmax(hidden @ weight.T) at `target`; the logits are never in memory.

    Args:
        hidden: [.., K] fp16 or bf16.
        weight: [V, K] of the same type.
        target: [..] int64.  Tokens whose target is `ignore_index` have loss 0 and no gradient; any other number outside
            0 .. V - 1 makes the loss NaN.

    Returns (loss, lse), both [..] fp32: the loss of every token, for the caller to weigh and add up, and the logarithm of the sum of
    exp(logits), which `linear_cross_entropy_backward` takes.  Under autograd the loss carries the backward pass (once: no
    gradient of a gradient, no forward mode), and lse none; neither the call nor that pass is captured into a graph.
    """
    if not torch.compiler.is_compiling():
        direct = _direct.linear_cross_entropy(hidden, weight, target, ignore_index)   # (no gradient is asked for)
        if direct is not None:
            return direct
    if records("linear_cross_entropy", hidden, weight):
        return _LinearCrossEntropy.apply(hidden, weight, target, ignore_index)
    return _forward(hidden, weight, target, ignore_index)


def linear_cross_entropy_backward(
    grad_loss: torch.Tensor,
    hidden: torch.Tensor,
    weight: torch.Tensor,
    target: torch.Tensor,
    lse: torch.Tensor,
    ignore_index: int = -100,
) -> Tuple[torch.Tensor, torch.Tensor]:
    """Gradients of hidden and weight, of their type, from that of the loss [..] (fp32) and the lse of the forward call.

    The vocabulary is done in pieces; what is held of a piece are its softmax gradients in 16 bits, which is where they are
    rounded: relative to the largest |grad_loss|, so that no weight of a mean is too small for fp16.  They have the power of two in
    a token's grad_loss; what is left of it is rounded with hidden, where tokens differ in it.  A grad_loss of an ignored
    token is not looked at; tokens with a target outside the vocabulary make NaN of the gradients they have a part in."""
    if not torch.compiler.is_compiling():
        direct = _direct.linear_cross_entropy_backward(grad_loss, hidden, weight, target, lse, ignore_index)
        if direct is not None:
            return direct
    refuse_transforms("linear_cross_entropy_backward", grad_loss, hidden, weight, lse)
    return _backward(grad_loss, hidden, weight, target, lse, ignore_index, True, True)
