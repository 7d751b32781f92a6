"""When the operators with a backward pass record it."""

from typing import Any

import torch
from torch.autograd import forward_ad


def not_captured(op: str) -> None:
    """Refuses a call that is recorded, or the backward pass of one that was, while a stream is being captured.

    A captured backward pass that accumulates into leaves of which an eager graph is alive as well ends the process, and
    a call cannot see whether there is one.  The `*_backward` functions are what is captured."""
    if not torch.compiler.is_compiling() and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            f"{op}: autograd does not record calls that are captured into a graph; "
            f"capture {op} under torch.no_grad() and {op}_backward"
        )


def refuse_transforms(op: str, *tensors: Any) -> None:
    """Refuses inputs that carry a derivative which nothing here passes on: a tangent, or the wrapper of a transform of torch.func.

    The operators write into tensors of their own, whose derivative would be zero without a word."""
    functorch = torch._C._functorch
    for t in tensors:
        if forward_ad._current_level >= 0 and forward_ad.unpack_dual(t).tangent is not None:
            raise RuntimeError(f"{op}: there are no forward-mode derivatives")
        # (compiled code can ask whether a transform is at work, and not whether it is on t)
        if functorch.maybe_current_level() is not None and (torch.compiler.is_compiling() or functorch.is_functorch_wrapped_tensor(t)):
            raise RuntimeError(f"{op}: does not work under torch.func's transforms")


def records(op: str, *tensors: torch.Tensor) -> bool:
    """Whether a call on `tensors` is to be recorded for autograd."""
    refuse_transforms(op, *tensors)
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)):
        return False
    not_captured(op)
    return True
