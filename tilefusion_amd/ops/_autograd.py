"""When the operators with a backward pass record it."""

import torch


def not_captured(op: str) -> None:
    """Refuses a call that is recorded, or the backward pass of one that was, while a stream is being captured.

    A captured backward pass that accumulates into leaves of which an eager graph is alive as well ends the process, and
    a call cannot see whether there is one.  The `*_backward` functions are what is captured."""
    if not torch.compiler.is_compiling() and torch.cuda.is_available() and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(
            f"{op}: autograd does not record calls that are captured into a graph; "
            f"capture {op} under torch.no_grad() and {op}_backward"
        )


def records(op: str, *tensors: torch.Tensor) -> bool:
    """Whether a call on `tensors` is to be recorded for autograd."""
    if not (torch.is_grad_enabled() and any(t.requires_grad for t in tensors)):
        return False
    not_captured(op)
    return True
