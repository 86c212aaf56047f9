"""A captured backward beside a living eager graph.

The autograd engine ends a backward by waiting for the streams of the leaves' gradient
accumulators.  An accumulator lives as long as any graph of its leaf and keeps the stream
that it was made on, so where an eager graph of the same leaf is alive while a backward is
captured into a HIP graph, that wait leaves the capture, and the runtime ends the process
at its end.  The operators' functions note here, on each leaf's accumulator, whether it was made
outside a capture, and their backward raises before the engine gets that far.  Torch does not
tell the age of an accumulator, so they see leaves that are their own inputs, in eager graphs
that went through them; graphs of other operators alone, and leaves further up, torch's engine
meets as it meets any model's.
"""

from __future__ import annotations

import torch

from opake_amd.exceptions import OperationError

_MARK = "opake_amd_made_in_capture"


def note_leaves(ctx) -> None:
    """In a function's forward, which the gradients will go through."""
    # Holding the accumulators' Python objects keeps their marks as long as this graph.
    ctx.accumulators = [fn for fn, _ in ctx.next_functions
                        if fn is not None and fn.name() == "torch::autograd::AccumulateGrad"]
    if ctx.accumulators:
        captured = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        for fn in ctx.accumulators:
            fn.metadata.setdefault(_MARK, captured)


def check_leaves(ctx) -> None:
    """In that function's backward."""
    if any(not fn.metadata[_MARK] for fn in ctx.accumulators) and \
            torch.cuda.is_current_stream_capturing():
        raise OperationError(
            "a backward pass is captured while an eager graph of the same leaves is alive: "
            "delete what was computed from them outside the capture first")


__all__ = ["check_leaves", "note_leaves"]
