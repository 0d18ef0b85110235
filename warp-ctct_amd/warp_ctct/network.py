"""Operators beside the losses: what makes the label scores of a transducer, and
the rules put on the joiner's logits before a token is taken from them.

The losses start from scores.  These are the operators on either side of them
that a model of the same kind runs: :func:`layer_norm` for a prediction network
or an encoder, in training.  Hand-written HIP kernels
like the losses', through the same binding: float32, float16 and bfloat16 are
read as they are (another type is converted to float32), sums and states are
kept in float32, a result is rounded once.  Nothing synchronises with the host;
work is enqueued on the current stream of the input's GPU.  A wrong shape, type
or device raises RuntimeError.  The backward passes are not differentiable
themselves (``create_graph=True`` raises).  Forward and backward can be captured
into a graph; as with any operator of torch, an eager autograd graph that hangs
on the same leaves must be gone before a backward pass is captured.

The reference has no counterpart: its callers take these from torch.
"""
from typing import Optional

import torch

from . import _C as core


def layer_norm(x: torch.Tensor,
               weight: Optional[torch.Tensor] = None,
               bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """``(x - mean) / sqrt(var + eps) * weight + bias`` over the last dimension.

    Args:
        x: (..., D).  Rows may lie anywhere, up to two strides in front of a
            dense last dimension (a transposed batch, a slice of a wider tensor)
            are read in place; other layouts are copied first.
        weight, bias: (D,) or None.  Both of the input's type, or converted to
            float32.
        eps: added to the (biased) variance.

    Differentiable with respect to ``x``, ``weight`` and ``bias``.  The gradients
    of the parameters are added up in a fixed order: the same on every call."""
    return core.layer_norm(x, weight, bias, float(eps))
