"""Operators beside the losses: what makes the label scores of a transducer, and
the rules put on the joiner's logits before a token is taken from them.

The losses start from scores.  These are the operators on either side of them
that a model of the same kind runs: :func:`layer_norm`, :func:`causal_conv` and
:func:`selective_scan` for a prediction network or an encoder, in training and
over prompts, :func:`causal_conv_step` and :func:`selective_scan_step` for
decoding a token at a time; :func:`adjust_logits` before a token is taken.
Hand-written HIP kernels like the losses', through the same binding: float32,
float16 and bfloat16 are read as they are (another type is converted to
float32), sums and states are kept in float32, a result is rounded once.  Nothing synchronises with the host;
work is enqueued on the current stream of the input's GPU.  A wrong shape, type
or device raises RuntimeError.  The backward passes are not differentiable
themselves (``create_graph=True`` raises), and inputs with a forward-mode tangent
are refused.  Forward and backward can be captured
into a graph; as with any operator of torch, an eager autograd graph that hangs
on the same leaves must be gone before a backward pass is captured.

The reference has no counterpart: its callers take these from torch.
"""
from typing import Optional, Union

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


def _activation(name: Optional[str]) -> bool:
    if name not in (None, "silu"):
        raise RuntimeError("activation must be None or 'silu', got %r" % (name,))
    return name == "silu"


def causal_conv(x: torch.Tensor,
                weight: torch.Tensor,
                bias: Optional[torch.Tensor] = None,
                lengths: Optional[torch.Tensor] = None,
                initial_state: Optional[torch.Tensor] = None,
                activation: Optional[str] = None,
                return_state: bool = False):
    """A short convolution along time, every channel with its own taps:
    ``out[n, t, e] = act(bias[e] + sum_k weight[e, k] * x[n, t - (K-1) + k, e])``.

    Args:
        x: (N, T, E).  A view with a dense last dimension is read in place.
        weight: (E, K), K from 1 to 8; the last tap is the current step's.
        bias: (E,) or None.
        lengths: (N,) steps of each sequence; the steps behind them are not read
            and their outputs (and gradients) are zero.  None: all T.
        initial_state: (N, K-1, E), the inputs in front of ``x``, in the type of
            ``x`` (float32 or float64 where that is float64).  None: zeros.
        activation: None or ``'silu'``.
        return_state: also return (N, K-1, E), the last K-1 inputs of every
            sequence: the ``initial_state`` of a call that goes on from there, and
            the ``state`` of :func:`causal_conv_step`.

    Returns out (N, T, E), or ``(out, state)``.  Differentiable with respect to
    ``x``, ``weight``, ``bias`` and ``initial_state``, through both results; the
    gradients of the parameters are added up in a fixed order.  The gradient of
    ``x`` is formed whether it is asked for or not."""
    got = core.causal_conv(x, weight, bias, lengths, initial_state, _activation(activation), bool(return_state))
    return (got[0], got[1]) if return_state else got[0]


def causal_conv_step(x: torch.Tensor,
                     state: torch.Tensor,
                     weight: torch.Tensor,
                     bias: Optional[torch.Tensor] = None,
                     activation: Optional[str] = None,
                     advance: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of :func:`causal_conv` for N sequences: ``x`` (N, E) comes in,
    ``state`` (N, K-1, E), in the type of the result, moves on in place, out
    (N, E) is returned.

    ``advance`` (N,) bool, None for all: a sequence that does not advance keeps
    its state, and its row of the result is zero (a hypothesis that took blank
    keeps the output of its last label).  Not differentiable: call it under
    ``torch.no_grad()``."""
    return core.causal_conv_step(x, state, weight, bias, _activation(activation), advance)


def selective_scan(x: torch.Tensor,
                   dt: torch.Tensor,
                   a: torch.Tensor,
                   b: torch.Tensor,
                   c: torch.Tensor,
                   skip: Optional[torch.Tensor] = None,
                   gate: Optional[torch.Tensor] = None,
                   dt_bias: Optional[torch.Tensor] = None,
                   softplus: bool = False,
                   lengths: Optional[torch.Tensor] = None,
                   initial_state: Optional[torch.Tensor] = None,
                   return_state: bool = False):
    """Selective state space scan: every channel drives S states of its own::

        d = softplus(dt + dt_bias)            # softplus=False: the sum itself
        h[s] = exp(d * a[s]) * h[s] + d * x * b[s]
        out = (sum_s c[s] * h[s] + skip * x) * silu(gate)

    Args:
        x, dt, gate: (N, T, E) in one type; gate may be None.  Views with a dense
            last dimension (the halves of one projection) are read in place.
        a: (E, S), S up to 64; converted to float32 like skip and dt_bias.
        b, c: (N, T, S), or (N, T, G, S) for G groups of E/G channels next to each
            other, in the type of ``x``.
        skip, dt_bias: (E,) or None.
        lengths: (N,) steps of each sequence; the steps behind them are not read
            and their outputs (and gradients) are zero.  None: all T.
        initial_state: (N, E, S) float32 (or float64, converted), the states in
            front of the first step.  None: zeros.
        return_state: also return the states behind the last step of every
            sequence, (N, E, S) float32: the ``initial_state`` of a call that goes
            on from there, and the ``state`` of :func:`selective_scan_step`.

    Returns out (N, T, E), or ``(out, state)``.  Differentiable with respect to
    everything but ``lengths``, through both results; every sum is added up in a
    fixed order.  All gradients are formed, whichever are asked for.  Where a gradient is tracked, the states in front of every 8
    steps are kept for it: T/8 * N * E * S floats for 16 states."""
    got = core.selective_scan(x, dt, a, b, c, skip, gate, dt_bias, bool(softplus), lengths, initial_state,
                              bool(return_state))
    return (got[0], got[1]) if return_state else got[0]


def selective_scan_step(x: torch.Tensor,
                        state: torch.Tensor,
                        dt: torch.Tensor,
                        a: torch.Tensor,
                        b: torch.Tensor,
                        c: torch.Tensor,
                        skip: Optional[torch.Tensor] = None,
                        gate: Optional[torch.Tensor] = None,
                        dt_bias: Optional[torch.Tensor] = None,
                        softplus: bool = False,
                        advance: Optional[torch.Tensor] = None) -> torch.Tensor:
    """One step of :func:`selective_scan` for N sequences: ``x``, ``dt``, ``gate``
    (N, E), ``b``, ``c`` (N, S) or (N, G, S); ``state`` (N, E, S) float32 moves on
    in place, out (N, E) is returned.

    ``advance`` (N,) bool, None for all: a sequence that does not advance keeps
    its state, and its row of the result is zero.  Not differentiable: call it
    under ``torch.no_grad()``."""
    return core.selective_scan_step(x, state, dt, a, b, c, skip, gate, dt_bias, bool(softplus), advance)


def adjust_logits(logits: torch.Tensor,
                  tokens: Optional[torch.Tensor] = None,
                  tokens_lengths: Optional[torch.Tensor] = None,
                  repetition_penalty: Union[float, torch.Tensor] = 1.0,
                  presence_penalty: Union[float, torch.Tensor] = 0.0,
                  frequency_penalty: Union[float, torch.Tensor] = 0.0,
                  bias: Optional[torch.Tensor] = None,
                  allowed: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The rules that a decoder puts on logits before it takes a token, in one
    pass: penalties for the tokens a row holds already, then a bias, then a mask.
    For every column ``v`` that stands ``count > 0`` times among a row's tokens::

        l = l / repetition_penalty if l > 0 else l * repetition_penalty
        l = l - presence_penalty - frequency_penalty * count

    then ``l + bias``, and minus infinity where ``allowed`` is not set.

    Args:
        logits: (N, V).
        tokens: (N, H) whole numbers, H up to 2^30, or None; values outside [0, V)
            (padding) count for nothing.
        tokens_lengths: (N,) how many of a row's tokens count.  None: all H.
        repetition_penalty, presence_penalty, frequency_penalty: a number, or
            (N,) with one for each row.  A repetition penalty is positive.
        bias: (V,) or (N, V): of an outer language model, of words to be heard.
        allowed: what a grammar lets follow: (V,) or (N, V) bool, or the same in
            bits, int32 (ceil(V/32),) or (N, ceil(V/32)) with bit ``v % 32`` of
            word ``v // 32`` for column ``v``.  A row that allows nothing comes
            out as minus infinity throughout.

    Returns a new (N, V) tensor of the type of ``logits``.  Not differentiable:
    call it under ``torch.no_grad()`` where an input requires a gradient."""
    return core.adjust_logits(logits, tokens, tokens_lengths, repetition_penalty, presence_penalty,
                              frequency_penalty, bias, allowed)
