"""Sequence operators for predictors over histories of any length.

The Transformer predictors hold at most 48 slots in one tile and the recurrent ones roll a dense state
forward; these are the blocks between the two. `linear_attention` reads a history in chunks and leaves
a state of fixed size per head, `linear_attention_step` carries that state on slot by slot.

All take CUDA (ROCm) tensors of one type (float32, bfloat16 or float16), run on the current stream
and raise on anything the kernels do not serve. `linear_attention` has gradients (not twice
differentiable).
"""
import math

import torch

from . import ops  # noqa: F401


def linear_attention(q, k, v, log_decay, scale=None, initial_state=None, lengths=None):
    """q, k [B, T, H, K], v [B, T, H, V], log_decay float32 [H] -> (o [B, T, H, V], state float32
    [B, H, K, V]):

        S_t = exp(log_decay) S_{t-1} + k_t^T v_t,    o_t = scale * q_t S_t,

    S before the first slot = `initial_state` (float32 [B, H, K, V], zero if None), `state` = S after the
    last one; `scale` is K ** -0.5 by default; K, V <= 256. `lengths` (int32 or int64 [B] on the GPU, T
    everywhere if None, values outside [0, T] taken as the nearer end): slots at and behind a sequence's
    length are not read, their o and their gradients are zero, and the state stops before them. The
    decay is a constant: it has no gradient and is refused if it wants one. Any strides with a
    contiguous last axis are read in place where rows start on 16 bytes, copied once otherwise."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() and q.shape[-1] else 1.0
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay is a constant of linear_attention: it has no gradient (detach it)")
    return torch.ops.cet.linear_attention(q, k, v, log_decay, float(scale), initial_state, lengths)


def linear_attention_step(q, k, v, log_decay, state, scale=None, slots=None, inplace=False):
    """One slot of `linear_attention` for every stream: q, k [B, H, K], v [B, H, V] -> (o [B, H, V], state).

    Without `slots`, `state` is float32 [B, H, K, V]; the new state is a new tensor, or the same one
    with `inplace`. With `slots` (int32 or int64 [B] on the GPU) `state` is a pool [rows, H, K, V] that is
    updated in place: stream b owns row slots[b]. A negative slot is an idle stream (o = 0); a slot
    beyond the pool, or one that an earlier stream of the call already has, gives o = NaN and changes
    no state (the values are on the GPU: raising would wait for it). No gradients."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() and q.shape[-1] else 1.0
    if torch.is_grad_enabled() and any(t.requires_grad for t in (q, k, v, log_decay, state)):
        raise RuntimeError("linear_attention_step has no gradient: call it under torch.no_grad(), or "
                           "linear_attention with T = 1")
    if slots is not None or inplace:
        return torch.ops.cet.linear_attention_step_(q, k, v, log_decay, state, float(scale), slots), state
    return torch.ops.cet.linear_attention_step(q, k, v, log_decay, state, float(scale))
