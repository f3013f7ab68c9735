"""Sequence operators for predictors over histories of any length.

The Transformer predictors hold at most 48 slots in one tile and the recurrent ones roll a dense state
forward; these are the blocks between the two. `rotary` gives queries and keys their slots' positions
(the Transformer adds a fixed table of sinusoids), `linear_attention` reads a history in chunks and
leaves a state of fixed size per head, `linear_attention_step` carries that state on slot by slot, and
`gated_linear` is the first half of a gated feed-forward (the Transformer's is a plain one).

All take CUDA (ROCm) tensors of one type (float32, bfloat16 or float16), run on the current stream
and raise on anything the kernels do not serve. `rotary`, `linear_attention` and
`gated_linear` have gradients (`rotary`'s can be differentiated again; the transforms of torch.func and
forward-mode differentiation are refused). All can be captured into graphs; a training step is captured whole, with
no eager graph of the same leaves alive, as torch asks.
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
    contiguous last axis are read in place where rows start on 16 bytes, copied once otherwise. Slots are
    taken in chunks of up to 32: an infinity or NaN in a slot within its sequence's length can reach the
    outputs of the slots of its chunk before it, too (an infinity as NaN). Sums and states are float32, and o and the
    gradients are rounded once; for bfloat16 tensors scores and states enter their products with 16 bits."""
    if scale is None:
        scale = 1.0 / math.sqrt(q.shape[-1]) if q.dim() and q.shape[-1] else 1.0
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay is a constant of linear_attention: it has no gradient (detach it)")
    grad = ops.wants_grad(q, k, v, initial_state)
    if not ops.direct(q, k, v, log_decay, initial_state, lengths):
        run = torch.ops.cet.linear_attention
    else:
        run = ops.LinearAttention.apply if grad else ops.run_linear_attention
    return run(q, k, v, log_decay, float(scale), initial_state, lengths, grad)[:2]


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
    direct, args = ops.direct(q, k, v, log_decay, state, slots), (q, k, v, log_decay, state, float(scale))
    if slots is not None or inplace:
        return (ops.step_in_place if direct else torch.ops.cet.linear_attention_step_)(*args, slots), state
    return (ops.run_linear_attention_step if direct else torch.ops.cet.linear_attention_step)(*args)


def rotary_frequencies(dim, base=10000.0, scaling="none", factor=1.0, original_length=None, turns=(32.0, 1.0), device="cuda"):
    """Radians per slot of the dim / 2 pairs of `rotary`, base ** (-2 j / dim), and the gain to call it
    with: (float64 [dim / 2] on `device`, float). `scaling` stretches positions that were trained on
    `original_length` slots over `factor` times as many:

    * "linear": every rate divided by `factor`;
    * "ntk": the base times factor ** (dim / (dim - 2)), so that the slowest pair is stretched by
      `factor` and the fastest keeps its rate;
    * "yarn": pairs that turn more than turns[0] times within `original_length` keep their rate, those
      below turns[1] are divided by `factor`, a linear ramp over the pairs between, from the last of the
      former to the first of the latter (which may lie behind the last pair); gain 0.1 ln(factor) + 1."""
    dim = int(dim)
    if dim < 2 or dim % 2:
        raise RuntimeError(f"dim must be even and positive, got {dim}")
    if not (base > 1.0 and math.isfinite(base) and factor > 0.0 and math.isfinite(factor)):
        raise RuntimeError(f"base must exceed 1 and factor 0, got {base}, {factor}")
    if scaling not in ("none", "linear", "ntk", "yarn"):
        raise RuntimeError(f'scaling must be "none", "linear", "ntk" or "yarn", got {scaling!r}')
    if scaling == "ntk":
        base = base * factor ** (dim / max(dim - 2, 1))
    j = torch.arange(dim // 2, dtype=torch.float64)
    freq, gain = base ** (-2.0 * j / dim), 1.0
    if scaling == "linear":
        freq = freq / factor
    elif scaling == "yarn":
        if not original_length or original_length <= 0 or not turns[0] > turns[1] > 0:
            raise RuntimeError("yarn needs original_length > 0 and turns[0] > turns[1] > 0")
        pair = [dim * math.log(original_length / (n * 2 * math.pi)) / (2 * math.log(base)) for n in turns]
        low, high = max(math.floor(pair[0]), 0), min(math.ceil(pair[1]), dim - 1)
        ramp = ((j - low) / max(high - low, 0.001)).clamp(0, 1)
        ramp[j >= pair[1]] = 1.0  # (all of them where even the first turns less than turns[1] times)
        freq = freq / factor * ramp + freq * (1 - ramp)
        gain = 0.1 * math.log(factor) + 1.0 if factor > 1.0 else 1.0
    return freq.to(device), gain


def rotary(q, k, positions, inv_freq, layout="half", gain=1.0):
    """Turns the pairs of q [B, T, Hq, D] and k [B, T, Hk, D] (or None) by positions * inv_freq:
    (a, b) -> gain (a cos - b sin, a sin + b cos); returns the two turned tensors (contiguous; the
    second None without k). `positions`: int32 or int64 [T] or [B, T], any values; `inv_freq`: float64
    [pairs] with 2 pairs <= D (see `rotary_frequencies`); `layout`: pairs are (j, j + pairs) ("half") or
    (2j, 2j + 1) ("interleaved"). Features behind the pairs pass through. Angles are formed in float64."""
    if layout not in ("half", "interleaved"):
        raise RuntimeError(f'layout must be "half" or "interleaved", got {layout!r}')
    if inv_freq.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("inv_freq is a constant of rotary: it has no gradient (detach it)")
    run = ops.direct_rotary if ops.direct(q, k, positions, inv_freq) else torch.ops.cet.rotary
    a, b = run(q, k, positions, inv_freq, layout == "interleaved", float(gain), False)
    return a, (b if k is not None else None)


def gated_linear(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up) in one kernel: x [..., D], w_gate and w_up [F, D] (the
    layout of `torch.nn.Linear`, or two halves of one [2F, D]), biases [F] or None, one type for all;
    returns [..., F]. `activation`: "silu", "gelu" (erf form) or "relu". Projections and activation are
    formed in float32 and the result is rounded once; the projections are not kept for the gradient but
    formed again. Their gradients are rounded to the tensors' type before the products that dx and the weights'
    gradients are (an error of the size of the results' own rounding); in float16 they have that type's range, infinite
    beyond 65504 and zero below 3e-8, which is what loss scaling is for. Layers with D and F up to 64 keep them in
    float32."""
    if x.dim() < 1:
        raise RuntimeError("x must be [..., D]")
    args = x.reshape(-1, x.shape[-1]) if x.dim() != 2 else x, w_gate, w_up, b_gate, b_up, activation
    if not ops.direct(x, w_gate, w_up, b_gate, b_up):
        out = torch.ops.cet.gated_linear(*args)
    else:
        out = ops.GatedLinear.apply(*args) if ops.wants_grad(x, w_gate, w_up, b_gate, b_up) else ops.run_gated_linear(*args)
    return out if x.dim() == 2 else out.reshape(*x.shape[:-1], w_gate.shape[0])
