"""Plain float64 statements of the sequence operators (CPU) for their tests."""
import math

import torch


def half_step(dtype):
    """Largest relative error of one rounding to `dtype`."""
    return torch.finfo(dtype).eps / 2


def linear_attention(q, k, v, log_decay, scale, s0=None, lengths=None):
    """Slot by slot; every product and sum as written in the definition."""
    B, T, H, K = q.shape
    V = v.shape[3]
    d = log_decay.double().exp().view(1, H, 1, 1)
    S = torch.zeros(B, H, K, V, dtype=torch.float64) if s0 is None else s0
    n = torch.full((B,), T) if lengths is None else lengths.clamp(0, T)
    out = []
    for t in range(T):
        live = (t < n).view(B, 1, 1, 1)
        S = torch.where(live, S * d + k[:, t, :, :, None] * v[:, t, :, None, :], S)
        o = scale * (q[:, t, :, :, None] * S).sum(-2)
        out.append(torch.where(live[..., 0], o, torch.zeros_like(o)))
    return (torch.stack(out, 1) if out else v.new_zeros(B, 0, H, V)), S


def linear_attention_with_gradients(q, k, v, log_decay, scale, s0, lengths, d_o, d_state):
    x = [t.detach().requires_grad_() for t in (q, k, v)] + ([s0.detach().requires_grad_()] if s0 is not None else [])
    o, S = linear_attention(x[0], x[1], x[2], log_decay, scale, x[3] if s0 is not None else None, lengths)
    loss = (o * d_o).sum() + (S * d_state).sum()
    grads = torch.autograd.grad(loss, x, allow_unused=True)
    return o.detach(), S.detach(), [torch.zeros_like(a) if g is None else g for a, g in zip(x, grads)]


def clean(x, lengths):
    """The operand with zeros behind the sequences: what lies there must not matter."""
    if lengths is None:
        return x
    live = torch.arange(x.shape[1])[None] < lengths[:, None]
    return torch.where(live.view(*live.shape, 1, 1), x, torch.zeros_like(x))


def geometric(H):
    return torch.log1p(-torch.exp2(-2.0 - 8.0 * torch.arange(H).float() / max(H, 1)))


def sqrt_scale(K):
    return 1.0 / math.sqrt(K)


def rotary(x, positions, freq, layout, gain):
    """x [B, T, H, D] float64."""
    P = freq.shape[0]
    angle = (positions.double()[..., None] * freq).expand(x.shape[0], x.shape[1], P)[:, :, None]
    c, s = gain * angle.cos(), gain * angle.sin()
    y = x.clone()
    ia = torch.arange(P) if layout == "half" else 2 * torch.arange(P)
    ib = ia + (P if layout == "half" else 1)
    y[..., ia] = x[..., ia] * c - x[..., ib] * s
    y[..., ib] = x[..., ia] * s + x[..., ib] * c
    return y
