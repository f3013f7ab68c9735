"""PyTorch custom ops (`torch.ops.cet.*`) in front of the C ABI.

Each op checks device / dtype / contiguity, allocates the outputs with torch (the library
never allocates results) and enqueues the HIP kernel on torch's current stream through the
ctypes binding. Handles are created and owned by the host-side model objects.
"""
import contextlib
import ctypes
import math
from typing import Optional

import torch
from torch.autograd import forward_ad

from . import _cabi

_NO_ARG = torch.empty(0)


def _dev_check(*tensors):
    dev = tensors[0].device
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError(
                "channelestimationtransformer_amd computes on the GPU only: got a tensor on "
                f"{t.device}; move inputs to a ROCm device (there is no CPU path)")
        if t.device != dev:
            raise RuntimeError(f"tensors on different devices: {t.device} vs {dev}")
    return dev


def _f32(name, t, *shape):
    """A contiguous float32 tensor of exactly this shape (None = any size in that position):
    the kernels index raw pointers, so a wrong dtype or a short buffer would read out of bounds."""
    if t.dtype != torch.float32:
        raise RuntimeError(f"{name} must be float32, got {t.dtype}")
    if t.shape != shape and (  # (the comparison alone where every size is given)
            t.dim() != len(shape) or any(s is not None and int(d) != int(s) for d, s in zip(t.shape, shape))):
        raise RuntimeError(f"{name} must have shape {list(shape)}, got {list(t.shape)}")
    t = t.contiguous() if t.numel() > 1 else t.contiguous().resolve_neg()  # (a single value may carry a flag for its sign)
    return t.clone() if t.data_ptr() % 16 else t  # a slice may start anywhere; the C ABI wants 16 B


def _noise(no, no_mode, N, Nr):
    """The noise operand of the per-resource-element kernels for `no_mode`."""
    if no_mode == 0:
        return None
    if no_mode == 1:
        return _f32("no", no, N)
    if no_mode == 2:
        return _f32("no", no, N, Nr)
    raise RuntimeError(f"no_mode must be 0, 1 or 2, got {no_mode}")


def _ptr(t):
    return ctypes.c_void_p(t.data_ptr()) if t is not None and t.numel() else None


@torch.library.custom_op("cet::informer_forward", mutates_args=())
def informer_forward(x_enc: torch.Tensor, x_dec: torch.Tensor, handle: int, pred_len: int,
                     c_out: int, attn_floats_per_sample: int) -> tuple[torch.Tensor, torch.Tensor]:
    dev = _dev_check(x_enc, x_dec)
    x_enc = x_enc.contiguous().float()
    x_dec = x_dec.contiguous().float()
    B = x_enc.shape[0]
    out = torch.empty((B, pred_len, c_out), dtype=torch.float32, device=dev)
    attn = torch.empty((B * attn_floats_per_sample,), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        rc = _cabi.lib().cet_informer_forward(
            ctypes.c_void_p(handle), _ptr(x_enc), _ptr(x_dec), _ptr(out), _ptr(attn), B,
            _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_informer_forward")
    return out, attn


@informer_forward.register_fake
def _(x_enc, x_dec, handle, pred_len, c_out, attn_floats_per_sample):
    B = x_enc.shape[0]
    return (x_enc.new_empty((B, pred_len, c_out)), x_enc.new_empty((B * attn_floats_per_sample,)))


@torch.library.custom_op("cet::rnn_rollout", mutates_args=())
def rnn_rollout(x: torch.Tensor, handle: int, pred_len: int) -> torch.Tensor:
    dev = _dev_check(x)
    x = x.contiguous().float()
    B, seq_len, F = x.shape
    out = torch.empty((B, pred_len, F), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        rc = _cabi.lib().cet_rnn_rollout(ctypes.c_void_p(handle), _ptr(x), _ptr(out), B, seq_len,
                                         pred_len, _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_rnn_rollout")
    return out


@rnn_rollout.register_fake
def _(x, handle, pred_len):
    return x.new_empty((x.shape[0], pred_len, x.shape[2]))


@torch.library.custom_op("cet::lmmse", mutates_args=())
def lmmse(y: torch.Tensor, H: torch.Tensor, no: torch.Tensor, no_scalar: float,
          no_mode: int, direct: bool, h_share: int = 1) -> tuple[torch.Tensor, torch.Tensor]:
    """y [N,Nr,2], H [ceil(N/h_share),Nr,Ns,2] float32 (interleaved complex) -> x_hat [N,Ns,2],
    no_eff [N,Ns]. h_share > 1: block fading, RE n uses H[n // h_share]."""
    dev = _dev_check(y, H) if no_mode == 0 else _dev_check(y, H, no)
    y = _f32("y", y, None, None, 2)
    N, Nr = y.shape[0], y.shape[1]
    H = _f32("H", H, None, Nr, None, 2)
    Ns = H.shape[2]
    _block_check(N, H.shape[0], h_share, direct)
    x_hat = torch.empty((N, Ns, 2), dtype=torch.float32, device=dev)
    no_eff = torch.empty((N, Ns), dtype=torch.float32, device=dev)
    no_dev = _noise(no, no_mode, N, Nr)
    L = _cabi.lib()
    with torch.cuda.device(dev):
        if h_share > 1:
            rc = L.cet_lmmse_block(_ptr(y), _ptr(H), no_mode, ctypes.c_float(no_scalar), _ptr(no_dev),
                                   _ptr(x_hat), _ptr(no_eff), ctypes.c_long(N), h_share, Nr, Ns,
                                   _cabi.current_stream_ptr(dev))
        else:
            fn = L.cet_lmmse_direct if direct else L.cet_lmmse
            rc = fn(_ptr(y), _ptr(H), no_mode, ctypes.c_float(no_scalar), _ptr(no_dev), _ptr(x_hat),
                    _ptr(no_eff), ctypes.c_long(N), Nr, Ns, _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_lmmse")
    return x_hat, no_eff


def _block_check(N, n_h, h_share, direct=False):
    if h_share < 1 or n_h != -(-N // h_share):
        raise RuntimeError(f"H holds {n_h} matrices; {N} REs with h_share={h_share} need {-(-N // max(h_share, 1))}")
    if direct and h_share > 1:
        raise RuntimeError("the direct kernel has no block-fading entry point")


@lmmse.register_fake
def _(y, H, no, no_scalar, no_mode, direct, h_share=1):
    N, Ns = y.shape[0], H.shape[2]
    return y.new_empty((N, Ns, 2)), y.new_empty((N, Ns))


@torch.library.custom_op("cet::nmse_sums", mutates_args=())
def nmse_sums(pred: torch.Tensor, truth: torch.Tensor) -> torch.Tensor:
    """pred, truth [B,P,C] float32 -> float64 [2,P]: (sum (truth-pred)^2, sum truth^2) per slot."""
    dev = _dev_check(pred, truth)
    pred = pred.contiguous().float()
    truth = truth.contiguous().float()
    B, P, C = pred.shape
    sums = torch.empty((2, P), dtype=torch.float64, device=dev)
    with torch.cuda.device(dev):
        rc = _cabi.lib().cet_nmse_sums(_ptr(pred), _ptr(truth), ctypes.c_void_p(sums.data_ptr()),
                                       ctypes.c_long(B), P, C, _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_nmse_sums")
    return sums


@nmse_sums.register_fake
def _(pred, truth):
    return pred.new_empty((2, pred.shape[1]), dtype=torch.float64)


@torch.library.custom_op("cet::qpsk_bit_errors", mutates_args=())
def qpsk_bit_errors(x_hat: torch.Tensor, x_true: torch.Tensor) -> torch.Tensor:
    """x_hat, x_true [..., 2] float32 (interleaved complex) -> float64 [2]: (bit errors, bits)."""
    dev = _dev_check(x_hat, x_true)
    x_hat = x_hat.contiguous().float()
    x_true = x_true.contiguous().float()
    x_hat = x_hat.clone() if x_hat.data_ptr() % 8 else x_hat  # (re, im) pairs are read as one piece
    x_true = x_true.clone() if x_true.data_ptr() % 8 else x_true
    N = x_hat.numel() // 2
    out = torch.empty((2,), dtype=torch.float64, device=dev)
    with torch.cuda.device(dev):
        rc = _cabi.lib().cet_qpsk_bit_errors(_ptr(x_hat), _ptr(x_true), ctypes.c_void_p(out.data_ptr()),
                                             ctypes.c_long(N), _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_qpsk_bit_errors")
    return out


@qpsk_bit_errors.register_fake
def _(x_hat, x_true):
    return x_hat.new_empty((2,), dtype=torch.float64)


@torch.library.custom_op("cet::lmmse_llr", mutates_args=())
def lmmse_llr(y: torch.Tensor, H: torch.Tensor, no: torch.Tensor, no_scalar: float,
              no_mode: int, h_share: int = 1) -> torch.Tensor:
    """y [N,Nr,2], H [ceil(N/h_share),Nr,Ns,2] float32 -> QPSK bit LLRs [N,Ns,2] (equalizer +
    demapper fused)."""
    dev = _dev_check(y, H) if no_mode == 0 else _dev_check(y, H, no)
    y = _f32("y", y, None, None, 2)
    N, Nr = y.shape[0], y.shape[1]
    H = _f32("H", H, None, Nr, None, 2)
    Ns = H.shape[2]
    _block_check(N, H.shape[0], h_share)
    llr = torch.empty((N, Ns, 2), dtype=torch.float32, device=dev)
    no_dev = _noise(no, no_mode, N, Nr)
    L = _cabi.lib()
    with torch.cuda.device(dev):
        if h_share > 1:
            rc = L.cet_lmmse_block_llr(_ptr(y), _ptr(H), no_mode, ctypes.c_float(no_scalar),
                                       _ptr(no_dev), _ptr(llr), ctypes.c_long(N), h_share, Nr, Ns,
                                       _cabi.current_stream_ptr(dev))
        else:
            rc = L.cet_lmmse_llr(_ptr(y), _ptr(H), no_mode, ctypes.c_float(no_scalar),
                                 _ptr(no_dev), _ptr(llr), ctypes.c_long(N), Nr, Ns,
                                 _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_lmmse_llr")
    return llr


@lmmse_llr.register_fake
def _(y, H, no, no_scalar, no_mode, h_share=1):
    return y.new_empty((y.shape[0], H.shape[2], 2))


@torch.library.custom_op("cet::ls_nn", mutates_args=())
def ls_nn(y: torch.Tensor, src: torch.Tensor, pinv: torch.Tensor, pabs2inv: torch.Tensor,
          no: float) -> tuple[torch.Tensor, torch.Tensor]:
    """y [planes, plane, 2] float32 (interleaved complex), tables of T entries ->
    h_hat [planes, T, 2], err_var [planes, T]."""
    dev = _dev_check(y, src, pinv, pabs2inv)
    y = _f32("y", y, None, None, 2)
    planes, plane = y.shape[0], y.shape[1]
    T = src.numel()
    if src.dtype != torch.int32 or src.dim() != 1:
        raise RuntimeError(f"src must be a 1-d int32 table, got {src.dtype} {list(src.shape)}")
    src = src.contiguous()
    pinv = _f32("pinv", pinv, T, 2)
    pabs2inv = _f32("pabs2inv", pabs2inv, T)
    h_hat = torch.empty((planes, T, 2), dtype=torch.float32, device=dev)
    err_var = torch.empty((planes, T), dtype=torch.float32, device=dev)
    with torch.cuda.device(dev):
        rc = _cabi.lib().cet_ls_nn(_ptr(y), _ptr(src), _ptr(pinv), _ptr(pabs2inv), ctypes.c_float(no),
                                   _ptr(h_hat), _ptr(err_var), ctypes.c_long(planes), plane, T,
                                   _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_ls_nn")
    return h_hat, err_var


@ls_nn.register_fake
def _(y, src, pinv, pabs2inv, no):
    return y.new_empty((y.shape[0], src.numel(), 2)), y.new_empty((y.shape[0], src.numel()))


@torch.library.custom_op("cet::lmmse_grid", mutates_args=())
def lmmse_grid(y: torch.Tensor, h_hat: torch.Tensor, err_var: torch.Tensor, no: torch.Tensor,
               no_scalar: float, no_mode: int, data_sym: torch.Tensor,
               eff_sc: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """y [B,Nr,n_sym,fft,2], h_hat [B,Nr,Ns,n_sym,n_sc,2] float32 (interleaved complex), err_var
    empty or [B,Nr,Ns,n_sym,n_sc]; index tables int32 -> x_hat [B,Ns,n_ds*n_sc,2], no_eff
    [B,Ns,n_ds*n_sc]."""
    dev = _dev_check(y, h_hat, data_sym, eff_sc)
    y = _f32("y", y, None, None, None, None, 2)
    B, Nr, n_sym, fft = y.shape[:4]
    h_hat = _f32("h_hat", h_hat, B, Nr, None, n_sym, None, 2)
    Ns, n_sc = h_hat.shape[2], h_hat.shape[4]
    n_ds = data_sym.numel()
    for name, t in (("data_sym", data_sym), ("eff_sc", eff_sc)):
        if t.dtype != torch.int32 or t.dim() != 1:
            raise RuntimeError(f"{name} must be a 1-d int32 table, got {t.dtype} {list(t.shape)}")
    data_sym, eff_sc = data_sym.contiguous(), eff_sc.contiguous()
    if eff_sc.numel() != n_sc or n_sc > fft or n_ds > n_sym:
        raise RuntimeError(f"inconsistent shapes: y {tuple(y.shape)}, h_hat {tuple(h_hat.shape)}, "
                           f"{n_ds} data symbols, {eff_sc.numel()} effective subcarriers")
    ev = _f32("err_var", err_var, B, Nr, Ns, n_sym, n_sc) if err_var.numel() else None
    if ev is not None:
        _dev_check(y, ev)
    x_hat = torch.empty((B, Ns, n_ds * n_sc, 2), dtype=torch.float32, device=dev)
    no_eff = torch.empty((B, Ns, n_ds * n_sc), dtype=torch.float32, device=dev)
    if no_mode not in (0, 1, 2):
        raise RuntimeError(f"no_mode must be 0, 1 or 2, got {no_mode}")
    no_dev = None
    if no_mode != 0:
        _dev_check(y, no)
        no_dev = _f32("no", no, B) if no_mode == 1 else _f32("no", no, B, Nr)
    with torch.cuda.device(dev):
        rc = _cabi.lib().cet_lmmse_grid(_ptr(y), _ptr(h_hat), _ptr(ev), no_mode, ctypes.c_float(no_scalar),
                                        _ptr(no_dev), _ptr(data_sym), _ptr(eff_sc), _ptr(x_hat),
                                        _ptr(no_eff), B, Nr, Ns, n_sym, fft, n_sc, n_ds,
                                        _cabi.current_stream_ptr(dev))
    _cabi.check(rc, "cet_lmmse_grid")
    return x_hat, no_eff


@lmmse_grid.register_fake
def _(y, h_hat, err_var, no, no_scalar, no_mode, data_sym, eff_sc):
    B, Ns, n = y.shape[0], h_hat.shape[2], data_sym.numel() * h_hat.shape[4]
    return y.new_empty((B, Ns, n, 2)), y.new_empty((B, Ns, n))


# -- sequence operators -----------------------------------------------------------------------

_SEQ_TYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}


def _seq_check(name, t, dtype, *shape):
    """A tensor of the call's type and of this shape (None = any size in that position) whose last axis
    is contiguous."""
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {dtype}, got {t.dtype}")
    have = t.shape
    if have != shape and (len(have) != len(shape) or any(s is not None and s != d for s, d in zip(shape, have))):
        raise RuntimeError(f"{name} must have shape {list(shape)}, got {list(have)}")
    return t if have[-1] > 1 and t.stride(-1) == 1 else _rows(t)


def _rows(t):
    """A contiguous last axis, and values as they lie in memory: the imaginary part of a conjugate is a view with a flag that
    turns its sign (a copy does so, and every view of more than one such value in a row is copied)."""
    return t.contiguous() if t.shape[-1] > 1 else t.resolve_neg()


def _seq_first(name, t, dim):
    """The tensor that gives a call its type and sizes."""
    have = t.shape
    if len(have) != dim:
        raise RuntimeError(f"{name} must have shape {[None] * dim}, got {list(have)}")
    return t if have[-1] > 1 and t.stride(-1) == 1 else _rows(t)


def _seq_type(t):
    if t.dtype not in _SEQ_TYPES:
        raise RuntimeError(f"float32, bfloat16 or float16 tensors are served, got {t.dtype}")
    return _SEQ_TYPES[t.dtype]


def _index(name, t, n):
    """An int32 / int64 [n] table -> (contiguous, holds int64)."""
    if t.dtype not in (torch.int32, torch.int64) or t.dim() != 1 or t.shape[0] != n:
        raise RuntimeError(f"{name} must be int32 or int64 [{n}], got {t.dtype} {list(t.shape)}")
    return t.contiguous(), int(t.dtype == torch.int64)


def _linattn(q, k, v, log_decay, scale, initial_state, lengths, d_o=None):
    """Checked operands of the linear attention calls and their descriptor."""
    dev = _dev_check(*[t for t in (q, k, v, log_decay, initial_state, lengths, d_o) if t is not None])
    code = _seq_type(q)
    q = _seq_first("q", q, 4)
    B, T, H, K = q.shape
    if T > 1 << 30 or B * H > 1 << 22:  # (the descriptor holds 32 bits of each)
        raise RuntimeError(f"up to 2^30 slots and 2^22 heads of all sequences are served, got {T} and {B} x {H}")
    k = _seq_check("k", k, q.dtype, B, T, H, K)
    v = _seq_check("v", v, q.dtype, B, T, H, None)
    V = v.shape[3]
    if not (1 <= K <= 256 and 1 <= V <= 256):
        raise RuntimeError(f"head sizes from 1 to 256 are served, got K = {K}, V = {V}")
    if not math.isfinite(scale):
        raise RuntimeError(f"scale must be finite, got {scale}")
    log_decay = _f32("log_decay", log_decay, H)
    if initial_state is not None:
        initial_state = _f32("initial_state", initial_state, B, H, K, V)
    wide = 0
    if lengths is not None:
        lengths, wide = _index("lengths", lengths, B)
    if d_o is not None:
        d_o = _seq_check("d_o", d_o, q.dtype, B, T, H, V)
    d = _cabi.LinattnDesc(code, B, T, H, K, V, wide, scale)
    d.q[:], d.k[:], d.v[:] = q.stride()[:3], k.stride()[:3], v.stride()[:3]
    if d_o is not None:
        d.d_o[:] = d_o.stride()[:3]
    return dev, d, q, k, v, log_decay, initial_state, lengths, d_o


def _workspace(n, dev):
    return torch.empty((n,), dtype=torch.uint8, device=dev) if n else None


def _at(t):
    """Address of a tensor's first element (None without one), as the C entry points take it."""
    return t.data_ptr() or None if t is not None else None


_HERE = contextlib.nullcontext()
_TWO = ctypes.c_int64 * 2


def _on(dev):
    """`dev` as the current device; nothing to do, and no time spent, where it is already."""
    return _HERE if torch.cuda.current_device() == dev.index else torch.cuda.device(dev)


def _stream(dev):
    return torch._C._cuda_getCurrentRawStream(dev.index)  # torch.cuda.current_stream without the object (1.5 us)


def run_linear_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float,
                         initial_state: Optional[torch.Tensor] = None, lengths: Optional[torch.Tensor] = None,
                         keep: bool = False) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """q, k [B,T,H,K], v [B,T,H,V] -> o [B,T,H,V], state float32 [B,H,K,V], and with `keep` the states between
    segments of a long time axis for the backward call (else empty)."""
    dev, d, q, k, v, log_decay, s0, lengths, _ = _linattn(q, k, v, log_decay, scale, initial_state, lengths)
    o = q.new_empty((d.B, d.T, d.H, d.V))
    state = torch.empty((d.B, d.H, d.K, d.V), dtype=torch.float32, device=dev)
    L = _cabi.lib()
    with _on(dev):
        kept = L.cet_linear_attention_states(d) if keep else 0
        segments = torch.empty((kept // 4,), dtype=torch.float32, device=dev)
        n = L.cet_linear_attention_workspace(d, _at(q), _at(k), _at(v), None, 0) - kept
        ws = _workspace(n, dev)
        rc = L.cet_linear_attention(d, _at(q), _at(k), _at(v), _at(log_decay), _at(s0), _at(lengths), _at(o), _at(state),
                                    _at(segments), _at(ws), n, _stream(dev))
    _cabi.check(rc, "cet_linear_attention")
    return o, state, segments


linear_attention = torch.library.custom_op("cet::linear_attention", mutates_args=())(run_linear_attention)


@linear_attention.register_fake
def _(q, k, v, log_decay, scale, initial_state=None, lengths=None, keep=False):
    B, T, H, K = q.shape
    segments = torch.library.get_ctx().new_dynamic_size() if keep else 0
    return (q.new_empty((B, T, H, v.shape[3])), q.new_empty((B, H, K, v.shape[3]), dtype=torch.float32),
            q.new_empty((segments,), dtype=torch.float32))


def run_linear_attention_backward(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor, scale: float,
                                  initial_state: Optional[torch.Tensor], lengths: Optional[torch.Tensor],
                                  segments: Optional[torch.Tensor], d_o: torch.Tensor, d_state: Optional[torch.Tensor],
                                  want_initial: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> dq, dk, dv, d_initial (empty unless `want_initial`). `segments`: what the forward call on the same
    operands kept (None: formed again)."""
    dev, d, q, k, v, log_decay, s0, lengths, d_o = _linattn(q, k, v, log_decay, scale, initial_state, lengths, d_o)
    if d_state is not None:
        _dev_check(q, d_state)
        d_state = _f32("d_state", d_state, d.B, d.H, d.K, d.V)
    dq, dk, dv = q.new_empty(q.shape), q.new_empty(q.shape), q.new_empty(v.shape)
    ds = torch.empty((d.B, d.H, d.K, d.V) if want_initial else (0,), dtype=torch.float32, device=dev)
    L = _cabi.lib()
    with _on(dev):
        kept = 0
        if segments is not None and segments.numel():
            _dev_check(q, segments)
            kept = L.cet_linear_attention_states(d)
            segments = _f32("segments", segments, kept // 4)
        n = L.cet_linear_attention_workspace(d, _at(q), _at(k), _at(v), _at(d_o), 1) - kept
        ws = _workspace(n, dev)
        rc = L.cet_linear_attention_backward(d, _at(q), _at(k), _at(v), _at(log_decay), _at(s0), _at(lengths), _at(segments),
                                             _at(d_o), _at(d_state), _at(dq), _at(dk), _at(dv), _at(ds), _at(ws), n,
                                             _stream(dev))
    _cabi.check(rc, "cet_linear_attention_backward")
    return dq, dk, dv, ds


linear_attention_backward = torch.library.custom_op("cet::linear_attention_backward", mutates_args=())(
    run_linear_attention_backward)


@linear_attention_backward.register_fake
def _(q, k, v, log_decay, scale, initial_state, lengths, segments, d_o, d_state, want_initial):
    B, T, H, K = q.shape
    shape = (B, H, K, v.shape[3]) if want_initial else (0,)
    return (q.new_empty(q.shape), k.new_empty(k.shape), v.new_empty(v.shape), q.new_empty(shape, dtype=torch.float32))


def _linattn_setup(ctx, inputs, output):
    q, k, v, log_decay, scale, initial_state, lengths, keep = inputs
    if ctx.needs_input_grad[3]:
        raise RuntimeError("log_decay is a constant of linear_attention: it has no gradient (detach it)")
    ctx.save_for_backward(q, k, v, log_decay, initial_state, lengths, output[2] if keep else None)
    ctx.scale = scale
    ctx.set_materialize_grads(False)


def _linattn_backward(ctx, d_o, d_state, _, run=linear_attention_backward):
    q, k, v, log_decay, s0, lengths, segments = ctx.saved_tensors
    if d_o is None:
        if d_state is None:
            return (None,) * 8
        d_o = q.new_zeros((*q.shape[:3], v.shape[3]))
    want = s0 is not None and ctx.needs_input_grad[5]
    dq, dk, dv, ds = run(q, k, v, log_decay, ctx.scale, s0, lengths, segments, d_o, d_state, want)
    return dq, dk, dv, None, None, ds if want else None, None, None


linear_attention.register_autograd(_linattn_backward, setup_context=_linattn_setup)


class LinearAttention(torch.autograd.Function):
    """The same operator without the dispatcher (eager calls on plain tensors: a third of the host time; a forward
    that takes `ctx` saves the binding of its arguments, 12 us)."""

    @staticmethod
    def forward(ctx, *args):
        output = run_linear_attention(*args)
        _linattn_setup(ctx, args, output)
        ctx.mark_non_differentiable(output[2])
        return output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_state, _):
        return _linattn_backward(ctx, d_o, d_state, None, run_linear_attention_backward if direct_gradient(d_o, d_state) else linear_attention_backward)


def _step(q, k, v, log_decay, state, out_state, scale, slots):
    dev = _dev_check(q, k, v, log_decay, state) if slots is None else _dev_check(q, k, v, log_decay, state, slots)
    code = _seq_type(q)
    q = _seq_first("q", q, 3)
    B, H, K = q.shape
    if B * H > 1 << 21:
        raise RuntimeError(f"up to 2^21 heads of all streams are served, got {B} x {H}")
    k = _seq_check("k", k, q.dtype, B, H, K)
    v = _seq_check("v", v, q.dtype, B, H, None)
    V = v.shape[2]
    if not (1 <= K <= 256 and 1 <= V <= 256):
        raise RuntimeError(f"head sizes from 1 to 256 are served, got K = {K}, V = {V}")
    log_decay = _f32("log_decay", log_decay, H)
    if slots is not None:
        slots, wide = _index("slots", slots, B)
        rows = state.shape[0]
        if rows >= 1 << 31:
            raise RuntimeError(f"pools of up to 2^31 - 1 states are served, got {rows}")
    o = q.new_empty((B, H, V))
    strides = [_TWO(*t.stride()[:2]) for t in (q, k, v)]
    L = _cabi.lib()
    with _on(dev):
        if slots is None:
            rc = L.cet_linear_attention_step(
                code, B, H, K, V, *strides, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), scale,
                state.data_ptr(), out_state.data_ptr(), B, None, 0, o.data_ptr(), _stream(dev))
        else:
            n = L.cet_linear_attention_step_pool_workspace(B, rows)
            ws = _workspace(n, dev)
            rc = L.cet_linear_attention_step_pool(
                code, B, H, K, V, *strides, q.data_ptr(), k.data_ptr(), v.data_ptr(), log_decay.data_ptr(), scale,
                state.data_ptr(), rows, slots.data_ptr(), wide, o.data_ptr(), _at(ws), n, _stream(dev))
    _cabi.check(rc, "cet_linear_attention_step")
    return o


def run_linear_attention_step(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                          state: torch.Tensor, scale: float) -> tuple[torch.Tensor, torch.Tensor]:
    """q, k [B,H,K], v [B,H,V], state float32 [B,H,K,V] -> o [B,H,V], the next state."""
    if q.dim() != 3 or v.dim() != 3:
        raise RuntimeError(f"q, k, v must be [B, H, features], got {list(q.shape)}, {list(v.shape)}")
    state = _f32("state", state, q.shape[0], q.shape[1], q.shape[2], v.shape[2])
    out = torch.empty_like(state)
    return _step(q, k, v, log_decay, state, out, scale, None), out


linear_attention_step = torch.library.custom_op("cet::linear_attention_step", mutates_args=())(run_linear_attention_step)


@linear_attention_step.register_fake
def _(q, k, v, log_decay, state, scale):
    return v.new_empty(v.shape), state.new_empty(state.shape)


def run_linear_attention_step_(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, log_decay: torch.Tensor,
                           state: torch.Tensor, scale: float, slots: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The same with the state (with `slots`: a pool of them) updated in place."""
    if q.dim() != 3 or v.dim() != 3:
        raise RuntimeError(f"q, k, v must be [B, H, features], got {list(q.shape)}, {list(v.shape)}")
    want = (None if slots is not None else q.shape[0], q.shape[1], q.shape[2], v.shape[2])
    if state.dtype != torch.float32 or not state.is_contiguous() or state.dim() != 4 or any(
            w is not None and s != w for s, w in zip(state.shape, want)) or (state.numel() == 1 and state.is_neg()):
        raise RuntimeError(f"state must be contiguous float32 {list(want)}, got {state.dtype} {list(state.shape)}")
    return _step(q, k, v, log_decay, state, state, scale, slots)


linear_attention_step_ = torch.library.custom_op("cet::linear_attention_step_", mutates_args=("state",))(run_linear_attention_step_)


@linear_attention_step_.register_fake
def _(q, k, v, log_decay, state, scale, slots=None):
    return v.new_empty(v.shape)


def run_rotary(q: torch.Tensor, k: Optional[torch.Tensor], positions: torch.Tensor, inv_freq: torch.Tensor, interleaved: bool,
           gain: float, inverse: bool) -> tuple[torch.Tensor, torch.Tensor]:
    """q [B,T,Hq,D], k [B,T,Hk,D] or None, positions int32 / int64 [T] or [B,T], inv_freq float64 [pairs]
    -> the turned q and k (empty without k)."""
    dev = _dev_check(q, positions, inv_freq) if k is None else _dev_check(q, k, positions, inv_freq)
    code = _seq_type(q)
    q = _seq_first("q", q, 4)
    B, T, Hq, D = q.shape
    if k is not None:
        k = _seq_check("k", k, q.dtype, B, T, None, D)
    if inv_freq.dtype != torch.float64 or inv_freq.dim() != 1 or not 1 <= inv_freq.shape[0] <= D // 2:
        raise RuntimeError(f"inv_freq must be float64 [pairs] with 1 <= pairs <= D / 2, got {inv_freq.dtype} "
                           f"{list(inv_freq.shape)} for D = {D}")
    inv_freq = inv_freq.contiguous()
    if positions.dtype not in (torch.int32, torch.int64) or positions.shape not in ((T,), (B, T)):
        raise RuntimeError(f"positions must be int32 or int64 [{T}] or [{B}, {T}], got {positions.dtype} {list(positions.shape)}")
    if not math.isfinite(gain):
        raise RuntimeError(f"gain must be finite, got {gain}")
    Hk = 0 if k is None else k.shape[2]
    if B * T > 2 * 10 ** 9 or Hq > 65536 or Hk > 65536:
        raise RuntimeError(f"up to 2e9 slots and 65536 heads are served, got {B} x {T}, {Hq} and {Hk}")
    if D > 1024:
        raise RuntimeError(f"heads of up to 1024 features are served, got D = {D}")
    d = _cabi.RotaryDesc(code, B, T, Hq, Hk, D, inv_freq.shape[0], int(interleaved), int(positions.dtype == torch.int64), gain)
    d.q[:] = q.stride()[:3]
    if k is not None:
        d.k[:] = k.stride()[:3]
    d.pos[:] = positions.stride() if positions.dim() == 2 else (0, positions.stride(0))
    qo = q.new_empty((B, T, Hq, D))
    ko = q.new_empty((B, T, Hk, D) if k is not None else (0,))
    with _on(dev):
        rc = _cabi.lib().cet_rotary(d, q.data_ptr(), _at(k), positions.data_ptr(), inv_freq.data_ptr(), int(inverse),
                                    qo.data_ptr(), ko.data_ptr(), _stream(dev))
    _cabi.check(rc, "cet_rotary")
    return qo, ko


rotary = torch.library.custom_op("cet::rotary", mutates_args=())(run_rotary)


@rotary.register_fake
def _(q, k, positions, inv_freq, interleaved, gain, inverse):
    return q.new_empty(q.shape), q.new_empty(k.shape if k is not None else (0,))


def _rotary_setup(ctx, inputs, output):
    q, k, positions, inv_freq, ctx.interleaved, ctx.gain, ctx.inverse = inputs
    ctx.save_for_backward(positions, inv_freq)
    ctx.set_materialize_grads(False)


def _rotary_backward(ctx, dq, dk, run=rotary):
    positions, inv_freq = ctx.saved_tensors
    if not ctx.needs_input_grad[1]:
        dk = None
    if not ctx.needs_input_grad[0]:
        dq = None
    turn = lambda a, b: run(a, b, positions, inv_freq, ctx.interleaved, ctx.gain, not ctx.inverse)  # noqa: E731
    if dq is None:
        dk = turn(dk, None)[0] if dk is not None else None
    elif dk is None:
        dq = turn(dq, None)[0]
    else:
        dq, dk = turn(dq, dk)
    return dq, dk, None, None, None, None, None


rotary.register_autograd(_rotary_backward, setup_context=_rotary_setup)


class Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        output = run_rotary(*args)
        _rotary_setup(ctx, args, output)
        return output

    @staticmethod
    def backward(ctx, dq, dk):
        return _rotary_backward(ctx, dq, dk, direct_rotary if direct_gradient(dq, dk) else rotary)


def direct_rotary(q, k, *rest):
    grad = torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad))
    return (Rotary.apply if grad else run_rotary)(q, k, *rest)


GATED_ACTIVATIONS = {"silu": 0, "gelu": 1, "relu": 2}


def _gated(x, w_gate, w_up, b_gate, b_up, activation, dy=None):
    """Checked operands of the gated projection and their descriptor; x and dy as matrices."""
    dev = _dev_check(*[t for t in (x, w_gate, w_up, b_gate, b_up, dy) if t is not None])
    code = _seq_type(x)
    if activation not in GATED_ACTIVATIONS:
        raise RuntimeError(f"activation must be one of {sorted(GATED_ACTIVATIONS)}, got {activation!r}")
    x = _seq_first("x", x, 2)
    N, D = x.shape
    w_gate = _seq_check("w_gate", w_gate, x.dtype, None, D)
    F = w_gate.shape[0]
    w_up = _seq_check("w_up", w_up, x.dtype, F, D)
    if D < 1 or F < 1 or D > 1 << 20 or F > 1 << 20 or N > 1 << 28:
        raise RuntimeError(f"x [N, D] and weights [F, D] with N up to 2^28, D and F from 1 to 2^20 are served, got {N}, {D}, {F}")
    b_gate = None if b_gate is None else _seq_check("b_gate", b_gate, x.dtype, F)
    b_up = None if b_up is None else _seq_check("b_up", b_up, x.dtype, F)
    if dy is not None:
        dy = _seq_check("dy", dy, x.dtype, N, F)
    d = _cabi.GatedDesc(code, GATED_ACTIVATIONS[activation], N, D, F, x.stride(0), w_gate.stride(0), w_up.stride(0),
                        0 if dy is None else dy.stride(0))
    return dev, d, x, w_gate, w_up, b_gate, b_up, dy


def run_gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor],
                 b_up: Optional[torch.Tensor], activation: str) -> torch.Tensor:
    """x [N,D], w_gate, w_up [F,D], b_gate, b_up [F] or None -> act(x w_gate^T + b_gate) * (x w_up^T + b_up) [N,F]."""
    dev, d, x, w_gate, w_up, b_gate, b_up, _ = _gated(x, w_gate, w_up, b_gate, b_up, activation)
    out = x.new_empty((d.N, d.F))
    L = _cabi.lib()
    with _on(dev):
        n = L.cet_gated_linear_workspace(d, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), 0)
        ws = _workspace(n, dev)
        rc = L.cet_gated_linear(d, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _at(b_gate), _at(b_up), out.data_ptr(), _at(ws), n,
                                _stream(dev))
    _cabi.check(rc, "cet_gated_linear")
    return out


gated_linear = torch.library.custom_op("cet::gated_linear", mutates_args=())(run_gated_linear)


@gated_linear.register_fake
def _(x, w_gate, w_up, b_gate, b_up, activation):
    return x.new_empty((x.shape[0], w_gate.shape[0]))


def run_gated_linear_backward(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, b_gate: Optional[torch.Tensor],
                          b_up: Optional[torch.Tensor], activation: str, dy: torch.Tensor, want_x: bool, want_w: bool,
                          want_b: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """-> dx, dw_gate, dw_up, db_gate, db_up; empty where not wanted."""
    dev, d, x, w_gate, w_up, b_gate, b_up, dy = _gated(x, w_gate, w_up, b_gate, b_up, activation, dy)
    new = lambda want, *shape: x.new_empty(shape if want else (0,))  # noqa: E731
    dx, dw_gate, dw_up = new(want_x, d.N, d.D), new(want_w, d.F, d.D), new(want_w, d.F, d.D)
    db_gate, db_up = new(want_b, d.F), new(want_b, d.F)
    L = _cabi.lib()
    with _on(dev):
        n = L.cet_gated_linear_workspace(d, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), 1)
        ws = _workspace(n, dev)
        rc = L.cet_gated_linear_backward(
            d, x.data_ptr(), w_gate.data_ptr(), w_up.data_ptr(), _at(b_gate), _at(b_up), dy.data_ptr(), dx.data_ptr(),
            dw_gate.data_ptr(), dw_up.data_ptr(), db_gate.data_ptr(), db_up.data_ptr(), _at(ws), n, _stream(dev))
    _cabi.check(rc, "cet_gated_linear_backward")
    return dx, dw_gate, dw_up, db_gate, db_up


gated_linear_backward = torch.library.custom_op("cet::gated_linear_backward", mutates_args=())(run_gated_linear_backward)


@gated_linear_backward.register_fake
def _(x, w_gate, w_up, b_gate, b_up, activation, dy, want_x, want_w, want_b):
    shapes = ((want_x, x.shape), (want_w, w_gate.shape), (want_w, w_up.shape), (want_b, w_gate.shape[:1]), (want_b, w_up.shape[:1]))
    return tuple(x.new_empty(s if want else (0,)) for want, s in shapes)


def _gated_setup(ctx, inputs, output):
    x, w_gate, w_up, b_gate, b_up, ctx.activation = inputs
    ctx.save_for_backward(x, w_gate, w_up, b_gate, b_up)


def _gated_backward(ctx, dy, run=gated_linear_backward):
    x, w_gate, w_up, b_gate, b_up = ctx.saved_tensors
    need = ctx.needs_input_grad
    dx, dwg, dwu, dbg, dbu = run(
        x, w_gate, w_up, b_gate, b_up, ctx.activation, dy, need[0], need[1] or need[2], need[3] or need[4])
    return tuple(t if n else None for t, n in zip((dx, dwg, dwu, dbg, dbu), need)) + (None,)


gated_linear.register_autograd(_gated_backward, setup_context=_gated_setup)


class GatedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, *args):
        output = run_gated_linear(*args)
        _gated_setup(ctx, args, output)
        return output

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        return _gated_backward(ctx, dy, run_gated_linear_backward if direct_gradient(dy) else gated_linear_backward)


_PLAIN = {torch.Tensor, torch.nn.Parameter, type(None)}


def step_in_place(q, k, v, log_decay, state, scale, slots):
    """run_linear_attention_step_, and autograd told of the write as the dispatcher would."""
    o = run_linear_attention_step_(q, k, v, log_decay, state, scale, slots)
    torch.autograd.graph.increment_version(state)
    return o


_compiling, _tracing = torch.compiler.is_compiling, torch._C._is_tracing
_dispatch_modes, _function_modes = torch._C._len_torch_dispatch_stack, torch._C._len_torch_function_stack


def _modes():
    """Whether a mode wants to see the calls (a default device does not)."""
    return any(not isinstance(torch._C._get_function_stack_at(n), torch.utils._device.DeviceContext)
               for n in range(_function_modes()))


def direct(*tensors):
    """Whether a call may pass the dispatcher by: eager, on plain tensors, with no tracer and no mode active (they
    would see the allocations of the results and not what fills them)."""
    if _compiling() or _tracing() or _dispatch_modes() or (_function_modes() and _modes()):
        return False
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError("forward-mode differentiation is not supported")  # the tangents would be dropped in silence
    for t in tensors:
        if type(t) not in _PLAIN:
            return False
    return True


def direct_gradient(*tensors):
    """The same for gradients on their way back, in fewer questions (the engine's thread takes twice as long for each)."""
    if _dispatch_modes() or _function_modes() or _tracing():
        return False
    for t in tensors:
        if type(t) not in _PLAIN:
            return False
    return True


def wants_grad(*tensors):
    if torch.is_grad_enabled():
        for t in tensors:
            if t is not None and t.requires_grad:
                return True
    return False
