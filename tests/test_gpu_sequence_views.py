"""Operands of the sequence operators that are real parts of complex channels: the imaginary part of a conjugate is a
view whose values lie in memory with the other sign."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref

pytestmark = pytest.mark.gpu


def parts(*shape, seed=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(*shape, dtype=torch.complex64, generator=g).cuda().conj().imag


@pytest.mark.parametrize("K, V", [(1, 1), (1, 8), (8, 1), (4, 4)])
def test_attention_of_imaginary_parts(K, V):
    B, T, H = 2, 9, 3
    q, k, v, dec = parts(B, T, H, K, seed=1), parts(B, T, H, K, seed=2), parts(B, T, H, V, seed=3), ref.geometric(H).cuda()
    if K == 1 and V == 1:
        q, k, v = (parts(B, T, H, seed=s).unsqueeze(-1) for s in (1, 2, 3))
    assert q.is_neg() and v.is_neg()
    plain = [t.clone() for t in (q, k, v)]
    for got, want in zip(cet.linear_attention(q, k, v, dec), cet.linear_attention(*plain, dec)):
        assert torch.equal(got, want)
    state = torch.randn(B, H, K, V, device="cuda")
    got, want = (cet.linear_attention_step(*(t[:, 0] for t in x), dec, state) for x in ((q, k, v), plain))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    leaves = [t.requires_grad_() for t in plain]
    o, _ = cet.linear_attention(*leaves, dec)
    d = parts(B, T, H, V, seed=4) if V > 1 else parts(B, T, H, seed=4).unsqueeze(-1)
    for got, want in zip(torch.autograd.grad(o, leaves, d, retain_graph=True), torch.autograd.grad(o, leaves, d.clone())):
        assert torch.equal(got, want)


def test_a_single_decay_and_state():
    q = torch.randn(1, 4, 1, 1, device="cuda")
    dec, s0 = parts(1, seed=5), parts(1, 1, 1, 1, seed=6)
    assert dec.is_neg() and s0.is_neg()
    got, want = cet.linear_attention(q, q, q, dec, initial_state=s0), cet.linear_attention(q, q, q, dec.clone(), initial_state=s0.clone())
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    with pytest.raises(RuntimeError, match="state"):
        cet.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], dec, s0, inplace=True)


@pytest.mark.parametrize("N, D, F", [(20, 1, 5), (20, 5, 1), (100, 1, 70), (100, 70, 1)])
def test_projection_of_imaginary_parts(N, D, F):
    x, w = (parts(*s, seed=n) for n, s in enumerate(((N, D), (F, D))))
    if D == 1:
        x, w = parts(N, seed=7).unsqueeze(-1), parts(F, seed=8).unsqueeze(-1)
    b = parts(F, seed=9)
    assert torch.equal(cet.gated_linear(x, w, w, b, b), cet.gated_linear(*(t.clone() for t in (x, w, w, b, b))))
