"""Linear attention within bounds that leave no room for operands of fewer bits, and with heads that remember
thousands of slots.

An output or gradient element is off by one rounding to the tensors' type and by (K + T + 64) fp32 roundings of the sum of
the terms' absolute values (the same recurrence on absolute values, "mass"). In bfloat16 every term of the sum holds a score or a
state that enters the matrix instructions in two bfloat16 terms: the first leaves 2^-8 of it, the second 2^-8 of
that, 2^-16 of the mass. 1 % on top for products of errors."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref
from channelestimationtransformer_amd import _cabi
from test_gpu_linear_attention import TYPES, gpu, make, within

pytestmark = pytest.mark.gpu


def expected(x, scale, dtype, T, K):
    a = {n: t.abs() if torch.is_tensor(t) and n not in ("lengths", "g") else t for n, t in x.items()}
    want = ref.linear_attention_with_gradients(x["q"], x["k"], x["v"], x["g"], scale, x["s0"], x["lengths"], x["d_o"], x["d_state"])
    mass = ref.linear_attention_with_gradients(a["q"], a["k"], a["v"], a["g"], scale, a["s0"], a["lengths"], a["d_o"], a["d_state"])
    c = (K + T + 64) * 2.0 ** -24
    inner = 2.0 ** -16 if dtype == torch.bfloat16 else 0.0
    tiny = 1e-30 + (1e-7 if dtype == torch.float16 else 0.0)
    typed = lambda w, m: 1.01 * (ref.half_step(dtype) * w.abs() + (inner + c) * m) + tiny  # noqa: E731
    whole = lambda m: 1.01 * c * m + 1e-30  # noqa: E731
    lim = [typed(want[0], mass[0]), whole(mass[1])] + [typed(w, m) if j < 3 else whole(m) for j, (w, m) in enumerate(zip(want[2], mass[2]))]
    return [want[0], want[1], *want[2]], lim


def check(x, dtype, y=None, pick=None):
    """`pick`: the sequences that are compared (all are computed)."""
    T, K = x["q"].shape[1], x["q"].shape[3]
    y = gpu(x, dtype) if y is None else y
    leaves = [y[n].detach().requires_grad_() for n in ("q", "k", "v", "s0") if y[n] is not None]
    out = cet.linear_attention(*leaves[:3], y["g"], initial_state=leaves[3] if len(leaves) > 3 else None, lengths=y["lengths"])
    got = [*out, *torch.autograd.grad(out, leaves, (y["d_o"], y["d_state"]))]
    if pick is not None:
        x = {n: t[pick] if torch.is_tensor(t) and n != "g" else t for n, t in x.items()}
        got = [t[pick] for t in got]
    want, lim = expected(x, ref.sqrt_scale(K), dtype, T, K)
    for n, a, b, c in zip(("o", "state", "dq", "dk", "dv", "d_initial"), got, want, lim):
        within(a.detach(), b, c, n)


def segments(dtype, B, T, H, K, V):
    d = _cabi.LinattnDesc({torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dtype], B, T, H, K, V, 0, 1.0)
    return _cabi.lib().cet_linear_attention_states(d) > 0


@pytest.mark.parametrize("shape", [(2, 40, 2, 16, 16), (2, 100, 2, 24, 40), (2, 65, 2, 64, 64), (1, 33, 3, 128, 128), (2, 130, 2, 100, 130),
                                   (1, 200, 2, 40, 200), (1, 97, 1, 160, 50), (2, 70, 1, 192, 256), (1, 300, 1, 256, 256), (3, 500, 1, 64, 16)])
def test_bfloat16_is_rounded_once(shape):
    """Scores and states keep more bits than the tensors, in the outputs and in all gradients."""
    check(make(*shape, torch.bfloat16, seed=sum(shape)), torch.bfloat16)

SLOW = torch.log1p(-torch.exp2(-torch.tensor([8.0, 9.0, 10.0, 12.0])))  # 256 to 4096 slots


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("ragged", [False, True])
@pytest.mark.parametrize("K, V", [(24, 40), (128, 128), (16, 8)])
def test_far_weights_over_segments(K, V, ragged, dtype):
    """The time axis cut into segments whose joined states still weigh in the outputs, the last state and its
    gradient; one head forgets nothing."""
    B, T = (2, 1100) if K < 128 else (1, 700)
    x = make(B, T, 5, K, V, dtype, seed=K + V, ragged=ragged)
    x["g"] = torch.cat([SLOW, torch.zeros(1)])
    if ragged:
        x["lengths"][0] = T - 37
    assert segments(dtype, B, T, 5, K, V)
    check(x, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B, K, V", [(128, 20, 40), (128, 100, 33), (512, 40, 16)])
def test_a_state_multiplied_out_within_a_segment(B, K, V, dtype):
    """Enough heads that the axis is not cut: decays that make the kept state's factor leave its range
    several times, once, and never within the history."""
    T, pick = 700, [0, B // 2, B - 1]
    g = torch.Generator().manual_seed(B + K)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = {"q": r(B, T, 4, K), "k": r(B, T, 4, K), "v": r(B, T, 4, V), "d_o": r(B, T, 4, V)}
    x = {n: t.to(dtype) for n, t in x.items()}
    x.update(s0=r(B, 4, K, V), d_state=r(B, 4, K, V), lengths=torch.randint(0, T + 1, (B,), generator=g),
             g=torch.cat([torch.log(torch.tensor([0.75, 0.97])), SLOW[:1], torch.zeros(1)]))
    x["lengths"][pick[0]], x["lengths"][pick[1]] = T, T - 19
    assert not segments(dtype, B, T, 4, K, V)
    y = {n: t.cuda() for n, t in x.items()}
    check({n: t.double() if n not in ("g", "lengths") else t for n, t in x.items()}, dtype, y=y, pick=pick)
