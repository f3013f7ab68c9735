"""Linear attention within bounds that leave no room for operands of fewer bits.

An output or gradient element is off by one rounding to the tensors' type and by (K + T + 64) fp32 roundings of the sum of
the terms' absolute values (the same recurrence on absolute values, "mass"). In bfloat16 every term of the sum holds a score or a
state that enters the matrix instructions in two bfloat16 terms: the first leaves 2^-8 of it, the second 2^-8 of
that, 2^-16 of the mass. 1 % on top for products of errors."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref
from test_gpu_linear_attention import gpu, make, within

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


@pytest.mark.parametrize("shape", [(2, 40, 2, 16, 16), (2, 100, 2, 24, 40), (2, 65, 2, 64, 64), (1, 33, 3, 128, 128), (2, 130, 2, 100, 130),
                                   (1, 200, 2, 40, 200), (1, 97, 1, 160, 50), (2, 70, 1, 192, 256), (1, 300, 1, 256, 256), (3, 500, 1, 64, 16)])
def test_bfloat16_is_rounded_once(shape):
    """Scores and states keep more bits than the tensors, in the outputs and in all gradients."""
    check(make(*shape, torch.bfloat16, seed=sum(shape)), torch.bfloat16)
