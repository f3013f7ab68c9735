"""The sequence operators in a compiled training step: the same bits as eager calls, in one graph."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref

pytestmark = pytest.mark.gpu


def step(x, wq, wg, wu, decay, positions, freq, lengths):
    B, T, _ = x.shape
    q, k, v = (x @ wq).reshape(B, T, 3, 2, 16).unbind(2)
    q, k = cet.rotary(q, k, positions, freq)
    o, state = cet.linear_attention(q, k, v, decay, lengths=lengths)
    return cet.gated_linear(o.reshape(B, T, 32), wg, wu, activation="gelu"), state


@pytest.mark.parametrize("T", [20, 700])  # one segment, and several whose states the forward call keeps
@pytest.mark.parametrize("dynamic", [False, True])
def test_compiled_and_eager(T, dynamic):
    g = torch.Generator().manual_seed(T)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    leaves = [r(2, T, 32), r(32, 96) * 0.2, r(48, 32) * 0.2, r(48, 32) * 0.2]
    rest = ref.geometric(2).cuda(), torch.arange(T, device="cuda"), cet.rotary_frequencies(16)[0], torch.tensor([T, T // 2], device="cuda")
    d = r(2, T, 48), r(2, 2, 16, 16)
    torch._dynamo.reset()
    compiled = torch.compile(step, backend="aot_eager", fullgraph=True, dynamic=dynamic)
    got = []
    for fn in (step, compiled, compiled):
        x = [t.clone().requires_grad_() for t in leaves]
        out = fn(*x, *rest)
        got.append([*out, *torch.autograd.grad(out, x, d)])
    for a, b, c in zip(*got):
        assert torch.equal(a, b) and torch.equal(a, c)
    with torch.no_grad():
        for a, b in zip(step(*leaves, *rest), compiled(*leaves, *rest)):
            assert torch.equal(a, b)
