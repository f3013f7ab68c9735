"""The sequence operators under tracers and modes: a call has to be recorded as an operator (the direct call into the C
library would leave nothing in the record but its allocations). The CPU tests put a stand-in in the library's
place; the GPU test replays what was traced with other inputs."""
import contextlib

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx
from torch.overrides import TorchFunctionMode
from torch.utils._python_dispatch import TorchDispatchMode

import channelestimationtransformer_amd as cet
import seq_ref as ref
from channelestimationtransformer_amd import _cabi, ops


class Library:
    """Every entry point succeeds and needs no workspace."""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def stand_in(monkeypatch):
    monkeypatch.setattr(ops, "_dev_check", lambda *tensors: tensors[0].device)
    monkeypatch.setattr(ops, "_on", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(ops, "_stream", lambda dev: None)
    monkeypatch.setattr(_cabi, "lib", Library)


def calls(dev):
    """name of the operator -> (function of one tensor, such a tensor, none of those that the function holds)"""
    g = torch.Generator().manual_seed(0)
    q, x, w = (torch.randn(*s, generator=g).to(dev) for s in ((2, 5, 3, 8), (6, 8), (4, 8)))
    decay, state = ref.geometric(3).to(dev), torch.randn(2, 3, 8, 8, generator=g).to(dev)
    pos, f = torch.arange(5, device=dev), cet.rotary_frequencies(8, device=dev)[0]

    def in_place(t):
        s = state.clone()
        return cet.linear_attention_step(t, q[:, 1], q[:, 2], decay, s, inplace=True)[0] + s.sum()

    return {"cet::linear_attention": (lambda t: cet.linear_attention(t, q, q, decay)[0], q.clone()),
            "cet::linear_attention_step": (lambda t: cet.linear_attention_step(t, q[:, 1], q[:, 2], decay, state)[0], q[:, 0].clone()),
            "cet::linear_attention_step_": (in_place, q[:, 0].clone()),
            "cet::rotary": (lambda t: cet.rotary(t, q, pos, f)[0], q.clone()),
            "cet::gated_linear": (lambda t: cet.gated_linear(t, w, w), x.clone())}


NAMES = list(calls("cpu"))


def recorded(graph):
    return [n.target.name().split(".")[0] for n in graph.graph.nodes if n.op == "call_function" and isinstance(n.target, torch._ops.OpOverload)]


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("mode", ["real", "fake", "symbolic"])
def test_in_a_graph_of_make_fx(stand_in, name, mode):
    fn, x = calls("cpu")[name]
    assert name in recorded(make_fx(fn, tracing_mode=mode, _allow_non_fake_inputs=True)(x))


@pytest.mark.parametrize("name", NAMES)
def test_in_a_traced_script(stand_in, name):
    fn, x = calls("cpu")[name]
    assert name in {n.kind() for n in torch.jit.trace(fn, (x,), check_trace=False).graph.nodes()}


class Seen(TorchDispatchMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_dispatch__(self, func, types, args=(), kwargs=None):
        self.names.append(func.name().split(".")[0])
        return func(*args, **(kwargs or {}))


class SeenFunctions(TorchFunctionMode):
    def __init__(self):
        super().__init__()
        self.names = []

    def __torch_function__(self, func, types, args=(), kwargs=None):
        self.names.append(str(func).replace(".", "::", 1).split(".")[0])
        return func(*args, **(kwargs or {}))


@pytest.mark.parametrize("name", NAMES)
@pytest.mark.parametrize("mode", [Seen, SeenFunctions])
def test_a_mode_sees_the_call(stand_in, name, mode):
    fn, x = calls("cpu")[name]
    with mode() as seen:
        fn(x)
    assert name in seen.names


@pytest.mark.parametrize("name", ["cet::linear_attention", "cet::rotary", "cet::gated_linear"])
def test_a_mode_sees_the_gradient(stand_in, name):
    """Also where the mode is entered after the forward call."""
    fn, x = calls("cpu")[name]
    out = fn(x.detach().requires_grad_())
    with Seen() as seen:
        out.sum().backward()
    assert {"cet::linear_attention": "cet::linear_attention_backward", "cet::rotary": "cet::rotary",
            "cet::gated_linear": "cet::gated_linear_backward"}[name] in seen.names


def test_the_default_device_is_no_reason_to_dispatch():
    with torch.device("cpu"):
        assert ops.direct(torch.zeros(2))
    assert ops.direct(torch.zeros(2), None)


@pytest.mark.gpu
@pytest.mark.parametrize("name", NAMES)
def test_what_was_traced_computes_with_new_inputs(name):
    fn, x = calls("cuda")[name]
    graph, script = make_fx(fn)(x), torch.jit.trace(fn, (x,), check_trace=False)
    for turn in range(3):
        y = x.flip(0) * (turn + 1) + turn
        want = fn(y)
        assert torch.equal(graph(y), want) and torch.equal(script(y), want)
