"""The sequence operators together, as the block of a predictor uses them, and through the dispatcher."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref

pytestmark = pytest.mark.gpu

H, K, D, F = 4, 16, 64, 96


def block(p, x, positions, state, lengths=None, step=False):
    """x [B, T, D] (a step: [B, D]) -> the block's output and the attention state."""
    B = x.shape[0]
    q, k, v = (x @ p["qkv"].t()).reshape(*x.shape[:-1], 3, H, K).unbind(-3)
    if step:
        q, k = (t[:, 0] for t in cet.rotary(q[:, None], k[:, None], positions[:, None], p["f"]))
        o, state = cet.linear_attention_step(q, k, v, p["g"], state)
    else:
        q, k = cet.rotary(q, k, positions, p["f"])
        o, state = cet.linear_attention(q, k, v, p["g"], initial_state=state, lengths=lengths)
    x = x + o.reshape(*x.shape[:-1], H * K) @ p["out"].t()
    return x + cet.gated_linear(x, p["wg"], p["wu"], p["bg"], p["bu"]) @ p["down"].t(), state


def plain_block(p, x, positions, lengths):
    B, T, _ = x.shape
    q, k, v = (x @ p["qkv"].t()).reshape(B, T, 3, H, K).unbind(2)
    f = p["f"]
    angle = positions.double()[..., None] * f
    c, s = angle.cos()[:, :, None], angle.sin()[:, :, None]
    turn = lambda t: torch.cat([t[..., :K // 2] * c - t[..., K // 2:] * s, t[..., :K // 2] * s + t[..., K // 2:] * c], -1)  # noqa: E731
    o, state = ref.linear_attention(turn(q), turn(k), v, p["g"], K ** -0.5, None, lengths)
    x = x + o.reshape(B, T, H * K) @ p["out"].t()
    g, u = x @ p["wg"].t() + p["bg"], x @ p["wu"].t() + p["bu"]
    return x + (torch.nn.functional.silu(g) * u) @ p["down"].t(), state


def parameters(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g) / s[-1] ** 0.5  # noqa: E731
    p = {"qkv": r(3 * H * K, D), "out": r(D, H * K), "wg": r(F, D), "wu": r(F, D), "bg": r(F), "bu": r(F), "down": r(D, F)}
    p["g"] = ref.geometric(H)
    p["f"] = cet.rotary_frequencies(K, device="cpu")[0]
    return p


NAMES = ("qkv", "out", "wg", "wu", "bg", "bu", "down")


def test_a_block_trains_on_ragged_histories():
    """Outputs and every gradient against the float64 block: relative to each tensor's norm within the fp32
    roundings of the longest chain, (T + D + F + 3 D) sums of 2^-24, times the 8 products in a row."""
    p = parameters()
    B, T = 5, 40
    g = torch.Generator().manual_seed(1)
    x, dy = torch.randn(B, T, D, generator=g), torch.randn(B, T, D, generator=g)
    lengths = torch.tensor([40, 1, 17, 33, 0])
    positions = torch.arange(T)[None] + torch.tensor([0, 5, 1000, 30, 2])[:, None]
    dy = ref.clean(dy[:, :, None], lengths)[:, :, 0]
    leaves = {n: p[n].double().requires_grad_() for n in NAMES}
    xd = x.double().requires_grad_()
    want, _ = plain_block({**p, **leaves}, xd, positions, lengths)
    wants = torch.autograd.grad((want * dy).sum(), [xd, *leaves.values()])
    dev = {n: t.cuda() for n, t in p.items()}
    got_leaves = {n: dev[n].clone().requires_grad_() for n in NAMES}
    xg = x.cuda().requires_grad_()
    got, _ = block({**dev, **got_leaves}, xg, positions.cuda(), None, lengths.cuda())
    gots = torch.autograd.grad((got * dy.cuda()).sum(), [xg, *got_leaves.values()])
    lim = 8 * (T + 4 * D + F) * 2.0 ** -24
    live = ref.clean(torch.ones(B, T, 1, 1), lengths)[:, :, 0].bool()
    for a, b, n in zip((torch.where(live, got.cpu(), 0.0), *gots), (torch.where(live, want, 0.0), *wants), ("out", "x", *NAMES)):
        off = float((a.double().cpu() - b).norm() / b.norm())
        assert off <= lim, (n, off, lim)


def test_a_history_and_then_one_slot_at_a_time():
    p = {n: t.cuda() for n, t in parameters().items()}
    B, T, more = 6, 50, 8
    g = torch.Generator().manual_seed(2)
    x = torch.randn(B, T + more, D, generator=g).cuda()
    with torch.no_grad():
        whole, last = block(p, x, torch.arange(T + more, device="cuda"), None)
        y, state = block(p, x[:, :T], torch.arange(T, device="cuda"), None)
        outs = [y]
        for t in range(T, T + more):
            y, state = block(p, x[:, t], torch.full((B,), t, device="cuda"), state, step=True)
            outs.append(y[:, None])
    got = torch.cat(outs, 1)
    lim = 16 * (T + more + 4 * D + F) * 2.0 ** -24  # two computations, each off by the bound of the test above
    assert float((got - whole).norm() / whole.norm()) <= lim and float((state - last).norm() / last.norm()) <= lim


def test_through_the_dispatcher():
    """torch.ops.cet.* (what a traced program calls) and the functions give the same bits; schemas, fake
    shapes and autograd registrations hold."""
    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    q, k, v, s0, dec = r(2, 20, 3, 16), r(2, 20, 3, 16), r(2, 20, 3, 24), r(2, 3, 16, 24), ref.geometric(3).cuda()
    lengths, pos, f = torch.tensor([20, 7], device="cuda"), torch.arange(20, device="cuda"), cet.rotary_frequencies(16)[0]
    x, wg, wu, b = r(30, 16), r(24, 16), r(24, 16), r(24)
    ops = torch.ops.cet
    leaves = [t.clone().requires_grad_() for t in (q, k, v, s0)]
    d = r(2, 20, 3, 24), r(2, 3, 16, 24)
    one = cet.linear_attention(*leaves[:3], dec, 0.3, leaves[3], lengths)
    two = ops.linear_attention(*leaves[:3], dec, 0.3, leaves[3], lengths)[:2]
    assert all(torch.equal(a, c) for a, c in zip(one, two))
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(one, leaves, d), torch.autograd.grad(two, leaves, d)))
    one, two = cet.rotary(leaves[0], leaves[1], pos, f), ops.rotary(leaves[0], leaves[1], pos, f, False, 1.0, False)
    assert all(torch.equal(a, c) for a, c in zip(one, two))
    dd = r(2, 20, 3, 16), r(2, 20, 3, 16)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(one, leaves[:2], dd), torch.autograd.grad(two, leaves[:2], dd)))
    gl = [t.clone().requires_grad_() for t in (x, wg, wu, b, b)]
    one, two = cet.gated_linear(*gl, "gelu"), ops.gated_linear(*gl, "gelu")
    dy = r(30, 24)
    assert torch.equal(one, two)
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(one, gl, dy), torch.autograd.grad(two, gl, dy)))
    sa, sb = s0.clone(), s0.clone()
    assert torch.equal(cet.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], dec, sa, 0.3, inplace=True)[0],
                       ops.linear_attention_step_(q[:, 0], k[:, 0], v[:, 0], dec, sb, 0.3, None)) and torch.equal(sa, sb)
    checks = ("test_schema", "test_faketensor", "test_autograd_registration")
    for op, args in ((ops.linear_attention, (*leaves[:3], dec, 0.3, leaves[3], lengths)), (ops.rotary, (leaves[0], leaves[1], pos, f, True, 1.5, False)),
                     (ops.gated_linear, (*gl, "silu")), (ops.linear_attention_step, (q[:, 0], k[:, 0], v[:, 0], dec, s0, 0.3)),
                     (ops.linear_attention_step_, (q[:, 0], k[:, 0], v[:, 0], dec, s0.clone(), 0.3, None)),
                     (ops.linear_attention_backward, (q, k, v, dec, 0.3, s0, lengths, None, d[0], d[1], True)),
                     (ops.gated_linear_backward, (x, wg, wu, b, None, "relu", dy, True, False, True))):
        torch.library.opcheck(op, args, test_utils=checks)


def test_a_state_written_in_place_is_noticed():
    """A state that a gradient still needs cannot be overwritten unnoticed, nor a gradient be taken twice."""
    g = torch.Generator().manual_seed(4)
    q = torch.randn(2, 5, 3, 8, generator=g).cuda().requires_grad_()
    s0, dec = torch.randn(2, 3, 8, 8, generator=g).cuda(), ref.geometric(3).cuda()
    o, _ = cet.linear_attention(q, q.detach(), q.detach(), dec, initial_state=s0)
    with torch.no_grad():
        cet.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], dec, s0, inplace=True)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        o.sum().backward()
    o, _ = cet.linear_attention(q, q.detach(), q.detach(), dec)
    dq, = torch.autograd.grad(o.square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError):
        dq.sum().backward()


def test_refusals_on_the_gpu():
    z = lambda *s, **kw: torch.zeros(*s, device="cuda", **kw)  # noqa: E731
    q, g = z(2, 4, 2, 8), z(2)
    f = cet.rotary_frequencies(8)[0]
    bad = [
        lambda: cet.linear_attention(q, q[:, :3], q, g), lambda: cet.linear_attention(q, q, q.bfloat16(), g), lambda: cet.linear_attention(q.double(), q.double(), q.double(), g),
        lambda: cet.linear_attention(q, q, q, z(3)), lambda: cet.linear_attention(q, q, q, g.double()), lambda: cet.linear_attention(q, q, q, g, initial_state=z(2, 2, 8, 7)),
        lambda: cet.linear_attention(q, q, q, g, lengths=z(3, dtype=torch.int64)), lambda: cet.linear_attention(q, q, q, g, lengths=z(2)),
        lambda: cet.linear_attention(z(1, 1, 1, 257), z(1, 1, 1, 257), z(1, 1, 1, 8), z(1)), lambda: cet.linear_attention(q, q, q, g, scale=float("inf")),
        lambda: cet.linear_attention(q[0], q[0], q[0], g), lambda: cet.linear_attention(q, q, q, g.cpu()),
        lambda: cet.linear_attention_step(q, q, q, g, z(2, 2, 8, 8)), lambda: cet.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g, z(3, 2, 8, 8)),
        lambda: cet.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g, z(2, 2, 8, 8).transpose(0, 1), inplace=True),
        lambda: cet.linear_attention_step(q[:, 0], q[:, 0], q[:, 0], g, z(2, 2, 8, 8), slots=z(3, dtype=torch.int32)),
        lambda: cet.rotary(q, q, torch.arange(3, device="cuda"), f), lambda: cet.rotary(q, q, torch.arange(4, device="cuda").float(), f),
        lambda: cet.rotary(q, q, torch.arange(4, device="cuda"), f.float()), lambda: cet.rotary(q, q, torch.arange(4, device="cuda"), cet.rotary_frequencies(16)[0]),
        lambda: cet.rotary(q, z(2, 4, 2, 16), torch.arange(4, device="cuda"), f), lambda: cet.rotary(q, q, torch.arange(4), f),
        lambda: cet.gated_linear(z(4, 8), z(6, 8), z(5, 8)), lambda: cet.gated_linear(z(4, 8), z(6, 7), z(6, 7)), lambda: cet.gated_linear(z(4, 8), z(6, 8), z(6, 8), z(5)),
        lambda: cet.gated_linear(z(4, 8), z(6, 8), z(6, 8), activation="tanh"), lambda: cet.gated_linear(z(4, 8), z(6, 8).half(), z(6, 8)),
        lambda: cet.gated_linear(z(4, 8).double(), z(6, 8).double(), z(6, 8).double()), lambda: cet.gated_linear(z(4, 0), z(6, 0), z(6, 0))]
    for n, call in enumerate(bad):
        try:
            call()
        except RuntimeError:
            continue
        pytest.fail(f"call {n} was not refused")


def test_function_transforms_are_refused():
    """Not silently without gradients."""
    q, dec = torch.randn(2, 5, 3, 8).cuda(), ref.geometric(3).cuda()
    for call in (lambda t: cet.linear_attention(t, q, q, dec)[0].sum(), lambda t: cet.gated_linear(t[0, 0], q[0, 1], q[0, 2]).sum(),
                 lambda t: cet.rotary(t, None, torch.arange(5, device="cuda"), cet.rotary_frequencies(8)[0])[0].sum()):
        with pytest.raises(RuntimeError):
            torch.func.grad(call)(q)


def test_forward_mode_differentiation_is_refused():
    """Not silently without tangents."""
    q, dec = torch.randn(2, 5, 3, 8).cuda(), ref.geometric(3).cuda()
    with torch.autograd.forward_ad.dual_level():
        t = torch.autograd.forward_ad.make_dual(q, torch.ones_like(q))
        for call in (lambda: cet.linear_attention(t, q, q, dec), lambda: cet.gated_linear(t[0, 0], q[0, 1], q[0, 2]),
                     lambda: cet.rotary(t, None, torch.arange(5, device="cuda"), cet.rotary_frequencies(8)[0])):
            with pytest.raises((RuntimeError, NotImplementedError)):
                call()
