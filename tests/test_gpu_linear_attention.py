"""Linear attention with a decay per head against the recurrence in float64.

Bound of an output element: one rounding to the tensors' type, for bfloat16 one more of each score and of
the state in the products (they enter the matrix instructions as bfloat16), and (K + T + 64) fp32
roundings of sums, products and powers, each relative to the sum of the absolute values of the terms:
the same recurrence on absolute values ("mass"). The state is only subject to the fp32 part. 1 % on top for
products of errors. The gradients are the same recurrence with other operands."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


def make(B, T, H, K, V, dtype, seed=0, state=True, ragged=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    x = {"q": r(B, T, H, K), "k": r(B, T, H, K), "v": r(B, T, H, V), "d_o": r(B, T, H, V)}
    x = {n: t.to(dtype).double() for n, t in x.items()}  # what the GPU gets, exactly
    x["s0"] = r(B, H, K, V).double() if state else None
    x["d_state"] = r(B, H, K, V).double()
    x["lengths"] = torch.randint(0, T + 1, (B,), generator=g) if ragged else None
    x["g"] = ref.geometric(H)
    return x


def bounds(x, scale, dtype, T, K):
    a = {n: t.abs() if torch.is_tensor(t) and n not in ("lengths", "g") else t for n, t in x.items()}
    o, S, grads = ref.linear_attention_with_gradients(x["q"], x["k"], x["v"], x["g"], scale, x["s0"], x["lengths"], x["d_o"], x["d_state"])
    mo, mS, mg = ref.linear_attention_with_gradients(a["q"], a["k"], a["v"], a["g"], abs(scale), a["s0"], a["lengths"], a["d_o"], a["d_state"])
    c = (K + T + 64) * 2.0 ** -24
    inner = ref.half_step(torch.bfloat16) if dtype == torch.bfloat16 else 0.0
    lim = lambda want, mass, typed: 1.01 * ((ref.half_step(dtype) if typed else 0.0) * want.abs() + ((inner if typed else 0.0) + c) * mass) + 1e-30 + (1e-7 if typed and dtype == torch.float16 else 0)  # noqa: E731,E501
    typed = [True] * 3 + [False]
    return (o, S, grads), (lim(o, mo, True), lim(S, mS, False), [lim(g, m, t) for g, m, t in zip(grads, mg, typed)])


def gpu(x, dtype):
    out = {n: x[n].to(dtype).cuda() for n in ("q", "k", "v", "d_o")}
    out["s0"] = x["s0"].float().cuda() if x["s0"] is not None else None
    out["d_state"] = x["d_state"].float().cuda()
    out["lengths"] = x["lengths"].cuda() if x["lengths"] is not None else None
    out["g"] = x["g"].cuda()
    return out


def within(got, want, lim, what):
    bad = ((got.double().cpu() - want).abs() > lim) | ~torch.isfinite(got.cpu())
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got.double().cpu() - want).abs() / lim).nan_to_num(9e9).max()):.3g} of the bound, first {bad.nonzero()[0].tolist()}"


def check(x, dtype, scale=None, y=None):
    T, K = x["q"].shape[1], x["q"].shape[3]
    s = ref.sqrt_scale(K) if scale is None else scale
    (o, S, grads), (lo, lS, lg) = bounds(x, s, dtype, T, K)
    y = y or gpu(x, dtype)
    leaves = [y[n].detach().requires_grad_() for n in ("q", "k", "v")] + ([y["s0"].detach().requires_grad_()] if y["s0"] is not None else [])
    got_o, got_S = cet.linear_attention(leaves[0], leaves[1], leaves[2], y["g"], scale=scale,
                                        initial_state=leaves[3] if len(leaves) > 3 else None, lengths=y["lengths"])
    assert got_o.dtype == dtype and got_S.dtype == torch.float32
    within(got_o, o, lo, "o")
    within(got_S, S, lS, "state")
    got = torch.autograd.grad((got_o, got_S), leaves, (y["d_o"], y["d_state"]))
    for n, a, b, c in zip(("dq", "dk", "dv", "d_initial"), got, grads, lg):
        within(a, b, c, n)
    return got_o, got_S, got


SHAPES = [  # B, T, H, K, V
    (2, 1, 2, 8, 8), (1, 2, 1, 1, 1), (3, 15, 2, 16, 16), (2, 16, 1, 32, 32), (2, 17, 3, 20, 24), (1, 31, 2, 8, 100), (2, 32, 2, 64, 64),
    (2, 33, 1, 40, 72), (1, 63, 2, 128, 128), (1, 64, 1, 128, 64), (2, 65, 1, 100, 33), (1, 80, 2, 256, 256),
    (1, 129, 1, 256, 8), (1, 97, 1, 8, 256), (1, 200, 1, 192, 130), (1, 70, 1, 3, 5),
    (9, 25, 3, 8, 8), (70, 32, 5, 16, 7), (5, 11, 2, 5, 16), (3, 33, 2, 16, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, dtype):
    check(make(*shape, dtype, seed=sum(shape)), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("V", [12, 50, 130])
@pytest.mark.parametrize("K", [10, 24, 40, 56, 72, 100, 160, 200])
def test_every_number_of_blocks(K, V, dtype):
    """Each number of blocks of K that a kernel is built for with each width of its slices, in segments, to ragged
    lengths; the gradients are the same with K and V exchanged."""
    check(make(2, 270, 1, K, V, dtype, seed=K + V, ragged=True), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("K, V", [(100, 128), (40, 33), (256, 200), (130, 70)])
def test_gradients_that_share_a_launch(K, V, dtype):
    """Heads whose K and V differ but are served by one kernel, and some where only two of the gradients are."""
    check(make(2, 150, 2, K, V, dtype, seed=K, ragged=True), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(2, 700, 1, 32, 16), (1, 1500, 2, 64, 64), (1, 1031, 1, 128, 128), (1, 900, 1, 16, 16)])
def test_time_axis_in_segments(shape, dtype):
    """Few sequences and heads: the time axis is cut and the pieces' states are joined."""
    check(make(*shape, dtype, seed=3), dtype)
    check(make(*shape, dtype, seed=4, state=False), dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [1, 40, 700])
@pytest.mark.parametrize("K, V", [(24, 40), (8, 12)])
def test_ragged_lengths_and_what_lies_behind_them(dtype, T, K, V):
    """Lengths of zero, one, T and beyond both ends; NaN and infinity behind the last slot are not read."""
    x = make(6, T, 2, K, V, dtype, seed=T, ragged=True)
    x["lengths"][:4] = torch.tensor([0, 1, T, min(T, 33)])
    y = gpu(x, dtype)
    for n in ("q", "k", "v", "d_o"):
        y[n] = torch.where((torch.arange(T)[None] < x["lengths"][:, None])[:, :, None, None].cuda(), y[n],
                           torch.tensor(float("nan") if n != "k" else float("inf"), dtype=dtype, device="cuda"))
    y["lengths"][0], y["lengths"][2] = -5, T + 1000  # taken as the nearer end
    o, _, (dq, dk, dv, _) = check(x, dtype, y=y)
    for b in range(6):
        for t in (o, dq, dk, dv):
            assert (t[b, int(x["lengths"][b]):] == 0).all()
    y["lengths"] = y["lengths"].int()
    check(x, dtype, y=y)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("T", [45, 29])
def test_strides_and_alignment(dtype, T):
    """Slices of one packed projection, heads before slots, and rows that start off 16 bytes."""
    B, H, K = 2, 3, 16
    x = make(B, T, H, K, K, dtype, seed=5)
    want = check(x, dtype)
    y = gpu(x, dtype)
    packed = torch.cat([y["q"], y["k"], y["v"]], -1)
    heads_first = {n: y[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v")}
    room = {n: torch.full((B, T, H, K + 3), float("nan"), dtype=dtype, device="cuda") for n in ("q", "k", "v")}
    for n in room:
        room[n][..., 1:K + 1] = y[n]
    for variant in (dict(zip(("q", "k", "v"), packed.split(K, -1))), heads_first, {n: room[n][..., 1:K + 1] for n in room}):
        got = check(x, dtype, y={**y, **variant})
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert all(torch.equal(a, b) for a, b in zip(got[2], want[2]))
    # a gradient that is one value spread over all of o
    leaves = [y[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o, _ = cet.linear_attention(*leaves, y["g"])
    spread = torch.autograd.grad(o.float().sum(), leaves)
    o, _ = cet.linear_attention(*leaves, y["g"])
    full = torch.autograd.grad(o, leaves, torch.ones_like(o))
    assert all(torch.equal(a, b) for a, b in zip(spread, full))


@pytest.mark.parametrize("dtype", TYPES)
def test_decays_at_their_ends(dtype):
    """No memory at all, none lost, and one that fades inside a block."""
    x = make(2, 70, 4, 16, 16, dtype, seed=6)
    x["g"] = torch.tensor([float("-inf"), 0.0, -20.0, -0.5])
    check(x, dtype)
    check(x, dtype, scale=-0.3)
    check(x, dtype, scale=0.0)


def test_many_small_heads_over_many_slots():
    """A lane per column also for long histories where there are heads enough for it; the far weights hold."""
    B, T, H, K = 4200, 130, 4, 8
    g = torch.Generator(device="cuda").manual_seed(16)
    q, k, v = (torch.randn(B, T, H, K, generator=g, device="cuda") for _ in range(3))
    dec = torch.log1p(-torch.exp2(-torch.tensor([5.0, 8.0, 11.0, 14.0], device="cuda")))
    o, s = cet.linear_attention(q, k, v, dec, scale=0.3)
    pick = [0, 1, 2099, 4198, 4199]
    x = [t[pick].double().cpu() for t in (q, k, v)]
    want, S = ref.linear_attention(*x, dec.cpu(), 0.3)
    mass, mS = ref.linear_attention(*(t.abs() for t in x), dec.cpu(), 0.3)
    c = 1.01 * (K + T + 64) * 2.0 ** -24
    within(o[pick], want, c * mass, "o")
    within(s[pick], S, c * mS, "state")


def test_a_thousand_single_slots_keep_far_weights():
    """The state after many steps against the recurrence: (steps + 64) fp32 roundings, none of them the decay's own
    raised to the number of steps."""
    H, K, n = 2, 4, 3000
    dec = torch.log1p(-torch.exp2(-torch.tensor([12.0, 16.0], device="cuda")))
    s = torch.ones(1, H, K, K, device="cuda")
    z = torch.zeros(1, H, K, device="cuda")
    for _ in range(n):
        cet.linear_attention_step(z, z, z, dec, s, inplace=True)
    want = (n * dec.double()).exp().cpu().view(1, H, 1, 1).expand(1, H, K, K)
    # each step rounds twice: 2 n / 2 units of 2^-24 at the worst
    within(s, want, n * 2.0 ** -24 * want, "state")


def test_histories_without_slots():
    q = torch.zeros(2, 0, 3, 8, device="cuda")
    s0 = torch.randn(2, 3, 8, 8, device="cuda")
    g = ref.geometric(3).cuda()
    o, s = cet.linear_attention(q, q, q, g, initial_state=s0)
    assert o.shape == (2, 0, 3, 8) and torch.equal(s, s0)
    o, s = cet.linear_attention(q, q, q, g)
    assert (s == 0).all()
    o, s = cet.linear_attention(q[:0], q[:0], q[:0], g)
    assert s.shape == (0, 3, 8, 8)


def test_gradients_against_differences():
    """o and the state are linear in each operand, so a central difference along any direction is the
    derivative up to fp32 rounding of the two sums (2^-24 of the terms' absolute sum each, times their
    number, here bounded through the float64 oracle's mass)."""
    x = make(2, 50, 2, 16, 24, torch.float32, seed=7)
    y = gpu(x, torch.float32)
    leaves = [y[n].detach().requires_grad_() for n in ("q", "k", "v", "s0")]

    def loss(a):
        o, s = cet.linear_attention(a[0], a[1], a[2], y["g"], initial_state=a[3])
        return (o.double() * y["d_o"].double()).sum() + (s.double() * y["d_state"].double()).sum()

    grads = torch.autograd.grad(loss(leaves), leaves)
    _, (lo, lS, _) = bounds(x, 0.25, torch.float32, 50, 16)
    slack = float((lo * x["d_o"].abs()).sum() + (lS * x["d_state"].abs()).sum())
    gen = torch.Generator(device="cuda").manual_seed(1)
    with torch.no_grad():
        for j in range(4):
            # a direction of at most the operand's own size: the difference's terms stay within twice the mass
            step = y[("q", "k", "v", "s0")[j]].abs() * (torch.randint(0, 2, leaves[j].shape, generator=gen, device="cuda") * 2 - 1)
            up, down = ([t + (s * step if i == j else 0) for i, t in enumerate(leaves)] for s in (1.0, -1.0))
            want = float((loss(up) - loss(down)) / 2)
            got = float((grads[j].double() * step.double()).sum())
            assert abs(got - want) <= 4 * slack, (j, got, want, slack)


def test_history_then_single_slots():
    """A history in one call, or in two that hand the state over, or slot by slot."""
    B, T, H, K, V = 3, 90, 2, 32, 48
    x = make(B, T, H, K, V, torch.float32, seed=8)
    y = gpu(x, torch.float32)
    whole, last = cet.linear_attention(y["q"], y["k"], y["v"], y["g"], initial_state=y["s0"])
    (o, S, _), (lo, lS, _) = bounds(x, ref.sqrt_scale(K), torch.float32, T, K)
    a, s = cet.linear_attention(y["q"][:, :57], y["k"][:, :57], y["v"][:, :57], y["g"], initial_state=y["s0"])
    outs = [a]
    for t in range(57, T):
        step, s = cet.linear_attention_step(y["q"][:, t], y["k"][:, t], y["v"][:, t], y["g"], s)
        outs.append(step[:, None])
    within(whole, o, lo, "whole")
    within(torch.cat(outs, 1), o, lo, "in pieces")
    within(last, S, lS, "state")
    within(s, S, lS, "state in pieces")


STEP_SHAPES = [(1, 1, 1, 1), (3, 2, 8, 8), (2, 3, 20, 24), (5, 2, 64, 64), (2, 1, 100, 33), (4, 2, 128, 128), (1, 2, 256, 256), (700, 2, 16, 40), (600, 4, 8, 7)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", STEP_SHAPES)
def test_single_slots(shape, dtype):
    B, H, K, V = shape
    x = make(B, 1, H, K, V, dtype, seed=9)
    y = gpu(x, dtype)
    (o, S, _), (lo, lS, _) = bounds({**x}, ref.sqrt_scale(K), torch.float32 if dtype == torch.bfloat16 else dtype, 1, K)
    lo = lo + 1.01 * ref.half_step(dtype) * o.abs()  # scores and state stay in fp32: one rounding to the type
    args = [y[n][:, 0] for n in ("q", "k", "v")]
    before = y["s0"].clone()
    got, s = cet.linear_attention_step(*args, y["g"], y["s0"])
    assert torch.equal(y["s0"], before)
    within(got[:, None], o, lo, "o")
    within(s, S, lS, "state")
    got2, same = cet.linear_attention_step(*args, y["g"], y["s0"], inplace=True)
    assert same is y["s0"] and torch.equal(got, got2) and torch.equal(s, same)
    # a pool with the streams in other places, one of them idle, one beyond it, one twice
    pool = torch.randn(B + 3, H, K, V, device="cuda")
    place = torch.randperm(B + 3)[:B].cuda()
    pool[place] = before
    kept = pool.clone()
    got3, _ = cet.linear_attention_step(*args, y["g"], pool, slots=place)
    assert torch.equal(got3, got) and torch.equal(pool[place], s)
    rest = torch.ones(B + 3, dtype=torch.bool, device="cuda")
    rest[place] = False
    assert torch.equal(pool[rest], kept[rest])


def test_slots_that_cannot_be_served():
    B, H, K, V = 6, 2, 16, 16
    y = gpu(make(B, 1, H, K, V, torch.float32, seed=10), torch.float32)
    args = [y[n][:, 0] for n in ("q", "k", "v")]
    pool = torch.randn(8, H, K, V, device="cuda")
    for kind in (torch.int32, torch.int64):
        p = pool.clone()
        slots = torch.tensor([3, -1, 8, 3, 0, 1 << 30], dtype=kind, device="cuda")
        o, _ = cet.linear_attention_step(*args, y["g"], p, slots=slots)
        want, s = cet.linear_attention_step(*args, y["g"], pool[[3, 0, 0, 0, 0, 0]])
        assert torch.equal(o[0], want[0]) and torch.equal(o[4], want[4]) and (o[1] == 0).all()
        assert torch.isnan(o[[2, 3, 5]]).all()
        assert torch.equal(p[3], s[0]) and torch.equal(p[0], s[4])
        assert torch.equal(p[[1, 2, 4, 5, 6, 7]], pool[[1, 2, 4, 5, 6, 7]])


def test_graphs_and_streams():
    """Captured forward, gradients and steps, replayed with other inputs between eager calls; two graphs
    share nothing; calls on a side stream."""
    xs = [make(2, 300, 2, 32, 32, torch.bfloat16, seed=s) for s in (11, 12)]
    ys = [gpu(x, torch.bfloat16) for x in xs]

    def forward_backward(y):
        leaves = [y[n].detach().requires_grad_() for n in ("q", "k", "v", "s0")]
        o, s = cet.linear_attention(*leaves[:3], y["g"], initial_state=leaves[3])
        return (o.detach(), s.detach(), *torch.autograd.grad((o, s), leaves, (y["d_o"], y["d_state"])))

    def steps(y):
        s = y["s0"].clone()
        outs = [cet.linear_attention_step(y["q"][:, t], y["k"][:, t], y["v"][:, t], y["g"], s, inplace=True)[0] for t in range(4)]
        return (*outs, s)

    for fn in (forward_backward, steps):
        want = [fn(y) for y in ys]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            on_side = fn(ys[0])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(on_side, want[0]))
        static = [{n: t.clone() if torch.is_tensor(t) else t for n, t in ys[0].items()} for _ in range(2)]
        graphs, outs = [], []
        for st in static:
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                outs.append(fn(st))
            graphs.append(g)
        for turn in range(4):
            for j, (g, st) in enumerate(zip(graphs, static)):
                y = ys[(turn + j) % 2]
                for n, t in st.items():
                    if torch.is_tensor(t):
                        t.copy_(y[n])
            for g in graphs:
                g.replay()
            fn(ys[turn % 2])
            torch.cuda.synchronize()
            for j, out in enumerate(outs):
                assert all(torch.equal(a, b) for a, b in zip(out, want[(turn + j) % 2]))


def test_states_of_segments_kept_or_formed_again():
    """The gradient from the states that the forward call kept and from formed ones: the same bits."""
    y = gpu(make(1, 1200, 2, 48, 32, torch.bfloat16, seed=15), torch.bfloat16)
    args = y["q"], y["k"], y["v"], y["g"], 0.2, y["s0"], None
    kept = torch.ops.cet.linear_attention(*args, True)[2]
    assert kept.numel() >= 2 * 48 * 32
    one = torch.ops.cet.linear_attention_backward(*args, kept, y["d_o"], y["d_state"], True)
    two = torch.ops.cet.linear_attention_backward(*args, None, y["d_o"], y["d_state"], True)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    with pytest.raises(RuntimeError, match="segments"):
        torch.ops.cet.linear_attention_backward(*args, kept[:-4], y["d_o"], y["d_state"], True)


def test_same_bits_every_time():
    y = gpu(make(1, 2000, 2, 64, 64, torch.bfloat16, seed=13), torch.bfloat16)
    first = cet.linear_attention(y["q"], y["k"], y["v"], y["g"])
    for _ in range(3):
        again = cet.linear_attention(y["q"], y["k"], y["v"], y["g"])
        assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])


def test_only_the_state_or_only_the_outputs_are_used():
    x = make(2, 40, 2, 16, 16, torch.float32, seed=14)
    y = gpu(x, torch.float32)
    for keep in (0, 1):
        z = dict(x)
        z["d_o"], z["d_state"] = (x["d_o"], torch.zeros_like(x["d_state"])) if keep == 0 else (torch.zeros_like(x["d_o"]), x["d_state"])
        _, (_, _, lg) = bounds(z, 0.25, torch.float32, 40, 16)
        _, _, want = ref.linear_attention_with_gradients(z["q"], z["k"], z["v"], z["g"], 0.25, z["s0"], None, z["d_o"], z["d_state"])
        leaves = [y[n].detach().requires_grad_() for n in ("q", "k", "v", "s0")]
        out = cet.linear_attention(*leaves[:3], y["g"], initial_state=leaves[3])[keep]
        got = torch.autograd.grad(out, leaves, y["d_o"] if keep == 0 else y["d_state"])
        for a, b, c in zip(got, want, lg):
            within(a, b, c, "gradient")
