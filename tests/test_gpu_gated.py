"""The gated projection and its gradients against float64.

With c = (D + 32) 2^-24 a projection is off by c M, M = sum |x||w| + |b| (products and sums in fp32); the
activations' slopes stay below 1.2 and their curvatures below 1, their functions within c |g|. So the result is off by
c (1.2 Mg |u| + |act| Mu + |g u|) and one rounding; the projections' gradients dg, du by dy times
c (1.2 Mu + |u| Mg + |u|) and c (1.2 Mg + |g|), and one rounding to the tensors' type (they enter the last
products in it); relu's slope is free where |g| <= c Mg. These errors go through the last products with
the absolute values of the other operand, whose own fp32 sums add (terms + 32) 2^-24 of the absolute sum.
1 % on top for products of errors."""
import pytest
import torch

import channelestimationtransformer_amd as cet
import seq_ref as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
E = 2.0 ** -24


def make(N, D, F, dtype, bias, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, by=1.0: (torch.randn(*s, generator=g, device="cuda") * by).to(dtype)  # noqa: E731
    w = [r(F, D, by=D ** -0.5) for _ in range(2)]
    b = [r(F, by=0.3) if bias else None for _ in range(2)]
    return r(N, D), w[0], w[1], b[0], b[1], r(N, F)


def expected(x, wg, wu, bg, bu, dy, kind, dtype):
    """(values, bounds) of out, dx, dwg, dwu, dbg, dbu."""
    h, c = ref.half_step(dtype), (x.shape[1] + 32) * E
    x, wg, wu, dy = (t.double() for t in (x, wg, wu, dy))
    zero = torch.zeros(wg.shape[0], dtype=torch.float64, device="cuda")
    bg, bu = (zero if b is None else b.double() for b in (bg, bu))
    g, u = x @ wg.t() + bg, x @ wu.t() + bu
    Mg, Mu = x.abs() @ wg.abs().t() + bg.abs(), x.abs() @ wu.abs().t() + bu.abs()
    if kind == "silu":
        s = torch.sigmoid(g)
        a, slope = g * s, s * (1 + g * (1 - s))
    elif kind == "gelu":
        p = torch.special.ndtr(g)
        a, slope = g * p, p + g * torch.exp(-g * g / 2) * 0.3989422804014327
    else:
        a, slope = g.clamp(min=0), (g > 0).double()
    out = a * u
    e_out = h * out.abs() + c * (1.2 * Mg * u.abs() + a.abs() * Mu + (g * u).abs())
    dg, du = dy * u * slope, dy * a
    e_g = dy.abs() * c * (1.2 * Mu + u.abs() * Mg + u.abs())
    if kind == "relu":
        e_g = e_g + (g.abs() <= c * Mg) * (dy * u).abs()
    e_u = dy.abs() * c * (1.2 * Mg + g.abs())
    r_g, r_u = e_g + h * dg.abs(), e_u + h * du.abs()
    dx, dwg, dwu = dg @ wg + du @ wu, dg.t() @ x, du.t() @ x
    n, f = (x.shape[0] + 32) * E, (2 * wg.shape[0] + 32) * E
    e_dx = h * dx.abs() + r_g @ wg.abs() + r_u @ wu.abs() + f * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    e_dw = [h * t.abs() + r.t() @ x.abs() + n * (d.abs().t() @ x.abs()) for t, r, d in ((dwg, r_g, dg), (dwu, r_u, du))]
    e_db = [h * d.sum(0).abs() + e.sum(0) + n * d.abs().sum(0) for d, e in ((dg, e_g), (du, e_u))]
    tiny = 6e-8 if dtype == torch.float16 else 1e-30
    # float16: dg and du below its smallest normal number are rounded in steps of 6e-8
    few = tiny * (1 + torch.stack([x.abs().sum(0).max(), wg.abs().sum(0).max(), wu.abs().sum(0).max()]).max())
    return (out, dx, dwg, dwu, dg.sum(0), du.sum(0)), [1.01 * e + few for e in (e_out, e_dx, *e_dw, *e_db)]


def check(args, kind, dtype, scale_ok=True):
    x, wg, wu, bg, bu, dy = args
    want, lim = expected(*args, kind, dtype)
    leaves = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu) if t is not None]
    it = iter(leaves)
    a = [next(it) if t is not None else None for t in (x, wg, wu, bg, bu)]
    out = cet.gated_linear(*a, activation=kind)
    grads = torch.autograd.grad(out, leaves, dy)
    assert out.dtype == dtype and all(g.shape == t.shape and g.dtype == dtype for g, t in zip(grads, leaves))
    for n, got, w, e in zip(("out", "dx", "dw_gate", "dw_up", "db_gate", "db_up"), (out.detach(), *grads), want, lim):
        err = (got.double() - w).abs()
        assert torch.isfinite(got).all() and (err <= e).all(), (n, float((err / e).nan_to_num(9e9).max()))
    return out, grads


SHAPES = [(1, 1, 1), (1, 64, 64), (5, 33, 17), (16, 128, 48), (40, 100, 130), (64, 256, 64), (65, 64, 64), (100, 16, 500), (129, 136, 128),
          (300, 72, 200), (70, 32, 32), (333, 20, 60), (90, 64, 7), (1000, 33, 64), (9000, 64, 64), (700, 256, 520), (17, 2050, 31), (2000, 64, 64), (257, 513, 9), (5000, 40, 24)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind, bias", [("silu", False), ("gelu", True), ("relu", True)])
@pytest.mark.parametrize("shape", SHAPES)
def test_forward_and_gradients(shape, kind, bias, dtype):
    check(make(*shape, dtype, bias, seed=sum(shape)), kind, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_large_tiles_and_split_sums(dtype):
    check(make(4100, 520, 4104, dtype, True, seed=1), "silu", dtype)  # tiles of 256
    check(make(4100, 512, 1030, dtype, False, seed=2), "gelu", dtype)
    check(make(20000, 64, 72, dtype, True, seed=3), "gelu", dtype)  # few tiles, long sums


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_alignment_and_leading_axes(dtype):
    args = make(70, 64, 96, dtype, True, seed=4)
    want = check(args, "silu", dtype)
    x, wg, wu, bg, bu, dy = args
    both = torch.cat([wg, wu])  # two halves of one projection
    wide = torch.full((70, 64 + 24), float("nan"), dtype=dtype, device="cuda")
    wide[:, 8:72] = x
    odd = torch.full((70, 67), float("nan"), dtype=dtype, device="cuda")
    odd[:, 1:65] = x
    dwide = torch.full((70, 99), float("nan"), dtype=dtype, device="cuda")
    dwide[:, 2:98] = dy
    for variant in ((x, both[:96], both[96:], bg, bu, dy), (wide[:, 8:72], wg, wu, bg, bu, dwide[:, 2:98]), (odd[:, 1:65], wg, wu, bg, bu, dy),
                    (x.t().contiguous().t(), wg.t().contiguous().t(), wu, bg, bu, dy.t().contiguous().t())):
        got = check(variant, "silu", dtype)
        assert torch.equal(got[0], want[0]) and all(torch.equal(a, b) for a, b in zip(got[1], want[1]))
    cube = cet.gated_linear(x.reshape(7, 10, 64), wg, wu, bg, bu)
    assert cube.shape == (7, 10, 96) and torch.equal(cube.reshape(70, 96), want[0])
    one = cet.gated_linear(x[3], wg, wu, bg, bu)  # a single row takes the kernel for few rows
    assert one.shape == (96,)
    lim = expected(*args, "silu", dtype)[1][0][3]
    assert ((one.double() - expected(*args, "silu", dtype)[0][0][3]).abs() <= lim).all()


def test_one_bias_no_rows_and_gradients_of_some():
    x, wg, wu, bg, bu, dy = make(90, 32, 40, torch.float32, True, seed=5)
    zero = torch.zeros_like(bg)
    assert torch.equal(cet.gated_linear(x, wg, wu, bg), cet.gated_linear(x, wg, wu, bg, zero))
    assert torch.equal(cet.gated_linear(x, wg, wu, None, bu), cet.gated_linear(x, wg, wu, zero, bu))
    leaves = [t.clone().requires_grad_() for t in (x[:0], wg, wu, bg, bu)]
    out = cet.gated_linear(*leaves)
    assert out.shape == (0, 40)
    assert all((g == 0).all() for g in torch.autograd.grad(out, leaves, dy[:0]))
    full = check((x, wg, wu, bg, bu, dy), "silu", torch.float32)[1]
    for keep in range(5):
        a = [t.clone() for t in (x, wg, wu, bg, bu)]
        a[keep].requires_grad_()
        got, = torch.autograd.grad(cet.gated_linear(*a), a[keep], dy)
        assert torch.equal(got, full[keep])


def test_gradient_against_differences():
    """The projections are linear in x and both weights and the loss is smooth (silu): a central difference
    with step t along a direction is off by t^2 / 6 of the third derivative, held here below one part in
    10^3 of the sum of the absolute terms by t = 1/64, and the fp32 bounds of both losses over 2 t."""
    args = make(66, 32, 48, torch.float32, True, seed=6)
    _, lim = expected(*args, "silu", torch.float32)
    x, wg, wu, bg, bu, dy = args
    leaves = [t.clone().requires_grad_() for t in (x, wg, wu, bg, bu)]
    grads = torch.autograd.grad(cet.gated_linear(*leaves), leaves, dy)
    t = 1.0 / 64
    g = torch.Generator(device="cuda").manual_seed(7)
    for j, leaf in enumerate((x, wg, wu, bg, bu)):
        step = leaf.abs() * (torch.randint(0, 2, leaf.shape, generator=g, device="cuda") * 2 - 1)
        loss = []
        for s in (t, -t):
            a = [x, wg, wu, bg, bu]
            a[j] = leaf + s * step
            loss.append(float((cet.gated_linear(*a).double() * dy.double()).sum()))
        want, got = (loss[0] - loss[1]) / (2 * t), float((grads[j].double() * step.double()).sum())
        mass = float((grads[j].double() * step.double()).abs().sum())
        slack = 1e-3 * mass + float((lim[0] * dy.abs()).sum()) / t + float((lim[j + 1] * step.abs()).sum())
        assert abs(got - want) <= slack, (j, got, want, slack)


def test_graphs_and_streams():
    cases = [make(300, 128, 200, torch.bfloat16, True, seed=s) for s in (8, 9)]

    def both_ways(x, wg, wu, bg, bu, dy):
        leaves = [t.detach().requires_grad_() for t in (x, wg, wu, bg, bu)]
        out = cet.gated_linear(*leaves)
        return (out.detach(), *torch.autograd.grad(out, leaves, dy))

    def few(x, wg, wu, bg, bu, dy):
        return (cet.gated_linear(x[:20], wg, wu, bg, bu),)

    for fn in (both_ways, few):
        want = [fn(*c) for c in cases]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = fn(*cases[0])
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want[0]))
        static = [[t.clone() for t in cases[0]] for _ in range(2)]
        graphs, outs = [], []
        for st in static:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                outs.append(fn(*st))
            graphs.append(graph)
        for turn in range(4):
            for j, st in enumerate(static):
                for a, b in zip(st, cases[(turn + j) % 2]):
                    a.copy_(b)
            for graph in graphs:
                graph.replay()
            fn(*cases[0])
            torch.cuda.synchronize()
            for j, out in enumerate(outs):
                assert all(torch.equal(a, b) for a, b in zip(out, want[(turn + j) % 2]))


@pytest.mark.parametrize("kind", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("N, D, F", [(9, 40, 24), (40, 100, 130), (300, 136, 150)])
def test_nan_is_not_swallowed(N, D, F, kind):
    """A NaN in a weight of the gate reaches its column of the result, whatever the activation, and no other."""
    x, wg, wu, _, _, _ = make(N, D, F, torch.float32, False, seed=8)
    wg[3, 5] = float("nan")
    out = cet.gated_linear(x, wg, wu, activation=kind)
    assert torch.isnan(out[:, 3]).all()
    assert torch.isfinite(out[:, [c for c in range(F) if c != 3]]).all()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("F", [129, 255, 257, 263, 1299])
def test_rows_of_an_odd_number_of_features(F, dtype):
    """Rows that start between two words, over one tile and several, with whole and broken last pieces."""
    check(make(300, 72, F, dtype, True, seed=F), "silu", dtype)
    check(make(4100, 40, F, dtype, False, seed=F), "relu", dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("N, D, F", [(90, 130, 70), (1073, 264, 2177), (600, 2056, 300), (3000, 128, 66)])
def test_tiles_of_every_size(N, D, F, dtype):
    """Few tiles (the smallest), several rounds of them, long sums in pieces."""
    check(make(N, D, F, dtype, True, seed=N), "gelu", dtype)
