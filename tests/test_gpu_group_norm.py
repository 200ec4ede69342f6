"""Group norm with an activation per graph, against the formula in float64.

Bounds are derived from roundings of u = 2^-24 (half a step of fp32): the normalised value takes four of them and the affine
map one, the activation four; the sums are exact at this scale (fp64).  They are evaluated element by element below.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def act64(z, kind):
    if kind == "none":
        return z, torch.ones_like(z)
    if kind == "relu":
        return z.clamp(min=0), (z > 0).double()
    if kind == "silu":
        s = torch.sigmoid(z)
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
    return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)


def values8(x):
    """The 8-bit values of x (exact in any precision)."""
    out = []
    for cols in torch.split(x.double(), 32, dim=1):
        top = cols.abs().amax(1, keepdim=True)
        e = torch.floor(torch.log2(top.clamp(min=2.0 ** -200))) - 6
        e = torch.where(top >= 127.5 * torch.exp2(e), e + 1, e).clamp(min=-126, max=121)
        out.append(torch.round(cols * torch.exp2(-e)).clamp(-127, 127) * torch.exp2(e))
    return torch.cat(out, 1)


def reference(x, sizes, groups, w, b, kind, eps, g=None, keep8=False):
    """(out, its bound) or, with g, also (gx, gw, gb) and their bounds, all float64."""
    n, c = x.shape
    per = c // groups
    x64 = x.double()
    w64 = torch.ones(c, dtype=torch.float64, device=x.device) if w is None else w.double()
    b64 = torch.zeros(c, dtype=torch.float64, device=x.device) if b is None else b.double()
    kept = values8(x) if keep8 else x64
    out, out_b = torch.zeros_like(x64), torch.zeros_like(x64)
    gx, gx_b = torch.zeros_like(x64), torch.zeros_like(x64)
    gw, gb, gw_b, gb_b = (torch.zeros(c, dtype=torch.float64, device=x.device) for _ in range(4))
    at = 0
    for s in sizes:
        if s == 0:
            continue
        r = slice(at, at + s)
        at += s
        grp = x64[r].reshape(s, groups, per)
        mean = grp.mean((0, 2))
        rs = 1.0 / torch.sqrt(((grp - mean[None, :, None]) ** 2).mean((0, 2)) + eps)
        mean, rs = mean.repeat_interleave(per), rs.repeat_interleave(per)

        def at_values(v):
            xh = (v - mean) * rs
            z = xh * w64 + b64
            return xh, z, 4 * U * (xh * w64).abs() + U * z.abs()

        xh, z, dz_err = at_values(x64[r])
        out[r] = act64(z, kind)[0]
        out_b[r] = 1.13 * dz_err + 4 * U * z.abs() + 1e-37
        if g is None:
            continue
        xh, z, z_err = at_values(kept[r])
        da = act64(z, kind)[1]
        g64 = g[r].double()
        dz = g64 * da
        dz_err = g64.abs() * (z_err + 6 * U) + U * dz.abs()          # |act''| <= 1
        gw += (dz * xh).sum(0)
        gb += dz.sum(0)
        gw_b += (dz_err * xh.abs() + 4 * U * (dz * xh).abs()).sum(0)
        gb_b += dz_err.sum(0)
        a, a_err = dz * w64, dz_err * w64.abs()

        def mean_of(t):
            return t.reshape(s, groups, per).mean((0, 2)).repeat_interleave(per)

        m1, m2 = mean_of(a), mean_of(a * xh)
        m1_err = mean_of(a_err) + U * m1.abs()
        m2_err = mean_of(a_err * xh.abs() + 4 * U * (a * xh).abs()) + U * m2.abs()
        gx[r] = rs * (a - m1 - xh * m2)
        gx_b[r] = rs * (a_err + m1_err + xh.abs() * m2_err + 6 * U * (a.abs() + m1.abs() + (xh * m2).abs()))
    if g is None:
        return out, out_b
    return (out, gx, gw, gb), (out_b, gx_b, gw_b + U * gw.abs() + 1e-37, gb_b + U * gb.abs() + 1e-37)


def within(got, want, bound, what):
    err = (got.double() - want).abs()
    assert got.shape == want.shape, what
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound.clamp(min=1e-300))[bad].max()):.3g} bounds"


def make(sizes, c, seed, offset=True):
    gen = torch.Generator(device=dev()).manual_seed(seed)
    n = sum(sizes)
    x = torch.randn(n, c, generator=gen, device=dev())
    if offset:
        x = x * (torch.rand(c, generator=gen, device=dev()) + 0.5) + torch.randn(c, generator=gen, device=dev())
    w = torch.rand(c, generator=gen, device=dev()) + 0.5
    b = torch.randn(c, generator=gen, device=dev()) * 0.3
    g = torch.randn(n, c, generator=gen, device=dev())
    return x, w, b, g


SHAPES = [
    # sizes, columns, groups
    ([1], 1, 1), ([1, 1, 1], 4, 2), ([138] * 4, 138, 6), ([5, 0, 138, 2, 0, 454], 138, 23), ([3, 7], 30, 30),
    ([2627, 454, 1], 256, 32), ([1500], 138, 138), ([700, 705], 46, 2), ([40], 320, 1), ([300], 1100, 1), ([9, 2000], 1100, 1),
    ([64] * 70, 12, 3), ([5000, 1, 4999], 6, 1), ([33], 1028, 257),
]


@pytest.mark.parametrize("sizes,c,groups", SHAPES, ids=[f"{len(s)}x{max(s)}-{c}-{g}" for s, c, g in SHAPES])
@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("keep8", [False, True])
def test_group_norm_act_matches_float64(sizes, c, groups, act, keep8):
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    x, w, b, g = make(sizes, c, seed=c + groups)
    if act == "relu":                       # no gradient where the sign of z is a matter of rounding
        for kept in (False, keep8):
            xs = values8(x).float() if kept else x
            _, bound = reference(x, sizes, groups, w, b, "none", 1e-5)
            mean_out = reference(x, sizes, groups, w, b, "none", 1e-5)[0]
            g = torch.where(mean_out.abs() > 4 * bound, g, 0.0)
        if keep8:
            g = torch.where(kept_z(x, sizes, groups, w, b).abs() > 1e-5, g, 0.0)
    xr, wr, br = (t.clone().requires_grad_() for t in (x, w, b))
    seg = Segments.from_sizes(sizes, dev())
    out = Fn.group_norm_act(xr, seg, groups, wr, br, act=act, keep8=keep8)
    grads = torch.autograd.grad(out, (xr, wr, br), g)
    want, bound = reference(x, sizes, groups, w, b, act, 1e-5, g, keep8)
    for name, a, e, t in zip(("out", "gx", "gw", "gb"), (out, *grads), want, bound):
        within(a.detach(), e, t, name)


def kept_z(x, sizes, groups, w, b):
    per = x.size(1) // groups
    v, out, at = values8(x), [], 0
    for s in sizes:
        if s:
            grp = x[at:at + s].double().reshape(s, groups, per)
            mean = grp.mean((0, 2), keepdim=True)
            rs = 1 / torch.sqrt(((grp - mean) ** 2).mean((0, 2), keepdim=True) + 1e-5)
            out.append(((v[at:at + s].reshape(s, groups, per) - mean) * rs).reshape(s, -1) * w.double() + b.double())
        at += s
    return torch.cat(out)


@pytest.mark.parametrize("layout", ["contiguous", "padded", "slice", "transposed", "offset", "expanded_g"])
@pytest.mark.parametrize("sizes", [[60, 61], [2000, 3]])
def test_layouts(layout, sizes):
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    from hgvae_amd.graph import new_padded
    c, groups = 30, 5
    x, w, b, g = make(sizes, c, 5)
    n = x.size(0)
    if layout == "padded":
        p = new_padded(n, c, dev())
        p.copy_(x)
        x = p
    elif layout == "slice":
        wide = torch.full((n, 64), float("nan"), device=dev())
        wide[:, 8:8 + c] = x
        x = wide[:, 8:8 + c]
    elif layout == "transposed":
        x = x.t().contiguous().t()
    elif layout == "offset":
        flat = torch.empty(n * c + 1, device=dev())
        flat[1:] = x.reshape(-1)
        x = flat[1:].view(n, c)
    elif layout == "expanded_g":
        g = torch.randn(1, c, device=dev()).expand(n, c)
    xr = x.detach().requires_grad_()
    out = Fn.group_norm_act(xr, Segments.from_sizes(sizes, dev()), groups, w, b)
    (gx,) = torch.autograd.grad(out, (xr,), g)
    want, bound = reference(x, sizes, groups, w, b, "silu", 1e-5, g)
    within(out.detach(), want[0], bound[0], "out")
    within(gx, want[1], bound[1], "gx")
    if layout == "slice":
        assert bool(wide[:, :8].isnan().all()) and bool(wide[:, 8 + c:].isnan().all())


def test_outputs_have_zero_pad_columns():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    for sizes in ([50], [1200], [30, 1500]):
        x, w, b, g = make(sizes, 30, 1)
        x.requires_grad_()
        out = Fn.group_norm_act(x, Segments.from_sizes(sizes, dev()), 3, w, b)
        (gx,) = torch.autograd.grad(out, (x,), g)
        for t in (out, gx):
            assert t.stride(0) == 32 and not bool(torch.as_strided(t.detach(), (t.size(0), 2), (32, 1), 30).any())


def test_columns_far_from_zero_and_constant_columns():
    """mean / std = 1e5: x itself has 7 digits, the two-piece mean adds nothing to that; constant groups give xh = 0."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    for sizes in ([200], [3000]):
        x, w, b, _ = make(sizes, 8, 3, offset=False)
        x[:, :4] += 1e5
        x[:, 4:] = 7.25
        out = Fn.group_norm_act(x, Segments.from_sizes(sizes, dev()), 2, w, b, act="none")
        want, bound = reference(x, sizes, 2, w, b, "none", 1e-5)
        within(out, want, bound, "out")
        assert torch.equal(out[:, 4:], b[4:].expand(sum(sizes), 4))


def test_a_bad_graph_stays_alone():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    for sizes in ([50, 60, 70], [1500, 1400, 1600]):
        x, w, b, g = make(sizes, 12, 4)
        clean = Fn.group_norm_act(x, Segments.from_sizes(sizes, dev()), 3, w, b)
        x[sizes[0] + 5, 5] = float("inf")
        x[sizes[0] + 6, 9] = float("nan")
        out = Fn.group_norm_act(x, Segments.from_sizes(sizes, dev()), 3, w, b)
        mid = slice(sizes[0], sizes[0] + sizes[1])
        assert torch.equal(out[:sizes[0]], clean[:sizes[0]]) and torch.equal(out[mid.stop:], clean[mid.stop:])
        assert torch.equal(out[mid, :4], clean[mid, :4]) and bool(out[mid, 4:].isnan().any(0).all())


def test_one_read_and_chunked_kernels_agree_on_a_mixed_batch():
    """A graph's result does not depend on the graphs beside it, nor on how often the call is repeated."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes = [10, 3000, 500, 1, 900, 15200]
    x, w, b, g = make(sizes, 138, 9)
    xr = x.clone().requires_grad_()

    def run():
        out = Fn.group_norm_act(xr, Segments.from_sizes(sizes, dev()), 6, w, b)
        return out.detach(), torch.autograd.grad(out, (xr,), g)[0]

    first, again = run(), run()
    assert torch.equal(first[0], again[0]) and torch.equal(first[1], again[1])
    want, bound = reference(x, sizes, 6, w, b, "silu", 1e-5, g)
    within(first[0], want[0], bound[0], "out")
    within(first[1], want[1], bound[1], "gx")


def test_no_affine_and_single_gradients():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    for sizes in ([40, 3], [1300]):
        x, w, b, g = make(sizes, 24, 2)
        seg = Segments.from_sizes(sizes, dev())
        xr = x.clone().requires_grad_()
        out = Fn.group_norm_act(xr, seg, 4, act="gelu")
        want, bound = reference(x, sizes, 4, None, None, "gelu", 1e-5, g)
        within(torch.autograd.grad(out, (xr,), g)[0], want[1], bound[1], "gx")
        wr = w.clone().requires_grad_()
        out = Fn.group_norm_act(x, seg, 4, wr, b)
        want, bound = reference(x, sizes, 4, w, b, "silu", 1e-5, g)
        within(torch.autograd.grad(out, (wr,), g)[0], want[2], bound[2], "gw")
        br = b.clone().requires_grad_()
        out = Fn.group_norm_act(x, seg, 4, w, br)
        within(torch.autograd.grad(out, (br,), g)[0], want[3], bound[3], "gb")


def test_gradients_against_differences():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes = [7, 5]
    x, w, b, g = make(sizes, 6, 11)
    seg = Segments.from_sizes(sizes, dev())
    xr, wr, br = (t.clone().requires_grad_() for t in (x, w, b))
    grads = torch.autograd.grad(Fn.group_norm_act(xr, seg, 2, wr, br), (xr, wr, br), g)
    # central differences of the float64 formula: error h^2 * third derivative ~ 1e-9, far below fp32's
    for t, got in zip((x, w, b), grads):
        t64 = t.double()
        for idx in range(0, t.numel(), 5):
            vals = []
            for h in (1e-5, -1e-5):
                p = t64.clone()
                p.view(-1)[idx] += h
                args = [p if t is u else u.double() for u in (x, w, b)]
                vals.append(float((reference(args[0], sizes, 2, args[1], args[2], "silu", 1e-5)[0] * g.double()).sum()))
            d = (vals[0] - vals[1]) / 2e-5
            assert abs(d - float(got.reshape(-1)[idx])) <= 1e-6 + 2e-6 * float(got.abs().max())


def test_batch_vector_streams_and_captured_graph():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes = [100, 0, 2000]
    x, w, b, g = make(sizes, 30, 6)
    seg = Segments.from_sizes(sizes, dev())
    batch = torch.repeat_interleave(torch.arange(3, device=dev()), torch.tensor(sizes, device=dev()))
    xr = x.clone().requires_grad_()
    want = Fn.group_norm_act(xr, seg, 3, w, b)
    (wgx,) = torch.autograd.grad(want, (xr,), g)
    assert torch.equal(Fn.group_norm_act(x, batch, 3, w, b), want)
    assert torch.equal(Fn.group_norm_act(x, Segments.from_ptr(torch.tensor([0, 100, 100, 2100], device=dev())), 3, w, b), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = Fn.group_norm_act(x, seg, 3, w, b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, want)
    static = x.clone().requires_grad_()
    with torch.cuda.stream(side):
        Fn.group_norm_act(static, seg, 3, w, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = Fn.group_norm_act(static, seg, 3, w, b, keep8=True)
        (gx,) = torch.autograd.grad(out, (static,), g)
    x2 = x.flip(0).contiguous()
    for data in (x, x2, x, x2):
        with torch.no_grad():
            static.copy_(data)
        graph.replay()
        torch.cuda.synchronize()
        r = data.clone().requires_grad_()
        e = Fn.group_norm_act(r, seg, 3, w, b, keep8=True)
        (egx,) = torch.autograd.grad(e, (r,), g)
        assert torch.equal(out, e) and torch.equal(gx, egx)


def test_empty_batches():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    x = torch.zeros(0, 12, device=dev(), requires_grad=True)
    w = torch.ones(12, device=dev(), requires_grad=True)
    out = Fn.group_norm_act(x, Segments.from_sizes([0, 0], dev()), 3, w)
    out.sum().backward()
    assert out.shape == (0, 12) and float(w.grad.abs().max()) == 0.0
    assert Fn.group_norm_act(x.detach(), Segments.from_sizes([], dev()), 3).shape == (0, 12)


def test_refusals():
    from hgvae_amd import Segments, _lib
    from hgvae_amd import functional as Fn
    seg = Segments.from_sizes([4, 6], dev())
    x = torch.randn(10, 12, device=dev())
    for call in (lambda: Fn.group_norm_act(x, seg, 5), lambda: Fn.group_norm_act(x, seg, 0), lambda: Fn.group_norm_act(x[:9], seg, 3),
                 lambda: Fn.group_norm_act(x.half(), seg, 3), lambda: Fn.group_norm_act(x[0], seg, 3), lambda: Fn.group_norm_act(x, seg, 3, act="tanh"),
                 lambda: Fn.group_norm_act(x, seg, 3, torch.ones(11, device=dev())), lambda: Fn.group_norm_act(x, seg, 3, torch.ones(12)),
                 lambda: Fn.group_norm_act(x, seg, 3, eps=-1.0), lambda: Fn.group_norm_act(x, [4, 6], 3), lambda: Fn.group_norm_act(x.cpu(), seg, 3),
                 lambda: Segments.from_batch(torch.tensor([0, 1, 0], device=dev())), lambda: Segments.from_batch(torch.tensor([-1, 0], device=dev())),
                 lambda: Segments.from_batch(torch.tensor([0, 3], device=dev()), num_graphs=3), lambda: Segments.from_ptr(torch.tensor([1, 3], device=dev())),
                 lambda: Segments.from_ptr(torch.tensor([0, 3, 2], device=dev())), lambda: Segments.from_sizes([2 ** 31 - 1, 1], dev()),
                 lambda: Segments.from_sizes([1.5], dev()), lambda: Segments.from_sizes([3], "cpu")):
        with pytest.raises(_lib.HgvError):
            call()


@pytest.mark.parametrize("sizes", [[700, 2500], [3, 0, 2100], [1100]])
@pytest.mark.parametrize("c,groups", [(36, 3), (64, 4), (65, 5), (138, 6), (256, 8), (1100, 2)])
def test_kept_input_is_its_8bit_form(sizes, c, groups):
    """What the forward pass leaves for the backward pass, with its last pass or by itself: the bytes of pack8(x)."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    n = sum(sizes)
    wide = torch.randn(n, c + 7, device=dev()) * torch.logspace(-3, 3, c + 7, device=dev())
    wide[n // 2, c // 2], wide[n // 3, 0], wide[1, c - 1] = float("nan"), float("inf"), 3e38
    seg = Segments.from_sizes(sizes, dev())
    for x in (wide[:, :c].contiguous(), wide[:, 3:c + 3], wide[:, 7:]):
        out = Fn.group_norm_act(x.detach().requires_grad_(), seg, groups, keep8=True)
        want = Fn.pack8(x)
        kept = [t for t in out.grad_fn.saved_tensors if t is not None and t.dtype in (torch.int8, torch.uint8)]
        assert torch.equal(kept[0][:, :c], want.q[:, :c]) and torch.equal(kept[1], want.scale)
        assert torch.equal(Fn.group_norm_act(x, seg, groups).isnan(), out.isnan())
        assert torch.equal(Fn.group_norm_act(x, seg, groups).nan_to_num(), out.detach().nan_to_num())


@pytest.mark.parametrize("c,groups", [(138, 6), (256, 8)])
def test_many_graphs_of_both_kinds(c, groups):
    """More than 64 MB of graphs of 100 and 300 rows: some read at once, some in chunks, whatever the rule picks."""
    test_group_norm_act_matches_float64([300] * 250 + [100] * 450 + [1, 0, 161, 160], c, groups, "silu", True)
