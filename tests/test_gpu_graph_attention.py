"""Attention within graphs against the formula in float64, row by row bounds.

An operand is two fp16 pieces (relative error 2^-22, an absolute floor 2^-38 of the longest row), a product drops the product of
the two small pieces (2^-22), and sums round in fp32: with u = 2^-24 at most once per four terms and piece.  The bounds below carry
these through the softmax and its gradient.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def make(sizes, h, hk, d, seed, spread=1.0):
    gen = torch.Generator(device=dev()).manual_seed(seed)
    n = sum(sizes)
    q, k, v, g = (torch.randn(n, x, d, generator=gen, device=dev()) for x in (h, hk, hk, h))
    return q * 1.5 * spread, k, v, g


def reference(q, k, v, sizes, mask, scale, g=None):
    """Values and bounds of (out, dq, dk, dv)."""
    n, h, d = q.shape
    r = h // k.size(1)
    q, k, v = q.double(), k.double(), v.double()
    if mask is not None:                                    # masked rows of k and v do not matter
        k = torch.where(mask[:, None, None], k, 0.0)
        v = torch.where(mask[:, None, None], v, 0.0)
    vals = [torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)]
    bnds = [torch.full_like(t, 1e-37) for t in vals]
    at = 0
    for size in sizes:
        rows = slice(at, at + size)
        at += size
        ok = torch.ones(size, dtype=torch.bool, device=q.device) if mask is None else mask[rows]
        if size == 0 or not bool(ok.any()):
            continue
        for head in range(h):
            Q, K, V = q[rows, head].contiguous(), k[rows, head // r].contiguous(), v[rows, head // r].contiguous()
            # longest rows, over the heads that share a scale
            top = lambda t, hs: float(t[rows, hs].norm(dim=-1).max())
            shared = slice(head // r * r, head // r * r + r)
            nq, nk, nv = top(q, shared), float(K.norm(dim=-1).max()), float(V.norm(dim=-1).max())
            per = 4 * 2.0 ** -22                                # two splits, the dropped product, margin for the floors' rounding

            def acc(terms):
                return per + 3 * U * (terms / 4 + 2)

            S = scale * Q @ K.t().contiguous()
            dS = scale * (acc(d) * Q.abs() @ K.abs().t().contiguous() + 2.0 ** -36 * math.sqrt(d) * nq * nk) + 3 * U * S.abs()
            S = S.masked_fill(~ok, -math.inf)
            lse = torch.logsumexp(S, dim=1, keepdim=True)
            P = torch.exp(S - lse)
            # relative error of a probability: its logit, the exponent's rounding, exp2, and the same of the sum
            E = torch.where(ok, dS, 0.0) + torch.where(ok, (S - lse).abs().clamp(max=200.0), 0.0) * 4 * U + 4 * U
            E = E + (P * E).sum(1, keepdim=True) + size / 16 * U
            O = P @ V
            out_b = (P * (E + acc(size))) @ V.abs() + 2.0 ** -30 * size ** 0.5 * nv * 2.0 ** -2 + 4 * U * O.abs()
            vals[0][rows, head], bnds[0][rows, head] = O, out_b
            if g is None:
                continue
            G = g[rows, head].double().contiguous()
            ng = top(g.double(), shared)
            dV, dV_b = P.t().contiguous() @ G, (P * (E + acc(size * r) + 4 * U)).t().contiguous() @ G.abs() + 2.0 ** -36 * size ** 0.5 * ng
            dP = G @ V.t().contiguous()
            dP_b = acc(d) * G.abs() @ V.abs().t().contiguous() + 2.0 ** -36 * math.sqrt(d) * ng * nv
            D = (G * O).sum(1, keepdim=True)
            D_b = (d / 8 + 4) * U * (G * O).abs().sum(1, keepdim=True) + (G.abs() * out_b).sum(1, keepdim=True)
            T = P * (dP - D)
            T_b = P * ((E + 4 * U) * (dP - D).abs() + dP_b + D_b + 2 * U * (dP.abs() + D.abs())) + 2.0 ** -36 * ng * nv * ok
            Tq, Tb = scale * T, scale * (T_b + acc(size * r) * T.abs())
            vals[1][rows, head], bnds[1][rows, head] = Tq @ K, Tb @ K.abs() + 2.0 ** -36 * nk * (scale * T.abs()).sum(1, keepdim=True)
            vals[2][rows, head // r] += torch.where(ok[:, None], Tq.t().contiguous() @ Q, 0.0)
            bnds[2][rows, head // r] += Tb.t().contiguous() @ Q.abs() + 2.0 ** -36 * nq * (scale * T.abs()).sum(0)[:, None]
            vals[3][rows, head // r] += torch.where(ok[:, None], dV, 0.0)
            bnds[3][rows, head // r] += dV_b
    return vals, bnds


def check(got, want, bound, what):
    assert got.shape == want.shape
    err = (got.double() - want).abs()
    bad = ~(err <= bound)
    assert not bool(bad.any()), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float((err / bound)[bad].max()):.3g} bounds, err {float(err.max()):.3g}"


def run(q, k, v, seg, g, mask=None, scale=None):
    from hgvae_amd import functional as Fn
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = Fn.graph_attention(*leaves, seg, mask=mask, scale=scale)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


SHAPES = [([1], 1, 1, 1), ([1, 1, 1], 2, 1, 5), ([2, 0, 3], 1, 1, 32), ([64], 2, 2, 64), ([65, 63], 4, 2, 23), ([138] * 3, 4, 4, 64),
          ([127, 128, 129, 1], 3, 1, 96), ([300], 2, 1, 128), ([454, 7], 6, 2, 23), ([200], 1, 1, 127), ([90, 300], 2, 2, 33), ([1000], 1, 1, 64),
          ([17] * 20, 2, 2, 16), ([700], 3, 3, 97), ([8] * 600, 1, 1, 16)]


@pytest.mark.parametrize("sizes,h,hk,d", SHAPES, ids=[f"{len(s)}x{max(s)}-{h}-{hk}-{d}" for s, h, hk, d in SHAPES])
@pytest.mark.parametrize("masked", [False, True])
def test_matches_float64(sizes, h, hk, d, masked):
    from hgvae_amd import Segments
    q, k, v, g = make(sizes, h, hk, d, seed=sum(sizes) + d)
    mask = None
    if masked:
        mask = torch.rand(sum(sizes), generator=torch.Generator(device=dev()).manual_seed(d), device=dev()) < 0.6
        mask[:sizes[0]] = False                                 # the first graph has no keys
    got = run(q, k, v, Segments.from_sizes(sizes, dev()), g, mask)
    want, bound = reference(q, k, v, sizes, mask, d ** -0.5, g)
    for name, a, e, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        check(a, e, b, name)
    if masked:
        assert not bool(got[0][:sizes[0]].any()) and not bool(got[1][:sizes[0]].any())
        assert not bool(got[2][~mask].any()) and not bool(got[3][~mask].any())


@pytest.mark.parametrize("spread", [1e-12, 1e-3, 8.0, 40.0])
@pytest.mark.parametrize("d", [20, 64])
def test_flat_and_peaked_probabilities(spread, d):
    from hgvae_amd import Segments
    sizes = [150, 333]
    q, k, v, g = make(sizes, 2, 2, d, seed=3, spread=spread)
    got = run(q, k, v, Segments.from_sizes(sizes, dev()), g)
    want, bound = reference(q, k, v, sizes, None, d ** -0.5, g)
    for name, a, e, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
        check(a, e, b, name)


def test_logits_that_grow_along_the_keys():
    """Every tile of keys brings a larger maximum (the running maximum moves each time), or a smaller one."""
    from hgvae_amd import Segments
    sizes = [640]
    q, k, v, g = make(sizes, 1, 1, 64, seed=4)
    ramp = torch.linspace(-60, 60, 640, device=dev())
    q[:, 0] = 0.0
    q[:, 0, 0] = 8.0
    for sign in (1.0, -1.0):
        k[:, 0, 0] = sign * ramp
        got = run(q, k, v, Segments.from_sizes(sizes, dev()), g)
        want, bound = reference(q, k, v, sizes, None, 0.125, g)
        for name, a, e, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
            check(a, e, b, name)


@pytest.mark.parametrize("factor", [1e-25, 1e-6, 1e6, 1e15])
def test_scales_of_the_operands_do_not_matter(factor):
    """v and the incoming gradient times a power of two: the same bits, scaled; q up and k down: the same result."""
    from hgvae_amd import Segments
    f = 2.0 ** round(math.log2(factor))
    sizes = [70, 140]
    q, k, v, g = make(sizes, 2, 1, 40, seed=5)
    seg = Segments.from_sizes(sizes, dev())
    base = run(q, k, v, seg, g)
    out, dq, dk, dv = run(q, k, v * f, seg, g)
    assert torch.equal(out, base[0] * f) and torch.equal(dq, base[1] * f) and torch.equal(dk, base[2] * f) and torch.equal(dv, base[3])
    out, dq, dk, dv = run(q, k, v, seg, g * f)
    assert torch.equal(out, base[0]) and torch.equal(dq, base[1] * f) and torch.equal(dk, base[2] * f) and torch.equal(dv, base[3] * f)
    out, dq, dk, dv = run(q * f, k / f, v, seg, g)
    assert torch.equal(out, base[0]) and torch.equal(dq, base[1] / f) and torch.equal(dk, base[2] * f) and torch.equal(dv, base[3])


def test_bad_values_in_masked_rows_do_not_matter():
    from hgvae_amd import Segments
    sizes = [100, 64]
    q, k, v, g = make(sizes, 2, 2, 24, seed=6)
    mask = torch.ones(164, dtype=torch.bool, device=dev())
    mask[10:20] = mask[163] = mask[100] = False
    seg = Segments.from_sizes(sizes, dev())
    want = run(q, k, v, seg, g, mask)
    for value in (float("nan"), float("inf"), -float("inf"), torch.finfo(torch.float32).min):
        kb, vb = k.clone(), v.clone()
        kb[~mask], vb[~mask] = value, value
        got = run(q, kb, vb, seg, g, mask)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_bad_row_stays_where_it_belongs():
    """NaN in one query: that row of out and dq, and what its gradient reaches.  Other graphs keep their bits."""
    from hgvae_amd import Segments
    sizes = [80, 90, 100]
    q, k, v, g = make(sizes, 1, 1, 32, seed=7)
    seg = Segments.from_sizes(sizes, dev())
    want = run(q, k, v, seg, g)
    q[85, 0, 3] = float("nan")
    got = run(q, k, v, seg, g)
    keep = torch.arange(270, device=dev()) != 85
    assert torch.equal(got[0][keep], want[0][keep]) and bool(got[0][85].isnan().all())
    assert torch.equal(got[1][keep], want[1][keep]) and bool(got[1][85].isnan().all())
    for a, b in zip(got[2:], want[2:]):
        assert torch.equal(a[:80], b[:80]) and torch.equal(a[170:], b[170:])


@pytest.mark.parametrize("layout", ["slices", "heads_first", "transposed", "offset", "expanded_g"])
def test_layouts(layout):
    from hgvae_amd import Segments
    sizes, h, hk, d = [70, 60], 4, 2, 20
    n = sum(sizes)
    q, k, v, g = make(sizes, h, hk, d, seed=8)
    seg = Segments.from_sizes(sizes, dev())
    want = run(q, k, v, seg, g)
    if layout == "slices":
        wide = torch.full((n, (h + 2 * hk) * d + 3), float("nan"), device=dev())
        wide[:, 1:1 + h * d] = q.reshape(n, -1)
        wide[:, 1 + h * d:1 + (h + hk) * d] = k.reshape(n, -1)
        wide[:, 1 + (h + hk) * d:1 + (h + 2 * hk) * d] = v.reshape(n, -1)
        q, k, v = (wide[:, a:b].unflatten(1, (-1, d)) for a, b in
                   ((1, 1 + h * d), (1 + h * d, 1 + (h + hk) * d), (1 + (h + hk) * d, 1 + (h + 2 * hk) * d)))
    elif layout == "heads_first":
        q, k, v, g = (t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k, v, g))
    elif layout == "transposed":
        q, k, v, g = (t.permute(2, 1, 0).contiguous().permute(2, 1, 0) for t in (q, k, v, g))
    elif layout == "offset":
        q, k, v, g = (torch.cat([t.new_zeros(1), t.reshape(-1)])[1:].view(t.shape) for t in (q, k, v, g))
    else:
        g = torch.randn(1, 1, d, device=dev()).expand(n, h, d)
        want = run(q, k, v, seg, g.contiguous())
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, seg, g), want))


def test_single_gradients_and_repeatability():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes = [200, 31]
    q, k, v, g = make(sizes, 4, 2, 64, seed=9)
    seg = Segments.from_sizes(sizes, dev())
    want = run(q, k, v, seg, g)
    assert all(torch.equal(a, b) for a, b in zip(run(q, k, v, seg, g), want))
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == j) for j, t in enumerate((q, k, v))]
        (got,) = torch.autograd.grad(Fn.graph_attention(*leaves, seg), [leaves[i]], g)
        assert torch.equal(got, want[1 + i])
    with torch.no_grad():
        assert torch.equal(Fn.graph_attention(q, k, v, seg), want[0])
    # the graphs beside a graph do not matter
    alone = run(q[200:], k[200:], v[200:], Segments.from_sizes([31], dev()), g[200:])
    assert all(torch.equal(a, b[200:]) for a, b in zip(alone, want))


def test_gradients_against_differences():
    from hgvae_amd import Segments
    sizes, d = [6, 9], 5
    q, k, v, g = make(sizes, 2, 1, d, seed=10)
    grads = run(q, k, v, Segments.from_sizes(sizes, dev()), g)[1:]
    base = [t.double() for t in (q, k, v)]
    for which, got in enumerate(grads):
        for idx in range(0, base[which].numel(), 7):
            vals = []
            for step in (1e-5, -1e-5):
                args = [t.clone() for t in base]
                args[which].view(-1)[idx] += step
                vals.append(float((reference(*args, sizes, None, d ** -0.5)[0][0] * g.double()).sum()))
            # differences of a float64 formula: h^2 * third derivative < 1e-9; fp32 carries 2^-24 of the largest entry a few times
            assert abs((vals[0] - vals[1]) / 2e-5 - float(got.reshape(-1)[idx])) <= 1e-7 + 40 * U * float(got.abs().max())


def test_streams_and_captured_graph():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes = [138, 0, 300]
    q, k, v, g = make(sizes, 2, 2, 48, seed=11)
    mask = torch.rand(438, device=dev()) < 0.8
    seg = Segments.from_sizes(sizes, dev())
    want = run(q, k, v, seg, g, mask)
    batch = torch.repeat_interleave(torch.arange(3, device=dev()), torch.tensor(sizes, device=dev()))
    assert torch.equal(Fn.graph_attention(q, k, v, batch, mask=mask), want[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = run(q, k, v, seg, g, mask)
        again = run(q, k, v, seg, g, mask)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, other, again))
    torch.cuda.synchronize()
    static = [t.clone() for t in (q, k, v, g)]
    graphs, outs = [], []
    for _ in range(2):                                          # two captures share nothing
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(run(*static[:3], seg, static[3], mask))
        graphs.append(graph)
    for flip in (False, True, False, True):
        for t, s in zip((q, k, v, g), static):
            s.copy_(t.flip(0) if flip else t)
        graphs[0].replay()
        graphs[1].replay()
        torch.cuda.synchronize()
        eager = run(*static[:3], seg, static[3], mask)
        for got in outs:
            assert all(torch.equal(a, b) for a, b in zip(got, eager))


def test_empty_and_refusals():
    from hgvae_amd import Segments, _lib
    from hgvae_amd import functional as Fn
    q = torch.zeros(0, 2, 8, device=dev(), requires_grad=True)
    out = Fn.graph_attention(q, q, q, Segments.from_sizes([0], dev()))
    out.sum().backward()
    assert out.shape == (0, 2, 8) and q.grad.shape == q.shape
    seg = Segments.from_sizes([4, 6], dev())
    q, k = torch.randn(10, 4, 8, device=dev()), torch.randn(10, 2, 8, device=dev())
    for call in (lambda: Fn.graph_attention(q, k, k[:, :1], seg), lambda: Fn.graph_attention(q[:, :3], k, k, seg), lambda: Fn.graph_attention(q.half(), k, k, seg),
                 lambda: Fn.graph_attention(q[:9], k[:9], k[:9], seg), lambda: Fn.graph_attention(q, k[..., :7], k[..., :7], seg),
                 lambda: Fn.graph_attention(q.cpu(), k, k, seg), lambda: Fn.graph_attention(q, k, k, seg, scale=0.0), lambda: Fn.graph_attention(q, k, k, seg, scale=float("nan")),
                 lambda: Fn.graph_attention(q, k, k, seg, mask=torch.ones(10, device=dev())), lambda: Fn.graph_attention(q, k, k, seg, mask=torch.ones(9, dtype=torch.bool, device=dev())),
                 lambda: Fn.graph_attention(q[:, 0], k, k, seg), lambda: Fn.graph_attention(torch.randn(10, 1, 129, device=dev()), torch.randn(10, 1, 129, device=dev()), torch.randn(10, 1, 129, device=dev()), seg),
                 lambda: Fn.graph_attention(q, k, k, Segments.from_sizes([4, 5], dev()))):
        with pytest.raises(_lib.HgvError):
            call()
