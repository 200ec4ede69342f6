"""Attention within graphs where single rows or single keys decide."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def make(n, h, hk, d, seed):
    gen = torch.Generator(device=dev()).manual_seed(seed)
    return tuple(torch.randn(n, x, d, generator=gen, device=dev()) for x in (h, hk, hk, h))


def run(q, k, v, sizes, g, mask=None):
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    out = Fn.graph_attention(*leaves, Segments.from_sizes(sizes, dev()), mask=mask)
    return (out.detach(), *torch.autograd.grad(out, leaves, g))


@pytest.mark.parametrize("h,hk,d", [(1, 1, 1), (4, 2, 9), (4, 2, 23), (4, 4, 64), (3, 1, 128)])
@pytest.mark.parametrize("sizes,keys", [([1] * 17, None), ([1, 5, 1, 0, 700, 1], None), ([200], [130]), ([40, 600, 3], [7, 40, 642]),
                                        ([5, 130], [0, 4, 5, 134])])
def test_gradients_through_a_single_key_are_zero(h, hk, d, sizes, keys):
    """A query with one key has the probability 1 whatever its logit is: dq and dk are zero, to the last bit."""
    n = sum(sizes)
    q, k, v, g = make(n, h, hk, d, seed=n + d)
    mask = None
    if keys is not None:
        mask = torch.zeros(n, dtype=torch.bool, device=dev())
        mask[torch.tensor(keys, device=dev())] = True
    out, dq, dk, dv = run(q, k, v, sizes, g, mask)
    at = 0
    for size in sizes:
        rows = torch.arange(at, at + size, device=dev())
        at += size
        live = rows if mask is None else rows[mask[rows]]
        if live.numel() == 1:
            assert not bool(dq[rows].any()) and not bool(dk[rows].any())
            # out is the one value, dv the sum of the gradients: pieces of 22 bits, a rounding or two in fp32, and dv's sum
            want = v[live].repeat_interleave(h // hk, 1).expand(size, h, d).double()
            assert bool(((out[rows].double() - want).abs() <= 2.0 ** -20 * v[live].abs().amax()).all())
            parts = g[rows].double().view(size, hk, h // hk, d)
            bound = (2.0 ** -20 + U * size) * parts.abs().sum((0, 2)) + 1e-9
            assert bool(((dv[live[0]].double() - parts.sum((0, 2))).abs() <= bound).all())
        elif live.numel() > 1:
            assert bool(dq[rows].any()) and bool(dk[live].any())


@pytest.mark.parametrize("n,h,hk,d", [(300, 2, 1, 23), (300, 1, 1, 64), (5000, 1, 1, 64), (5000, 2, 2, 40), (2600, 1, 1, 128)])
@pytest.mark.parametrize("factor", [2.0 ** 10, 2.0 ** 14, 2.0 ** 20])
def test_dq_of_ordinary_rows_beside_one_with_a_large_gradient(n, h, hk, d, factor):
    """dq of a row depends on that row's gradient alone, and is as exact as if the others' were of its size."""
    q, k, v, g = make(n, h, hk, d, seed=n + d)
    g[n // 3] *= factor
    dq = run(q, k, v, [n], g)[1].double()
    scale = d ** -0.5
    for head in range(h):
        Q, K, V, G = (t[:, i].double() for t, i in ((q, head), (k, head * hk // h), (v, head * hk // h), (g, head)))
        P = torch.softmax(scale * Q @ K.t().contiguous(), 1)
        dP = G @ V.t().contiguous()
        D = (P * dP).sum(1, keepdim=True)
        want = scale * (P * (dP - D)) @ K
        # relative to sum_j p_j (|dP_j| + |D|) |k_j|: logits of about 25 at most from 22-bit pieces and fp32 (their errors times the
        # probability), dP and D likewise, a split of the sum's terms, sums of n terms a fourth at a time;  and the two floors
        # 2^-39 of the pieces against the row's and the graph's own norms
        terms = scale * (P * (dP.abs() + D.abs())) @ K.abs()
        norms = G.norm(dim=1, keepdim=True) * V.norm(dim=1).max() * K.norm(dim=1).max() * scale
        logit = scale * (Q.norm(dim=1) * K.norm(dim=1).max()).max()
        bound = terms * (logit * 2.0 ** -20 + 2.0 ** -20 + n / 4 * U) + norms * 2.0 ** -34 * n ** 0.5
        err = (dq[:, head] - want).abs()
        assert bool((err <= bound).all()), f"{float((err / bound).max()):.3g} bounds"
        # by row: pieces of 22 bits in q, k, v and g, and fp32 sums
        off = (dq[:, head] - want).norm(dim=1) / want.norm(dim=1)
        assert float(off.max()) <= 2.0 ** -15, float(off.max())


@pytest.mark.parametrize("sizes", [[40, 70], [600, 90]])
@pytest.mark.parametrize("value", [float("nan"), float("inf"), -float("inf")])
def test_bad_queries_of_a_graph_without_keys_give_zeros(sizes, value):
    """A graph without keys gives zeros and zero gradients, whatever its rows of q, k, v and g hold; the other keeps its bits."""
    n, first = sum(sizes), sizes[0]
    q, k, v, g = make(n, 4, 2, 24, seed=n)
    mask = torch.arange(n, device=dev()) >= first
    want = run(q, k, v, sizes, g, mask)
    for t in (q, k, v, g):
        t[3], t[first - 1, 0, 5] = value, value
    got = run(q, k, v, sizes, g, mask)
    for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
        assert not bool(a[:first].any()) and torch.equal(a[first:], b[first:]), name


@pytest.mark.parametrize("h,hk,d", [(2, 1, 23), (1, 1, 64)])
@pytest.mark.parametrize("sizes", [[8] * 40 + [513, 512], [512, 511, 1, 64], [600] + [3] * 30])
def test_graphs_on_both_sides_of_the_limit_of_the_small_kernel(sizes, h, hk, d):
    """Batches whose largest graph takes images of the operands, with graphs of a few rows beside it, and batches that do without."""
    from test_gpu_graph_attention import check, reference
    n = sum(sizes)
    q, k, v, g = make(n, h, hk, d, seed=n + d)
    mask = torch.rand(n, generator=torch.Generator(device=dev()).manual_seed(d), device=dev()) < 0.7
    for m in (None, mask):
        got = run(q, k, v, sizes, g, m)
        want, bound = reference(q, k, v, sizes, m, d ** -0.5, g)
        for name, a, e, b in zip(("out", "dq", "dk", "dv"), got, want, bound):
            check(a, e, b, name)


@pytest.mark.parametrize("mean", [0.0, 1.0])
@pytest.mark.parametrize("h,hk,d", [(2, 1, 4), (1, 1, 23), (1, 1, 64), (1, 1, 128)])
def test_long_sums(h, hk, d, mean):
    """Sums over the 9 000 nodes of a graph, of values and gradients with and without a mean, against float64 by their norms.

    The sums: parts of 1 024 rows in the matrix cores, six roundings per 64 rows, nine parts.  Where the terms do not cancel a part
    grows to a ninth of the whole: sqrt(9 * 96 / 3) / 9 = 1.9, and nine additions sqrt(9 / 3) = 1.7;  where they cancel to a third:
    sqrt(9 * 96 / 2) / 3 = 6.9, and sqrt(9 / 2) = 2.1;  10 in units of 2^-24 of the result holds both.  dv of heads of 33 ... 64 and 97 ...
    128 columns has no second sum: sqrt(850 / 2) = 20.6 by the same count, and the cuts of one sign beside it: 40.
    The terms: a probability is off by ln 2 times its logit's error (the exponent's rounding, |logit - M| < 32: 2^-20; three
    sums of |logit| < 16: 3 * 2^-21; three times the pieces' 2^-24 of the products, below 16: 3 * 2^-23), exp2's 2^-23, its split's 2^-22: 5 * 2^-21
    together, which also holds the relative error of dP and D in units of |dP| + |D| + the root of the products' squares.  Errors of
    single terms are independent and add in squares.
    dq: what D = sum_j p_j dP_j has from out's sum moves all terms of the row alike."""
    n = 9000
    q, k, v, g = make(n, h, hk, d, seed=d)
    q *= 1.5
    v += mean
    g += mean
    got = run(q, k, v, [n], g)
    want, single = ([torch.zeros_like(t, dtype=torch.float64) for t in (q, q, k, v)] for _ in range(2))
    common = torch.zeros_like(q, dtype=torch.float64)
    scale = d ** -0.5
    for i in range(h):
        j = i * hk // h
        Q, K, V, G = (t[:, x].double().contiguous() for t, x in ((q, i), (k, j), (v, j), (g, i)))
        P = torch.softmax(scale * Q @ K.t().contiguous(), 1)
        O = P @ V
        D = (G * O).sum(1, keepdim=True)
        dP = G @ V.t().contiguous()
        T = scale * P * (dP - D)
        M = (scale * P * (dP.abs() + D.abs() + ((G * G) @ (V * V).t().contiguous()).sqrt())) ** 2
        want[0][:, i], want[1][:, i], common[:, i] = O, T @ K, scale * D * (P @ K)
        want[2][:, j] += T.t().contiguous() @ Q
        want[3][:, j] += P.t().contiguous() @ G
        single[0][:, i], single[1][:, i] = (P * P) @ (V * V), M @ (K * K)
        single[2][:, j] += M.t().contiguous() @ (Q * Q)
        single[3][:, j] += (P * P).t().contiguous() @ (G * G)
    for name, a, e, s in zip(("out", "dq", "dk", "dv"), got, want, single):
        second = name != "dv" or d <= 32 or 64 < d <= 96
        allowed = (10 if second else 40) * U * e.norm() + 5 * 2.0 ** -21 * s.sum().sqrt()
        if name == "dq":
            allowed = allowed + 10 * U * common.norm()
        off = (a.double() - e).norm()
        assert float(off) <= float(allowed), f"{name}: {float(off / allowed):.3g} of what is allowed"


@pytest.mark.parametrize("h,hk,d", [(1, 1, 64), (2, 1, 23), (1, 1, 96)])
@pytest.mark.parametrize("which", ["g", "v"])
@pytest.mark.parametrize("factor", [2.0 ** 6, 2.0 ** 10, 2.0 ** 16])
def test_dq_and_dk_beside_one_large_row(h, hk, d, which, factor):
    """One row of g or of v far larger than the others of its graph: dq and dk as a whole stay as exact as fp32 is.

    The logits' gradient is split with an absolute floor 2^-25 under a bound of 2^14 that holds for the largest gradient and the largest
    probability of 1 024 rows (dk) or of the row (dq).  A term of ordinary size, |dP| about |do| |v| / 8, next to its bound: 2^11.  With a large row of v
    the bound is F times too high for all others: 2^11 / F, at F = 2^10 2^1 with errors of 2^-26, and the large row's own
    terms, p F |do| |v|, of which n are summed, are as many times larger: 6 000 errors of 2^-26 against 2^11, 2^-31 of the whole.
    So the bound is that of the long sums, 10 * 2^-24 of the norm, and of single terms' errors, 5 * 2^-21 in squares, where they cancel in
    full: 50 * 2^-24 at most."""
    n = 6000
    q, k, v, g = make(n, h, hk, d, seed=d)
    (g if which == "g" else v)[n // 3] *= factor
    _, dq, dk, _ = run(q, k, v, [n], g)
    want = [torch.zeros_like(t, dtype=torch.float64) for t in (q, k)]
    scale = d ** -0.5
    for i in range(h):
        j = i * hk // h
        Q, K, V, G = (t[:, x].double().contiguous() for t, x in ((q, i), (k, j), (v, j), (g, i)))
        P = torch.softmax(scale * Q @ K.t().contiguous(), 1)
        T = scale * P * (G @ V.t().contiguous() - (G * (P @ V)).sum(1, keepdim=True))
        want[0][:, i] = T @ K
        want[1][:, j] += T.t().contiguous() @ Q
    for name, a, e in zip(("dq", "dk"), (dq, dk), want):
        off = float((a.double() - e).norm() / e.norm())
        assert off <= 50 * U, f"{name}: {off:.3g}"
