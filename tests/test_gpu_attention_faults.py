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
