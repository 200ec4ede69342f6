"""Group norm: gradients that are zero by definition."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu"])
@pytest.mark.parametrize("sizes,c", [([1, 1, 1], 198), ([1], 1), ([1, 3000, 1, 0, 1], 37), ([1, 700, 1], 64), ([1] * 300, 5)])
def test_the_gradient_of_a_single_value_is_zero(sizes, c, act):
    """One value per (graph, group) is its own mean: the level's output does not depend on it, and gx is zero, to the last bit."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(c + sum(sizes))
    n = sum(sizes)
    x = (torch.randn(n, c, generator=gen, device=dev()) * 3.0 + 5.0).requires_grad_()
    w, b = torch.rand(c, generator=gen, device=dev()) + 0.5, torch.randn(c, generator=gen, device=dev())
    g = torch.randn(n, c, generator=gen, device=dev())
    out = Fn.group_norm_act(x, Segments.from_sizes(sizes, dev()), c, w, b, act=act)
    (gx,) = torch.autograd.grad(out, x, g)
    single = torch.repeat_interleave(torch.tensor(sizes) == 1, torch.tensor(sizes)).to(dev())
    assert not bool(gx[single].any())
    if act != "relu" and not bool(single.all()):
        assert bool(gx[~single].any())


@pytest.mark.parametrize("keep8", [False, True])
def test_row_layouts_agree_where_the_kernels_differ(keep8):
    """More than 64 MB in columns whose pieces are not whole lines: graphs of 300 rows run in chunks where rows are multiples of 16
    bytes apart, else one workgroup reads each at once, in the forward and in the backward pass by themselves."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes, c, groups = [300] * 300 + [100] * 450 + [1, 0, 161, 160], 138, 6
    n = sum(sizes)
    gen = torch.Generator(device=dev()).manual_seed(2)
    x, g = (torch.randn(n, c, generator=gen, device=dev()) for _ in range(2))
    w, b = torch.rand(c, generator=gen, device=dev()) + 0.5, torch.randn(c, generator=gen, device=dev())
    seg = Segments.from_sizes(sizes, dev())

    def padded(t):
        wide = torch.full((n, 140), float("nan"), device=dev())
        wide[:, :c] = t
        return wide[:, :c]

    def run(x, g):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        out = Fn.group_norm_act(leaves[0], seg, groups, *leaves[1:], keep8=keep8)
        return (out.detach(), *torch.autograd.grad(out, leaves, g))

    want = run(x, g)
    assert seg._norm_plan(c, groups, False)[1][2] > seg._norm_plan(c, groups, True)[1][2] > 0
    for other in (run(padded(x), padded(g)), run(padded(x), g), run(x, padded(g))):
        for a, e in zip(other, want):
            # sums in 64 bits in another order, rounded to 32: the statistics, then a handful of operations on them
            assert bool(((a - e).abs() <= 8 * 2.0 ** -24 * e.abs().max()).all())
