"""linear8: sums over a long axis, and operands whose rows are followed by foreign values."""
import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


def grads(x, w, b, g):
    from hgvae_amd import functional as Fn
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = Fn.linear8(*leaves)
    return (y.detach(), *torch.autograd.grad(y, leaves, g))


@pytest.mark.parametrize("mean", [0.0, 1.0, -1.0])
@pytest.mark.parametrize("n,k,m", [(1000003, 20, 12), (500000, 33, 138)])
def test_long_sums_do_not_drift(n, k, m, mean):
    """Weight and bias gradients over many rows.  The products are exact; sums of a tile, of eight tiles and of all tiles of a
    workgroup are fp32, workgroups are added in fp64.  Roundings that do not lean to one side add in squares: a workgroup adds
    about 130 tiles, so with a rounding of 2^-24 of the sum so far, which grows like the root of the tiles added, they stay below
    sqrt(130 / 8 * 8 * 8 / 130 / 2 + 130 / 8 / 2) * 2^-24 < 4 * 2^-24 of it; twice that is allowed."""
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(n + k)
    x = torch.nn.functional.silu(torch.randn(n, k, generator=gen, device=dev()))
    w, b = torch.randn(m, k, generator=gen, device=dev()), torch.randn(m, generator=gen, device=dev())
    g = (torch.randn(n, m, generator=gen, device=dev()) + mean) * 1e-2
    _, _, gw, gb = grads(x, w, b, g)
    for got, want in ((gw, g.double().t().contiguous() @ Fn.pack8(x).unpack().double()), (gb, g.double().sum(0))):
        assert float((got.double() - want).norm() / want.norm()) <= 8 * U


# widths that run in each of the product's kernels: short and long sources, weights in registers, in LDS whole, in two parts, streamed
WIDTHS = [(5, 3), (20, 12), (28, 138), (90, 33), (97, 40), (105, 256), (138, 138), (141, 20), (150, 30), (203, 138), (270, 50), (285, 287)]


def followed_by(t, width, value, first=0):
    """The matrix as columns ``first`` ... of one that is ``width`` wide and holds ``value`` elsewhere."""
    wide = torch.full((t.size(0), width), value, device=dev())
    wide[:, first:first + t.size(1)] = t
    return wide[:, first:first + t.size(1)]


@pytest.mark.parametrize("k,m", WIDTHS)
@pytest.mark.parametrize("n", [1, 37, 4100])
def test_what_lies_behind_the_last_column_does_not_matter(k, m, n):
    """Operands and gradients as slices of wider matrices, of the next multiple of 4 columns and beyond: the same bits."""
    gen = torch.Generator(device=dev()).manual_seed(k + m + n)
    x, w, b, g = (torch.randn(*s, generator=gen, device=dev()) for s in ((n, k), (m, k), (m,), (n, m)))
    want = grads(x, w, b, g)
    for value in (1e6, float("inf"), float("nan")):
        for first, more in ((0, 0), (0, 4), (0, 13), (8, 8)):         # the last: a slice that ends the buffer
            xs, gs = (followed_by(t, (t.size(1) + more + 3) // 4 * 4, value, first) for t in (x, g))
            for got in (grads(xs, w, b, g), grads(x, w, b, gs)):
                assert all(torch.equal(a, c) for a, c in zip(got, want)), (value, first, more)


@pytest.mark.parametrize("k,m", [(90, 33), (97, 138), (138, 138), (30, 20)])
def test_gradients_handed_on_by_a_concatenation(k, m):
    """The gradient of the first part of a concatenation is a slice of the whole, with the other part's behind it."""
    from hgvae_amd import functional as Fn
    n, other = 300, 4 - m % 4
    gen = torch.Generator(device=dev()).manual_seed(k + m)
    x, w, g = (torch.randn(*s, generator=gen, device=dev()) for s in ((n, k), (m, k), (n, m + other)))
    want = grads(x, w, torch.zeros(m, device=dev()), g[:, :m].contiguous())
    for value in (1.0, 1e30, float("inf")):
        g[:, m:] = value
        args = [t.clone().requires_grad_() for t in (x, w)]
        z = torch.randn(n, other, generator=gen, device=dev())
        got = torch.autograd.grad(torch.cat([Fn.linear8(*args), z], 1), args, g)
        assert torch.equal(got[0], want[1]) and torch.equal(got[1], want[2])


@pytest.mark.parametrize("kind", ["f16x3", "bf16x6", "fp32", "auto"])
def test_foreign_columns_in_every_arithmetic_and_without_a_weight_gradient(kind):
    from hgvae_amd import functional as Fn
    n, k, m = 200, 106, 138
    x, w, b, g = (torch.randn(*s, generator=torch.Generator(device=dev()).manual_seed(5), device=dev()) for s in ((n, k), (m, k), (m,), (n, m)))
    before = Fn._projection
    try:
        Fn.set_projection(kind)
        want = grads(x, w, b, g)
        xs, gs = followed_by(x, 108, float("nan")), followed_by(g, 140, float("nan"))
        assert all(torch.equal(a, c) for a, c in zip(grads(xs, w, b, gs), want))
        with torch.no_grad():
            assert torch.equal(Fn.linear8(xs, w, b), want[0])
        xr, br = xs.detach().requires_grad_(), b.clone().requires_grad_()
        gx, gb = torch.autograd.grad(Fn.linear8(xr, w, br), (xr, br), gs)
        assert torch.equal(gx, want[1])
        assert bool(((gb.double() - g.double().sum(0)).abs() <= n * U * g.double().abs().sum(0)).all())
    finally:
        Fn.set_projection(before)
