"""linear8: sums over a long axis."""
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
