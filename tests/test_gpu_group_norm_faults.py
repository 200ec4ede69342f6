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
