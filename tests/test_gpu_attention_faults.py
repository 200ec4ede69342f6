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
