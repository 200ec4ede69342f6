"""Projections of column slices: nothing behind a slice of whole 16-byte chunks is read, also where its last row ends the buffer."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", ["f16x3", "bf16x6", "fp32"])
@pytest.mark.parametrize("k,m", [(4, 20), (12, 138), (20, 64), (60, 33), (100, 138), (148, 40), (204, 138), (284, 288)])
def test_slices_of_whole_chunks(kind, k, m):
    from hgvae_amd import functional as Fn
    if Fn._CHECK_PADS:
        pytest.skip("such a matrix is refused under HGVAE_CHECK_PADS")
    dev = torch.device("cuda:0")
    n = 128
    gen = torch.Generator(device=dev).manual_seed(k + m)
    x, w, b = (torch.randn(*s, generator=gen, device=dev) for s in ((n, k), (m, k), (m,)))
    w2 = torch.randn(m, k, generator=gen, device=dev)
    before = Fn._projection
    try:
        Fn.set_projection(kind)
        want, want2 = Fn.dual_linear(x, w, bias=b), Fn.dual_linear(x, w, x, w2, b)
        for first, width in ((0, k + 8), (8, k + 8), (4, k + 12)):
            wide = torch.full((n, width), float("nan"), device=dev)
            wide[:, first:first + k] = x
            part = wide[:, first:first + k]
            assert torch.equal(Fn.dual_linear(part, w, bias=b), want)
            assert torch.equal(Fn.dual_linear(part, w, part, w2, b), want2)
    finally:
        Fn.set_projection(before)
