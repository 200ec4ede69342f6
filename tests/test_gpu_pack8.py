"""Activation checkpoints in 8 bits: the packed form bit for bit, and the projection that keeps its input that way."""
import pytest
import torch

from test_gpu_group_norm import values8

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def dev():
    return torch.device("cuda:0")


@pytest.mark.parametrize("n,c", [(1, 1), (3, 31), (5, 32), (7, 33), (1000, 138), (4, 256), (2, 1100), (70001, 5), (33, 1025)])
@pytest.mark.parametrize("layout", ["contiguous", "slice", "transposed"])
def test_pack8_round_trip_is_exact(n, c, layout):
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(n + c)
    x = torch.randn(n, c, generator=gen, device=dev()) * torch.exp2(torch.randint(-30, 30, (n, 1), generator=gen, device=dev()).float())
    if layout == "slice":
        wide = torch.full((n, c + 13), float("nan"), device=dev())
        wide[:, 4:4 + c] = x
        x = wide[:, 4:4 + c]
    elif layout == "transposed":
        x = x.t().contiguous().t()
    p = Fn.pack8(x)
    assert torch.equal(p.unpack().double(), values8(x))
    assert p.q.shape == (n, (c + 15) // 16 * 16) and p.scale.shape == (n, (c + 31) // 32)
    assert not bool(p.q[:, c:].any()) and int(p.q.min()) >= -127 and p.nbytes() == p.q.numel() + p.scale.numel()
    # half a step, and a step is at most 1/63 of the block's largest magnitude
    for j, cols in enumerate(torch.split(x.double(), 32, dim=1)):
        step = torch.exp2(p.scale[:, j:j + 1].double() - 127)
        assert bool(((values8(x)[:, 32 * j:32 * j + 32] - cols).abs() <= step / 2).all())
        assert bool((step <= cols.abs().amax(1, keepdim=True) / 63).all())


def test_pack8_borders():
    """Ties to even, the carry into the next power of two, zeros, the smallest and largest numbers, infinities and NaN."""
    from hgvae_amd import functional as Fn
    big, tiny = torch.finfo(torch.float32).max, torch.finfo(torch.float32).tiny
    rows = [[64.0, 0.5, 1.5, 2.5, -0.5, -1.5], [127.0, 126.5, 125.5, -126.5, 0.0, 0.0], [127.4, 1.0, 0.0, 0.0, 0.0, 0.0],
            [127.5, 1.0, 3.0, 5.0, -1.0, -3.0], [127.99, 1.0, 0.0, 0.0, 0.0, 0.0], [0.0] * 6, [-0.0] * 6, [big, -big, 1.0, 0.0, 0.0, 0.0],
            [tiny, -tiny, tiny / 2, 0.0, 0.0, 0.0], [2.0 ** -149, 2.0 ** -140, 0.0, 0.0, 0.0, 0.0], [2.0 ** -120, 2.0 ** -127, 2.0 ** -126, 1.5 * 2.0 ** -126, 0.0, 0.0]]
    x = torch.tensor(rows, device=dev())
    p = Fn.pack8(x)
    assert torch.equal(p.unpack().double(), values8(x))
    assert p.q[0, :6].tolist() == [64, 0, 2, 2, 0, -2] and p.q[3, :6].tolist() == [64, 0, 2, 2, 0, -2]
    bad = torch.zeros(3, 70, device=dev())
    bad[0, 40], bad[1, 69], bad[2, 0] = float("inf"), float("nan"), -float("inf")
    bad[:, 33] = 2.0
    got = Fn.pack8(bad).unpack()
    nan = torch.zeros(3, 70, dtype=torch.bool, device=dev())
    nan[0, 32:64] = nan[1, 64:] = nan[2, :32] = True
    assert torch.equal(got.isnan(), nan) and float(got[2, 33]) == 2.0


def reference(x, w, b, g):
    x, w, g = x.double(), w.double(), g.double()
    v = values8(x)
    y = x @ w.t() + (0 if b is None else b.double())
    k, m, n = x.size(1), w.size(0), x.size(0)
    # products: two fp16 pieces per operand drop 3 * 2^-22 of a term, the sums round once per 32 terms and piece
    per = 4 * 2.0 ** -22
    return ((y, per * (x.abs() @ w.abs().t()) + 4 * U * (1 + k / 8) * (x.abs() @ w.abs().t()) + 2 * U * y.abs()),
            (g @ w, (per + 4 * U * (1 + m / 8)) * (g.abs() @ w.abs())),
            (g.t() @ v, (4 * U + U * (8 + n / 16)) * (g.abs().t() @ v.abs())),
            (g.sum(0), (4 * U + U * (8 + n / 16)) * g.abs().sum(0)))


@pytest.mark.parametrize("n,k,m", [(1, 1, 1), (2, 5, 7), (31, 32, 33), (138, 138, 138), (4416, 138, 138), (5000, 105, 256), (777, 288, 288),
                                   (20011, 256, 12), (9001, 9, 138), (33, 144, 144), (64, 17, 280), (70825, 60, 145)])
@pytest.mark.parametrize("bias", [True, False])
def test_linear8_matches_float64(n, k, m, bias):
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(n + k + m)
    x = torch.nn.functional.silu(torch.randn(n, k, generator=gen, device=dev()))
    w = torch.randn(m, k, generator=gen, device=dev()) / k ** 0.5
    b = torch.randn(m, generator=gen, device=dev()) if bias else None
    g = torch.randn(n, m, generator=gen, device=dev())
    args = [t.clone().requires_grad_() for t in (x, w) + ((b,) if bias else ())]
    y = Fn.linear8(*args)
    got = (y.detach(), *torch.autograd.grad(y, args, g))
    for name, a, (want, bound) in zip(("y", "gx", "gw", "gb"), got, reference(x, w, b, g)):
        err = (a.double() - want).abs()
        assert a.shape == want.shape and bool((err <= bound + 1e-37).all()), f"{name}: {float((err / (bound + 1e-37)).max()):.3g} bounds"


def test_linear8_gradients_one_at_a_time_and_repeatable():
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(1)
    x, w, b, g = (torch.randn(*s, generator=gen, device=dev()) for s in ((3000, 138), (140, 138), (140,), (3000, 140)))
    full = [t.clone().requires_grad_() for t in (x, w, b)]
    want = torch.autograd.grad(Fn.linear8(*full), full, g)
    for i in range(3):
        args = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(Fn.linear8(*args), [args[i]], g)
        if i < 2:
            assert torch.equal(got, want[i])
        else:
            assert float((got - want[i]).abs().max()) <= 3000 * U * float(g.abs().sum(0).max())
    assert all(torch.equal(a, c) for a, c in zip(torch.autograd.grad(Fn.linear8(*full), full, g), want))


def test_linear8_layouts_and_foreign_columns():
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(2)
    n, k, m = 600, 105, 70
    x, w, g = (torch.randn(*s, generator=gen, device=dev()) for s in ((n, k), (m, k), (n, m)))
    wide = torch.full((n, 140), float("nan"), device=dev())
    wide[:, :k] = x
    gwide = torch.full((n, 88), float("nan"), device=dev())
    gwide[:, :m] = g
    for xs, ws, gs in ((wide[:, :k], w, g), (x.t().contiguous().t(), w.t().contiguous().t(), gwide[:, :m]),
                       (x, w, torch.randn(1, m, generator=gen, device=dev()).expand(n, m))):
        xr, wr = xs.detach().requires_grad_(), ws.detach().requires_grad_()
        y = Fn.linear8(xr, wr)
        got = (y.detach(), *torch.autograd.grad(y, (xr, wr), gs))
        for a, (want, bound) in zip(got, reference(xs, ws, None, gs)):
            assert bool(((a.double() - want).abs() <= bound).all())


def test_linear8_keeps_a_quarter():
    """What a level holds between the passes is the 8-bit form, not the matrix."""
    from hgvae_amd import functional as Fn
    w = torch.randn(16, 256, device=dev(), requires_grad=True)
    x = torch.randn(1 << 16, 256, device=dev(), requires_grad=True)
    y = Fn.linear8(x * 1.0, w)
    kept = {t.data_ptr(): t.untyped_storage().nbytes() for t in y.grad_fn.saved_tensors if t is not w}
    assert sum(kept.values()) <= 1.04 * x.numel() and not any(t.dtype == torch.float32 and t.shape == x.shape for t in y.grad_fn.saved_tensors)


def test_linear8_captured_and_on_another_stream():
    from hgvae_amd import functional as Fn
    if Fn._CHECK_PADS:
        pytest.skip("HGVAE_CHECK_PADS synchronises")
    gen = torch.Generator(device=dev()).manual_seed(3)
    x, w, b, g = (torch.randn(*s, generator=gen, device=dev()) for s in ((4416, 138), (138, 138), (138,), (4416, 138)))

    def step(x):
        args = [t.detach().requires_grad_() for t in (x, w, b)]
        y = Fn.linear8(*args)
        return (y.detach(), *torch.autograd.grad(y, args, g))

    want = step(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(other, want))
    static = x.clone()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(static)
    for data in (x, x * 2, x.flip(0).contiguous(), x):
        static.copy_(data)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(out, step(data)))


def test_pack8_linear8_empty_and_refusals():
    from hgvae_amd import _lib
    from hgvae_amd import functional as Fn
    assert Fn.pack8(torch.zeros(0, 5, device=dev())).unpack().shape == (0, 5)
    w = torch.randn(4, 5, device=dev(), requires_grad=True)
    y = Fn.linear8(torch.zeros(0, 5, device=dev()), w)
    y.sum().backward()
    assert y.shape == (0, 4) and float(w.grad.abs().max()) == 0.0
    x = torch.randn(6, 5, device=dev())
    for call in (lambda: Fn.pack8(x.half()), lambda: Fn.pack8(x[0]), lambda: Fn.pack8(x.cpu()), lambda: Fn.pack8(torch.zeros(4, 0, device=dev())),
                 lambda: Fn.linear8(x, torch.randn(4, 6, device=dev())), lambda: Fn.linear8(x, w.detach().cpu()),
                 lambda: Fn.linear8(x, w, torch.randn(5, device=dev())), lambda: Fn.linear8(torch.randn(6, 300, device=dev()), torch.randn(4, 300, device=dev())),
                 lambda: Fn.linear8(x, torch.randn(300, 5, device=dev())), lambda: Fn.linear8(x, w.detach().double())):
        with pytest.raises(_lib.HgvError):
            call()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 4113, 8191])
@pytest.mark.parametrize("k,m", [(96, 40), (97, 40), (100, 138), (105, 256), (128, 33), (138, 138), (140, 100), (144, 144), (145, 144), (256, 64)])
def test_projection_keeps_the_8bit_form(n, k, m):
    """What the product leaves for the weight gradient, in one launch or by itself: pack8(x) byte for byte, zeros behind the last
    column; and the product itself is what it is without."""
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(n + k)
    x = torch.randn(n, k, generator=gen, device=dev()) * torch.exp2(torch.randint(-40, 40, (n, 1), generator=gen, device=dev()).float())
    x[:, k - 1] *= 1e-3
    x[n // 2] = 0.0
    w, b = torch.randn(m, k, generator=gen, device=dev()), torch.randn(m, generator=gen, device=dev())
    y = Fn.linear8(x, w.clone().requires_grad_(), b)
    q, scale = (t for t in y.grad_fn.saved_tensors if t.dtype in (torch.int8, torch.uint8))
    want = Fn.pack8(x)
    assert torch.equal(q, want.q) and torch.equal(scale, want.scale)
    assert torch.equal(y.detach(), Fn.linear8(x, w, b))


@pytest.mark.parametrize("k", [97, 138, 143])
def test_kept_form_ignores_what_lies_behind_the_last_column(k):
    """Row pitch K rounded up to 4, foreign values there: they are not part of the last block."""
    from hgvae_amd import functional as Fn
    if Fn._CHECK_PADS:
        pytest.skip("such a matrix is refused under HGVAE_CHECK_PADS")
    wide = torch.randn(500, (k + 3) // 4 * 4, device=dev())
    wide[:, k:] = 1e4
    x = wide[:, :k]
    y = Fn.linear8(x, torch.randn(40, k, device=dev(), requires_grad=True))
    q, scale = (t for t in y.grad_fn.saved_tensors if t.dtype in (torch.int8, torch.uint8))
    want = Fn.pack8(x.contiguous())
    assert torch.equal(q, want.q) and torch.equal(scale, want.scale)


@pytest.mark.parametrize("n,m", [(1, 5), (700, 138), (70001, 33)])
def test_bias_gradient_beside_a_frozen_weight(n, m):
    """Only the bias (and the input) learn: nothing is packed, the bias gradient is the column sums, also in a captured pass."""
    from hgvae_amd import functional as Fn
    x, w, g = (torch.randn(*s, device=dev()) for s in ((n, 100), (m, 100), (n, m)))
    b = torch.randn(m, device=dev(), requires_grad=True)

    def step():
        y = Fn.linear8(x, w, b)
        assert len(y.grad_fn.saved_tensors) == 1
        return torch.autograd.grad(y, b, g)[0]

    # sums of n values: one rounding per partial sum, at most n / 16 of them on the longest chain of the kernel
    want = g.double().sum(0)
    bound = (n / 16 + 8) * U * g.double().abs().sum(0)
    assert bool(((step().double() - want).abs() <= bound).all())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        g.normal_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, step())


def test_guarded_arithmetic_in_a_captured_step():
    """projection "auto": the device decides launch by launch which arithmetic runs, on every replay anew."""
    from hgvae_amd import functional as Fn
    torch.manual_seed(1)
    calm = torch.randn(300, 100, device=dev()).sign() * (torch.rand(300, 100, device=dev()) + 0.5)
    wild = calm.clone()
    wild[7, 3] = 1e-9                                            # outside the range of the two fp16 pieces
    w, g = torch.randn(64, 100, device=dev(), requires_grad=True), calm[:, :64].contiguous()
    before = Fn._projection
    Fn.set_projection("auto")
    try:
        static = calm.clone()

        def step(x):
            y = Fn.linear8(x, w)
            return (y.detach(), *torch.autograd.grad(y, w, g))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(static)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(static)
        for x in (calm, wild, calm, wild, wild, calm):
            static.copy_(x)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, step(x)))
    finally:
        Fn.set_projection(before)
