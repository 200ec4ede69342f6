"""The per-graph operators together, as levels of a deeper encoder use them: norm and activation, projection, attention, residual."""
import gc
import math

import pytest
import torch
from torch import nn

from test_gpu_group_norm import values8

pytestmark = pytest.mark.gpu

FWD_RTOL, BWD_RTOL = 1e-5, 1e-4          # norm-wise, the tolerances of the other operators of the package


def dev():
    return torch.device("cuda:0")


class Level(nn.Module):
    """x + attention(linear(act(norm(x))))"""

    def __init__(self, channels, groups, heads, kv_heads, keep8):
        super().__init__()
        from hgvae_amd.nn import GraphAttention, GroupNormAct, Linear8
        self.norm = GroupNormAct(channels, groups, "silu", keep8=keep8)
        self.lin = Linear8(channels, channels) if keep8 else nn.Linear(channels, channels)
        self.att = GraphAttention(channels, heads, kv_heads, head_dim=channels // heads, keep8=keep8)
        self.keep8 = keep8

    def forward(self, x, segments, mask=None):
        from hgvae_amd import functional as Fn
        h = self.norm(x, segments)
        h = self.lin(h) if self.keep8 else Fn.dual_linear(h, self.lin.weight, bias=self.lin.bias)
        return x + self.att(h, segments, mask)


def reference(level, x, sizes, mask):
    """The same level in float64 torch operations on parameters given by name."""
    p = {k: v for k, v in level.items()}
    n, c = x.shape
    heads, kv, groups = p["heads"], p["kv"], p["groups"]
    out, at = [], 0
    for s in sizes:
        r = slice(at, at + s)
        at += s
        if s == 0:
            continue
        g = x[r].reshape(s, groups, c // groups)
        mean = g.mean((0, 2), keepdim=True)
        xh = (g - mean) / torch.sqrt(((g - mean) ** 2).mean((0, 2), keepdim=True) + 1e-5)
        z = xh.reshape(s, c) * p["norm.weight"] + p["norm.bias"]
        h = (z * torch.sigmoid(z)) @ p["lin.weight"].t() + p["lin.bias"]
        q, k, v = ((h @ p[f"att.lin_{t}.weight"].t()).unflatten(1, (-1, c // heads)).transpose(0, 1) for t in "qkv")
        k, v = (t.repeat_interleave(heads // kv, 0) for t in (k, v))
        a = q @ k.transpose(1, 2) / math.sqrt(c // heads)
        if mask is not None:
            a = a.masked_fill(~mask[r], -math.inf)
        o = (torch.softmax(a, -1) @ v).transpose(0, 1).reshape(s, c)
        out.append(x[r] + o @ p["att.lin_out.weight"].t() + p["att.lin_out.bias"])
    return torch.cat(out)


@pytest.mark.parametrize("sizes,c,groups,heads,kv", [([138, 1, 60], 138, 6, 6, 2), ([40, 0, 300], 64, 8, 4, 4), ([2], 96, 1, 1, 1)])
@pytest.mark.parametrize("masked", [False, True])
def test_two_levels_match_float64(sizes, c, groups, heads, kv, masked):
    from hgvae_amd import Segments
    torch.manual_seed(c)
    n = sum(sizes)
    levels = [Level(c, groups, heads, kv, False).to(dev()) for _ in range(2)]
    x = torch.randn(n, c, device=dev())
    g = torch.randn(n, c, device=dev())
    mask = None
    if masked:
        mask = torch.rand(n, device=dev()) < 0.7
        at = 0
        for s in sizes:
            if s:
                mask[at] = True                                 # the dense softmax of the reference has no empty rows
            at += s
    seg = Segments.from_sizes(sizes, dev())
    xr = x.clone().requires_grad_()
    out = levels[1](levels[0](xr, seg, mask), seg, mask)
    out.backward(g)
    x64 = x.double().cpu().requires_grad_()
    params = []
    h = x64
    for level in levels:
        p = {k: v.detach().double().cpu().requires_grad_() for k, v in level.named_parameters()}
        params.append(p)
        h = reference({**p, "heads": heads, "kv": kv, "groups": groups}, h, sizes, None if mask is None else mask.cpu())
    h.backward(g.double().cpu())

    def close(a, b, rtol, what):
        a, b = a.detach().double().cpu(), b.detach()
        assert (a - b).abs().max() <= rtol * b.abs().max() + 1e-6, what

    close(out, h, FWD_RTOL, "out")
    close(xr.grad, x64.grad, BWD_RTOL, "x")
    for level, p in zip(levels, params):
        for name, q in level.named_parameters():
            close(q.grad, p[name].grad, BWD_RTOL, name)


def test_8bit_level_is_the_sum_of_its_parts():
    """Autograd through a level whose inputs are kept in 8 bits, against its operators called one by one with the gradients
    handed on by hand.  The forward result is that of the level which keeps everything."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    sizes, c = [70, 300], 64
    torch.manual_seed(3)
    level = Level(c, 8, 4, 2, True).to(dev())
    seg = Segments.from_sizes(sizes, dev())
    x, g = torch.randn(370, c, device=dev()), torch.randn(370, c, device=dev())
    xr = x.clone().requires_grad_()
    out = level(xr, seg)
    out.backward(g)
    full = Level(c, 8, 4, 2, False).to(dev())
    full.load_state_dict(level.state_dict())
    assert torch.equal(full(x, seg), out)

    def leaf(t):
        return t.detach().requires_grad_()

    a = level.att
    x0 = leaf(x)
    h0 = Fn.group_norm_act(x0, seg, 8, level.norm.weight, level.norm.bias, keep8=True)
    x1 = leaf(h0)
    h1 = Fn.linear8(x1, level.lin.weight, level.lin.bias)
    x2 = leaf(h1)
    qkv = [Fn.linear8(x2, lin.weight) for lin in (a.lin_q, a.lin_k, a.lin_v)]
    q, k, v = (leaf(t.unflatten(1, (-1, 16))) for t in qkv)
    o = Fn.graph_attention(q, k, v, seg)
    x3 = leaf(o.reshape(370, c))
    y = Fn.linear8(x3, a.lin_out.weight, a.lin_out.bias)
    grads = {}
    g3, grads["att.lin_out.weight"], grads["att.lin_out.bias"] = torch.autograd.grad(y, (x3, a.lin_out.weight, a.lin_out.bias), g)
    gq = torch.autograd.grad(o, (q, k, v), g3.view(370, 4, 16))
    parts = [torch.autograd.grad(t, (x2, lin.weight), gt.reshape(370, -1)) for t, lin, gt in zip(qkv, (a.lin_q, a.lin_k, a.lin_v), gq)]
    for name, (_, gw) in zip("qkv", parts):
        grads[f"att.lin_{name}.weight"] = gw
    g1, grads["lin.weight"], grads["lin.bias"] = torch.autograd.grad(h1, (x1, level.lin.weight, level.lin.bias), parts[2][0] + parts[1][0] + parts[0][0])
    g0, grads["norm.weight"], grads["norm.bias"] = torch.autograd.grad(h0, (x0, level.norm.weight, level.norm.bias), g1)
    for name, p in level.named_parameters():
        # autograd may add the three gradients of h in another order: one rounding of each of two sums
        bound = 0.0 if name.startswith("att") else 1e-5 * float(grads[name].abs().max())
        assert float((p.grad - grads[name]).abs().max()) <= bound, name
    assert float((xr.grad - (g0 + g)).abs().max()) <= 1e-5 * float(g0.abs().max())


def test_8bit_weight_gradient_is_within_half_a_step():
    from hgvae_amd import functional as Fn
    gen = torch.Generator(device=dev()).manual_seed(5)
    x, w, g = (torch.randn(*s, generator=gen, device=dev()) for s in ((900, 138), (40, 138), (900, 40)))
    wr = w.clone().requires_grad_()
    (g8,) = torch.autograd.grad(Fn.linear8(x, wr), (wr,), g)
    exact = g.double().t() @ x.double()
    off = (values8(x) - x.double()).abs()
    bound = g.double().abs().t() @ off
    assert bool(((g8.double() - exact).abs() <= bound + 1e-4 * exact.abs().max()).all())
    assert float((g8.double() - exact).norm() / exact.norm()) < 0.01        # steps of 1/63 at most, errors of both signs


def test_captured_training_step_replays_as_eager():
    """Forward and backward of an 8-bit level replayed from one HIP graph, eager steps between the replays.  While an eager
    graph of the same leaves lives, the captured backward pass is refused with an error; once it is gone the capture works."""
    from hgvae_amd import Segments
    from hgvae_amd._lib import HgvError
    sizes, c = [138, 90], 64
    torch.manual_seed(6)
    level = Level(c, 8, 4, 4, True).to(dev())
    seg = Segments.from_sizes(sizes, dev())
    data = [torch.randn(228, c, device=dev()) for _ in range(2)]
    g = torch.randn(228, c, device=dev())
    params = list(level.parameters())
    static = data[0].clone()

    def step(x):
        out = level(x, seg)
        return (out.detach(), *torch.autograd.grad(out, params, g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    alive = level(data[1], seg)                                  # an eager graph over the same leaves
    with pytest.raises(HgvError, match="alive"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            step(static)
    torch.autograd.grad(alive, params, g)                        # the eager graph itself is as good as before
    del alive
    gc.collect()                                                 # what the refused call left
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i in (0, 1, 0, 1):
        static.copy_(data[i])
        graph.replay()
        torch.cuda.synchronize()
        want = step(data[i])
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_modules_repr_and_second_derivatives_are_refused():
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    from hgvae_amd.nn import GraphAttention, GroupNormAct
    assert "groups=3" in repr(GroupNormAct(12, 3)) and "heads=4" in repr(GraphAttention(64, 4, 2))
    seg = Segments.from_sizes([5, 4], dev())
    x = torch.randn(9, 12, device=dev(), requires_grad=True)
    w = torch.randn(12, 12, device=dev(), requires_grad=True)
    q = torch.randn(9, 2, 6, device=dev(), requires_grad=True)
    for out, leaf in ((Fn.group_norm_act(x, seg, 3), x), (Fn.linear8(x, w), x), (Fn.graph_attention(q, q, q, seg), q)):
        (first,) = torch.autograd.grad((out ** 2).sum(), (leaf,), create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), (leaf,))


def test_evaluation_keeps_nothing(monkeypatch):
    """Under no_grad a module's parameters still ask for gradients: no 8-bit forms, statistics or leaves are kept for them."""
    from hgvae_amd import Segments, _lib
    from hgvae_amd import functional as Fn
    level = Level(64, 8, 4, 2, True).to(dev())
    seg = Segments.from_sizes([1500, 300], dev())
    x = torch.randn(1800, 64, device=dev())
    want = level(x, seg).detach()
    names, real = [], _lib.call
    count = len(Fn._leaf_streams)
    monkeypatch.setattr(_lib, "call", lambda name, *args: (names.append(name), real(name, *args))[1])
    with torch.no_grad():
        got = level(x, seg)
    assert torch.equal(got, want) and not [n for n in names if n.endswith("8") or n == "hgv_pack8"]
    assert len(Fn._leaf_streams) == count
    names.clear()
    level(x, seg)
    assert "hgv_group_norm_fwd8" in names and ("hgv_gemm_nt16h_keep8" in names or "hgv_pack8" in names)


def test_plan_dropped_while_another_stream_reads_it():
    """A plan used on a second stream and dropped at once: its memory is not handed out before that stream is done."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    n = 300 * 700
    x = torch.randn(n, 64, device=dev())
    want = Fn.group_norm_act(x, Segments.from_sizes([300] * 700, dev()), 8)
    side = torch.cuda.Stream()
    for _ in range(5):
        seg = Segments.from_sizes([300] * 700, dev())
        size = seg._buf.numel()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(8):
                got = Fn.group_norm_act(x, seg, 8)
        del seg
        torch.zeros(size, dtype=torch.int32, device=dev())        # would land in the plan's memory, on the first stream
        torch.cuda.synchronize()
        assert torch.equal(got, want)


def test_copies_of_a_plan_have_arrays_of_their_own():
    import copy
    import pickle
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    x = torch.randn(430, 24, device=dev())
    seg = Segments.from_sizes([400, 0, 30], dev())
    want = Fn.group_norm_act(x, seg, 3), Fn.graph_attention(*(x.view(430, 3, 8),) * 3, seg)
    for other in (copy.deepcopy(seg), copy.copy(seg), pickle.loads(pickle.dumps(seg))):
        assert other.sizes == seg.sizes and other.device == seg.device and other._ptr.data_ptr() != seg._ptr.data_ptr()
        assert other._attention_plan[0] == other._ptr.data_ptr()
        got = Fn.group_norm_act(x, other, 3), Fn.graph_attention(*(x.view(430, 3, 8),) * 3, other)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_empty_batches_through_the_modules():
    from hgvae_amd import Segments
    level = Level(24, 3, 4, 2, True).to(dev())
    for sizes in ([], [0, 0]):
        x = torch.zeros(0, 24, device=dev(), requires_grad=True)
        out = level(x, Segments.from_sizes(sizes, dev()))
        assert out.shape == (0, 24)
        out.sum().backward()
        assert x.grad.shape == (0, 24) and all(not bool(p.grad.any()) for p in level.parameters())
        level.zero_grad()


def test_plans_are_made_before_a_capture():
    """A batch vector or a new plan inside a capture is an error that leaves the capture usable."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    from hgvae_amd._lib import HgvError
    x = torch.randn(50, 12, device=dev())
    batch = torch.zeros(50, dtype=torch.long, device=dev())
    seg = Segments.from_sizes([50], dev())
    want = Fn.group_norm_act(x, seg, 3)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in (lambda: Fn.group_norm_act(x, batch, 3), lambda: Segments.from_sizes([50], dev()), lambda: Segments.from_ptr(batch[:1])):
            with pytest.raises(HgvError, match="before the capture"):
                call()
        out = Fn.group_norm_act(x, seg, 3)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want)


@pytest.mark.parametrize("op", ["norm", "linear8", "attention"])
def test_offsets_beyond_32_bits(op):
    """Matrices of more than 2^31 elements: the last graph's rows give what they give by themselves (to rounding: the order of sums
    follows the plan)."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    rows, last = 16_000_000, 1000
    if op == "norm":
        x, g = torch.randn(rows, 140, device=dev()), torch.randn(last, 140, device=dev())
        assert x.numel() > 2 ** 31
        w = torch.randn(140, device=dev(), requires_grad=True)
        seg = Segments.from_sizes([8000] * ((rows - last) // 8000) + [(rows - last) % 8000, last], dev())
        xr = x.requires_grad_()
        out = Fn.group_norm_act(xr, seg, 7, w, keep8=True)
        tail = out[-last:].detach().clone()
        full = torch.zeros_like(out)
        full[-last:] = g
        gx, gw = torch.autograd.grad(out, (xr, w), full)
        small = x.detach()[-last:].clone().requires_grad_()
        ref = Fn.group_norm_act(small, Segments.from_sizes([last], dev()), 7, w, keep8=True)
        rx, rw = torch.autograd.grad(ref, (small, w), g)
        pairs = ((tail, ref), (gx[-last:], rx), (gw, rw))
    elif op == "linear8":
        x = torch.randn(rows, 140, device=dev())
        w = torch.randn(24, 140, device=dev(), requires_grad=True)
        xr = x.requires_grad_()
        out = Fn.linear8(xr, w)
        tail = out[-last:].detach().clone()
        full = torch.zeros_like(out)
        full[-last:] = 1.0
        gx, gw = torch.autograd.grad(out, (xr, w), full)
        small = x.detach()[-last:].clone().requires_grad_()
        ref = Fn.linear8(small, w)
        rx, rw = torch.autograd.grad(ref, (small, w), torch.ones_like(ref))
        pairs = ((tail, ref), (gx[-last:], rx), (gw, rw))
    else:
        rows, h, d = 9_000_000, 4, 64
        q = torch.randn(rows, h, d, device=dev()).requires_grad_()
        assert q.numel() > 2 ** 31
        k, v = (torch.randn(rows, h, d, device=dev()).requires_grad_() for _ in range(2))
        seg = Segments.from_sizes([100] * ((rows - last) // 100) + [last], dev())
        out = Fn.graph_attention(q, k, v, seg)
        tail = out[-last:].detach().clone()
        g = torch.randn(last, h, d, device=dev())
        full = torch.zeros_like(out)
        full[-last:] = g
        grads = torch.autograd.grad(out, (q, k, v), full)
        small = [t.detach()[-last:].clone().requires_grad_() for t in (q, k, v)]
        ref = Fn.graph_attention(*small, Segments.from_sizes([last], dev()))
        refs = torch.autograd.grad(ref, small, g)
        pairs = ((tail, ref), *((a[-last:], b) for a, b in zip(grads, refs)))
    for a, b in pairs:
        b = b.detach()
        assert float((a.detach() - b).abs().max()) <= 1e-5 * float(b.abs().max())
    torch.cuda.empty_cache()


def test_capture_after_a_warm_up_whose_results_live_on():
    """The usual recipe: warm up on a side stream, keep the last loss, capture, replay."""
    from hgvae_amd import Segments
    torch.manual_seed(8)
    level = Level(64, 8, 4, 2, False).to(dev())
    seg = Segments.from_sizes([100, 40], dev())
    static = torch.randn(140, 64, device=dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            level.zero_grad(set_to_none=True)
            loss = (level(static, seg) ** 2).mean()
            loss.backward()
    torch.cuda.current_stream().wait_stream(side)
    level.zero_grad(set_to_none=True)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = (level(static, seg) ** 2).mean()
        out.backward()
    del loss
    got = {n: p.grad for n, p in level.named_parameters()}
    for _ in range(3):
        static.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = torch.autograd.grad((level(static, seg) ** 2).mean(), list(level.parameters()))
        for (n, g), w in zip(got.items(), want):
            assert float((g - w).abs().max()) <= 1e-6 * float(w.abs().max()), n
