"""nn.GraphAttention with keep8: its three projections of one input keep one 8-bit form of it."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def dev():
    return torch.device("cuda:0")


def kept(out):
    """8-bit matrices that the graph behind ``out`` holds: {address: (rows, columns, bytes)}."""
    found, todo, seen = {}, [out.grad_fn], set()
    while todo:
        node = todo.pop()
        if node is None or node in seen:
            continue
        seen.add(node)
        for t in getattr(node, "saved_tensors", ()):
            if t is not None and t.dtype in (torch.int8, torch.uint8):
                found[t.data_ptr()] = t.numel()
        todo += [n for n, _ in node.next_functions]
    return found


@pytest.mark.parametrize("c,heads,kv", [(64, 4, 2), (138, 6, 2)])
def test_the_input_is_kept_once(c, heads, kv):
    from hgvae_amd import Segments
    from hgvae_amd.nn import GraphAttention
    sizes = [300, 1, 900]
    n = sum(sizes)
    torch.manual_seed(c)
    att = GraphAttention(c, heads, kv, keep8=True).to(dev())
    x = torch.randn(n, c, device=dev(), requires_grad=True)
    out = att(x, Segments.from_sizes(sizes, dev()))
    # the input, and the attention's output in front of the last projection: 1 byte per element in rows of whole 16 columns, and a byte per block
    row = (c + 15) // 16 * 16 + (c + 31) // 32
    assert sum(kept(out).values()) == 2 * n * row


@pytest.mark.parametrize("c,heads,kv,frozen", [(64, 4, 2, ""), (138, 6, 2, ""), (138, 6, 6, "q"), (30, 5, 1, "qkv"), (64, 4, 4, "x")])
def test_gradients_are_those_of_three_projections(c, heads, kv, frozen):
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    from hgvae_amd.nn import GraphAttention
    sizes = [70, 0, 300, 3]
    n = sum(sizes)
    torch.manual_seed(c + kv)
    att = GraphAttention(c, heads, kv, keep8=True).to(dev())
    x, g = torch.randn(n, c, device=dev()), torch.randn(n, c, device=dev())
    lins = {"q": att.lin_q, "k": att.lin_k, "v": att.lin_v}
    for name in frozen.replace("x", ""):
        lins[name].weight.requires_grad_(False)
    seg = Segments.from_sizes(sizes, dev())

    def grads(out, xr):
        leaves = [p for p in (xr, *att.parameters()) if p.requires_grad]
        return torch.autograd.grad(out, leaves, g)

    xr = x.clone().requires_grad_("x" not in frozen)
    out = att(xr, seg)
    got = grads(out, xr)
    xs = x.clone().requires_grad_("x" not in frozen)
    q, k, v = (Fn.linear8(xs, lin.weight).unflatten(1, (-1, att.head_dim)) for lin in lins.values())
    one = Fn.linear8(Fn.graph_attention(q, k, v, seg).reshape(n, -1), att.lin_out.weight, att.lin_out.bias)
    want = grads(one, xs)
    assert torch.equal(out, one)
    if "x" not in frozen:                                       # a sum of three, in this order or another: two roundings
        assert bool(((got[0] - want[0]).abs() <= 2 * 2.0 ** -23 * want[0].abs().max()).all())
        got, want = got[1:], want[1:]
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    with torch.no_grad():
        assert torch.equal(att(x, seg), out) and not kept(out.detach() * out.new_ones(1).requires_grad_())


def test_captured_and_a_part_without_a_gradient():
    """Replays of a captured pass; and a value projection whose result is not used, so its gradient is zero."""
    from hgvae_amd import Segments
    from hgvae_amd import functional as Fn
    from hgvae_amd.nn import GraphAttention
    torch.manual_seed(1)
    att = GraphAttention(138, 6, 2, keep8=True).to(dev())
    seg = Segments.from_sizes([138] * 4, dev())
    static, g = torch.randn(552, 138, device=dev()), torch.randn(552, 138, device=dev())

    def step(x):
        leaf = x.detach().requires_grad_()
        out = att(leaf, seg)
        return (out.detach(), *torch.autograd.grad(out, (leaf, *att.parameters()), g))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(static)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(static)
    for i in range(4):
        static.copy_(torch.randn(552, 138, device=dev(), generator=torch.Generator(device=dev()).manual_seed(i)))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, step(static)))
    x = static.clone().requires_grad_()
    q, k, v = Fn._linear8_each(x, [lin.weight for lin in (att.lin_q, att.lin_k, att.lin_v)])
    gx, gq, gv = torch.autograd.grad((q * 2.0).sum() + k.sum(), (x, att.lin_q.weight, att.lin_v.weight))
    want = torch.autograd.grad((Fn.linear8(x, att.lin_q.weight) * 2.0).sum() + Fn.linear8(x, att.lin_k.weight).sum(), (x, att.lin_q.weight))
    assert torch.equal(gq, want[1]) and not bool(gv.any())
    assert bool(((gx - want[0]).abs() <= 2.0 ** -23 * want[0].abs().max()).all())
