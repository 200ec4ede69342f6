"""No-GPU checks of the per-graph operators: plans, refusals through Python and through the C ABI, the exported sizes."""
import ctypes

import numpy as np
import pytest
import torch


def test_segments_refuse_what_they_cannot_hold():
    from hgvae_amd import Segments, _lib
    for call in (lambda: Segments.from_sizes([3], "cpu"), lambda: Segments.from_sizes([-1, 3]), lambda: Segments.from_sizes([2 ** 31]),
                 lambda: Segments.from_sizes([2 ** 31 - 1, 2]), lambda: Segments.from_sizes([0.5]), lambda: Segments.from_sizes(np.zeros((2, 2), dtype=np.int64)),
                 lambda: Segments.from_ptr(torch.tensor([1, 2])), lambda: Segments.from_ptr(torch.tensor([0, 3, 2])), lambda: Segments.from_ptr(torch.zeros(0, dtype=torch.long)),
                 lambda: Segments.from_ptr(torch.tensor([0.0, 1.0])), lambda: Segments.from_batch(torch.tensor([1, 0])), lambda: Segments.from_batch(torch.tensor([-1, 0])),
                 lambda: Segments.from_batch(torch.tensor([0, 2]), num_graphs=2), lambda: Segments.from_batch(torch.tensor([0, 2 ** 40])), lambda: Segments.from_batch(torch.zeros(2, 2, dtype=torch.long))):
        with pytest.raises(_lib.HgvError):
            call()


def test_operators_refuse_cpu_tensors():
    from hgvae_amd import _lib
    from hgvae_amd import functional as Fn
    x, batch = torch.randn(4, 6), torch.zeros(4, dtype=torch.long)
    for call in (lambda: Fn.pack8(x), lambda: Fn.linear8(x, torch.randn(3, 6)), lambda: Fn.group_norm_act(x, batch, 2),
                 lambda: Fn.graph_attention(x.view(4, 2, 3), x.view(4, 2, 3), x.view(4, 2, 3), batch)):
        with pytest.raises(_lib.HgvError):
            call()


def test_modules_refuse_widths_that_do_not_divide():
    from hgvae_amd.nn import GraphAttention, GroupNormAct, Linear8
    for call in (lambda: GroupNormAct(10, 3), lambda: GroupNormAct(10, 0), lambda: GraphAttention(10, 3), lambda: GraphAttention(12, 4, 3), lambda: GraphAttention(12, 0)):
        with pytest.raises(ValueError):
            call()
    a = GraphAttention(138, 6, 2, keep8=True)
    assert a.lin_q.weight.shape == (138, 138) and a.lin_k.weight.shape == (46, 138) and a.lin_out.weight.shape == (138, 138)
    assert Linear8(5, 3).weight.shape == (3, 5)


def test_tiles_cover_every_row_once():
    """The plan's arrays, built on the host: row chunks, tiles of 64 rows and blocks of 64 and 128 rows."""
    from hgvae_amd.graph import Segments
    rng = np.random.default_rng(0)
    for _ in range(20):
        sizes = rng.integers(0, 700, size=rng.integers(1, 9))
        ptr = np.concatenate([[0], np.cumsum(sizes)])
        for rows in (64, 128):
            for order in (np.flatnonzero(sizes), np.argsort(sizes, kind="stable")[int((sizes == 0).sum()):][::-1]):
                t = Segments._tiles_of(sizes, ptr, order, rows)
                seen = np.zeros(int(sizes.sum()), dtype=int)
                for k, (graph, row, first, count) in enumerate(t):
                    seen[row:min(row + rows, ptr[graph + 1])] += 1
                    assert ptr[graph] <= row < ptr[graph + 1] and first <= k < first + count and count == -(-sizes[graph] // rows)
                assert (seen == 1).all()


def test_captured_backward_is_refused_while_an_older_graph_holds_the_leaves(monkeypatch):
    """The book-keeping on the CPU: streams and the capture are numbers that the test sets."""
    from hgvae_amd import _lib
    from hgvae_amd import functional as Fn
    state = {"stream": 0, "capturing": False}
    monkeypatch.setattr(_lib, "stream", lambda: state["stream"])
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: state["capturing"])

    class Twice(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x):
            ctx.leaves = Fn._leaves_of(x, None)
            return x * 2

        @staticmethod
        @Fn._first_order
        def backward(ctx, g):
            return g * 2

    w = torch.ones(3, requires_grad=True)
    count = len(Fn._leaf_streams)
    alive = Twice.apply(w)                                       # an eager graph on stream 0
    state.update(stream=7, capturing=True)
    for _ in range(2):                                           # a later graph on the capture's stream does not hide it
        with pytest.raises(_lib.HgvError, match="alive"):
            torch.autograd.grad(Twice.apply(w).sum(), w)
    assert len(Fn._leaf_streams) == count + 1
    del alive
    assert len(Fn._leaf_streams) == count
    assert torch.autograd.grad(Twice.apply(w).sum(), w)[0].tolist() == [2.0] * 3
    state.update(capturing=False)
    late = Twice.apply(w)
    state.update(stream=0)
    assert torch.autograd.grad(Twice.apply(w).sum() + late.sum(), w)[0].tolist() == [4.0] * 3
    del late
    state.update(stream=5)
    warm = Twice.apply(w)                                        # a graph of a warm-up stream may live on
    state.update(stream=7, capturing=True)
    assert torch.autograd.grad(Twice.apply(w).sum(), w)[0].tolist() == [2.0] * 3
    del warm
    assert Fn._leaves_of(torch.ones(2), w * 1) == []             # no leaf, or none that asks for a gradient


def test_c_abi_refusals_without_a_gpu():
    from hgvae_amd import _lib
    lib = _lib.load()

    def refused(code, name, *args):
        assert getattr(lib, name)(*args) == code and lib.hgv_last_error(), name

    one = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(one) + 255) // 256 * 256
    refused(-1, "hgv_pack8", None, 4, 4, 4, None, 16, None, None)
    refused(-1, "hgv_pack8", at, 4, 4, 0, at, 16, at, None)
    refused(-1, "hgv_pack8", at, 4, 4, 4, at, 20, at, None)                     # rows of q that are not multiples of 16
    refused(-1, "hgv_pack8", at, 4, 4, 4, at, 48, at, None)                     # behind the last block
    refused(-1, "hgv_unpack8", at, 16, at, 4, 5, at, 4, None)
    refused(-1, "hgv_gemm_tn8", at, 8, 8, at, 16, at, 0, 4, at, 8, None, at, 4096, None)
    refused(-1, "hgv_gemm_tn8", at, 6, 6, at, 16, at, 8, 4, at, 8, None, at, 4096, None)
    refused(-4, "hgv_gemm_tn8", at, 8, 8, at, 16, at, 8, 4, at, 8, None, at, 16, None)
    norm = lambda c, groups, small, rows, ws: (at, 16, c, groups, 0, 1e-5, None, None, at, at, at, at, 2, 2, small, rows, 0, 4, at, 16, at, at, at, ws, None)
    refused(-1, "hgv_group_norm_fwd", *norm(10, 3, 0, 0, 4096))
    refused(-1, "hgv_group_norm_fwd", *norm(12, 3, 3, 4, 4096))                 # more small graphs than graphs
    refused(-1, "hgv_group_norm_fwd", *norm(12, 3, 1, 10 ** 6, 4096))           # a small graph that does not fit
    refused(-4, "hgv_group_norm_fwd", *norm(12, 3, 0, 0, 16))
    att = lambda h, hk, d, scale, ws: (at, 8, 8, at, 8, 8, at, 8, 8, 4, 1, h, hk, d, scale, None, at, 4, at, 1, at, 1, 1, at, None, at, ws, None)
    refused(-1, "hgv_graph_attention_fwd", *att(3, 2, 8, 1.0, 4096))
    refused(-2, "hgv_graph_attention_fwd", *att(2, 2, 129, 1.0, 4096))
    refused(-1, "hgv_graph_attention_fwd", *att(2, 2, 8, 0.0, 4096))
    refused(-1, "hgv_graph_attention_fwd", *att(2, 2, 8, float("nan"), 4096))
    refused(-4, "hgv_graph_attention_fwd", *att(2, 2, 8, 1.0, 16))
    assert lib.hgv_group_norm_small_rows(10, 3) == 0 and lib.hgv_group_norm_small_rows(138, 6) > 0
    assert lib.hgv_graph_attention_ws(0, 1, 1, 1, 8, 1, 0) == 0 and lib.hgv_graph_attention_ws(100, 1, 2, 1, 8, 2, 1) > lib.hgv_graph_attention_ws(100, 1, 2, 1, 8, 2, 0) > 0


def test_header_and_bindings_agree_on_the_number_of_arguments():
    import os
    import re
    from hgvae_amd import _lib
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    with open(os.path.join(root, "include", "hgvae_hip.h")) as f:
        text = re.sub(r"/\*.*?\*/", "", f.read(), flags=re.S)
    for name, (_, args) in _lib.SIGNATURES.items():
        found = re.search(rf"\b{name}\s*\(([^)]*)\)", text)
        assert found, name
        params = found.group(1).strip()
        assert (0 if params in ("", "void") else params.count(",") + 1) == len(args), name


def test_c_abi_refusals_of_the_packing_forms():
    from hgvae_amd import _lib
    lib = _lib.load()
    room = ctypes.create_string_buffer(8192)
    at = (ctypes.addressof(room) + 255) // 256 * 256

    def norm(q, ldq, scale, rows=16):
        return lib.hgv_group_norm_fwd8(at, 16, 12, 3, 0, 1e-5, None, None, at, at, at, at, 2, 2, 0, 0, 0, 4, rows, q, ldq, scale, at, 16, at, at,
                                       at, 16, None)

    for bad in ((None, 16, at), (at, 16, None), (at, 12, at), (at, 48, at), (at + 4, 16, at)):
        assert norm(*bad) == -1 and b"fwd8" in lib.hgv_last_error()
    assert norm(at, 16, at, rows=0) == -1
    assert norm(at, 16, at) == -4                                # ... and a good form reaches the check of the workspace

    def product(q, ldq, scale, lda=100):
        return lib.hgv_gemm_nt16h_keep8(at, lda, 100, at, None, 4, 40, at, 40, q, ldq, scale, None)

    for bad in ((None, 112, at), (at, 112, None), (at, 100, at), (at, 144, at), (at + 8, 112, at)):
        assert product(*bad) == -1 and b"keep8" in lib.hgv_last_error()
    assert product(at, 112, at, lda=98) == -1 and b"source 1" in lib.hgv_last_error()
