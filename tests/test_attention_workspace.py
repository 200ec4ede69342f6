"""Workspace of the attention's forward pass: no images of the operands where no graph is large."""
import ctypes


def test_small_graphs_need_next_to_none():
    from hgvae_amd import _lib
    lib = _lib.load()
    sizes = (500000, 2000, 4, 4, 64, 8000)
    images = lib.hgv_graph_attention_ws(*sizes, 0)
    assert images > 3 * 500000 * 4 * 64 * 4
    assert 0 < lib.hgv_graph_attention_fwd_ws(*sizes, 512) <= 4096
    assert lib.hgv_graph_attention_fwd_ws(*sizes, 513) == images
    assert lib.hgv_graph_attention_fwd_ws(0, 1, 1, 1, 8, 1, 8) == 0


def test_the_entry_point_asks_for_what_it_uses():
    from hgvae_amd import _lib
    lib = _lib.load()
    room = ctypes.create_string_buffer(4096)
    at = (ctypes.addressof(room) + 255) // 256 * 256

    def forward(max_rows, ws, ws_bytes):                        # 4 rows, out not there: the check behind that of the workspace
        return lib.hgv_graph_attention_fwd(at, 8, 8, at, 8, 8, at, 8, 8, 4, 1, 2, 2, 8, 1.0, None, at, max_rows, at, 1, at, 1, 1, None, None, ws,
                                           ws_bytes, None)

    assert forward(4, at, 255) == -4 and forward(4, at + 8, 256) == -4 and forward(513, at, 256) == -4
    assert forward(4, at, 256) == -1 and b"buffer" in lib.hgv_last_error()
