"""Device-resident graph structure (CSR by target, CSR by source) built once per batch.

PyG operators take a COO ``edge_index`` on every call (reference call sites
gvae/gvae_skipcon.py:105-118).  Here the first operator that sees an
``edge_index`` tensor builds a :class:`Graph` with the radix-sort kernel and every
later layer, both encode passes and the backward pass reuse it.
"""
from __future__ import annotations

import bisect
import weakref
from typing import Optional, Sequence

import numpy as np
import torch

from . import _lib


def pad4(n: int) -> int:
    return (n + 3) // 4 * 4


def new_padded(rows: int, cols: int, device, zero_pad: bool = True) -> torch.Tensor:
    """[rows, cols] fp32 view of a buffer whose rows are padded to a multiple of 4 floats."""
    ld = pad4(cols)
    buf = torch.empty(rows, ld, dtype=torch.float32, device=device)
    if zero_pad and ld != cols:
        buf[:, cols:].zero_()
    return buf.as_strided((rows, cols), (ld, 1))                # buf[:, :cols] in half the time


def ld_of(t: torch.Tensor) -> int:
    """Leading dimension (elements per row) of a 2-D tensor whose rows are unit-stride."""
    sh, st = t.shape, t.stride()
    if len(sh) != 2 or (sh[1] > 1 and st[1] != 1):
        raise _lib.HgvError(f"expected a row-major 2-D tensor, got shape {tuple(sh)} strides {st}")
    return st[0] if sh[0] > 1 else max(st[0], sh[1])


def rowmajor(t: torch.Tensor) -> torch.Tensor:
    """Return t if its rows are unit-stride with ld >= cols, else a padded copy."""
    if t.dim() == 2 and t.dtype == torch.float32 and (t.size(1) <= 1 or t.stride(1) == 1) \
            and (t.size(0) <= 1 or t.stride(0) >= t.size(1)):
        return t
    out = new_padded(t.size(0), t.size(1), t.device)
    out.copy_(t)
    return out


def is_vec4(t: torch.Tensor) -> bool:
    ld = ld_of(t)
    return t.data_ptr() % 16 == 0 and ld % 4 == 0 and ld >= pad4(t.size(1))


def as_padded(t: torch.Tensor) -> torch.Tensor:
    """Row-major fp32 tensor laid out for the 16-byte kernel paths (copy only if needed)."""
    t = rowmajor(t)
    if is_vec4(t):
        return t
    out = new_padded(t.size(0), t.size(1), t.device)
    out.copy_(t)
    return out


class _LongRows:
    """Rows of a CSR that are far longer than the average (hubs), listed on the device once per CSR.  Whether there
    are any reaches the host through an asynchronous copy; until it has arrived the answer is "maybe"."""
    __slots__ = ("threshold", "rows", "count", "cap", "_host", "_event", "_known")

    def __init__(self, rowptr: torch.Tensor, n_rows: int, n_entries: int):
        dev = rowptr.device
        self.threshold = max(64, 4 * -(-n_entries // max(n_rows, 1)))
        self.cap = n_entries // self.threshold + 1
        self.rows = torch.empty(self.cap, dtype=torch.int32, device=dev)
        self.count = torch.zeros(1, dtype=torch.int32, device=dev)
        _lib.call("hgv_csr_long_rows", rowptr.data_ptr(), n_rows, self.threshold, self.rows.data_ptr(), self.cap,
                  self.count.data_ptr(), _lib.stream())
        self._known: Optional[int] = None
        self._host = self._event = None
        if not torch.cuda.is_current_stream_capturing():      # a capture must not hold host copies or foreign events
            self._host = torch.empty(1, dtype=torch.int32, pin_memory=True)
            self._host.copy_(self.count, non_blocking=True)
            self._event = torch.cuda.Event()
            self._event.record()

    def maybe_any(self) -> bool:
        """False only once the device has reported an empty list (never blocks)."""
        if self._known is None and self._event is not None and self._event.query():
            self._known = int(self._host[0])
        return self._known is None or self._known > 0


class _Csr:
    __slots__ = ("rowptr", "col", "perm", "_long")

    def __init__(self, rowptr, col, perm):
        self.rowptr, self.col, self.perm = rowptr, col, perm
        self._long = None

    def long_rows(self, n_rows: int) -> _LongRows:
        if self._long is None:
            self._long = _LongRows(self.rowptr, n_rows, int(self.col.numel()))
        return self._long


def _build_csr(edge_index: torch.Tensor, n: int, by_src: bool, status: torch.Tensor) -> _Csr:
    e = edge_index.size(1)
    dev = edge_index.device
    rowptr = torch.empty(n + 1, dtype=torch.int32, device=dev)
    col = torch.empty(e, dtype=torch.int32, device=dev)
    perm = torch.empty(e, dtype=torch.int32, device=dev)
    lib = _lib.load()
    ws_bytes = lib.hgv_csr_build_ws(e, n)
    ws = torch.empty(max(ws_bytes, 256), dtype=torch.uint8, device=dev)
    _lib.call("hgv_csr_build", edge_index.data_ptr(), edge_index.stride(0), edge_index.stride(1), e, n,
              1 if by_src else 0, rowptr.data_ptr(), col.data_ptr(), perm.data_ptr(), status.data_ptr(),
              ws.data_ptr(), ws.numel(), _lib.stream())
    return _Csr(rowptr, col, perm)


class Graph:
    """CSR views of one (batched) graph with ``num_nodes`` nodes.

    ``by_dst``: row i lists the sources of the edges into i, in stable edge order
    (forward aggregation).  ``by_src``: row j lists the targets of the edges out of
    j (backward aggregation); built on first use.
    """

    def __init__(self, edge_index: torch.Tensor, num_nodes: int, hold: bool = True):
        _lib.require_cuda(edge_index)
        if edge_index.dim() != 2 or edge_index.size(0) != 2 or edge_index.dtype != torch.int64:
            raise _lib.HgvError(f"edge_index must be int64 [2, E], got {edge_index.dtype} {tuple(edge_index.shape)}")
        self.num_nodes = int(num_nodes)
        self.num_edges = int(edge_index.size(1))
        # graph_of() keys its cache by the caller's tensor and passes hold=False: a strong
        # reference from the cached Graph would keep that cache entry alive forever.
        self._ei_ref = weakref.ref(edge_index)
        self._ei_hold = edge_index if hold else None
        self.status = torch.zeros(1, dtype=torch.int32, device=edge_index.device)
        self.by_dst = _build_csr(edge_index, self.num_nodes, False, self.status)
        self._by_src: Optional[_Csr] = None
        self._inv_deg = None
        self._loops: Optional["Graph"] = None
        self._t2f = None

    @classmethod
    def from_parts(cls, edge_index: torch.Tensor, num_nodes: int, by_dst: _Csr, by_src: Optional[_Csr]) -> "Graph":
        """Graph around CSR arrays that already exist (e.g. assembled from a packed shard): nothing is sorted."""
        g = cls.__new__(cls)
        g.num_nodes, g.num_edges = int(num_nodes), int(edge_index.size(1))
        g._ei_ref, g._ei_hold = weakref.ref(edge_index), edge_index
        g.status = torch.zeros(1, dtype=torch.int32, device=edge_index.device)
        g.by_dst, g._by_src = by_dst, by_src
        g._inv_deg = g._loops = g._t2f = None
        return g

    @property
    def edge_index(self) -> torch.Tensor:
        ei = self._ei_ref()
        if ei is None:
            raise _lib.HgvError("the edge_index tensor this Graph was built from no longer exists")
        return ei

    @property
    def by_src(self) -> _Csr:
        if self._by_src is None:
            self._by_src = _build_csr(self.edge_index, self.num_nodes, True, self.status)
        return self._by_src

    @property
    def in_degree(self) -> torch.Tensor:
        rp = self.by_dst.rowptr
        return rp[1:] - rp[:-1]

    @property
    def inv_deg(self) -> torch.Tensor:
        """1 / max(in-degree, 1) as fp32 [N]."""
        if self._inv_deg is None:
            self._inv_deg = self.in_degree.clamp(min=1).to(torch.float32).reciprocal()
        return self._inv_deg

    @property
    def gcn_dis(self) -> torch.Tensor:
        """in-degree^-1/2 as fp32 [N] (0 for isolated targets): GCNConv's symmetric normalisation, meant for the
        loop-augmented graph where every degree is >= 1."""
        if getattr(self, "_gcn_dis", None) is None:
            d = self.in_degree.to(torch.float32).pow(-0.5)
            self._gcn_dis = torch.where(torch.isinf(d), torch.zeros_like(d), d)
        return self._gcn_dis

    @property
    def src_pos_to_dst_pos(self) -> torch.Tensor:
        """For each position of the by-source CSR, the position of the same edge in the by-target CSR."""
        if self._t2f is None:
            inv = torch.empty(self.num_edges, dtype=torch.int64, device=self.by_dst.perm.device)
            inv[self.by_dst.perm.long()] = torch.arange(self.num_edges, device=inv.device)
            self._t2f = inv[self.by_src.perm.long()]
        return self._t2f

    def with_self_loops(self) -> "Graph":
        """Graph of (edges minus existing self loops) followed by one loop per node.

        This is the edge list GATConv (remove_self_loops + add_self_loops) and GCNConv
        (add_remaining_self_loops, unweighted) aggregate over.
        """
        if self._loops is None:
            ei = self.edge_index
            keep = ei[0] != ei[1]
            if not bool(keep.all()):
                ei = ei[:, keep]
            loop = torch.arange(self.num_nodes, dtype=torch.int64, device=ei.device)
            self._loops = Graph(torch.cat([ei, loop.unsqueeze(0).expand(2, -1)], dim=1).contiguous(), self.num_nodes,
                                hold=True)
        return self._loops

    def check(self) -> None:
        """Synchronising validity check: raises if an index was outside [0, num_nodes)."""
        if int(self.status.item()) != 0:
            raise _lib.HgvError("edge_index holds node indices outside [0, num_nodes)")


# edge_index tensor object -> Graph, dropped when the tensor dies
_cache: "dict[int, tuple]" = {}


def graph_of(edge_index, num_nodes: Optional[int] = None) -> Graph:
    """Graph for an ``edge_index`` tensor (cached per tensor object and version) or pass-through."""
    if isinstance(edge_index, Graph):
        return edge_index
    key = id(edge_index)
    hit = _cache.get(key)
    if hit is not None:
        ref, version, n, g = hit
        if ref() is edge_index and version == edge_index._version and (num_nodes is None or n == num_nodes):
            if torch.is_grad_enabled():
                g.by_src  # the caller's tensor may be gone by the time backward runs
            return g
    if num_nodes is None:
        raise _lib.HgvError("num_nodes is required to build a Graph")
    g = Graph(edge_index, num_nodes, hold=False)
    g.by_dst.long_rows(g.num_nodes)
    if torch.is_grad_enabled():
        # built now: the caller's tensor may be gone by the time backward runs - and everything the backward pass reads
        # exists before any of it can run on a second stream
        g.by_src.long_rows(g.num_nodes)
        g.inv_deg
    ref = weakref.ref(edge_index, lambda _r, k=key: _cache.pop(k, None))
    _cache[key] = (ref, edge_index._version, num_nodes, g)
    return g


def _not_captured() -> None:
    if torch.cuda.is_current_stream_capturing():
        raise _lib.HgvError("Segments copies between host and device: make it before the capture")


class Segments:
    """Which rows of a batched matrix belong to which graph: the plan that the per-graph operators
    (:func:`~hgvae_amd.functional.group_norm_act`, :func:`~hgvae_amd.functional.graph_attention`) take.

    Rows of a graph are consecutive and graphs follow one another, as ``Batch.from_data_list`` lays them out; a graph may
    have no rows.  Building one uploads a few arrays (and, from a device tensor, reads the sizes back: one host
    synchronisation); a plan serves every call, stream and captured graph afterwards, so a loop keeps it next to its batch.
    """
    MAX_ROWS = 2 ** 31 - 2 ** 16                                # row numbers are 32 bits, and loops step beyond the last one

    def __init__(self, sizes: Sequence[int], device):
        sizes = np.asarray(list(sizes) if not isinstance(sizes, np.ndarray) else sizes)
        if sizes.ndim != 1 or (sizes.size and sizes.dtype.kind not in "iu"):
            raise _lib.HgvError("Segments: sizes must be a sequence of integers")
        sizes = sizes.astype(np.int64)
        if sizes.size and (int(sizes.min()) < 0 or int(sizes.max()) > self.MAX_ROWS or int(sizes.sum()) > self.MAX_ROWS):
            raise _lib.HgvError(f"Segments: sizes must be >= 0 and sum to at most {self.MAX_ROWS} rows")
        self.device = torch.device(device)
        if self.device.type != "cuda":
            raise _lib.HgvError("hgvae_amd operators run on the GPU only (Segments needs a cuda device)")
        if self.device.index is None:
            self.device = torch.device("cuda", torch.cuda.current_device())
        _not_captured()
        self.sizes = [int(s) for s in sizes]
        self.num_graphs, self.num_rows = len(self.sizes), int(sizes.sum())
        ptr = np.zeros(self.num_graphs + 1, dtype=np.int64)
        np.cumsum(sizes, out=ptr[1:])
        # graphs that have rows, smallest first (stable): operators split this list at a size of their own
        order = np.argsort(sizes, kind="stable")
        order = order[int((sizes == 0).sum()):]
        self._sorted = sizes[order].tolist()
        # row chunks of the norm's passes: 64 rows (32 where that leaves fewer than 2 048 of them), at most 512 per graph
        rows = 64 if self.num_rows >= 64 * 2048 else 32
        per = np.maximum(rows, -(-sizes[order] // 512))
        counts = -(-sizes[order] // per)
        first = np.zeros(order.size + 1, dtype=np.int64)
        np.cumsum(counts, out=first[1:])
        total = int(first[-1])
        self._first_host = first.tolist()
        which = np.repeat(np.arange(order.size), counts)
        start = ptr[order][which] + (np.arange(total) - first[which]) * per[which]
        chunks = np.zeros((total, 4), dtype=np.int64)
        chunks[:, 0], chunks[:, 1] = order[which], start
        chunks[:, 2] = np.minimum(start + per[which], ptr[order + 1][which])
        # attention: tiles of 64 rows in row order, each with the first tile of its graph and their number, and blocks of 64
        # and of 128 rows, those of the largest graphs first
        tiles, blocks = self._tiles_of(sizes, ptr, np.flatnonzero(sizes), 64), [self._tiles_of(sizes, ptr, order[::-1], r) for r in (64, 128)]
        self._n_tiles = len(tiles)
        parts = [chunks.ravel(), tiles.ravel(), np.concatenate(blocks).ravel(), ptr, order, first]
        host = np.concatenate(parts).astype(np.int32)
        self._buf = torch.from_numpy(host).to(self.device)          # copied before the call returns: any stream may read it
        self._home = _lib.stream_of(self.device.index)
        at = np.cumsum([0] + [p.size for p in parts])
        self._chunks, self._tiles, self._blocks, self._ptr, self._order, self._first = (self._buf[at[i]:at[i + 1]] for i in range(6))
        self._norm_plans: "dict[tuple, tuple]" = {}
        self._attention_plan = (self._ptr.data_ptr(), self._sorted[-1] if self._sorted else 0, self._tiles.data_ptr(), self._n_tiles,
                                self._blocks.data_ptr(), *map(len, blocks))

    def __reduce__(self):
        return Segments, (self.sizes, str(self.device))             # copies and pickles get arrays of their own

    @staticmethod
    def _tiles_of(sizes, ptr, graphs, rows: int) -> np.ndarray:
        """(graph, first row, first tile of the graph, tiles of the graph) of every tile of ``rows`` rows, graph by graph."""
        counts = -(-sizes[graphs] // rows)
        first = np.cumsum(counts) - counts
        total = int(counts.sum())
        which = np.repeat(np.arange(len(graphs)), counts)
        out = np.empty((total, 4), dtype=np.int64)
        out[:, 0], out[:, 2], out[:, 3] = graphs[which], first[which], counts[which]
        out[:, 1] = ptr[graphs][which] + (np.arange(total) - first[which]) * rows
        return out

    @classmethod
    def from_sizes(cls, sizes: Sequence[int], device="cuda") -> "Segments":
        """From the number of rows of each graph, in order."""
        return cls(sizes, device)

    @classmethod
    def from_ptr(cls, ptr: torch.Tensor, device=None) -> "Segments":
        """From the first row of each graph and the end (``Batch.ptr``)."""
        if ptr.dim() != 1 or ptr.numel() < 1 or ptr.dtype not in (torch.int32, torch.int64):
            raise _lib.HgvError("Segments: ptr must be a 1-D integer tensor with at least one entry")
        if ptr.is_cuda:
            _not_captured()
        host = ptr.detach().cpu().numpy().astype(np.int64)
        if host[0] != 0:
            raise _lib.HgvError("Segments: ptr must start at 0")
        return cls(np.diff(host), ptr.device if device is None else device)

    @classmethod
    def from_batch(cls, batch: torch.Tensor, num_graphs: Optional[int] = None) -> "Segments":
        """From the graph number of each row (``Batch.batch``), which must not decrease."""
        if batch.dim() != 1 or batch.dtype not in (torch.int32, torch.int64):
            raise _lib.HgvError("Segments: batch must be a 1-D integer tensor")
        if batch.is_cuda:
            _not_captured()
        host = batch.detach().cpu().numpy().astype(np.int64)
        if host.size and (host[0] < 0 or (np.diff(host) < 0).any()):
            raise _lib.HgvError("Segments: the rows of a graph must be consecutive and graphs in order")
        count = int(host[-1]) + 1 if host.size else 0
        if num_graphs is not None:
            if int(num_graphs) < count:
                raise _lib.HgvError(f"Segments: batch names graph {count - 1} of {num_graphs}")
            count = int(num_graphs)
        if count > cls.MAX_ROWS:
            raise _lib.HgvError(f"Segments: {count} graphs")
        return cls(np.bincount(host, minlength=count) if host.size else np.zeros(count, dtype=np.int64), batch.device)

    def _norm_plan(self, columns: int, groups: int, wide: bool):
        """What a call of the norm passes on: (device arrays), (graphs, graphs with rows, how many of them one workgroup reads at
        once, rows of the largest of those, first chunk of the others, end of the chunks), workspace bytes forward and backward.
        ``wide``: the matrices' rows are multiples of 16 bytes apart."""
        plan = self._norm_plans.get((columns, groups, wide))
        if plan is None:
            lib = _lib.load()
            limit = lib.hgv_group_norm_small_rows(columns, groups)
            per = columns // groups
            slab = per * max(1, -(-32 // per))                  # the columns that a workgroup takes
            if wide and slab < columns and slab % 32 and 4 * self.num_rows * columns > 64 << 20:
                # one read of a whole graph per workgroup saves launches and passes.  Where memory is what counts and its pieces of rows
                # are not whole lines, long graphs run faster in chunks of 16-byte reads (forward and backward, one read / chunks, 50 M values:
                # slabs of 33 columns, graphs of 130 rows 477 / 473 us, of 200 466 / 435, of 300 516 / 362;  of 46 columns 430 / 439, 512 / 413,
                # 460 / 353;  of 60 columns 485 / 380, 419 / 382;  256 columns in slabs of 32: 2 500 of 200 rows 778 / 1 049).  Chunks in
                # 4-byte reads are slower (138 columns without pads: 130 rows 432 / 587, 200 rows 514 / 595, 300 rows 461 / 493)
                limit = min(limit, 160)
            n, listed = bisect.bisect_right(self._sorted, limit), len(self._sorted)
            if n < listed and 8 * sum(self._sorted[:n]) < self.num_rows:
                n = 0                   # a few small graphs beside large ones: not worth a launch of their own
            chunks = (self._first_host[n], self._first_host[-1])
            ws = [lib.hgv_group_norm_ws(chunks[1] - chunks[0], self.num_graphs, listed, n, columns, groups, b) for b in (0, 1)]
            plan = (tuple(t.data_ptr() for t in (self._ptr, self._order, self._chunks, self._first)),
                    (self.num_graphs, listed, n, self._sorted[n - 1] if n else 0, *chunks), *ws)
            self._norm_plans[columns, groups, wide] = plan
        return plan

    def __repr__(self):
        return f"Segments({self.num_graphs} graphs, {self.num_rows} rows, {self.device})"


def segments_of(segments, num_rows: int) -> Segments:
    """A :class:`Segments`, or one built for this call from a ``batch`` vector (one host synchronisation)."""
    if not isinstance(segments, Segments):
        if not isinstance(segments, torch.Tensor):
            raise _lib.HgvError("expected Segments or a batch vector")
        segments = Segments.from_batch(segments)
    if segments.num_rows != num_rows:
        raise _lib.HgvError(f"the matrix has {num_rows} rows but the graphs have {segments.num_rows}")
    index = segments.device.index
    if _lib.stream_of(index) != segments._home and not torch.cuda.is_current_stream_capturing():
        segments._buf.record_stream(torch.cuda.current_stream(index))       # a plan that is dropped outlives what reads it there
    return segments
