"""The neighbourhood softmax with a learned relative bias.

Every edge ``e = (i <- j)`` lies in a bucket (a ring of distance, a side, whatever
its owner sorts edges by), and head h learns one number a bucket,

    s_h   = scale <q_i,h, rho(g_ij) k_j,h> + bias(e) + table[bucket(e), h],
    alpha = softmax of s_h over i's edges inside the window,

so that a layer's weights can depend on where a neighbour sits beside what it
holds.  The table's gradient is the sum, over a bucket's edges, of the scores'.

Edges outside the window count for nothing, whatever their rows hold and whatever the
row's other scores are, nor do edges of weight zero in a gradient; a target with no
edge inside has only zero weights (and zero gradients).

The op reads an edge set through :class:`RelativeEdgeTables`, which its owner builds
once and keeps.  On the GPU (``gm_relative_*``) neither the scores nor the learned
bias of an edge is written; the backward reads the weights the forward gave.
bfloat16 rows take float32 tables, arithmetic and weights, and get bfloat16
gradients, rounded once; the learned table's sums are in a fixed order.  CPU
tensors take the formulas in torch.
"""

from __future__ import annotations

import functools
import math
from typing import Any

import torch
from torch import Tensor

from gm_attention_amd import _native
from gm_attention_amd.nn import differential, fused_attention
from gm_attention_amd.nn.differential import EdgeTables
from gm_attention_amd.representations.field_type import SO2FieldType

MAX_H, MAX_F, MAX_D = fused_attention.MAX_H, fused_attention.MAX_F, fused_attention.MAX_D
MAX_BUCKETS = 256
# up to here the scores' rows of more than 8 steps, not 32, take four waves.  5,120 waves run at once (five a SIMD);
# while the targets are about three times as many the launch ends with its longest rows, which four waves shorten
# (2,048 targets 14.2 -> 9.1 us, 12,285 46 -> 34), beyond it the waves' sharing costs more (32,768: 131 -> 174)
FEW_TARGETS = 16384
MAX_SOURCES = 2**24  # of float32 tables: a record's word holds the source and the bucket


def distance_buckets(distances: Tensor, cutoff: float, n_buckets: int) -> Tensor:
    """Every edge's ring of distance, ``n_buckets`` of equal width up to ``cutoff``.

    A ring begins a thousandth of its width early: a lattice's distances lie on the
    borders, and their roundings must not tell equal ones apart."""
    rings = torch.floor(distances * (n_buckets / cutoff) + 1e-3)
    return rings.clamp_(0, n_buckets - 1).to(torch.int32)


class RelativeEdgeTables(EdgeTables):
    """:class:`differential.EdgeTables` with every edge's bucket ``(n_edges,)``, whole
    numbers in ``0 .. n_buckets - 1`` (checked here, once).

    The backward's lane kernels read pairs of neighbouring targets, and of sources, each
    with the list of the nodes that either has an edge with: neighbours on a grid share
    most of theirs, whose rows are then loaded once for both.  The lists are found with
    the first call that a backward can follow (or by :meth:`group_sources`), outside a
    capture, and kept: of each side 48 bytes an entry at three orders, four entries for
    seven edges or fewer on a grid."""

    def __init__(self, row_ptr: Tensor, source: Tensor, transport: Tensor, bias: Tensor, inside: Tensor,
                 buckets: Tensor, n_buckets: int, *, n_sources: int | None = None) -> None:
        differential._outside_capture(row_ptr, "RelativeEdgeTables")
        if not 1 <= n_buckets <= MAX_BUCKETS:
            raise ValueError(f"n_buckets must lie in 1..{MAX_BUCKETS}, got {n_buckets}.")
        if buckets.dtype not in (torch.uint8, torch.int16, torch.int32, torch.int64) or buckets.shape != source.shape:
            raise ValueError(f"buckets must be integers ({source.shape[0]},).")
        if buckets.device != row_ptr.device:
            raise ValueError("every table must live on the same device.")
        if buckets.numel() and bool((buckets.amin() < 0) | (buckets.amax() >= n_buckets)):
            raise ValueError(f"every bucket must lie in 0 .. {n_buckets - 1}.")
        nodes = row_ptr.shape[0] - 1 if n_sources is None else int(n_sources)
        if transport.dtype == torch.float32 and nodes > MAX_SOURCES:
            raise ValueError(f"float32 tables hold at most {MAX_SOURCES} sources, got {nodes}.")
        self.n_buckets = int(n_buckets)
        self.buckets = buckets.detach().to(torch.uint8, copy=True)
        self._pairs: dict[str, tuple[Tensor, Tensor]] = {}
        super().__init__(row_ptr, source, transport, bias, inside, n_sources=n_sources)

    def _hold(self, source: Tensor, phases: Tensor, masked: Tensor) -> None:
        super()._hold(source, phases, masked)
        if self.device.type == "cuda":
            self._kept.append(_native.Made(self.buckets))

    def __getstate__(self) -> dict:
        return {n: v for n, v in super().__getstate__().items() if n != "_pairs"}

    def __setstate__(self, state: dict) -> None:
        self._pairs = {}
        super().__setstate__(state)
        if self.device.type == "cuda" and "records" in state:
            self._kept.append(_native.Made(self.buckets))

    def group_sources(self) -> tuple[Tensor, Tensor]:
        """Finds what a backward reads beside the edges, once: the pairs of targets and of sources
        (``(ptr, entries)`` of the sources'), or for float64 tables the edges sorted by source."""
        if self.dtype == torch.float64:
            return super().group_sources()
        self._paired("targets")
        return self._paired("sources")

    def sources(self, slots: int) -> tuple[Tensor | None, Tensor | None]:
        """``(src_ptr, records_s)`` for the simple kernels (``slots`` 0)."""
        return (None, None) if slots else super().group_sources()

    def pairs(self, side: str, slots: int) -> tuple:
        """The pairs of ``"targets"`` or ``"sources"`` as the entry points take them, for lane
        kernels with ``slots`` edge slots a wave (0: none, the simple kernels)."""
        if slots == 0:
            return None, None, None, None
        ptr, entries = self._paired(side)
        # rows beyond 16 steps of a wave are a workgroup's: 32 times these slots
        order, counts = self._rows((f"{side}' pairs", max(1, slots // 2)), lambda: ptr)
        # an edge set without edges has entries of no pair, and an address all the same
        return entries.data_ptr(), _native._ptr(ptr), _native._ptr(order), counts

    def lane_rows(self, slots: int) -> tuple[Tensor | None, Any]:
        """The targets in classes for the forward's lane kernels: rows beyond 32 steps of a wave are a
        workgroup's, of few targets, where the longest row decides, beyond 8."""
        return self.target_rows(max(1, slots // 4) if slots and self.n_targets <= FEW_TARGETS else slots)

    def _paired(self, side: str) -> tuple[Tensor, Tensor]:
        held = self._pairs.get(side)
        if held is None:
            with _native.LOCK:
                held = self._pairs.get(side)
                if held is None:
                    held = self._pairs[side] = self._pair(side == "targets")
        return held

    def _pair(self, targets: bool) -> tuple[Tensor, Tensor]:
        """``(ptr, entries)``: every pair's entries, in order of their nodes."""
        differential._outside_capture(self.row_ptr, "RelativeEdgeTables' pairs (a first call with these tables)")
        self.found()
        target = torch.repeat_interleave(torch.arange(self.n_targets, device=self.device),
                                         self.row_ptr[1:] - self.row_ptr[:-1], output_size=self.n_edges)
        source = self._unpacked(self.records)
        row, node, rows, nodes = ((target, source, self.n_targets, self.n_sources) if targets else
                                  (source, target, self.n_sources, self.n_targets))
        # by pair, node and row; edges of one row to one node stand apart
        key, edge = torch.sort(((row >> 1) * nodes + node) * 2 + (row & 1), stable=True)
        again = torch.zeros_like(key)
        if self.n_edges > 1 and bool((key[1:] == key[:-1]).any()):
            place = torch.arange(self.n_edges, device=self.device)
            first = torch.ones_like(key, dtype=torch.bool)
            first[1:] = key[1:] != key[:-1]
            again = place - torch.cummax(torch.where(first, place, 0), 0).values
            by = torch.sort(again, stable=True).indices
            by = by[torch.sort(key[by] >> 1, stable=True).indices]
            key, edge, again = key[by], edge[by], again[by]
        second, key = key & 1, key >> 1
        new = torch.ones_like(key, dtype=torch.bool)
        new[1:] = (key[1:] != key[:-1]) | (again[1:] != again[:-1])
        entry = torch.cumsum(new, 0) - 1
        key = key[new]
        n = key.shape[0]
        ptr = torch.searchsorted(key // max(nodes, 1), torch.arange((rows + 1) // 2 + 1, device=self.device))
        edges = torch.full((n, 2), -1, dtype=torch.int64, device=self.device)
        edges.view(-1)[2 * entry + second] = edge
        there, at = edges >= 0, edges.clamp_min(0)
        entries = torch.zeros(max(n, 1), 4 * self.orders, dtype=torch.float32, device=self.device)
        words = entries.view(torch.int32)
        words[:n, 0] = key % max(nodes, 1)
        words[:n, 1], words[:n, 3] = edges.unbind(1)
        phases = self.records[at][:, :, 2:].reshape(n, 2, self.orders - 1, 2).masked_fill(~there[:, :, None, None], 0.0)
        entries[:n, 4:] = phases.transpose(1, 2).flatten(1)
        self._kept.append(_native.Made(entries, ptr))
        return ptr, entries

    def _packed(self, source: Tensor) -> Tensor:
        buckets = self.buckets.long()
        if self.dtype == torch.float64:
            return source + (buckets << 32)
        word = source + (buckets << 24)
        return torch.where(word >= 2**31, word - 2**32, word)  # the same 32 bits

    def _unpacked(self, records: Tensor) -> Tensor:
        mask = 0xFFFFFF if self.dtype == torch.float32 else 0xFFFFFFFF
        return super()._unpacked(records) & mask

    def _source_records(self, target: Tensor, edge: Tensor, records: Tensor) -> Tensor:
        records_s = torch.empty(self.n_edges, 2 * self.orders, dtype=self.dtype, device=self.device)
        words = records_s.view(differential._WORD[self.dtype])
        words[:, 0] = target
        words[:, 1] = edge
        records_s[:, 2:] = records[:, 2:]
        return records_s


class Heads:
    """The rows' ``heads`` heads of ``head_type`` as the entry points take them."""

    def __init__(self, head_type: SO2FieldType, heads: int) -> None:
        if not 1 <= heads <= MAX_H:
            raise ValueError(f"heads must lie in 1..{MAX_H}, got {heads}.")
        full = head_type.scaled(heads)
        if len(head_type) > MAX_F or full.dimension > MAX_D:
            raise ValueError(f"the heads must hold at most {MAX_F} frequencies and {MAX_D} numbers a row, "
                             f"got {full!r} ({full.dimension}).")
        self.heads, self.scale = heads, 1.0 / math.sqrt(head_type.dimension)
        self.plan = fused_attention.plan_of(head_type, full, heads)
        self.top = head_type.max_frequency
        # rows of more than 32 of these go to a workgroup where ds is formed: a wave holds 12 steps of 64 / heads edges
        self.score_slots = max(1, 12 * (64 // heads) // 32)
        # read on the host, whatever the default device of the call that makes the (kept) heads
        self.desc = torch.tensor([list(row) for row in self.plan.rows], dtype=torch.int64, device="cpu")
        self._slots: dict[int, int] = {}
        self._served: dict[tuple[int, torch.dtype], Heads] = {}

    def served(self, tables: EdgeTables) -> Heads:
        """The heads as the kernels take them: these, or with copies of zeros where that gives the lane kernels
        whole units (rows are repacked: little beside an edge set's many edges a row)."""
        held = self._served.get((tables.orders, tables.dtype))
        if held is None:
            held = self
            if tables.dtype != torch.float64 and not self.slots(tables):
                copies = _native.relative_padded(self.desc, self.plan.width, tables.orders, self.heads)
                held = heads_of(SO2FieldType(copies), self.heads) if copies else self
            self._served[tables.orders, tables.dtype] = held
        return held

    def slots(self, tables: EdgeTables) -> int:
        """Edge slots of a wave of the lane kernels (0: the simple kernels serve)."""
        if tables.dtype == torch.float64:
            return 0
        held = self._slots.get(tables.orders)
        if held is None:
            held = self._slots[tables.orders] = _native.relative_slots(self.desc, self.plan.width, tables.orders,
                                                                       self.heads)
        return held


heads_of = functools.lru_cache(maxsize=256)(Heads)


class RelativeSoftmax(torch.autograd.Function):
    """``alpha (n_edges, H)`` from the heads' rows and ``table (n_buckets, H)``; ``dq``,
    ``dk`` in the rows' dtype and ``dtable`` back."""

    @staticmethod
    def forward(ctx: Any, q: Tensor, k: Tensor, table: Tensor, tables: RelativeEdgeTables, heads: Heads, scale: float,
                train: bool) -> Tensor:
        if train:  # found here: the backward runs on a thread and perhaps a stream of its own
            slots = heads.served(tables).slots(tables)
            tables.sources(slots)
            tables.pairs("targets", slots)
            tables.pairs("sources", slots)
            tables.target_rows(heads.score_slots)
        with _native.span("gm::attention/relative_softmax"):
            alpha = _native.relative_forward(q, k, table, tables, heads, scale)
        if train:
            ctx.save_for_backward(q, k, alpha)
            ctx.rest = (tables, heads, scale)
        return alpha

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_alpha: Tensor) -> tuple:
        q, k, alpha = ctx.saved_tensors
        with _native.span("gm::attention/relative_softmax_backward"):
            dq, dk, dtable = _native.relative_backward(grad_alpha.contiguous(), alpha, q, k, *ctx.rest)
        return dq, dk, dtable, None, None, None, None


def relative_softmax(q: Tensor, k: Tensor, table: Tensor, tables: RelativeEdgeTables, head_type: SO2FieldType,
                     heads: int, scale: float | None = None) -> Tensor:
    """The heads' attention weights ``(n_edges, heads)`` of ``q (n_targets, D)`` and
    ``k (n_sources, D)``, rows of ``heads`` heads of ``head_type``, under the learned
    ``table (n_buckets, heads)``; ``scale`` is ``1 / sqrt(dim head_type)`` by default."""
    if not isinstance(head_type, SO2FieldType):
        raise TypeError(f"head_type must be an SO2FieldType, got {type(head_type).__name__}.")
    layout = heads_of(head_type, heads)
    width = layout.plan.width
    if not isinstance(tables, RelativeEdgeTables):
        raise TypeError(f"tables must be RelativeEdgeTables, got {type(tables).__name__}.")
    dtype = torch.float32 if q.dtype == torch.bfloat16 else q.dtype
    if dtype != tables.dtype or k.dtype != q.dtype:
        raise ValueError(f"q and k must share a dtype, {tables.dtype} (or bfloat16 with float32 tables), "
                         f"got {q.dtype} and {k.dtype}.")
    if tuple(q.shape) != (tables.n_targets, width) or tuple(k.shape) != (tables.n_sources, width):
        raise ValueError(f"q and k must be ({tables.n_targets}, {width}) and ({tables.n_sources}, {width}), "
                         f"got {tuple(q.shape)} and {tuple(k.shape)}.")
    if tuple(table.shape) != (tables.n_buckets, heads) or not table.is_floating_point():
        raise ValueError(f"table must be ({tables.n_buckets}, {heads}) real numbers, "
                         f"got {tuple(table.shape)} of {table.dtype}.")
    if any(t.device != tables.device for t in (q, k, table)):
        raise ValueError("q, k and table must live on the tables' device.")
    if layout.top >= tables.orders:
        raise ValueError(f"the tables hold orders below {tables.orders}, the heads need {layout.top}.")
    scale = layout.scale if scale is None else float(scale)
    if q.device.type != "cuda":
        return _eager(q, k, table, tables, layout.plan, scale)
    # whether a backward can follow: inside the op a parameter looks the same under no_grad
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or table.requires_grad)
    return RelativeSoftmax.apply(differential._whole(q), differential._whole(k), table.to(dtype).contiguous(), tables,
                                 layout, scale, train)


def enabled(mhsa: Any, x: Any, edges: Any) -> bool:
    """Whether a layer's scores with a relative bias take the fused op on the GPU."""
    if fused_attention.MODE == "0" or x.device.type != "cuda" or edges.n_edges == 0:
        return False
    if x.dtype not in (torch.float32, torch.float64, torch.bfloat16) or mhsa.num_heads > MAX_H:
        return False
    head = mhsa.field_type_attn
    n_nodes = edges.row_ptr.shape[0] - 1
    return (len(head) <= MAX_F and mhsa.field_type_in.dimension <= MAX_D and head.max_frequency <= edges.max_frequency
            and (n_nodes <= MAX_SOURCES or x.dtype == torch.float64))


def _kind(top: int, n_buckets: int) -> differential._Kind:
    """The tables of an edge set whose buckets are rings of distance up to its cutoff."""
    def make(g: fused_attention.Geometry, row_ptr: Tensor, source: Tensor, n_sources: int | None) -> EdgeTables:
        return RelativeEdgeTables(row_ptr, source, g.transport[:, : top + 1], g.bias, g.inside,
                                  distance_buckets(g.rho, 1.0, n_buckets), n_buckets, n_sources=n_sources)

    return differential._Kind(("relative", top, n_buckets), make)


def attention_weights(mhsa: Any, q: Tensor, k: Tensor, edges: Any) -> Tensor:
    """The weights ``(n_edges, n_heads)`` of a layer with a learned bias a ring of distance
    from its flat query and key rows: the fused op where it serves, else its formulas in torch."""
    head, table, window = mhsa.field_type_attn, mhsa.relative_bias, mhsa.heads[0].window
    dtype = torch.float32 if q.dtype == torch.bfloat16 else q.dtype
    scale = float(mhsa.heads[0]._score_scale)
    if not enabled(mhsa, q, edges):  # of any size, unlike the op's
        g = fused_attention.geometry(edges, mhsa.cutoff, window, dtype)
        buckets = distance_buckets(g.rho, 1.0, table.shape[0]).long()
        return _weights(q, k, table, buckets, g.row_ptr, g.source, g.transport[:, 1:].flatten(1),
                        g.bias.masked_fill(g.inside == 0, -math.inf),
                        fused_attention.plan_of(head, mhsa.field_type_in, mhsa.num_heads), scale)
    top = head.max_frequency
    kind = _kind(top, table.shape[0])
    if fused_attention.chunk_of(edges) is not None:
        tables, first, source = differential.chunk_tables(edges, mhsa.cutoff, window, dtype, top, kind)
        q, k = q[first:first + tables.n_targets], k[source:source + tables.n_sources]
    else:
        tables = differential.edge_tables(edges, mhsa.cutoff, window, dtype, top, kind)
    return relative_softmax(q, k, table, tables, head, mhsa.num_heads, scale)


def _eager(q: Tensor, k: Tensor, table: Tensor, tables: RelativeEdgeTables, plan: fused_attention.Plan,
           scale: float) -> Tensor:
    return _weights(q, k, table, tables.buckets.long(), tables.row_ptr, tables._source, tables._phases, tables._bias,
                    plan, scale)


def _weights(q: Tensor, k: Tensor, table: Tensor, buckets: Tensor, row_ptr: Tensor, source: Tensor, phases: Tensor,
             bias: Tensor, plan: fused_attention.Plan, scale: float) -> Tensor:
    """The formulas in torch, in the bias's arithmetic (``-inf`` outside the window)."""
    learned = table.to(bias.dtype).index_select(0, buckets)
    return differential.torch_weights(q, k, row_ptr, source, phases, bias, plan, scale, learned)[0]
