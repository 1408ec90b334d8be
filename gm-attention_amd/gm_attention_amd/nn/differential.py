"""The differential neighbourhood softmax: per head the difference of two maps.

Head h scores every edge ``e = (i <- j)`` twice, with the maps ``p = 2h, 2h + 1``
of ``map_type`` each,

    s_p   = scale <q_i,p , rho(g_ij) k_j,p> + bias(e),
    a_p   = softmax of s_p over i's edges inside the window,
    alpha = a_2h - lambda_h a_2h+1,

``lambda`` one learned number a head.  What both maps give to every neighbour
cancels, so the weights keep what tells neighbours apart.  A map's copies sit
side by side in the rows (map-major within each frequency), so rows of H heads
with an even number of copies hold H heads of two maps of half the copies each:
the layers' query and key rows serve as they are.

Edges outside the window count for nothing, whatever their rows hold; a target
with no edge inside has only zero weights (and zero gradients).

The op reads an edge set through :class:`EdgeTables`, which its owner builds once
and keeps.  On the GPU (``gm_differential_*``) neither the maps nor their
gradients are written: the forward keeps two numbers a target and map for
the backward.  bfloat16 rows take float32 tables, arithmetic and weights, and get
bfloat16 gradients, rounded once.  CPU tensors take the formulas in torch.
"""

from __future__ import annotations

import ctypes
import functools
import math
from collections import OrderedDict
from collections.abc import Callable
from typing import Any, NamedTuple

import numpy as np
import torch
from torch import Tensor

from gm_attention_amd import _native
from gm_attention_amd.nn import fused_attention
from gm_attention_amd.representations.field_type import SO2FieldType

MAX_H, MAX_F, MAX_D = fused_attention.MAX_H, fused_attention.MAX_F, fused_attention.MAX_D


class EdgeTables:
    """What the op reads of one edge set: the CSR over targets (``row_ptr``,
    ``source``), the transport phases ``(E, orders, 2)``, the softmax bias and the
    window's support (:class:`fused_attention.Geometry`'s tables).

    ``n_sources`` is the number of key rows (the targets' by default).  The
    indices are checked here, once; the GPU's copies of the tables are packed here,
    so a table written to afterwards is not seen.  A step under graph capture needs
    its tables (for training :meth:`group_sources` too) from before the capture."""

    def __init__(self, row_ptr: Tensor, source: Tensor, transport: Tensor, bias: Tensor, inside: Tensor, *,
                 n_sources: int | None = None) -> None:
        _outside_capture(row_ptr, "EdgeTables")
        n_edges = source.shape[0]
        if row_ptr.dtype != torch.int64 or row_ptr.ndim != 1 or row_ptr.shape[0] < 1:
            raise ValueError("row_ptr must be int64 (n_targets + 1,).")
        if source.dtype != torch.int64 or source.ndim != 1:
            raise ValueError("source must be int64 (n_edges,).")
        if transport.ndim != 3 or transport.shape[0] != n_edges or transport.shape[1] < 1 or transport.shape[2] != 2:
            raise ValueError(f"transport must be ({n_edges}, orders, 2), got {tuple(transport.shape)}.")
        if transport.dtype not in (torch.float32, torch.float64):
            raise ValueError(f"the tables must be float32 or float64, got {transport.dtype}.")
        if bias.dtype != transport.dtype or tuple(bias.shape) != (n_edges,):
            raise ValueError(f"bias must be ({n_edges},) in transport's dtype.")
        if inside.dtype not in (torch.uint8, torch.bool) or tuple(inside.shape) != (n_edges,):
            raise ValueError(f"inside must be uint8 or bool ({n_edges},).")
        if any(t.device != row_ptr.device for t in (source, transport, bias, inside)):
            raise ValueError("every table must live on the same device.")
        self.n_targets = row_ptr.shape[0] - 1
        self.n_sources = self.n_targets if n_sources is None else int(n_sources)
        self.n_edges = n_edges
        if max(self.n_targets, self.n_sources, n_edges) >= 2**31:
            raise ValueError("nodes and edges are indexed in 32 bits.")
        bad = (row_ptr[0] != 0) | (row_ptr[-1] != n_edges) | (row_ptr[1:] < row_ptr[:-1]).any()
        if n_edges:
            bad = bad | (source.amin() < 0) | (source.amax() >= self.n_sources)
        if bool(bad):
            raise ValueError("row_ptr must rise from 0 to n_edges and every source lie in 0 .. n_sources - 1.")
        self.device, self.dtype, self.orders = transport.device, transport.dtype, transport.shape[1]
        self.row_ptr = row_ptr.detach().clone()
        self._sources, self._classes = None, {}
        masked = bias.detach().masked_fill(inside == 0, -math.inf)
        phases = transport.detach()[:, 1:].reshape(n_edges, 2 * (self.orders - 1))
        self._hold(source.detach(), phases, masked)

    def _hold(self, source: Tensor, phases: Tensor, masked: Tensor) -> None:
        """The checked tables in the form their device reads."""
        if self.device.type != "cuda":
            with torch.inference_mode(False):  # a later step may train: autograd saves no inference tensor
                self._source, self._phases, self._bias = (t.clone() if t.is_inference() else t
                                                          for t in (source, phases, masked))
            return
        records = torch.empty(self.n_edges, 2 * self.orders, dtype=self.dtype, device=self.device)
        words = records.view(_WORD[self.dtype])
        words[:, 0] = self._packed(source)
        # in units of log 2; the type's lowest value stays a finite one
        lowest = torch.finfo(self.dtype).min
        records[:, 1] = torch.where(masked == -math.inf, masked, (masked * _LOG2E).clamp_min(lowest))
        records[:, 2:] = phases
        self.records = records
        self._kept = [_native.Made(self.row_ptr, records)]

    def __getstate__(self) -> dict:
        """A copy (of the edge set that keeps them too) takes the tables alone: what is
        found from them is found again, and a stream's events are not copied."""
        if self.device.type == "cuda":
            self.found()
        return {n: v for n, v in self.__dict__.items() if n not in ("_kept", "_sources", "_classes")}

    def __setstate__(self, state: dict) -> None:
        self.__dict__.update(state, _sources=None, _classes={}, device=state["row_ptr"].device)
        if self.device.type == "cuda" and "records" in state:
            self._kept = [_native.Made(self.row_ptr, self.records)]
        elif self.device.type == "cuda":  # read back on another device than the one they were written from
            self._hold(*(self.__dict__.pop(n) for n in ("_source", "_phases", "_bias")))
        elif "records" in state:
            records = self.__dict__.pop("records")
            self._hold(self._unpacked(records), records[:, 2:], records[:, 1] / _LOG2E)

    def _packed(self, source: Tensor) -> Tensor:
        """The records' first words."""
        return source

    def _unpacked(self, records: Tensor) -> Tensor:
        """The sources in the records."""
        return records.view(_WORD[self.dtype])[:, 0].long()

    def group_sources(self) -> tuple[Tensor, Tensor]:
        """``(src_ptr, records_s)``: the edges sorted by source, each with its target,
        its place and its tables, for the backward; found once."""
        if self._sources is None:
            with _native.LOCK:
                if self._sources is None:
                    self._sources = self._group()
        return self._sources

    def _group(self) -> tuple[Tensor, Tensor]:
        _outside_capture(self.row_ptr, "EdgeTables.group_sources")
        self.found()
        sorted_source, order = torch.sort(self._unpacked(self.records).to(torch.int32), stable=True)
        bounds = torch.arange(self.n_sources + 1, dtype=torch.int32, device=self.device)
        src_ptr = torch.searchsorted(sorted_source, bounds)
        target = torch.repeat_interleave(torch.arange(self.n_targets, device=self.device),
                                         self.row_ptr[1:] - self.row_ptr[:-1], output_size=self.n_edges)
        records_s = self._source_records(target.index_select(0, order), order, self.records.index_select(0, order))
        self._kept.append(_native.Made(src_ptr, records_s))
        return src_ptr, records_s

    def _source_records(self, target: Tensor, edge: Tensor, records: Tensor) -> Tensor:
        records_s = torch.empty(self.n_edges, 2 + 2 * self.orders, dtype=self.dtype, device=self.device)
        words = records_s.view(_WORD[self.dtype])
        words[:, 0] = target
        words[:, 1] = edge
        words[:, 3] = 0
        records_s[:, 2] = records[:, 1]
        records_s[:, 4:] = records[:, 2:]
        return records_s

    def target_rows(self, slots: int) -> tuple[Tensor | None, Any]:
        """The targets in the classes of degree that the lane kernels with ``slots``
        edge slots a wave take, and the classes' counts as the entry points read
        them; ``(None, None)`` for ``slots`` 0, the simple kernels."""
        return self._rows(("targets", slots), lambda: self.row_ptr)

    def source_rows(self, slots: int) -> tuple[Tensor | None, Any]:
        """The same of the sources and their edges."""
        return self._rows(("sources", slots), lambda: self.group_sources()[0])

    def _rows(self, key: tuple[str, int], ptr: Any) -> tuple[Tensor | None, Any]:
        if key[1] == 0:
            return None, None
        held = self._classes.get(key)
        if held is None:
            with _native.LOCK:
                held = self._classes.get(key)
                if held is None:
                    held = self._classes[key] = self._in_classes(ptr(), key[1])
        return held

    def _in_classes(self, ptr: Tensor, slots: int) -> tuple[Tensor, Any]:
        _outside_capture(ptr, "EdgeTables' rows in classes (a first call with these tables and heads)")
        self.found()
        degree = ptr[1:] - ptr[:-1]
        rank = (degree <= 128 * slots).to(torch.uint8) + (degree <= 32 * slots).to(torch.uint8)
        order = torch.sort(rank, stable=True).indices.to(torch.int32)
        counts = torch.stack([(rank == c).sum() for c in range(3)]).tolist()
        self._kept.append(_native.Made(order))
        return order, (ctypes.c_int64 * 3)(*counts)

    def found(self) -> None:
        """The current stream reads what is kept from here on."""
        here = _native.stream_handle(self.device)
        for made in self._kept:
            if made.handle != here:
                made.found()


_LOG2E = 1.0 / math.log(2.0)
_WORD = {torch.float32: torch.int32, torch.float64: torch.int64}


def _outside_capture(t: Tensor, what: str) -> None:
    if t.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError(f"{what} waits for the device: build it before the capture.")


class Maps:
    """The rows' ``2 heads`` maps of ``map_type`` as the entry points take them."""

    def __init__(self, map_type: SO2FieldType, heads: int) -> None:
        if not isinstance(map_type, SO2FieldType):
            raise TypeError(f"map_type must be an SO2FieldType, got {type(map_type).__name__}.")
        if not 1 <= heads <= MAX_H:
            raise ValueError(f"heads must lie in 1..{MAX_H}, got {heads}.")
        full = map_type.scaled(2 * heads)
        if len(map_type) > MAX_F or full.dimension > MAX_D:
            raise ValueError(f"the maps must hold at most {MAX_F} frequencies and {MAX_D} numbers a row, "
                             f"got {full!r} ({full.dimension}).")
        self.heads, self.scale = heads, 1.0 / math.sqrt(map_type.dimension)
        self.plan = fused_attention.plan_of(map_type, full, 2 * heads)
        self.top = max(n for n, *_ in self.plan.rows)
        # read on the host, whatever the default device of the call that makes the (kept) maps
        self.desc = torch.tensor([list(row) for row in self.plan.rows], dtype=torch.int64, device="cpu")
        self._slots: dict[int, int] = {}

    def slots(self, tables: EdgeTables) -> int:
        """Edge slots of a wave of the lane kernels (0: the simple kernels serve)."""
        if tables.dtype == torch.float64:
            return 0
        held = self._slots.get(tables.orders)
        if held is None:
            held = self._slots[tables.orders] = _native.differential_slots(self.desc, self.plan.width, tables.orders,
                                                                           self.heads)
        return held


maps_of = functools.lru_cache(maxsize=256)(Maps)


class DifferentialSoftmax(torch.autograd.Function):
    """``alpha (n_edges, H)`` from the maps' rows and ``lam (H,)``; ``dq``, ``dk``
    in the rows' dtype and ``dlam`` back."""

    @staticmethod
    def forward(ctx: Any, q: Tensor, k: Tensor, lam: Tensor, tables: EdgeTables, maps: Maps, scale: float,
                train: bool) -> Tensor:
        if train:  # found here: the backward runs on a thread and perhaps a stream of its own
            tables.group_sources()
            tables.source_rows(maps.slots(tables))
        with _native.span("gm::attention/differential_softmax"):
            alpha, stats = _native.differential_forward(q, k, lam, tables, maps, scale, train)
        if train:
            ctx.save_for_backward(q, k, lam, stats)
            ctx.rest = (tables, maps, scale)
        return alpha

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, grad_alpha: Tensor) -> tuple:
        q, k, lam, stats = ctx.saved_tensors
        with _native.span("gm::attention/differential_softmax_backward"):
            dq, dk, dlam = _native.differential_backward(grad_alpha.contiguous(), q, k, lam, stats, *ctx.rest)
        return dq, dk, dlam, None, None, None, None


def differential_softmax(q: Tensor, k: Tensor, lam: Tensor, tables: EdgeTables, map_type: SO2FieldType, heads: int,
                         scale: float | None = None) -> Tensor:
    """The heads' attention weights ``(n_edges, heads)`` of ``q (n_targets, D)`` and
    ``k (n_sources, D)``, rows of ``2 heads`` maps of ``map_type``, under ``lam
    (heads,)``; ``scale`` is ``1 / sqrt(dim map_type)`` by default."""
    maps = maps_of(map_type, heads)
    width = maps.plan.width
    table = torch.float32 if q.dtype == torch.bfloat16 else q.dtype
    if table != tables.dtype or k.dtype != q.dtype:
        raise ValueError(f"q and k must share a dtype, {tables.dtype} (or bfloat16 with float32 tables), "
                         f"got {q.dtype} and {k.dtype}.")
    if tuple(q.shape) != (tables.n_targets, width) or tuple(k.shape) != (tables.n_sources, width):
        raise ValueError(f"q and k must be ({tables.n_targets}, {width}) and ({tables.n_sources}, {width}), "
                         f"got {tuple(q.shape)} and {tuple(k.shape)}.")
    if tuple(lam.shape) != (heads,):
        raise ValueError(f"lam must be ({heads},), got {tuple(lam.shape)}.")
    if any(t.device != tables.device for t in (q, k, lam)):
        raise ValueError("q, k and lam must live on the tables' device.")
    if maps.top >= tables.orders:
        raise ValueError(f"the tables hold orders below {tables.orders}, the maps need {maps.top}.")
    scale = maps.scale if scale is None else float(scale)
    if q.device.type != "cuda":
        return _eager(q, k, lam, tables, maps.plan, scale)
    # whether a backward can follow: inside the op a parameter looks the same under no_grad
    train = torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or lam.requires_grad)
    return DifferentialSoftmax.apply(_whole(q), _whole(k), lam.to(table).contiguous(), tables, maps, scale, train)


def enabled(mhsa: Any, x: Any, edges: Any) -> bool:
    """Whether a differential layer's scores take the fused op on the GPU."""
    if fused_attention.MODE == "0" or x.device.type != "cuda" or edges.n_edges == 0:
        return False
    if x.dtype not in (torch.float32, torch.float64, torch.bfloat16) or mhsa.num_heads > MAX_H:
        return False
    maps = mhsa.field_type_map
    return (len(maps) <= MAX_F and mhsa.field_type_in.dimension <= MAX_D
            and maps.max_frequency <= edges.max_frequency)


class _Kind(NamedTuple):
    """Which tables of an edge set: their name among what is kept of its geometry, and how
    they are made of a geometry and the CSR ``(row_ptr, source)`` over ``n_sources`` rows."""

    name: tuple
    make: Callable[..., EdgeTables]


def _kind(top: int) -> _Kind:
    return _Kind((top,), lambda g, row_ptr, source, n_sources: EdgeTables(
        row_ptr, source, g.transport[:, : top + 1], g.bias, g.inside, n_sources=n_sources))


def edge_tables(edges: Any, cutoff: float, window: str, dtype: torch.dtype, top: int,
                kind: _Kind | None = None) -> EdgeTables:
    """The tables of ``edges`` under a cutoff and window, with the transport's orders
    up to ``top``: built once and kept with the edge set's geometry."""
    kind = _kind(top) if kind is None else kind
    g = fused_attention.geometry(edges, cutoff, window, dtype)
    key = ("differential", *kind.name)
    held = g.derived.get(key)
    if held is None:
        with _native.LOCK:
            held = g.derived.get(key)
            if held is None:
                held = g.derived[key] = kind.make(g, g.row_ptr, g.source, None)
    return held


class _Ranges:
    """The tables of an edge set's chunks, ``{(e0, e1): (tables, first target, first source)}``:
    the ranges found last, up to ``limit`` edges of them.  A range that a captured graph
    reads stays."""

    def __init__(self, limit: int) -> None:
        self.limit, self.edges = limit, 0
        self.held: OrderedDict[tuple[int, int], tuple[EdgeTables, int, int]] = OrderedDict()
        self.captured: dict[tuple[int, int], tuple[EdgeTables, int, int]] = {}

    def find(self, span: tuple[int, int]) -> tuple[EdgeTables, int, int] | None:
        with _native.LOCK:
            found = self.captured.get(span)
            if found is None and (found := self.held.get(span)) is not None:
                if found[0].device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                    self.captured[span] = self.held.pop(span)
                    self.edges -= found[0].n_edges
                else:
                    self.held.move_to_end(span)
            return found

    def keep(self, span: tuple[int, int], made: tuple[EdgeTables, int, int]) -> tuple[EdgeTables, int, int]:
        with _native.LOCK:
            found = self.find(span)
            if found is not None:  # another thread was first
                return found
            self.held[span] = made
            self.edges += made[0].n_edges
            while self.edges > self.limit:
                self.edges -= self.held.popitem(last=False)[1][0].n_edges
            return made


def chunk_tables(chunk: Any, cutoff: float, window: str, dtype: torch.dtype, top: int,
                 kind: _Kind | None = None) -> tuple[EdgeTables, int, int]:
    """The tables of a chunk (``EdgeGeometry.chunks``) over its own targets and the range of
    nodes its sources lie in, and the first of each.  Chunks are made anew for every pass:
    the tables are kept with the edge set they are ranges of, as many as two passes over all
    of its edges take, where a range's lists of nodes take no more than its edges (a chunk
    with sources all over a large set keeps its own)."""
    kind = _kind(top) if kind is None else kind
    parent, e0, e1 = fused_attention.chunk_of(chunk)
    outer = fused_attention.geometry(parent, cutoff, window, dtype)
    ranges = outer.derived.get(("differential ranges", *kind.name))
    if ranges is None:
        with _native.LOCK:
            ranges = outer.derived.setdefault(("differential ranges", *kind.name), _Ranges(2 * int(parent.n_edges)))
    # an edge set registered as a chunk under numbers of its own is not the range of its span
    same = (chunk.edge_index.data_ptr() == parent.edge_index[:, e0:].data_ptr()
            and chunk.row_ptr.shape == parent.row_ptr.shape)
    found = ranges.find((e0, e1)) if same else None
    if found is not None:
        return found
    g = fused_attention.geometry(chunk, cutoff, window, dtype)
    found = g.derived.get(("differential range", *kind.name))
    if found is not None:
        return found
    _outside_capture(g.row_ptr, "EdgeTables")
    ptr, begin = (outer.host_row_ptr(), e0) if same else (g.host_row_ptr(), 0)
    first = int(np.searchsorted(ptr, begin, side="right")) - 1
    last = int(np.searchsorted(ptr, begin + e1 - e0, side="left"))
    source, behind = int(g.source.min()), int(g.source.max()) + 1
    made = kind.make(g, g.row_ptr[first:last + 1], g.source - source, behind - source), first, source
    # 12 bytes a node of either list, 24 and 32 an edge at two orders
    if same and made[0].n_targets + made[0].n_sources <= 4 * (e1 - e0):
        return ranges.keep((e0, e1), made)
    with _native.LOCK:
        return g.derived.setdefault(("differential range", *kind.name), made)


def attention_weights(mhsa: Any, q: Tensor, k: Tensor, edges: Any) -> Tensor:
    """A differential layer's weights ``(n_edges, n_heads)`` from its flat query and
    key rows: the fused op where it serves, else the single softmax's eager
    arithmetic over the ``2 n_heads`` maps and their difference."""
    lam, maps = mhsa.lambdas(), mhsa.field_type_map
    window = mhsa.heads[0].window
    if enabled(mhsa, q, edges):
        table = torch.float32 if q.dtype == torch.bfloat16 else q.dtype
        if fused_attention.chunk_of(edges) is not None:
            tables, first, source = chunk_tables(edges, mhsa.cutoff, window, table, maps.max_frequency)
            q, k = q[first:first + tables.n_targets], k[source:source + tables.n_sources]
        else:
            tables = edge_tables(edges, mhsa.cutoff, window, table, maps.max_frequency)
        return differential_softmax(q, k, lam, tables, maps, mhsa.num_heads)
    plan = fused_attention.plan_of(maps, mhsa.field_type_in, 2 * mhsa.num_heads)  # of any size, unlike the op's
    weights = fused_attention.softmax_eager(plan, q, k, edges, mhsa.cutoff, window, 1.0 / math.sqrt(maps.dimension))
    return weights[:, 0::2] - lam.to(weights.dtype) * weights[:, 1::2]


def _whole(rows: Tensor) -> Tensor:
    """Contiguous rows at a multiple of 16 bytes, as the lane kernels load them."""
    rows = rows.contiguous()
    return rows if rows.data_ptr() % 16 == 0 else rows.clone()


def torch_weights(q: Tensor, k: Tensor, row_ptr: Tensor, source: Tensor, phases: Tensor, bias: Tensor,
                  plan: fused_attention.Plan, scale: float, learned: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """``(weights, none)``, both ``(n_edges, plan.heads)``: the softmax of every head (or map) in torch, in the
    arithmetic of ``bias (n_edges,)`` (``-inf`` outside the window), ``learned (n_edges, plan.heads)`` added to the
    scores; ``none`` marks the weights of zero, whose edges count for nothing in a gradient.

    An edge outside the window, or of a score of -inf, has weight zero in any row: one whose other scores are not
    numbers too."""
    n, heads, dtype = row_ptr.shape[0] - 1, plan.heads, bias.dtype
    target = torch.repeat_interleave(torch.arange(n, device=q.device), row_ptr[1:] - row_ptr[:-1])
    # an edge outside the window reads nothing: its row may hold anything
    outside = (bias == -math.inf).unsqueeze(-1)
    qe = q.to(dtype).index_select(0, target).masked_fill(outside, 0.0)
    ke = k.to(dtype).index_select(0, source).masked_fill(outside, 0.0)
    score = 0.0
    for f, a, off, _, dim in plan.rows:
        block = slice(off, off + heads * a * dim)
        if f == 0:
            score = score + (qe[:, block] * ke[:, block]).reshape(-1, heads, a).sum(-1)
        else:
            qr, qi = qe[:, block].reshape(-1, heads, a, 2).unbind(-1)
            kr, ki = ke[:, block].reshape(-1, heads, a, 2).unbind(-1)
            cos, sin = phases[:, 2 * f - 2, None], phases[:, 2 * f - 1, None]
            score = score + cos * (qr * kr + qi * ki).sum(-1) + sin * (qi * kr - qr * ki).sum(-1)
    score = scale * score + (bias.unsqueeze(-1) if learned is None else bias.unsqueeze(-1) + learned)
    out = outside | (score == -math.inf)
    index = target.unsqueeze(-1).expand(-1, heads)
    top = score.new_full((n, heads), -math.inf).scatter_reduce(0, index, score.detach().masked_fill(out, -math.inf),
                                                               "amax")
    weight = torch.exp(score - top.masked_fill(top == -math.inf, 0.0).index_select(0, target)).masked_fill(out, 0.0)
    total = score.new_zeros(n, heads).index_add(0, target, weight)
    weight = weight / total.masked_fill(total == 0, 1.0).index_select(0, target)
    none = out | (weight == 0)

    # a factor of zero is not enough where the other one is infinite or no number (no gradient: undefined, or a second
    # derivative's that does not depend on it)
    def over_scores(g: Tensor | None) -> Tensor | None:
        return None if g is None else g.masked_fill(none, 0.0)

    def over_rows(g: Tensor | None) -> Tensor | None:
        if g is None:
            return None
        return g.masked_fill(torch.cat([none.repeat_interleave(a * dim, 1) for _, a, _, _, dim in plan.rows], 1), 0.0)

    for t, kept in ((score, over_scores), (qe, over_rows), (ke, over_rows)):
        if t.requires_grad:
            t.register_hook(kept)
    return weight.masked_fill(none, 0.0), none


def _eager(q: Tensor, k: Tensor, lam: Tensor, tables: EdgeTables, plan: fused_attention.Plan, scale: float) -> Tensor:
    """The formulas in torch, in the tables' arithmetic."""
    weight, none = torch_weights(q, k, tables.row_ptr, tables._source, tables._phases, tables._bias, plan, scale)
    alpha = weight[:, 0::2] - lam.to(tables.dtype) * weight[:, 1::2]
    return alpha.masked_fill(none[:, 0::2] & none[:, 1::2], 0.0)
