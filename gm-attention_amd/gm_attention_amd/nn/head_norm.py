"""The norm and rotation of query and key rows, head by head, in one pass.

For every head's numbers ``x`` of a row (P of them, every frequency's together),

    xhat = x / sqrt(mean x^2 + eps),
    y    = exp(i theta) (gain xhat),

with one learned gain a copy of the head type (the same for every head) and an
angle a complex copy that is linear in the row's node's position,

    theta(node, slot) = sum_axis positions(node, axis) frequencies(axis, slot).

A copy of a frequency above zero turns as the complex number it is; copies of
frequency zero turn in pairs, a last odd one stays.  The norm sees only the sizes
of copies and a common phase of a copy commutes with any turn of the frames, so
both are gauge equivariant; the scores of rotated queries and keys depend on the
nodes' positions through their differences alone.  Positions are whatever scalars a
node has (latitude, height, time; longitude with whole frequencies).

A head's slots are, in order, its pairs of frequency-0 copies (``a_0 // 2``) and
then every copy of the frequencies above.  Angles are formed in 64 bits from the
positions and frequencies, which are constants to autograd.

On the GPU (``gm_head_norm_*``) both sets of rows take one pass each way; rows may
be strided views (of one product's output).  bfloat16 rows take float32 gains and
arithmetic and are rounded once.  CPU tensors, and rows beyond the kernel's bounds,
take the formulas in torch.
"""

from __future__ import annotations

import functools
from collections.abc import Sequence
from typing import Any

import torch
from torch import Tensor, nn

from gm_attention_amd import _native
from gm_attention_amd.nn import fused_attention
from gm_attention_amd.representations.field_type import SO2FeatureField, SO2FieldType

MAX_HEADS, MAX_F, MAX_D, MAX_AXES = 64, fused_attention.MAX_F, fused_attention.MAX_D, 8


class HeadRows:
    """Rows of ``heads`` heads of ``head_type``: a head's ``copies``, ``slots`` and numbers."""

    def __init__(self, head_type: SO2FieldType, heads: int) -> None:
        if heads < 1:
            raise ValueError(f"heads must be at least 1, got {heads}.")
        self.heads, self.width, self.numbers = heads, heads * head_type.dimension, head_type.dimension
        self.copies = sum(a for _, a in head_type.items())
        self.pairs = head_type.multiplicity(0) // 2 if 0 in head_type else 0
        self.slots = self.pairs + sum(a for f, a in head_type.items() if f)
        self.plan = fused_attention.plan_of(head_type, head_type.scaled(heads), heads)
        # read on the host, whatever the default device of the call that makes the (kept) rows
        self.desc = torch.tensor([list(row) for row in self.plan.rows], dtype=torch.int64, device="cpu")
        self.serves = heads <= MAX_HEADS and len(head_type) <= MAX_F and self.width <= MAX_D


rows_of = functools.lru_cache(maxsize=256)(HeadRows)


def rotary_frequencies(head_type: SO2FieldType, highest: Sequence[float], lowest: Sequence[float],
                       whole: Sequence[bool] | None = None) -> Tensor:
    """Frequencies ``(axes, slots)`` in radians a unit of each axis: the slots are dealt to
    the axes in turn, an axis's from its ``highest`` down to its ``lowest`` in equal
    ratios, rounded to whole numbers (one at least) on a periodic axis (``whole``)."""
    axes = len(highest)
    if not axes or len(lowest) != axes or (whole is not None and len(whole) != axes):
        raise ValueError("highest, lowest and whole hold a value an axis.")
    if any(not (0 < lo <= hi) for lo, hi in zip(lowest, highest)):
        raise ValueError(f"every axis needs 0 < lowest <= highest, got {lowest} and {highest}.")
    slots = rows_of(head_type, 1).slots
    out = torch.zeros(axes, slots, dtype=torch.float64)
    for axis in range(axes):
        mine = range(axis, slots, axes)
        for j, slot in enumerate(mine):
            ratio = (lowest[axis] / highest[axis]) ** (j / max(1, len(mine) - 1))
            value = highest[axis] * ratio
            out[axis, slot] = max(1.0, round(value)) if whole is not None and whole[axis] else value
    return out


class HeadNormOp(torch.autograd.Function):
    """The sets' outputs from ``sets`` rows and then their gains (None: ones)."""

    @staticmethod
    def forward(ctx: Any, layout: HeadRows, eps: float | None, positions: Tensor | None, frequencies: Tensor | None,
                train: bool, sets: int, *given: Tensor | None):
        ctx.set_materialize_grads(False)
        rows, gains = given[:sets], given[sets:]
        with _native.span("gm::pointwise/head_norm"):
            out = _native.head_norm_forward(rows, gains, layout, eps, positions, frequencies)
        if train:
            ctx.save_for_backward(positions, frequencies, *given)
            ctx.rest = (layout, eps)
        return tuple(out)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx: Any, *grads: Tensor | None):
        positions, frequencies, *given = ctx.saved_tensors
        layout, eps = ctx.rest
        sets = len(grads)
        need = ctx.needs_input_grad[6:]
        mine = [i for i in range(sets) if grads[i] is not None and (need[i] or need[sets + i])]
        out: list[Tensor | None] = [None] * (2 * sets)
        if mine:
            with _native.span("gm::pointwise/head_norm_backward"):
                dx, dgain = _native.head_norm_backward(
                    [grads[i].contiguous() for i in mine], [given[i] for i in mine], [given[sets + i] for i in mine],
                    layout, eps, positions, frequencies, any(need[sets + i] for i in mine))
            for at, i in enumerate(mine):
                out[i] = dx[at]
                out[sets + i] = dgain[at] if need[sets + i] else None
        return (None,) * 6 + tuple(out)


def head_norm(rows: Tensor, head_type: SO2FieldType, heads: int, gain: Tensor | None = None, *,
              eps: float | None = 1e-6, positions: Tensor | None = None,
              frequencies: Tensor | None = None) -> Tensor:
    """``rows (N, D)`` of ``heads`` heads of ``head_type`` normalised head by head (not with
    ``eps`` None), multiplied by ``gain (copies,)`` and turned by the angles of ``positions
    (N, axes)`` and ``frequencies (axes, slots)`` (not without them)."""
    return _run([rows], [gain], head_type, heads, eps, positions, frequencies)[0]


def query_key_norm(q: Tensor, k: Tensor, head_type: SO2FieldType, heads: int, q_gain: Tensor | None = None,
                   k_gain: Tensor | None = None, *, eps: float | None = 1e-6, positions: Tensor | None = None,
                   frequencies: Tensor | None = None) -> tuple[Tensor, Tensor]:
    """:func:`head_norm` of the queries and keys ``(N, D)`` of one node set, in one pass: the
    angles are formed once for both.  (Rows of different node sets take :func:`head_norm`.)"""
    if k.shape != q.shape or k.dtype != q.dtype or k.device != q.device:
        raise ValueError(f"q and k must share a shape, dtype and device, got {tuple(q.shape)} {q.dtype} on {q.device} "
                         f"and {tuple(k.shape)} {k.dtype} on {k.device}.")
    q, k = _run([q, k], [q_gain, k_gain], head_type, heads, eps, positions, frequencies)
    return q, k


def _run(rows: list[Tensor], gains: list[Tensor | None], head_type: SO2FieldType, heads: int, eps: float | None,
         positions: Tensor | None, frequencies: Tensor | None) -> Sequence[Tensor]:
    if not isinstance(head_type, SO2FieldType):
        raise TypeError(f"head_type must be an SO2FieldType, got {type(head_type).__name__}.")
    layout, first = rows_of(head_type, heads), rows[0]
    dtype, device = first.dtype, first.device
    if dtype not in (torch.float32, torch.float64, torch.bfloat16):
        raise ValueError(f"rows must be float32, float64 or bfloat16, got {dtype}.")
    if first.ndim != 2 or first.shape[1] != layout.width:
        raise ValueError(f"rows must be (N, {layout.width}), got {tuple(first.shape)}.")
    if eps is not None and not eps > 0.0:
        raise ValueError(f"eps must be positive (None: no norm), got {eps}.")
    if (positions is None) != (frequencies is None):
        raise ValueError("positions and frequencies go together.")
    if eps is None and positions is None and all(g is None for g in gains):
        raise ValueError("nothing to do: neither a norm nor gains nor positions.")
    if positions is not None and frequencies is not None:
        axes = frequencies.shape[0] if frequencies.ndim else 0
        if tuple(frequencies.shape) != (axes, layout.slots) or not 1 <= axes <= MAX_AXES:
            raise ValueError(f"frequencies must be (axes, {layout.slots}) of 1..{MAX_AXES} axes, "
                             f"got {tuple(frequencies.shape)}.")
        if tuple(positions.shape) != (first.shape[0], axes):
            raise ValueError(f"positions must be ({first.shape[0]}, {axes}), got {tuple(positions.shape)}.")
        if positions.is_complex() or frequencies.is_complex():
            raise ValueError("positions and frequencies must be real.")
        if positions.device != device or frequencies.device != device:
            raise ValueError(f"positions and frequencies must live on the rows' device, {device}.")
        if positions.requires_grad or frequencies.requires_grad:
            raise ValueError("positions and frequencies are constants: they get no gradient here.")
        positions, frequencies = positions.double().contiguous(), frequencies.double().contiguous()
    pd = _native.param_dtype(dtype)
    for i, g in enumerate(gains):
        if g is None:
            continue
        if tuple(g.shape) != (layout.copies,) or not g.is_floating_point() or g.device != device:
            raise ValueError(f"a gain must be ({layout.copies},) real numbers on {device}, "
                             f"got {tuple(g.shape)} of {g.dtype} on {g.device}.")
        gains[i] = g if g.dtype == pd and g.is_contiguous() else g.to(pd).contiguous()
    if device.type != "cuda" or not layout.serves:
        return [_eager(x, g, layout, eps, positions, frequencies) for x, g in zip(rows, gains)]
    # whether a backward can follow: inside the op a parameter looks the same under no_grad
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (*rows, *gains))
    return HeadNormOp.apply(layout, eps, positions, frequencies, train, len(rows), *map(_rows, rows), *gains)


def _rows(x: Tensor) -> Tensor:
    """Rows as the kernel reads them: each row's numbers side by side, rows apart."""
    n, width = x.shape
    if (width == 1 or x.stride(1) == 1) and (n <= 1 or x.stride(0) >= width):
        return x
    return x.contiguous()


def _eager(x: Tensor, gain: Tensor | None, layout: HeadRows, eps: float | None, positions: Tensor | None,
           frequencies: Tensor | None) -> Tensor:
    """The formulas in torch, in the parameters' arithmetic."""
    v = x.to(_native.param_dtype(x.dtype))
    n, heads = x.shape[0], layout.heads
    blocks = [v[:, off:off + heads * a * dim].reshape(n, heads, a, dim) for _, a, off, _, dim in layout.plan.rows]
    if eps is not None:  # in 64 bits: squares and their sums, forward and back, pass 32 bits' range
        wide = [b.double() for b in blocks]
        mean = sum(b.square().sum((2, 3)) for b in wide) / layout.numbers
        inv = torch.rsqrt(mean + eps)[:, :, None, None]
        blocks = [(b * inv).to(v.dtype) for b in wide]
    if gain is not None:
        at = gain.split([a for _, a, *_ in layout.plan.rows])
        blocks = [b * g[None, None, :, None] for b, g in zip(blocks, at)]
    if positions is not None and frequencies is not None:
        theta = positions @ frequencies
        cos, sin = torch.cos(theta).to(v.dtype), torch.sin(theta).to(v.dtype)
        slot, turned = 0, []
        for (f, a, *_), b in zip(layout.plan.rows, blocks):
            count = a if f else a // 2
            pairs = b if f else b[:, :, :2 * count].reshape(n, heads, count, 2)
            c, s = cos[:, None, slot:slot + count], sin[:, None, slot:slot + count]
            re, im = pairs.unbind(-1)
            out = torch.stack([c * re - s * im, c * im + s * re], dim=-1)
            turned.append(out if f else torch.cat([out.reshape(n, heads, 2 * count, 1), b[:, :, 2 * count:]], dim=2))
            slot += count
        blocks = turned
    return torch.cat([b.flatten(1) for b in blocks], dim=1).to(x.dtype)


class SO2QueryKeyNorm(nn.Module):
    """The norm, gains and rotation of an attention layer's queries and keys: ``norm`` and
    ``gain`` leave their part out, ``frequencies (axes, slots)`` (radians a unit of each
    axis, e.g. from :func:`rotary_frequencies`) turn the rows by their nodes' positions.

    The frequencies are part of the construction, kept in 64 bits whatever the module is
    cast to; they are not in its state.  A device's copy is made by the first call there,
    which a captured step needs to have been made before the capture."""

    def __init__(self, head_type: SO2FieldType, heads: int, *, eps: float = 1e-6, norm: bool = True,
                 gain: bool = True, frequencies: Tensor | Sequence[Sequence[float]] | None = None, dtype=None,
                 device=None) -> None:
        super().__init__()
        if not isinstance(head_type, SO2FieldType):
            raise TypeError(f"head_type must be an SO2FieldType, got {type(head_type).__name__}.")
        if not (eps > 0.0):
            raise ValueError(f"eps must be positive, got {eps}.")
        layout = rows_of(head_type, heads)
        self.head_type, self.heads = head_type, heads
        self.eps = float(eps) if norm else None
        if frequencies is None:
            self.frequencies = None
        else:
            held = torch.as_tensor(frequencies, dtype=torch.float64, device="cpu").detach()
            if held.ndim != 2 or held.shape[1] != layout.slots or not 1 <= held.shape[0] <= MAX_AXES:
                raise ValueError(f"frequencies must be (axes, {layout.slots}) of 1..{MAX_AXES} axes, "
                                 f"got {tuple(held.shape)}.")
            self.frequencies = tuple(map(tuple, held.tolist()))
        if not norm and not gain and frequencies is None:
            raise ValueError("nothing to do: neither a norm nor gains nor frequencies.")
        for name in ("query_gain", "key_gain"):
            self.register_parameter(name, nn.Parameter(torch.empty(layout.copies, dtype=dtype, device=device))
                                    if gain else None)
        self.reset_parameters()

    def reset_parameters(self) -> None:
        for p in self.parameters():
            nn.init.ones_(p)

    def _on(self, device: torch.device) -> Tensor | None:
        if self.frequencies is None:
            return None
        key = f"_frequencies {device}"
        held = self.__dict__.get(key)
        if held is None:
            if device.type == "cuda" and torch.cuda.is_current_stream_capturing():
                raise RuntimeError("the first call of an SO2QueryKeyNorm on a device waits for the device: make it "
                                   "before the capture.")
            with torch.inference_mode(False):  # a later step may train
                held = torch.tensor(self.frequencies, dtype=torch.float64, device=device)
            _native.complete(held.device)  # other streams and threads find it unchecked
            self.__dict__[key] = held
        return held

    def __getstate__(self) -> dict:
        return {n: v for n, v in self.__dict__.items() if not n.startswith("_frequencies ")}

    def forward_flat(self, q: Tensor, k: Tensor, positions: Tensor | None = None) -> tuple[Tensor, Tensor]:
        """Query and key rows ``(N, D)`` of one node set, with its ``positions (N, axes)``."""
        if (positions is None) != (self.frequencies is None):
            raise ValueError("positions must be given exactly where there are frequencies.")
        return query_key_norm(q, k, self.head_type, self.heads, self.query_gain, self.key_gain, eps=self.eps,
                              positions=positions, frequencies=self._on(q.device))

    def forward(self, q: SO2FeatureField, k: SO2FeatureField,
                positions: Tensor | None = None) -> tuple[SO2FeatureField, SO2FeatureField]:
        """The same of fields of the heads side by side (``head_type.scaled(heads)``), with positions a node."""
        full = self.head_type.scaled(self.heads)
        for given in (q, k):
            if given.field_type != full:
                raise ValueError(f"Expected a field of type {full!r}, got {given.field_type!r}.")
        rows, keys = q._rows(), k._rows()
        batch = rows.shape[:-1]
        if keys.shape != rows.shape:
            raise ValueError(f"q and k must be fields on the same nodes, got {tuple(batch)} "
                             f"and {tuple(keys.shape[:-1])}.")
        if positions is not None:
            if positions.shape[:-1] != batch:
                raise ValueError(f"positions must be ({', '.join(map(str, batch))}, axes), "
                                 f"got {tuple(positions.shape)}.")
            positions = positions.reshape(-1, positions.shape[-1])
        out = self.forward_flat(rows.reshape(-1, rows.shape[-1]), keys.reshape(-1, rows.shape[-1]), positions)
        turned_q, turned_k = (SO2FeatureField.from_flat(full, t.reshape(*batch, -1)) for t in out)
        return turned_q, turned_k

    def extra_repr(self) -> str:
        axes = 0 if self.frequencies is None else len(self.frequencies)
        return (f"head_type={self.head_type!r}, heads={self.heads}, eps={self.eps}, "
                f"gain={self.query_gain is not None}, axes={axes}")
