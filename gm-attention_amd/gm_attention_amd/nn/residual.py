"""``SO2ResidualNorm``: the residual sum between two sub-layers, with their norms.

A block that normalises before and after its sub-layers (the mixer, the
feed-forward) joins a sub-layer's output ``u`` to its rows ``x`` by

    x' = x + s * act(z) * (gamma_p * norm(u) + beta_p),
    h  = gamma_n * norm(x') + beta_n,

``norm`` the merged equivariant normalisation of :class:`SO2LayerNorm`, ``s`` one
learned scale a copy, ``act(z)`` one gate a copy (``sigmoid``, or ``2 sigmoid``,
which is one at zero) from pre-activations affine in the sub-layer's scalar
inputs, and ``h`` the next sub-layer's input.  Scales and gates multiply both
coordinates of a copy, so the sum is as equivariant as its parts.  Any of the
branch's norm, the gate, the scale and the next norm may be left out.

On the GPU the sum and both norms are one HIP pass each way over flat rows
(``gm_residual_norm_*``; parameter gradients reduced in a fixed order) for
float32, float64 and bfloat16 rows; bfloat16 rows keep float32 parameters and
arithmetic, take a branch in bfloat16 or float32 (the gates' pre-activations in
the rows' type), and are rounded once: ``h`` is normalised from the sum before
its rounding.  CPU tensors take the same
formulas in torch.
"""

from __future__ import annotations

from typing import Literal

import torch
from torch import Tensor, nn

from gm_attention_amd import _native
from gm_attention_amd.nn.linear import FlatLinear
from gm_attention_amd.nn.normalization import MAX_WIDTH, SO2LayerNorm
from gm_attention_amd.representations.field_type import SO2FeatureField, SO2FieldType

GateKind = Literal["sigmoid", "double_sigmoid"]
_GATES = {"sigmoid": 1.0, "double_sigmoid": 2.0}


class ResidualNormOp(torch.autograd.Function):
    """``(x', h)`` (``x'`` alone without a next norm) from the rows, the branch, the
    gates' pre-activations and the parameters, a vector a frequency; ``counts``
    how many of ``params`` each group has (the branch's gains and offset, the
    scales, the next norm's gains and offset), zero for a group left out;
    ``train`` whether a backward can follow."""

    @staticmethod
    def forward(ctx, x: Tensor, u: Tensor, z: Tensor | None, layout, factor: float, eps: float, next_eps: float,
                counts: tuple[int, ...], train: bool, *params: Tensor):
        ctx.set_materialize_grads(False)
        with _native.span("gm::pointwise/residual_norm"):
            y, normed, stats = _native.residual_norm_forward(x, u, z, counts, params, layout, factor, eps, next_eps,
                                                             train)
        if train:
            ctx.save_for_backward(x, u, z, stats, *params)
            ctx.rest = (layout, factor, counts)
        return y if normed is None else (y, normed)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy: Tensor | None, dn: Tensor | None = None):
        x, u, z, stats, *params = ctx.saved_tensors
        if dy is None and dn is None:
            return (None,) * len(ctx.needs_input_grad)
        layout, factor, counts = ctx.rest
        with _native.span("gm::pointwise/residual_norm_backward"):
            dx, du, dz, dparams = _native.residual_norm_backward(
                None if dy is None else dy.contiguous(), None if dn is None else dn.contiguous(), x, u, z, counts,
                params, stats, layout, factor)
        # dparams: the groups' gradients in order, a left-out group's too
        copies, sizes, held = layout.a0 + layout.G, [], []
        lengths = iter(layout.parameter_slots(counts)[2])
        for group, count in enumerate(counts):
            sizes += [next(lengths) for _ in range(count)] if count else [layout.a0 if group in (1, 4) else copies]
            held += [True] * count or [False]
        return (dx, du, dz, None, None, None, None, None, None,
                *(g for g, h in zip(dparams.split(sizes), held, strict=True) if h))


def _by_key(held: nn.ParameterDict, keys: list[str]) -> list[Tensor]:
    """A dictionary's vectors under ``keys`` (its own order is its keys' as texts, 10 before 2)."""
    own = held._parameters
    if all(k in own for k in keys):
        return [own[k] for k in keys]
    return [held[k] for k in keys]  # a replica's are plain attributes, a pruned or parametrised one's is computed


class SO2ResidualNorm(nn.Module):
    """The residual sum of ``field_type`` rows: ``post_norm`` normalises the
    branch, ``gate`` names its gates' activation, ``scale`` is the scales' initial
    value, ``norm`` normalises behind the sum (each left out by False or None)."""

    def __init__(self, field_type: SO2FieldType, *, eps: float = 1e-5, bias: bool = True, post_norm: bool = True,
                 gate: GateKind | None = None, scale: float | None = None, norm: bool = True, dtype=None,
                 device=None) -> None:
        super().__init__()
        if not isinstance(field_type, SO2FieldType):
            raise TypeError(f"field_type must be an SO2FieldType, got {type(field_type).__name__}.")
        if not (eps > 0.0):
            raise ValueError(f"eps must be positive, got {eps}.")
        if gate is not None and gate not in _GATES:
            raise ValueError(f"gate must be None or one of {tuple(_GATES)}, got {gate!r}.")
        self.field_type = field_type
        self.gate = gate
        self.width, self.copies = field_type.dimension, sum(m for _, m in field_type.items())
        kw = dict(dtype=dtype, device=device)
        self.post = SO2LayerNorm(field_type, eps=eps, bias=bias, **kw) if post_norm else None
        self.norm = SO2LayerNorm(field_type, eps=eps, bias=bias, **kw) if norm else None
        self.initial_scale = None if scale is None else float(scale)
        self.scale = None if scale is None else nn.ParameterDict({
            str(f): nn.Parameter(torch.full((m,), float(scale), **kw)) for f, m in field_type.items()})
        # the gates read the sub-layer's scalars; a field without any takes its pre-activations from the caller
        self.gate_linear = (nn.Linear(field_type.multiplicity(0), self.copies, **kw)
                            if gate is not None and 0 in field_type else None)

    def reset_parameters(self) -> None:
        for norm in (self.post, self.norm):
            if norm is not None:
                norm.reset_parameters()
        if self.scale is not None:
            for p in self.scale.values():
                nn.init.constant_(p, self.initial_scale)
        if self.gate_linear is not None:
            self.gate_linear.reset_parameters()

    def pre_activations(self, scalars: Tensor) -> Tensor:
        """The gates' pre-activations ``(N, copies)`` from scalars ``(N, a_0)``: one product."""
        if self.gate_linear is None:
            raise ValueError("pre_activations needs a gate and frequency-0 channels to condition it on, "
                             f"but got gate={self.gate!r} and {self.field_type!r}.")
        return FlatLinear.apply(scalars, self.gate_linear.weight.t(), self.gate_linear.bias)

    def _layout(self):
        layout = self.__dict__.get("_pw_layout")
        if layout is None:
            layout = _native.PointwiseLayout(self.field_type)
            self.__dict__["_pw_layout"] = layout
        return layout

    def _params(self) -> tuple[tuple[int, ...], list[Tensor]]:
        """``(counts, params)`` as the op takes them: every group's vectors by frequency, a
        group left out where the module was made without it."""
        post, norm, keys = self.post, self.norm, [str(f) for f in self.field_type.frequencies]
        groups = [[] if post is None else _by_key(post.gamma, keys),
                  [post.beta] if post is not None and post.has_bias else [],
                  [] if self.scale is None else _by_key(self.scale, keys),
                  [] if norm is None else _by_key(norm.gamma, keys),
                  [norm.beta] if norm is not None and norm.has_bias else []]
        return tuple(map(len, groups)), [p for group in groups for p in group]

    def uses_hip(self, flat: Tensor) -> bool:
        return flat.is_cuda and flat.dtype in (torch.float32, torch.float64, torch.bfloat16) \
            and self.width <= MAX_WIDTH

    def _check(self, rows: Tensor, branch: Tensor, pre: Tensor | None) -> None:
        width = self.width
        if rows.ndim != 2 or rows.shape[1] != width:
            raise ValueError(f"rows must be (N, {width}), got {tuple(rows.shape)}.")
        if branch.shape != rows.shape:
            raise ValueError(f"branch must have the rows' shape {tuple(rows.shape)}, got {tuple(branch.shape)}.")
        if (pre is None) != (self.gate is None):
            raise ValueError(f"pre must be given exactly where there is a gate (gate={self.gate!r}).")
        if pre is not None and tuple(pre.shape) != (rows.shape[0], self.copies):
            raise ValueError(f"pre must be ({rows.shape[0]}, {self.copies}), got {tuple(pre.shape)}.")

    def forward_flat(self, rows: Tensor, branch: Tensor, pre: Tensor | None = None) -> tuple[Tensor, Tensor | None]:
        """``(x', h)`` on flat rows ``(N, D)``, both in the rows' dtype (``h`` None
        without a next norm); ``pre (N, copies)`` the gates' pre-activations."""
        self._check(rows, branch, pre)
        if not self.uses_hip(rows):
            return self._eager(rows, branch, pre)
        if branch.dtype != rows.dtype and not (rows.dtype == torch.bfloat16 and branch.dtype == torch.float32):
            branch = branch.to(rows.dtype)
        pd, (counts, params) = _native.param_dtype(rows.dtype), self._params()
        params = [p if p.dtype == pd and p.is_contiguous() else p.to(pd).contiguous() for p in params]
        # inside the op a parameter looks the same under no_grad
        train = torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (rows, branch, pre, *params))
        out = ResidualNormOp.apply(rows.contiguous(), branch.contiguous(),
                                   None if pre is None else pre.to(rows.dtype).contiguous(), self._layout(),
                                   _GATES.get(self.gate, 1.0), self.post.eps if self.post is not None else 1.0,
                                   self.norm.eps if self.norm is not None else 1.0,
                                   counts, train, *params)
        return out if self.norm is not None else (out, None)

    def forward(self, x: SO2FeatureField, branch: SO2FeatureField,
                pre: Tensor | None = None) -> tuple[SO2FeatureField, SO2FeatureField | None]:
        for given in (x, branch):
            if given.field_type != self.field_type:
                raise ValueError(f"Expected a field of type {self.field_type!r}, got {given.field_type!r}.")
        rows, u = x._rows(), branch._rows()
        batch = rows.shape[:-1]
        y, normed = self.forward_flat(rows.reshape(-1, rows.shape[-1]), u.reshape(-1, u.shape[-1]),
                                      None if pre is None else pre.reshape(-1, pre.shape[-1]))
        fields = [None if t is None else SO2FeatureField.from_flat(self.field_type, t.reshape(*batch, -1))
                  for t in (y, normed)]
        return fields[0], fields[1]

    def _eager(self, rows: Tensor, branch: Tensor, pre: Tensor | None) -> tuple[Tensor, Tensor | None]:
        """The formulas in torch, in the parameters' arithmetic."""
        dtype = _native.param_dtype(rows.dtype)

        def normed(norm: SO2LayerNorm, flat: Tensor) -> Tensor:
            return norm._eager(SO2FeatureField.from_flat(self.field_type, flat))._rows()

        def per_coordinate(values: Tensor) -> Tensor:
            parts = values.split([m for _, m in self.field_type.items()], dim=-1)
            return torch.cat([p if f == 0 else p.repeat_interleave(2, dim=-1)
                              for f, p in zip(self.field_type.frequencies, parts, strict=True)], dim=-1)

        out = branch.to(dtype)
        if self.post is not None:
            out = normed(self.post, out)
        if pre is not None:
            out = per_coordinate(_GATES[self.gate] * torch.sigmoid(pre.to(dtype))) * out
        if self.scale is not None:
            out = per_coordinate(torch.cat([self.scale[str(f)] for f in self.field_type.frequencies])) * out
        out = rows.to(dtype) + out
        return out.to(rows.dtype), None if self.norm is None else normed(self.norm, out).to(rows.dtype)

    def extra_repr(self) -> str:
        return (f"field_type={self.field_type!r}, post_norm={self.post is not None}, gate={self.gate!r}, "
                f"scale={self.initial_scale}, norm={self.norm is not None}")
