"""Differential attention and the sandwich block as layers: the batched
``SO2MHSA(differential=True)`` and ``SO2TransformerBlock`` with
``norm_placement="sandwich"``, alone and together, on the GPU against the same
module in float64 on the CPU, whose arithmetic is torch's (and is checked here
against the oracle's single softmax over the maps and the block's formulas).

The windows taper (``quartic``), so that an edge on the cutoff's rounding weighs
nothing either way.  Bounds are the layers' own (test_attention_gpu.close: 1e-5
relative and 1e-6 of the largest entry for float32, 1e-10 for float64, parameter
gradients within 1e-5 of their norm; 2e-2 of the largest entry for bfloat16 rows).
"""

import math

import pytest
import torch

import problems
from gm_attention_amd.discretization.discretization import SphericalDiscretization
from gm_attention_amd.discretization.frames import build_tangent_frames, rotate_tangent_frames
from gm_attention_amd.discretization.grid import build_equiangular_grid
from gm_attention_amd.nn.attention import SO2MHSA, weighted_segment_sum
from gm_attention_amd.nn.blocks import SO2TransformerBlock
from gm_attention_amd.nn.linear import flat_forward
from gm_attention_amd.representations.field_type import SO2FeatureField, SO2FieldType
from oracle import eager
from test_attention_gpu import close

D64 = torch.float64


def edges_of(batch=1, nlat=10, nlon=20):
    disc = problems.discretization(nlat, nlon)
    e = disc.edge_geometry.tile(batch, n_sources=disc.n_nodes) if batch > 1 else disc.edge_geometry
    return e, disc.coverage_radius


def stirred(module):
    with torch.no_grad():
        g = torch.Generator().manual_seed(5)
        for p in module.parameters():
            p.add_(0.1 * torch.randn(p.shape, generator=g, dtype=D64).to(p))
    return module


def layer(field, heads, dtype=D64, device="cpu"):
    torch.manual_seed(0)
    _, cutoff = edges_of()
    return stirred(SO2MHSA(SO2FieldType(field), heads, cutoff=cutoff, window="quartic", batched=True,
                           differential=True, lambda_init=0.5, dtype=dtype, device=device))


def block(field, heads, differential, gate="double_sigmoid", scale=0.5, multiplier=2, dtype=D64, device="cpu"):
    torch.manual_seed(0)
    _, cutoff = edges_of()
    return stirred(SO2TransformerBlock(SO2FieldType(field), heads, ffn_multiplier=multiplier, cutoff=cutoff,
                                       window="quartic", attention_batched=True, attention_differential=differential,
                                       norm_placement="sandwich", residual_gate=gate, residual_scale=scale, dtype=dtype,
                                       device=device))


def run(module, flat, edges, probe, chunk=None):
    leaf = flat.clone().requires_grad_(True)
    module.zero_grad(set_to_none=True)
    ft = module.field_type_in if isinstance(module, SO2MHSA) else module.field_type
    x = SO2FeatureField.from_flat(ft, leaf)
    out = module(x, edges) if chunk is None else module.forward_chunked(x, edges, chunk_size=chunk)
    out = out.to_flat()
    (out.double() * probe.to(out.device)).sum().backward()
    return out.detach(), leaf.grad, {n: p.grad for n, p in module.named_parameters() if p.grad is not None}


def on_gpu(make, module, dtype, cuda):
    gpu = make(dtype, cuda)
    gpu.load_state_dict({k: v.to(dtype) for k, v in module.state_dict().items()})
    return gpu


def compare(make, dtype, cuda, rows=None, batch=2):
    """The module on the GPU in ``dtype`` (its rows in ``rows``) against float64 on the CPU on the same numbers."""
    module = make(D64, "cpu")
    edges, _ = edges_of(batch)
    width = (module.field_type_in if isinstance(module, SO2MHSA) else module.field_type).dimension
    x, probe = problems.normal((edges.row_ptr.shape[0] - 1, width), 1), problems.normal(
        (edges.row_ptr.shape[0] - 1, width), 7)
    if dtype == torch.float32:
        module.load_state_dict({k: v.float().double() for k, v in module.state_dict().items()})
        x = x.to(rows or torch.float32).double()
        edges = edges.to(None, torch.float32).to(None, D64)
    want = run(module, x, edges, probe)
    gpu = on_gpu(make, module, dtype, cuda)
    got = run(gpu, x.to(cuda, rows or dtype), edges.to(cuda, dtype), probe)
    assert set(got[2]) == set(want[2])
    return got, want


LAYERS = [({0: 16, 1: 16, 2: 16}, 4), ({0: 8, 1: 8, 2: 8}, 2), ({0: 24, 1: 12, 2: 12}, 6), ({0: 8, 1: 4}, 2),
          ({0: 32, 1: 32, 2: 32}, 8)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, D64])
@pytest.mark.parametrize("field,heads", LAYERS)
def test_differential_layer_equals_float64(field, heads, dtype, cuda):
    print(f"differential layer {field} H={heads} {dtype}", flush=True)
    got, want = compare(lambda d, dev: layer(field, heads, d, dev), dtype, cuda)
    close(got[0], want[0], dtype, "out", scaled=True)
    close(got[1], want[1], dtype, "dx", scaled=True)
    for n in want[2]:
        close(got[2][n], want[2][n], dtype, f"d{n}", reduction=True)
    assert float(want[2]["lambda_query"].abs().max()) > 1e-3


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, D64])
@pytest.mark.parametrize("differential,gate,scale", [(True, "double_sigmoid", 0.5), (True, None, None),
                                                     (False, "sigmoid", 0.1)])
def test_sandwich_block_equals_float64(differential, gate, scale, dtype, cuda):
    print(f"sandwich {differential} {gate} {scale} {dtype}", flush=True)
    got, want = compare(lambda d, dev: block({0: 8, 1: 8, 2: 8}, 2, differential, gate, scale, dtype=d, device=dev),
                        dtype, cuda)
    close(got[0], want[0], dtype, "out", scaled=True)
    close(got[1], want[1], dtype, "dx", scaled=True)
    for n in want[2]:
        close(got[2][n], want[2][n], dtype, f"d{n}", reduction=True)


@pytest.mark.gpu
def test_bf16_rows_within_2e2_of_float64(cuda):
    """bfloat16 rows through both operators: the mixer hands back float32, the feed-forward bfloat16."""
    got, want = compare(lambda d, dev: block({0: 32, 1: 32, 2: 32}, 8, True, multiplier=4, dtype=d, device=dev),
                        torch.float32, cuda, rows=torch.bfloat16, batch=1)
    for g, w, name in ((got[0], want[0], "out"), (got[1], want[1], "dx")):
        assert g.dtype == torch.bfloat16
        err = float((g.double().cpu() - w).abs().max()) / float(w.abs().max())
        assert err <= 2e-2, f"{name}: {err:.3e} of the largest entry"
    for n in want[2]:
        err = float((got[2][n].double().cpu() - want[2][n]).norm()) / max(float(want[2][n].norm()), 1e-30)
        assert err <= 2e-2 or float(want[2][n].abs().max()) < 1e-6, f"d{n}: {err:.3e}"


@pytest.mark.gpu
def test_the_block_runs_both_operators(cuda, monkeypatch):
    """A training step of the block reaches the kernels it is there for."""
    from gm_attention_amd import _native

    called = []
    inner = _native._call
    monkeypatch.setattr(_native, "_call", lambda name, *args: (called.append(name), inner(name, *args))[1])
    module = block({0: 16, 1: 16, 2: 16}, 4, True, dtype=torch.float32, device=cuda)
    edges, _ = edges_of()
    n = edges.row_ptr.shape[0] - 1
    run(module, problems.normal((n, 80), 1).float().to(cuda), edges.to(cuda, torch.float32),
        problems.normal((n, 80), 7))
    for name, times in (("gm_differential_forward_f32", 1), ("gm_differential_backward_f32", 1),
                        ("gm_residual_norm_forward_f32", 2), ("gm_residual_norm_backward_f32", 2)):
        assert called.count(name) == times, name
    assert not any(name.startswith("gm_softmax") for name in called)


@pytest.mark.gpu
def test_chunked_equals_whole(cuda):
    module = block({0: 8, 1: 8, 2: 8}, 2, True, device=cuda)
    edges, _ = edges_of(2)
    edges = edges.to(cuda, D64)
    n = edges.row_ptr.shape[0] - 1
    x, probe = problems.normal((n, 40), 1).to(cuda), problems.normal((n, 40), 7)
    whole, chunked = run(module, x, edges, probe), run(module, x, edges, probe, chunk=37)
    close(chunked[0], whole[0], D64, "out")
    close(chunked[1], whole[1], D64, "dx")
    for n in whole[2]:
        close(chunked[2][n], whole[2][n], D64, f"d{n}")


@pytest.mark.gpu
def test_block_is_gauge_equivariant(cuda):
    grid = build_equiangular_grid(10, 20)
    cutoff = 3.0 * math.pi / 9
    frames = build_tangent_frames(grid.nodes)
    theta = torch.rand(grid.n_nodes, dtype=D64, generator=torch.Generator().manual_seed(4)) * 2 * math.pi
    base, turned = (SphericalDiscretization.from_grid(grid, cutoff, frames=f).edge_geometry.to(cuda, D64)
                    for f in (frames, rotate_tangent_frames(frames, theta)))
    module = block({0: 8, 1: 8, 2: 8}, 2, True, device=cuda)
    x = SO2FeatureField.from_flat(module.field_type, problems.normal((grid.n_nodes, 40), 1).to(cuda))
    with torch.no_grad():
        y, y_turned = module(x, base), module(x.gauge_transform(theta.to(cuda)), turned)
    expected = y.gauge_transform(theta.to(cuda))
    torch.testing.assert_close(y_turned.to_flat(), expected.to_flat(), rtol=1e-9, atol=1e-9)
    assert float((y.to_flat() - expected.to_flat()).abs().max()) > 1e-3


@pytest.mark.gpu
def test_forward_graph_replays_equal_the_eager_forward(cuda):
    module = block({0: 16, 1: 16, 2: 16}, 4, True, dtype=torch.float32, device=cuda).eval()
    edges, _ = edges_of()
    edges = edges.to(cuda, torch.float32)
    x = problems.normal((edges.row_ptr.shape[0] - 1, 80), 3).float().to(cuda)

    def forward():
        return module.forward_flat(x, edges)

    with torch.no_grad():
        want = forward().clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            forward()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = forward()
        for replay in range(3):
            out.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, want), replay
            assert torch.equal(forward(), want), replay
            torch.cuda.synchronize()


@pytest.mark.gpu
def test_switched_off_the_layer_runs_in_torch(cuda, monkeypatch):
    from gm_attention_amd.nn import fused_attention

    module = layer({0: 8, 1: 8, 2: 8}, 2, device=cuda)
    edges, _ = edges_of()
    edges = edges.to(cuda, D64)
    x, probe = problems.normal((edges.row_ptr.shape[0] - 1, 40), 1).to(cuda), problems.normal(
        (edges.row_ptr.shape[0] - 1, 40), 7)
    fused = run(module, x, edges, probe)
    monkeypatch.setattr(fused_attention, "MODE", "0")
    plain = run(module, x, edges, probe)
    close(plain[0], fused[0], D64, "out")
    for n in fused[2]:
        close(plain[2][n], fused[2][n], D64, f"d{n}")


@pytest.mark.gpu
@pytest.mark.parametrize("gate,scale", [("sigmoid", 0.5), (None, None)])
def test_a_replica_of_a_block_gives_its_results(gate, scale, cuda):
    """A data-parallel step's replica, whose parameters are plain attributes."""
    from torch.nn.parallel import replicate

    module = block({0: 8, 1: 8, 2: 8}, 2, True, gate, scale, dtype=torch.float32, device=cuda)
    edges = edges_of()[0].to(cuda, torch.float32)
    x = problems.normal((edges.row_ptr.shape[0] - 1, 40), 1).float().to(cuda)
    (replica,) = replicate(module, [cuda])
    params = list(module.parameters())

    def step(m):
        out = m.forward_flat(x, edges)
        return [out, *torch.autograd.grad((out * x).sum(), params, allow_unused=True)]

    want = step(module)
    for a, b, name in zip(step(replica), want, ["out", *(n for n, _ in module.named_parameters())], strict=True):
        b = torch.zeros_like(a) if b is None else b
        if name.endswith("key.bias"):  # moves all of a row's scores alike: zero but for both sides' roundings
            b = torch.zeros_like(b)
        # a replica's matrices are built, not assembled: the same numbers in another order
        close(a, b, torch.float32, name, reduction=True)


@pytest.mark.gpu
def test_edge_sets_are_copied_and_saved_after_a_step(cuda):
    """An edge set that a differential layer has run on is copied and pickled as any other."""
    import copy
    import pickle

    module = layer({0: 8, 1: 8, 2: 8}, 2, torch.float32, cuda)
    edges = edges_of(2)[0].to(cuda, torch.float32)
    n = edges.row_ptr.shape[0] - 1
    x, probe = problems.normal((n, 40), 1).float().to(cuda), problems.normal((n, 40), 7)
    want = run(module, x, edges, probe)
    for other in (copy.deepcopy(edges), pickle.loads(pickle.dumps(edges))):
        got = run(module, x, other, probe)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
@pytest.mark.parametrize("train", [True, False])
def test_a_chunked_step_builds_its_tables_once_and_is_captured(train, cuda, monkeypatch):
    from gm_attention_amd.nn import differential

    module = layer({0: 16, 1: 16, 2: 16}, 4, torch.float32, cuda).train(train)
    edges = edges_of(2)[0].to(cuda, torch.float32)
    n = edges.row_ptr.shape[0] - 1
    x, up = (problems.normal((n, 80), i).float().to(cuda) for i in (1, 7))
    built, init = [], differential.EdgeTables.__init__
    monkeypatch.setattr(differential.EdgeTables, "__init__",
                        lambda self, *a, **kw: (built.append(1), init(self, *a, **kw))[1])

    def step():
        leaf = x.detach().requires_grad_(train)
        with torch.set_grad_enabled(train):
            out = module.forward_chunked(SO2FeatureField.from_flat(module.field_type_in, leaf), edges,
                                         chunk_size=75).to_flat()
        return [out.detach(), *(torch.autograd.grad(out, leaf, up) if train else ())]

    want = [t.clone() for t in step()]
    chunks = sum(1 for _ in edges.chunks(75))
    assert len(built) == chunks == 6
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        got = step()
    assert len(built) == chunks
    for size in (40, 50, 60, 90):  # other chunkings, beyond what is kept of them
        with torch.no_grad():
            module.forward_chunked(SO2FeatureField.from_flat(module.field_type_in, x), edges, chunk_size=size)
    for replay in range(3):
        for t in got:
            t.zero_()
        captured.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want, strict=True)), replay
        assert all(torch.equal(a, b) for a, b in zip(step(), want, strict=True)), replay
        torch.cuda.synchronize()


# ---------------------------------------------------------------- without a GPU


def test_cpu_layer_is_its_formulas():
    """The layer's heads, from the oracle's softmax over the 2 H maps, their difference and the value kernels."""
    module = layer({0: 8, 1: 4, 2: 4}, 2)
    edges, cutoff = edges_of()
    n = edges.row_ptr.shape[0] - 1
    x = problems.normal((n, module.field_type_in.dimension), 1)
    field = SO2FeatureField.from_flat(module.field_type_in, x)
    t = problems.tables(10, 20, window="quartic")
    heads = []
    q1k1, q2k2 = (module.lambda_query * module.lambda_key).sum(-1)
    lam = q1k1.exp() - q2k2.exp() + 0.5
    torch.testing.assert_close(module.lambdas(), lam)
    for h, head in enumerate(module.heads):
        q, k = flat_forward(head.query, x), flat_forward(head.key, x)
        # the head's rows: two maps of half its copies each, side by side at every frequency
        rows, at = [], 0
        for f, m in head.field_type_attn.items():
            rows.append((f, m // 2, at, 0, 1 if f == 0 else 2))
            at += m * (1 if f == 0 else 2)
        maps = eager.softmax_op(q, k, t.transport, t.bias, t.inside, rows, t.row_ptr, t.source, 2, (at / 2) ** -0.5)
        alpha = maps[:, 0] - lam[h] * maps[:, 1]
        messages = head.value(SO2FeatureField(field.field_type, {
            f: field[f].index_select(0, edges.source_index) for f in field.frequencies}), edges)
        heads.append(weighted_segment_sum(alpha, messages.coefficients, edges.row_ptr))
    whole = SO2FeatureField(module.field_type_in, {
        f: torch.cat([o[f] for o in heads], dim=-1 if f == 0 else -2) for f in field.frequencies})
    want = module.output_projection(whole).to_flat()
    torch.testing.assert_close(module(field, edges).to_flat(), want, rtol=1e-10, atol=1e-10)


def test_cpu_block_is_its_formulas():
    module = block({0: 8, 1: 4}, 2, True, gate="sigmoid")
    edges, _ = edges_of()
    x = problems.normal((edges.row_ptr.shape[0] - 1, 16), 1)
    ft = module.field_type

    def per_coordinate(v):
        return torch.cat([v[..., :8], v[..., 8:].repeat_interleave(2, dim=-1)], dim=-1)

    def joined(residual, rows, u, given):
        z = given[:, :8] @ residual.gate_linear.weight.t() + residual.gate_linear.bias
        scale = per_coordinate(torch.cat(list(residual.scale.values())))
        return rows + scale * per_coordinate(torch.sigmoid(z)) * residual.post.forward_flat(u)

    h = module.norm1.forward_flat(x)
    mixed = module.attention(SO2FeatureField.from_flat(ft, h), edges).to_flat()
    rows = joined(module.residual1, x, mixed, h)
    h = module.residual1.norm.forward_flat(rows)
    hidden = flat_forward(module.linear2, module.activation.forward_flat(flat_forward(module.linear1, h)))
    want = joined(module.residual2, rows, hidden, h)
    got = module(SO2FeatureField.from_flat(ft, x), edges).to_flat()
    torch.testing.assert_close(got, want, rtol=1e-12, atol=1e-12)


def test_the_default_block_is_as_it_was():
    """No parameter of the new forms in a block that does not ask for them."""
    names = {n for n, _ in SO2TransformerBlock(SO2FieldType({0: 4, 1: 4}), 2, cutoff=1.0).named_parameters()}
    assert not any("residual" in n or "lambda" in n for n in names)
    assert "norm2.gamma.0" in names


def test_refusals():
    ft = SO2FieldType({0: 4, 1: 4})
    with pytest.raises(ValueError, match="needs batched=True"):
        SO2MHSA(ft, 2, cutoff=1.0, differential=True)
    with pytest.raises(ValueError, match="twice num_heads"):
        SO2MHSA(SO2FieldType({0: 4, 1: 2}), 2, cutoff=1.0, batched=True, differential=True)
    with pytest.raises(ValueError, match="norm_placement must be"):
        SO2TransformerBlock(ft, 2, cutoff=1.0, norm_placement="post")
    for kw in (dict(residual_gate="sigmoid"), dict(residual_scale=1.0)):
        with pytest.raises(ValueError, match="belong to norm_placement='sandwich'"):
            SO2TransformerBlock(ft, 2, cutoff=1.0, **kw)
    with pytest.raises(ValueError, match="gate must be None or one of"):
        SO2TransformerBlock(ft, 2, cutoff=1.0, norm_placement="sandwich", residual_gate="silu")
    with pytest.raises(ValueError, match="needs mixer='attention'"):
        SO2TransformerBlock(ft, 2, cutoff=1.0, mixer="convolution", attention_differential=True)


def test_modules_pickled_before_there_were_the_options_run_as_they_did():
    import pickle

    edges, cutoff = edges_of()
    torch.manual_seed(0)
    for make, option in ((lambda: SO2MHSA(SO2FieldType({0: 4, 1: 4}), 2, cutoff=cutoff, batched=True, dtype=D64),
                          "differential"),
                         (lambda: SO2TransformerBlock(SO2FieldType({0: 4, 1: 4}), 2, cutoff=cutoff,
                                                      attention_batched=True, dtype=D64), "norm_placement")):
        module = make()
        older = pickle.loads(pickle.dumps(module))
        for m in older.modules():
            m.__dict__.pop(option, None)
            m.__dict__.pop("differential", None)
        x = problems.normal((edges.row_ptr.shape[0] - 1, 12), 1)
        probe = problems.normal(x.shape, 2)
        for chunk in (None, 50):
            want, got = run(module, x, edges, probe, chunk), run(older, x, edges, probe, chunk)
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        assert repr(older) == repr(module)


@pytest.mark.parametrize("field,heads", [({0: 34, 1: 34}, 17), ({f: 2 for f in range(9)}, 1), ({0: 1028}, 1)])
def test_layers_beyond_the_ops_bounds_run_in_torch(field, heads):
    """More heads, frequencies or numbers a row than the fused op takes."""
    from gm_attention_amd.nn import differential

    cutoff = math.pi / 3
    edges = SphericalDiscretization.from_grid(build_equiangular_grid(10, 20), cutoff, max_frequency=8).edge_geometry
    module = SO2MHSA(SO2FieldType(field), heads, cutoff=cutoff, window="quartic", batched=True, differential=True,
                     dtype=D64)
    q, k = (problems.normal((edges.row_ptr.shape[0] - 1, module.field_type_in.dimension), i) for i in range(2))
    got = differential.attention_weights(module, q, k, edges)
    t = problems.tables(10, 20, window="quartic")
    transport = torch.view_as_real(edges.transport_phases)
    rows, at = [], 0
    for f, m in field.items():
        rows.append((f, m // (2 * heads), at, 0, 1 if f == 0 else 2))
        at += m * (1 if f == 0 else 2)
    maps = eager.softmax_op(q, k, transport, t.bias, t.inside, rows, t.row_ptr, t.source, 2 * heads,
                            (at / (2 * heads)) ** -0.5)
    torch.testing.assert_close(got, maps[:, 0::2] - module.lambdas() * maps[:, 1::2], rtol=1e-10, atol=1e-12)


def replica_of(module):
    """A module's replica as a data-parallel step makes one (torch.nn.parallel.replicate, which needs a GPU)."""
    replica = module._replicate_for_data_parallel()
    replica._former_parameters = {}
    for key, child in module._modules.items():
        setattr(replica, key, None if child is None else replica_of(child))
    for key, p in module._parameters.items():
        if p is None:
            replica._parameters[key] = None
        else:
            setattr(replica, key, p * 1.0)
            replica._former_parameters[key] = getattr(replica, key)
    return replica


@pytest.mark.parametrize("placement,mixer", [("pre", "attention"), ("pre", "convolution"), ("sandwich", "attention"),
                                             ("sandwich", "convolution")])
def test_replicas_of_blocks_give_their_results(placement, mixer):
    edges, cutoff = edges_of()
    torch.manual_seed(0)
    module = stirred(SO2TransformerBlock(SO2FieldType({0: 4, 1: 4}), 2, cutoff=cutoff, attention_batched=True,
                                         mixer=mixer, norm_placement=placement, dtype=D64))
    replica = replica_of(module)
    assert not list(replica.parameters())
    x = problems.normal((edges.row_ptr.shape[0] - 1, 12), 1)
    for chunk in (None, 50):
        assert torch.equal(replica.forward_flat(x, edges, chunk), module.forward_flat(x, edges, chunk))
    if placement == "sandwich":
        for a, b in ((replica.residual1, module.residual1), (replica.residual2, module.residual2)):
            (counts, mine), (want, theirs) = a._params(), b._params()
            assert counts == want and all(torch.equal(p, q) for p, q in zip(mine, theirs, strict=True))


def test_chunks_tables_are_kept_with_the_edge_set():
    """Every pass over the chunks finds the tables of the first, over the chunk's own targets and the range of
    its sources, and its weights are the whole edge set's."""
    from gm_attention_amd.nn import differential

    edges, cutoff = edges_of(2)
    n, maps, heads = edges.row_ptr.shape[0] - 1, SO2FieldType({0: 2, 1: 1}), 2
    q, k = (problems.normal((n, 16), i) for i in range(2))
    lam = torch.tensor([0.3, 0.6], dtype=D64)
    whole = differential.edge_tables(edges, cutoff, "quartic", D64, 1)
    want = differential.differential_softmax(q, k, lam, whole, maps, heads)
    first_pass, got = [], []
    for chunk in edges.chunks(37):
        tables, first, source = differential.chunk_tables(chunk, cutoff, "quartic", D64, 1)
        first_pass.append(tables)
        assert tables.n_targets <= 37 and tables.n_sources < n  # but for a sample's border, a band of rows
        got.append(differential.differential_softmax(q[first:first + tables.n_targets],
                                                     k[source:source + tables.n_sources], lam, tables, maps, heads))
    torch.testing.assert_close(torch.cat(got), want, rtol=1e-13, atol=1e-15)
    for chunk, held in zip(edges.chunks(37), first_pass, strict=True):
        assert differential.chunk_tables(chunk, cutoff, "quartic", D64, 1)[0] is held
    # other chunkings: what is kept stays within two passes over the edges
    for size in (11, 50, 60, 90):
        for chunk in edges.chunks(size):
            differential.chunk_tables(chunk, cutoff, "quartic", D64, 1)
    from gm_attention_amd.nn import fused_attention

    ranges = fused_attention.geometry(edges, cutoff, "quartic", D64).derived["differential ranges", 1]
    assert sum(t.n_edges for t, *_ in ranges.held.values()) == ranges.edges <= 2 * edges.n_edges


def test_a_chunk_under_numbers_of_its_own_has_tables_of_its_own():
    """An edge set registered as a chunk keeps its own: another may have its span with other numbers."""
    from gm_attention_amd.nn import differential, fused_attention

    edges, cutoff = edges_of()
    (chunk, *_), n = list(edges.chunks(50)), edges.row_ptr.shape[0] - 1
    own = chunk.select(torch.arange(chunk.n_edges), n_nodes=n)  # copies, not views
    fused_attention.register_chunk(own, edges, 0, chunk.n_edges)
    mine = differential.chunk_tables(own, cutoff, "quartic", D64, 1)
    theirs = differential.chunk_tables(chunk, cutoff, "quartic", D64, 1)
    assert mine[0] is not theirs[0] and mine[1:] == theirs[1:]
    assert torch.equal(mine[0].row_ptr, theirs[0].row_ptr) and torch.equal(mine[0]._source, theirs[0]._source)
    assert differential.chunk_tables(own, cutoff, "quartic", D64, 1)[0] is mine[0]
