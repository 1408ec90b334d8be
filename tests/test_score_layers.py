"""What enters a batched attention layer's scores: ``SO2MHSA`` and
``SO2TransformerBlock`` with a learned bias a ring of distance, normalised queries
and keys and rotations by position, alone and together, on the GPU against the same
module in float64 on the CPU, whose arithmetic is torch's (and is checked here
against the formulas written with the oracle's softmax).

The windows taper (``quartic``), so that an edge on the cutoff's rounding weighs
nothing either way.  Bounds are the layers' own (test_attention_gpu.close: 1e-5
relative and 1e-6 of the largest entry for float32, 1e-10 for float64, parameter
gradients within 1e-5 of their norm; 2e-2 of the largest entry for bfloat16 rows).
"""

import copy
import math
import pickle

import pytest
import torch

import problems
from gm_attention_amd.discretization.discretization import SphericalDiscretization
from gm_attention_amd.discretization.frames import build_tangent_frames, rotate_tangent_frames
from gm_attention_amd.discretization.grid import build_equiangular_grid
from gm_attention_amd.nn import attention, fused_attention, relative
from gm_attention_amd.nn.attention import SO2MHSA, weighted_segment_sum
from gm_attention_amd.nn.blocks import SO2TransformerBlock
from gm_attention_amd.nn.head_norm import query_key_norm, rotary_frequencies
from gm_attention_amd.nn.linear import flat_forward
from gm_attention_amd.nn.relative import RelativeEdgeTables, distance_buckets, relative_softmax
from gm_attention_amd.representations.field_type import SO2FeatureField, SO2FieldType
from oracle import eager
from test_attention_gpu import close
from test_differential_layers import edges_of, on_gpu, stirred

D64 = torch.float64
#: every option alone, and together
OPTIONS = {"bias": dict(relative_bias=9), "norm": dict(query_key_norm=True), "turn": dict(rotary=True),
           "norm+turn": dict(query_key_norm=True, rotary=True),
           "all": dict(relative_bias=16, query_key_norm=True, rotary=True),
           "differential+norm+turn": dict(differential=True, query_key_norm=True, rotary=True)}


def frequencies(field, heads, kw):
    maps = 2 * heads if kw.get("differential") else heads
    return rotary_frequencies(SO2FieldType({f: m // maps for f, m in field.items()}), (6.0, 5.0), (0.5, 1.0),
                              (False, True))


def layer(field, heads, option, dtype=D64, device="cpu"):
    torch.manual_seed(0)
    kw = dict(OPTIONS[option])
    if kw.get("rotary"):
        kw["rotary"] = frequencies(field, heads, kw)
    return stirred(SO2MHSA(SO2FieldType(field), heads, cutoff=edges_of()[1], window="quartic", batched=True,
                           dtype=dtype, device=device, **kw))


def block(field, heads, option, placement="pre", multiplier=2, dtype=D64, device="cpu"):
    torch.manual_seed(0)
    kw = dict(OPTIONS[option])
    if kw.get("rotary"):
        kw["rotary"] = frequencies(field, heads, kw)
    kw = {f"attention_{n}": v for n, v in kw.items()}
    return stirred(SO2TransformerBlock(SO2FieldType(field), heads, ffn_multiplier=multiplier, cutoff=edges_of()[1],
                                       window="quartic", attention_batched=True, norm_placement=placement,
                                       dtype=dtype, device=device, **kw))


def positions_of(n, batch=1, nlat=10, nlon=20):
    """Latitude and longitude of the grid's nodes, sample by sample."""
    nodes = build_equiangular_grid(nlat, nlon).nodes.double()
    at = torch.stack([torch.asin(nodes[:, 2].clamp(-1, 1)), torch.atan2(nodes[:, 1], nodes[:, 0])], dim=1)
    return at.repeat(n // at.shape[0], 1)


def run(module, flat, edges, probe, chunk=None, positions=None):
    leaf = flat.clone().requires_grad_(True)
    module.zero_grad(set_to_none=True)
    layer_ = module if isinstance(module, SO2MHSA) else module.attention
    ft = module.field_type_in if isinstance(module, SO2MHSA) else module.field_type
    x = SO2FeatureField.from_flat(ft, leaf)
    given = {}
    if layer_.rotated:
        given["positions"] = (positions_of(flat.shape[0]) if positions is None else positions).to(flat.device)
    out = module(x, edges, **given) if chunk is None else module.forward_chunked(x, edges, chunk_size=chunk, **given)
    out = out.to_flat()
    (out.double() * probe.to(out.device)).sum().backward()
    return out.detach(), leaf.grad, {n: p.grad for n, p in module.named_parameters() if p.grad is not None}


def compare(make, dtype, cuda, rows=None, batch=2):
    module = make(D64, "cpu")
    edges, _ = edges_of(batch)
    width = (module.field_type_in if isinstance(module, SO2MHSA) else module.field_type).dimension
    n = edges.row_ptr.shape[0] - 1
    x, probe = problems.normal((n, width), 1), problems.normal((n, width), 7)
    if dtype == torch.float32:
        module.load_state_dict({k: v.float().double() for k, v in module.state_dict().items()})
        x = x.to(rows or torch.float32).double()
        edges = edges.to(None, torch.float32).to(None, D64)
    want = run(module, x, edges, probe)
    got = run(on_gpu(make, module, dtype, cuda), x.to(cuda, rows or dtype), edges.to(cuda, dtype), probe)
    assert set(got[2]) == set(want[2])
    return got, want


def close_gradients(got, want, dtype):
    for n in want:
        if n.endswith("key.bias") and float(want[n].abs().max()) < 1e-9:
            continue  # moves all of a row's scores alike: zero but for both sides' roundings
        close(got[n], want[n], dtype, f"d{n}", reduction=True)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, D64])
@pytest.mark.parametrize("option", OPTIONS)
@pytest.mark.parametrize("field,heads", [({0: 16, 1: 16, 2: 16}, 4), ({0: 24, 1: 12, 2: 12}, 6), ({0: 8, 1: 4}, 2)])
def test_layer_equals_float64(field, heads, option, dtype, cuda):
    print(f"layer {field} H={heads} {option} {dtype}", flush=True)
    got, want = compare(lambda d, dev: layer(field, heads, option, d, dev), dtype, cuda)
    close(got[0], want[0], dtype, "out", scaled=True)
    close(got[1], want[1], dtype, "dx", scaled=True)
    close_gradients(got[2], want[2], dtype)
    if "bias" in option or option == "all":
        assert float(want[2]["relative_bias"].abs().max()) > 1e-4


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, D64])
@pytest.mark.parametrize("placement", ["pre", "sandwich"])
def test_block_equals_float64(placement, dtype, cuda):
    got, want = compare(lambda d, dev: block({0: 8, 1: 8, 2: 8}, 2, "all", placement, dtype=d, device=dev), dtype,
                        cuda)
    close(got[0], want[0], dtype, "out", scaled=True)
    close(got[1], want[1], dtype, "dx", scaled=True)
    close_gradients(got[2], want[2], dtype)


@pytest.mark.gpu
@pytest.mark.parametrize("placement", ["pre", "sandwich"])
def test_bf16_rows_within_2e2_of_float64(placement, cuda, monkeypatch):
    """A query's or key's bias has a gradient of one term a node, of both signs: terms off by 2e-2 of themselves, as the
    rows here are allowed to be, leave their sum off by 2e-2 of the sum of their absolute values."""
    scored, projected = attention._scored, []

    def kept(mhsa, queries, keys, positions):
        for rows in (queries, keys):
            rows.retain_grad()
            projected.append(rows)
        return scored(mhsa, queries, keys, positions)

    monkeypatch.setattr(attention, "_scored", kept)
    got, want = compare(lambda d, dev: block({0: 32, 1: 32, 2: 32}, 8, "all", placement, 4, d, dev), torch.float32,
                        cuda, rows=torch.bfloat16, batch=1)
    terms = {s: rows.grad.abs().sum(0) for s, rows in zip(("query", "key"), projected)}  # float64's: the first run
    for g, w, name in ((got[0], want[0], "out"), (got[1], want[1], "dx")):
        assert g.dtype == torch.bfloat16
        err = float((g.double().cpu() - w).abs().max()) / float(w.abs().max())
        assert err <= 2e-2, f"{name}: {err:.3e} of the largest entry"
    for n in want[2]:
        size = float(want[2][n].norm())
        if n.endswith(("query.bias", "key.bias")):
            head = int(n.split(".")[2])
            size = float(terms[n.split(".")[3]][4 * head:4 * head + 4].norm())
        err = float((got[2][n].double().cpu() - want[2][n]).norm()) / max(size, 1e-30)
        assert err <= 2e-2 or float(want[2][n].abs().max()) < 1e-6, f"d{n}: {err:.3e}"


@pytest.mark.gpu
@pytest.mark.parametrize("rows,suffix", [(torch.float32, "f32"), (torch.bfloat16, "bf16")])
def test_the_block_runs_both_operators(rows, suffix, cuda, monkeypatch):
    """A training step of the block reaches the kernels it is there for."""
    from gm_attention_amd import _native

    called = []
    inner = _native._call
    monkeypatch.setattr(_native, "_call", lambda name, *args: (called.append(name), inner(name, *args))[1])
    module = block({0: 32, 1: 32, 2: 32}, 8, "all", dtype=torch.float32, device=cuda)
    edges, _ = edges_of()
    n = edges.row_ptr.shape[0] - 1
    run(module, problems.normal((n, 160), 1).to(rows).to(cuda), edges.to(cuda, torch.float32),
        problems.normal((n, 160), 7))
    for name in ("gm_relative_forward_", "gm_relative_backward_", "gm_head_norm_forward_", "gm_head_norm_backward_"):
        assert called.count(name + suffix) == 1, name
    assert not any(name.startswith("gm_softmax") for name in called)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, D64])
def test_both_operators_in_a_row(rows, cuda):
    """As a program calls them: normalised and turned queries and keys into the softmax with a learned bias, forward and
    backward, against the same calls in float64 on the CPU."""
    heads, head = 4, SO2FieldType({0: 4, 1: 4, 2: 4})
    t = problems.tables(10, 20, batch=2, window="quartic")
    n, E = t.n_nodes, t.source.shape[0]
    given = dict(q=problems.normal((n, 80), 1), k=problems.normal((n, 80), 2),
                 q_gain=1 + 0.2 * problems.normal((12,), 3), k_gain=1 + 0.2 * problems.normal((12,), 4), table=problems.normal((12, heads), 5))
    at, f = positions_of(n), rotary_frequencies(head, (6.0, 4.0), (0.5, 1.0), (False, True))
    up = problems.normal((E, heads), 6)
    given, up = {name: v.to(rows).double() for name, v in given.items()}, up.to(rows).double()
    tables = [t.transport[:, :3].to(rows).double(), t.bias.to(rows).double()]
    buckets = distance_buckets(t.rho, 1.0, 12)

    def step(dtype, device):
        edges = RelativeEdgeTables(t.row_ptr.to(device), t.source.to(device),
                                   *(x.to(dtype).to(device) for x in tables), t.inside.to(device), buckets.to(device),
                                   12)
        leaves = {name: v.to(dtype).to(device).requires_grad_(True) for name, v in given.items()}
        q, k = query_key_norm(leaves["q"], leaves["k"], head, heads, leaves["q_gain"], leaves["k_gain"],
                              positions=at.to(device), frequencies=f.to(device))
        alpha = relative_softmax(q, k, leaves["table"], edges, head, heads)
        return [alpha, *torch.autograd.grad(alpha, list(leaves.values()), up.to(dtype).to(device))]

    for got, want, name in zip(step(rows, cuda), step(D64, "cpu"), ("alpha", *given)):
        close(got, want, rows, name, scaled=True, reduction=name.endswith(("gain", "table")))


@pytest.mark.gpu
@pytest.mark.parametrize("option", ["all", "differential+norm+turn", "norm"])
def test_chunked_equals_whole(option, cuda):
    module = block({0: 8, 1: 8, 2: 8}, 2, option, device=cuda)
    edges, _ = edges_of(2)
    edges = edges.to(cuda, D64)
    n = edges.row_ptr.shape[0] - 1
    x, probe = problems.normal((n, 40), 1).to(cuda), problems.normal((n, 40), 7)
    whole, chunked = run(module, x, edges, probe), run(module, x, edges, probe, chunk=37)
    close(chunked[0], whole[0], D64, "out")
    close(chunked[1], whole[1], D64, "dx")
    for name in whole[2]:
        close(chunked[2][name], whole[2][name], D64, f"d{name}")


@pytest.mark.gpu
def test_block_is_gauge_equivariant(cuda):
    grid = build_equiangular_grid(10, 20)
    cutoff = 3.0 * math.pi / 9
    frames = build_tangent_frames(grid.nodes)
    theta = torch.rand(grid.n_nodes, dtype=D64, generator=torch.Generator().manual_seed(4)) * 2 * math.pi
    base, turned = (SphericalDiscretization.from_grid(grid, cutoff, frames=f).edge_geometry.to(cuda, D64)
                    for f in (frames, rotate_tangent_frames(frames, theta)))
    module = block({0: 8, 1: 8, 2: 8}, 2, "all", device=cuda)
    at = positions_of(grid.n_nodes).to(cuda)
    x = SO2FeatureField.from_flat(module.field_type, problems.normal((grid.n_nodes, 40), 1).to(cuda))
    with torch.no_grad():
        y, y_turned = module(x, base, at), module(x.gauge_transform(theta.to(cuda)), turned, at)
    expected = y.gauge_transform(theta.to(cuda))
    torch.testing.assert_close(y_turned.to_flat(), expected.to_flat(), rtol=1e-9, atol=1e-9)
    assert float((y.to_flat() - expected.to_flat()).abs().max()) > 1e-3


@pytest.mark.gpu
def test_forward_graph_replays_equal_the_eager_forward(cuda):
    module = block({0: 16, 1: 16, 2: 16}, 4, "all", dtype=torch.float32, device=cuda).eval()
    edges, _ = edges_of()
    edges = edges.to(cuda, torch.float32)
    n = edges.row_ptr.shape[0] - 1
    x, at = problems.normal((n, 80), 3).float().to(cuda), positions_of(n).to(cuda)

    def forward():
        return module.forward_flat(x, edges, positions=at)

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
    module = layer({0: 8, 1: 8, 2: 8}, 2, "all", device=cuda)
    edges, _ = edges_of()
    edges = edges.to(cuda, D64)
    n = edges.row_ptr.shape[0] - 1
    x, probe = problems.normal((n, 40), 1).to(cuda), problems.normal((n, 40), 7)
    fused = run(module, x, edges, probe)
    monkeypatch.setattr(fused_attention, "MODE", "0")
    plain = run(module, x, edges, probe)
    close(plain[0], fused[0], D64, "out")
    for name in fused[2]:
        close(plain[2][name], fused[2][name], D64, f"d{name}")


@pytest.mark.gpu
def test_edge_sets_and_modules_are_copied_after_a_step(cuda):
    module = layer({0: 8, 1: 8, 2: 8}, 2, "all", torch.float32, cuda)
    edges = edges_of(2)[0].to(cuda, torch.float32)
    n = edges.row_ptr.shape[0] - 1
    x, probe = problems.normal((n, 40), 1).float().to(cuda), problems.normal((n, 40), 7)
    want = run(module, x, edges, probe)
    for m, e in ((copy.deepcopy(module), edges), (pickle.loads(pickle.dumps(module)), copy.deepcopy(edges)),
                 (module, pickle.loads(pickle.dumps(edges)))):
        got = run(m, x, e, probe)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.gpu
def test_a_replica_of_a_block_gives_its_results(cuda):
    """A data-parallel step's replica, whose parameters are plain attributes."""
    from torch.nn.parallel import replicate

    module = block({0: 8, 1: 8, 2: 8}, 2, "all", dtype=torch.float32, device=cuda)
    edges = edges_of()[0].to(cuda, torch.float32)
    n = edges.row_ptr.shape[0] - 1
    x, at = problems.normal((n, 40), 1).float().to(cuda), positions_of(n).to(cuda)
    (replica,) = replicate(module, [cuda])
    params = list(module.parameters())

    def step(m):
        out = m.forward_flat(x, edges, positions=at)
        return [out, *torch.autograd.grad((out * x).sum(), params, allow_unused=True)]

    want = step(module)
    for a, b, name in zip(step(replica), want, ["out", *(p for p, _ in module.named_parameters())], strict=True):
        close(a, torch.zeros_like(a) if b is None else b, torch.float32, name, reduction=True)


# ---------------------------------------------------------------- without a GPU


def test_cpu_layer_is_its_formulas():
    """The layer's heads, from normalised and turned rows by hand, the oracle's softmax with the learned numbers in its
    bias, and the value kernels."""
    module = layer({0: 8, 1: 4, 2: 4}, 2, "all")
    edges, cutoff = edges_of()
    n = edges.row_ptr.shape[0] - 1
    x, at = problems.normal((n, module.field_type_in.dimension), 1), positions_of(n)
    field = SO2FeatureField.from_flat(module.field_type_in, x)
    t = problems.tables(10, 20, window="quartic")
    rings = torch.floor(16 * t.rho + 1e-3).clamp(0, 15).long()
    theta = at @ torch.tensor(module.query_key.frequencies, dtype=D64)  # slots: two pairs of scalars, 2 + 2 copies

    def scored(rows, gain):
        """One head's rows: four scalars, two copies each of frequencies 1 and 2."""
        rows = rows / (rows.square().mean(1, keepdim=True) + 1e-6).sqrt()
        rows = rows * torch.cat([gain[:4], gain[4:].repeat_interleave(2)])
        z = torch.view_as_complex(rows.reshape(n, 6, 2).contiguous()) * torch.polar(torch.ones_like(theta), theta)
        return torch.view_as_real(z).reshape(n, 12)

    heads = []
    for h, head in enumerate(module.heads):
        q = scored(flat_forward(head.query, x), module.query_key.query_gain)
        k = scored(flat_forward(head.key, x), module.query_key.key_gain)
        rows, begin = [], 0
        for f, m in head.field_type_attn.items():
            rows.append((f, m, begin, 0, 1 if f == 0 else 2))
            begin += m * (1 if f == 0 else 2)
        alpha = eager.softmax_op(q, k, t.transport, t.bias + module.relative_bias[:, h][rings], t.inside, rows,
                                 t.row_ptr, t.source, 1, begin ** -0.5)[:, 0]
        messages = head.value(SO2FeatureField(field.field_type, {
            f: field[f].index_select(0, edges.source_index) for f in field.frequencies}), edges)
        heads.append(weighted_segment_sum(alpha, messages.coefficients, edges.row_ptr))
    whole = SO2FeatureField(module.field_type_in, {
        f: torch.cat([o[f] for o in heads], dim=-1 if f == 0 else -2) for f in field.frequencies})
    want = module.output_projection(whole).to_flat()
    torch.testing.assert_close(module(field, edges, at).to_flat(), want, rtol=1e-10, atol=1e-10)


def test_a_bias_of_zeros_is_the_layer_without_it():
    torch.manual_seed(0)
    edges, cutoff = edges_of()
    ft = SO2FieldType({0: 4, 1: 4})
    plain = SO2MHSA(ft, 2, cutoff=cutoff, window="quartic", batched=True, dtype=D64)
    torch.manual_seed(0)
    biased = SO2MHSA(ft, 2, cutoff=cutoff, window="quartic", batched=True, relative_bias=5, dtype=D64)
    assert {n for n, _ in biased.named_parameters()} - {n for n, _ in plain.named_parameters()} == {"relative_bias"}
    x = SO2FeatureField.from_flat(ft, problems.normal((edges.row_ptr.shape[0] - 1, 12), 1))
    torch.testing.assert_close(biased(x, edges).to_flat(), plain(x, edges).to_flat(), rtol=1e-12, atol=1e-12)


def test_the_default_block_is_as_it_was():
    names = {n for n, _ in SO2TransformerBlock(SO2FieldType({0: 4, 1: 4}), 2, cutoff=1.0).named_parameters()}
    assert not any("relative" in n or "query_key" in n for n in names)


def test_modules_pickled_before_there_were_the_options_run_as_they_did():
    edges, cutoff = edges_of()
    torch.manual_seed(0)
    module = SO2TransformerBlock(SO2FieldType({0: 4, 1: 4}), 2, cutoff=cutoff, attention_batched=True, dtype=D64)
    older = pickle.loads(pickle.dumps(module))
    for m in older.modules():
        for option in ("rings", "scored", "rotated", "differential"):
            m.__dict__.pop(option, None)
    x = problems.normal((edges.row_ptr.shape[0] - 1, 12), 1)
    probe = problems.normal(x.shape, 2)
    for chunk in (None, 50):
        want, got = run(module, x, edges, probe, chunk), run(older, x, edges, probe, chunk)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("field,heads", [({0: 34, 1: 34}, 17), ({f: 2 for f in range(9)}, 1), ({0: 1028}, 1)])
def test_layers_beyond_the_ops_bounds_run_in_torch(field, heads):
    torch.manual_seed(0)
    module = SO2MHSA(SO2FieldType(field), heads, cutoff=1.0, batched=True, relative_bias=3, query_key_norm=True)

    class Rows:
        device, dtype = torch.device("cuda"), torch.float32

    class Edges:
        n_edges, max_frequency, row_ptr = 10, 16, torch.zeros(5)

    assert not relative.enabled(module, Rows(), Edges())


def test_chunks_tables_are_kept_with_the_edge_set():
    """A second pass over the same chunks builds no tables, and gives what the whole edge set gives."""
    module = layer({0: 8, 1: 4}, 2, "bias")
    edges = edges_of(2)[0]
    n = edges.row_ptr.shape[0] - 1
    x = SO2FeatureField.from_flat(module.field_type_in, problems.normal((n, 16), 1))
    kind = relative._kind(1, 9)
    from gm_attention_amd.nn import differential

    for _ in range(2):
        found = [differential.chunk_tables(c, module.cutoff, "quartic", D64, 1, kind)[0] for c in edges.chunks(60)]
    assert all(isinstance(t, RelativeEdgeTables) and t.n_buckets == 9 for t in found)
    again = [differential.chunk_tables(c, module.cutoff, "quartic", D64, 1, kind)[0] for c in edges.chunks(60)]
    assert all(a is b for a, b in zip(found, again))
    other = [differential.chunk_tables(c, module.cutoff, "quartic", D64, 1)[0] for c in edges.chunks(60)]
    assert not any(isinstance(t, RelativeEdgeTables) for t in other)
    torch.testing.assert_close(module.forward_chunked(x, edges, chunk_size=60).to_flat(), module(x, edges).to_flat(),
                               rtol=1e-10, atol=1e-12)


def test_refusals():
    ft = SO2FieldType({0: 4, 1: 4})
    f = torch.ones(1, 3)
    for kw in (dict(relative_bias=4), dict(query_key_norm=True), dict(rotary=f)):
        with pytest.raises(ValueError, match="need batched=True"):
            SO2MHSA(ft, 2, cutoff=1.0, **kw)
        with pytest.raises(ValueError, match="need mixer='attention'"):
            SO2TransformerBlock(ft, 2, cutoff=1.0, mixer="convolution", **{f"attention_{n}": v for n, v in kw.items()})
    with pytest.raises(ValueError, match="takes no relative_bias"):
        SO2MHSA(ft, 2, cutoff=1.0, batched=True, differential=True, relative_bias=4)
    for rings in (0, 257):
        with pytest.raises(ValueError, match="relative_bias must lie in"):
            SO2MHSA(ft, 2, cutoff=1.0, batched=True, relative_bias=rings)
    with pytest.raises(ValueError, match=r"frequencies must be \(axes, 3\)"):
        SO2MHSA(ft, 2, cutoff=1.0, batched=True, rotary=torch.ones(1, 4))
    edges, cutoff = edges_of()
    x = SO2FeatureField.from_flat(ft, torch.zeros(200, 12))
    at = torch.zeros(200, 1)
    plain = SO2MHSA(ft, 2, cutoff=cutoff, batched=True)
    turned = SO2MHSA(ft, 2, cutoff=cutoff, batched=True, rotary=f)
    for module, given in ((plain, at), (turned, None)):
        for call in (lambda: module(x, edges, given),
                     lambda: module.forward_chunked(x, edges, chunk_size=50, positions=given)):
            with pytest.raises(ValueError, match="positions must be given exactly"):
                call()
    with pytest.raises(ValueError, match=r"positions must be \(200, 1\)"):
        turned(x, edges, at[:7])
    conv = SO2TransformerBlock(ft, 2, cutoff=cutoff, mixer="convolution")
    with pytest.raises(ValueError, match="positions belong to"):
        conv(x, edges, at)
