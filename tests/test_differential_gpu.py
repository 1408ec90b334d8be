"""The differential neighbourhood softmax (nn/differential.py) against its
formulas and their derivatives written out in float64.

Tolerances follow the roundings.  A score of n products is off by at most
n + 4 half steps of its terms' absolute sum M (scaled, the bias with them); a
weight a = exp(s - m) / l by the score's, its row's largest score's and the
sum's: rel = (eps / 2) (64 + (n + 4) (M + max M of the row) + degree) of itself,
``64`` for the exponentials, quotients and shuffles and the logarithm's |s - lse|
(below 30 here).  T = sum a g is off by rel of sum a |g|, an edge's gradient by
2 rel of a (|g| + sum a |g|), and a row's gradient by that, summed with the
absolute values of what it multiplies, and by a half step an edge for the sum
itself.  A result held in bfloat16 is off by another eps / 2 = 2^-8 of its value.
"""

import concurrent.futures
import copy
import itertools
import math
import pickle

import pytest
import torch

import problems
from gm_attention_amd.nn import differential
from gm_attention_amd.nn.differential import EdgeTables, differential_softmax
from gm_attention_amd.representations.field_type import SO2FieldType


class Graph:
    """An edge set with float64 tables as the op's tables round them."""

    def __init__(self, row_ptr, source, transport, bias, inside, n_sources, dtype):
        self.row_ptr, self.source, self.n_sources, self.inside = row_ptr, source, n_sources, inside
        self.transport, self.bias = transport.to(dtype).double(), bias.to(dtype).double()
        self.n_targets = row_ptr.shape[0] - 1
        self.target = torch.repeat_interleave(torch.arange(self.n_targets), row_ptr[1:] - row_ptr[:-1])

    def tables(self, dtype, device):
        return EdgeTables(self.row_ptr.to(device), self.source.to(device), self.transport.to(dtype).to(device),
                          self.bias.to(dtype).to(device), self.inside.to(device), n_sources=self.n_sources)


def sphere(nlat, nlon, batch=1, window="hard", dtype=torch.float32, order=2):
    t = problems.tables(nlat, nlon, batch=batch, window=window)
    return Graph(t.row_ptr, t.source, t.transport[:, : order + 1], t.bias, t.inside, t.n_nodes, dtype)


def scattered(degrees, n_sources, dtype, outside=0.2, order=2, seed=0):
    """Rows of the given degrees with sources at random (some twice), random
    phases, biases and support; every fourth row has no edge inside."""
    g = torch.Generator().manual_seed(seed)
    row_ptr = torch.tensor([0, *itertools.accumulate(degrees)])
    E = int(row_ptr[-1])
    source = torch.randint(0, n_sources, (E,), generator=g)
    angle = 2 * math.pi * torch.rand(E, generator=g, dtype=torch.float64)
    orders = torch.arange(order + 1) * angle.unsqueeze(-1)
    inside = (torch.rand(E, generator=g) >= outside).to(torch.uint8)
    for i in range(0, len(degrees), 4):
        inside[row_ptr[i]:row_ptr[i + 1]] = 0
    bias = torch.randn(E, generator=g, dtype=torch.float64) - 3.0
    return Graph(row_ptr, source, torch.stack([torch.cos(orders), torch.sin(orders)], -1), bias, inside, n_sources,
                 dtype)


def oracle(graph, q, k, lam, g, copies, heads, eps):
    """``{name: (value, tolerance)}`` of alpha, dq, dk and dlam; a row an excluded
    edge would read is replaced by zeros there."""
    maps, n, E = 2 * heads, graph.n_targets, graph.source.numel()
    t, j = graph.target, graph.source
    scale = sum(c * (1 if f == 0 else 2) for f, c in copies.items()) ** -0.5
    use = graph.inside.bool()
    out = {name: torch.zeros(shape, dtype=torch.float64) for name, shape in
           (("alpha", (E, heads)), ("dq", q.shape), ("dk", k.shape), ("dlam", (heads,)))}
    tol = {name: torch.zeros_like(v) for name, v in out.items()}
    degree = (graph.row_ptr[1:] - graph.row_ptr[:-1]).double()
    in_degree = torch.bincount(j, minlength=k.shape[0]).double()

    def rows_of(x, index, p):
        at, got = 0, []
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            got.append(x[:, at + p * w: at + (p + 1) * w].index_select(0, index))
            at += maps * w
        return torch.where(use.unsqueeze(-1), torch.cat(got, 1), 0.0)

    def turn(x, sign):
        at, got = 0, []
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            b = x[:, at:at + w]
            if f:
                z = torch.complex(graph.transport[:, f, 0], sign * graph.transport[:, f, 1]).unsqueeze(-1)
                b = torch.view_as_real(z * torch.view_as_complex(b.reshape(E, c, 2).contiguous())).reshape(E, w)
            got.append(b)
            at += w
        return torch.cat(got, 1)

    def turn_abs(x):
        """What the turned numbers' terms sum to in absolute value."""
        at, got = 0, []
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            b = x[:, at:at + w].abs()
            if f:
                pair = b.reshape(E, c, 2)
                cos, sin = graph.transport[:, f, 0].abs()[:, None, None], graph.transport[:, f, 1].abs()[:, None, None]
                b = (cos * pair + sin * pair.flip(-1)).reshape(E, w)
            got.append(b)
            at += w
        return torch.cat(got, 1)

    def put(x, p, v, index):
        at, mine = 0, 0
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            x[:, at + p * w: at + (p + 1) * w] = torch.zeros(x.shape[0], w, dtype=x.dtype).index_add_(
                0, index, v[:, mine:mine + w])
            at, mine = at + maps * w, mine + w

    def per_target(v):
        return torch.zeros(n, dtype=torch.float64).index_add_(0, t, v)

    for p in range(maps):
        h, factor = p // 2, 1.0 if p % 2 == 0 else -lam[p // 2]
        qe, ke = rows_of(q, t, p), rows_of(k, j, p)
        tk, tka = turn(ke, 1.0), turn_abs(ke)
        s = scale * (qe * tk).sum(-1) + graph.bias
        terms = scale * (qe.abs() * tka).sum(-1) + graph.bias.abs()
        logit = torch.where(use, s, -math.inf)
        top = torch.full((n,), -math.inf, dtype=torch.float64).scatter_reduce(0, t, logit, "amax")
        w = torch.where(use, torch.exp(logit - top[t]), 0.0)
        total = per_target(w)
        w = torch.where(use, w / total[t], 0.0)
        most = torch.zeros(n, dtype=torch.float64).scatter_reduce(0, t, torch.where(use, terms, 0.0), "amax")
        products = 4 * qe.shape[1] + 4
        rel = eps / 2 * (64 + products * (terms + most[t]) + degree[t])
        out["alpha"][:, h] += factor * w
        tol["alpha"][:, h] += abs(factor) * w * (rel + eps)
        ge = torch.where(use, g[:, h], 0.0)
        T, Ta = per_target(w * ge), per_target(w * ge.abs())
        if p % 2:
            out["dlam"][h] = -T.sum()
            tol["dlam"][h] = (w * ge.abs() * rel).sum() + eps * T.abs().sum()
        ds = scale * factor * w * (ge - T[t])
        row_rel = torch.zeros(n, dtype=torch.float64).scatter_reduce(0, t, torch.where(use, rel, 0.0), "amax")[t]
        dsa = scale * abs(factor) * w * (ge.abs() + Ta[t])
        put(out["dq"], p, ds.unsqueeze(-1) * tk, t)
        put(tol["dq"], p, (dsa * (2 * row_rel + eps / 2 * degree[t])).unsqueeze(-1) * tka, t)
        put(out["dk"], p, ds.unsqueeze(-1) * turn(qe, -1.0), j)
        put(tol["dk"], p, (dsa * (2 * row_rel + eps / 2 * in_degree[j])).unsqueeze(-1) * turn_abs(qe), j)
    return {name: (out[name], tol[name]) for name in out}


def compare(got, want, name):
    value, tol = want
    if got.dtype == torch.bfloat16:
        tol = tol + torch.finfo(torch.bfloat16).eps / 2 * (value.abs() + tol)
    tol = tol + torch.finfo(torch.float32).tiny
    off = (got.detach().double().cpu() - value).abs()
    assert got.shape == value.shape, name
    assert bool((off <= tol).all()), f"{name}: {float((off / tol).nan_to_num(math.inf).max())} of the tolerance"


def inputs(graph, copies, heads, rows, seed=0):
    D = 2 * heads * sum(c * (1 if f == 0 else 2) for f, c in copies.items())
    table = torch.float64 if rows == torch.float64 else torch.float32
    q = problems.normal((graph.n_targets, D), seed).to(rows).double()
    k = problems.normal((graph.n_sources, D), seed + 1).to(rows).double()
    lam = (0.2 + 0.6 * problems.normal((heads,), seed + 2).abs()).to(table).double()
    g = problems.normal((graph.source.numel(), heads), seed + 3).to(table).double()
    return q, k, lam, g


def run(graph, tables, q, k, lam, g, copies, heads, rows, device):
    leaves = [q.to(rows).to(device).requires_grad_(True), k.to(rows).to(device).requires_grad_(True),
              lam.to(tables.dtype).to(device).requires_grad_(True)]
    alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
    assert alpha.dtype == tables.dtype
    with torch.no_grad():
        assert torch.equal(differential_softmax(*leaves, tables, SO2FieldType(copies), heads), alpha)
    grads = torch.autograd.grad(alpha, leaves, g.to(tables.dtype).to(device))
    assert [x.dtype for x in grads] == [rows, rows, tables.dtype]
    return dict(zip(("alpha", "dq", "dk", "dlam"), (alpha, *grads)))


def check(graph, copies, heads, rows, device, seed=0):
    print(f"differential {copies} H={heads} {rows} N={graph.n_targets} E={graph.source.numel()}", flush=True)
    table = torch.float64 if rows == torch.float64 else torch.float32
    values = inputs(graph, copies, heads, rows, seed)
    got = run(graph, graph.tables(table, device), *values, copies, heads, rows, device)
    want = oracle(graph, *values, copies, heads, torch.finfo(table).eps)
    for name in want:
        compare(got[name], want[name], name)


#: copies a map and heads: every lane arrangement, odd copies, three frequencies with a gap, one frequency alone
LAYOUTS = [({0: 2, 1: 2, 2: 2}, 8), ({0: 2, 1: 2, 2: 2}, 4), ({0: 2, 1: 2, 2: 2}, 1), ({0: 2, 1: 2, 2: 2}, 16),
           ({0: 4, 1: 4, 2: 4}, 8), ({0: 4, 1: 4, 2: 4}, 16), ({0: 8, 1: 8, 2: 8}, 2), ({0: 1, 1: 1, 2: 1}, 8),
           ({0: 1, 1: 1, 2: 1}, 1), ({0: 2, 1: 1, 2: 1}, 6), ({0: 4, 1: 2, 2: 2}, 4), ({0: 8, 1: 4, 2: 4}, 8),
           ({0: 2, 1: 2}, 4), ({0: 1, 1: 1}, 3), ({0: 4, 1: 2, 2: 1}, 8), ({0: 3, 1: 2, 2: 1}, 6),
           ({0: 3, 1: 2, 2: 1}, 5),
           ({0: 2, 2: 2}, 4), ({1: 2}, 2), ({0: 5}, 7), ({0: 3, 1: 5, 2: 2}, 3), ({0: 2, 1: 2, 2: 2}, 6)]
ROWS = [torch.float32, torch.bfloat16, torch.float64]


def tables_dtype(rows):
    return torch.float64 if rows == torch.float64 else torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", LAYOUTS)
def test_every_layout_and_type(copies, heads, rows, cuda):
    check(sphere(10, 20, window="quartic", dtype=tables_dtype(rows)), copies, heads, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 2, 1: 2, 2: 2}, 8), ({0: 2, 1: 2, 2: 2}, 2), ({0: 4, 1: 4, 2: 4}, 16),
                                          ({0: 3, 1: 5, 2: 2}, 3)])
def test_lengths_of_rows(copies, heads, rows, cuda):
    """No edge, one, and around every number of edges a step, a batch, a wave and a
    workgroup hold; sources twice in a row, rows with nothing inside, more and
    fewer sources than targets."""
    degrees = [0, 1, 1, 2, 3, 0, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 130, 200, 255,
               256, 257, 300, 511, 512, 513, 700, 1, 0]
    for n_sources in (11, 400):
        check(scattered(degrees, n_sources, tables_dtype(rows)), copies, heads, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("copies,heads", [({0: 2, 1: 2, 2: 2}, 8), ({0: 2, 1: 2, 2: 2}, 4), ({0: 4, 1: 4, 2: 4}, 16)])
def test_rows_longer_than_a_workgroup_holds(copies, heads, rows, cuda):
    check(scattered([5, 1023, 2048, 2049, 4500, 3], 50, torch.float32), copies, heads, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
def test_masked_rows_may_hold_anything(rows, cuda):
    """Nodes whose every edge is outside hold NaN, infinities and the type's extremes,
    and the bias of those edges too: nothing of them is seen."""
    dtype, copies, heads = tables_dtype(rows), {0: 2, 1: 2, 2: 2}, 4
    graph = sphere(10, 20, dtype=dtype)
    gone = torch.zeros(graph.n_targets, dtype=torch.bool)
    gone[30:95] = True
    graph.inside = graph.inside * (~(gone[graph.target] | gone[graph.source])).to(torch.uint8)
    assert bool((torch.zeros(graph.n_targets).index_add_(0, graph.target, graph.inside.float()) == 0).any())
    q, k, lam, g = inputs(graph, copies, heads, rows)
    odd = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(rows).min, torch.finfo(rows).max])
    for x in (q, k):
        x[gone] = odd.double()[torch.arange(int(gone.sum()) * x.shape[1]) % 5].reshape(-1, x.shape[1])
    out = graph.inside == 0
    graph.bias[out] = odd.double()[torch.arange(int(out.sum())) % 4]
    g = torch.where(out.unsqueeze(-1), math.nan, g)
    got = run(graph, graph.tables(dtype, cuda), q, k, lam, g, copies, heads, rows, cuda)
    clean = [torch.where(gone.unsqueeze(-1), 0.0, x) for x in (q, k)]
    graph.bias[out] = 0.0
    want = oracle(graph, *clean, lam, torch.where(out.unsqueeze(-1), 0.0, g), copies, heads, torch.finfo(dtype).eps)
    for name in want:
        compare(got[name], want[name], name)
    assert bool((got["dq"][gone.to(cuda)] == 0).all()) and bool((got["dk"][gone.to(cuda)] == 0).all())
    assert bool((got["alpha"][out.to(cuda)] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 2, 1: 2, 2: 2}, 8), ({0: 4, 1: 4, 2: 4}, 16), ({0: 3, 1: 2, 2: 1}, 3)])
def test_rows_of_no_number_leave_the_edges_outside(copies, heads, rows, cuda):
    """A key that is no number makes the weights of the rows that read it no numbers, of its head alone and not those of
    the edges outside the window: these stay zero and add nothing to any gradient."""
    edges_outside(copies, heads, rows, cuda)


@pytest.mark.parametrize("rows", ROWS)
def test_rows_of_no_number_on_the_cpu(rows):
    edges_outside({0: 3, 1: 2, 2: 1}, 2, rows, "cpu")


def edges_outside(copies, heads, rows, device):
    dtype = tables_dtype(rows)
    graph = scattered([1, 2, 9, 40, 6, 300, 1, 700, 3, 2100, 5200, 64], 60, dtype, outside=0.4)
    q, k, lam, g = inputs(graph, copies, heads, rows)
    use = graph.inside.bool()
    bad = torch.zeros(graph.n_targets, dtype=torch.bool)
    bad[graph.target[use & (graph.source == 7)]] = True
    assert 3 <= int(bad.sum()) < graph.n_targets - 3
    nan = use & bad[graph.target]
    tables, results = graph.tables(dtype, device), []
    for value in (0.0, math.nan):
        k[7, 2 * copies[0]] = value  # the first number of the second head's first map
        leaves = [x.to(to).to(device, copy=True).requires_grad_(True)
                  for x, to in ((q, rows), (k, rows), (lam, dtype))]
        alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
        grads = torch.autograd.grad(alpha, leaves[:2], g.to(dtype).to(device))
        results.append([x.detach().cpu() for x in (alpha, *grads)])
    columns, at = torch.zeros(q.shape[1], dtype=torch.bool), 0
    for f, c in copies.items():
        w = c * (1 if f == 0 else 2)
        columns[at + 2 * w:at + 3 * w] = True
        at += 2 * heads * w
    sources = torch.zeros(graph.n_sources, dtype=torch.bool)
    sources[graph.source[nan]] = True
    expected = (nan.unsqueeze(1) & (torch.arange(heads) == 1), bad.unsqueeze(1) & columns,
                sources.unsqueeze(1) & columns)
    assert bool((results[1][0][~use] == 0).all())
    for name, clean, got, where in zip(("alpha", "dq", "dk"), *results, expected):
        assert torch.equal(got.isnan(), where), name
        assert torch.equal(got[~where], clean[~where]), name


@pytest.mark.gpu
def test_biases_of_the_lowest_value_inside_the_window(cuda):
    """A row whose every bias is the type's lowest is uniform; beside an ordinary
    one such an edge has weight zero; a row of -inf biases has none inside."""
    lowest = torch.finfo(torch.float32).min
    graph = scattered([4, 4, 4], 6, torch.float32, outside=0.0)
    graph.inside[:] = 1
    graph.bias[:] = torch.tensor([lowest] * 4 + [0.0, lowest, 0.0, lowest] + [-math.inf] * 4).double()
    q, k, lam, g = inputs(graph, {0: 2, 1: 2, 2: 2}, 2, torch.float32)
    got = run(graph, graph.tables(torch.float32, cuda), q, k, lam, g, {0: 2, 1: 2, 2: 2}, 2, torch.float32, cuda)
    alpha = got["alpha"].cpu()
    torch.testing.assert_close(alpha[:4], (0.25 - 0.25 * lam).float().expand(4, 2))
    assert bool((alpha[[5, 7]] == 0).all()) and bool((alpha[8:] == 0).all())
    assert all(bool(torch.isfinite(x).all()) for x in got.values())


def bounds(graph, q, k, lam, g, copies, eps):
    """What a row's gradient may be off by where its weights sum to one: (64 + degree) half steps of the weights and
    as many of T, of a sum of a (|g| + T) |tau k| <= 2 max|g| sqrt(2) max|k|; a source's of its edges' sum."""
    q, k, lam, g = (t.detach() for t in (q, k, lam, g))
    scale = sum(c * (1 if f == 0 else 2) for f, c in copies.items()) ** -0.5
    degree = float((graph.row_ptr[1:] - graph.row_ptr[:-1]).max())
    sources = float(torch.bincount(graph.source).max())
    each = eps * scale * max(1.0, float(lam.abs().max())) * 2 * float(g.abs().max()) * 2 ** 0.5
    return (64 + degree) * each * float(k.abs().max()), (64 + degree + sources) * each * float(q.abs().max()) * sources


def assert_within(got, want, name, tol):
    if got.dtype == torch.bfloat16:
        tol = tol + torch.finfo(torch.bfloat16).eps / 2 * (want.abs() + tol)
    off = (got.detach().double().cpu() - want).abs()
    assert bool((off <= tol).all()), f"{name}: off by {float(off.max())}"


BIASED = [({0: 2, 1: 2, 2: 2}, 8, torch.float32), ({0: 2, 1: 2, 2: 2}, 8, torch.bfloat16),
          ({0: 4, 1: 4, 2: 4}, 4, torch.float32), ({0: 3, 1: 2}, 3, torch.float32), ({0: 3, 1: 2}, 3, torch.bfloat16),
          ({0: 2, 1: 2, 2: 2}, 2, torch.float64)]
DEGREES = [4, 1, 0, 7, 40, 140, 600]


@pytest.mark.gpu
@pytest.mark.parametrize("copies,heads,rows", BIASED)
def test_gradients_of_rows_whose_biases_are_all_the_lowest_value(copies, heads, rows, cuda):
    """Such a row's scores are all its bias, in any type: its weights are 1 / degree, forward and backward."""
    table = tables_dtype(rows)
    graph = scattered(DEGREES, 30, table, outside=0.0)
    graph.inside[:] = 1
    graph.bias[:] = torch.finfo(table).min
    q, k, lam, g = inputs(graph, copies, heads, rows)
    got = run(graph, graph.tables(table, cuda), q, k, lam, g, copies, heads, rows, cuda)
    want = run(graph, graph.tables(torch.float64, "cpu"), q, k, lam, g, copies, heads, torch.float64, "cpu")
    uniform = (1.0 / (graph.row_ptr[1:] - graph.row_ptr[:-1]).double())[graph.target]
    torch.testing.assert_close(want["alpha"], uniform.unsqueeze(-1) * (1 - lam), rtol=1e-12, atol=1e-14)
    eps = torch.finfo(table).eps
    tol_q, tol_k = bounds(graph, q, k, lam, g, copies, eps)
    assert_within(got["alpha"], want["alpha"], "alpha", 2 * (64 + max(DEGREES)) * eps * want["alpha"].abs() + eps)
    assert_within(got["dq"], want["dq"], "dq", tol_q)
    assert_within(got["dk"], want["dk"], "dk", tol_k)
    assert_within(got["dlam"], want["dlam"], "dlam", len(DEGREES) * (64 + max(DEGREES)) * eps * float(g.abs().max()))


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [12, 20, 29])
@pytest.mark.parametrize("copies,heads,rows", BIASED)
def test_weights_of_the_backward_are_the_forwards_beside_large_biases(copies, heads, rows, exponent, cuda):
    """A gradient that is the same for every edge meets weights that sum to one: nothing is left of it in the
    rows, whatever the scores' own rounding beside biases of up to -2^29 (-2^60 in float64)."""
    table = tables_dtype(rows)
    graph = scattered(DEGREES, 30, table, outside=0.0)
    graph.inside[:] = 1
    graph.bias -= 2.0 ** (exponent if table == torch.float32 else 2 * exponent + 2)
    graph.bias = graph.bias.to(table).double()
    q, k, lam, g = inputs(graph, copies, heads, rows)
    g = g[:1].expand_as(g)
    got = run(graph, graph.tables(table, cuda), q, k, lam, g, copies, heads, rows, cuda)
    eps = torch.finfo(table).eps
    tol_q, tol_k = bounds(graph, q, k, lam, g, copies, eps)
    assert_within(got["dq"], torch.zeros_like(q), "dq", tol_q)
    assert_within(got["dk"], torch.zeros_like(k), "dk", tol_k)
    filled = sum(d > 0 for d in DEGREES)
    assert_within(got["dlam"], -filled * g[0], "dlam", filled * (64 + max(DEGREES)) * eps * float(g.abs().max()))
    sums = torch.zeros(len(DEGREES), heads, dtype=torch.float64).index_add_(0, graph.target, got["alpha"].detach().double().cpu())
    assert_within(sums, (torch.tensor(DEGREES) > 0).double().unsqueeze(-1) * (1 - lam), "sums", 2 * (64 + max(DEGREES)) * eps)


@pytest.mark.gpu
@pytest.mark.parametrize("common", [0.0, 10.0, 1000.0])
@pytest.mark.parametrize("copies,heads,rows", BIASED)
def test_gradients_with_a_common_part(copies, heads, rows, common, cuda):
    """What a smooth field's values give: the weights' gradients of a row nearly alike, and its keys too.  The
    part they share cancels, and leaves the roundings it had (the oracle's bounds count |g| whole)."""
    table = tables_dtype(rows)
    graph = scattered(DEGREES, 30, table)
    q, k, lam, g = inputs(graph, copies, heads, rows)
    k = (k + common / 100).to(rows).double()
    g = (g + common).to(table).double()
    got = run(graph, graph.tables(table, cuda), q, k, lam, g, copies, heads, rows, cuda)
    want = oracle(graph, q, k, lam, g, copies, heads, torch.finfo(table).eps)
    for name in want:
        compare(got[name], want[name], name)


@pytest.mark.gpu
def test_sources_at_the_far_end_of_a_large_table(cuda):
    """Key rows whose offsets pass 2^31 numbers."""
    copies, heads, n = {0: 2, 1: 2, 2: 2}, 8, 13_600_000  # 160 numbers a row: 2.2e9
    graph = scattered([3, 40, 70, 0, 5], 64, torch.float32)
    near = graph.source.clone()
    q, k, lam, g = inputs(graph, copies, heads, torch.bfloat16)
    want = oracle(graph, q, k, lam, g, copies, heads, torch.finfo(torch.float32).eps)
    graph.source, graph.n_sources = near + (n - 64), n
    tables = graph.tables(torch.float32, cuda)
    far = torch.zeros(n, 160, dtype=torch.bfloat16, device=cuda)
    far[n - 64:] = k.to(torch.bfloat16).to(cuda)
    leaves = [q.bfloat16().to(cuda).requires_grad_(True), far.requires_grad_(True), lam.float().to(cuda)]
    alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
    dq, dk = torch.autograd.grad(alpha, leaves[:2], g.float().to(cuda))
    compare(alpha, want["alpha"], "alpha")
    compare(dq, want["dq"], "dq")
    compare(dk[n - 64:], want["dk"], "dk")
    assert not bool(dk[: n - 64].any())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_rows_at_odd_addresses_and_strides(rows, cuda):
    copies, heads = {0: 2, 1: 2, 2: 2}, 4
    graph = sphere(10, 20)
    q, k, lam, g = inputs(graph, copies, heads, rows)
    want = oracle(graph, q, k, lam, g, copies, heads, torch.finfo(torch.float32).eps)
    tables = graph.tables(torch.float32, cuda)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape).copy_(t)

    def strided(t):
        return torch.empty(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device=cuda)[:, 3:-2].copy_(t)

    for view in (shifted, strided):
        leaves = [view(q.to(rows)).requires_grad_(True), view(k.to(rows)).requires_grad_(True),
                  lam.float().to(cuda).requires_grad_(True)]
        alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
        up = view(g.float())  # a gradient with gaps between its rows
        grads = torch.autograd.grad(alpha, leaves, up)
        for name, x in zip(("alpha", "dq", "dk", "dlam"), (alpha, *grads)):
            compare(x, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("copies,heads", [({0: 2, 1: 2, 2: 2}, 8), ({0: 3, 1: 2}, 2)])
def test_gradients_against_differences(copies, heads, cuda):
    """In float64, along random directions: the fourth-order difference at step
    1e-3 is off by h^4 f^(5) / 30, about 1e-13 here, and by roundings of 1e-16 / h
    of the loss's magnitude."""
    graph = sphere(8, 16, window="quartic", dtype=torch.float64)
    values = inputs(graph, copies, heads, torch.float64)
    tables = graph.tables(torch.float64, cuda)
    start, up = [v.to(cuda) for v in values[:3]], values[3].to(cuda)
    map_type = SO2FieldType(copies)
    leaves = [v.clone().requires_grad_(True) for v in start]
    grads = torch.autograd.grad(differential_softmax(*leaves, tables, map_type, heads), leaves, up)
    for i in range(3):
        step = problems.normal(start[i].shape, 70 + i).to(cuda)

        def at(h):
            moved = [v + h * step if n == i else v for n, v in enumerate(start)]
            return float((differential_softmax(*moved, tables, map_type, heads) * up).sum())

        h = 1e-3
        slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        want = float((grads[i] * step).sum())
        assert abs(slope - want) <= 1e-7 * (1 + abs(want)), (i, slope, want)


@pytest.mark.gpu
def test_turning_the_frames_leaves_the_weights(cuda):
    """Gauge equivariance: turning every node's frame turns its rows and the
    transports with them; the weights stay."""
    copies, heads = {0: 2, 1: 2, 2: 2}, 4
    graph = sphere(10, 20, dtype=torch.float64)
    q, k, lam, _ = inputs(graph, copies, heads, torch.float64)
    theta = 6.0 * problems.normal((graph.n_targets,), 9)

    def turned(x):
        blocks, at = [], 0
        for f, c in copies.items():
            w = 2 * heads * c * (1 if f == 0 else 2)
            b = x[:, at:at + w]
            if f:
                z = torch.polar(torch.ones_like(theta), f * theta).unsqueeze(-1)
                b = torch.view_as_real(z * torch.view_as_complex(b.reshape(len(x), -1, 2).contiguous()))
                b = b.reshape(len(x), w)
            blocks.append(b)
            at += w
        return torch.cat(blocks, 1)

    def alpha(g, q, k):
        return differential_softmax(q.to(cuda), k.to(cuda), lam.to(cuda), g.tables(torch.float64, cuda),
                                    SO2FieldType(copies), heads)

    before = alpha(graph, q, k)
    phase = torch.view_as_complex(graph.transport.contiguous())
    shift = (theta[graph.target] - theta[graph.source]).unsqueeze(-1) * torch.arange(3)
    graph.transport = torch.view_as_real(phase * torch.polar(torch.ones_like(shift), shift))
    torch.testing.assert_close(alpha(graph, turned(q), turned(k)), before, rtol=1e-11, atol=1e-13)


@pytest.mark.gpu
def test_replays_of_a_captured_step_equal_the_eager_one(cuda):
    copies, heads = {0: 2, 1: 2, 2: 2}, 8
    graph = sphere(12, 24, batch=2)
    q, k, lam, g = (v.float().to(cuda) for v in inputs(graph, copies, heads, torch.float32))
    tables = graph.tables(torch.float32, cuda)

    def step():
        leaves = [v.detach().requires_grad_(True) for v in (q, k, lam)]
        alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
        return [alpha.detach(), *torch.autograd.grad(alpha, leaves, g)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        got = step()
    for replay in range(3):
        for t in got:
            t.zero_()
        captured.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), replay
        assert all(torch.equal(a, b) for a, b in zip(step(), want)), replay
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_tables_are_built_before_a_capture(cuda):
    graph = sphere(8, 16)
    q, k, lam, g = (v.float().to(cuda) for v in inputs(graph, {0: 2, 1: 2}, 2, torch.float32))
    tables = graph.tables(torch.float32, cuda)
    given = [graph.row_ptr.to(cuda), graph.source.to(cuda), graph.transport.float().to(cuda),
             graph.bias.float().to(cuda), graph.inside.to(cuda)]
    torch.cuda.synchronize()
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        held = q * 1.0
        with pytest.raises(RuntimeError, match="before the capture"):
            EdgeTables(*given)
        with pytest.raises(RuntimeError, match="before the capture"):
            differential_softmax(q.requires_grad_(True), k, lam, tables, SO2FieldType({0: 2, 1: 2}), 2)
    captured.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, q)


@pytest.mark.gpu
def test_inference_needs_no_source_side(cuda):
    """Under no_grad a layer's parameters still require gradients: the op neither sorts
    the edges by source nor needs that done before a capture."""
    copies, heads = {0: 2, 1: 2, 2: 2}, 8
    graph = sphere(8, 16)
    q, k, lam, g = (v.float().to(cuda) for v in inputs(graph, copies, heads, torch.float32))
    tables, maps = graph.tables(torch.float32, cuda), SO2FieldType(copies)
    lam = torch.nn.Parameter(lam)
    with torch.no_grad():
        want = differential_softmax(q, k, lam, tables, maps, heads)
        torch.cuda.synchronize()
        captured = torch.cuda.CUDAGraph()
        with torch.cuda.graph(captured):
            got = differential_softmax(q, k, lam, tables, maps, heads)
        for _ in range(3):
            got.zero_()
            captured.replay()
            torch.cuda.synchronize()
            assert torch.equal(got, want)
            assert torch.equal(differential_softmax(q, k, lam, tables, maps, heads), want)
    assert tables._sources is None
    alpha = differential_softmax(q, k, lam, tables, maps, heads)
    assert torch.equal(alpha, want) and tables._sources is not None


@pytest.mark.gpu
def test_two_threads_at_once(cuda):
    """Two threads' first steps over the same new tables, each on its own stream."""
    copies, heads = {0: 2, 1: 2, 2: 2}, 8
    graph = sphere(12, 24, batch=2)
    q, k, lam, g = (v.float().to(cuda) for v in inputs(graph, copies, heads, torch.float32))

    def step(tables):
        leaves = [v.detach().requires_grad_(True) for v in (q, k, lam)]
        alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
        return [alpha.detach(), *torch.autograd.grad(alpha, leaves, g)]

    want = step(graph.tables(torch.float32, cuda))
    tables = graph.tables(torch.float32, cuda)
    torch.cuda.synchronize()

    def work(_):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            out = [step(tables) for _ in range(5)]
        stream.synchronize()
        return out

    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        runs = list(pool.map(work, range(2)))
    assert all(torch.equal(a, b) for run in runs for got in run for a, b in zip(got, want))


@pytest.mark.gpu
def test_on_another_stream(cuda):
    """Tables built on one stream behind other work, read on another at once."""
    copies, heads = {0: 2, 1: 2, 2: 2}, 8
    graph = sphere(24, 48)
    q, k, lam, g = (v.float().to(cuda) for v in inputs(graph, copies, heads, torch.float32))

    def step(tables):
        leaves = [v.detach().requires_grad_(True) for v in (q, k, lam)]
        alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
        return [alpha.detach(), *torch.autograd.grad(alpha, leaves, g)]

    want = step(graph.tables(torch.float32, cuda))
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=cuda)
    for _ in range(20):
        busy = busy @ busy * 1e-3
    tables = graph.tables(torch.float32, cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(tables)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_tables_written_to_afterwards_are_not_seen(cuda):
    copies, heads = {0: 2, 1: 2, 2: 2}, 8
    graph = sphere(10, 20)
    q, k, lam, g = (v.float().to(cuda) for v in inputs(graph, copies, heads, torch.float32))
    given = [graph.row_ptr.to(cuda), graph.source.to(cuda), graph.transport.float().to(cuda),
             graph.bias.float().to(cuda), graph.inside.to(cuda)]
    tables = EdgeTables(*given)

    def step():
        leaves = [v.detach().requires_grad_(True) for v in (q, k, lam)]
        alpha = differential_softmax(*leaves, tables, SO2FieldType(copies), heads)
        return [alpha.detach(), *torch.autograd.grad(alpha, leaves, g)]

    want = step()
    for t in given[2:]:
        t.zero_()
    assert all(torch.equal(a, b) for a, b in zip(step(), want))


@pytest.mark.gpu
def test_no_targets_and_no_edges(cuda):
    map_type = SO2FieldType({0: 2, 1: 2})
    for n, m in ((0, 0), (0, 5), (4, 0), (4, 5)):
        tables = EdgeTables(torch.zeros(n + 1, dtype=torch.int64, device=cuda),
                            torch.zeros(0, dtype=torch.int64, device=cuda), torch.zeros(0, 2, 2, device=cuda),
                            torch.zeros(0, device=cuda), torch.zeros(0, dtype=torch.uint8, device=cuda), n_sources=m)
        leaves = [torch.ones(*shape, device=cuda, requires_grad=True) for shape in ((n, 24), (m, 24), (2,))]
        alpha = differential_softmax(*leaves, tables, map_type, 2)
        assert alpha.shape == (0, 2)
        for x, grad in zip(leaves, torch.autograd.grad(alpha, leaves, alpha.detach())):
            assert grad.shape == x.shape and not bool(grad.any())


# ---------------------------------------------------------------- without a GPU


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 2, 1: 2, 2: 2}, 3), ({1: 1, 2: 3}, 2), ({0: 5}, 1)])
def test_cpu_rows_take_the_formulas_in_torch(copies, heads, rows):
    check(scattered([0, 1, 5, 9, 40, 3, 70, 0, 8], 13, tables_dtype(rows)), copies, heads, rows, "cpu")


def test_the_oracle_is_the_single_softmax_at_lambda_zero():
    from oracle import eager

    t = problems.tables(8, 16, window="quartic")
    copies, heads = {0: 2, 1: 2, 2: 2}, 3
    graph = Graph(t.row_ptr, t.source, t.transport[:, :3], t.bias, t.inside, t.n_nodes, torch.float64)
    q, k, _, g = inputs(graph, copies, heads, torch.float64)
    want = oracle(graph, q, k, torch.zeros(heads, dtype=torch.float64), g, copies, heads, 1e-16)["alpha"][0]
    plan = differential.maps_of(SO2FieldType(copies), heads).plan
    single = eager.softmax_op(q, k, graph.transport, graph.bias, graph.inside, plan.rows, graph.row_ptr, graph.source,
                              2 * heads, 10 ** -0.5)
    torch.testing.assert_close(want, single[:, 0::2], rtol=1e-12, atol=1e-14)


def test_refusals():
    row_ptr, source = torch.tensor([0, 2, 3]), torch.tensor([0, 1, 1])
    phases, bias, inside = torch.zeros(3, 2, 2), torch.zeros(3), torch.ones(3, dtype=torch.uint8)

    def tables(**kw):
        given = dict(row_ptr=row_ptr, source=source, transport=phases, bias=bias, inside=inside)
        n = kw.pop("n_sources", None)
        given.update(kw)
        return EdgeTables(*given.values(), n_sources=n)

    for kw, message in ((dict(row_ptr=row_ptr.int()), "row_ptr must be int64"),
                        (dict(source=source.int()), "source must"),
                        (dict(transport=phases[:2]), r"transport must be \(3, orders, 2\)"),
                        (dict(transport=phases.half()), "float32 or float64"),
                        (dict(bias=bias.double()), "bias must be"),
                        (dict(bias=bias[:2]), "bias must be"), (dict(inside=inside.long()), "inside must be"),
                        (dict(row_ptr=torch.tensor([0, 2, 2])), "row_ptr must rise"),
                        (dict(row_ptr=torch.tensor([1, 2, 3])), "row_ptr must rise"),
                        (dict(row_ptr=torch.tensor([0, 4, 3])), "row_ptr must rise"),
                        (dict(source=torch.tensor([0, 2, 1])), "every source"),
                        (dict(source=torch.tensor([0, -1, 1])), "every source"), (dict(n_sources=1), "every source")):
        with pytest.raises(ValueError, match=message):
            tables(**kw)
    t, map_type = tables(), SO2FieldType({0: 2, 1: 1})
    q, lam = torch.zeros(2, 16), torch.zeros(2)
    assert differential_softmax(q, q, lam, t, map_type, 2).shape == (3, 2)
    for call, message in (((q.double(), q.double(), lam), "share a dtype"), ((q, q.double(), lam), "share a dtype"),
                          ((q.half(), q.half(), lam), "share a dtype"), ((q[:1], q, lam), "q and k must be"),
                          ((q, q[:, :8], lam), "q and k must be"), ((q, q, lam[:1]), r"lam must be \(2,\)")):
        with pytest.raises(ValueError, match=message):
            differential_softmax(*call, t, map_type, 2)
    with pytest.raises(ValueError, match="heads must lie in 1..16"):
        differential_softmax(q, q, lam, t, map_type, 17)
    with pytest.raises(ValueError, match="at most 8 frequencies and 1024"):
        differential_softmax(q, q, lam, t, SO2FieldType({0: 600}), 1)
    with pytest.raises(ValueError, match="orders below 2, the maps need 2"):
        differential_softmax(torch.zeros(2, 16), torch.zeros(2, 16), lam, t, SO2FieldType({0: 2, 2: 1}), 2)


def test_the_library_refuses_bad_arguments():
    """Through the C interface, before anything is launched (no GPU touched)."""
    import ctypes

    from gm_attention_amd import _native

    lib = _native.library()

    def forward(rows=((0, 2, 0, 0, 1), (1, 1, 8, 0, 2)), n=0, D=16, orders=2, H=2, F=None):
        flat = [x for row in rows for x in row]
        desc = (ctypes.c_int64 * len(flat))(*flat)
        return lib.gm_differential_forward_f32(None, None, None, None, ctypes.cast(desc, ctypes.c_void_p), None, None,
                                               None, n, 0, 0, D, orders, len(rows) if F is None else F, H, 1.0, None,
                                               None, None)

    assert forward() == 0
    for kw, message in ((dict(n=-1), b"non-negative"), (dict(n=1), b"device pointers"),
                        (dict(H=17), b"at most 16 heads"), (dict(D=1025), b"D must be in"),
                        (dict(D=20), b"fill the flat width"), (dict(orders=1), b"exceeds"),
                        (dict(F=9), b"1 to 8"), (dict(n=2**31), b"32 bits"),
                        (dict(rows=((1, 1, 0, 0, 2), (0, 2, 8, 0, 1))), b"must rise"),
                        (dict(rows=((0, 2, 4, 0, 1), (1, 1, 8, 0, 2))), b"follow each other")):
        assert forward(**kw) == 1
        assert message in lib.gm_last_error(), kw


def test_maps_made_under_a_default_device_serve_every_call():
    """The layout the library reads on the host is in host memory, whatever device was the default."""
    map_type, graph = SO2FieldType({0: 4, 1: 4, 2: 4}), scattered([3, 1, 4], 5, torch.float32)
    tables = graph.tables(torch.float32, "cpu")
    with torch.device("meta"):
        held = differential.maps_of(map_type, 3)
    assert differential.maps_of(map_type, 3) is held
    assert held.desc.device.type == "cpu" and held.slots(tables) == 4


# ------------------------------------------------------------- copies of the tables


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.float64])
def test_copied_tables_give_the_same_results(rows, cuda, tmp_path):
    copies, heads = {0: 2, 1: 2, 2: 2}, 4
    graph = scattered([3, 0, 70, 9, 1, 200], 40, rows)
    tables = graph.tables(rows, cuda)
    values = inputs(graph, copies, heads, rows)
    want = run(graph, tables, *values, copies, heads, rows, cuda)
    torch.save(tables, tmp_path / "tables")
    for other in (copy.deepcopy(tables), pickle.loads(pickle.dumps(tables)),
                  torch.load(tmp_path / "tables", weights_only=False)):
        got = run(graph, other, *values, copies, heads, rows, cuda)
        assert all(torch.equal(got[n], want[n]) for n in want)
    read = torch.load(tmp_path / "tables", weights_only=False, map_location="cpu")
    assert read.device.type == "cpu"
    got = run(graph, read, *values, copies, heads, rows, "cpu")
    want = oracle(graph, *values, copies, heads, torch.finfo(rows).eps)
    for name in want:  # the biases were kept in units of log 2: two roundings, of the many the bound counts for them
        compare(got[name], want[name], name)


@pytest.mark.parametrize("rows", ROWS)
def test_masked_rows_may_hold_anything_on_the_cpu(rows):
    test_masked_rows_may_hold_anything(rows, "cpu")


def test_derivatives_of_every_kind_on_the_cpu():
    """Backward, forward and second derivatives, and functions of functions."""
    copies, heads = {0: 2, 1: 1}, 2
    graph = scattered([1, 3, 4, 6], 5, torch.float64, outside=0.3)
    *leaves, _ = inputs(graph, copies, heads, torch.float64)
    tables = graph.tables(torch.float64, "cpu")

    def weights(q, k, extra):
        return differential_softmax(q, k, extra, tables, SO2FieldType(copies), heads)

    given = [x.requires_grad_(True) for x in leaves]
    assert torch.autograd.gradcheck(weights, given, check_forward_ad=True)
    assert torch.autograd.gradgradcheck(weights, given)
    q, k, extra = (x.detach() for x in leaves)

    def loss(q):
        return weights(q, k, extra).square().sum()

    (want,) = torch.autograd.grad(loss(given[0]), given[:1])
    torch.testing.assert_close(torch.func.grad(loss)(q), want)
    torch.testing.assert_close(torch.func.vmap(torch.func.grad(loss))(torch.stack([q, 2 * q]))[0], want)


def test_copied_tables_on_the_cpu_give_the_same_results():
    copies, heads, rows = {0: 2, 1: 2}, 2, torch.float64
    graph = scattered([3, 0, 70, 9, 1], 40, rows)
    tables = graph.tables(rows, "cpu")
    values = inputs(graph, copies, heads, rows)
    want = run(graph, tables, *values, copies, heads, rows, "cpu")
    for other in (copy.deepcopy(tables), pickle.loads(pickle.dumps(tables))):
        got = run(graph, other, *values, copies, heads, rows, "cpu")
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_what_a_stream_made_stays_out_of_a_copy():
    """Beside the tables their owner keeps the events of the streams that made them, which are not copied."""
    tables = scattered([3, 0, 7], 4, torch.float64).tables(torch.float64, "cpu")
    tables._kept = [torch.cuda.Event.__new__(torch.cuda.Event)]
    tables._classes[("targets", 4)] = (None, tables._kept[0])
    assert copy.deepcopy(tables)._classes == {} and not hasattr(pickle.loads(pickle.dumps(tables)), "_kept")
