"""The neighbourhood softmax with a learned relative bias (nn/relative.py) against
its formulas and their derivatives written out in float64.

Tolerances follow the roundings.  A score of n products is off by at most n + 4
half steps of its terms' absolute sum M (scaled, both biases with them); a weight
a = exp(s - m) / l by the score's, its row's largest score's and the sum's: rel =
(eps / 2) (64 + (n + 4) (M + max M of the row) + degree) of itself, ``64`` for the
exponentials, quotients and shuffles.  T = sum a g is off by rel of sum a |g|, an
edge's ds by 2 rel of a (|g| + sum a |g|); a row's gradient by that, summed with the
absolute values of what it multiplies, and by a half step an edge for the sum itself;
a bucket's sum by its edges' and a half step an edge of it.  A result held in
bfloat16 is off by another eps / 2 = 2^-8 of its value.
"""

import concurrent.futures
import copy
import math
import pickle

import pytest
import torch

import problems
from gm_attention_amd.nn import relative
from gm_attention_amd.nn.relative import RelativeEdgeTables, distance_buckets, relative_softmax
from gm_attention_amd.representations.field_type import SO2FieldType
from test_differential_gpu import ROWS, compare, scattered, sphere, tables_dtype


def bucketed(graph, n_buckets, seed=0):
    """The graph with a bucket an edge, at random, one of every five edges in the last."""
    gen = torch.Generator().manual_seed(1000 + seed)
    graph.buckets = torch.randint(0, n_buckets, graph.source.shape, generator=gen)
    graph.buckets[::5] = n_buckets - 1
    graph.n_buckets = n_buckets
    return graph


def tables_of(graph, dtype, device):
    return RelativeEdgeTables(graph.row_ptr.to(device), graph.source.to(device), graph.transport.to(dtype).to(device),
                              graph.bias.to(dtype).to(device), graph.inside.to(device), graph.buckets.to(device),
                              graph.n_buckets, n_sources=graph.n_sources)


def oracle(graph, q, k, table, g, copies, heads, eps):
    """``{name: (value, tolerance)}`` of alpha, dq, dk and dtable; a row an excluded
    edge would read is replaced by zeros there."""
    n, E = graph.n_targets, graph.source.numel()
    t, j, b = graph.target, graph.source, graph.buckets
    scale = sum(c * (1 if f == 0 else 2) for f, c in copies.items()) ** -0.5
    use = graph.inside.bool()
    out = {name: torch.zeros(shape, dtype=torch.float64) for name, shape in
           (("alpha", (E, heads)), ("dq", q.shape), ("dk", k.shape), ("dtable", table.shape))}
    tol = {name: torch.zeros_like(v) for name, v in out.items()}
    degree = (graph.row_ptr[1:] - graph.row_ptr[:-1]).double()
    in_degree = torch.bincount(j, minlength=k.shape[0]).double()
    members = torch.bincount(b, minlength=table.shape[0]).double()

    def blocks():
        at = 0
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            yield f, w, at
            at += heads * w

    def rows_of(x, index, h):
        got = [x[:, at + h * w: at + (h + 1) * w].index_select(0, index) for _, w, at in blocks()]
        return torch.where(use.unsqueeze(-1), torch.cat(got, 1), 0.0)

    def turn(x, sign, absolute=False):
        got, at = [], 0
        for f, w, _ in blocks():
            v = x[:, at:at + w]
            if f:
                cos, sin = graph.transport[:, f, 0, None], sign * graph.transport[:, f, 1, None]
                re, im = v.reshape(E, -1, 2).unbind(-1)
                if absolute:
                    re, im, cos, sin = re.abs(), im.abs(), cos.abs(), sin.abs()
                    v = torch.stack([cos * re + sin * im, cos * im + sin * re], -1).reshape(E, w)
                else:
                    v = torch.stack([cos * re - sin * im, cos * im + sin * re], -1).reshape(E, w)
            got.append(v.abs() if absolute else v)
            at += w
        return torch.cat(got, 1)

    def put(x, h, v, index):
        mine = 0
        for _, w, at in blocks():
            x[:, at + h * w: at + (h + 1) * w] = torch.zeros(x.shape[0], w, dtype=x.dtype).index_add_(
                0, index, v[:, mine:mine + w])
            mine += w

    def per(index, v, size=n):
        return torch.zeros(size, dtype=torch.float64).index_add_(0, index, v)

    for h in range(heads):
        qe, ke = rows_of(q, t, h), rows_of(k, j, h)
        tk, tka = turn(ke, 1.0), turn(ke, 1.0, absolute=True)
        learned = table[:, h][b]
        s = scale * (qe * tk).sum(-1) + graph.bias + learned
        terms = scale * (qe.abs() * tka).sum(-1) + graph.bias.abs() + learned.abs()
        logit = torch.where(use, s, -math.inf)
        top = torch.full((n,), -math.inf, dtype=torch.float64).scatter_reduce(0, t, logit, "amax")
        w = torch.where(use, torch.exp(logit - top[t]), 0.0)
        w = torch.where(use, w / per(t, w)[t], 0.0)
        most = torch.zeros(n, dtype=torch.float64).scatter_reduce(0, t, torch.where(use, terms, 0.0), "amax")
        rel = eps / 2 * (64 + (4 * qe.shape[1] + 4) * (terms + most[t]) + degree[t])
        out["alpha"][:, h] = w
        tol["alpha"][:, h] = w * (rel + eps)
        ge = torch.where(use, g[:, h], 0.0)
        T, Ta = per(t, w * ge), per(t, w * ge.abs())
        ds = w * (ge - T[t])
        row_rel = torch.zeros(n, dtype=torch.float64).scatter_reduce(0, t, torch.where(use, rel, 0.0), "amax")[t]
        dsa = w * (ge.abs() + Ta[t])
        out["dtable"][:, h] = per(b, ds, table.shape[0])
        tol["dtable"][:, h] = per(b, dsa * 2 * row_rel, table.shape[0]) + \
            eps / 2 * (members + 1) * per(b, dsa, table.shape[0])
        ds, dsa = scale * ds, scale * dsa
        put(out["dq"], h, ds.unsqueeze(-1) * tk, t)
        put(tol["dq"], h, (dsa * (2 * row_rel + eps / 2 * degree[t])).unsqueeze(-1) * tka, t)
        put(out["dk"], h, ds.unsqueeze(-1) * turn(qe, -1.0), j)
        put(tol["dk"], h, (dsa * (2 * row_rel + eps / 2 * in_degree[j])).unsqueeze(-1) *
            turn(qe, -1.0, absolute=True), j)
    return {name: (out[name], tol[name]) for name in out}


def inputs(graph, copies, heads, rows, seed=0):
    D = heads * sum(c * (1 if f == 0 else 2) for f, c in copies.items())
    dtype = tables_dtype(rows)
    q = problems.normal((graph.n_targets, D), seed).to(rows).double()
    k = problems.normal((graph.n_sources, D), seed + 1).to(rows).double()
    table = problems.normal((graph.n_buckets, heads), seed + 2).to(dtype).double()
    g = problems.normal((graph.source.numel(), heads), seed + 3).to(dtype).double()
    return q, k, table, g


def run(tables, q, k, table, g, copies, heads, rows, device):
    leaves = [q.to(rows).to(device).requires_grad_(True), k.to(rows).to(device).requires_grad_(True),
              table.to(tables.dtype).to(device).requires_grad_(True)]
    alpha = relative_softmax(*leaves, tables, SO2FieldType(copies), heads)
    assert alpha.dtype == tables.dtype
    with torch.no_grad():
        assert torch.equal(relative_softmax(*leaves, tables, SO2FieldType(copies), heads), alpha)
    grads = torch.autograd.grad(alpha, leaves, g.to(tables.dtype).to(device), retain_graph=True)
    again = torch.autograd.grad(alpha, leaves, g.to(tables.dtype).to(device))
    # masked rows may hold NaN, their gradients are zeros
    assert all(torch.equal(a, b) for a, b in zip(grads, again)), "two backward passes differ"
    assert [x.dtype for x in grads] == [rows, rows, tables.dtype]
    return dict(zip(("alpha", "dq", "dk", "dtable"), (alpha, *grads)))


def check(graph, copies, heads, rows, device, seed=0):
    print(f"relative {copies} H={heads} B={graph.n_buckets} {rows} N={graph.n_targets} E={graph.source.numel()}",
          flush=True)
    dtype = tables_dtype(rows)
    values = inputs(graph, copies, heads, rows, seed)
    got = run(tables_of(graph, dtype, device), *values, copies, heads, rows, device)
    want = oracle(graph, *values, copies, heads, torch.finfo(dtype).eps)
    for name in want:
        compare(got[name], want[name], name)


#: copies a head and heads: every lane arrangement, odd copies, frequencies with gaps and alone, above two
LAYOUTS = [({0: 4, 1: 4, 2: 4}, 8), ({0: 4, 1: 4, 2: 4}, 4), ({0: 4, 1: 4, 2: 4}, 1), ({0: 4, 1: 4, 2: 4}, 16),
           ({0: 2, 1: 2, 2: 2}, 8), ({0: 2, 1: 2, 2: 2}, 16), ({0: 2, 1: 2, 2: 2}, 1), ({0: 8, 1: 8, 2: 8}, 4),
           ({0: 8, 1: 8, 2: 8}, 16), ({0: 1, 1: 1, 2: 1}, 8), ({0: 1, 1: 1, 2: 1}, 1), ({0: 2, 1: 1, 2: 1}, 6),
           ({0: 4, 1: 2, 2: 2}, 6), ({0: 8, 1: 4, 2: 4}, 4), ({0: 8, 1: 4, 2: 2}, 8), ({0: 4, 1: 4}, 4),
           ({0: 2, 1: 2}, 4), ({0: 1, 1: 1}, 3), ({0: 4, 1: 2, 2: 1}, 8), ({0: 3, 1: 2, 2: 1}, 6),
           ({0: 3, 1: 2, 2: 1}, 5), ({0: 5, 1: 3, 2: 3}, 7), ({0: 12}, 8), ({0: 4}, 16), ({1: 4, 2: 4}, 8),
           ({0: 2, 2: 2}, 4), ({1: 2}, 2), ({2: 4}, 4), ({0: 5}, 7), ({0: 3, 1: 5, 2: 2}, 3), ({0: 2, 3: 2}, 4),
           ({0: 4, 1: 4, 2: 4}, 6), ({0: 16, 1: 16, 2: 16}, 2), ({0: 32, 1: 32, 2: 32}, 1)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", LAYOUTS)
def test_every_layout_and_type(copies, heads, rows, cuda):
    order = max(copies)
    check(bucketed(sphere(10, 20, window="quartic", dtype=tables_dtype(rows), order=order), 7), copies, heads, rows,
          cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 4, 1: 4}, 4), ({0: 12}, 8), ({1: 4}, 2)])
def test_tables_of_more_orders_than_the_heads_read(copies, heads, rows, cuda):
    check(bucketed(sphere(8, 16, dtype=tables_dtype(rows), order=4), 5), copies, heads, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 2, 1: 2, 2: 2}, 2), ({0: 1, 1: 1, 2: 1}, 4),
                                          ({0: 8, 1: 8, 2: 8}, 16), ({0: 3, 1: 5, 2: 2}, 3)])
def test_lengths_of_rows(copies, heads, rows, cuda):
    """No edge, one, and around every number of edges a step, a batch, a wave and a
    workgroup hold; sources twice in a row, rows with nothing inside, more and
    fewer sources than targets."""
    degrees = [0, 1, 1, 2, 3, 0, 4, 5, 7, 8, 9, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100, 127, 128, 129, 130, 200, 255,
               256, 257, 300, 511, 512, 513, 700, 1, 0]
    for n_sources in (11, 400):
        check(bucketed(scattered(degrees, n_sources, tables_dtype(rows)), 9), copies, heads, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 4, 1: 4, 2: 4}, 4), ({0: 8, 1: 8, 2: 8}, 16),
                                          ({0: 1, 1: 1, 2: 1}, 2)])
def test_rows_longer_than_a_workgroup_holds(copies, heads, rows, cuda):
    check(bucketed(scattered([1, 5000, 3, 2100, 17, 9000], 500, torch.float32), 33), copies, heads, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.float64])
@pytest.mark.parametrize("n_buckets", [1, 2, 31, 32, 33, 64, 65, 96, 128, 129, 255, 256])
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 1, 1: 1, 2: 1}, 16), ({0: 3, 1: 1}, 5)])
def test_numbers_of_buckets(copies, heads, n_buckets, rows, cuda):
    check(bucketed(sphere(9, 18, batch=3, dtype=rows), n_buckets), copies, heads, rows, cuda)


@pytest.mark.gpu
def test_many_targets_for_each_workgroup(cuda):
    """More rows than the backward has workgroups: their sums are carried over rows of every length."""
    gen = torch.Generator().manual_seed(5)
    degrees = torch.randint(0, 9, (40_000,), generator=gen).tolist()
    for i in range(0, 40_000, 1000):
        degrees[i] = 200 + i // 100
    check(bucketed(scattered(degrees, 3000, torch.float32), 11), {0: 1, 1: 1, 2: 1}, 4, torch.float32, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads,n_buckets", [({0: 1, 1: 1, 2: 1}, 4, 11), ({0: 4, 1: 4, 2: 4}, 8, 32),
                                                    ({0: 3, 1: 1}, 5, 3), ({0: 2, 1: 2, 2: 2}, 16, 256)])
def test_the_tables_gradient_over_every_edge(copies, heads, n_buckets, rows, cuda):
    """Sums over more rows than the workgroups hold at once, of numbers whose sums are exact.  Queries of zeros and
    equal biases make a row of 2^d edges uniform, 2^-d; under whole g up to 2 its ds are whole in 2^-2d, 2^-12 at most
    here, and sum to at most 4.  A workgroup has at most 160 rows here, one workgroup a CU: its sums stay below 2^12,
    24 bits above 2^-12; those of the workgroups are in double.  So every edge counts once, to the last bit."""
    gen = torch.Generator().manual_seed(n_buckets)
    degrees = (2 ** torch.randint(0, 5, (40_000,), generator=gen)).tolist()
    degrees[::7] = [0] * len(degrees[::7])
    degrees[3::997] = [64] * len(degrees[3::997])
    graph = bucketed(scattered(degrees, 3000, torch.float32, outside=0.0, order=max(copies)), n_buckets)
    graph.inside[:] = 1
    graph.bias[:] = 0.0
    E, D = graph.source.numel(), heads * SO2FieldType(copies).dimension
    dtype = tables_dtype(rows)
    g = torch.randint(-2, 3, (E, heads), generator=gen).double()
    leaves = [torch.zeros(graph.n_targets, D), torch.ones(graph.n_sources, D), torch.zeros(n_buckets, heads)]
    leaves = [x.to(t).to(cuda).requires_grad_(True) for x, t in zip(leaves, (rows, rows, dtype))]
    alpha = relative_softmax(*leaves, tables_of(graph, dtype, cuda), SO2FieldType(copies), heads)
    degree = (graph.row_ptr[1:] - graph.row_ptr[:-1]).double()[graph.target].unsqueeze(1)
    assert torch.equal(alpha.detach().cpu().double(), (1 / degree).expand(E, heads))
    (got,) = torch.autograd.grad(alpha, leaves[2:], g.to(dtype).to(cuda))
    total = torch.zeros(graph.n_targets, heads, dtype=torch.float64).index_add_(0, graph.target, g / degree)
    ds = (g - total[graph.target]) / degree
    want = torch.zeros(n_buckets, heads, dtype=torch.float64).index_add_(0, graph.buckets, ds)
    assert torch.equal(got.cpu(), want.to(dtype)) and float((want != 0).double().mean()) > 0.9


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 1, 1: 1, 2: 1}, {0: 4, 1: 4, 2: 4}])
def test_long_rows_among_many_targets(copies, cuda):
    """Rows that a wave takes alone though its scores fill more than it holds, beside some of a workgroup."""
    degrees = [1] * 17_000
    degrees[5], degrees[700], degrees[16_999], degrees[9000] = 300, 470, 511, 2000
    check(bucketed(scattered(degrees, 3000, torch.float32), 11), copies, 4, torch.float32, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 1}])
def test_masked_rows_may_hold_anything(copies, rows, cuda):
    """Nodes whose every edge is outside hold NaN, infinities and the type's extremes,
    and the bias of those edges too: nothing of them is seen."""
    dtype, heads = tables_dtype(rows), 4
    graph = bucketed(sphere(10, 20, dtype=dtype), 6)
    gone = torch.zeros(graph.n_targets, dtype=torch.bool)
    gone[30:95] = True
    graph.inside = graph.inside * (~(gone[graph.target] | gone[graph.source])).to(torch.uint8)
    assert bool((torch.zeros(graph.n_targets).index_add_(0, graph.target, graph.inside.float()) == 0).any())
    q, k, table, g = inputs(graph, copies, heads, rows)
    odd = torch.tensor([math.nan, math.inf, -math.inf, torch.finfo(rows).min, torch.finfo(rows).max])
    for x in (q, k):
        x[gone] = odd.double()[torch.arange(int(gone.sum()) * x.shape[1]) % 5].reshape(-1, x.shape[1])
    out = graph.inside == 0
    graph.bias[out] = odd.double()[torch.arange(int(out.sum())) % 4]
    g = torch.where(out.unsqueeze(-1), math.nan, g)
    got = run(tables_of(graph, dtype, cuda), q, k, table, g, copies, heads, rows, cuda)
    clean = [torch.where(gone.unsqueeze(-1), 0.0, x) for x in (q, k)]
    graph.bias[out] = 0.0
    want = oracle(graph, *clean, table, torch.where(out.unsqueeze(-1), 0.0, g), copies, heads, torch.finfo(dtype).eps)
    for name in want:
        compare(got[name], want[name], name)
    assert bool((got["dq"][gone.to(cuda)] == 0).all()) and bool((got["dk"][gone.to(cuda)] == 0).all())
    assert bool((got["alpha"][out.to(cuda)] == 0).all())


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 1}])
def test_biases_of_the_lowest_value_inside_the_window(copies, cuda):
    """A row whose every bias is the type's lowest is uniform; beside an ordinary
    one such an edge has weight zero; a row of -inf biases has none inside."""
    lowest = torch.finfo(torch.float32).min
    graph = bucketed(scattered([4, 4, 4], 6, torch.float32, outside=0.0), 3)
    graph.inside[:] = 1
    graph.bias[:] = torch.tensor([lowest] * 4 + [0.0, lowest, 0.0, lowest] + [-math.inf] * 4).double()
    q, k, table, g = inputs(graph, copies, 2, torch.float32)
    got = run(tables_of(graph, torch.float32, cuda), q, k, table, g, copies, 2, torch.float32, cuda)
    alpha = got["alpha"].cpu()
    torch.testing.assert_close(alpha[:4], torch.full((4, 2), 0.25))
    assert bool((alpha[[5, 7]] == 0).all()) and bool((alpha[8:] == 0).all())
    assert all(bool(torch.isfinite(x).all()) for x in got.values())


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 1}])
def test_learned_biases_of_minus_infinity_shut_their_buckets(copies, cuda):
    graph = bucketed(scattered([6, 40, 1, 300], 20, torch.float32, outside=0.0), 4)
    graph.inside[:] = 1
    graph.buckets[graph.target == 2] = 1
    q, k, table, g = inputs(graph, copies, 3, torch.float32)
    table[1] = -math.inf
    got = run(tables_of(graph, torch.float32, cuda), q, k, table, g, copies, 3, torch.float32, cuda)
    graph.inside = graph.inside * (graph.buckets != 1).to(torch.uint8)
    table[1] = 0.0
    want = oracle(graph, q, k, table, g, copies, 3, torch.finfo(torch.float32).eps)
    for name in want:
        compare(got[name], want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 4, 1: 4, 2: 4}, 16), ({0: 1, 1: 1, 2: 1}, 4),
                                          ({0: 3, 1: 2, 2: 1}, 5), ({0: 2, 3: 2}, 4)])
def test_rows_of_no_number_leave_the_edges_that_are_shut(copies, heads, rows, cuda):
    """A key that is no number makes the weights of the rows that read it no numbers, of its head alone and not those of
    the edges outside the window or of a learned -inf: these stay zero and add nothing to any gradient."""
    shut_edges(copies, heads, rows, cuda)


@pytest.mark.parametrize("rows", ROWS)
def test_rows_of_no_number_on_the_cpu(rows):
    shut_edges({0: 3, 1: 2, 2: 1}, 2, rows, "cpu")


def shut_edges(copies, heads, rows, device):
    dtype = tables_dtype(rows)
    graph = bucketed(scattered([1, 2, 9, 40, 6, 300, 1, 700, 3, 2100, 5200, 64], 60, dtype, outside=0.4,
                               order=max(copies)), 4)
    q, k, table, g = inputs(graph, copies, heads, rows)
    lost = graph.source == 7
    shut = (graph.buckets == 0) & ~lost
    use = graph.inside.bool() & ~shut
    bad = torch.zeros(graph.n_targets, dtype=torch.bool)
    bad[graph.target[use & lost]] = True
    assert 3 <= int(bad.sum()) < graph.n_targets - 3
    nan = use & bad[graph.target]
    graph.buckets = torch.where(nan, 1, torch.where(shut, 0, 2 + graph.source % 2))
    table[0] = -math.inf
    tables, results = tables_of(graph, dtype, device), []
    for value in (0.0, math.nan):
        k[7, copies[0]] = value  # the second head's first number
        leaves = [x.to(to).to(device, copy=True).requires_grad_(True)
                  for x, to in ((q, rows), (k, rows), (table, dtype))]
        alpha = relative_softmax(*leaves, tables, SO2FieldType(copies), heads)
        grads = torch.autograd.grad(alpha, leaves, g.to(dtype).to(device))
        results.append([x.detach().cpu() for x in (alpha, *grads)])
    head, at = torch.zeros(q.shape[1], dtype=torch.bool), 0
    for f, c in copies.items():
        w = c * (1 if f == 0 else 2)
        head[at + w:at + 2 * w] = True
        at += heads * w
    sources = torch.zeros(graph.n_sources, dtype=torch.bool)
    sources[graph.source[nan]] = True
    second = torch.arange(heads) == 1
    expected = (nan.unsqueeze(1) & second, bad.unsqueeze(1) & head, sources.unsqueeze(1) & head,
                (torch.arange(4) == 1).unsqueeze(1) & second)
    assert bool((results[1][0][~use] == 0).all())
    for name, clean, got, where in zip(("alpha", "dq", "dk", "dtable"), *results, expected):
        assert torch.equal(got.isnan(), where), name
        assert torch.equal(got[~where], clean[~where]), name


@pytest.mark.gpu
@pytest.mark.parametrize("common", [0.0, 10.0, 1000.0])
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 3, 1: 1}, 3)])
def test_gradients_with_a_common_part(copies, heads, common, cuda):
    """What a row's g share cancels: the gradients are those without it, but for T's rounding."""
    graph = bucketed(sphere(10, 20), 5)
    q, k, table, g = inputs(graph, copies, heads, torch.float32)
    g = (g + common).float().double()
    got = run(tables_of(graph, torch.float32, cuda), q, k, table, g, copies, heads, torch.float32, cuda)
    want = oracle(graph, q, k, table, g, copies, heads, torch.finfo(torch.float32).eps)
    for name in want:
        compare(got[name], want[name], name)


@pytest.mark.gpu
def test_a_single_bucket_leaves_the_softmax_as_it_is(cuda):
    """One learned number for every edge cancels, and its gradient is zero but for rounding."""
    from gm_attention_amd.nn.fused_attention import Softmax

    graph, copies, heads = bucketed(sphere(10, 20), 1), {0: 4, 1: 4, 2: 4}, 8
    q, k, table, g = inputs(graph, copies, heads, torch.float32)
    got = run(tables_of(graph, torch.float32, cuda), q, k, table, g, copies, heads, torch.float32, cuda)
    plan = relative.heads_of(SO2FieldType(copies), heads).plan
    desc = torch.tensor([list(r) for r in plan.rows], dtype=torch.int64, device=cuda)
    single = Softmax.apply(q.float().to(cuda), k.float().to(cuda), graph.transport.float().to(cuda).contiguous(),
                           graph.bias.float().to(cuda), graph.inside.to(cuda), desc, graph.row_ptr.to(cuda),
                           graph.source.to(cuda), heads, 20 ** -0.5, 64)
    want = oracle(graph, q, k, table, g, copies, heads, torch.finfo(torch.float32).eps)
    compare(single, want["alpha"], "single")
    compare(got["alpha"], want["alpha"], "alpha")
    compare(got["dtable"], want["dtable"], "dtable")


@pytest.mark.gpu
def test_sources_at_the_far_end_of_a_large_table(cuda):
    """Key rows whose offsets pass 2^31 numbers, the last source a record can name."""
    copies, heads, n = {0: 4, 1: 4, 2: 4}, 8, 2**24  # 160 numbers a row: 2.7e9
    graph = bucketed(scattered([3, 40, 70, 0, 5], 64, torch.float32), 256)
    graph.source[0] = 63
    near = graph.source.clone()
    q, k, table, g = inputs(graph, copies, heads, torch.bfloat16)
    want = oracle(graph, q, k, table, g, copies, heads, torch.finfo(torch.float32).eps)
    graph.source, graph.n_sources = near + (n - 64), n
    tables = tables_of(graph, torch.float32, cuda)
    far = torch.zeros(n, 160, dtype=torch.bfloat16, device=cuda)
    far[n - 64:] = k.to(torch.bfloat16).to(cuda)
    leaves = [q.bfloat16().to(cuda).requires_grad_(True), far.requires_grad_(True),
              table.float().to(cuda).requires_grad_(True)]
    alpha = relative_softmax(*leaves, tables, SO2FieldType(copies), heads)
    dq, dk, dtable = torch.autograd.grad(alpha, leaves, g.float().to(cuda))
    compare(alpha, want["alpha"], "alpha")
    compare(dq, want["dq"], "dq")
    compare(dk[n - 64:], want["dk"], "dk")
    compare(dtable, want["dtable"], "dtable")
    assert not bool(dk[: n - 64].any())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_rows_at_odd_addresses_and_strides(rows, cuda):
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    graph = bucketed(sphere(10, 20), 5)
    q, k, table, g = inputs(graph, copies, heads, rows)
    want = oracle(graph, q, k, table, g, copies, heads, torch.finfo(torch.float32).eps)
    tables = tables_of(graph, torch.float32, cuda)

    def shifted(t):
        return torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape).copy_(t)

    def strided(t):
        return torch.empty(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device=cuda)[:, 3:-2].copy_(t)

    for view in (shifted, strided):
        leaves = [view(q.to(rows)).requires_grad_(True), view(k.to(rows)).requires_grad_(True),
                  view(table.float()).requires_grad_(True)]
        alpha = relative_softmax(*leaves, tables, SO2FieldType(copies), heads)
        grads = torch.autograd.grad(alpha, leaves, view(g.float()))  # a gradient with gaps between its rows
        for name, x in zip(("alpha", "dq", "dk", "dtable"), (alpha, *grads)):
            compare(x, want[name], name)


@pytest.mark.gpu
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 3, 1: 2}, 2)])
def test_gradients_against_differences(copies, heads, cuda):
    """In float64, central differences of a weighted sum of the weights along random directions: a step of h = 1e-5 is
    off by h^2 / 6 of the third derivative, of order one, and by eps / h = 2e-11 of the sum's terms."""
    graph = bucketed(sphere(8, 16, dtype=torch.float64), 5)
    values = inputs(graph, copies, heads, torch.float64)
    tables = tables_of(graph, torch.float64, cuda)
    q, k, table, g = (v.to(cuda) for v in values)
    got = run(tables, *values, copies, heads, torch.float64, cuda)

    def loss(*leaves):
        return float((relative_softmax(*leaves, tables, SO2FieldType(copies), heads) * g).sum())

    for i, name in enumerate(("dq", "dk", "dtable")):
        leaves = [q, k, table]
        step = torch.randn(leaves[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)).to(cuda)
        h = 1e-5
        up, down = (loss(*(x + s * h * step if i == j else x for j, x in enumerate(leaves))) for s in (1, -1))
        want = float((got[name] * step).sum())
        assert abs((up - down) / (2 * h) - want) <= 1e-6 * float((got[name] * step).abs().sum()), name


@pytest.mark.gpu
def test_turning_the_frames_leaves_the_weights(cuda):
    """Frames turned by any angle a node: rows and transport follow, the weights stay."""
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    graph = bucketed(sphere(10, 20, dtype=torch.float64), 5)
    q, k, table, _ = inputs(graph, copies, heads, torch.float64)
    psi = problems.normal((graph.n_targets,), 9)
    field = SO2FieldType({f: heads * c for f, c in copies.items()})

    def turned(x):
        out = x.clone()
        for f, c in field.items():
            if f:
                s = field.slices()[f]
                z = torch.view_as_complex(x[:, s].reshape(-1, c, 2).contiguous())
                z = z * torch.polar(torch.ones_like(psi), -f * psi).unsqueeze(-1)
                out[:, s] = torch.view_as_real(z).reshape(-1, 2 * c)
        return out

    args = (table.to(cuda),)
    want = relative_softmax(q.to(cuda), k.to(cuda), *args, tables_of(graph, torch.float64, cuda),
                            SO2FieldType(copies), heads)
    shift = psi[graph.source] - psi[graph.target]
    tau = torch.view_as_complex(graph.transport.contiguous())
    tau = tau * torch.polar(torch.ones_like(shift), shift).unsqueeze(-1) ** torch.arange(tau.shape[1])
    graph.transport = torch.view_as_real(tau)
    got = relative_softmax(turned(q).to(cuda), turned(k).to(cuda), *args, tables_of(graph, torch.float64, cuda),
                           SO2FieldType(copies), heads)
    torch.testing.assert_close(got, want, rtol=1e-11, atol=1e-13)


# ------------------------------------------------------------- streams, captures, threads


def stepper(graph, copies, heads, device):
    q, k, table, g = (v.float().to(device) for v in inputs(graph, copies, heads, torch.float32))

    def step(tables):
        leaves = [v.detach().requires_grad_(True) for v in (q, k, table)]
        alpha = relative_softmax(*leaves, tables, SO2FieldType(copies), heads)
        return [alpha.detach(), *torch.autograd.grad(alpha, leaves, g)]

    return step


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 1}])
def test_replays_of_two_captured_steps_equal_the_eager_ones(copies, cuda):
    """Two graphs over the same tables, replayed in turn with eager steps between."""
    graphs = [bucketed(sphere(12, 24, batch=2), 9), bucketed(sphere(12, 24, batch=2), 9, seed=1)]
    steps = [stepper(g, copies, 8, cuda) for g in graphs]
    kept = [tables_of(g, torch.float32, cuda) for g in graphs]
    want = [[t.clone() for t in s(k)] for s, k in zip(steps, kept)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for s, k in zip(steps, kept):
            s(k)
    torch.cuda.current_stream().wait_stream(side)
    captured, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for c, s, k in zip(captured, steps, kept):
        with torch.cuda.graph(c):
            got.append(s(k))
    for replay in range(3):
        for out in got:
            for t in out:
                t.zero_()
        for c in captured:
            c.replay()
        torch.cuda.synchronize()
        for out, w, s, k in zip(got, want, steps, kept):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), replay
            assert all(torch.equal(a, b) for a, b in zip(s(k), w)), replay
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_tables_are_built_before_a_capture(cuda):
    graph = bucketed(sphere(8, 16), 4)
    q, k, table, g = (v.float().to(cuda) for v in inputs(graph, {0: 4, 1: 4}, 2, torch.float32))
    tables = tables_of(graph, torch.float32, cuda)
    given = [graph.row_ptr.to(cuda), graph.source.to(cuda), graph.transport.float().to(cuda),
             graph.bias.float().to(cuda), graph.inside.to(cuda), graph.buckets.to(cuda), 4]
    torch.cuda.synchronize()
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        held = q * 1.0
        with pytest.raises(RuntimeError, match="before the capture"):
            RelativeEdgeTables(*given)
        with pytest.raises(RuntimeError, match="before the capture"):
            relative_softmax(q.requires_grad_(True), k, table, tables, SO2FieldType({0: 4, 1: 4}), 2)
    captured.replay()
    torch.cuda.synchronize()
    assert torch.equal(held, q)


@pytest.mark.gpu
def test_inference_needs_no_source_side(cuda):
    copies, heads = {0: 4, 1: 4, 2: 4}, 8
    graph = bucketed(sphere(8, 16), 4)
    q, k, table, g = (v.float().to(cuda) for v in inputs(graph, copies, heads, torch.float32))
    tables, head = tables_of(graph, torch.float32, cuda), SO2FieldType(copies)
    table = torch.nn.Parameter(table)
    with torch.no_grad():
        want = relative_softmax(q, k, table, tables, head, heads)
    assert not tables._pairs
    alpha = relative_softmax(q, k, table, tables, head, heads)
    assert torch.equal(alpha, want) and set(tables._pairs) == {"sources", "targets"}


@pytest.mark.gpu
def test_two_threads_at_once(cuda):
    """Two threads' first steps over the same new tables, each on its own stream."""
    graph = bucketed(sphere(12, 24, batch=2), 8)
    step = stepper(graph, {0: 4, 1: 4, 2: 4}, 8, cuda)
    want = step(tables_of(graph, torch.float32, cuda))
    tables = tables_of(graph, torch.float32, cuda)
    torch.cuda.synchronize()

    def work(_):
        stream = torch.cuda.Stream()
        with torch.cuda.stream(stream):
            out = [step(tables) for _ in range(5)]
        stream.synchronize()
        return out

    with concurrent.futures.ThreadPoolExecutor(2) as pool:
        runs = list(pool.map(work, range(2)))
    assert all(torch.equal(a, b) for got in runs for out in got for a, b in zip(out, want))


@pytest.mark.gpu
def test_on_another_stream(cuda):
    """Tables built on one stream behind other work, read on another at once."""
    graph = bucketed(sphere(24, 48), 8)
    step = stepper(graph, {0: 4, 1: 4, 2: 4}, 8, cuda)
    want = step(tables_of(graph, torch.float32, cuda))
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=cuda)
    for _ in range(20):
        busy = busy @ busy * 1e-3
    tables = tables_of(graph, torch.float32, cuda)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = step(tables)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_no_targets_and_no_edges(cuda):
    nothing(cuda)


def test_no_targets_and_no_edges_on_the_cpu():
    nothing("cpu")


def nothing(cuda):
    for copies in ({0: 4, 1: 4}, {0: 3, 1: 1}):
        head = SO2FieldType(copies)
        for n, m in ((0, 0), (0, 5), (4, 0), (4, 5)):
            tables = RelativeEdgeTables(
                torch.zeros(n + 1, dtype=torch.int64, device=cuda), torch.zeros(0, dtype=torch.int64, device=cuda),
                torch.zeros(0, 2, 2, device=cuda), torch.zeros(0, device=cuda),
                torch.zeros(0, dtype=torch.uint8, device=cuda), torch.zeros(0, dtype=torch.int32, device=cuda), 3,
                n_sources=m)
            width = 2 * head.dimension
            leaves = [torch.ones(*s, device=cuda, requires_grad=True) for s in ((n, width), (m, width), (3, 2))]
            alpha = relative_softmax(*leaves, tables, head, 2)
            assert alpha.shape == (0, 2)
            for x, grad in zip(leaves, torch.autograd.grad(alpha, leaves, alpha.detach())):
                assert grad.shape == x.shape and not bool(grad.any())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.float64])
def test_copied_tables_give_the_same_results(rows, cuda, tmp_path):
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    graph = bucketed(scattered([3, 0, 70, 9, 1, 200], 40, rows), 200)  # buckets on both sides of a word's sign
    tables = tables_of(graph, rows, cuda)
    values = inputs(graph, copies, heads, rows)
    want = run(tables, *values, copies, heads, rows, cuda)
    torch.save(tables, tmp_path / "tables")
    for other in (copy.deepcopy(tables), pickle.loads(pickle.dumps(tables)),
                  torch.load(tmp_path / "tables", weights_only=False)):
        got = run(other, *values, copies, heads, rows, cuda)
        assert all(torch.equal(got[n], want[n]) for n in want)
    read = torch.load(tmp_path / "tables", weights_only=False, map_location="cpu")
    assert read.device.type == "cpu" and torch.equal(read.buckets.long(), graph.buckets)
    got = run(read, *values, copies, heads, rows, "cpu")
    want = oracle(graph, *values, copies, heads, torch.finfo(rows).eps)
    for name in want:  # the biases were kept in units of log 2: two roundings, of the many the bound counts for them
        compare(got[name], want[name], name)


# ---------------------------------------------------------------- without a GPU


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 2, 1: 2, 2: 2}, 3), ({1: 1, 2: 3}, 2), ({0: 5}, 1)])
def test_cpu_rows_take_the_formulas_in_torch(copies, heads, rows):
    check(bucketed(scattered([0, 1, 5, 9, 40, 3, 70, 0, 8], 13, tables_dtype(rows)), 4), copies, heads, rows, "cpu")


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 1}])
def test_masked_rows_may_hold_anything_on_the_cpu(copies, rows):
    test_masked_rows_may_hold_anything(copies, rows, "cpu")


def test_learned_biases_of_minus_infinity_on_the_cpu():
    test_learned_biases_of_minus_infinity_shut_their_buckets({0: 4, 1: 4, 2: 4}, "cpu")


def test_edges_of_weight_zero_on_the_cpu():
    """Inside the window too they add nothing to a gradient, whatever their g, the learned number or the row
    that made their score -inf hold."""
    tables = RelativeEdgeTables(torch.tensor([0, 5]), torch.arange(5), torch.ones(5, 1, 2), torch.zeros(5),
                                torch.tensor([1, 1, 1, 1, 0], dtype=torch.uint8), torch.arange(5), 5, n_sources=5)
    q = torch.ones(1, 1, requires_grad=True)
    k = torch.tensor([[0.5], [-0.25], [-math.inf], [-400.0], [math.nan]], requires_grad=True)
    table = torch.tensor([[0.0], [0.25], [0.0], [0.0], [math.nan]], requires_grad=True)
    alpha = relative_softmax(q, k, table, tables, SO2FieldType({0: 1}), 1)
    w = 1 / (1 + math.exp(-0.5))  # of the scores 0.5 and 0
    torch.testing.assert_close(alpha, torch.tensor([[w], [1 - w], [0.0], [0.0], [0.0]]))
    dq, dk, dtable = torch.autograd.grad(alpha, (q, k, table),
                                         torch.tensor([[1.0], [3.0], [math.inf], [math.nan], [math.nan]]))
    ds = w * (1 - w) * (1 - 3)
    zeros = [[0.0]] * 3
    torch.testing.assert_close(dq, torch.tensor([[ds * 0.75]]))
    torch.testing.assert_close(dk, torch.tensor([[ds], [-ds], *zeros]))
    torch.testing.assert_close(dtable, torch.tensor([[ds], [-ds], *zeros]))


def test_derivatives_of_every_kind_on_the_cpu():
    """Backward, forward and second derivatives, and functions of functions."""
    copies, heads = {0: 2, 1: 1}, 2
    graph = bucketed(scattered([1, 3, 4, 6], 5, torch.float64, outside=0.3), 3)
    *leaves, _ = inputs(graph, copies, heads, torch.float64)
    tables = tables_of(graph, torch.float64, "cpu")

    def weights(q, k, extra):
        return relative_softmax(q, k, extra, tables, SO2FieldType(copies), heads)

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
    graph = bucketed(scattered([3, 0, 70, 9, 1], 40, torch.float64), 256)
    values = inputs(graph, {0: 2, 1: 2}, 2, torch.float64)
    tables = tables_of(graph, torch.float64, "cpu")
    want = run(tables, *values, {0: 2, 1: 2}, 2, torch.float64, "cpu")
    for other in (copy.deepcopy(tables), pickle.loads(pickle.dumps(tables))):
        got = run(other, *values, {0: 2, 1: 2}, 2, torch.float64, "cpu")
        assert all(torch.equal(got[n], want[n]) for n in want)


def test_tables_made_in_inference_mode_train():
    copies, heads = {0: 2, 1: 2}, 2
    graph = bucketed(scattered([3, 0, 70, 9, 1], 40, torch.float64), 6)
    values = inputs(graph, copies, heads, torch.float64)
    want = run(tables_of(graph, torch.float64, "cpu"), *values, copies, heads, torch.float64, "cpu")
    with torch.inference_mode():
        for name in ("row_ptr", "source", "transport", "bias", "inside", "buckets"):
            setattr(graph, name, getattr(graph, name).clone())
        tables = tables_of(graph, torch.float64, "cpu")
    got = run(tables, *values, copies, heads, torch.float64, "cpu")
    assert all(torch.equal(got[n], want[n]) for n in want)


def test_rings_of_distance():
    """Equal distances share a ring whatever their last bit, the borders' too; every distance has one."""
    step = math.pi / 31
    distances = torch.tensor([0.0, 1e-9, 0.5, 1.0, 1.5, 2.0, 3.0, 7.0], dtype=torch.float64) * step
    want = [0, 0, 1, 2, 3, 4, 5, 5]
    for dtype in (torch.float64, torch.float32):
        for off in (0.0, 1e-7, -1e-7):
            got = distance_buckets((distances * (1 + off)).to(dtype), 3 * step, 6)
            assert got.tolist() == want, (dtype, off)


def test_refusals():
    row_ptr, source = torch.tensor([0, 2, 3]), torch.tensor([0, 1, 1])
    phases, bias, inside = torch.zeros(3, 2, 2), torch.zeros(3), torch.ones(3, dtype=torch.uint8)
    buckets = torch.tensor([0, 2, 1], dtype=torch.int32)

    def tables(n_buckets=3, n_sources=None, **kw):
        given = dict(row_ptr=row_ptr, source=source, transport=phases, bias=bias, inside=inside, buckets=buckets)
        given.update(kw)
        return RelativeEdgeTables(*given.values(), n_buckets, n_sources=n_sources)

    for kw, message in ((dict(n_buckets=0), "n_buckets must lie in 1..256"),
                        (dict(n_buckets=257), "n_buckets must lie in 1..256"),
                        (dict(n_buckets=2), r"every bucket must lie in 0 \.\. 1"),
                        (dict(buckets=buckets - 1), "every bucket"), (dict(buckets=buckets[:2]), "buckets must be"),
                        (dict(buckets=buckets.float()), "buckets must be"),
                        (dict(n_sources=2**24 + 1), "at most 16777216 sources"),
                        (dict(source=torch.tensor([0, 2, 1])), "every source"),
                        (dict(row_ptr=torch.tensor([0, 2, 2])), "row_ptr must rise")):
        with pytest.raises(ValueError, match=message):
            tables(**kw)
    t, head = tables(), SO2FieldType({0: 4, 1: 2})
    q, table = torch.zeros(2, 16), torch.zeros(3, 2)
    assert relative_softmax(q, q, table, t, head, 2).shape == (3, 2)
    for call, message in (((q.double(), q.double(), table), "share a dtype"), ((q, q.double(), table), "share a dtype"),
                          ((q.half(), q.half(), table), "share a dtype"), ((q[:1], q, table), "q and k must be"),
                          ((q, q[:, :8], table), "q and k must be"), ((q, q, table[:2]), r"table must be \(3, 2\)"),
                          ((q, q, table[:, :1]), r"table must be"), ((q, q, table.long()), r"table must be")):
        with pytest.raises(ValueError, match=message):
            relative_softmax(*call, t, head, 2)
    with pytest.raises(ValueError, match="heads must lie in 1..16"):
        relative_softmax(q, q, table, t, head, 17)
    with pytest.raises(ValueError, match="at most 8 frequencies and 1024"):
        relative_softmax(q, q, table, t, SO2FieldType({0: 1030}), 1)
    with pytest.raises(ValueError, match="orders below 2, the heads need 2"):
        relative_softmax(q, q, table, t, SO2FieldType({0: 4, 2: 2}), 2)
    with pytest.raises(TypeError, match="head_type must be"):
        relative_softmax(q, q, table, t, {0: 8}, 2)
    from gm_attention_amd.nn.differential import EdgeTables

    with pytest.raises(TypeError, match="tables must be RelativeEdgeTables"):
        relative_softmax(q, q, table, EdgeTables(row_ptr, source, phases, bias, inside), head, 2)


@pytest.mark.parametrize("copies,heads,orders,padded", [
    ({0: 4, 1: 4, 2: 4}, 8, 3, None), ({0: 3, 1: 2, 2: 1}, 6, 3, {0: 4, 1: 2, 2: 1}), ({0: 12}, 8, 1, {0: 16}),
    ({0: 5, 1: 3, 2: 3}, 7, 3, {0: 8, 1: 4, 2: 4}), ({0: 4, 1: 4}, 4, 3, {0: 8, 1: 4, 2: 2}),
    ({2: 4}, 4, 3, {1: 4, 2: 4}), ({0: 2, 3: 2}, 4, 4, None), ({0: 4, 1: 4}, 4, 4, None), ({0: 1024}, 1, 1, None)])
def test_layouts_filled_up_to_whole_units(copies, heads, orders, padded):
    """The layout that the lane kernels take in a layout's place, or the simple kernels with the layout itself."""
    phases = torch.zeros(1, orders, 2)
    tables = RelativeEdgeTables(torch.tensor([0, 1]), torch.tensor([0]), phases, torch.zeros(1),
                                torch.ones(1, dtype=torch.uint8), torch.zeros(1, dtype=torch.uint8), 1)
    given = relative.heads_of(SO2FieldType(copies), heads)
    served = given.served(tables)
    if padded is None:
        assert served is given
    else:
        assert served is relative.heads_of(SO2FieldType(padded), heads) and served.slots(tables) > 0
        assert given.slots(tables) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_rows_are_repacked_as_they_are(rows, cuda):
    from gm_attention_amd import _native

    heads = 5
    small, large = (relative.heads_of(SO2FieldType(c), heads) for c in ({0: 3, 2: 1}, {0: 4, 1: 2, 2: 2}))
    x = problems.normal((7001, small.plan.width), 1).to(rows).to(cuda)
    big = _native.relative_repack(x, small, large)
    want = torch.zeros(7001, 60, dtype=rows, device=cuda)
    for h in range(heads):
        want[:, 4 * h:4 * h + 3] = x[:, 3 * h:3 * h + 3]
        want[:, 40 + 4 * h:42 + 4 * h] = x[:, 15 + 2 * h:17 + 2 * h]
    assert torch.equal(big, want)
    assert torch.equal(_native.relative_repack(big, large, small), x)
    with pytest.raises(RuntimeError, match="rows must be contiguous"):
        _native.relative_repack(x, large, small)


def test_the_library_refuses_bad_arguments():
    """Through the C interface, before anything is launched (no GPU touched)."""
    import ctypes

    from gm_attention_amd import _native

    lib = _native.library()

    def forward(rows=((0, 4, 0, 0, 1), (1, 2, 8, 0, 2)), n=0, m=0, D=16, orders=2, H=2, F=None, buckets=3):
        flat = [x for row in rows for x in row]
        desc = (ctypes.c_int64 * len(flat))(*flat)
        return lib.gm_relative_forward_f32(None, None, None, None, ctypes.cast(desc, ctypes.c_void_p), None, None,
                                           None, n, m, 0, D, orders, len(rows) if F is None else F, H, buckets, 1.0,
                                           None, None)

    assert forward() == 0
    for kw, message in ((dict(n=-1), b"non-negative"), (dict(n=1), b"device pointers"),
                        (dict(H=17), b"at most 16 heads"), (dict(D=1025), b"D must be in"),
                        (dict(D=20), b"fill the flat width"), (dict(orders=1), b"exceeds"),
                        (dict(F=9), b"1 to 8"), (dict(n=2**31), b"32 bits"), (dict(m=2**24 + 1), b"24 bits"),
                        (dict(buckets=0), b"1 to 256 buckets"), (dict(buckets=257), b"1 to 256 buckets"),
                        (dict(rows=((1, 2, 0, 0, 2), (0, 4, 8, 0, 1))), b"must rise"),
                        (dict(rows=((0, 4, 4, 0, 1), (1, 2, 8, 0, 2))), b"follow each other")):
        assert forward(**kw) == 1
        assert message in lib.gm_last_error(), kw
