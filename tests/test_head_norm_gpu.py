"""The norm and rotation of rows of heads (nn/head_norm.py) against its formulas and
their derivatives written out in float64.

Tolerances follow the roundings, in half steps (eps / 2).  A lane adds up to 24 squares in
two sums (12 additions and the last: 13), the head in double: 1 / sqrt is off by 6.5 and
its own rounding, 7; xhat by 8, gain xhat by 9; the angle's fraction of a turn by 2^-26 of
a turn in float (1.6 half steps of a radian), its sine and cosine by two steps (4), the
turned pair by three: 18 half steps of what the pair's terms sum to.  An angle in double is
off by 2^-52 (axes + 3) of the sum of its terms' absolute values.  Backward: d as a pair
alone, 8.6, t = gain d by one more, mean(t xhat) by 9.6 + 13 (its sum) + 7 + 1 = 31 of mean
|t xhat|, dx by 8 + 31 + 2 (product, difference) + 8 (1 / sqrt and its product) = 49, 50 of
its terms' absolute sum; a gain's gradient by 8.6 + 8 + 1, 20 of each term, and one an
addition, of which there are one a node and head.  A result held in bfloat16 is off by
another eps / 2 = 2^-8 of its value.
"""

import copy
import math
import pickle

import pytest
import torch

import problems
from gm_attention_amd.nn import head_norm
from gm_attention_amd.nn.head_norm import SO2QueryKeyNorm, query_key_norm, rotary_frequencies
from gm_attention_amd.representations.field_type import SO2FeatureField, SO2FieldType
from test_differential_gpu import ROWS, compare, tables_dtype


def parts_of(copies, heads):
    """A head's parts in the flat row: ``(columns, copies, slot)`` of every pair, or odd scalar."""
    out, at = [], 0
    for h in range(heads):
        mine, slot, copy_at, base = [], 0, 0, 0
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            first = base + h * w
            for u in range(0, c, 2 if f == 0 else 1):
                if f:
                    mine.append(((first + 2 * u, first + 2 * u + 1), (copy_at + u, copy_at + u), slot))
                    slot += 1
                elif u + 1 < c:
                    mine.append(((first + u, first + u + 1), (copy_at + u, copy_at + u + 1), slot))
                    slot += 1
                else:
                    mine.append(((first + u,), (copy_at + u,), None))
            copy_at += c
            base += heads * w
        out.append(mine)
    return out


def oracle(x, gain, dy, copies, heads, eps_norm, positions, frequencies, eps):
    """``{name: (value, tolerance)}`` of y, dx and dgain in float64."""
    n, numbers, copies_n = x.shape[0], sum(c * (1 if f == 0 else 2) for f, c in copies.items()), sum(copies.values())
    half = eps / 2
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    ty, tx = torch.zeros_like(x), torch.zeros_like(x)
    dgain, tg = torch.zeros(copies_n, dtype=torch.float64), torch.zeros(copies_n, dtype=torch.float64)
    g = torch.ones(copies_n, dtype=torch.float64) if gain is None else gain
    if positions is not None:
        theta = positions @ frequencies
        wrong = 2.0 ** -52 * (positions.shape[1] + 3) * (positions.abs() @ frequencies.abs())
    for mine in parts_of(copies, heads):
        columns = [c for cols, _, _ in mine for c in cols]
        inv = torch.ones(n, dtype=torch.float64) if eps_norm is None else \
            (x[:, columns].square().mean(1) + eps_norm) ** -0.5
        mean, size, back = torch.zeros(n, dtype=torch.float64), torch.zeros(n, dtype=torch.float64), []
        for cols, us, slot in mine:
            hat = [inv * x[:, c] for c in cols]
            z = [g[u] * v for u, v in zip(us, hat)]
            d = [dy[:, c] for c in cols]
            off = torch.zeros(n, dtype=torch.float64)
            if slot is not None and positions is not None:
                cos, sin = torch.cos(theta[:, slot]), torch.sin(theta[:, slot])
                z, za = [cos * z[0] - sin * z[1], cos * z[1] + sin * z[0]], z[0].abs() + z[1].abs()
                d, da = [cos * d[0] + sin * d[1], cos * d[1] - sin * d[0]], d[0].abs() + d[1].abs()
                off = wrong[:, slot]
            else:
                za, da = sum(v.abs() for v in z), sum(v.abs() for v in d)
            for i, c in enumerate(cols):
                y[:, c] = z[i]
                ty[:, c] = (18 * half + off) * za
                t = g[us[i]] * d[i]
                dgain[us[i]] += (d[i] * hat[i]).sum()
                tg[us[i]] += ((20 * half + off) * da * hat[i].abs()).sum() + \
                    half * 2 * n * heads * (da * hat[i].abs()).sum()
                mean += t * hat[i]
                size += (1 + off / (31 * half)) * g[us[i]].abs() * da * hat[i].abs()
                back.append((c, t, hat[i], g[us[i]].abs() * da * (1 + off / (50 * half))))
        for c, t, hat, ta in back:
            if eps_norm is None:
                dx[:, c], tx[:, c] = t, 50 * half * ta
            else:
                dx[:, c] = inv * (t - hat * mean / numbers)
                tx[:, c] = 50 * half * inv * (ta + hat.abs() * size / numbers)
    return {"y": (y, ty), "dx": (dx, tx), "dgain": (dgain, tg)}


def inputs(copies, heads, n, axes, rows, seed=0, gains=True):
    D = heads * sum(c * (1 if f == 0 else 2) for f, c in copies.items())
    slots = copies.get(0, 0) // 2 + sum(c for f, c in copies.items() if f)
    dtype = tables_dtype(rows)
    made = dict(q=problems.normal((n, D), seed).to(rows), k=(3 * problems.normal((n, D), seed + 1) + 1).to(rows),
                up=[problems.normal((n, D), seed + 2 + i).to(rows) for i in range(2)], positions=None, frequencies=None,
                q_gain=None, k_gain=None)
    if gains:
        for i, name in enumerate(("q_gain", "k_gain")):
            made[name] = (1 + 0.3 * problems.normal((sum(copies.values()),), seed + 4 + i)).to(dtype)
    if axes:
        scale = torch.tensor([1.0, 3.0, 1e6, 2e5][:axes], dtype=torch.float64)
        made["positions"] = problems.normal((n, axes), seed + 6).double() * scale
        made["frequencies"] = problems.normal((axes, slots), seed + 7).double() * 2.0
    return made


def run(made, copies, heads, eps, device, need=("q", "k", "q_gain", "k_gain")):
    leaves = {}
    for name in ("q", "k", "q_gain", "k_gain"):
        if made[name] is not None:
            leaves[name] = made[name].to(device).requires_grad_(name in need)
    place = {n: None if made[n] is None else made[n].to(device) for n in ("positions", "frequencies")}
    args = (leaves["q"], leaves["k"], SO2FieldType(copies), heads, leaves.get("q_gain"), leaves.get("k_gain"))
    outs = query_key_norm(*args, eps=eps, **place)
    with torch.no_grad():
        for a, b in zip(query_key_norm(*args, eps=eps, **place), outs):
            torch.testing.assert_close(a, b, rtol=0, atol=0, equal_nan=True)
    names = [n for n in leaves if n in need]
    grads = torch.autograd.grad(outs, [leaves[n] for n in names], [u.to(device) for u in made["up"]])
    return dict(zip(("yq", "yk", *("d" + n for n in names)), (*outs, *grads)))


def wanted(made, copies, heads, eps_norm, eps):
    out = {}
    for i, s in enumerate("qk"):
        gain = made[s + "_gain"]
        got = oracle(made[s].double(), None if gain is None else gain.double(), made["up"][i].double(), copies, heads,
                     eps_norm, made["positions"], made["frequencies"], eps)
        out["y" + s], out["d" + s] = got["y"], got["dx"]
        if gain is not None:
            out[f"d{s}_gain"] = got["dgain"]
    return out


def check(copies, heads, n, axes, rows, device, eps=1e-6, gains=True, seed=0):
    print(f"head norm {copies} H={heads} N={n} axes={axes} {rows}", flush=True)
    made = inputs(copies, heads, n, axes, rows, seed, gains)
    got = run(made, copies, heads, eps, device)
    want = wanted(made, copies, heads, eps, torch.finfo(tables_dtype(rows)).eps)
    assert set(got) == set(want)
    for name in want:
        compare(got[name], want[name], name)


LAYOUTS = [({0: 4, 1: 4, 2: 4}, 8), ({0: 4, 1: 4, 2: 4}, 1), ({0: 8, 1: 8, 2: 8}, 16), ({0: 2, 1: 2, 2: 2}, 4),
           ({0: 1, 1: 1, 2: 1}, 8), ({0: 11, 1: 5, 2: 3}, 3), ({0: 3, 1: 2, 2: 1}, 5), ({0: 12}, 8), ({0: 1}, 1),
           ({0: 1}, 7), ({1: 1}, 1), ({1: 4, 2: 4}, 8), ({2: 3}, 2), ({0: 5, 3: 2, 10: 1}, 4), ({0: 4, 1: 4}, 6),
           ({f: 1 for f in range(8)}, 9), ({0: 2, 1: 1}, 64), ({0: 4, 1: 2}, 33), ({0: 3}, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", LAYOUTS)
def test_every_layout_and_type(copies, heads, rows, cuda):
    check(copies, heads, 37, 2, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 1024}, 1), ({0: 1023}, 1), ({0: 15}, 64), ({1: 512}, 1), ({1: 8}, 64),
                                          ({0: 64, 1: 64, 2: 64}, 3), ({0: 256, 1: 128, 2: 256}, 1),
                                          ({0: 1, 1: 1}, 64)])
def test_the_widest_rows(copies, heads, rows, cuda):
    check(copies, heads, 21, 1, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 3, 7, 16, 31, 32, 33, 255, 4097, 60_001])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 3, 1: 1}, 3)])
def test_numbers_of_rows(copies, heads, n, rows, cuda):
    check(copies, heads, n, 2, rows, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 4097, 12_289, 60_001, 200_001])
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("eps", [None, 3.0])
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 8), ({0: 11, 1: 5, 2: 3}, 3), ({0: 12}, 8)])
def test_gains_gradients_over_every_row(copies, heads, eps, rows, n, cuda):
    """Sums over more rows than the workgroups hold at once, of numbers whose sums are exact: rows of 1 and -1 (under
    the norm, mean 1 and eps 3, of halves), gradients of whole numbers up to 2.  All the terms together, 2 n
    heads of up to 2, stay below 2^24 of their units (6.4 million), so every row counts once, to the last bit, in any
    order."""
    head = SO2FieldType(copies)
    gen = torch.Generator(device=cuda).manual_seed(n)
    D = heads * head.dimension
    q, k = (2.0 * torch.randint(0, 2, (n, D), generator=gen, device=cuda) - 1 for _ in range(2))
    up = [torch.randint(-2, 3, (n, D), generator=gen, device=cuda).double() for _ in range(2)]
    gains = [torch.ones(sum(copies.values()), dtype=tables_dtype(rows), device=cuda, requires_grad=True)
             for _ in range(2)]
    outs = query_key_norm(q.to(rows), k.to(rows), head, heads, *gains, eps=eps)
    grads = torch.autograd.grad(outs, gains, [u.to(rows) for u in up])
    for x, u, got in zip((q, k), up, grads):
        terms, want, at = (x * u).sum(0), [], 0  # whole numbers in double
        for f, c in copies.items():
            w = c * (1 if f == 0 else 2)
            want.append(terms[at:at + heads * w].reshape(heads, c, -1).sum((0, 2)))
            at += heads * w
        want = torch.cat(want) * (1.0 if eps is None else 0.5)
        assert torch.equal(got.double(), want)
        assert n == 1 or bool((want != 0).any())


@pytest.mark.gpu
@pytest.mark.parametrize("eps,gains,axes", [(1e-6, True, 0), (1e-6, False, 2), (1e-6, False, 0), (None, True, 2),
                                            (None, False, 1), (None, True, 0), (0.5, True, 8)])
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 5}])
def test_every_part_left_out(copies, eps, gains, axes, cuda):
    made = inputs(copies, 4, 200, min(axes, 4), torch.float32, gains=gains)
    if axes == 8:
        made["positions"] = made["positions"].repeat(1, 2)
        made["frequencies"] = made["frequencies"].repeat(2, 1)
    got = run(made, copies, 4, eps, cuda)
    for name, want in wanted(made, copies, 4, eps, torch.finfo(torch.float32).eps).items():
        compare(got[name], want, name)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 4), ({0: 3, 1: 2}, 5)])
def test_rows_at_odd_addresses_and_strides(copies, heads, rows, cuda):
    """Halves of one product's output, columns of a wider table, a shifted address, a transposed table, gradients with
    gaps and rows all the same."""
    made = inputs(copies, heads, 45, 2, rows)
    want = wanted(made, copies, heads, 1e-6, torch.finfo(tables_dtype(rows)).eps)
    n, D = made["q"].shape

    def halves(q, k):
        both = torch.cat([q, k], 1).to(cuda)
        return both[:, :D], both[:, D:]

    def columns(*ts):
        return [torch.empty(n, D + 7, dtype=t.dtype, device=cuda)[:, 3:3 + D].copy_(t) for t in ts]

    def shifted(*ts):
        return [torch.empty(t.numel() + 1, dtype=t.dtype, device=cuda)[1:].view(t.shape).copy_(t) for t in ts]

    def turned(*ts):
        return [torch.empty(D, n, dtype=t.dtype, device=cuda).t().copy_(t) for t in ts]

    place = dict(positions=made["positions"].to(cuda).float().double(), frequencies=made["frequencies"].to(cuda))
    place["positions"] = made["positions"].to(cuda)
    gains = [made[s].to(cuda).requires_grad_(True) for s in ("q_gain", "k_gain")]
    for view in (halves, columns, shifted, turned):
        leaves = [t.detach().requires_grad_(True) for t in view(made["q"], made["k"])]
        outs = query_key_norm(*leaves, SO2FieldType(copies), heads, *gains, **place)
        assert all(o.is_contiguous() for o in outs)
        grads = torch.autograd.grad(outs, [*leaves, *gains], columns(*made["up"]))
        for name, t in zip(("yq", "yk", "dq", "dk", "dq_gain", "dk_gain"), (*outs, *grads)):
            compare(t, want[name], (view.__name__, name))
    one = made["q"][:1].to(cuda).expand(n, D)
    same = query_key_norm(one, one, SO2FieldType(copies), heads, **place)[0]
    alone = query_key_norm(one.contiguous(), one.contiguous(), SO2FieldType(copies), heads, **place)[0]
    assert torch.equal(same, alone)


@pytest.mark.gpu
def test_whichever_gradients_are_asked_for(cuda):
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    made = inputs(copies, heads, 77, 2, torch.float32)
    every = run(made, copies, heads, 1e-6, cuda)
    for need in (("q",), ("k",), ("q_gain",), ("k_gain",), ("q", "k"), ("q", "k_gain"), ("q_gain", "k_gain")):
        got = run(made, copies, heads, 1e-6, cuda, need)
        assert set(got) == {"yq", "yk", *("d" + n for n in need)}
        for name in got:
            torch.testing.assert_close(got[name], every[name], rtol=1e-5, atol=1e-5)
    # one output used alone: the other's rows get no gradient
    leaves = [made[n].to(cuda).requires_grad_(True) for n in ("q", "k", "q_gain", "k_gain")]
    out = query_key_norm(leaves[0], leaves[1], SO2FieldType(copies), heads, leaves[2], leaves[3],
                         positions=made["positions"].to(cuda), frequencies=made["frequencies"].to(cuda))[1]
    grads = torch.autograd.grad(out, leaves, made["up"][1].to(cuda), allow_unused=True)
    assert grads[0] is None and grads[2] is None
    torch.testing.assert_close(grads[1], every["dk"])
    torch.testing.assert_close(grads[3], every["dk_gain"], rtol=1e-5, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_the_smallest_and_largest_numbers(rows, cuda):
    """Rows whose squares pass the type's range, or vanish in it, are normalised as any other; a row of zeros stays."""
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    made = inputs(copies, heads, 6, 2, rows)
    for i, size in enumerate((1e30, 1e-30, 3e37, 1e-3, 0.0)):
        made["q"][i] = (made["q"][i].double().clamp(-3, 3) * size).to(rows)
    got = run(made, copies, heads, 1e-6, cuda)
    for name, want in wanted(made, copies, heads, 1e-6, torch.finfo(torch.float32).eps).items():
        compare(got[name], want, name)
    assert not bool(got["yq"][4].any())


@pytest.mark.gpu
@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 4), ({0: 1, 1: 1}, 2), ({0: 11, 1: 5, 2: 3}, 3)])
def test_products_that_cancel(copies, heads, rows, cuda):
    """Whole numbers: sums of a piece's products are often zero though its terms are not."""
    made = inputs(copies, heads, 500, 0, rows, gains=False)
    for t in (made["q"], made["k"], *made["up"]):
        t.copy_(t.round().clamp(-2, 2))
    got = run(made, copies, heads, 1e-6, cuda)
    for name, want in wanted(made, copies, heads, 1e-6, torch.finfo(tables_dtype(rows)).eps).items():
        compare(got[name], want, name)


@pytest.mark.gpu
def test_infinite_and_nan_heads_stay_in_their_heads(cuda):
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    made = inputs(copies, heads, 20, 2, torch.float32)
    want = run(made, copies, heads, 1e-6, cuda)
    for row, value in ((3, math.nan), (7, math.inf), (19, -math.inf)):
        made["q"][row, 5] = value  # a scalar of the second head
    got = run(made, copies, heads, 1e-6, cuda)
    head = torch.zeros(80, dtype=torch.bool)
    for first, width in ((0, 4), (16, 8), (48, 8)):
        head[first + width:first + 2 * width] = True
    bad = torch.zeros(20, dtype=torch.bool)
    bad[[3, 7, 19]] = True
    for name in ("yq", "dq"):
        assert bool(got[name].cpu()[bad][:, head].isnan().any(1).all())
        clean = ~(bad.unsqueeze(1) & head)
        assert torch.equal(got[name].cpu()[clean], want[name].cpu()[clean])
    for name in ("yk", "dk", "dk_gain"):
        assert torch.equal(got[name], want[name])


@pytest.mark.gpu
def test_angles_of_far_positions(cuda):
    """A position of 2^31 hours and one beside it differ by their frequency's angle."""
    copies, heads = {0: 4, 1: 4}, 2
    head, n = SO2FieldType(copies), 64
    made = inputs(copies, heads, 1, 1, torch.float32)
    q = made["q"].expand(n, -1).contiguous()
    frequencies = torch.full((1, 6), 2 * math.pi / 24, dtype=torch.float64)
    hours = (2.0 ** 31 + torch.arange(n, dtype=torch.float64)).unsqueeze(1)
    got = query_key_norm(q.to(cuda), q.to(cuda), head, heads, positions=hours.to(cuda),
                         frequencies=frequencies.to(cuda))[0]
    near = (hours - 2.0 ** 31) + 2.0 ** 31 % 24  # whole days earlier
    want = query_key_norm(q.to(cuda), q.to(cuda), head, heads, positions=near.to(cuda),
                          frequencies=frequencies.to(cuda))[0]
    # both angles to 2^-52 of 2^31 pi / 12: 1.2e-7, of rows of 2 / sqrt(mean) at most sqrt(12)
    torch.testing.assert_close(got, want, rtol=0, atol=2e-6)


@pytest.mark.gpu
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 4, 2: 4}, 4), ({0: 3, 1: 2}, 2)])
def test_gradients_against_differences(copies, heads, cuda):
    """In float64, central differences along random directions: a step of h = 1e-5 is off by h^2 / 6 of the third
    derivative, of order one, and by eps / h = 2e-11 of the sum's terms."""
    made = inputs(copies, heads, 25, 2, torch.float64)
    got = run(made, copies, heads, 1e-6, cuda)
    place = {n: made[n].to(cuda) for n in ("positions", "frequencies")}
    names = ("q", "k", "q_gain", "k_gain")
    base = [made[n].to(cuda) for n in names]

    def loss(q, k, qg, kg):
        outs = query_key_norm(q, k, SO2FieldType(copies), heads, qg, kg, **place)
        return float(sum((o * u.to(cuda)).sum() for o, u in zip(outs, made["up"])))

    h = 1e-5
    for i, name in enumerate(names):
        step = torch.randn(base[i].shape, dtype=torch.float64, generator=torch.Generator().manual_seed(i)).to(cuda)
        up, down = (loss(*(x + s * h * step if i == j else x for j, x in enumerate(base))) for s in (1, -1))
        terms = got["d" + name] * step
        assert abs((up - down) / (2 * h) - float(terms.sum())) <= 1e-6 * float(terms.abs().sum()), name


@pytest.mark.gpu
def test_scores_depend_on_differences_of_positions(cuda):
    """All nodes moved by the same amounts: every pair's score stays."""
    copies, heads = {0: 4, 1: 4, 2: 4}, 2
    made = inputs(copies, heads, 30, 2, torch.float64, gains=False)
    q, k, f = (made[n].to(cuda) for n in ("q", "k", "frequencies"))
    for axis, moved in ((0, 0.7), (1, -12.5)):
        scores = []
        for shift in (0.0, moved):
            at = made["positions"].clone()
            at[:, axis] += shift
            qr, kr = query_key_norm(q, k, SO2FieldType(copies), heads, positions=at.to(cuda), frequencies=f)
            scores.append(qr @ kr.t())
        torch.testing.assert_close(*scores, rtol=1e-11, atol=1e-11)


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 4, 1: 4, 2: 4}, {0: 3, 1: 1}])
def test_replays_of_two_captured_steps_equal_the_eager_ones(copies, cuda):
    made = [{n: v.to(cuda) for n, v in inputs(copies, 8, 300, 2, torch.float32, seed=s).items() if n != "up"}
            for s in (0, 20)]
    ups = [[u.to(cuda) for u in inputs(copies, 8, 300, 2, torch.float32, seed=s)["up"]] for s in (0, 20)]

    def step(m, up):
        leaves = [m[n].detach().requires_grad_(True) for n in ("q", "k", "q_gain", "k_gain")]
        outs = query_key_norm(leaves[0], leaves[1], SO2FieldType(copies), 8, leaves[2], leaves[3],
                              positions=m["positions"], frequencies=m["frequencies"])
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, up)]

    want = [[t.clone() for t in step(m, u)] for m, u in zip(made, ups)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for m, u in zip(made, ups):
            step(m, u)
    torch.cuda.current_stream().wait_stream(side)
    captured, got = [torch.cuda.CUDAGraph() for _ in range(2)], []
    for c, m, u in zip(captured, made, ups):
        with torch.cuda.graph(c):
            got.append(step(m, u))
    for replay in range(3):
        for out in got:
            for t in out:
                t.zero_()
        for c in captured:
            c.replay()
        torch.cuda.synchronize()
        for out, w, m, u in zip(got, want, made, ups):
            assert all(torch.equal(a, b) for a, b in zip(out, w)), replay
            assert all(torch.equal(a, b) for a, b in zip(step(m, u), w)), replay
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_no_rows(cuda):
    for device in (cuda, "cpu"):
        leaves = [torch.zeros(0, 80, device=device, requires_grad=True) for _ in range(2)]
        gains = [torch.ones(12, device=device, requires_grad=True) for _ in range(2)]
        outs = query_key_norm(*leaves, SO2FieldType({0: 4, 1: 4, 2: 4}), 4, *gains,
                              positions=torch.zeros(0, 1, device=device), frequencies=torch.ones(1, 10, device=device))
        assert all(o.shape == (0, 80) for o in outs)
        for x, g in zip((*leaves, *gains), torch.autograd.grad(outs, (*leaves, *gains), outs)):
            assert g.shape == x.shape and not bool(g.any())


@pytest.mark.gpu
def test_rows_beyond_the_kernels_bounds_run_in_torch(cuda):
    check({0: 1030}, 1, 9, 1, torch.float32, cuda)
    check({0: 2, 1: 1}, 65, 9, 1, torch.float32, cuda)
    check({f: 1 for f in range(9)}, 2, 9, 1, torch.float32, cuda)


@pytest.mark.gpu
def test_on_another_stream_and_the_modules_tables(cuda):
    """A module's first call on one stream behind other work, its next on another at once."""
    head = SO2FieldType({0: 4, 1: 4, 2: 4})
    made = inputs({0: 4, 1: 4, 2: 4}, 4, 500, 2, torch.float32)
    q, k, at = (made[n].to(cuda) for n in ("q", "k", "positions"))
    module = SO2QueryKeyNorm(head, 4, frequencies=made["frequencies"], device=cuda)
    want = module.forward_flat(q, k, at)
    torch.cuda.synchronize()
    busy = torch.randn(4096, 4096, device=cuda)
    for _ in range(20):
        busy = busy @ busy * 1e-3
    other = SO2QueryKeyNorm(head, 4, frequencies=made["frequencies"], device=cuda)
    other.forward_flat(q, k, at)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = other.forward_flat(q, k, at)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_modules_first_call_is_before_a_capture(cuda):
    head = SO2FieldType({0: 4, 1: 4, 2: 4})
    made = inputs({0: 4, 1: 4, 2: 4}, 4, 50, 2, torch.float32)
    q, k, at = (made[n].to(cuda) for n in ("q", "k", "positions"))
    module, other = (SO2QueryKeyNorm(head, 4, frequencies=made["frequencies"], device=cuda).requires_grad_(False)
                     for _ in range(2))
    want = [t.clone() for t in module.forward_flat(q, k, at)]
    torch.cuda.synchronize()
    captured = torch.cuda.CUDAGraph()
    with torch.cuda.graph(captured):
        with pytest.raises(RuntimeError, match="before the capture"):
            other.forward_flat(q, k, at)
        got = module.forward_flat(q, k, at)
    for _ in range(2):
        for t in got:
            t.zero_()
        captured.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))
    assert all(torch.equal(a, b) for a, b in zip(other.forward_flat(q, k, at), want))


@pytest.mark.gpu
def test_a_module_called_in_inference_mode_trains_on_the_gpu(cuda):
    inference_first(cuda)


# ---------------------------------------------------------------- without a GPU


def test_a_module_called_in_inference_mode_trains():
    inference_first("cpu")


def inference_first(device):
    """What its first call keeps serves a later step's backward."""
    copies, heads = {0: 4, 1: 4, 2: 4}, 4
    made = inputs(copies, heads, 9, 2, torch.float32)
    at, up = made["positions"].to(device), [u.to(device) for u in made["up"]]
    modules = [SO2QueryKeyNorm(SO2FieldType(copies), heads, frequencies=made["frequencies"], device=device)
               for _ in range(2)]
    with torch.inference_mode():
        modules[0].forward_flat(made["q"].to(device), made["k"].to(device), at)
    assert not modules[0]._on(at.device).is_inference()
    grads = []
    for module in modules:
        leaves = [made[n].to(device).requires_grad_(True) for n in ("q", "k")] + list(module.parameters())
        grads.append(torch.autograd.grad(module.forward_flat(*leaves[:2], at), leaves, up))
    assert all(torch.equal(a, b) for a, b in zip(*grads))


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("copies,heads", [({0: 4, 1: 2, 2: 1}, 3), ({0: 3, 1: 1}, 2), ({0: 5}, 1), ({2: 2}, 4)])
def test_cpu_rows_take_the_formulas_in_torch(copies, heads, rows):
    # torch sums a head's squares in the rows' arithmetic: a half step a number more, few of the bound's
    check(copies, heads, 12, 2, rows, "cpu")


@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_the_smallest_and_largest_numbers_on_the_cpu(rows):
    test_the_smallest_and_largest_numbers(rows, "cpu")


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [torch.float32, torch.bfloat16])
def test_the_largest_numbers_beyond_the_kernels_bounds(rows, cuda):
    """As within them: 65 heads run in torch."""
    copies, heads = {0: 2, 1: 1}, 65
    made = inputs(copies, heads, 4, 1, rows)
    for i, size in enumerate((1e30, 3e37, 1e20)):
        made["q"][i] = (made["q"][i].double().clamp(-3, 3) * size).to(rows)
    got = run(made, copies, heads, 1e-6, cuda)
    for name, want in wanted(made, copies, heads, 1e-6, torch.finfo(torch.float32).eps).items():
        compare(got[name], want, name)


def test_module_is_its_function_and_survives_casts_and_copies():
    head = SO2FieldType({0: 4, 1: 2})
    frequencies = rotary_frequencies(head, (8.0, 5.0), (0.3, 1.0), (False, True))
    module = SO2QueryKeyNorm(head, 2, frequencies=frequencies)
    q, k = (problems.normal((9, 16), i).float() for i in range(2))
    at = problems.normal((9, 2), 2).double()
    want = query_key_norm(q, k, head, 2, module.query_gain, module.key_gain, positions=at, frequencies=frequencies)
    for other in (module, copy.deepcopy(module), pickle.loads(pickle.dumps(module)),
                  copy.deepcopy(module).to(torch.bfloat16).float()):
        assert all(torch.equal(a, b) for a, b in zip(other.forward_flat(q, k, at), want))
    assert set(module.state_dict()) == {"query_gain", "key_gain"} and "query_gain" in dir(module)
    assert not list(SO2QueryKeyNorm(head, 2, gain=False).parameters())


@pytest.mark.gpu
def test_the_module_takes_fields_on_the_gpu(cuda):
    fields_of(cuda)


def test_the_module_takes_fields():
    fields_of("cpu")


def fields_of(device):
    """Called, it gives what its flat form does, in the fields' shape, and its hooks run."""
    head, heads = SO2FieldType({0: 4, 1: 2}), 3
    full = head.scaled(heads)
    frequencies = rotary_frequencies(head, (8.0, 5.0), (0.3, 1.0), (False, True))
    at = problems.normal((2, 7, 2), 2).double().to(device)
    q, k = (problems.normal((2, 7, full.dimension), i).float().to(device) for i in range(2))
    for module, given in ((SO2QueryKeyNorm(head, heads, frequencies=frequencies, device=device), (at,)),
                          (SO2QueryKeyNorm(head, heads, device=device), ())):
        called = []
        module.register_forward_hook(lambda *_: called.append(1))
        got = module(*(SO2FeatureField.from_flat(full, x) for x in (q, k)), *given)
        want = module.forward_flat(q.flatten(0, 1), k.flatten(0, 1), *(p.flatten(0, 1) for p in given))
        assert called == [1]
        for a, b in zip(got, want):
            assert a.field_type == full and torch.equal(a.to_flat(), b.reshape(2, 7, -1))
    field = SO2FeatureField.from_flat(full, q)
    for call, message in (((SO2FeatureField.from_flat(SO2FieldType({0: 24}), q), field), "Expected a field of type"),
                          ((field, SO2FeatureField.from_flat(full, k[:1])), "on the same nodes"),
                          ((field, field, at), "exactly where there are frequencies"),
                          ((field, field, at[0]), r"positions must be \(2, 7, axes\)")):
        with pytest.raises(ValueError, match=message):
            module(*call)


def test_frequencies_are_dealt_to_the_axes():
    got = rotary_frequencies(SO2FieldType({0: 5, 1: 3}), (16.0, 7.3), (1.0, 0.2), (False, True))
    assert got.shape == (2, 5) and got.dtype == torch.float64
    torch.testing.assert_close(got[0], torch.tensor([16.0, 0.0, 4.0, 0.0, 1.0], dtype=torch.float64))
    torch.testing.assert_close(got[1], torch.tensor([0.0, 7.0, 0.0, 1.0, 0.0], dtype=torch.float64))
    for highest, lowest, whole in (((1.0,), (2.0,), None), ((1.0,), (0.0,), None), ((), (), None),
                                   ((1.0,), (1.0, 1.0), None), ((1.0,), (1.0,), (True, True))):
        with pytest.raises(ValueError):
            rotary_frequencies(SO2FieldType({1: 1}), highest, lowest, whole)


def test_refusals():
    head = SO2FieldType({0: 4, 1: 2})
    q, gain = torch.zeros(3, 16), torch.ones(6)
    at, f = torch.zeros(3, 1), torch.ones(1, 4)

    def call(q=q, k=None, q_gain=gain, eps=1e-6, positions=at, frequencies=f, heads=2, head=head):
        return query_key_norm(q, q if k is None else k, head, heads, q_gain, gain, eps=eps, positions=positions,
                              frequencies=frequencies)

    assert call()[0].shape == (3, 16)
    for kw, message in ((dict(k=q.double()), "share a shape, dtype"), (dict(k=q[:2]), "share a shape"),
                        (dict(q=q.half()), "float32, float64 or bfloat16"), (dict(q=q[:, :15]), "rows must be"),
                        (dict(q=q[0]), "rows must be"), (dict(heads=3), "rows must be"), (dict(heads=0), "at least 1"),
                        (dict(eps=0.0), "eps must be positive"), (dict(eps=-1.0), "eps must be positive"),
                        (dict(eps=math.nan), "eps must be positive"),
                        (dict(positions=None), "go together"), (dict(frequencies=None), "go together"),
                        (dict(positions=at[:2]), r"positions must be \(3, 1\)"),
                        (dict(frequencies=f[:, :3]), r"frequencies must be \(axes, 4\)"),
                        (dict(frequencies=torch.ones(9, 4), positions=torch.ones(3, 9)), "1..8 axes"),
                        (dict(frequencies=torch.ones(0, 4), positions=torch.ones(3, 0)), "1..8 axes"),
                        (dict(positions=at.clone().requires_grad_(True)), "constants"),
                        (dict(positions=at.cfloat()), "must be real"),
                        (dict(q_gain=gain[:5]), "a gain must be"), (dict(q_gain=gain.long()), "a gain must be")):
        with pytest.raises(ValueError, match=message):
            call(**kw)
    with pytest.raises(TypeError, match="head_type must be"):
        call(head={0: 8})
    with pytest.raises(ValueError, match="nothing to do"):
        query_key_norm(q, q, head, 2, eps=None)
    for kw, message in ((dict(eps=0.0), "eps must be positive"),
                        (dict(frequencies=torch.ones(1, 3)), "frequencies must"),
                        (dict(norm=False, gain=False), "nothing to do")):
        with pytest.raises(ValueError, match=message):
            SO2QueryKeyNorm(head, 2, **kw)
    with pytest.raises(ValueError, match="exactly where there are frequencies"):
        SO2QueryKeyNorm(head, 2).forward_flat(q, q, at)
    with pytest.raises(ValueError, match="exactly where there are frequencies"):
        SO2QueryKeyNorm(head, 2, frequencies=f).forward_flat(q, q)


def test_the_library_refuses_bad_arguments():
    """Through the C interface, before anything is launched (no GPU touched)."""
    import ctypes

    from gm_attention_amd import _native

    lib = _native.library()
    pair, strides = (ctypes.c_void_p * 2)(None, None), (ctypes.c_int64 * 2)(16, 16)

    def forward(rows=((0, 4, 0, 0, 1), (1, 2, 8, 0, 2)), n=0, D=16, H=2, sets=2, axes=0, eps=1e-6, x=pair):
        flat = [v for row in rows for v in row]
        desc = (ctypes.c_int64 * len(flat))(*flat)
        return lib.gm_head_norm_forward_f32(x, strides, pair, sets, ctypes.cast(desc, ctypes.c_void_p), n, D,
                                            len(rows), H, None, None, axes, 1, eps, pair, None)

    assert forward() == 0
    for kw, message in ((dict(n=-1), b"non-negative"), (dict(n=1), b"device pointers"), (dict(sets=3), b"one set"),
                        (dict(sets=0), b"one set"), (dict(axes=9), b"at most 8 axes"), (dict(H=65), b"at most 64"),
                        (dict(D=20), b"fill the flat width"), (dict(eps=-1.0), b"eps must not"),
                        (dict(x=None), b"host arrays"),
                        (dict(rows=((1, 2, 0, 0, 2), (0, 4, 8, 0, 1))), b"must rise")):
        assert forward(**kw) == 1
        assert message in lib.gm_last_error(), kw
