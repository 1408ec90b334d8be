"""The neighbourhood softmax with a learned relative bias, and the norm and
rotation of queries and keys, as training and inference programs call them.

* ``relative``: every head's softmax over each target's edges of ``scale <q_i,
  tau k_j> + bias(e) + table[bucket(e), head]``, ``table`` learned, the buckets a
  property of the edge (its ring of distance and side here); inference, or
  training with the gradients of the rows and of the table.
* ``query_key``: the query and key rows' heads normalised by their root mean
  square, multiplied by a gain a copy and turned by an angle a copy that is
  linear in the node's position; any of the three may be missing; inference, or
  training with the gradients of the rows and gains.

With ``own`` false both run in their plain form, elementary tensor operations in
32 bits (the angles, of far positions too, in 64); with ``own`` true they are the
package's operators.
"""

from __future__ import annotations

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

EPS = 1e-6
FILL = 1e20  # what a data set writes where it has no value


# ---------------------------------------------------------------- the cases


def _relative(name, nlat, nlon, batch, heads, copies, buckets, rows=3.0, window="hard", missing=0.0, bf16=False,
              train=True):
    return dict(name=name, kind="relative", nlat=nlat, nlon=nlon, batch=batch, heads=heads, copies=copies,
                buckets=buckets, rows=rows, window=window, missing=missing, bf16=bf16, train=train)


def _query_key(name, nodes, heads, copies, axes=2, norm=True, gain=True, packed=False, bf16=False, train=True):
    return dict(name=name, kind="query_key", nodes=nodes, heads=heads, copies=copies, axes=axes, norm=norm, gain=gain,
                packed=packed, bf16=bf16, train=train)


def listed():
    return [
        # one small sample through a trained layer, four heads: latency
        _relative("relative-infer-32x64", 32, 64, 1, 4, "16,16,16", 16, train=False),
        # a training step on a small odd grid: six heads, fewer copies at the higher frequencies, a taper, and nodes
        # without data (some targets keep no neighbour)
        _relative("relative-train-45x91-uneven", 45, 91, 3, 6, "24,12,12", 21, rows=2.5, window="quartic",
                  missing=0.2),
        # a training step with bfloat16 rows, the block's usual ones
        _relative("relative-train-bf16-64x128", 64, 128, 4, 8, "32,32,32", 32, bf16=True),
        # a training step of a wider layer with a fine table
        _relative("relative-train-128x256-wide", 128, 256, 2, 16, "64,64,64", 96),
        # inference on a whole-degree grid, one sample, bfloat16 rows
        _relative("relative-infer-bf16-181x360", 181, 360, 1, 8, "32,32,32", 32, bf16=True, train=False),
        # the headline layer's training step: 63 M edges, degrees from 42 to 2,048
        _relative("relative-train-256x512", 256, 512, 4, 8, "32,32,32", 32),
        # a single node's query and key: latency
        _query_key("query-key-infer-one", 1, 8, "32,32,32", bf16=True, train=False),
        # one small sample through a trained layer: latency
        _query_key("query-key-infer-32x64", 32 * 64, 4, "16,16,16", train=False),
        # odd multiplicities, three heads, three samples of a small odd grid, both rows from one product
        _query_key("query-key-train-45x91-odd", 3 * 45 * 91, 3, "33,15,9", axes=3, packed=True),
        # the headline layer's nodes in float32
        _query_key("query-key-train-256x512", 4 * 256 * 512, 8, "32,32,32"),
        # the same layer of a block with bfloat16 rows
        _query_key("query-key-train-bf16-256x512", 4 * 256 * 512, 8, "32,32,32", bf16=True),
        # inference of a model's wide stage, both rows from one product
        _query_key("query-key-infer-bf16-64x128-wide", 8 * 64 * 128, 16, "128,128,128", axes=3, packed=True,
                   bf16=True, train=False),
    ]


#: copies a head at frequencies 0, 1, 2 that layers are drawn with
_PER_HEAD = ((4, 4, 4), (4, 4, 4), (4, 4, 4), (2, 2, 2), (8, 8, 8), (1, 1, 1), (4, 2, 2), (2, 1, 1), (4, 4), (8, 4, 2),
             (3, 2, 1), (5, 3, 3), (12,), (0, 4, 4))
#: a drawn case's points times copies a point, and its rows' numbers, stay within the largest listed ones
_MOST_RELATIVE = 4 * 256 * 512 * 96
_MOST_QUERY_KEY = 4 * 256 * 512 * 160


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    heads = rng.choice((1, 2, 4, 4, 6, 8, 8, 8, 16))
    per = rng.choice(_PER_HEAD)
    if heads * sum(c * (1 if f == 0 else 2) for f, c in enumerate(per)) > 640:
        per = (2, 2, 2)
    copies = ",".join(str(heads * c) for c in per)
    width = heads * sum(c * (1 if f == 0 else 2) for f, c in enumerate(per))
    bf16, train = rng.random() < 0.4, rng.random() < 0.65
    if rng.random() < 0.55:
        nlat = _log_uniform(rng, 12, 250)
        nlon = max(8, 2 * nlat + rng.choice((0, 0, -1, 1, 5)))
        batch = rng.randint(1, 4)
        while batch > 1 and nlat * nlon * batch * heads * sum(per) > _MOST_RELATIVE:
            batch -= 1
        if nlat * nlon * heads * sum(per) > _MOST_RELATIVE:
            nlat, nlon = 120, 241
        case = _relative("", nlat, nlon, batch, heads, copies, _log_uniform(rng, 1, 256),
                         round(rng.uniform(1.6, 3.0), 2), rng.choice(("hard", "quartic")),
                         rng.choice((0.0, 0.0, 0.1, 0.3)), bf16, train)
    else:
        nodes = _log_uniform(rng, 1, min(524288, _MOST_QUERY_KEY // width))
        axes, norm = rng.choice((0, 1, 2, 2, 3)), rng.random() < 0.85
        if axes == 0:
            norm = True
        case = _query_key("", nodes, heads, copies, axes, norm, norm and rng.random() < 0.85, rng.random() < 0.4,
                          bf16, train)
    del case["name"]
    return case


def _copies(case):
    return {f: int(c) for f, c in enumerate(case["copies"].split(",")) if int(c)}


def _width(copies):
    return sum(c * (1 if f == 0 else 2) for f, c in copies.items())


def _head(case):
    return {f: c // case["heads"] for f, c in _copies(case).items()}


# ---------------------------------------------------------------- what a program has in hand


def _row_pairs(nlat, nlon, radius):
    """Per grid row the neighbours of its first node, as ``(row, steps east)``
    pairs with their distance and the angle that turns the neighbour's frame into
    the node's; the other nodes of a row see the same ones turned with them."""
    theta = np.pi * np.arange(nlat) / (nlat - 1)
    step = 2 * np.pi / nlon
    starts, rows, steps, distances, angles, sides = [0], [], [], [], [], []
    for i in range(nlat):
        for j in range(max(0, i - 4), min(nlat, i + 5)):
            d = np.arange(-((nlon - 1) // 2), nlon // 2 + 1)
            c = np.cos(theta[i]) * np.cos(theta[j]) + np.sin(theta[i]) * np.sin(theta[j]) * np.cos(d * step)
            near = np.arccos(np.clip(c, -1, 1)) <= radius + 1e-7
            d, c = d[near], c[near]
            phi = d * step
            p = [np.stack([np.sin(t) * np.cos(a), np.sin(t) * np.sin(a), np.cos(t) + 0 * a], -1)
                 for t, a in ((theta[i], 0 * phi), (theta[j], phi))]
            south = [np.stack([np.cos(t) * np.cos(a), np.cos(t) * np.sin(a), -np.sin(t) + 0 * a], -1)
                     for t, a in ((theta[i], 0 * phi), (theta[j], phi))]
            east = [np.stack([-np.sin(a), np.cos(a), 0 * a], -1) for a in (0 * phi, phi)]
            chord = p[1] - p[0]
            here = np.arctan2((chord * east[0]).sum(-1), (chord * south[0]).sum(-1))
            there = np.arctan2((chord * east[1]).sum(-1), (chord * south[1]).sum(-1))
            distance = 2 * np.arcsin(np.clip(np.linalg.norm(chord, axis=-1) / 2, 0, 1))
            # coincident nodes (a pole's) differ by their frames' own turn about it
            turn = np.where(distance > 1e-9, here - there, np.where(i == 0, phi, -phi))
            rows.append(np.full(d.shape, j))
            steps.append(d)
            distances.append(distance)
            angles.append(turn)
            sides.append(np.full(d.shape, int(np.sign(j - i)) + 1))
        starts.append(sum(len(r) for r in rows))
    return np.array(starts), *(np.concatenate(x) for x in (rows, steps, distances, angles, sides)), theta


def _neighbours(case, device):
    """The edges of an equiangular grid within ``rows`` row spacings, target by
    target, one disjoint copy a sample: ``row_ptr``, ``source``, ``target``, the
    transport phases of orders 0.., the log window and quadrature weight, the
    window's support, and every edge's bucket: its ring of distance, on its side
    (north, the same row, south) where there are three buckets or more."""
    nlat, nlon = case["nlat"], case["nlon"]
    cutoff = case["rows"] * math.pi / (nlat - 1)
    starts, rows, steps, distances, angles, sides, theta = _row_pairs(nlat, nlon, cutoff)
    rings = case["buckets"] // 3 if case["buckets"] >= 3 else case["buckets"]
    buckets = np.minimum(np.floor(rings * distances / cutoff), rings - 1).astype(np.int64)
    if case["buckets"] >= 3:
        buckets += rings * sides
    starts, rows, steps, buckets = (torch.from_numpy(x).to(device) for x in (starts, rows, steps, buckets))
    distances, angles = (torch.from_numpy(x).to(device) for x in (distances, angles))
    degree = starts[1:] - starts[:-1]
    per_node = degree.repeat_interleave(nlon).repeat(case["batch"])
    row_ptr = torch.cat([per_node.new_zeros(1), per_node.cumsum(0)])
    n_edges = int(row_ptr[-1])
    target = torch.repeat_interleave(torch.arange(per_node.numel(), device=device), per_node, output_size=n_edges)
    at = torch.arange(n_edges, device=device) - row_ptr[target]
    node = target % (nlat * nlon)
    pair = starts[node // nlon] + at
    source = target - node + rows[pair] * nlon + (node % nlon + steps[pair]) % nlon
    top = max(_copies(case))
    orders = torch.arange(top + 1, device=device) * angles.unsqueeze(-1)
    phases = torch.stack([torch.cos(orders), torch.sin(orders)], dim=-1)
    window = torch.ones_like(distances) if case["window"] == "hard" else \
        torch.relu(1.0 - (distances / cutoff) ** 2) ** 2
    weight = torch.from_numpy(np.sin(theta).clip(0.25 * math.pi / (nlat - 1))).to(device)[rows] * \
        (math.pi / (nlat - 1)) * (2 * math.pi / nlon)
    tiny = torch.finfo(torch.float32).tiny
    bias = torch.log(window.clamp_min(tiny)) + torch.log(weight)
    return dict(row_ptr=row_ptr, source=source, target=target, transport=phases.float()[pair].contiguous(),
                bias=bias.float()[pair].contiguous(), inside=(window > 0)[pair].to(torch.uint8),
                buckets=buckets.to(torch.int32)[pair])


def _relative_inputs(case, device, gen, dtype):
    D = _width(_copies(case))
    state = dict(case=case, **_neighbours(case, device))
    n = state["row_ptr"].numel() - 1
    q, k = (torch.randn(n, D, generator=gen, device=device) for _ in range(2))
    if case["missing"]:
        # whole runs of nodes hold no data, and none of their edges count, in or out
        runs = torch.rand((n + 63) // 64, generator=gen, device=device) < case["missing"]
        gone = runs.repeat_interleave(64)[:n]
        state["inside"] *= (~(gone[state["target"]] | gone[state["source"]])).to(torch.uint8)
        q, k = (t.masked_fill(gone.unsqueeze(-1), FILL) for t in (q, k))
    state.update(q=q.to(dtype), k=k.to(dtype),
                 table=0.5 * torch.randn(case["buckets"], case["heads"], generator=gen, device=device))
    if case["train"]:
        state["upstream"] = torch.randn(state["source"].numel(), case["heads"], generator=gen, device=device)
    return state


def _relative_ranges(state):
    """Ranges of targets whose edges' rows fit in memory beside the rest."""
    ptr = state["row_ptr"].cpu().numpy()
    most, ends, last = 320_000_000 // state["q"].shape[1], [0], 0
    while last < len(ptr) - 1:
        last = max(last + 1, int(np.searchsorted(ptr, ptr[last] + most, side="right")) - 1)
        ends.append(last)
    state["ranges"] = [(a, b, int(ptr[a]), int(ptr[b])) for a, b in zip(ends, ends[1:])]


def _relative_kept(state):
    """The package's tables of the edge set, which a program builds once for it."""
    from gm_attention_amd.nn.relative import RelativeEdgeTables
    from gm_attention_amd.representations.field_type import SO2FieldType

    case = state["case"]
    del state["target"]
    state["head_type"] = SO2FieldType(_head(case))
    state["tables"] = RelativeEdgeTables(state["row_ptr"], state["source"], state["transport"], state["bias"],
                                         state["inside"], state["buckets"], case["buckets"])
    if case["train"]:
        state["tables"].group_sources()
        for name in ("q", "k", "table"):
            state[name].requires_grad_(True)


def _slots(head):
    """The copies of a head that have an angle: pairs of scalar copies, then every copy above frequency 0."""
    return head.get(0, 0) // 2 + sum(c for f, c in head.items() if f)


def _positions(case, device, gen):
    """Latitude, longitude and a time in hours since an epoch, the first ``axes`` of them; and each slot's
    radians a unit of its one axis: whole wave numbers of longitude, periods of time from hours to decades."""
    n, axes, slots = case["nodes"], case["axes"], _slots(_head(case))
    columns = [torch.linspace(-0.5 * math.pi, 0.5 * math.pi, n, dtype=torch.float64, device=device),
               2 * math.pi * torch.rand(n, generator=gen, device=device, dtype=torch.float64),
               torch.floor(1e6 * torch.rand(n, generator=gen, device=device, dtype=torch.float64))]
    frequencies = torch.zeros(axes, slots, dtype=torch.float64)
    for i in range(slots):
        step = i // axes
        frequencies[i % axes, i] = (2.0 ** step, 1.0 + step, 2 * math.pi / 6.0 * 0.05 ** step)[i % axes]
    return torch.stack(columns[:axes], dim=1), frequencies.to(device)


def _query_key_inputs(case, device, gen, dtype):
    copies = _copies(case)
    n, D = case["nodes"], _width(copies)
    rows = (1.3 * torch.randn(n, 2 * D, generator=gen, device=device) + 0.1).to(dtype)
    q, k = rows[:, :D], rows[:, D:]
    if not case["packed"]:
        q, k = q.contiguous(), k.contiguous()
    state = dict(case=case, q=q, k=k)
    if case["gain"]:
        for name in ("q_gain", "k_gain"):
            state[name] = 1.0 + 0.1 * torch.randn(sum(_head(case).values()), generator=gen, device=device)
    if case["axes"]:
        state["positions"], state["frequencies"] = _positions(case, device, gen)
    if case["train"]:
        state["upstream"] = [torch.randn(n, D, generator=gen, device=device).to(dtype) for _ in range(2)]
    return state


def _query_key_kept(state):
    from gm_attention_amd.representations.field_type import SO2FieldType

    state["head_type"] = SO2FieldType(_head(state["case"]))
    if state["case"]["train"]:
        for name in ("q", "k", "q_gain", "k_gain"):
            if name in state:
                state[name].requires_grad_(True)


def _inputs(case, seed):
    device = torch.device("cuda")
    gen = torch.Generator(device=device).manual_seed(seed)
    make = _relative_inputs if case["kind"] == "relative" else _query_key_inputs
    return make(case, device, gen, torch.bfloat16 if case["bf16"] else torch.float32)


def prepare(case, seed):
    state = _inputs(case, seed)
    relative = case["kind"] == "relative"
    if own:
        package = str(Path.cwd() / "gm-attention_amd")
        if package not in sys.path:
            sys.path.insert(0, package)
        (_relative_kept if relative else _query_key_kept)(state)
    elif relative:
        _relative_ranges(state)
    return state


# ---------------------------------------------------------------- one pass


def _turned(rows, copies, phases, sign):
    """Every pair of the rows turned by its frequency's phase (``sign`` -1: back)."""
    out, at = [], 0
    for f, c in copies.items():
        w = c * (1 if f == 0 else 2)
        block = rows[:, at:at + w]
        if f:
            re, im = block.reshape(-1, c, 2).unbind(-1)
            cos, sin = phases[:, f, 0:1], sign * phases[:, f, 1:2]
            block = torch.stack([cos * re - sin * im, cos * im + sin * re], dim=-1).reshape(-1, w)
        out.append(block)
        at += w
    return torch.cat(out, dim=1)


def _by_head(rows, copies, heads):
    """The rows' numbers as ``(heads, numbers of one head)``, frequency by frequency."""
    out, at = [], 0
    for f, c in copies.items():
        w = c * (1 if f == 0 else 2)
        out.append(rows[:, at:at + w].reshape(-1, heads, w // heads))
        at += w
    return torch.cat(out, dim=2)


def _by_row(heads, copies):
    """The inverse of :func:`_by_head`."""
    out, at = [], 0
    for f, c in copies.items():
        w = c * (1 if f == 0 else 2) // heads.shape[1]
        out.append(heads[:, :, at:at + w].reshape(heads.shape[0], -1))
        at += w
    return torch.cat(out, dim=1)


def _relative_plain(s):
    case, copies = s["case"], _copies(s["case"])
    heads = case["heads"]
    scale = 1.0 / math.sqrt(_width(copies) / heads)
    q, k, table = s["q"].float(), s["k"].float(), s["table"]
    alpha = q.new_empty(s["source"].numel(), heads)
    if case["train"]:
        dq, dk = torch.zeros_like(q), torch.zeros_like(k)
        # millions of edges a bucket: in 64 bits, every 4,096th edge's sum first (few numbers meet in one place)
        dtable = torch.zeros(4096 * table.shape[0], heads, dtype=torch.float64, device=q.device)
    for a, b, e0, e1 in s["ranges"]:
        at, source, phases = s["target"][e0:e1] - a, s["source"][e0:e1], s["transport"][e0:e1]
        bucket = s["buckets"][e0:e1]
        qe = _by_head(q[a:b].index_select(0, at), copies, heads)
        ke = _by_head(_turned(k.index_select(0, source), copies, phases, 1.0), copies, heads)
        score = scale * (qe * ke).sum(-1) + s["bias"][e0:e1].unsqueeze(-1) + table.index_select(0, bucket)
        score = score.masked_fill((s["inside"][e0:e1] == 0).unsqueeze(-1), float("-inf"))
        index = at.unsqueeze(-1).expand(-1, heads)
        most = score.new_full((b - a, heads), float("-inf")).scatter_reduce_(0, index, score, "amax")
        most = most.masked_fill(most == float("-inf"), 0.0)  # nothing inside: every weight is zero
        weight = torch.exp(score - most.index_select(0, at))
        total = score.new_zeros(b - a, heads).index_add_(0, at, weight)
        weight = weight / total.masked_fill(total == 0, 1.0).index_select(0, at)
        alpha[e0:e1] = weight
        if not case["train"]:
            continue
        g = s["upstream"][e0:e1]
        mean = score.new_zeros(b - a, heads).index_add_(0, at, weight * g)
        ds = weight * (g - mean.index_select(0, at))
        dtable.index_add_(0, 4096 * bucket.long() + torch.arange(e1 - e0, device=q.device) % 4096, ds.double())
        ds = (scale * ds).unsqueeze(-1)
        dq[a:b].index_add_(0, at, _by_row(ds * ke, copies))
        dk.index_add_(0, source, _turned(_by_row(ds * qe, copies), copies, phases, -1.0))
    if not case["train"]:
        return dict(alpha=alpha)
    dtable = dtable.reshape(-1, 4096, heads).sum(1).float()
    return dict(alpha=alpha, dq=dq.to(s["q"].dtype), dk=dk.to(s["k"].dtype), dtable=dtable)


def _query_key_plain(s):
    case, copies, head = s["case"], _copies(s["case"]), _head(s["case"])
    heads, train = case["heads"], case["train"]
    a0, spans = head.get(0, 0), [c * (1 if f == 0 else 2) for f, c in head.items()]
    if case["axes"]:
        angle = s["positions"] @ s["frequencies"]
        cos, sin = torch.cos(angle).float().unsqueeze(1), torch.sin(angle).float().unsqueeze(1)

    def one(rows, gain):
        x = _by_head(rows.float(), copies, heads)
        if case["norm"]:
            x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS)
        if gain is not None:
            x = x * torch.cat([g if f == 0 else g.repeat_interleave(2)
                               for f, g in zip(head, gain.split(list(head.values())))])
        if case["axes"]:
            scalars, rest = x.split([a0, sum(spans) - a0], dim=-1)
            kept = scalars[..., a0 - a0 % 2:]
            pairs = torch.cat([scalars[..., :a0 - a0 % 2], rest], dim=-1)
            re, im = pairs.reshape(*pairs.shape[:2], -1, 2).unbind(-1)
            pairs = torch.stack([cos * re - sin * im, cos * im + sin * re], dim=-1).flatten(2)
            x = torch.cat([pairs[..., :a0 - a0 % 2], kept, pairs[..., a0 - a0 % 2:]], dim=-1)
        return _by_row(x, copies).to(rows.dtype)

    with torch.set_grad_enabled(train):
        v = {n: s[n].detach().requires_grad_(train) for n in ("q", "k", "q_gain", "k_gain") if n in s}
        outs = [one(v["q"], v.get("q_gain")), one(v["k"], v.get("k_gain"))]
        if not train:
            return outs
        grads = torch.autograd.grad(outs, list(v.values()), s["upstream"])
    return [o.detach() for o in outs] + list(grads)


def _relative_own(s):
    from gm_attention_amd.nn.relative import relative_softmax

    case = s["case"]
    with torch.set_grad_enabled(case["train"]):
        alpha = relative_softmax(s["q"], s["k"], s["table"], s["tables"], s["head_type"], case["heads"])
        if not case["train"]:
            return dict(alpha=alpha)
        dq, dk, dtable = torch.autograd.grad(alpha, (s["q"], s["k"], s["table"]), s["upstream"])
    return dict(alpha=alpha.detach(), dq=dq, dk=dk, dtable=dtable)


def _query_key_own(s):
    from gm_attention_amd.nn.head_norm import query_key_norm

    case = s["case"]
    with torch.set_grad_enabled(case["train"]):
        outs = query_key_norm(s["q"], s["k"], s["head_type"], case["heads"], s.get("q_gain"), s.get("k_gain"),
                              eps=EPS if case["norm"] else None, positions=s.get("positions"),
                              frequencies=s.get("frequencies"))
        if not case["train"]:
            return list(outs)
        grads = torch.autograd.grad(outs, [s[n] for n in ("q", "k", "q_gain", "k_gain") if n in s], s["upstream"])
    return [o.detach() for o in outs] + list(grads)


def run(state):
    if state["case"]["kind"] == "relative":
        return _relative_own(state) if own else _relative_plain(state)
    return _query_key_own(state) if own else _query_key_plain(state)


# ---------------------------------------------------------------- what a pass cannot do without


def _edges(case):
    starts = _row_pairs(case["nlat"], case["nlon"], case["rows"] * math.pi / (case["nlat"] - 1))[0]
    return int(starts[-1]) * case["nlon"] * case["batch"]


def work(case):
    copies = _copies(case)
    D = _width(copies)
    b = 2 if case["bf16"] else 4
    if case["kind"] == "relative":
        n, e, h = case["nlat"] * case["nlon"] * case["batch"], _edges(case), case["heads"]
        # ids, bias, support, bucket, phases of the orders above 0
        tables = e * (8 + 4 + 1 + 4 + 8 * max(copies)) + 8 * n
        # a score: a product a scalar copy, four a pair and the turn; the gradients of q and k as much each
        flops = 2.0 * e * sum(c * (1 if f == 0 else 4) for f, c in copies.items())
        if not case["train"]:
            return dict(bytes=tables + 2 * n * D * b + 4 * e * h, flops=flops)
        return dict(bytes=tables + 4 * n * D * b + 8 * e * h, flops=3 * flops)
    n = case["nodes"]
    rows, flops = 4 * n * D * b + 8 * n * case["axes"], 14.0 * n * D
    if case["train"]:
        # the gradients of both outputs in, those of both rows out
        rows += 4 * n * D * b
        flops *= 3
    return dict(bytes=rows, flops=flops)


# ---------------------------------------------------------------- the definition in 64 bits


def _relative_exact(s):
    """Head by head over the whole edge set, in complex double arithmetic."""
    case, copies = s["case"], _copies(s["case"])
    heads, train = case["heads"], case["train"]
    source, target, bucket = s["source"], s["target"], s["buckets"].long()
    n = s["row_ptr"].numel() - 1
    tau = {f: torch.complex(s["transport"][:, f, 0].double(), s["transport"][:, f, 1].double()) for f in copies if f}
    scale = (_width(copies) / heads) ** -0.5
    outside = s["inside"] == 0
    table = s["table"].double()
    starts = dict(zip(copies, np.cumsum([0] + [c * (1 if f == 0 else 2) for f, c in copies.items()])))

    def column(rows, f, c):
        """Copy ``c`` of frequency ``f``: a real column, or a complex one."""
        if f == 0:
            return rows[:, starts[f] + c].double()
        return torch.complex(rows[:, starts[f] + 2 * c].double(), rows[:, starts[f] + 2 * c + 1].double())

    def put(rows, f, c, v):
        if f == 0:
            rows[:, starts[f] + c] = v
        else:
            rows[:, starts[f] + 2 * c], rows[:, starts[f] + 2 * c + 1] = v.real, v.imag

    def sums(index, v, size=n):
        if v.is_complex():
            return torch.complex(sums(index, v.real.contiguous(), size), sums(index, v.imag.contiguous(), size))
        return torch.zeros(size, dtype=torch.float64, device=v.device).index_add_(0, index, v)

    q, k = s["q"], s["k"]
    alpha = torch.zeros(source.numel(), heads, dtype=torch.float64, device=q.device)
    if train:
        dq, dk = (torch.zeros(t.shape, dtype=torch.float64, device=t.device) for t in (q, k))
        dtable = torch.zeros_like(table)
    for h in range(heads):
        mine = [(f, h * (c // heads) + u) for f, c in copies.items() for u in range(c // heads)]
        score = torch.zeros(source.numel(), dtype=torch.float64, device=q.device)
        for f, c in mine:
            a, b = column(q, f, c)[target], column(k, f, c)[source]
            score += a * b if f == 0 else (a.conj() * tau[f] * b).real
        score = scale * score + s["bias"].double() + table[:, h][bucket]
        score[outside] = -math.inf
        top = torch.full((n,), -math.inf, dtype=torch.float64, device=q.device)
        top.scatter_reduce_(0, target, score, "amax")
        w = torch.exp(score - torch.where(top.isinf(), torch.zeros_like(top), top)[target])
        w /= sums(target, w).clamp_min(1e-300)[target]
        alpha[:, h] = w
        if train:
            g = s["upstream"][:, h].double()
            ds = w * (g - sums(target, w * g)[target])
            # a bucket's sum by every 4,096th edge first: few numbers meet in one place
            spread = bucket * 4096 + torch.arange(bucket.numel(), device=q.device) % 4096
            dtable[:, h] = sums(spread, ds, 4096 * table.shape[0]).reshape(-1, 4096).sum(1)
            ds = scale * ds
            for f, c in mine:
                a, b = column(q, f, c)[target], column(k, f, c)[source]
                put(dq, f, c, sums(target, ds * b if f == 0 else ds * tau[f] * b))
                put(dk, f, c, sums(source, ds * a if f == 0 else ds * tau[f].conj() * a))
    return dict(alpha=alpha, dq=dq, dk=dk, dtable=dtable) if train else dict(alpha=alpha)


def _query_key_exact(s):
    """The formulas and their derivatives column by column in double."""
    case, copies, head = s["case"], _copies(s["case"]), _head(s["case"])
    heads, dev = case["heads"], s["q"].device
    starts = dict(zip(copies, np.cumsum([0] + [c * (1 if f == 0 else 2) for f, c in copies.items()])))
    firsts = dict(zip(head, np.cumsum([0] + list(head.values()))))
    numbers = _width(head)
    # a head's parts: (the column of its first number, of its second or None, their copies, its angle's slot or None)
    parts = []
    for h in range(heads):
        mine, slot = [], 0
        for f, c in head.items():
            base = int(starts[f]) + h * c * (1 if f == 0 else 2)
            for u in range(0, c, 2 if f == 0 else 1):
                copy = int(firsts[f]) + u
                if f:
                    mine.append((base + 2 * u, base + 2 * u + 1, copy, copy, slot))
                elif u + 1 < c:
                    mine.append((base + u, base + u + 1, copy, copy + 1, slot))
                else:
                    mine.append((base + u, None, copy, copy, None))
                slot += mine[-1][4] is not None
        parts.append(mine)
    turn = torch.polar(torch.ones((), dtype=torch.float64, device=dev),
                       s["positions"] @ s["frequencies"]) if case["axes"] else None

    def one(rows, gain, g):
        x = rows.double()
        out = torch.empty_like(x)
        dx = torch.empty_like(x) if g is not None else None
        dgain = torch.zeros(sum(head.values()), dtype=torch.float64, device=dev)
        gains = torch.ones_like(dgain) if gain is None else gain.double()
        for mine in parts:
            columns = [c for p in mine for c in p[:2] if c is not None]
            inv = (x[:, columns].pow(2).sum(1) / numbers + EPS).pow(-0.5) if case["norm"] else \
                torch.ones(x.shape[0], dtype=torch.float64, device=dev)
            mean, back = torch.zeros_like(inv), {}
            for c0, c1, u0, u1, slot in mine:
                if c1 is None:
                    hat = inv * x[:, c0]
                    out[:, c0] = gains[u0] * hat
                    if g is not None:
                        d = g[:, c0].double()
                        dgain[u0] += (d * hat).sum()
                        back[c0] = gains[u0] * d
                        mean += back[c0] * hat
                    continue
                z = torch.complex(gains[u0] * inv * x[:, c0], gains[u1] * inv * x[:, c1])
                if turn is not None:
                    z = z * turn[:, slot]
                out[:, c0], out[:, c1] = z.real, z.imag
                if g is not None:
                    d = torch.complex(g[:, c0].double(), g[:, c1].double())
                    if turn is not None:
                        d = d * turn[:, slot].conj()
                    for c, u, v in ((c0, u0, d.real), (c1, u1, d.imag)):
                        hat = inv * x[:, c]
                        dgain[u] += (v * hat).sum()
                        back[c] = gains[u] * v
                        mean += back[c] * hat
            if g is not None:
                for c, v in back.items():
                    dx[:, c] = inv * (v - inv * x[:, c] * mean / numbers) if case["norm"] else v
        return out, dx, dgain

    up = s.get("upstream", (None, None))
    got = [one(s[n], s.get(n + "_gain"), u) for n, u in zip(("q", "k"), up)]
    outs = [g[0] for g in got]
    if case["train"]:
        outs += [g[1] for g in got]
        if case["gain"]:
            outs += [g[2] for g in got]
    return outs


def exact(case, seed):
    state = _inputs(case, seed)
    with torch.no_grad():
        return _relative_exact(state) if case["kind"] == "relative" else _query_key_exact(state)
