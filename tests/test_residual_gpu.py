"""The residual sum between two norms (nn/residual.py) against its formulas and
their derivatives written out in float64.

Tolerances: every result is compared within ``ROUNDINGS * eps / 2`` of the
magnitude its own chain of roundings can reach -- the formula with every term's
absolute value in its place (a centred value counts |x| + mean |x|) -- with
ROUNDINGS = 96: the longest chain takes two row sums (of at most 16 numbers a
lane and six shuffle steps each, twice), a sum over a lane's rows and one over
workgroups (pairwise in blocks, under 40 in sequence at these sizes), and under
twenty products, quotients and exponentials.  A result held in bfloat16 is off by
another eps / 2 = 2^-8 of its value.
"""

import copy
import itertools
import pickle

import pytest
import torch

import problems
from gm_attention_amd.nn import residual
from gm_attention_amd.nn.nonlinearities import SO2ScalarGatedNonlinearity
from gm_attention_amd.nn.normalization import SO2LayerNorm
from gm_attention_amd.nn.residual import SO2ResidualNorm
from gm_attention_amd.representations.field_type import SO2FieldType

ROUNDINGS = 96


def _copy_index(copies):
    out, at = [], 0
    for f, c in copies.items():
        out.append(torch.arange(at, at + c).repeat_interleave(1 if f == 0 else 2))
        at += c
    return torch.cat(out)


def oracle(copies, v, post, gate, scale, norm, eps=1e-5):
    """Values and magnitudes of every output and gradient: ``{name: (value, magnitude)}``."""
    index, C, a0, present = _copy_index(copies), sum(copies.values()), copies.get(0, 0), len(copies)
    D = index.numel()
    scalar = torch.arange(D) < a0
    share = torch.cat([torch.full((c * (1 if f == 0 else 2),), 1.0 / (present * c * (1 if f == 0 else 2)),
                                  dtype=torch.float64) for f, c in copies.items()])

    def mean0(x):
        return torch.where(scalar, x[:, :a0].mean(1, keepdim=True), 0.0) if a0 else torch.zeros_like(x)

    def spread(x):
        return torch.zeros(*x.shape[:-1], C, dtype=x.dtype).index_add_(-1, index, x)

    def offset(b):
        return torch.cat([b, b.new_zeros(D - a0)])

    x, u = v["x"], v["u"]
    if post:
        c = u - mean0(u)
        inv = 1.0 / (c.square() @ share + eps).sqrt().unsqueeze(1)
        uh, muh = c * inv, (u.abs() + mean0(u.abs())) * inv
        gain, off = v["post.gamma"][index], offset(v["post.beta"])
    else:
        uh, muh, inv = u, u.abs(), 1.0
        gain, off = torch.ones(D, dtype=torch.float64), torch.zeros(D, dtype=torch.float64)
    factor = {"": 1.0, "sigmoid": 1.0, "double_sigmoid": 2.0}[gate]
    sig = torch.sigmoid(v["z"]) if gate else None
    act = factor * sig[:, index] if gate else torch.ones_like(x)
    s = v["scale"][index] if scale else torch.ones(D, dtype=torch.float64)
    b, mb = gain * uh + off, gain.abs() * muh + off.abs()
    y, my = x + s * act * b, x.abs() + s.abs() * act * mb
    out = {"y": (y, my)}
    G, mG = v["dy"], v["dy"].abs()
    if norm:
        c2 = y - mean0(y)
        inv2 = 1.0 / (c2.square() @ share + eps).sqrt().unsqueeze(1)
        xh, mxh = c2 * inv2, (my + mean0(my)) * inv2
        g2, b2 = v["norm.gamma"][index], offset(v["norm.beta"])
        out["normed"] = (g2 * xh + b2, g2.abs() * mxh + b2.abs())
        gh = g2 * v["dn"]
        G = G + inv2 * (gh - mean0(gh) - (gh * xh).sum(1, keepdim=True) * share * xh)
        mG = mG + inv2 * (gh.abs() + mean0(gh.abs()) + (gh.abs() * mxh).sum(1, keepdim=True) * share * mxh)
        out["norm.gamma"] = (spread((v["dn"] * xh).sum(0)), spread((v["dn"].abs() * mxh).sum(0)))
        out["norm.beta"] = (v["dn"][:, :a0].sum(0), v["dn"][:, :a0].abs().sum(0))
    out["x"] = (G, mG)
    if gate:
        d = factor * sig * (1 - sig)
        out["z"] = (spread(G * s * b) * d, spread(mG * s.abs() * mb) * factor * sig)
    inner, minner = G * act * s, mG * act * s.abs()
    if post:
        gu, mgu = inner * gain, minner * gain.abs()
        out["u"] = (inv * (gu - mean0(gu) - (gu * uh).sum(1, keepdim=True) * share * uh),
                    inv * (mgu + mean0(mgu) + (mgu * muh).sum(1, keepdim=True) * share * muh))
        out["post.gamma"] = (spread((inner * uh).sum(0)), spread((minner * muh).sum(0)))
        out["post.beta"] = (inner[:, :a0].sum(0), minner[:, :a0].sum(0))
    else:
        out["u"] = (inner, minner)
    if scale:
        out["scale"] = (spread((G * act * b).sum(0)), spread((mG * act * mb).sum(0)))
    return out


def values(copies, nodes, post, gate, scale, norm, dtype, branch, seed=0):
    """Seeded inputs as the rows' types hold them, in float64."""
    C, a0 = sum(copies.values()), copies.get(0, 0)
    D = sum(c * (1 if f == 0 else 2) for f, c in copies.items())
    pd = torch.float64 if dtype == torch.float64 else torch.float32

    def normal(i, *shape, to=dtype):
        return problems.normal(shape, 10 * seed + i).to(to).double()

    v = {"x": (1.5 * normal(0, nodes, D) + 0.3).to(dtype).double(),
         "u": (0.5 * normal(1, nodes, D)).to(branch).double(), "dy": normal(2, nodes, D)}
    if gate:
        v["z"] = normal(3, nodes, C)
    if norm:
        v["dn"] = normal(4, nodes, D)
    for i, name in enumerate((["post"] if post else []) + (["norm"] if norm else [])):
        v[name + ".gamma"] = (1 + 0.2 * normal(5 + i, C, to=pd)).to(pd).double()
        v[name + ".beta"] = (0.2 * normal(7 + i, a0, to=pd)).to(pd).double()
    if scale:
        v["scale"] = (0.5 + 0.2 * normal(9, C, to=pd)).to(pd).double()
    return v


def module_of(copies, v, post, gate, scale, norm, dtype, device):
    pd = torch.float64 if dtype == torch.float64 else torch.float32
    m = SO2ResidualNorm(SO2FieldType(copies), post_norm=post, gate=gate or None, scale=0.5 if scale else None,
                        norm=norm, dtype=pd, device=device)
    named = {}
    for kind in ("post", "norm"):
        if getattr(m, kind) is not None:
            named[kind + ".gamma"] = [getattr(m, kind).gamma[str(f)] for f in copies]
            if 0 in copies:
                named[kind + ".beta"] = [getattr(m, kind).beta]
    if m.scale is not None:
        named["scale"] = [m.scale[str(f)] for f in copies]
    with torch.no_grad():
        for name, ps in named.items():
            for p, w in zip(ps, v[name].split([p.numel() for p in ps])):
                p.copy_(w)
    return m, named


def compare(got, want, what, dtype):
    value, magnitude = want
    eps = torch.finfo(torch.float64 if dtype == torch.float64 else torch.float32).eps
    tol = ROUNDINGS * eps / 2 * magnitude
    if got.dtype == torch.bfloat16:
        tol = tol + torch.finfo(torch.bfloat16).eps / 2 * (value.abs() + tol)
    off = (got.detach().double().cpu() - value).abs()
    assert got.shape == value.shape, what
    assert bool((off <= tol).all()), f"{what}: {float((off / tol.clamp_min(1e-300)).max())} of the tolerance"


def check(copies, nodes, post, gate, scale, norm, dtype, branch, device, view=None):
    print(f"residual {copies} n={nodes} post={post} gate={gate} scale={scale} norm={norm} {dtype} {branch}", flush=True)
    v = values(copies, nodes, post, gate, scale, norm, dtype, branch)
    want = oracle(copies, v, post, gate, scale, norm)
    m, named = module_of(copies, v, post, gate, scale, norm, dtype, device)
    put = (lambda t, to: t.to(to).to(device)) if view is None else (lambda t, to: view(t.to(to).to(device)))
    leaves = {"x": put(v["x"], dtype).requires_grad_(True), "u": put(v["u"], branch).requires_grad_(True)}
    if gate:
        leaves["z"] = put(v["z"], dtype).requires_grad_(True)
    outs = m.forward_flat(leaves["x"], leaves["u"], leaves.get("z"))
    assert (outs[1] is None) == (not norm)
    outs = [o for o in outs if o is not None]
    for o, name in zip(outs, ("y", "normed")):
        assert o.dtype == dtype
        compare(o, want[name], name, dtype)
    inputs = list(leaves.values()) + [p for ps in named.values() for p in ps]
    ups = [put(v["dy"], dtype)] + ([put(v["dn"], dtype)] if norm else [])
    grads = iter(torch.autograd.grad(outs, inputs, ups))
    for name, leaf in leaves.items():
        g = next(grads)
        assert g.dtype == leaf.dtype
        compare(g, want[name], "d" + name, dtype)
    for name, ps in named.items():
        compare(torch.cat([next(grads) for _ in ps]), want[name], "d" + name, dtype)
    with torch.no_grad():  # without a backward to follow: the same numbers
        again = [o for o in m.forward_flat(leaves["x"], leaves["u"], leaves.get("z")) if o is not None]
    for a, b in zip(outs, again):
        assert torch.equal(a, b)


FIELDS = [{0: 32, 1: 32, 2: 32}, {0: 33, 1: 17, 2: 9}, {0: 8, 1: 8}, {0: 4, 1: 2}, {1: 3, 2: 5}, {0: 1}, {0: 7},
          {0: 64, 1: 64, 2: 64}, {0: 1, 1: 1}, {1: 16}, {0: 24, 1: 12, 2: 6}]
FLOATS = [(torch.float32, torch.float32), (torch.float64, torch.float64), (torch.bfloat16, torch.bfloat16),
          (torch.bfloat16, torch.float32)]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,branch", FLOATS)
@pytest.mark.parametrize("copies", FIELDS)
def test_every_field_and_type(copies, dtype, branch, cuda):
    check(copies, 77, True, "double_sigmoid", True, True, dtype, branch, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("post,gate,scale,norm", list(itertools.product((True, False), ("", "sigmoid"), (True, False),
                                                                         (True, False))))
@pytest.mark.parametrize("copies", [{0: 8, 1: 8, 2: 8}, {0: 3, 1: 5}])
def test_every_part_left_out(post, gate, scale, norm, copies, cuda):
    check(copies, 50, post, gate, scale, norm, torch.float32, torch.float32, cuda)
    check(copies, 50, post, gate, scale, norm, torch.bfloat16, torch.float32, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("nodes", [1, 2, 31, 33, 4096, 20011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_numbers_of_rows(nodes, dtype, cuda):
    check({0: 16, 1: 16, 2: 16}, nodes, True, "sigmoid", True, True, dtype, dtype, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 1024}, {0: 1023}, {1: 512}, {0: 256, 1: 384}, {0: 204, 1: 205, 2: 205},
                                    {0: 128, 1: 128, 2: 128}])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
def test_the_widest_rows(copies, dtype, cuda):
    check(copies, 9, True, "sigmoid", True, True, dtype, dtype, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_rows_at_odd_addresses_and_strides(dtype, cuda):
    """Views whose first row is not at a multiple of 16 bytes, and rows of a wider table."""
    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        return flat[1:].view(t.shape).copy_(t)

    def strided(t):
        return torch.empty(t.shape[0], t.shape[1] + 5, dtype=t.dtype, device=t.device)[:, 3:-2].copy_(t)

    for view in (shifted, strided):
        check({0: 8, 1: 8}, 21, True, "sigmoid", True, True, dtype, dtype, cuda,
              view=lambda t: view(t.detach()))


@pytest.mark.gpu
def test_no_rows(cuda):
    m = SO2ResidualNorm(SO2FieldType({0: 4, 1: 4}), scale=1.0, device=cuda)
    x, u = (torch.zeros(0, 12, device=cuda, requires_grad=True) for _ in range(2))
    y, h = m.forward_flat(x, u)
    assert y.shape == h.shape == (0, 12)
    for g in torch.autograd.grad([y, h], [x, u, *m.parameters()], [y, h]):
        assert bool((g == 0).all())


@pytest.mark.gpu
def test_one_output_used_alone(cuda):
    """The gradient of the norm alone, or of the sum alone, with the other unused."""
    copies, dtype = {0: 16, 1: 16}, torch.float32
    v = values(copies, 40, True, "sigmoid", True, True, dtype, dtype)
    m, named = module_of(copies, v, True, "sigmoid", True, True, dtype, cuda)
    leaves = [v[n].float().to(cuda).requires_grad_(True) for n in ("x", "u", "z")]
    for used in ("dy", "dn"):
        w = dict(v, **{n: torch.zeros_like(v[n]) for n in ("dy", "dn") if n != used})
        want = oracle(copies, w, True, "sigmoid", True, True)
        outs = m.forward_flat(*leaves)
        grads = torch.autograd.grad(outs[0 if used == "dy" else 1], leaves, v[used].float().to(cuda))
        for g, name in zip(grads, ("x", "u", "z")):
            compare(g, want[name], f"d{name} of {used}", dtype)


@pytest.mark.gpu
def test_gradients_against_differences(cuda):
    """In float64, along random directions of every input and parameter: the
    fourth-order difference at step 1e-3 is off by about 1e-12 h^-4 f^(5) h^4 / 30
    and by roundings of 1e-16 / h = 1e-13 of the loss's magnitude."""
    copies, dtype = {0: 5, 1: 4, 2: 3}, torch.float64
    v = values(copies, 12, True, "double_sigmoid", True, True, dtype, dtype)
    m, named = module_of(copies, v, True, "double_sigmoid", True, True, dtype, cuda)
    leaves = [v[n].to(cuda).requires_grad_(True) for n in ("x", "u", "z")]
    params = [p for ps in named.values() for p in ps]
    ups = [v["dy"].to(cuda), v["dn"].to(cuda)]

    def loss(moved):
        with torch.no_grad():
            for p, w in zip(params, moved[3:]):
                p.copy_(w)
        return sum((o * g).sum() for o, g in zip(m.forward_flat(*moved[:3]), ups))

    start = [t.detach().clone() for t in leaves + params]
    grads = torch.autograd.grad(loss([*leaves, *start[3:]]), leaves + params)
    for i in range(len(start)):
        step = problems.normal(start[i].shape, 90 + i).to(cuda)

        def at(h):
            with torch.no_grad():
                return float(loss([t + h * step if j == i else t for j, t in enumerate(start)]))

        h = 1e-3
        slope = (8 * (at(h) - at(-h)) - (at(2 * h) - at(-2 * h))) / (12 * h)
        want = float((grads[i] * step).sum())
        assert abs(slope - want) <= 1e-8 * (1 + abs(want)), (i, slope, want)


@pytest.mark.gpu
def test_replays_of_a_captured_step_equal_the_eager_one(cuda):
    copies, dtype = {0: 32, 1: 32, 2: 32}, torch.float32
    v = values(copies, 3000, True, "sigmoid", True, True, dtype, dtype)
    m, named = module_of(copies, v, True, "sigmoid", True, True, dtype, cuda)
    params = [p for ps in named.values() for p in ps]
    x, u, z = (v[n].float().to(cuda) for n in ("x", "u", "z"))
    ups = [v["dy"].float().to(cuda), v["dn"].float().to(cuda)]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, u, z)]
        outs = m.forward_flat(*leaves)
        return [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves + params, ups)]

    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for replay in range(3):
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), replay
        assert all(torch.equal(a, b) for a, b in zip(step(), want)), replay
        torch.cuda.synchronize()


@pytest.mark.gpu
def test_on_another_stream(cuda):
    copies, dtype = {0: 16, 1: 16, 2: 16}, torch.float32
    v = values(copies, 500, True, "", True, True, dtype, dtype)
    m, _ = module_of(copies, v, True, "", True, True, dtype, cuda)
    x, u = v["x"].float().to(cuda), v["u"].float().to(cuda)
    with torch.no_grad():
        want = m.forward_flat(x, u)
        torch.cuda.synchronize()
        side = torch.cuda.Stream()
        with torch.cuda.stream(side):
            got = m.forward_flat(x, u)
        side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_nothing_is_kept_for_a_backward_that_cannot_follow(cuda, monkeypatch):
    m = SO2ResidualNorm(SO2FieldType({0: 16, 1: 16}), scale=1.0, device=cuda)
    x, u = (problems.normal((50, 48), i).float().to(cuda) for i in range(2))
    given, real = [], residual._native.residual_norm_forward
    monkeypatch.setattr(residual._native, "residual_norm_forward", lambda *a: given.append(a[-1]) or real(*a))
    with torch.no_grad():
        without = m.forward_flat(x, u)
    with_graph = m.forward_flat(x, u)
    m.requires_grad_(False)
    m.forward_flat(x, u)
    assert given == [False, True, False]
    assert all(torch.equal(a, b) for a, b in zip(without, with_graph))


@pytest.mark.gpu
def test_gradients_hold_no_workspace(cuda):
    m = SO2ResidualNorm(SO2FieldType({0: 16, 1: 16}), scale=1.0, device=cuda)
    x, u = (problems.normal((5000, 48), i).float().to(cuda) for i in range(2))
    y, h = m.forward_flat(x, u)
    (y.sum() + h.sum()).backward()
    assert all(p.grad.untyped_storage().nbytes() <= 4 * (3 * 32 + 2 * 16) for p in m.parameters())


@pytest.mark.gpu
def test_infinite_and_nan_rows_stay_in_their_rows(cuda):
    m = SO2ResidualNorm(SO2FieldType({0: 16, 1: 16, 2: 16}), scale=1.0, device=cuda)
    x, u = (problems.normal((200, 80), i).float().to(cuda) for i in range(2))
    x[17, 3] = float("inf")
    u[90, 41] = float("nan")
    y, h = m.forward_flat(x, u)
    bad = torch.zeros(200, dtype=torch.bool, device=cuda)
    bad[[17, 90]] = True
    assert bool(torch.isfinite(y[~bad]).all()) and bool(torch.isfinite(h[~bad]).all())
    assert not bool(torch.isfinite(h[bad]).all(dim=1).any())


# ---------------------------------------------------------------- without a GPU


@pytest.mark.parametrize("post,gate,scale,norm", [(True, "double_sigmoid", True, True), (False, "", False, True),
                                                  (True, "", True, False), (False, "sigmoid", False, False)])
@pytest.mark.parametrize("copies", [{0: 6, 1: 4, 2: 3}, {1: 3, 2: 2}, {0: 5}])
def test_cpu_rows_take_the_formulas_in_torch(copies, post, gate, scale, norm):
    dtype = torch.float64
    v = values(copies, 20, post, gate, scale, norm, dtype, dtype)
    want = oracle(copies, v, post, gate, scale, norm)
    m, named = module_of(copies, v, post, gate, scale, norm, dtype, "cpu")
    leaves = {n: v[n].clone().requires_grad_(True) for n in ("x", "u", "z") if n in v}
    outs = [o for o in m.forward_flat(leaves["x"], leaves["u"], leaves.get("z")) if o is not None]
    for o, name in zip(outs, ("y", "normed")):
        compare(o, want[name], name, dtype)
    grads = torch.autograd.grad(outs, list(leaves.values()), [v["dy"]] + ([v["dn"]] if norm else []))
    for name, g in zip(leaves, grads):
        compare(g, want[name], "d" + name, dtype)


def test_refusals():
    ft = SO2FieldType({0: 4, 1: 4})
    with pytest.raises(TypeError, match="SO2FieldType"):
        SO2ResidualNorm({0: 4})
    with pytest.raises(ValueError, match="eps must be positive"):
        SO2ResidualNorm(ft, eps=0.0)
    with pytest.raises(ValueError, match="gate must be None or one of"):
        SO2ResidualNorm(ft, gate="silu")
    m, gated = SO2ResidualNorm(ft), SO2ResidualNorm(ft, gate="sigmoid")
    x = torch.zeros(3, 12)
    with pytest.raises(ValueError, match=r"rows must be \(N, 12\)"):
        m.forward_flat(x[:, :8], x[:, :8])
    with pytest.raises(ValueError, match="branch must have the rows' shape"):
        m.forward_flat(x, x[:2])
    with pytest.raises(ValueError, match="pre must be given exactly where there is a gate"):
        m.forward_flat(x, x, torch.zeros(3, 8))
    with pytest.raises(ValueError, match="pre must be given exactly where there is a gate"):
        gated.forward_flat(x, x)
    with pytest.raises(ValueError, match=r"pre must be \(3, 8\)"):
        gated.forward_flat(x, x, torch.zeros(3, 7))
    with pytest.raises(ValueError, match="pre_activations needs a gate"):
        m.pre_activations(x[:, :4])


def test_the_library_refuses_bad_arguments():
    """Through the C interface, before anything is launched (no GPU touched)."""
    import ctypes

    from gm_attention_amd import _native

    lib = _native.library()
    offsets, mults = (ctypes.c_int64 * 1)(4), (ctypes.c_int64 * 1)(4)
    params = (ctypes.c_void_p * 8)()

    def forward(n=1, D=12, a0=4, nf=1, eps=1e-5):
        return lib.gm_residual_norm_forward_f32(None, None, None, ctypes.cast(params, ctypes.c_void_p), n, D, a0, nf,
                                                ctypes.cast(offsets, ctypes.c_void_p),
                                                ctypes.cast(mults, ctypes.c_void_p), 1.0, eps, eps, None, None, None,
                                                None)

    for kw, message in ((dict(n=-1), b"non-negative"), (dict(D=1025), b"1..1024"), (dict(a0=13), b"a0 must lie"),
                        (dict(D=14), b"fill the flat width"), (dict(nf=9), b"at most 8"), (dict(eps=0.0), b"eps"),
                        (dict(), b"device pointers")):
        assert forward(**kw) == 1
        assert message in lib.gm_last_error(), kw
    assert forward(n=0) == 0
    params[1] = 64  # the gains of one frequency alone (an address nothing reads)
    assert forward(n=0) == 1 and b"every frequency" in lib.gm_last_error()


@pytest.mark.parametrize("make", [SO2LayerNorm, SO2ScalarGatedNonlinearity, SO2ResidualNorm])
def test_modules_are_copied_with_their_layouts(make):
    """Modules keep their layout for the entry points; copies have their own."""
    m = make(SO2FieldType({0: 4, 1: 3, 2: 2}))
    args = m._layout().args()
    for other in (copy.deepcopy(m), pickle.loads(pickle.dumps(m))):
        layout = other._layout()
        assert layout is not m._layout() and layout.args()[:3] == args[:3]
        assert list(layout.offsets) == [4, 10] and list(layout.mults) == [3, 2]
        assert layout.args()[3].value != args[3].value


def test_a_used_module_is_copied():
    m = SO2ResidualNorm(SO2FieldType({0: 4, 1: 3}), scale=0.5)
    counts, params = m._params()
    m._layout().parameter_slots(counts)
    other = copy.deepcopy(m)
    x, u = (problems.normal((7, 10), i).float() for i in range(2))
    assert all(torch.equal(a, b) for a, b in zip(m.forward_flat(x, u), other.forward_flat(x, u)))
    assert other._layout().parameter_slots(counts)[1:] == m._layout().parameter_slots(counts)[1:]


# ------------------------------------------------------- where the parameters are read


def replica_of(module):
    """A module's replica as a data-parallel step makes one: its parameters are plain attributes."""
    replica = module._replicate_for_data_parallel()
    for key, child in module._modules.items():
        setattr(replica, key, None if child is None else replica_of(child))
    for key, p in module._parameters.items():
        if p is None:
            replica._parameters[key] = None
        else:
            setattr(replica, key, p * 1.0)
    return replica


def by_name(module):
    """The vectors of every group in the order of the field's frequencies."""
    keys = [str(f) for f in module.field_type.frequencies]
    named = dict(module.named_parameters())
    return [named[n] for group in (["post.gamma." + k for k in keys], ["post.beta"], ["scale." + k for k in keys],
                                   ["norm.gamma." + k for k in keys], ["norm.beta"]) for n in group if n in named]


FORMS = [dict(scale=0.5), dict(scale=0.5, norm=False), dict(post_norm=False, scale=1.0), dict(norm=False),
         dict(scale=0.5, bias=False)]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("copies", [{0: 4, 1: 3, 2: 2}, {1: 3, 2: 3}, {0: 3, 2: 3, 10: 3}, {2: 2, 9: 4, 11: 5}])
def test_parameters_are_read_by_frequency_in_modules_and_replicas(copies, form):
    module = SO2ResidualNorm(SO2FieldType(copies), **form)
    with torch.no_grad():
        for i, p in enumerate(module.parameters()):
            p.add_(torch.arange(p.numel()) + 10.0 * i)
    want = by_name(module)
    counts, params = module._params()
    assert len(params) == len(want) and all(a is b for a, b in zip(params, want))
    replicated, copied = replica_of(module)._params()
    assert replicated == counts
    assert len(copied) == len(want) and all(torch.equal(a, b) for a, b in zip(copied, want))


def test_pruned_and_parametrised_vectors_are_read_as_they_act():
    from torch.nn.utils import parametrize, prune

    class Doubled(torch.nn.Module):
        def forward(self, p):
            return 2 * p

    module = SO2ResidualNorm(SO2FieldType({0: 4, 1: 4}), scale=0.5)
    prune.custom_from_mask(module.post.gamma, "1", torch.tensor([1.0, 0.0, 1.0, 0.0]))
    parametrize.register_parametrization(module.norm.gamma, "0", Doubled())
    counts, params = module._params()
    assert counts == (2, 1, 2, 2, 1)
    assert params[1].tolist() == [1.0, 0.0, 1.0, 0.0]  # the branch's gains of frequency 1
    assert params[5].tolist() == [2.0] * 4  # the next norm's of frequency 0


@pytest.mark.gpu
@pytest.mark.parametrize("copies", [{0: 4, 2: 3, 10: 3}, {0: 5, 2: 2, 10: 4}, {2: 4, 11: 8}])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_frequencies_of_two_digits(copies, dtype, cuda):
    check(copies, 40, True, "sigmoid", True, True, dtype, dtype, cuda)


@pytest.mark.gpu
@pytest.mark.parametrize("form", FORMS)
def test_a_replica_gives_the_modules_results(form, cuda):
    from torch.nn.parallel import replicate

    module = SO2ResidualNorm(SO2FieldType({0: 8, 1: 8, 2: 4}), gate="sigmoid", device=cuda, **form)
    with torch.no_grad():
        for i, p in enumerate(module.parameters()):
            p.add_(0.1 * problems.normal(p.shape, i).float().to(cuda))
    x, u, z = (problems.normal((50, w), 30 + w).float().to(cuda) for w in (32, 32, 20))
    u = u.flip(0)
    (replica,) = replicate(module, [cuda])
    params = list(module.parameters())

    def step(m):
        outs = [o for o in m.forward_flat(x, u, z) if o is not None]
        return outs + list(torch.autograd.grad(sum((o * x).sum() for o in outs), params, allow_unused=True))

    for a, b in zip(step(replica), step(module), strict=True):
        assert torch.equal(a, torch.zeros_like(a) if b is None else b)  # a copy's unused parameter: zeros
