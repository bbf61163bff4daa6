"""``residual_norm`` on B200 against its definition in float64, forward and gradients.

Tolerances.  Each result is a sum of a few products whose magnitudes (``_bounds``: the definition
with every term's absolute value) bound its error: a relative 2^-24 for each of fewer than 48
elementary steps (2 ulp for rsqrt, exp and tanh), and for a mean over d values at most
(d / 64 + 24) roundings in whatever order it is added.  Sums over T rows add at most T roundings.
On top stands the rounding to the output's type, eps / 2.
"""

import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
NAMES = ("x", "branch", "post", "pre", "gate")


def _bounds(t, act, rs, bs, eps, dy, dh):
    """Magnitudes of y, h and the gradients: each term of the definition by its absolute value (float64)."""
    x, u, post, pre, gate = (t.get(n) for n in NAMES)
    d = x.shape[-1]
    mean = lambda v: v.mean(dim=-1, keepdim=True)  # noqa: E731
    out = {}
    y, _ = ref.norm(x, u, post, gate, act, pre if u is not None else torch.ones(d).double(), rs, bs, eps)
    a = torch.ones(())
    n_abs = None
    if u is not None:
        ru = torch.rsqrt(mean(u * u) + eps)
        uh = (u * ru).abs()
        n_abs = u.abs() if post is None else uh * post.abs()
        if gate is not None:
            a = dict(none=lambda v: v, sigmoid=torch.sigmoid, tanh=torch.tanh)[act](gate).abs()
        y_abs = abs(rs) * x.abs() + abs(bs) * a * n_abs
    else:
        y_abs = x.abs()
    out["y"] = y_abs
    ry = torch.rsqrt(mean(y * y) + eps)
    # the norm's own relative error follows that of the mean square: mean(y_abs |y|) / mean(y^2)
    cond = mean(y_abs * y.abs()) * ry * ry
    yh = (y_abs + y.abs() * cond) * ry
    if pre is not None:
        out["h"] = yh * pre.abs()
    dz = dy.abs() if dy is not None else torch.zeros_like(x)
    if dh is not None:
        tt = (dh * pre).abs()
        dz = dz + ry * (1 + cond) * (tt + yh * mean(tt * yh))
        out["pre"] = (dh.abs() * yh).sum(0)
    out["x"] = dz * (abs(rs) if u is not None else 1.0)
    if u is not None:
        bz = abs(bs) * dz
        if gate is not None:
            dg = bz * n_abs
            out["gate"] = dg
            while out["gate"].ndim > gate.ndim:
                out["gate"] = out["gate"].sum(0)
            for i, s in enumerate(gate.shape):
                if s == 1 and out["gate"].shape[i] != 1:
                    out["gate"] = out["gate"].sum(i, keepdim=True)
        dn = bz * a
        if post is None:
            out["branch"] = dn
        else:
            tt = dn * post.abs()
            out["branch"] = ru * (tt + uh * mean(tt * uh))
            out["post"] = (dn * uh).sum(0)
    return out


def _case(T, d, xt, ut, post, pre, gate, seed, branch=True):
    g = torch.Generator().manual_seed(seed)

    def r(*s, std=1.0, mean=0.0):
        return torch.randn(*s, generator=g) * std + mean

    t = {"x": r(T, d).to(xt)}
    if branch:
        t["branch"] = r(T, d, std=0.5).to(ut)
        if post:
            t["post"] = r(d, std=0.2, mean=1.0)
        if gate is not None:
            t["gate"] = r(*gate, std=0.7, mean=0.2)
            if tuple(gate) == (T, d):
                t["gate"] = t["gate"].to(ut)
    if pre:
        t["pre"] = r(d, std=0.2, mean=1.0)
    return t, r(T, d).to(xt), r(T, d).to(ut)


def _check(pkg, t, dy, dh, act="none", rs=1.0, bs=1.0, eps=1e-6, train=True, view=None):
    dev = {n: v.to(DEV) for n, v in t.items()}
    if view:
        dev = {n: view(n, v) for n, v in dev.items()}
    leaves = {n: v.detach().requires_grad_(train) for n, v in dev.items()}
    kw = dict(residual_scale=rs, branch_scale=bs) if "branch" in t else {}
    y, h = pkg.residual_norm(leaves["x"], leaves.get("branch"), post_weight=leaves.get("post"),
                             gate=leaves.get("gate"), gate_activation=act, pre_weight=leaves.get("pre"), eps=eps, **kw)
    ref_leaves = {n: v.double().requires_grad_(True) for n, v in t.items()}
    ry, rh = ref.norm(ref_leaves["x"], ref_leaves.get("branch"), ref_leaves.get("post"), ref_leaves.get("gate"), act,
                      ref_leaves.get("pre"), rs, bs, eps)
    T, d = t["x"].shape
    b = _bounds({n: v.double() for n, v in t.items()}, act, rs, bs, eps, None if dy is None else dy.double(),
                None if h is None or dh is None else dh.double())
    unit = (48 + 2 * (d / 64 + 24)) * 2.0 ** -24

    def close(name, got, want, magnitude, rows=0):
        tiny = {torch.float16: 2.0 ** -25}.get(got.dtype, 2.0 ** -140)
        tol = (unit + rows * 2.0 ** -24) * magnitude + torch.finfo(got.dtype).eps / 2 * want.abs() + tiny
        err = (got.detach().cpu().double() - want).abs()
        assert (err <= tol).all(), f"{name}: error {float((err / tol).max()):.3g} times its bound"

    if "branch" in t:
        assert y.dtype == t["x"].dtype and y.is_contiguous()
        close("y", y, ry.detach(), b["y"])
    if h is not None:
        close("h", h, rh.detach(), b["h"])
    if not train:
        return y, h
    outs, grads, r_outs, r_grads = [], [], [], []
    for o, ro, go in ((y, ry, dy), (h, rh, dh)):
        if o is not None and go is not None:
            outs.append(o), grads.append(go.to(DEV)), r_outs.append(ro), r_grads.append(go.double())
    got = torch.autograd.grad(outs, list(leaves.values()), grads, allow_unused=True)
    want = torch.autograd.grad(r_outs, list(ref_leaves.values()), r_grads, allow_unused=True)
    for n, gg, wg in zip(leaves, got, want):
        if wg is None:
            wg = torch.zeros_like(ref_leaves[n])
        if gg is None:
            assert not wg.any(), n
            continue
        assert gg.dtype == t[n].dtype and gg.shape == t[n].shape
        close("d_" + n, gg, wg, b.get(n, torch.zeros(())), rows=T if n in ("pre", "post", "gate") else 0)
    return y, h


BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
SIZES = [(1, 1), (3, 7), (2, 31), (5, 64), (64, 256), (7, 1000), (33, 1001), (4, 2048), (130, 520), (3, 4096), (2, 8192),
         (2, 8200), (3, 16384)]


@pytest.mark.parametrize("T,d", SIZES)
@pytest.mark.parametrize("xt,ut", [(BF, BF), (HF, HF), (F32, F32), (F32, BF), (F32, HF), (BF, F32)])
def test_sizes_and_types(moe_pkg, T, d, xt, ut):
    t, dy, dh = _case(T, d, xt, ut, True, True, (d,), T + d)
    _check(moe_pkg, t, dy, dh, act="sigmoid", rs=0.9, bs=0.5)


@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("pre", [False, True])
@pytest.mark.parametrize("gate", [None, "channel", "token", "full"])
@pytest.mark.parametrize("act", ["none", "sigmoid", "tanh"])
@pytest.mark.parametrize("T,d", [(37, 192), (6, 45)])
def test_every_form(moe_pkg, post, pre, gate, act, T, d):
    shape = {None: None, "channel": (d,), "token": (T, 1), "full": (T, d)}[gate]
    t, dy, dh = _case(T, d, F32, F32, post, pre, shape, 5)
    _check(moe_pkg, t, dy, dh, act=act, bs=-1.25)
    t, dy, dh = _case(T, d, BF, BF, post, pre, shape, 6)
    _check(moe_pkg, t, dy, dh, act=act)


@pytest.mark.parametrize("gate", ["token", "full"])
@pytest.mark.parametrize("T,d", [(3, 8192), (5, 6000), (4, 2048), (300, 1032), (2, 1500), (2, 16384)])
@pytest.mark.parametrize("xt,ut", [(F32, F32), (F32, BF), (BF, BF)])
def test_gates_of_wide_rows(moe_pkg, gate, T, d, xt, ut):
    t, dy, dh = _case(T, d, xt, ut, True, True, (T, 1) if gate == "token" else (T, d), 31)
    _check(moe_pkg, t, dy, dh, act="sigmoid", bs=0.5)


@pytest.mark.parametrize("T,d", [(9, 64), (4, 2049)])
def test_mixed_types_outside_the_common_ones(moe_pkg, T, d):
    """A float32 gate on bf16 rows, a norm in another type than the branch."""
    t, dy, dh = _case(T, d, BF, BF, True, True, (T, d), 41)
    t["gate"] = t["gate"].float()
    _check(moe_pkg, t, dy, dh, act="tanh")
    t, dy, dh = _case(T, d, BF, BF, True, True, (d,), 42)
    dev = {n: v.to(DEV).requires_grad_(True) for n, v in t.items()}
    out = moe_pkg.residual_norm(dev["x"], dev["branch"], post_weight=dev["post"], gate=dev["gate"], pre_weight=dev["pre"])
    y, h = moe_pkg.residual_norm(dev["x"], dev["branch"], post_weight=dev["post"], gate=dev["gate"],
                                 pre_weight=dev["pre"], norm_dtype=F32)
    # two kernels add in another order: float32 values a few 2^-24 apart, which can round to neighbours in bf16
    assert h.dtype == F32
    assert ((h - out[1].float()).abs() <= (2.0 ** -8 + 2.0 ** -16) * h.abs()).all()
    assert ((y.float() - out[0].float()).abs() <= 2.0 ** -7 * out[0].float().abs()).all()
    got = torch.autograd.grad([y, h], list(dev.values()), [dy.to(DEV), dh.float().to(DEV)])
    want = torch.autograd.grad(list(out), list(dev.values()), [dy.to(DEV), dh.to(DEV)])
    for a, b in zip(got, want):  # the same sums in another order, rounded to the same type
        scale = float(b.float().abs().max())
        assert float((a.float() - b.float()).abs().max()) <= (2.0 ** -8 if b.dtype == BF else 2.0 ** -15) * scale


@pytest.mark.parametrize("dy_on,dh_on", [(True, False), (False, True)])
@pytest.mark.parametrize("d", [96, 37])
def test_one_output_used(moe_pkg, dy_on, dh_on, d):
    t, dy, dh = _case(9, d, F32, BF, True, True, (d,), 8)
    _check(moe_pkg, t, dy if dy_on else None, dh if dh_on else None)


@pytest.mark.parametrize("T,d,xt", [(5, 64, BF), (5, 65, F32), (1, 2048, BF), (40, 1024, F32)])
def test_norm_alone(moe_pkg, T, d, xt):
    t, dy, dh = _case(T, d, xt, xt, False, True, None, 4, branch=False)
    y, h = _check(moe_pkg, t, None, dh)
    x = t["x"].to(DEV)
    y, h = moe_pkg.residual_norm(x, pre_weight=t["pre"].to(DEV), norm_dtype=torch.bfloat16)
    assert y is x and h.dtype == torch.bfloat16


@pytest.mark.parametrize("shape", [(3, 40, 64), (3, 1, 64), (1, 40, 1), (3, 40, 1), (1, 1, 64), (64,), (1, 40, 64),
                                   (3, 1, 1), (1,), ()])
def test_gates_that_broadcast(moe_pkg, shape):
    g = torch.Generator().manual_seed(3)
    x, u = torch.randn(3, 40, 64, generator=g), torch.randn(3, 40, 64, generator=g)
    gate = torch.randn(shape, generator=g)
    post = torch.rand(64, generator=g) + 0.5
    dev = [v.to(DEV).requires_grad_(True) for v in (x, u, gate)]
    y, _ = moe_pkg.residual_norm(dev[0], dev[1], gate=dev[2], post_weight=post.to(DEV))
    gr = torch.autograd.grad(y, dev, torch.ones_like(y))
    leaf = [v.double().requires_grad_(True) for v in (x, u, gate)]
    ry, _ = ref.norm(leaf[0], leaf[1], post.double(), leaf[2])
    want = torch.autograd.grad(ry, leaf, torch.ones_like(ry))
    torch.testing.assert_close(y.detach().cpu().double(), ry.detach(), rtol=0, atol=2e-5)
    for a, b in zip(gr, want):
        # up to 7680 terms of a few units each: 7680 * 2^-24 * 8
        torch.testing.assert_close(a.cpu().double(), b, rtol=0, atol=4e-3 if a.numel() < 64 else 2e-4)


@pytest.mark.parametrize("groups,rows,d", [(5, 64, 96), (700, 32, 40), (3, 33, 300), (2, 40, 8200), (4, 31, 64)])
@pytest.mark.parametrize("act", ["none", "sigmoid"])
def test_one_gate_row_for_each_sequence(moe_pkg, groups, rows, d, act):
    """Column sums over groups of rows: each sequence's gate gradient, and the post norm's over all of them.
    A sum of n terms is off by at most (n + 48 + d / 32) * 2^-24 of its terms' magnitudes."""
    g = torch.Generator().manual_seed(groups)
    x, u, dy = (torch.randn(groups, rows, d, generator=g) for _ in range(3))
    gate, post = torch.randn(groups, 1, d, generator=g), torch.rand(d, generator=g) + 0.5
    dev = [v.to(DEV).requires_grad_(True) for v in (gate, post)]
    y, _ = moe_pkg.residual_norm(x.to(DEV), u.to(DEV), gate=dev[0], gate_activation=act, post_weight=dev[1], branch_scale=0.5)
    got = torch.autograd.grad(y, dev, dy.to(DEV))
    leaf = [v.double().requires_grad_(True) for v in (gate, post)]
    want_y, _ = ref.norm(x.double(), u.double(), leaf[1], leaf[0], act, None, 1.0, 0.5)
    want = torch.autograd.grad(want_y, leaf, dy.double())
    uh = u.double() * torch.rsqrt(u.double().square().mean(-1, keepdim=True) + 1e-6)
    terms = (0.5 * dy.double() * uh).abs()
    a = gate.double() if act == "none" else torch.sigmoid(gate.double())
    slope = torch.ones_like(a) if act == "none" else a * (1 - a)
    sizes = [(terms * post.double()).sum(1, keepdim=True) * slope, (terms * a.abs()).sum((0, 1))]
    for gg, wg, size, n in zip(got, want, sizes, (rows, groups * rows)):
        assert ((gg.cpu().double() - wg).abs() <= (n + 48 + d / 32) * 2.0 ** -24 * size + 1e-30).all()


def test_strides_and_offsets(moe_pkg):
    """Rows of a wider buffer, an odd first element, transposed and expanded inputs."""
    t, dy, dh = _case(20, 96, BF, BF, True, True, (20, 96), 9)

    def wide(n, v):
        if v.ndim != 2:
            return v
        buf = torch.zeros(20, 200, dtype=v.dtype, device=DEV)
        buf[:, 3:99] = v
        return buf[:, 3:99]

    a = _check(moe_pkg, t, dy, dh, view=wide)
    b = _check(moe_pkg, t, dy, dh, view=lambda n, v: v.t().contiguous().t() if v.ndim == 2 else v)
    c = _check(moe_pkg, t, dy, dh)
    for p, q, r in zip(a, b, c):
        torch.testing.assert_close(p, r, rtol=2.0 ** -7, atol=2.0 ** -7)
        assert torch.equal(q, r)
    x = t["x"][:1].to(DEV).expand(20, 96)
    y, h = moe_pkg.residual_norm(x, t["branch"][:1].to(DEV).expand(20, 96), pre_weight=t["pre"].to(DEV))
    assert torch.equal(y[0], y[19]) and torch.equal(h[0], h[19])


@pytest.mark.parametrize("rows,ld", [(40, (1 << 26) + 8), (3, (1 << 30) + 8)])
def test_rows_far_apart(moe_pkg, rows, ld):
    """Offsets that pass 32 bits, and row strides that the fast kernels do not take."""
    buf = torch.empty(rows * ld, dtype=BF, device=DEV)
    x = buf.as_strided((rows, 64), (ld, 1))
    g = torch.Generator().manual_seed(2)
    x.copy_(torch.randn(rows, 64, generator=g))
    u, w = torch.randn(rows, 64, generator=g).to(BF).to(DEV), torch.rand(64, generator=g).to(DEV)

    def run(t):
        leaf = t.detach().requires_grad_(True)
        y, h = moe_pkg.residual_norm(leaf, u, pre_weight=w, post_weight=w)
        return y.detach(), h.detach(), torch.autograd.grad([y, h], leaf, [u, u])[0]

    for a, b in zip(run(x), run(x.contiguous())):  # another kernel may add in another order: one bf16 step
        assert ((a.float() - b.float()).abs() <= 2.0 ** -6 * b.float().abs() + 2.0 ** -12).all()
    del buf, x
    torch.cuda.empty_cache()


def test_half_precision_weights_get_their_own_gradient_type(moe_pkg):
    t, dy, dh = _case(8, 64, BF, BF, True, True, None, 2)
    post, pre = t["post"].to(BF).to(DEV).requires_grad_(True), t["pre"].to(BF).to(DEV).requires_grad_(True)
    y, h = moe_pkg.residual_norm(t["x"].to(DEV), t["branch"].to(DEV), post_weight=post, pre_weight=pre)
    g = torch.autograd.grad([y, h], [post, pre], [dy.to(DEV), dh.to(DEV)])
    assert all(v.dtype == BF and torch.isfinite(v).all() for v in g)


def test_only_some_inputs_need_gradients(moe_pkg):
    t, dy, dh = _case(12, 96, BF, BF, True, True, (96,), 51)
    full = {n: v.to(DEV).requires_grad_(True) for n, v in t.items()}

    def run(leaves):
        y, h = moe_pkg.residual_norm(leaves["x"], leaves["branch"], post_weight=leaves["post"], gate=leaves["gate"],
                                     gate_activation="sigmoid", pre_weight=leaves["pre"])
        wanted = [n for n in NAMES if leaves[n].requires_grad]
        return dict(zip(wanted, torch.autograd.grad([y, h], [leaves[n] for n in wanted], [dy.to(DEV), dh.to(DEV)])))

    want = run(full)
    for n in NAMES:
        got = run({m: v.detach().requires_grad_(m == n) for m, v in full.items()})
        assert list(got) == [n] and torch.equal(got[n], want[n])
    # one tensor as stream and as branch: both gradients reach it
    both = full["x"].detach().clone().requires_grad_(True)
    y, _ = moe_pkg.residual_norm(both, both, branch_scale=2.0)
    (g,) = torch.autograd.grad(y, both, torch.ones_like(y))
    assert torch.equal(g, torch.full_like(g, 3.0))
    with pytest.raises(RuntimeError):  # differentiable once
        x = full["x"].detach().float().requires_grad_(True)
        _, h = moe_pkg.residual_norm(x, pre_weight=full["pre"].detach())
        (g,) = torch.autograd.grad(h.sum(), x, create_graph=True)
        g.sum().backward()


def test_zero_rows_zero_values_and_non_finite_rows(moe_pkg):
    w = torch.ones(64, device=DEV, requires_grad=True)
    x = torch.empty(0, 64, device=DEV, requires_grad=True)
    y, h = moe_pkg.residual_norm(x, torch.empty(0, 64, device=DEV), gate=w, pre_weight=w)
    assert y.shape == h.shape == (0, 64)
    gw, gx = torch.autograd.grad(h, [w, x], torch.empty(0, 64, device=DEV))
    assert not gw.any() and gx.shape == (0, 64)
    x = torch.zeros(3, 64, device=DEV, requires_grad=True)
    u = torch.zeros(3, 64, device=DEV, requires_grad=True)
    y, h = moe_pkg.residual_norm(x, u, post_weight=w, pre_weight=w)
    assert not y.any() and not h.any()
    gx, gu = torch.autograd.grad([y, h], [x, u], [torch.ones_like(y)] * 2)
    assert torch.isfinite(gx).all() and torch.isfinite(gu).all()
    bad = torch.randn(4, 64, device=DEV)
    bad[1, 5] = float("nan")
    bad[2, 7] = float("inf")
    y, h = moe_pkg.residual_norm(bad, torch.ones(4, 64, device=DEV), pre_weight=w)
    assert torch.isfinite(h[[0, 3]]).all() and not torch.isfinite(h[1]).any()


def test_gradient_against_differences(moe_pkg):
    """Central differences of the float64 definition in a random direction of each input."""
    t, dy, dh = _case(3, 40, F32, F32, True, True, (40,), 17)
    leaves = {n: v.to(DEV).requires_grad_(True) for n, v in t.items()}
    y, h = moe_pkg.residual_norm(leaves["x"], leaves["branch"], post_weight=leaves["post"], gate=leaves["gate"],
                                 gate_activation="tanh", pre_weight=leaves["pre"], branch_scale=0.7)
    got = torch.autograd.grad([y, h], list(leaves.values()), [dy.to(DEV), dh.to(DEV)])

    def value(v):
        a, b = ref.norm(v["x"], v["branch"], v["post"], v["gate"], "tanh", v["pre"], 1.0, 0.7)
        return float((a * dy.double()).sum() + (b * dh.double()).sum())

    g = torch.Generator().manual_seed(1)
    for n, gg in zip(leaves, got):
        way = torch.randn(t[n].shape, generator=g).double()
        way /= way.norm()
        e = 1e-5
        plus = {m: v.double() + (e * way if m == n else 0) for m, v in t.items()}
        minus = {m: v.double() - (e * way if m == n else 0) for m, v in t.items()}
        want = (value(plus) - value(minus)) / (2 * e)
        # e^2 / 6 times third derivatives of order 10, cancellation 1e-13 / 1e-5, float32 gradients of norm < 100
        assert abs(float((gg.cpu().double() * way).sum()) - want) < 1e-4


def test_runs_are_equal_and_capture_replays(moe_pkg):
    t, dy, dh = _case(700, 512, BF, BF, True, True, (512,), 23)
    leaves = {n: v.to(DEV).requires_grad_(True) for n, v in t.items()}
    dy, dh = dy.to(DEV), dh.to(DEV)

    def step():
        y, h = moe_pkg.residual_norm(leaves["x"], leaves["branch"], post_weight=leaves["post"], gate=leaves["gate"],
                                     pre_weight=leaves["pre"])
        return [y.detach(), h.detach(), *torch.autograd.grad([y, h], list(leaves.values()), [dy, dh])]

    first = step()
    assert all(torch.equal(a, b) for a, b in zip(first, step()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, on_side))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        leaves["x"].mul_(2)
    graph.replay()
    graph.replay()
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(out, want))
    with torch.no_grad():
        leaves["x"].mul_(0.5)
