"""``route_experts`` on B200 against its definition in float64.

Tolerances.  A weight is a quotient of at most 32 added ratios: exp within 2 ulp of a difference
of logits that is rounded to half an ulp (at most 64 here: 2^-24 * 64 = 2^-18 relative), and a
handful of products and sums of 2^-24 each; the same for the numerator.  That is below 2^-16.
A gradient is r (d - c) (1 - s) with |c| <= max|d|: the same relative error on terms of at most
2 |r| max|d|.
"""

import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
REL = 2.0 ** -16


def _logits(T, E, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(T, E, generator=g) * spread).to(dtype).to(DEV)


def _check(pkg, logits, k, d_w=None, **kw):
    names = dict(num_groups="groups", renormalize="renorm")
    args = {names.get(n, n): v for n, v in kw.items()}
    if "groups" in args and "top_groups" not in args:
        args["top_groups"] = args["groups"]
    leaf = logits.detach().requires_grad_(d_w is not None)
    w, ids, counts = pkg.route_experts(leaf, k, **kw)
    want = ref.route(logits, k, d_w=d_w, **args)
    assert w.dtype == torch.float32 and ids.dtype == torch.int32 and counts.dtype == torch.int32
    assert torch.equal(ids.cpu().long(), want[1])
    assert torch.equal(counts.cpu().long(), want[2])
    torch.testing.assert_close(w.detach().cpu().double(), want[0], rtol=REL, atol=2.0 ** -140, equal_nan=True)
    if d_w is not None:
        (g,) = torch.autograd.grad(w, leaf, d_w)
        assert g.dtype == logits.dtype and g.shape == logits.shape
        scale = abs(kw.get("scale", 1.0))
        bound = 2 * REL * scale * float(d_w.abs().max()) + 1e-30
        err = (g.cpu().double() - want[3]).abs()
        # terms of at most 2 scale max|d|, and the rounding to the logits' type
        assert (err <= bound + torch.finfo(logits.dtype).eps / 2 * want[3].abs()
                + (2.0 ** -25 if logits.dtype == torch.float16 else 0.0)).all(), float(err.max())
    return w, ids, counts


SHAPES = [(1, 1, 1), (1, 2, 2), (5, 7, 3), (64, 64, 8), (33, 40, 8), (17, 96, 6), (130, 128, 4), (9, 255, 32),
          (21, 256, 8), (6, 300, 11), (4, 512, 32)]


@pytest.mark.parametrize("T,E,k", SHAPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("with_bias", [False, True])
def test_against_the_definition(moe_pkg, T, E, k, score, renorm, with_bias):
    logits = _logits(T, E, torch.float32, T + E)
    g = torch.Generator().manual_seed(9)
    bias = (torch.randn(E, generator=g) * 0.05).to(DEV) if with_bias else None
    d_w = torch.randn(T, k, generator=g).to(DEV)
    _check(moe_pkg, logits, k, d_w, score=score, renormalize=renorm, bias=bias, scale=2.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups,group_score", [(1, 1, "top2"), (8, 3, "top2"), (8, 3, "max")])
def test_half_types_with_many_ties(moe_pkg, dtype, score, groups, top_groups, group_score):
    """bf16 logits on a coarse grid: the ids of equal keys have to come lowest first."""
    logits = (_logits(40, 64, torch.float32, 3) * 4).round().div(4).to(dtype)
    d_w = _logits(40, 6, torch.float32, 4)
    _check(moe_pkg, logits, 6, d_w, score=score, num_groups=groups, top_groups=top_groups, group_score=group_score)
    _check(moe_pkg, logits, 6, d_w, score=score, num_groups=groups, top_groups=top_groups, group_score=group_score,
           bias=torch.zeros(64, device=DEV), renormalize=False)


@pytest.mark.parametrize("E,groups,top_groups,k", [(8, 4, 2, 4), (64, 8, 4, 8), (64, 64, 9, 9), (256, 8, 4, 8),
                                                   (72, 8, 6, 16), (160, 5, 3, 6), (21, 7, 2, 5), (510, 255, 20, 32),
                                                   (512, 2, 1, 32), (12, 12, 12, 3)])
@pytest.mark.parametrize("group_score", ["top2", "max"])
@pytest.mark.parametrize("score,with_bias", [("sigmoid", True), ("sigmoid", False), ("softmax", True),
                                             ("softmax", False)])
def test_groups(moe_pkg, E, groups, top_groups, k, group_score, score, with_bias):
    logits = _logits(19, E, torch.float32, E + groups)
    g = torch.Generator().manual_seed(2)
    bias = (torch.randn(E, generator=g) * 0.1).to(DEV) if with_bias else None
    _check(moe_pkg, logits, k, _logits(19, k, torch.float32, 5), score=score, bias=bias, num_groups=groups,
           top_groups=top_groups, group_score=group_score, scale=2.5)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("groups,top_groups", [(1, 1), (4, 2)])
def test_keys_closer_than_float32_tells_apart(moe_pkg, score, groups, top_groups):
    """Keys s + b of neighbours that differ by less than a float32 step of the key: the order is
    that of exact arithmetic."""
    g = torch.Generator().manual_seed(7)
    T, E, k = 50, 32, 6
    logits = (torch.randn(T, E, generator=g) * 0.5).float()
    s = torch.sigmoid(logits.double()) if score == "sigmoid" else torch.softmax(logits.double(), 1)
    # one row fixes a bias that lifts every key to within a few float32 steps of 1
    bias = (1.0 - s[0]).float()
    logits = logits[:1].repeat(T, 1)
    logits = torch.nextafter(logits, logits + torch.randint(-1, 2, (T, E), generator=g))
    _check(moe_pkg, logits.to(DEV), k, None, score=score, bias=bias.to(DEV), num_groups=groups, top_groups=top_groups)


def test_large_logits_saturate_or_underflow(moe_pkg):
    logits = torch.tensor([[-200.0, -201.0, -300.0, -199.5], [60.0, 61.0, 59.0, 100.0], [30.0, -30.0, 0.0, 90.0],
                           [-80.0, -90.0, -85.0, -100.0]], device=DEV)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            w, _, _ = _check(moe_pkg, logits, 3, None, score=score, renormalize=renorm)
            assert torch.isfinite(w).all()
    w, _, _ = moe_pkg.route_experts(logits, 3, score="sigmoid")
    assert torch.allclose(w.sum(1), torch.ones(4, device=DEV))
    _check(moe_pkg, logits, 2, None, score="sigmoid", bias=torch.tensor([0.0, 1e-3, 0.0, -1e-3], device=DEV))


def test_masked_experts_and_rows(moe_pkg):
    logits = _logits(9, 24, torch.float32, 11)
    logits[0, :] = float("-inf")          # nothing left
    logits[1, 5:] = float("-inf")         # fewer than k
    logits[2, ::2] = float("-inf")
    logits[3, :] = float("nan")           # behind the padding mask
    logits[4, :] = float("inf")
    logits[5, :12] = float("-inf")        # two whole groups
    logits[6, 1:6] = float("-inf")        # one expert left in its group
    valid = torch.tensor([1, 1, 1, 0, 0, 1, 1, 1, 0], dtype=torch.bool, device=DEV)
    d_w = _logits(9, 8, torch.float32, 12)
    bias = torch.linspace(-0.1, 0.1, 24, device=DEV)
    bias[23] = float("-inf")
    for kw in (dict(), dict(bias=bias), dict(num_groups=4, top_groups=2), dict(num_groups=4, top_groups=2, bias=bias),
               dict(num_groups=4, top_groups=2, group_score="max", bias=bias)):
        for score in ("softmax", "sigmoid"):
            for renorm in (True, False):
                w, ids, _ = _check(moe_pkg, logits, 8, d_w, score=score, renormalize=renorm, valid=valid, **kw)
                assert (ids[0] == -1).all() and (w[0] == 0).all()
                assert (ids[3] == -1).all() and (w[3] == 0).all()
                assert (ids[1] >= 0).sum() <= 5


def test_nan_ranks_first_and_spoils_its_row_only(moe_pkg):
    logits = _logits(4, 16, torch.float32, 13)
    logits[1, 6] = float("nan")
    logits[2, 3] = float("inf")
    for score in ("softmax", "sigmoid"):
        w, ids, _ = moe_pkg.route_experts(logits, 4, score=score)
        assert ids[1, 0] == 6 and torch.isnan(w[1]).all()
        assert ids[2, 0] == 3
        assert torch.isfinite(w[[0, 3]]).all()
        assert torch.isnan(w[2]).any() == (score == "softmax")


def test_empty_and_strided_and_batched(moe_pkg):
    w, ids, counts = moe_pkg.route_experts(torch.empty(0, 8, device=DEV), 2)
    assert w.shape == (0, 2) and counts.sum() == 0
    wide = _logits(12, 80, torch.float32, 14)
    a = moe_pkg.route_experts(wide[:, 3:43], 5, score="sigmoid")
    b = moe_pkg.route_experts(wide[:, 3:43].contiguous(), 5, score="sigmoid")
    assert all(torch.equal(x, y) for x, y in zip(a, b))
    c = moe_pkg.route_experts(wide[:, 3:43].t().contiguous().t(), 5, score="sigmoid")
    assert all(torch.equal(x, y) for x, y in zip(c, b))
    d = moe_pkg.route_experts(wide[:1].expand(12, 80), 5)
    assert torch.equal(d[1][0], d[1][11])
    w3, i3, _ = moe_pkg.route_experts(wide.view(3, 4, 80), 5, valid=torch.ones(3, 4, device=DEV))
    assert w3.shape == (3, 4, 5) and torch.equal(i3.view(12, 5), moe_pkg.route_experts(wide, 5)[1])
    one = moe_pkg.route_experts(wide[0], 5)
    assert one[0].shape == (5,) and torch.equal(one[1], i3[0, 0])


def test_gradient_against_differences(moe_pkg):
    """Central differences of the float64 definition at points where no choice changes within the step."""
    T, E, k = 3, 12, 4
    logits = (torch.arange(T * E).remainder(7) * 0.3 + torch.linspace(0, 0.2, T * E)).view(T, E).to(DEV)
    d_w = _logits(T, k, torch.float32, 21)
    for score in ("softmax", "sigmoid"):
        for renorm in (True, False):
            leaf = logits.clone().requires_grad_(True)
            w, ids, _ = moe_pkg.route_experts(leaf, k, score=score, renormalize=renorm, scale=1.5)
            (g,) = torch.autograd.grad(w, leaf, d_w)
            h = 1e-4
            for t, e in ((0, 0), (1, int(ids[1, 0])), (2, int(ids[2, k - 1])), (0, E - 1)):
                step = torch.zeros(T, E, dtype=torch.float64)
                step[t, e] = h
                up, ui, _ = ref.route(logits.cpu().double() + step, k, score=score, renorm=renorm, scale=1.5)
                dn, di, _ = ref.route(logits.cpu().double() - step, k, score=score, renorm=renorm, scale=1.5)
                assert torch.equal(ui, di)
                want = float(((up - dn) / (2 * h) * d_w.cpu().double()).sum())
                # third derivative terms h^2/6 * O(1) and the kernel's own error
                assert abs(float(g[t, e]) - want) <= 1e-6 + 1e-4 * abs(want)


def test_runs_are_equal_and_capture_replays(moe_pkg):
    logits = _logits(5000, 64, torch.float32, 30)
    bias = torch.zeros(64, device=DEV)
    kw = dict(score="sigmoid", bias=bias, num_groups=8, top_groups=4)
    first = moe_pkg.route_experts(logits, 8, **kw)
    again = moe_pkg.route_experts(logits, 8, **kw)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    static = logits.clone().requires_grad_(True)
    d_w = _logits(5000, 8, torch.float32, 31)

    def step():
        w, ids, counts = moe_pkg.route_experts(static, 8, **kw)
        return w.detach(), ids, counts, torch.autograd.grad(w, static, d_w)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    other = _logits(5000, 64, torch.float32, 32)
    with torch.no_grad():
        static.copy_(other)
    graph.replay()
    graph.replay()
    want = moe_pkg.route_experts(other, 8, **kw)
    assert all(torch.equal(a, b) for a, b in zip(out[:3], want))
    leaf = other.clone().requires_grad_(True)
    assert torch.equal(out[3], torch.autograd.grad(moe_pkg.route_experts(leaf, 8, **kw)[0], leaf, d_w)[0])


def test_large_batches_and_two_streams(moe_pkg):
    """More rows than the CTAs that are resident, on two streams at once; strided, odd and masked rows
    are compared with the definition row by row on a sample."""
    wide = _logits(70001, 67, torch.bfloat16, 40)
    logits = wide[:, 1:62]
    valid = torch.rand(70001, generator=torch.Generator().manual_seed(3)).to(DEV) < 0.9
    bias = (torch.arange(61, device=DEV) % 7) * 1e-3
    kw = dict(score="sigmoid", bias=bias, valid=valid)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    outs = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            outs.append(moe_pkg.route_experts(logits, 6, **kw))
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for a, b in zip(*outs):
        assert torch.equal(a, b)
    w, ids, counts = outs[0]
    assert int(counts.sum()) == 6 * int(valid.sum())
    assert torch.equal(torch.bincount(ids[ids >= 0].reshape(-1).long(), minlength=61), counts.long())
    pick = torch.arange(0, 70001, 701)
    want = ref.route(logits[pick], 6, score="sigmoid", bias=bias, valid=valid[pick])
    assert torch.equal(ids[pick].cpu().long(), want[1])
    torch.testing.assert_close(w[pick].cpu().double(), want[0], rtol=REL, atol=0)


def test_rows_far_apart(moe_pkg):
    """Offsets that pass 32 bits."""
    ld = (1 << 27) + 3
    buf = torch.empty(20 * ld, dtype=torch.bfloat16, device=DEV)
    far = buf.as_strided((20, 40), (ld, 1))
    far.copy_(_logits(20, 40, torch.float32, 50))
    near = far.contiguous()
    d_w = _logits(20, 5, torch.float32, 51)
    results = []
    for t in (far, near):
        leaf = t.detach().requires_grad_(True)
        w, ids, counts = moe_pkg.route_experts(leaf, 5, renormalize=False)
        results.append((w.detach(), ids, counts, torch.autograd.grad(w, leaf, d_w)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*results))
    del buf, far
    torch.cuda.empty_cache()


def test_second_differentiation_is_refused(moe_pkg):
    logits = _logits(4, 16, torch.float32, 1).requires_grad_(True)
    w, _, _ = moe_pkg.route_experts(logits, 4)
    (g,) = torch.autograd.grad(w.square().sum(), logits, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_refusals_on_the_device(moe_pkg):
    logits = _logits(4, 16, torch.float32, 1)
    with pytest.raises(ValueError):
        moe_pkg.route_experts(logits, 4, bias=torch.zeros(16))  # another device
    with pytest.raises(ValueError):
        moe_pkg.route_experts(logits, 4, valid=torch.ones(4))
    with pytest.raises(ValueError):
        moe_pkg.route_experts(logits.double(), 4)
