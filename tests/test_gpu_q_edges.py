"""Calls at the borders of ``route_experts``, ``residual_norm``, ``adamw_step`` and their users on B200:
rows that are not finite, wrong lengths, captured and concurrent calls.  Routing is compared with its
definition in float64, with the tolerances derived in ``test_gpu_m_scores.py``."""

import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _rows(T, E, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, E, generator=g).to(dtype).to(DEV)


def _ids(pkg, logits, k, **kw):
    """ids and counts are those of the definition; returns the weights."""
    w, ids, counts = pkg.route_experts(logits, k, **kw)
    names = dict(num_groups="groups", renormalize="renorm")
    want = ref.route(logits, k, **{names.get(n, n): v for n, v in kw.items()})
    assert torch.equal(ids.cpu().long(), want[1])
    assert torch.equal(counts.cpu().long(), want[2])
    return w, want[0]


# ------------------------------------------------------------------ rows of NaN
@pytest.mark.parametrize("E", [1, 8, 64, 128, 256, 512])
@pytest.mark.parametrize("T", [3, 700])
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("with_bias", [False, True])
def test_rows_of_nan_alone(moe_pkg, E, T, score, with_bias):
    """Every lane's best key is NaN, in the first rows that a warp takes and in later ones."""
    k = min(E, 8)
    logits = _rows(T, E, E + T)
    bad = torch.zeros(T, dtype=torch.bool)
    bad[0] = bad[T // 2:T // 2 + 40] = True
    logits[bad.to(DEV)] = float("nan")
    bias = torch.linspace(-0.1, 0.1, E, device=DEV) if with_bias else None
    for renorm in (True, False):
        w, want = _ids(moe_pkg, logits, k, score=score, bias=bias, renormalize=renorm)
        assert torch.isnan(w[bad.to(DEV)]).all()
        torch.testing.assert_close(w.cpu().double()[~bad], want[~bad], rtol=2.0 ** -16, atol=0)
    w, _ = _ids(moe_pkg, torch.full((T, E), float("nan"), device=DEV), k, score=score, bias=bias)
    assert torch.isnan(w).all()


@pytest.mark.parametrize("E", [8, 64, 128, 256, 512])
@pytest.mark.parametrize("T", [3, 700])
@pytest.mark.parametrize("spoil", [float("nan"), float("inf")])
@pytest.mark.parametrize("groups", [1, 4])
def test_one_logit_spoils_every_key_of_a_softmax(moe_pkg, E, T, spoil, groups):
    """With a bias, or group sums, the keys are the softmax's: one NaN or +inf makes them all NaN."""
    logits = _rows(T, E, 3 * E + T)
    bad = torch.zeros(T, dtype=torch.bool)
    bad[0] = bad[1] = bad[T // 2] = True
    at = torch.arange(T) * 7 % E
    logits[bad.to(DEV), at[bad].to(DEV)] = spoil
    bias = torch.linspace(-0.1, 0.1, E, device=DEV)
    for kw in (dict(bias=bias), dict(bias=bias, renormalize=False)):
        w, want = _ids(moe_pkg, logits, min(E // groups, 6), num_groups=groups, top_groups=max(1, groups // 2), **kw)
        torch.testing.assert_close(w.cpu().double()[~bad], want[~bad], rtol=2.0 ** -16, atol=0)


@pytest.mark.parametrize("spoil", [float("nan"), float("inf")])
@pytest.mark.parametrize("kw", [dict(bias=True), dict(num_groups=4, top_groups=1), dict(bias=True, num_groups=4, top_groups=2)])
def test_a_spoilt_softmax_has_nan_weights(moe_pkg, spoil, kw):
    """Every score of the row is NaN, so are its weights, whichever experts the order of NaN keys picks."""
    for E in (8, 64, 256):
        logits = _rows(5, E, E)
        logits[1, E - 1] = logits[3, E // 2] = spoil
        args = dict(kw, bias=torch.linspace(-0.1, 0.1, E, device=DEV)) if "bias" in kw else kw
        for renorm in (True, False):
            w, _, _ = moe_pkg.route_experts(logits, 2, renormalize=renorm, **args)
            assert torch.isnan(w[[1, 3]]).all()
            assert torch.isfinite(w[[0, 2, 4]]).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("E", [2, 24, 64, 300])
@pytest.mark.parametrize("groups", [1, 2])
def test_a_masked_expert_stays_masked_in_a_row_of_nan(moe_pkg, score, E, groups):
    logits = _rows(6, E, E)
    logits[0] = float("nan")
    logits[2, E // 2] = float("nan")
    logits[3, 0] = float("inf")
    logits[4, E - 1] = float("-inf")
    bias = torch.linspace(-0.1, 0.1, E, device=DEV)
    bias[1::3] = float("-inf")
    for kw in (dict(), dict(renormalize=False)):
        _ids(moe_pkg, logits, min(8, E // groups), score=score, bias=bias, num_groups=groups, top_groups=1, **kw)


@pytest.mark.parametrize("kw", [dict(score_function="sigmoid", balance_bias=True), dict(balance_bias=True)])
@pytest.mark.parametrize("T", [40, 1500])
def test_a_nan_token_leaves_the_other_tokens(moe_pkg, kw, T):
    torch.manual_seed(0)
    layer = moe_pkg.SparseMoE(moe_pkg.MoEConfig(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2, **kw)).to(DEV)
    x = _rows(T, 256, 5, torch.bfloat16)
    spoilt = x.clone()
    spoilt[0] = float("nan")
    with torch.no_grad():
        a, b = layer(x)[0], layer(spoilt)[0]
    assert torch.equal(a[1:], b[1:])
    assert torch.isnan(b[0]).all()


# ------------------------------------------------------------------ wrong lengths
def _layer(pkg, **kw):
    torch.manual_seed(0)
    return pkg.SparseMoE(pkg.MoEConfig(**{**dict(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2), **kw})).to(DEV)


@pytest.mark.parametrize("kw", [dict(), dict(score_function="sigmoid"), dict(dense_subset_k=2)])
def test_a_logit_bias_of_another_length_is_refused(moe_pkg, kw):
    layer, x = _layer(moe_pkg, **kw), _rows(20, 256, 1, torch.bfloat16)
    layer.router_logit_bias = torch.zeros(7, device=DEV)
    with pytest.raises(ValueError, match="router_logit_bias"), torch.no_grad():
        layer(x)
    if "dense_subset_k" not in kw:
        with pytest.raises(ValueError, match="router_logit_bias"):
            layer(x.requires_grad_(True))
    layer.router_logit_bias = torch.zeros(8, device=DEV)
    with torch.no_grad():
        assert torch.isfinite(layer(x)[0]).all()


@pytest.mark.parametrize("kw", [dict(), dict(score_function="sigmoid"), dict(dense_subset_k=2)])
@pytest.mark.parametrize("n", [19, 21])
def test_a_mask_of_another_length_is_refused(moe_pkg, kw, n):
    layer, x = _layer(moe_pkg, **kw), _rows(20, 256, 1, torch.bfloat16)
    valid = torch.ones(n, dtype=torch.bool, device=DEV)
    with pytest.raises(ValueError, match="valid"), torch.no_grad():
        layer(x, valid)
    if "dense_subset_k" not in kw:
        with pytest.raises(ValueError, match="valid"):
            layer(x.requires_grad_(True), valid)
    x = x.detach()
    with pytest.raises(ValueError, match="valid"):
        layer.forward_dense_subset(x, [0, 3], valid=valid)
    with pytest.raises(ValueError, match="expert_weights"):
        layer.forward_dense_subset(x, [0, 3], expert_weights=torch.ones(n, 2, device=DEV))


# ------------------------------------------------------------------ the layer's scratch memory
SCORED = dict(score_function="sigmoid", balance_bias=True)


@pytest.mark.parametrize("kw", [dict(), SCORED])
def test_workspace_belongs_to_a_stream(moe_pkg, kw):
    layer, x = _layer(moe_pkg, **kw), _rows(20, 256, 1, torch.bfloat16)
    with torch.no_grad():
        layer(x)
        first = layer._ws
        layer(x)
        assert layer._ws is first
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(x)
        assert layer._ws is not first
    torch.cuda.current_stream().wait_stream(side)


@pytest.mark.parametrize("kw", [dict(), SCORED])
def test_layer_on_two_streams_at_once(moe_pkg, kw):
    layer = _layer(moe_pkg, **kw)
    xs = [_rows(3000, 256, 7 + i, torch.bfloat16) for i in range(2)]
    with torch.no_grad():
        want = [layer(x)[0].clone() for x in xs]
        streams = [torch.cuda.Stream() for _ in xs]
        torch.cuda.synchronize()
        got = [[], []]
        for _ in range(20):
            for s, x, g in zip(streams, xs, got):
                with torch.cuda.stream(s):
                    g.append(layer(x)[0])
        torch.cuda.synchronize()
    for w, g in zip(want, got):
        assert all(torch.equal(w, o) for o in g)


@pytest.mark.parametrize("kw", [dict(), SCORED])
def test_captured_layer_keeps_its_workspace(moe_pkg, kw):
    """Captured by hand; other calls of other sizes between the replays, and memory that takes what they freed."""
    layer, x = _layer(moe_pkg, **kw), _rows(500, 256, 3, torch.bfloat16)
    other = _rows(900, 256, 4, torch.bfloat16)
    static = torch.empty_like(x)
    with torch.no_grad():
        want = [t.clone() for t in layer(x)]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(static.copy_(x))
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer(static)
        captured = layer._ws
        layer(x)
        assert layer._ws is not captured
        del captured
        for _ in range(3):
            layer(other)
            taken = [torch.full((1 << 20,), 0xA5, dtype=torch.uint8, device=DEV) for _ in range(16)]
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, want))
            assert all(bool((t == 0xA5).all()) for t in taken)
            del taken


# ------------------------------------------------------------------ the optimizer
@pytest.mark.parametrize("bits", [32, 8])
def test_capturable_optimizer_resumes_from_another_device(moe_pkg, bits):
    """A checkpoint whose count has another device's name: the next steps are those of going on."""
    def make(values):
        params = [torch.nn.Parameter(v.detach().clone()) for v in values]
        return params, moe_pkg.AdamW(params, lr=1e-2, state_bits=bits, capturable=True, seed=4)

    def steps(params, opt, n, first):
        for i in range(first, first + n):
            for j, p in enumerate(params):
                p.grad = torch.full_like(p, 0.1 * (i + 1)) * torch.arange(1, p.numel() + 1, device=DEV)
            opt.step()

    params, opt = make([torch.linspace(-1, 1, n, device=DEV) for n in (300, 17)])
    steps(params, opt, 3, 0)
    saved = opt.state_dict()
    counts = saved["param_groups"][0]["step_counts"]
    assert list(counts) == ["cuda:0"] and int(counts["cuda:0"]) == 3
    saved["param_groups"][0]["step_counts"] = {"cuda:7": counts["cuda:0"].cpu()}
    again, resumed = make(params)
    resumed.load_state_dict(saved)
    steps(params, opt, 2, 3)
    steps(again, resumed, 2, 3)
    assert all(torch.equal(a, b) for a, b in zip(params, again))


def test_captures_that_could_not_replay_are_refused(moe_pkg):
    params = [torch.nn.Parameter(torch.ones(n, device=DEV)) for n in (300, 17)]
    for p in params:
        p.grad = torch.ones_like(p)
    eager, fresh = moe_pkg.AdamW(params), moe_pkg.AdamW(params, capturable=True)
    eager.step()
    torch.cuda.synchronize()
    before = [p.detach().clone() for p in params]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(RuntimeError, match="capturable"):
            eager.step()
        with pytest.raises(RuntimeError, match="eager"):
            fresh.step()
        params[0].detach().add_(1.0)
    graph.replay()
    eager.step()  # goes on eagerly, at step 2
    assert eager.state[params[0]]["step"] == 2 and not fresh.state
    assert not torch.equal(before[1], params[1])


def test_capturable_may_change_between_steps(moe_pkg):
    """The step count goes on.  The factors of a step come from powers in double on the host or on the
    device, at most one float32 rounding apart (2^-23 of an update of about lr), six times."""
    def run(kinds):
        p = torch.nn.Parameter(torch.linspace(-1, 1, 300, device=DEV))
        opt = moe_pkg.AdamW([p], lr=1e-2, capturable=kinds[0])
        for i, kind in enumerate(kinds):
            opt.param_groups[0]["capturable"] = kind
            p.grad = torch.full_like(p, 0.1 * (i + 1))
            opt.step()
        return p.detach(), opt

    want, _ = run([False] * 6)
    for kinds in ([False, False, False, True, True, True], [True, True, False, False, True, False]):
        got, opt = run(kinds)
        # the parameters round to 2^-24 of themselves with each update
        torch.testing.assert_close(got, want, rtol=6 * 2.0 ** -23, atol=6 * 1e-2 * 2.0 ** -22)
        assert ("step_counts" in opt.param_groups[0]) == kinds[-1]


# ------------------------------------------------------------------ experts that come and go
def test_scored_layer_grows_and_prunes(moe_pkg):
    """balance_bias and expert_groups change with the experts; until then the call is refused."""
    layer = _layer(moe_pkg, score_function="sigmoid", balance_bias=True, expert_groups=4, top_expert_groups=2)
    layer.update_balance_bias(torch.arange(8.0))
    x = _rows(40, 256, 2, torch.bfloat16)

    def experts(keep, new):
        added = [moe_pkg.SwiGLUExpert(256, 256).to(DEV) for _ in range(new)]
        layer.experts = torch.nn.ModuleList([layer.experts[i] for i in keep] + added)
        router = torch.nn.Linear(256, len(keep) + new, bias=False).to(DEV)
        router.weight[: len(keep)] = layer.router.weight[keep]
        layer.router = router

    def check(E):
        out, _, _, load = layer(x)
        logits = layer._router_logits(x, layer.router.weight.float().contiguous(), None)
        _, ids, _ = ref.route(logits, 2, score="sigmoid", bias=layer.balance_bias, groups=layer.expert_groups, top_groups=2)
        want = torch.zeros(40, E).scatter_(1, ids, 1.0)
        assert torch.equal(layer.last_selected_mask.cpu(), want) and torch.isfinite(out).all() and load.shape == (E,)

    with torch.no_grad():
        check(8)
        experts(list(range(8)), 2)
        with pytest.raises(ValueError, match="balance_bias"):
            layer(x)
        layer.balance_bias = torch.cat([layer.balance_bias, torch.zeros(2, device=DEV)])
        with pytest.raises(ValueError, match="expert_groups"):
            layer(x)
        layer.expert_groups = 5
        check(10)
        keep = [0, 1, 2, 4, 5, 7, 8, 9]
        experts(keep, 0)
        layer.balance_bias = layer.balance_bias[keep]
        layer.expert_groups = 4
        check(8)
    assert layer.state_dict()["balance_bias"].shape == (8,)


# ------------------------------------------------------------------ gates that broadcast
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("rows,shape", [((3, 40), shape) for shape in (
    (3, 1, 64), (1, 40, 64), (1, 40, 1), (3, 1, 1), (1, 1, 64), (64,), (1,), (3, 40, 1), (3, 40, 64))] + [
    ((12, 10), (12, 1, 64)), ((60, 2), (60, 1, 64)), ((60, 2), (60, 1, 1))])
@pytest.mark.parametrize("branch", [torch.float32, None])
def test_gradient_of_a_16_bit_gate_is_rounded_once(moe_pkg, dtype, rows, shape, branch):
    """d gate = sum of dy act'(g) n over what the gate stands for.  Its terms cancel to a small rest, which
    the rounding of single terms (2^-8 or 2^-11 of each) would bury; a sum of n float32 terms is off by
    at most (n + 64) 2^-24 of their magnitudes, the result by half a step of its type."""
    g = torch.Generator().manual_seed(5)
    (B, S), d = rows, 64
    kind = branch or dtype
    x, u = torch.randn(B, S, d, generator=g).to(kind), (torch.rand(B, S, d, generator=g) + 0.5).to(kind)
    dy = torch.randn(B, S, d, generator=g).sign() * (torch.rand(B, S, d, generator=g) + 0.5)
    dy = (dy - (dy * u.float()).mean() / (u.float() ** 2).mean() * u.float()).to(kind)
    gate = torch.randn(shape, generator=g).to(dtype)
    leaf = gate.to(DEV).requires_grad_(True)
    y, _ = moe_pkg.residual_norm(x.to(DEV), u.to(DEV), gate=leaf, gate_activation="sigmoid")
    (got,) = torch.autograd.grad(y, leaf, dy.to(DEV))
    assert got.dtype == dtype and got.shape == gate.shape
    want_leaf = gate.double().requires_grad_(True)
    want_y, _ = ref.norm(x.double(), u.double(), None, want_leaf, "sigmoid")
    (want,) = torch.autograd.grad(want_y, want_leaf, dy.double())
    s = torch.sigmoid(gate.double())
    terms = (dy.double() * u.double() * s * (1 - s)).abs()
    while terms.ndim > gate.ndim:
        terms = terms.sum(0)
    for i, size in enumerate(gate.shape):
        terms = terms.sum(i, keepdim=True) if size == 1 else terms
    n = B * S * d // max(1, gate.numel())
    tol = (n + 64) * 2.0 ** -24 * terms + torch.finfo(dtype).eps / 2 * want.abs() + 2.0 ** -25
    assert ((got.cpu().double() - want).abs() <= tol).all(), float(((got.cpu().double() - want).abs() / tol).max())


# ------------------------------------------------------------------ no tokens
@pytest.mark.parametrize("kw", [dict(), SCORED, dict(SCORED, expert_groups=4, top_expert_groups=2)])
@pytest.mark.parametrize("block", [False, True])
def test_training_step_without_tokens(moe_pkg, kw, block):
    torch.manual_seed(0)
    cfg = moe_pkg.MoEConfig(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2, **kw)
    layer = (moe_pkg.SparseMoEBlock if block else moe_pkg.SparseMoE)(cfg).to(DEV)
    x = torch.empty(2, 0, 256, dtype=torch.bfloat16, device=DEV).requires_grad_(True)
    out, aux, z, load = layer(x)
    assert out.shape == x.shape and float(aux.detach()) == float(z.detach()) == 0.0 and not load.any()
    (out.float().sum() + aux + z).backward()
    assert x.grad.shape == x.shape
    for n, p in layer.named_parameters():
        assert p.grad is not None and not p.grad.any(), n
    with torch.no_grad():
        assert layer(x)[0].shape == x.shape


# ------------------------------------------------------------------ the weights' NVFP4 copies
@pytest.mark.parametrize("kw", [dict(), SCORED])
def test_invalidated_cache_is_made_again(moe_pkg, kw):
    """Weights that change without their version (a replayed optimizer step, ``.data``)."""
    layer, x = _layer(moe_pkg, **kw), _rows(40, 256, 3, torch.bfloat16)
    with torch.no_grad():
        layer(x)
        for p in layer.experts.parameters():
            p.data.mul_(-1.5)
        moe_pkg.nvfp4.invalidate_cache(layer.experts)
        fresh = _layer(moe_pkg, **kw)
        fresh.load_state_dict(layer.state_dict())
        assert torch.equal(layer(x)[0], fresh(x)[0])


# ------------------------------------------------------------------ captured calls and those copies
def _side(fn):
    """Runs ``fn`` on a side stream, as before a capture."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        result = fn()
    torch.cuda.current_stream().wait_stream(side)
    return result


@pytest.mark.parametrize("kw", [dict(), SCORED])
def test_capture_after_the_weights_changed(moe_pkg, kw):
    """What a capture records has not run: an eager call behind it must not take its quantisation for done."""
    layer, x = _layer(moe_pkg, **kw), _rows(60, 256, 3, torch.bfloat16)
    static = x.clone()
    with torch.no_grad():
        old = layer(x)[0].clone()
        _side(lambda: layer(static))
        for p in layer.experts.parameters():
            p.mul_(-1.5)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = layer(static)[0]
        eager = layer(x)[0].clone()
        graph.replay()
        fresh = _layer(moe_pkg, **kw)
        fresh.load_state_dict(layer.state_dict())
        want = fresh(x)[0]
        assert torch.equal(eager, want) and torch.equal(captured, want) and not torch.equal(want, old)
        for p in layer.experts.parameters():  # once more, behind the capture
            p.mul_(2.0)
        fresh.load_state_dict(layer.state_dict())
        assert torch.equal(layer(x)[0], fresh(x)[0])


@pytest.mark.parametrize("kw", [dict(), SCORED])
@pytest.mark.parametrize("fresh_cache", [False, True])
def test_captured_training_step(moe_pkg, kw, fresh_cache):
    """Forward, gradients and optimizer step in one graph, replayed: the weights are those of eager steps
    (the same seeds of the stochastic rounding)."""
    import random

    x = _rows(200, 256, 6, torch.bfloat16)

    def make():
        layer = _layer(moe_pkg, **kw)
        return layer, list(layer.parameters()), moe_pkg.AdamW(layer.parameters(), lr=1e-2, capturable=True)

    def step(layer, params, opt, inp):
        random.seed(11)
        out, aux, z, _ = layer(inp)
        ones = [torch.ones_like(t) for t in (out, aux, z)]
        for p, g in zip(params, torch.autograd.grad([out, aux, z], params, ones)):
            p.grad = g
        opt.step()

    one, two = make(), make()
    for _ in range(5):
        step(*one, x)
    static = x.clone()
    _side(lambda: [step(*two, static) for _ in range(2)])
    if fresh_cache:  # an eager forward between the last step and the capture
        two[0](static)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(*two, static)
    for _ in range(3):
        two[0](_rows(333, 256, 9, torch.bfloat16))  # other calls between the replays
        graph.replay()
    for (n, p), q in zip(one[0].named_parameters(), two[1]):
        assert torch.equal(p, q), n
    moe_pkg.nvfp4.invalidate_cache(two[0].experts)
    with torch.no_grad():
        assert torch.equal(one[0](x)[0], two[0](x)[0])


@pytest.mark.parametrize("kw", [dict(), SCORED])
def test_first_calls_on_two_streams(moe_pkg, kw):
    """One call quantises the weights, the other takes what it wrote without a word from the user."""
    torch.manual_seed(0)
    cfg = moe_pkg.MoEConfig(d_model=2048, expert_hidden_dim=1024, num_experts=16, top_k=2, **kw)
    layer = moe_pkg.SparseMoE(cfg).to(DEV)
    x = _rows(64, 2048, 3, torch.bfloat16)
    streams = [torch.cuda.Stream() for _ in range(3)]
    with torch.no_grad():
        for scale in (1.0, -0.5, 2.0):
            for p in layer.experts.parameters():
                p.mul_(scale)
            moe_pkg.nvfp4.invalidate_cache(layer.experts)
            torch.cuda.synchronize()
            got = []
            for s in streams:
                with torch.cuda.stream(s):
                    got.append(layer(x)[0])
            torch.cuda.synchronize()
            want = layer(x)[0]
            assert all(torch.equal(want, g) for g in got)


def test_a_layer_with_its_cache_can_be_copied(moe_pkg):
    import copy

    layer, x = _layer(moe_pkg, **SCORED), _rows(64, 256, 3, torch.bfloat16)
    with torch.no_grad():
        want = layer(x)[0]
        other = copy.deepcopy(layer)
        assert torch.equal(other(x)[0], want)
        for p in other.experts.parameters():
            p.mul_(2.0)
        assert not torch.equal(other(x)[0], want) and torch.equal(layer(x)[0], want)


def test_broadcast_16_bit_gates_of_nothing_and_of_mixed_types(moe_pkg):
    """No rows; a bf16 gate on an fp16 stream and a float32 branch (the kernels of mixed types)."""
    for rows, shape in (((0, 5), (1, 5, 32)), ((3, 0), (3, 1, 32)), ((0, 5), (1, 1, 1))):
        x = torch.empty(*rows, 32, device=DEV, dtype=torch.bfloat16)
        gate = torch.ones(shape, device=DEV, dtype=torch.bfloat16).requires_grad_(True)
        y, _ = moe_pkg.residual_norm(x, x.clone(), gate=gate)
        (g,) = torch.autograd.grad(y, gate, torch.empty_like(y))
        assert g.shape == gate.shape and not g.any()
    gen = torch.Generator().manual_seed(2)
    x, u, dy = (torch.randn(4, 6, 40, generator=gen) for _ in range(3))
    gate = torch.randn(1, 6, 40, generator=gen).to(torch.bfloat16)
    leaf = gate.to(DEV).requires_grad_(True)
    y, _ = moe_pkg.residual_norm(x.half().to(DEV), u.to(DEV), gate=leaf)
    (got,) = torch.autograd.grad(y, leaf, dy.half().to(DEV))
    terms = dy.half().double() * u.double()
    want = terms.sum(0, keepdim=True)
    # four terms of a few float32 roundings, and half a step of bf16: eps / 2 = 2^-8 of the value
    tol = 68 * 2.0 ** -24 * terms.abs().sum(0, keepdim=True) + torch.finfo(torch.bfloat16).eps / 2 * want.abs()
    assert got.dtype == torch.bfloat16 and ((got.cpu().double() - want).abs() <= tol).all()
