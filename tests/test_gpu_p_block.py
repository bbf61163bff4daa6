"""The layer routed from scores, ``SparseMoEBlock`` and ``AdamW`` together, on B200.

* With zero balance bias and softmax scores the scored path computes the plain layer: same
  experts, same output.  The two round the routing weights apart by a few float32 steps, which
  the bf16 products see as at most one bf16 step of a term: 2^-8 of the k terms' magnitudes, at
  most of their largest sum, hence rtol 2^-6 with the largest output as scale.
* Sigmoid and group routing against the definition on the library's own router logits, the
  output against the experts run one by one (bf16 rounding of each term and of the sum).
* The training forward and backward, the optimizer's step and the next forward in a row.
"""

import random

import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _cfg(pkg, **kw):
    base = dict(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2)
    base.update(kw)
    return pkg.MoEConfig(**base)


def _layer(pkg, seed=0, cls="SparseMoE", **kw):
    torch.manual_seed(seed)
    return getattr(pkg, cls)(_cfg(pkg, **kw)).to(DEV)


def _x(T=96, d=256, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(T, d, generator=g).to(torch.bfloat16).to(DEV)


def _close(a, b, rel):
    scale = float(b.float().abs().max())
    assert float((a.float() - b.float()).abs().max()) <= rel * scale + 1e-30, (float((a.float() - b.float()).abs().max()), scale)


@pytest.mark.parametrize("masked", [False, True])
def test_scored_softmax_is_the_plain_layer(moe_pkg, masked):
    plain, scored = _layer(moe_pkg), _layer(moe_pkg, balance_bias=True)
    scored.load_state_dict(plain.state_dict(), strict=False)
    x = _x()
    valid = torch.arange(96, device=DEV) % 5 != 0 if masked else None
    with torch.no_grad():
        a, b = plain(x, valid), scored(x, valid)
    assert torch.equal(plain.last_selected_mask, scored.last_selected_mask)
    _close(b[0], a[0], 2.0 ** -6)
    for p, q in zip(a[1:], b[1:]):
        torch.testing.assert_close(p, q, rtol=1e-5, atol=1e-6)
    grads = []
    for layer in (plain, scored):
        random.seed(5)  # the stochastic rounding of the gradients
        xg = x.clone().requires_grad_(True)
        out, aux, z, _ = layer(xg, valid)
        torch.autograd.backward([out, aux, z], [torch.ones_like(out), torch.tensor(0.5, device=DEV), torch.tensor(0.1, device=DEV)])
        grads.append([xg.grad, layer.router.weight.grad] + [p.grad for p in layer.experts.parameters()])
        layer.zero_grad(set_to_none=True)
    for p, q in zip(*grads):
        # the same NVFP4 codes but for values next to a border of their rounding
        assert float((p.float() - q.float()).norm()) <= 0.05 * float(p.float().norm())


@pytest.mark.parametrize("kw", [dict(score_function="sigmoid", balance_bias=True, routed_scale=2.5),
                                dict(score_function="sigmoid", expert_groups=4, top_expert_groups=2),
                                dict(expert_groups=4, top_expert_groups=2, group_score="max", norm_topk_prob=False)])
def test_scored_routing_and_output(moe_pkg, kw):
    layer = _layer(moe_pkg, **kw)
    x = _x()
    valid = torch.arange(96, device=DEV) % 7 != 3
    if layer.balance_bias is not None:
        layer.balance_bias.copy_(torch.linspace(-0.2, 0.2, 8))
    with torch.no_grad():
        out, aux, z, load = layer(x, valid)
        logits = layer._router_logits(x, layer.router.weight.float().contiguous(), None)
        each = torch.stack([layer.forward_dense_subset(x, [e]) for e in range(8)]).float()
    w, ids, counts = ref.route(logits, 2, score=layer.score_function, bias=layer.balance_bias,
                               groups=layer.expert_groups, top_groups=layer.top_expert_groups or layer.expert_groups,
                               group_score=layer.group_score, renorm=layer.norm_topk_prob, scale=layer.routed_scale,
                               valid=valid)
    want_mask = torch.zeros(96, 9).scatter_(1, ids % 9, 1.0)[:, :8]
    assert torch.equal(layer.last_selected_mask.cpu(), want_mask)
    torch.testing.assert_close(load.cpu().double(), counts.double() / counts.sum(), rtol=1e-6, atol=0)
    w = w.float().to(DEV)
    pick = ids.clamp(min=0).to(DEV)
    terms = torch.stack([each[pick[:, j], torch.arange(96, device=DEV)] * w[:, j:j + 1] for j in range(2)])
    # a term: bf16 of the row, of the weight, of the product; the sum: bf16 again
    bound = 4 * 2.0 ** -8 * terms.abs().sum(0) + 2.0 ** -8 * terms.sum(0).abs() + 1e-6
    assert ((out.float() - terms.sum(0)).abs() <= bound).all()
    assert not out[~valid].any()
    l = logits[valid].double()
    s = torch.sigmoid(l) if layer.score_function == "sigmoid" else torch.softmax(l, -1)
    want = 8 * ((counts.double() / counts.sum()).to(DEV) * (s / s.sum(-1, keepdim=True)).mean(0)).sum()
    torch.testing.assert_close(aux.double(), want, rtol=1e-5, atol=0)
    torch.testing.assert_close(z.double(), torch.logsumexp(l, -1).square().mean(), rtol=1e-5, atol=0)


def test_masked_rows_may_hold_anything(moe_pkg):
    layer = _layer(moe_pkg, score_function="sigmoid", balance_bias=True)
    x = _x(40)
    valid = torch.arange(40, device=DEV) < 30
    bad = x.clone()
    bad[30:] = float("nan")
    results = []
    for v in (x, bad):
        random.seed(3)
        leaf = v.clone().requires_grad_(True)
        out, aux, z, _ = layer(leaf, valid)
        (out.float().sum() + aux + z).backward()
        results.append([out.detach(), aux.detach(), z.detach(), leaf.grad] + [p.grad.clone() for p in layer.parameters()])
        layer.zero_grad(set_to_none=True)
    for p, q in zip(*results):
        assert torch.isfinite(p).all() and torch.equal(p, q)
    out, aux, z, load = layer(x, torch.zeros(40, dtype=torch.bool, device=DEV))
    assert not out.any() and float(aux.detach()) == float(z.detach()) == 0.0 and not load.any()
    empty = layer(x[:0])
    assert empty[0].shape == (0, 256)


def test_balance_bias_moves_against_the_load_and_travels(moe_pkg):
    layer = _layer(moe_pkg, score_function="sigmoid", balance_bias=True)
    assert "balance_bias" in layer.state_dict()
    load = torch.tensor([0.5, 0.1, 0.1, 0.1, 0.1, 0.1, 0.0, 0.0], device=DEV)
    layer.update_balance_bias(load, rate=0.01)
    want = torch.tensor([-1, 1, 1, 1, 1, 1, 1, 1], device=DEV) * 0.01
    torch.testing.assert_close(layer.balance_bias, want)
    other = _layer(moe_pkg, seed=4, score_function="sigmoid", balance_bias=True)
    other.load_state_dict(layer.state_dict())
    x = _x(20)
    with torch.no_grad():
        assert torch.equal(layer(x)[0], other(x)[0])


def test_what_does_not_combine_is_refused(moe_pkg):
    layer = _layer(moe_pkg, score_function="sigmoid")
    with pytest.raises(NotImplementedError), torch.no_grad():
        layer(_x(), dense_subset_k=2)
    layer.mitotic_pairs = [(0, 1)]
    with pytest.raises(NotImplementedError), torch.no_grad():
        layer(_x())
    layer.mitotic_pairs = []
    with pytest.raises(NotImplementedError):
        layer.forward_details(_x())
    with pytest.raises(NotImplementedError, match="scores"):
        moe_pkg.ExpertParallelMoE.from_dense(layer)


@pytest.mark.parametrize("kw", [dict(), dict(post_norm=True, residual_gate="tanh", branch_scale=0.5),
                                dict(post_norm=True, residual_gate="linear", score_function="sigmoid", expert_groups=4,
                                     top_expert_groups=2, balance_bias=True)])
@pytest.mark.parametrize("stream", [torch.bfloat16, torch.float32])
def test_block_is_its_parts(moe_pkg, kw, stream):
    block = _layer(moe_pkg, cls="SparseMoEBlock", **kw)
    with torch.no_grad():
        for p in (block.moe_norm, block.post_norm, block.gate):
            if p is not None:
                p.add_(torch.randn(256, device=DEV) * 0.1)
    x = _x(48).to(stream).view(2, 24, 256)
    after = torch.rand(256, device=DEV) + 0.5
    with torch.no_grad():
        (y, h), aux, z, load = block(x, next_norm=after)
        _, normed = ref.norm(x.double(), pre=block.moe_norm.double())
        out = block.moe(normed.to(torch.bfloat16))[0]
    assert y.dtype == stream and y.shape == x.shape and h.dtype == torch.bfloat16
    act = dict(none="none", linear="none").get(block.residual_gate, block.residual_gate)
    want, want_h = ref.norm(x.double(), out.double(), None if block.post_norm is None else block.post_norm.double(),
                            None if block.gate is None else block.gate.double(), act, after.double(), 1.0,
                            block.branch_scale, block.eps)
    # the inner norm rounds to bf16 either way of a border now and then: the experts see one step of one input
    _close(y, want, 2.0 ** -5)
    _close(h, want_h, 2.0 ** -5)


def test_training_steps_in_a_row(moe_pkg):
    """Forward, backward, optimizer and the next forward, as a training loop has them: every
    parameter gets its gradient and moves, and the layer computes with the moved weights."""
    kw = dict(score_function="sigmoid", balance_bias=True, post_norm=True, residual_gate="sigmoid")
    for bits in (32, 8):
        block = _layer(moe_pkg, cls="SparseMoEBlock", **kw)
        opt = moe_pkg.AdamW(block.parameters(), lr=1e-2, state_bits=bits)
        x = _x(64).float()
        for _ in range(3):
            y, aux, z, load = block(x)
            (y.square().mean() + 0.01 * aux + 0.001 * z).backward()
            before = {n: p.detach().clone() for n, p in block.named_parameters()}
            for n, p in block.named_parameters():
                assert p.grad is not None and torch.isfinite(p.grad).all(), n
            clip = 1.0 / torch.clamp(torch.linalg.vector_norm(torch.stack([p.grad.norm() for p in block.parameters()])), min=1.0)
            opt.step(grad_scale=clip)
            opt.zero_grad()
            block.moe.update_balance_bias(load)
            assert all(not torch.equal(before[n], p) for n, p in block.named_parameters())
        fresh = _layer(moe_pkg, seed=9, cls="SparseMoEBlock", **kw)
        fresh.load_state_dict(block.state_dict())
        with torch.no_grad():
            assert torch.equal(block(x)[0], fresh(x)[0])


def test_adamw_class_follows_torch_and_its_checkpoint(moe_pkg):
    """32-bit moments against torch.optim.AdamW on float64 copies; resuming from a state dict is the
    same as going on, for both widths; parameters without a gradient wait with their count."""
    g = torch.Generator().manual_seed(0)
    shapes = [(7,), (33, 5), (300,), (1,)]
    init = [torch.randn(s, generator=g) for s in shapes]
    grads = [[torch.randn(s, generator=g) for s in shapes] for _ in range(6)]

    def run(make, dtype, steps, params=None, opt=None, start=0):
        params = params or [torch.nn.Parameter(t.to(dtype).to(DEV)) for t in init]
        opt = opt or make(params)
        for k in range(start, steps):
            for i, p in enumerate(params):
                p.grad = None if (k == 2 and i == 1) else grads[k][i].to(dtype).to(DEV)
            opt.step()
        return params, opt

    hyper = dict(lr=1e-2, betas=(0.8, 0.95), weight_decay=0.1)
    want, _ = run(lambda p: torch.optim.AdamW(p, **hyper), torch.float64, 6)
    got, _ = run(lambda p: moe_pkg.AdamW(p, **hyper), torch.float32, 6)
    for a, b in zip(got, want):
        # six updates of at most a few lr, each off by 2^-19 of itself, and six roundings of the parameter
        torch.testing.assert_close(a.double(), b.detach(), rtol=2.0 ** -20, atol=6 * 4e-2 * 2.0 ** -19)
    for bits in (32, 8):
        def make(p):
            return moe_pkg.AdamW(p, state_bits=bits, seed=3, **hyper)

        whole, _ = run(make, torch.float32, 6)
        half, opt = run(make, torch.float32, 3)
        again = [torch.nn.Parameter(p.detach().clone()) for p in half]
        second = make(again)
        second.load_state_dict(opt.state_dict())
        if bits == 8:
            assert second.state[again[0]]["exp_avg"].dtype == torch.float8_e4m3fn
            assert second.state[again[0]]["exp_avg_sq"].dtype == torch.float8_e5m2
        resumed, _ = run(make, torch.float32, 6, again, second, start=3)
        for a, b in zip(whole, resumed):
            assert torch.equal(a, b)


def test_adamw_class_masters_mixed_types_and_lr_tensor(moe_pkg):
    g = torch.Generator().manual_seed(1)
    p16 = torch.nn.Parameter(torch.randn(500, generator=g).to(torch.bfloat16).to(DEV))
    p32 = torch.nn.Parameter(torch.randn(40, generator=g).to(DEV))
    lr = torch.tensor(1e-4, device=DEV)
    opt = moe_pkg.AdamW([{"params": [p16]}, {"params": [p32], "weight_decay": 0.0}], lr=lr, master_weights=True)
    before = p16.detach().clone()
    for _ in range(40):
        p16.grad, p32.grad = torch.ones_like(p16), torch.ones_like(p32)
        opt.step()
    master = opt.state[p16]["master"]
    assert "master" not in opt.state[p32]
    # 40 steps of 1e-4 are below a bf16 step of most values: the master has them
    assert float((master - before.float()).abs().mean()) > 2e-3
    assert torch.equal(p16, master.to(torch.bfloat16))
    with pytest.raises(ValueError):
        moe_pkg.AdamW([p32], state_bits=16)
    with pytest.raises(ValueError):
        moe_pkg.AdamW([p32], lr=-1.0)


def test_adamw_class_captured(moe_pkg):
    for bits in (32, 8):
        params = [torch.nn.Parameter(torch.linspace(-1, 1, n, device=DEV)) for n in (300, 17)]
        eager = [torch.nn.Parameter(p.detach().clone()) for p in params]
        opt = moe_pkg.AdamW(params, lr=1e-2, state_bits=bits, capturable=True)
        other = moe_pkg.AdamW(eager, lr=1e-2, state_bits=bits)
        for p, q in zip(params, eager):
            p.grad, q.grad = torch.full_like(p, 0.5), torch.full_like(q, 0.5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            opt.step()  # step 1, eager: allocates the state
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            opt.step()
        graph.replay()
        graph.replay()
        for _ in range(3):
            other.step()
        for p, q in zip(params, eager):
            torch.testing.assert_close(p, q, rtol=2.0 ** -20, atol=2.0 ** -20)
