"""What ``route_experts``, ``residual_norm`` and ``adamw_step`` refuse, checked without a GPU:
the Python checks run before the device is asked for, the library's on null device pointers."""

import ctypes
from array import array

import pytest
import torch


def _route(pkg, logits=None, k=2, **kw):
    return pkg.route_experts(torch.zeros(3, 8) if logits is None else logits, k, **kw)


@pytest.mark.parametrize("kw", [
    dict(score="relu"), dict(group_score="sum"), dict(k=0), dict(k=9), dict(num_groups=3), dict(num_groups=0),
    dict(num_groups=4, top_groups=5), dict(num_groups=4, top_groups=0), dict(num_groups=4, top_groups=1, k=3),
    dict(bias=torch.zeros(7)), dict(bias=torch.zeros(8, 1)), dict(valid=torch.ones(4)), dict(valid=torch.ones(3, 1)),
    dict(logits=torch.zeros(3, 8, dtype=torch.float64)), dict(logits=torch.zeros(3, 8, dtype=torch.int32)),
    dict(logits=torch.zeros(3, 0)), dict(logits=torch.zeros(2, 513)), dict(logits=torch.zeros(2, 64), k=33),
    dict(logits=torch.zeros(())),
])
def test_route_refuses(moe_pkg, kw):
    with pytest.raises(ValueError):
        _route(moe_pkg, **kw)


def test_nothing_runs_on_the_cpu(moe_pkg):
    with pytest.raises(ValueError, match="CUDA"):
        _route(moe_pkg)
    with pytest.raises(ValueError, match="CUDA"):
        moe_pkg.residual_norm(torch.zeros(2, 8), torch.zeros(2, 8))
    t = [[torch.zeros(4)] for _ in range(4)]
    with pytest.raises(ValueError, match="CUDA"):
        moe_pkg.adamw_step(*t, step=1)


X, W = torch.zeros(2, 3, 8), torch.ones(8)


@pytest.mark.parametrize("args,kw", [
    ((X,), dict()), ((X,), dict(gate=W, pre_weight=W)), ((X,), dict(post_weight=W, pre_weight=W)),
    ((X,), dict(pre_weight=W, residual_scale=0.5)), ((X,), dict(pre_weight=W, branch_scale=0.5)),
    ((X, torch.zeros(2, 3, 4)), dict()), ((X, torch.zeros(3, 8)), dict()), ((X, X), dict(gate_activation="relu")),
    ((X, X), dict(post_weight=torch.ones(4))), ((X, X), dict(pre_weight=torch.ones(1, 8))),
    ((X, X), dict(gate=torch.ones(2, 8))), ((X, X), dict(gate=torch.ones(1, 2, 3, 8))),
    ((X, X), dict(gate=torch.ones(8, dtype=torch.float64))), ((X, X.double()), dict()),
    ((X, X), dict(pre_weight=W, norm_dtype=torch.float64)), ((torch.zeros(()), torch.zeros(())), dict()),
    ((torch.zeros(1, 16385), torch.zeros(1, 16385)), dict()), ((torch.zeros(2, 0), torch.zeros(2, 0)), dict()),
])
def test_norm_refuses(moe_pkg, args, kw):
    with pytest.raises(ValueError):
        moe_pkg.residual_norm(*args, **kw)


def _adam(**change):
    f = dict(params=[torch.zeros(300)], grads=[torch.zeros(300)], exp_avgs=[torch.zeros(300)],
             exp_avg_sqs=[torch.zeros(300)])
    f.update(change)
    return f


@pytest.mark.parametrize("change", [
    dict(step=0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(eps=float("nan")),
    dict(grads=[]), dict(grads=[torch.zeros(299)]), dict(exp_avgs=[torch.zeros(300, dtype=torch.bfloat16)]),
    dict(exp_avg_sqs=[torch.zeros(600)[::2]]), dict(params=[torch.zeros(300, dtype=torch.float64)]),
    dict(exp_avg_scales=[torch.ones(2)]), dict(masters=[torch.zeros(300, dtype=torch.float16)]),
    dict(exp_avg_scales=[torch.ones(2)], exp_avg_sq_scales=[torch.ones(2)]),  # the moments are not 8 bits
    dict(step=torch.ones(1)), dict(lr=torch.ones(2)), dict(grad_scale=torch.ones(1, dtype=torch.float64)),
    dict(indices=[0, 1]), dict(params=[torch.zeros(600)[::2]]),
])
def test_adamw_refuses(moe_pkg, change):
    f = _adam(**change)
    lists = [f.pop(n) for n in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    f.setdefault("step", 1)
    with pytest.raises(ValueError):
        moe_pkg.adamw_step(*lists, **f)


def test_adamw_refuses_a_tensor_given_twice(moe_pkg):
    t = torch.zeros(8)
    with pytest.raises(ValueError, match="twice"):
        moe_pkg.adamw_step([t, t], [torch.zeros(8)] * 2, [torch.zeros(8), torch.zeros(8)],
                           [torch.zeros(8), torch.zeros(8)], step=1)
    with pytest.raises(ValueError, match="twice"):
        moe_pkg.adamw_step([t], [torch.zeros(8)], [t], [torch.zeros(8)], step=1)
    scales = [torch.ones(1)], [torch.ones(2)]
    with pytest.raises(ValueError, match="exp_avg_sq_scales"):
        moe_pkg.adamw_step([t], [torch.zeros(8)], [torch.zeros(8).to(torch.float8_e4m3fn)],
                           [torch.zeros(8).to(torch.float8_e5m2)], step=1, exp_avg_scales=scales[0],
                           exp_avg_sq_scales=scales[1])


def test_library_refuses(moe_pkg):
    lib, L = moe_pkg.library(), moe_pkg._lib

    def route(T=4, E=8, k=2, dtype=1, ld=8, score=0, groups=1, top=1, gs=0, ptr=None):
        return lib.mcl4moe_route_scores(ptr, dtype, ld, None, None, T, E, k, score, groups, top, gs, 1, 1.0, ptr, ptr,
                                        None, None)

    assert route() == L.ERR_INVALID  # null pointers
    for bad in (dict(T=-1), dict(E=0), dict(k=0), dict(k=9), dict(dtype=3), dict(ld=7), dict(score=2), dict(groups=3),
                dict(groups=4, top=0), dict(groups=4, top=5), dict(groups=4, top=1, k=3), dict(gs=2)):
        assert route(**{**dict(T=0), **bad}) == L.ERR_INVALID, bad
    assert route(T=0, E=513, ld=513) == L.ERR_UNSUPPORTED
    assert route(T=0, E=64, k=33, ld=64) == L.ERR_UNSUPPORTED
    assert route(T=0) == L.OK
    assert lib.mcl4moe_route_scores_backward(None, 1, 8, None, None, 4, 8, 2, 0, 1, 1.0, None, None) == L.ERR_INVALID
    assert lib.mcl4moe_route_scores_backward(None, 1, 8, None, None, 0, 8, 2, 0, 1, 1.0, None, None) == L.OK

    def norm(backward=False, **kw):
        a = L.NormArgs(rows=0, cols=8, x_dtype=1, norm_dtype=1, ld_x=8)
        for n, v in kw.items():
            setattr(a, n, v)
        if backward:
            return lib.mcl4moe_residual_norm_backward(a, None, 0, None)
        return lib.mcl4moe_residual_norm(a, None)

    assert lib.mcl4moe_residual_norm(None, None) == L.ERR_INVALID
    assert norm() == L.OK
    for bad in (dict(rows=-1), dict(cols=0), dict(x_dtype=3), dict(ld_x=7), dict(rows=1), dict(gate_mode=1),
                dict(gate_mode=4), dict(branch=64, ld_branch=7), dict(branch=64, ld_branch=8, gate_mode=1, gate_rows=0),
                dict(norm_dtype=5), dict(gate_act=3)):
        assert norm(**bad) == L.ERR_INVALID, bad
        assert norm(backward=True, **bad) == L.ERR_INVALID, bad
    assert norm(cols=16385, ld_x=16385) == L.ERR_UNSUPPORTED
    assert lib.mcl4moe_residual_norm_workspace_size(64, 2048, 0, 0) >= 3 * 4 * 2048
    assert lib.mcl4moe_residual_norm_workspace_size(64, 16385, 0, 0) == 0

    def adam(**kw):
        a = L.AdamwArgs(n=0, param_dtype=1, grad_dtype=1, bits=32, beta1=0.9, beta2=0.99, eps=1e-8, step=1)
        for n, v in kw.items():
            setattr(a, n, v)
        return lib.mcl4moe_adamw_step(ctypes.byref(a), None)

    assert lib.mcl4moe_adamw_step(None, None) == L.ERR_INVALID
    assert adam() == L.OK
    for bad in (dict(n=-1), dict(n=1), dict(param_dtype=3), dict(grad_dtype=-1), dict(bits=4), dict(beta1=1.0),
                dict(beta2=-0.5), dict(eps=-1.0), dict(step=0)):
        assert adam(**bad) == L.ERR_INVALID, bad
    numels, null = array("q", [5]), array("Q", [0])
    at = null.buffer_info()[0]
    assert adam(n=1, numels=numels.buffer_info()[0], params=at, grads=at, exp_avgs=at, exp_avg_sqs=at) == L.ERR_INVALID


def test_config_of_scored_routing_and_block(moe_pkg):
    base = dict(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2)
    for bad in (dict(score_function="relu"), dict(group_score="sum"), dict(expert_groups=3), dict(expert_groups=0),
                dict(expert_groups=4, top_expert_groups=5), dict(expert_groups=8, top_expert_groups=1),
                dict(residual_gate="relu")):
        with pytest.raises(ValueError):
            moe_pkg.MoEConfig(**base, **bad)
    layer = moe_pkg.SparseMoE(moe_pkg.MoEConfig(**base))
    assert layer._routing_variant(None, None, None) is None and layer.balance_bias is None
    for kw in (dict(score_function="sigmoid"), dict(expert_groups=4, top_expert_groups=2), dict(routed_scale=2.0),
               dict(balance_bias=True)):
        assert moe_pkg.SparseMoE(moe_pkg.MoEConfig(**base, **kw))._routing_variant(None, None, None) == "scored"
    with pytest.raises(ValueError, match="balance_bias"):
        layer.update_balance_bias(torch.zeros(8))
    block = moe_pkg.SparseMoEBlock(moe_pkg.MoEConfig(**base))
    assert {"moe_norm", "moe.router.weight"} <= set(block.state_dict())
    assert block.post_norm is None and block.gate is None


def test_optimizer_arguments(moe_pkg):
    p = torch.nn.Parameter(torch.zeros(3))
    for bad in (dict(state_bits=4), dict(lr=-1e-3), dict(betas=(1.0, 0.9)), dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            moe_pkg.AdamW([p], **bad)
    opt = moe_pkg.AdamW([p])
    opt.step()  # nothing has a gradient
    assert not opt.state
