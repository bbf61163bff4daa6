"""Calls at the borders of the layer and of its operators that are refused, or decided on the host, checked
without a GPU."""

import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp
from torch.autograd import forward_ad

from test_ep_cpu import _free_port

HERE = Path(__file__).resolve().parent


def _layer(pkg, **kw):
    return pkg.SparseMoE(pkg.MoEConfig(**{**dict(d_model=256, expert_hidden_dim=256, num_experts=8, top_k=2), **kw}))


def test_logit_bias_has_one_entry_per_expert(moe_pkg):
    layer = _layer(moe_pkg)
    cpu = torch.device("cpu")
    assert layer._logit_bias(cpu, 8) is None
    for n in (7, 9):
        layer.router_logit_bias = torch.zeros(n)
        with pytest.raises(ValueError, match="router_logit_bias"):
            layer._logit_bias(cpu, 8)
    layer.router_logit_bias = torch.arange(8, dtype=torch.bfloat16)
    assert torch.equal(layer._logit_bias(cpu, 8), torch.arange(8, dtype=torch.float32))


def _expert_parallel_worker(rank, port):
    sys.path[:0] = [str(HERE.parent), str(HERE)]
    os.environ.update(MASTER_ADDR="127.0.0.1", MASTER_PORT=str(port))
    dist.init_process_group("gloo", rank=rank, world_size=1)
    try:
        from __graft_entry__ import load_package
        from ep_oracle_ops import OracleEPOps

        ep = load_package().ExpertParallelMoE.from_dense(_layer(load_package(), num_experts=4), ops=OracleEPOps())
        x = torch.zeros(6, 256, dtype=torch.bfloat16)
        for n in (5, 7):
            with pytest.raises(ValueError, match="valid"):
                ep(x, torch.ones(n))
        ep.router_logit_bias = torch.zeros(3)
        with pytest.raises(ValueError, match="router_logit_bias"):
            ep(x)
    finally:
        dist.destroy_process_group()


def test_expert_parallel_refuses_wrong_lengths():
    mp.spawn(_expert_parallel_worker, args=(_free_port(),), nprocs=1, join=True)


def _capturable(pkg, counts):
    """(a fresh optimizer of two parameters, a checkpoint of such a one with ``counts``)"""
    params = [torch.nn.Parameter(torch.zeros(5)), torch.nn.Parameter(torch.zeros(3))]
    opt = pkg.AdamW(params, capturable=True)
    saved = opt.state_dict()
    saved["state"] = {i: dict(step=0, exp_avg=torch.ones(p.shape), exp_avg_sq=torch.ones(p.shape))
                      for i, p in enumerate(params)}
    saved["param_groups"][0]["step_counts"] = {d: torch.tensor(n) for d, n in counts.items()}
    return opt, saved


@pytest.mark.parametrize("counts", [{"cpu": 41}, {"cuda:0": 41}, {"cuda:0": 41, "cuda:1": 41}, {"cpu": 41, "cuda:1": 41}])
def test_device_step_count_goes_on_after_loading(moe_pkg, counts):
    """A checkpoint of one device loaded on another: the count goes where the moments go."""
    opt, saved = _capturable(moe_pkg, counts)
    opt.load_state_dict(saved)
    group = opt.param_groups[0]
    assert {d: int(t) for d, t in group["step_counts"].items()} == {"cpu": 41}
    after = opt._device_counts(group, {(torch.device("cpu"), torch.float32): []})
    assert int(after[torch.device("cpu")]) == 42
    assert saved["param_groups"][0]["step_counts"] == {d: torch.tensor(41) for d in counts}


def test_device_step_counts_that_differ_are_not_guessed(moe_pkg):
    opt, saved = _capturable(moe_pkg, {"cuda:0": 41, "cuda:1": 40})
    with pytest.raises(ValueError, match="step counts"):
        opt.load_state_dict(saved)
    opt, saved = _capturable(moe_pkg, {})
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["step_counts"] == {}


def test_learning_rate_tensor_follows_the_parameters(moe_pkg):
    p = torch.nn.Parameter(torch.zeros(5))
    opt = moe_pkg.AdamW([p], lr=torch.tensor(1e-3))
    opt.load_state_dict(opt.state_dict())
    assert opt.param_groups[0]["lr"].device == p.device and float(opt.param_groups[0]["lr"]) == pytest.approx(1e-3)


def test_a_capture_needs_a_device_count_and_state(moe_pkg, monkeypatch):
    monkeypatch.setattr(torch.cuda, "is_initialized", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    p = torch.nn.Parameter(torch.zeros(5))
    opt = moe_pkg.AdamW([p])
    opt.step()  # nothing has a gradient
    p.grad = torch.ones(5)
    with pytest.raises(RuntimeError, match="capturable"):
        opt.step()
    assert not opt.state
    opt = moe_pkg.AdamW([p], capturable=True)
    with pytest.raises(RuntimeError, match="eager"):
        opt.step()
    assert not opt.state and "step_counts" not in opt.param_groups[0]


def test_a_changed_kind_of_step_count_goes_on(moe_pkg):
    params = [torch.nn.Parameter(torch.zeros(n)) for n in (5, 3)]
    opt = moe_pkg.AdamW(params, capturable=True)
    group, cpu = opt.param_groups[0], torch.device("cpu")
    states = [opt.state[p] for p in params]
    for s in states:
        s.update(opt._new_state(params[0], group), step=4)
    items = [(p, s, i) for i, (p, s) in enumerate(zip(params, states))]
    assert int(opt._device_counts(group, {(cpu, 4): items})[cpu]) == 5
    opt._host_counts(group)
    assert [s["step"] for s in states] == [5, 5] and "step_counts" not in group
    states[0]["step"] = 2
    with pytest.raises(ValueError, match="step count"):
        opt._device_counts(group, {(cpu, 2): items[:1], (cpu, 5): items[1:]})


def test_forward_mode_derivatives_are_refused(moe_pkg):
    x, w = torch.zeros(3, 8), torch.ones(8)
    with forward_ad.dual_level():
        dx, dw = forward_ad.make_dual(x, torch.ones_like(x)), forward_ad.make_dual(w, torch.ones_like(w))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            moe_pkg.route_experts(dx, 2)
        for args, kw in (((dx, x), {}), ((x, dx), {}), ((x, x), dict(gate=dw)), ((x, x), dict(post_weight=dw)),
                         ((x,), dict(pre_weight=dw))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                moe_pkg.residual_norm(*args, **kw)
        with pytest.raises(ValueError, match="CUDA"):  # nothing has a tangent
            moe_pkg.residual_norm(x, x)
    with pytest.raises((NotImplementedError, RuntimeError)):
        torch.func.jvp(lambda t: moe_pkg.route_experts(t, 2)[0], (x,), (x,))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float64])
def test_balance_bias_keeps_float32(moe_pkg, dtype):
    start = torch.linspace(-0.9, 0.9, 8) + 1e-4
    for make in (lambda m: m.to(dtype), lambda m: torch.nn.Sequential(m).to(dtype)[0]):
        layer = _layer(moe_pkg, balance_bias=True)
        layer.balance_bias.copy_(start)
        layer = make(layer)
        assert layer.router.weight.dtype == dtype
        assert layer.balance_bias.dtype == torch.float32 and torch.equal(layer.balance_bias, start)
        assert "balance_bias" in dict(layer.named_buffers())
        # loads that 8 significant bits do not tell apart, 1000 times
        counts = torch.tensor([1001, 1001, 1001, 1001, 999, 999, 999, 999])
        for _ in range(1000):
            layer.update_balance_bias(counts, rate=1e-3)
        # each of the 1000 sums rounds to 2^-24 of at most 2
        moved = torch.tensor([-1.0] * 4 + [1.0] * 4)
        torch.testing.assert_close(layer.balance_bias, start + moved, rtol=0, atol=1000 * 2.0 ** -23)
    assert _layer(moe_pkg).to(dtype).balance_bias is None


def test_balance_bias_of_a_checkpoint_in_bf16(moe_pkg):
    layer = _layer(moe_pkg, balance_bias=True)
    state = {n: t.to(torch.bfloat16) for n, t in layer.state_dict().items()}
    state["balance_bias"].fill_(0.75)
    layer.load_state_dict(state, assign=True)
    layer.update_balance_bias(torch.arange(8), rate=1e-3)
    want = 0.75 + 1e-3 * torch.tensor([1.0] * 4 + [-1.0] * 4)
    torch.testing.assert_close(layer.balance_bias, want, rtol=2.0 ** -23, atol=0)


def test_enable_cuda_graph_says_where_it_does_nothing(moe_pkg, recwarn):
    _layer(moe_pkg).enable_cuda_graph()
    _layer(moe_pkg, score_function="sigmoid").enable_cuda_graph(False)
    assert not recwarn.list
    with pytest.warns(UserWarning, match="routes from scores"):
        _layer(moe_pkg, score_function="sigmoid").enable_cuda_graph()


def _in_a_process(code):
    """What ``code`` prints with the library as ``lib``; a signal that ends the process shows."""
    run = subprocess.run([sys.executable, "-c", "from __graft_entry__ import load_package\npkg = load_package()\n"
                          "lib = pkg.library()\n" + code], cwd=HERE.parent, capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, (run.returncode, run.stderr[-500:])
    return run.stdout.split()


def test_norm_workspace_of_gates_that_do_not_fit(moe_pkg):
    """Gate rows that do not divide the rows, as many as there are and more: the call that would use them
    is refused, and so there is no workspace."""
    got = _in_a_process("for rows in (3, 9, 10, 11, 20, 1 << 40):\n"
                        "    print(lib.mcl4moe_residual_norm_workspace_size(10, 64, 1, rows))")
    assert [int(n) > 0 for n in got] == [False, False, True, False, False, False]


def test_sizes_whose_products_overflow_are_refused(moe_pkg):
    """Counts of rows and elements near the end of 64 bits, with addresses that are never used."""
    got = _in_a_process("""
import ctypes
from array import array
L = pkg._lib
at = 1 << 20
for T in (1 << 62, (1 << 63) - 1, (1 << 30) + 1, 1 << 29):
    for back in (False, True):
        if back:
            st = lib.mcl4moe_route_scores_backward(at, 1, 8, at, at, T, 8, 4, 0, 1, 1.0, at, None)
        else:
            st = lib.mcl4moe_route_scores(at, 1, 8, None, None, T, 8, 4, 0, 1, 1, 0, 1, 1.0, at, at, None, None)
        print(st == L.ERR_UNSUPPORTED)
pointers = array("Q", [at])
p = pointers.buffer_info()[0]
for n in ((1 << 63) - 1, (1 << 63) - 4000, 1 << 43):
    for bits in (8, 32):
        numels = array("q", [n])
        a = L.AdamwArgs(n=1, param_dtype=1, grad_dtype=1, bits=bits, beta1=0.9, beta2=0.99, eps=1e-8, step=1, params=p,
                        grads=p, exp_avgs=p, exp_avg_sqs=p, exp_avg_scales=p, exp_avg_sq_scales=p,
                        numels=numels.buffer_info()[0])
        print(lib.mcl4moe_adamw_step(ctypes.byref(a), None) == L.ERR_UNSUPPORTED)
""")
    assert got == ["True"] * 14


def test_invalidate_cache_leaves_no_bytes_to_carry_over(moe_pkg):
    layer, nv = _layer(moe_pkg), moe_pkg.nvfp4
    setattr(layer.experts, nv.CACHE_ATTR, {"up_proj": object()})
    for e in layer.experts:
        setattr(e.up_proj, nv.SLOT_ATTR, (object(), 0))
        setattr(e.down_proj, nv.SLOT_ATTR, (object(), 0))
    nv.invalidate_cache(layer.experts)
    assert getattr(layer.experts, nv.CACHE_ATTR) is None
    assert not any(hasattr(m, nv.SLOT_ATTR) for m in layer.modules())
