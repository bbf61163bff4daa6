"""``adamw_step`` on B200.

32-bit moments against float64: m and v are two products and a sum, 3 * 2^-24 of the terms'
magnitudes (the scale factor and the rounded coefficients add 3 more); the update takes a square
root, two quotients and three products, 16 * 2^-24 of it (approximate square root and quotient of
2 ulp each included).  8-bit codes and scales are equal, bit for bit, to a float32 restatement.
"""

import math

import numpy as np
import pytest
import torch

import operators_ref as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
HYPER = dict(lr=1e-2, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.1)
E4, E5 = torch.float8_e4m3fn, torch.float8_e5m2


def _lists(sizes, ptype, gtype, seed, bits=32, master=False):
    g = torch.Generator().manual_seed(seed)
    r = lambda n, s: torch.randn(n, generator=g) * s  # noqa: E731
    out = dict(params=[], grads=[], exp_avgs=[], exp_avg_sqs=[])
    if bits == 8:
        out.update(exp_avg_scales=[], exp_avg_sq_scales=[])
    if master:
        out["masters"] = []
    for n in sizes:
        p = r(n, 0.05)
        out["params"].append(p.to(ptype).to(DEV))
        if master:
            out["masters"].append(p.to(DEV))
        out["grads"].append(r(n, 1e-2).to(gtype).to(DEV))
        if bits == 32:
            out["exp_avgs"].append(r(n, 3e-3).to(DEV))
            out["exp_avg_sqs"].append((r(n, 1e-2).square() + 1e-9).to(DEV))
        else:
            b = -(-n // 256)
            out["exp_avgs"].append(r(n, 40.0).clamp(-250, 250).to(E4).to(DEV))
            out["exp_avg_sqs"].append((r(n, 100.0).square()).to(E5).to(DEV))
            out["exp_avg_scales"].append(torch.full((b,), 2.0 ** -14).to(DEV))
            out["exp_avg_sq_scales"].append(torch.full((b,), 2.0 ** -27).to(DEV))
    return out


def _call(pkg, lists, **kw):
    kw = {**HYPER, **kw}
    names = [n for n in lists if n not in ("params", "grads", "exp_avgs", "exp_avg_sqs")]
    pkg.adamw_step(lists["params"], lists["grads"], lists["exp_avgs"], lists["exp_avg_sqs"],
                   **{n: lists[n] for n in names}, **kw)


def _clone(lists):
    return {n: [t.clone() for t in v] for n, v in lists.items()}


SIZES = [1, 3, 255, 256, 257, 0, 1000, 8192, 8193, 30001]


@pytest.mark.parametrize("ptype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("gtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("master", [False, True])
def test_32_bit_moments(moe_pkg, ptype, gtype, master):
    lists = _lists(SIZES, ptype, gtype, 1, master=master)
    old = _clone(lists)
    scale = torch.tensor([0.75], device=DEV)
    _call(moe_pkg, lists, step=7, grad_scale=scale)
    lr, betas, eps, wd = (HYPER[n] for n in ("lr", "betas", "eps", "weight_decay"))
    for i, n in enumerate(SIZES):
        o = {k: v[i].cpu() for k, v in old.items()}
        main = o["masters"] if master else o["params"]
        p, m, v = ref.adamw32(main, o["grads"], o["exp_avgs"], o["exp_avg_sqs"], 7, lr, betas, eps, wd, 0.75)
        new = {k: v_[i].cpu().double() for k, v_ in lists.items()}
        gs = o["grads"].double().abs() * 0.75
        u = 2.0 ** -24
        m_abs = 0.9 * o["exp_avgs"].double().abs() + 0.1 * gs
        assert ((new["exp_avgs"] - m).abs() <= 6 * u * m_abs + 2.0 ** -148).all()
        assert ((new["exp_avg_sqs"] - v).abs() <= 8 * u * v + 2.0 ** -148).all()
        upd = lr / (1 - 0.9 ** 7) * m_abs / ((v / (1 - 0.99 ** 7)).sqrt() + eps)
        tol = 32 * u * upd + 4 * u * main.double().abs()
        if master:
            assert ((new["masters"] - p).abs() <= tol).all()
            assert torch.equal(lists["params"][i].cpu(), lists["masters"][i].cpu().to(ptype))
        else:
            tiny = 2.0 ** -25 if ptype == torch.float16 else 0.0
            assert ((new["params"] - p).abs() <= tol + torch.finfo(ptype).eps / 2 * p.abs() + tiny).all()


def _expect8(old, i, step, seed, grad_scale, index):
    g = old["grads"][i].float().cpu().numpy()
    n = g.size
    m = old["exp_avgs"][i].float().cpu().numpy() * np.repeat(old["exp_avg_scales"][i].cpu().numpy(), 256)[:n]
    v = old["exp_avg_sqs"][i].float().cpu().numpy() * np.repeat(old["exp_avg_sq_scales"][i].cpu().numpy(), 256)[:n]
    m, v = ref.moments_f32(g, m, v, HYPER["betas"], grad_scale)
    w = ref.noise(n, index, step, seed)
    return m, v, ref.encode8(m, w >> 16, 3, 7, 7), ref.encode8(v, w & 0xFFFF, 2, 15, 14)


@pytest.mark.parametrize("ptype,gtype,master", [(torch.float32, torch.float32, False),
                                                (torch.bfloat16, torch.bfloat16, True),
                                                (torch.float16, torch.float32, False)])
def test_8_bit_moments_bit_for_bit(moe_pkg, ptype, gtype, master):
    sizes = [1, 5, 256, 259, 0, 1027, 8200]
    lists = _lists(sizes, ptype, gtype, 2, bits=8, master=master)
    # blocks that are zero, tiny, huge, and with values that are not finite
    for t, val in ((lists["exp_avgs"], 0.0), (lists["exp_avg_sqs"], 0.0), (lists["grads"], 0.0)):
        t[5][:256] = val
    lists["grads"][5][256:512] *= 2.0 ** -70 if gtype == torch.float32 else 2.0 ** -8
    lists["exp_avg_scales"][5][1] = 2.0 ** -120
    lists["exp_avg_sq_scales"][5][1] = 2.0 ** -126
    lists["grads"][5][600] = float("inf")
    lists["grads"][5][700] = float("nan")
    lists["grads"][5][800] = -float("inf")
    old = _clone(lists)
    seed = 0x123456789ABCDEF0
    scale = torch.tensor(0.5, device=DEV)
    _call(moe_pkg, lists, step=11, seed=seed, grad_scale=scale)
    for i, n in enumerate(sizes):
        if n == 0:
            continue
        _, _, (mc, ms), (vc, vs) = _expect8(old, i, 11, seed, 0.5, i)
        np.testing.assert_array_equal(lists["exp_avg_scales"][i].cpu().numpy(), ms)
        np.testing.assert_array_equal(lists["exp_avg_sq_scales"][i].cpu().numpy(), vs)
        np.testing.assert_array_equal(lists["exp_avgs"][i].view(torch.uint8).cpu().numpy(), mc)
        np.testing.assert_array_equal(lists["exp_avg_sqs"][i].view(torch.uint8).cpu().numpy(), vc)
    ok = torch.ones(1027, dtype=torch.bool)
    ok[[600, 700, 800]] = False
    assert torch.isfinite(lists["params"][5].cpu().float()[ok]).all()
    assert not torch.isfinite(lists["params"][5].cpu().float()[~ok]).any()


def test_noise_is_keyed_by_seed_step_and_index(moe_pkg):
    base = _lists([5000, 5000], torch.float32, torch.float32, 3, bits=8)
    for k in base:
        base[k][1] = base[k][0].clone()

    def codes(**kw):
        lists = _clone(base)
        _call(moe_pkg, lists, **kw)
        return lists["exp_avgs"][0].view(torch.uint8), lists["exp_avgs"][1].view(torch.uint8)

    a0, a1 = codes(step=5, seed=1)
    b0, b1 = codes(step=5, seed=1)
    assert torch.equal(a0, b0) and torch.equal(a1, b1)
    assert not torch.equal(a0, a1)                      # the tensor's place
    assert not torch.equal(a0, codes(step=6, seed=1)[0])
    assert not torch.equal(a0, codes(step=5, seed=1 << 40)[0])
    c0, c1 = codes(step=5, seed=1, indices=[1, 0])
    assert torch.equal(c0, a1) and torch.equal(c1, a0)


def test_rounding_keeps_the_mean(moe_pkg):
    """The mean of 400 draws of a value lies within 6 standard errors (a draw is off by less than a
    step, 2^-3 or 2^-2 of the value or of the block's smallest normal): for 512 values, chance 1e-6."""
    base = _lists([256], torch.float32, torch.float32, 4, bits=8)
    m, v, (_, ms), (_, vs) = _expect8(base, 0, 1, 0, None, 0)
    sum_m, sum_v, reps = np.zeros(256), np.zeros(256), 400
    for s in range(reps):
        lists = _clone(base)
        _call(moe_pkg, lists, step=1, seed=s)
        sum_m += lists["exp_avgs"][0].float().cpu().numpy().astype(np.float64) * ms[0]
        sum_v += lists["exp_avg_sqs"][0].float().cpu().numpy().astype(np.float64) * vs[0]
    # a draw between two neighbours has a standard deviation of at most half their distance
    step_m = np.maximum(np.abs(m) * 2.0 ** -3, ms[0] * 2.0 ** -9)
    step_v = np.maximum(np.abs(v) * 2.0 ** -2, vs[0] * 2.0 ** -16)
    assert np.isfinite(m).all()
    assert (np.abs(sum_m / reps - m) <= 6 * 0.5 * step_m / math.sqrt(reps)).all()
    fine = np.isfinite(v)  # draws above the largest e5m2 value are inf, and NaN as a moment
    assert (np.abs(sum_v / reps - v) <= 6 * 0.5 * step_v / math.sqrt(reps))[fine].all()
    assert np.isnan(sum_v[~fine]).all()


def test_unaligned_views_and_many_tensors(moe_pkg):
    """Views at odd elements of one buffer, more of them than one launch's table holds."""
    rng = np.random.default_rng(0)
    sizes = [int(n) for n in rng.integers(1, 700, 900)]
    for bits in (32, 8):
        a = _lists(sizes, torch.float32, torch.bfloat16, 5, bits=bits)
        b = {}
        for k, v in a.items():
            flat = torch.cat([t.view(torch.uint8) for t in v])
            unit = v[0].element_size()
            buf = torch.zeros(flat.numel() + unit, dtype=torch.uint8, device=DEV)
            buf[unit:] = flat
            whole = buf.view(v[0].dtype)
            at, views = 1, []
            for t in v:
                views.append(whole[at:at + t.numel()])
                at += t.numel()
            b[k] = views
        _call(moe_pkg, a, step=3, seed=9)
        _call(moe_pkg, b, step=3, seed=9)
        for k in a:
            for s, t in zip(a[k], b[k]):
                assert torch.equal(s.view(torch.uint8), t.contiguous().view(torch.uint8)), k


def test_device_step_and_lr_and_capture(moe_pkg):
    for bits in (32, 8):
        a = _lists([700, 12], torch.float32, torch.float32, 6, bits=bits)
        b = _clone(a)
        step, lr = torch.tensor([0], device=DEV), torch.tensor(0.0, device=DEV)

        def one():
            step.add_(1)
            _call(moe_pkg, b, step=step, lr=lr, seed=4)

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            warm = _clone(b)
            _call(moe_pkg, warm, step=torch.tensor([1], device=DEV), lr=lr, seed=4)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one()
        step.zero_()
        for k in range(1, 4):
            lr.fill_(0.5 ** k)
            graph.replay()
            _call(moe_pkg, a, step=k, lr=0.5 ** k, seed=4)
        for k in a:
            for s, t in zip(a[k], b[k]):
                if k in ("params", "masters"):  # the same double-precision corrections, host and device pow
                    torch.testing.assert_close(s, t, rtol=2.0 ** -21, atol=2.0 ** -21, equal_nan=True)
                else:
                    assert torch.equal(s.view(torch.uint8), t.view(torch.uint8)), k


def test_versions_move_and_gradients_stay(moe_pkg):
    lists = _lists([100], torch.float32, torch.float32, 7)
    p, g = torch.nn.Parameter(lists["params"][0]), lists["grads"][0]
    before, vp, vg = g.clone(), p._version, g._version
    moe_pkg.adamw_step([p], [g], lists["exp_avgs"], lists["exp_avg_sqs"], step=1)
    assert p._version > vp and g._version == vg and torch.equal(g, before)
    with torch.enable_grad():
        q = torch.nn.Parameter(torch.ones(4, device=DEV))
        loss = (q * q).sum()
        m = [torch.zeros(4, device=DEV)], [torch.zeros(4, device=DEV)]
        moe_pkg.adamw_step([q], [torch.ones(4, device=DEV)], *m, step=1)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            loss.backward()


def test_strided_gradients_and_empty_calls(moe_pkg):
    p = torch.randn(6, 8, device=DEV)
    g = torch.randn(8, 6, device=DEV).t()
    a = [[p.clone()], [g], [torch.zeros_like(p)], [torch.zeros_like(p)]]
    b = [[p.clone()], [g.contiguous()], [torch.zeros_like(p)], [torch.zeros_like(p)]]
    moe_pkg.adamw_step(*a, step=1)
    moe_pkg.adamw_step(*b, step=1)
    assert torch.equal(a[0][0], b[0][0])
    moe_pkg.adamw_step([], [], [], [], step=1)
    e = [torch.empty(0, device=DEV) for _ in range(4)]
    moe_pkg.adamw_step(*[[t] for t in e], step=1)
