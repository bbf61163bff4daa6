"""Cases of the operators around the expert layer: routing from scores, the norms and
residual sum around the block, and the AdamW step over the layer's parameters.

``run`` computes a case in its plain form (elementary torch operations), or, where
``own`` is true, through the framework's entry points:

    route_experts   scores -> (weights, expert ids, counts), and its gradient
    residual_norm   post-norm, gate, residual sum and the next pre-norm, and its gradient
    adamw_step      one decoupled-weight-decay Adam step over a list of tensors, states in
                    32 bits or in 8 (a power-of-two scale for each 256 elements)
"""

import math
import random

import numpy as np
import torch

own = False

NEG_INF = float("-inf")
BLOCK = 256  # elements of a tensor that share one scale of an 8-bit state
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


def _entry():
    from __graft_entry__ import load_package

    return load_package()


# ---------------------------------------------------------------------------- cases


def listed():
    return [
        # one decode step's routing: 64 sequences, the latency of a call
        dict(name="route decode", op="route", tokens=64, experts=64, top_k=8, score="sigmoid", bias=True, groups=1,
             top_groups=1, group_score="top2", renorm=True, scale=1.0, dtype="float32", masked=False, train=False),
        # prefill with group-limited selection over the headline layer's experts
        dict(name="route prefill groups", op="route", tokens=32768, experts=64, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", renorm=True, scale=2.5, dtype="float32", masked=False,
             train=False),
        # the grown skewed layer: 40 experts, plain softmax scores kept as they are, bf16 logits, padded batch
        dict(name="route train softmax", op="route", tokens=65536, experts=40, top_k=8, score="softmax", bias=False,
             groups=1, top_groups=1, group_score="max", renorm=False, scale=1.0, dtype="bfloat16", masked=True,
             train=True),
        # many fine experts in groups, an odd token count, forward and gradient
        dict(name="route train wide", op="route", tokens=16383, experts=256, top_k=8, score="sigmoid", bias=True,
             groups=8, top_groups=4, group_score="top2", renorm=True, scale=2.5, dtype="float32", masked=False,
             train=True),
        # decode: both norms, the gate and the residual of 64 tokens
        dict(name="norm decode", op="norm", tokens=64, dim=2048, stream="bfloat16", branch="bfloat16", post=True,
             gate="channel", act="none", pre=True, train=False),
        # prefill at the headline width
        dict(name="norm prefill", op="norm", tokens=32768, dim=2048, stream="bfloat16", branch="bfloat16", post=True,
             gate="channel", act="none", pre=True, train=False),
        # training at the headline width: gradients of the stream, the branch, both norms and the gate
        dict(name="norm train", op="norm", tokens=32768, dim=2048, stream="bfloat16", branch="bfloat16", post=True,
             gate="channel", act="sigmoid", pre=True, train=True),
        # float32 residual stream with a bf16 block, one gate value for each token, an odd width and length
        dict(name="norm train ragged", op="norm", tokens=4099, dim=1001, stream="float32", branch="bfloat16",
             post=True, gate="token", act="tanh", pre=True, train=True),
        # a small layer's ten tensors: the latency of a step
        dict(name="adamw small", op="adamw", experts=4, dim=64, hidden=128, param="float32", grad="float32", bits=32,
             master=False, clip=True),
        # every tensor of the headline layer (129 and a norm weight), 32-bit states
        dict(name="adamw experts", op="adamw", experts=64, dim=2048, hidden=1024, param="float32", grad="float32",
             bits=32, master=False, clip=False),
        # the skewed layer's tensors with 8-bit states
        dict(name="adamw experts 8 bits", op="adamw", experts=40, dim=1536, hidden=512, param="float32",
             grad="float32", bits=8, master=False, clip=True),
        # bf16 parameters and gradients with float32 masters, 8-bit states, ragged blocks
        dict(name="adamw ragged 8 bits", op="adamw", experts=24, dim=777, hidden=391, param="bfloat16",
             grad="bfloat16", bits=8, master=True, clip=False),
    ]


def _spread(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, max(low, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    op = rng.choice(["route", "norm", "adamw"])
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        size = _spread(rng, 2, 256 // groups)
        experts = groups * size
        top_groups = rng.randint(1, groups)
        top_k = rng.randint(1, min(16, top_groups * size))
        tokens = min(_spread(rng, 1, 65536), (1 << 22) // experts)
        return dict(op=op, tokens=tokens, experts=experts, top_k=top_k, score=rng.choice(["softmax", "sigmoid"]),
                    bias=rng.random() < 0.5, groups=groups, top_groups=top_groups,
                    group_score=rng.choice(["top2", "max"]), renorm=rng.random() < 0.7,
                    scale=rng.choice([1.0, 2.5]), dtype=rng.choice(["float32", "bfloat16", "float16"]),
                    masked=rng.random() < 0.4, train=rng.random() < 0.6)
    if op == "norm":
        dim = _spread(rng, 32, 8192)
        dim = dim // 64 * 64 + (64 if dim < 64 else 0) if rng.random() < 0.6 else dim
        tokens = min(_spread(rng, 1, 32768), (1 << 26) // dim)
        stream, branch = rng.choice([("bfloat16", "bfloat16"), ("float16", "float16"), ("float32", "float32"),
                                     ("float32", "bfloat16"), ("float32", "float16")])
        return dict(op=op, tokens=tokens, dim=dim, stream=stream, branch=branch, post=rng.random() < 0.8,
                    gate=rng.choice(["none", "channel", "token", "full"]),
                    act=rng.choice(["none", "sigmoid", "tanh"]), pre=rng.random() < 0.8, train=rng.random() < 0.6)
    experts, dim = _spread(rng, 1, 64), _spread(rng, 16, 2048)
    hidden = _spread(rng, 16, 1024)
    param = rng.choice(["float32", "float32", "bfloat16"])
    return dict(op=op, experts=experts, dim=dim, hidden=hidden, param=param, grad=rng.choice(["float32", param]),
                bits=rng.choice([8, 32]), master=param != "float32" and rng.random() < 0.7, clip=rng.random() < 0.5)


# ---------------------------------------------------------------------------- inputs


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 17)


def prepare(case, seed):
    rnd = _generator(seed)
    return dict(route=_prepare_route, norm=_prepare_norm, adamw=_prepare_adamw)[case["op"]](case, rnd)


def _prepare_route(case, rnd):
    tokens, experts, top_k = case["tokens"], case["experts"], case["top_k"]
    # router rows of N(0, 0.02) on inputs of N(0, 1) at width 2048, some experts favoured
    skew = torch.randn(experts, generator=rnd, device="cuda") * 0.3
    logits = torch.randn(tokens, experts, generator=rnd, device="cuda") * 0.9 + skew
    s = dict(case=case, logits=logits.to(DTYPES[case["dtype"]]), bias=None, valid=None, d_weights=None)
    if case["bias"]:  # what a balance rule with steps of 0.001 has added up to
        s["bias"] = torch.randint(-60, 61, (experts,), generator=rnd, device="cuda").float() * 1e-3
    if case["masked"]:  # padding at the end of a batch
        s["valid"] = torch.arange(tokens, device="cuda") < tokens - tokens // 9
    if case["train"]:
        s["logits"].requires_grad_(True)
        s["d_weights"] = torch.randn(tokens, top_k, generator=rnd, device="cuda") * 0.1
    return s


def _prepare_norm(case, rnd):
    tokens, dim = case["tokens"], case["dim"]
    stream, branch = DTYPES[case["stream"]], DTYPES[case["branch"]]

    def normal(*shape, std=1.0, mean=0.0):
        return torch.randn(*shape, generator=rnd, device="cuda") * std + mean

    s = dict(case=case, x=normal(tokens, dim).to(stream), branch=normal(tokens, dim, std=0.3).to(branch),
             post=normal(dim, std=0.1, mean=1.0) if case["post"] else None,
             pre=normal(dim, std=0.1, mean=1.0) if case["pre"] else None, gate=None, d_stream=None, d_normed=None)
    if case["gate"] != "none":
        shape = dict(channel=(dim,), token=(tokens, 1), full=(tokens, dim))[case["gate"]]
        gate = normal(*shape, std=0.5, mean=0.3)
        s["gate"] = gate.to(branch) if case["gate"] == "full" else gate
    if case["train"]:
        s["d_stream"] = normal(tokens, dim, std=0.1).to(stream)
        s["d_normed"] = normal(tokens, dim, std=0.1).to(branch) if case["pre"] else None
        for name in ("x", "branch", "post", "pre", "gate"):
            if s[name] is not None:
                s[name].requires_grad_(True)
    return s


def _sizes(case):
    """Elements of the layer's tensors: gate/up and down projection of each expert, the router, a norm."""
    experts, dim, hidden = case["experts"], case["dim"], case["hidden"]
    return [2 * hidden * dim, hidden * dim] * experts + [experts * dim, dim]


def _views(flat, sizes, unit=1):
    """One view for each tensor of ``flat``, where each begins at a multiple of BLOCK elements."""
    starts = np.cumsum([0] + [-(-n // BLOCK) * BLOCK for n in sizes])
    return [flat[int(a) // unit:int(a) // unit + -(-n // unit)] for a, n in zip(starts, sizes)]


def _prepare_adamw(case, rnd):
    sizes = _sizes(case)
    total = sum(-(-n // BLOCK) * BLOCK for n in sizes)
    param = DTYPES[case["param"]]

    def normal(std):
        return torch.randn(total, generator=rnd, device="cuda") * std

    flat = {"params": normal(0.02)}
    if case["master"]:
        flat["masters"] = flat["params"]
    flat["params"] = flat["params"].to(param)
    flat["grads"] = normal(1e-3).to(DTYPES[case["grad"]])
    if case["bits"] == 32:
        flat["exp_avgs"] = normal(3e-4)
        flat["exp_avg_sqs"] = normal(1e-3).square_().add_(1e-7)
    else:
        flat["exp_avgs"] = (normal(32.0).clamp_(-240, 240)).to(torch.float8_e4m3fn)
        flat["exp_avg_sqs"] = (normal(1.0).square_().mul_(8e3).clamp_(max=3e4)).to(torch.float8_e5m2)
        flat["exp_avg_scales"] = torch.full((total // BLOCK,), 2.0 ** -17, device="cuda")
        flat["exp_avg_sq_scales"] = torch.full((total // BLOCK,), 2.0 ** -33, device="cuda")
    lists = {k: _views(v, sizes, BLOCK if k.endswith("scales") else 1) for k, v in flat.items()}
    clip = torch.rand(1, generator=rnd, device="cuda") * 0.5 + 0.5 if case["clip"] else None
    return dict(case=case, flat=flat, lists=lists, grad_scale=clip, seed=1234567890123, step=100, lr=1e-4,
                betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


# ---------------------------------------------------------------------------- one pass


def run(state):
    op = state["case"]["op"]
    if own:
        return dict(route=_own_route, norm=_own_norm, adamw=_own_adamw)[op](state)
    with torch.no_grad():
        return dict(route=_plain_route, norm=_plain_norm, adamw=_plain_adamw)[op](state)


def _own_route(s):
    c = s["case"]
    weights, ids, counts = _entry().route_experts(
        s["logits"], c["top_k"], score=c["score"], bias=s["bias"], num_groups=c["groups"],
        top_groups=c["top_groups"], group_score=c["group_score"], renormalize=c["renorm"], scale=c["scale"],
        valid=s["valid"])
    out = dict(weights=weights, ids=ids, counts=counts)
    if c["train"]:
        (out["d_logits"],) = torch.autograd.grad(weights, s["logits"], s["d_weights"])
    return out


def _plain_route(s):
    c = s["case"]
    k = c["top_k"]
    logits = s["logits"].double()  # 64 bits: the order of near neighbours is the result
    if c["score"] == "sigmoid":
        scores = 1.0 / (1.0 + torch.exp(-logits))
    else:
        e = torch.exp(logits - logits.max(dim=1, keepdim=True).values)
        scores = e / e.sum(dim=1, keepdim=True)
    values = scores if s["bias"] is None else scores + s["bias"].double()
    keys = logits if s["bias"] is None else values  # both scores rise with the logit
    if c["groups"] > 1:
        tokens, experts = logits.shape
        size = experts // c["groups"]
        if c["group_score"] == "max" or size == 1:
            group = keys.view(tokens, c["groups"], size).max(dim=2).values
        else:
            group = torch.sort(values.view(tokens, c["groups"], size), dim=2, descending=True).values[:, :, :2].sum(2)
        best = torch.sort(group, dim=1, descending=True, stable=True).indices[:, :c["top_groups"]]
        open_group = torch.zeros_like(group, dtype=torch.bool).scatter_(1, best, True)
        keys = torch.where(open_group.repeat_interleave(size, dim=1), keys, NEG_INF)
    ids = torch.sort(keys, dim=1, descending=True, stable=True).indices[:, :k]
    chosen = scores.gather(1, ids)
    total = chosen.sum(dim=1, keepdim=True) if c["renorm"] else torch.ones_like(chosen[:, :1])
    share = chosen / total
    weights = share * c["scale"]
    valid = s["valid"]
    if valid is not None:
        weights = torch.where(valid[:, None], weights, 0.0)
        ids = torch.where(valid[:, None], ids, -1)
    flat = ids.reshape(-1)
    counts = torch.bincount(flat[flat >= 0], minlength=logits.shape[1])
    out = dict(weights=weights.float(), ids=ids.int(), counts=counts.int())
    if c["train"]:
        d = s["d_weights"].double() * c["scale"]
        inner = (d * share).sum(dim=1, keepdim=True)
        at = ids.clamp(min=0).long()
        if c["score"] == "sigmoid":
            d_chosen = share * (d - inner) if c["renorm"] else share * d
            d_logits = torch.zeros_like(logits).scatter_(1, at, d_chosen * (1.0 - chosen))
        elif c["renorm"]:
            d_logits = torch.zeros_like(logits).scatter_(1, at, share * (d - inner))
        else:
            d_logits = torch.zeros_like(logits).scatter_(1, at, d * chosen) - scores * inner
        if valid is not None:
            d_logits = torch.where(valid[:, None], d_logits, 0.0)
        out["d_logits"] = d_logits.to(s["logits"].dtype)
    return out


EPS = 1e-6
BRANCH_SCALE = 0.5


def _own_norm(s):
    c = s["case"]
    y, h = _entry().residual_norm(s["x"], s["branch"], post_weight=s["post"], gate=s["gate"],
                                  gate_activation=c["act"], pre_weight=s["pre"], branch_scale=BRANCH_SCALE, eps=EPS)
    out = dict(stream=y, normed=h)
    if c["train"]:
        names = [n for n in ("x", "branch", "post", "pre", "gate") if s[n] is not None]
        outputs, grads = ([y], [s["d_stream"]]) if h is None else ([y, h], [s["d_stream"], s["d_normed"]])
        for n, g in zip(names, torch.autograd.grad(outputs, [s[n] for n in names], grads)):
            out["d_" + n] = g
    return out


def _plain_norm(s):
    c = s["case"]
    x, u = s["x"].float(), s["branch"].float()
    n, r_u, post = u, None, None
    if s["post"] is not None:
        post = s["post"].float()
        r_u = torch.rsqrt((u * u).mean(dim=1, keepdim=True) + EPS)
        n = u * r_u * post
    gate, slope = None, None
    if s["gate"] is not None:
        raw = s["gate"].float()
        if c["act"] == "sigmoid":
            gate = 1.0 / (1.0 + torch.exp(-raw))
            slope = gate * (1.0 - gate)
        elif c["act"] == "tanh":
            gate = torch.tanh(raw)
            slope = 1.0 - gate * gate
        else:
            gate, slope = raw, 1.0
    y = x + BRANCH_SCALE * (n if gate is None else gate * n)
    r_y, pre, h = None, None, None
    if s["pre"] is not None:
        pre = s["pre"].float()
        r_y = torch.rsqrt((y * y).mean(dim=1, keepdim=True) + EPS)
        h = (y * r_y * pre).to(s["branch"].dtype)
    out = dict(stream=y.to(s["x"].dtype), normed=h)
    if c["train"]:
        d_y = s["d_stream"].float()
        if pre is not None:
            d_h = s["d_normed"].float()
            y_hat = y * r_y
            t = d_h * pre
            d_y = d_y + r_y * (t - y_hat * (t * y_hat).mean(dim=1, keepdim=True))
            out["d_pre"] = (d_h * y_hat).sum(dim=0).to(s["pre"].dtype)
        out["d_x"] = d_y.to(s["x"].dtype)
        d_n = BRANCH_SCALE * d_y
        if gate is not None:
            d_gate = d_n * n * slope
            if c["gate"] == "channel":
                d_gate = d_gate.sum(dim=0)
            elif c["gate"] == "token":
                d_gate = d_gate.sum(dim=1, keepdim=True)
            out["d_gate"] = d_gate.to(s["gate"].dtype)
            d_n = d_n * gate
        d_u = d_n
        if post is not None:
            u_hat = u * r_u
            t = d_n * post
            d_u = r_u * (t - u_hat * (t * u_hat).mean(dim=1, keepdim=True))
            out["d_post"] = (d_n * u_hat).sum(dim=0).to(s["post"].dtype)
        out["d_branch"] = d_u.to(s["branch"].dtype)
    return out


def _own_adamw(s):
    lists = s["lists"]
    _entry().adamw_step(lists["params"], lists["grads"], lists["exp_avgs"], lists["exp_avg_sqs"], step=s["step"],
                        lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["weight_decay"],
                        exp_avg_scales=lists.get("exp_avg_scales"), exp_avg_sq_scales=lists.get("exp_avg_sq_scales"),
                        masters=lists.get("masters"), grad_scale=s["grad_scale"], seed=s["seed"])
    return {k: v for k, v in s["flat"].items() if k != "grads"}


def _plain_adamw(s):
    lists = s["lists"]
    _ = [_plain_adamw_tensor(s, i) for i in range(len(lists["params"]))]
    return {k: v for k, v in s["flat"].items() if k != "grads"}


def _plain_adamw_tensor(s, i):
    t = {k: v[i] for k, v in s["lists"].items()}
    (b1, b2), step = s["betas"], s["step"]
    g = t["grads"].float()
    if s["grad_scale"] is not None:
        g = g * s["grad_scale"]
    if "exp_avg_scales" in t:
        m = t["exp_avgs"].float() * _spread_scales(t["exp_avg_scales"], g)
        v = t["exp_avg_sqs"].float() * _spread_scales(t["exp_avg_sq_scales"], g)
    else:
        m, v = t["exp_avgs"], t["exp_avg_sqs"]
    m = m * b1 + g * (1.0 - b1)
    v = v * b2 + (g * g) * (1.0 - b2)
    main = t.get("masters", t["params"])
    denom = torch.sqrt(v) * (1.0 / math.sqrt(1.0 - b2 ** step)) + s["eps"]
    p = main.float() * (1.0 - s["lr"] * s["weight_decay"]) - (m / denom) * (s["lr"] / (1.0 - b1 ** step))
    main.copy_(p)
    if main is not t["params"]:
        t["params"].copy_(p)
    if "exp_avg_scales" not in t:
        t["exp_avgs"].copy_(m)
        t["exp_avg_sqs"].copy_(v)
        return
    noise = _noise(g.numel(), i, step, s["seed"], g.device)
    _store8(m, noise >> 16, t["exp_avgs"], t["exp_avg_scales"], mantissa=3, bias=7, top=7)
    _store8(v, noise & 0xFFFF, t["exp_avg_sqs"], t["exp_avg_sq_scales"], mantissa=2, bias=15, top=14)


def _spread_scales(scales, like):
    return scales[:, None].expand(-1, BLOCK).reshape(-1)[: like.numel()]


def _noise(n, tensor, step, seed, device):
    """A 32-bit word for each element: Philox4x32 of 7 rounds, counter (element / 4, tensor, step), key the seed."""
    low = 0xFFFFFFFF
    c0 = torch.arange(-(-n // 4), dtype=torch.int64, device=device)
    c1, c2, c3 = c0 >> 32, torch.full_like(c0, tensor), torch.full_like(c0, step & low)
    c0 = c0 & low
    k0, k1 = seed & low, (seed >> 32) & low
    for _ in range(7):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57  # wraps like the unsigned product: both halves are right
        c0, c1, c2, c3 = ((b >> 32) & low) ^ c1 ^ k0, b & low, ((a >> 32) & low) ^ c3 ^ k1, a & low
        k0, k1 = (k0 + 0x9E3779B9) & low, (k1 + 0xBB67AE85) & low
    return torch.stack((c0, c1, c2, c3), dim=1).reshape(-1)[:n]


def _power(exponent):
    """2 ** exponent in float32 from its bits, exact for -126 to 127."""
    return ((exponent.int() + 127) << 23).view(torch.float32)


def _store8(x, noise16, codes, scales, mantissa, bias, top):
    """Rounds x to 8-bit floats of ``mantissa`` bits, up with the probability that keeps the mean. A block's
    scale is the power of two that puts its largest finite magnitude into binade ``top``."""
    n = x.numel()
    finite = torch.isfinite(x)
    size = torch.where(finite, x.abs(), 0.0)
    padded = torch.zeros(scales.numel() * BLOCK, device=x.device)
    padded[:n] = size
    largest = padded.view(-1, BLOCK).max(dim=1).values
    exponent = (torch.frexp(largest).exponent - 1).clamp(min=-112)
    scales.copy_(torch.where(largest > 0, _power(exponent - top), 1.0))
    size = size * _spread_scales(_power(top - exponent), x)
    binade = (torch.frexp(size).exponent - 1).clamp(min=1 - bias)
    binade = torch.where(size > 0, binade, 1 - bias)
    steps = torch.floor(size * _power(mantissa - binade) + noise16.float() * 2.0 ** -16).int()
    code = ((binade + bias) << mantissa) + steps - (1 << mantissa)
    code = torch.where(finite, code, 0x7F) | torch.where(torch.signbit(x), 0x80, 0)
    codes.view(torch.uint8).copy_(code.to(torch.uint8))


# ---------------------------------------------------------------------------- work


def work(case):
    size = {"float32": 4, "bfloat16": 2, "float16": 2}
    if case["op"] == "route":
        t, e, k = case["tokens"], case["experts"], case["top_k"]
        matrix = t * e * size[case["dtype"]]
        n = matrix + 8 * t * k + 4 * e + (4 * e if case["bias"] else 0) + (t if case["masked"] else 0)
        if case["train"]:
            n += matrix + 4 * t * k
        return {"bytes": n, "flops": t * e * (20 if case["train"] else 12)}
    if case["op"] == "norm":
        t, d = case["tokens"], case["dim"]
        x, u = t * d * size[case["stream"]], t * d * size[case["branch"]]
        weights = 4 * d * (case["post"] + case["pre"])
        gate = dict(none=0, channel=4 * d, token=4 * t, full=u)[case["gate"]]
        n = 2 * x + u + weights + gate + (u if case["pre"] else 0)
        if case["train"]:  # each output's gradient in, each input's out
            n += 2 * x + u + weights + gate + (u if case["pre"] else 0)
        return {"bytes": n, "flops": t * d * (40 if case["train"] else 12)}
    n = sum(_sizes(case))
    per = 2 * size[case["param"]] + size[case["grad"]] + (16 if case["bits"] == 32 else 4 + 16 / BLOCK)
    if case["master"]:
        per += 8 - size[case["param"]]
    return {"bytes": n * per, "flops": 16 * n}


# ---------------------------------------------------------------------------- from the definitions, in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return dict(route=_exact_route, norm=_exact_norm, adamw=_exact_adamw)[case["op"]](state)


def _exact_route(s):
    """Selection by repeated maxima, gradient by differentiation of the weights' definition."""
    c = s["case"]
    logits = s["logits"].detach().double().requires_grad_(True)
    scores = torch.sigmoid(logits) if c["score"] == "sigmoid" else torch.softmax(logits, dim=1)
    with torch.no_grad():
        ranked = scores.clone() if s["bias"] is None else scores + s["bias"].double()
        tokens, experts = ranked.shape
        place = torch.arange(experts, device=ranked.device)

        def first_best(values):
            best = values.amax(dim=1, keepdim=True)
            return torch.where(values == best, place[: values.shape[1]], values.shape[1]).amin(dim=1)

        if c["groups"] > 1:
            parts = ranked.reshape(tokens * c["groups"], -1).clone()
            first = parts.amax(dim=1)
            value = first.clone()
            if c["group_score"] == "top2" and parts.shape[1] > 1:
                parts.scatter_(1, first_best(parts)[:, None], NEG_INF)
                value += parts.amax(dim=1)
            value = value.reshape(tokens, c["groups"])
            member = place // (experts // c["groups"])
            allowed = torch.zeros_like(ranked, dtype=torch.bool)
            for _ in range(c["top_groups"]):
                g = first_best(value)[:, None]
                allowed |= member[None, :] == g
                value.scatter_(1, g, NEG_INF)
            ranked = ranked.masked_fill(~allowed, NEG_INF)
        picks = []
        for _ in range(c["top_k"]):
            picks.append(first_best(ranked))
            ranked.scatter_(1, picks[-1][:, None], NEG_INF)
        picks = torch.stack(picks, dim=1)
    weights = scores.gather(1, picks)
    if c["renorm"]:
        weights = weights / weights.sum(dim=1, keepdim=True)
    weights = weights * c["scale"]
    if s["valid"] is not None:
        weights = weights * s["valid"][:, None]
    out = dict(weights=weights.detach(), ids=None, counts=None)
    if c["train"]:
        (out["d_logits"],) = torch.autograd.grad(weights, logits, s["d_weights"].double())
    return out


def _exact_norm(s):
    c = s["case"]
    leaf = {n: s[n].detach().double().requires_grad_(True) for n in ("x", "branch", "post", "pre", "gate")
            if s[n] is not None}

    def normed(t, weight):
        return t / torch.sqrt(torch.mean(t ** 2, dim=-1, keepdim=True) + EPS) * weight

    inner = normed(leaf["branch"], leaf["post"]) if "post" in leaf else leaf["branch"]
    if "gate" in leaf:
        act = dict(none=lambda t: t, sigmoid=torch.sigmoid, tanh=torch.tanh)[c["act"]]
        inner = act(leaf["gate"]) * inner
    y = leaf["x"] + BRANCH_SCALE * inner
    h = normed(y, leaf["pre"]) if "pre" in leaf else None
    out = dict(stream=y.detach(), normed=None if h is None else h.detach())
    if c["train"]:
        value = (y * s["d_stream"].double()).sum()
        if h is not None:
            value = value + (h * s["d_normed"].double()).sum()
        for n, g in zip(leaf, torch.autograd.grad(value, list(leaf.values()))):
            out["d_" + n] = g
    return out


def _exact_adamw(s):
    f, sizes = s["flat"], _sizes(s["case"])
    (b1, b2), step = s["betas"], s["step"]
    starts = np.cumsum([0] + [-(-n // BLOCK) * BLOCK for n in sizes])
    inside = torch.zeros(int(starts[-1]), dtype=torch.bool, device="cuda")
    for a, n in zip(starts, sizes):
        inside[int(a):int(a) + n] = True
    g = f["grads"].double()
    if s["grad_scale"] is not None:
        g *= s["grad_scale"].double()
    m, v = f["exp_avgs"].double(), f["exp_avg_sqs"].double()
    eight = s["case"]["bits"] == 8
    if eight:
        m = (m.view(-1, BLOCK) * f["exp_avg_scales"].double()[:, None]).view(-1)
        v = (v.view(-1, BLOCK) * f["exp_avg_sq_scales"].double()[:, None]).view(-1)
    new_m, new_v = torch.lerp(m, g, 1.0 - b1), torch.lerp(v, g ** 2, 1.0 - b2)
    old = f["masters" if "masters" in f else "params"].double()
    root = torch.sqrt(new_v / (1.0 - b2 ** step))
    new = old * (1.0 - s["lr"] * s["weight_decay"]) - s["lr"] * (new_m / (1.0 - b1 ** step)) / (root + s["eps"])
    new = torch.where(inside, new, old)
    out = {"params": torch.where(inside, new, f["params"].double())}
    if "masters" in f:
        out["masters"] = new
    if not eight:
        out["exp_avgs"], out["exp_avg_sqs"] = torch.where(inside, new_m, m), torch.where(inside, new_v, v)
        return out
    # the codes hang on the noise words, the scales on which side of a power of two a rounded maximum
    # falls: neither is a rounding of a value that 64 bits give
    for name in ("exp_avgs", "exp_avg_sqs", "exp_avg_scales", "exp_avg_sq_scales"):
        out[name] = None
    return out


if __name__ == "__main__":
    for one in listed() + [draw(random.Random(i)) for i in range(6)]:
        print(one, work(one))
