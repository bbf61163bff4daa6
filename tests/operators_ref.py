"""Plain float64 (and, for the 8-bit moments, bit-exact float32) forms of ``route_experts``,
``residual_norm`` and ``adamw_step`` for the tests, written from their definitions."""

import math

import numpy as np
import torch

NEG = -math.inf


# ------------------------------------------------------------------ routing
def _rank_key(v):
    """NaN before everything, then falling."""
    return (0, 0.0) if math.isnan(v) else (1, -v)


def route_row(row, k, score, bias, groups, top_groups, group_score):
    """(ids, scores of all experts) of one row of python floats, by the definition."""
    E = len(row)
    if score == "sigmoid":
        s = [math.nan if math.isnan(l) else (1.0 / (1.0 + math.exp(-l)) if l > -700 else math.exp(l)) for l in row]
    else:
        t = torch.softmax(torch.tensor(row, dtype=torch.float64), dim=0)
        s = t.tolist()
    key = list(row) if bias is None else [si + b for si, b in zip(s, bias)]
    val = s if bias is None else key
    masked = [l == NEG or (bias is not None and bias[e] == NEG) for e, l in enumerate(row)]
    open_ = [True] * E
    size = E // groups
    if groups > 1:
        values = []
        for g in range(groups):
            here = [e for e in range(g * size, (g + 1) * size) if not masked[e]]
            use = val if group_score == "top2" and size > 1 else key
            best = sorted((use[e] for e in here), key=_rank_key)
            if not here:
                values.append(NEG)
            elif group_score == "top2" and size > 1:
                values.append(math.nan if any(math.isnan(b) for b in best) else sum(best[:2]))
            else:
                values.append(best[0])
        order = sorted(range(groups), key=lambda g: (_rank_key(values[g]), g))
        chosen = set(order[:top_groups])
        open_ = [e // size in chosen for e in range(E)]
    left = [e for e in range(E) if open_[e] and not masked[e]]
    ids = sorted(left, key=lambda e: (_rank_key(key[e]), e))[:k]
    return ids + [-1] * (k - len(ids)), s


def route(logits, k, score="softmax", bias=None, groups=1, top_groups=1, group_score="top2", renorm=True, scale=1.0,
          valid=None, d_w=None):
    """(weights, ids, counts[, d_logits]) in float64 on the CPU."""
    l = logits.detach().double().cpu()
    T, E = l.shape
    b = None if bias is None else bias.double().cpu().tolist()
    ids = []
    for t in range(T):
        if valid is not None and not bool(valid[t]):
            ids.append([-1] * k)
        else:
            ids.append(route_row(l[t].tolist(), k, score, b, groups, top_groups, group_score)[0])
    ids = torch.tensor(ids, dtype=torch.long).view(T, k)
    leaf = l.clone().requires_grad_(True)
    has = ids >= 0
    got = leaf.gather(1, ids.clamp(min=0)) if T else leaf[:, :1].expand(0, k)
    if renorm:  # in logs: the ratio is defined where the scores themselves underflow
        logs = torch.nn.functional.logsigmoid(got) if score == "sigmoid" else got
        share = torch.softmax(logs.masked_fill(~has, NEG), dim=1)
    elif score == "sigmoid":
        share = torch.sigmoid(got)
    else:
        share = torch.softmax(leaf, dim=1).gather(1, ids.clamp(min=0))
    w = torch.where(has, share * scale, 0.0)
    counts = torch.bincount(ids[has].reshape(-1), minlength=E)
    if d_w is None:
        return w.detach(), ids, counts
    picked = torch.where(has, w, 0.0)
    (g,) = torch.autograd.grad(picked, leaf, torch.where(has, d_w.double().cpu(), 0.0))
    return w.detach(), ids, counts, torch.nan_to_num(g) if not torch.isfinite(l).all() else g


# ------------------------------------------------------------------ norms
def norm(x, branch=None, post=None, gate=None, act="none", pre=None, rs=1.0, bs=1.0, eps=1e-6):
    """(y, h) in float64, differentiable."""
    def rms(t, w):
        return t * torch.rsqrt(t.square().mean(dim=-1, keepdim=True) + eps) * w

    if branch is None:
        return x, rms(x, pre)
    n = branch if post is None else rms(branch, post)
    if gate is not None:
        n = dict(none=lambda t: t, sigmoid=torch.sigmoid, tanh=torch.tanh)[act](gate) * n
    y = rs * x + bs * n
    return y, None if pre is None else rms(y, pre)


# ------------------------------------------------------------------ AdamW
def philox7(c0, c1, c2, c3, seed):
    """Words [4, n] of Philox4x32-7 for uint64 counter arrays holding 32-bit values."""
    mask = np.uint64(0xFFFFFFFF)
    c = [np.asarray(v, dtype=np.uint64) & mask for v in np.broadcast_arrays(c0, c1, c2, c3)]
    k0, k1 = seed & 0xFFFFFFFF, (seed >> 32) & 0xFFFFFFFF
    for _ in range(7):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        s = np.uint64(32)
        c = [(b >> s) ^ c[1] ^ np.uint64(k0), b & mask, (a >> s) ^ c[3] ^ np.uint64(k1), a & mask]
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    return np.stack(c)


def noise(n, tensor, step, seed):
    q = np.arange(-(-n // 4), dtype=np.uint64)
    return philox7(q, q >> np.uint64(32), tensor, step, seed).T.reshape(-1)[:n].astype(np.uint32)


def encode8(x, noise16, mantissa, bias, top):
    """(codes uint8 [n], scales float32 [blocks]) of a float32 array by the definition, value by value in float64."""
    n = x.size
    blocks = -(-n // 256)
    codes, scales = np.zeros(n, np.uint8), np.ones(blocks, np.float32)
    for b in range(blocks):
        part = x[b * 256:(b + 1) * 256]
        size = np.where(np.isfinite(part), np.abs(part.astype(np.float64)), 0.0)
        big = size.max(initial=0.0)
        e = max(math.frexp(big)[1] - 1, -112) if big > 0 else -112
        if big > 0:
            scales[b] = 2.0 ** (e - top)
        for i, (v, a) in enumerate(zip(part, size)):
            sign = 0x80 if np.signbit(v) else 0
            if not np.isfinite(v):
                codes[b * 256 + i] = 0x7F | sign
                continue
            a = np.float64(a) * 2.0 ** (top - e) if big > 0 else 0.0
            be = max(math.frexp(a)[1] - 1, 1 - bias) if a > 0 else 1 - bias
            # the sum is rounded to float32 as the definition has it
            steps = int(math.floor(np.float32(np.float32(a * 2.0 ** (mantissa - be)) +
                                              np.float32(int(noise16[b * 256 + i]) * 2.0 ** -16))))
            codes[b * 256 + i] = ((be + bias) << mantissa) + steps - (1 << mantissa) | sign
    return codes, scales


def adamw32(p, g, m, v, step, lr, betas, eps, wd, grad_scale=1.0):
    """(p, m, v) in float64."""
    g = g.double() * grad_scale
    m = betas[0] * m.double() + (1 - betas[0]) * g
    v = betas[1] * v.double() + (1 - betas[1]) * g * g
    upd = (m / (1 - betas[0] ** step)) / ((v / (1 - betas[1] ** step)).sqrt() + eps)
    return p.double() * (1 - lr * wd) - lr * upd, m, v


def moments_f32(g, m, v, betas, grad_scale=None):
    """The new moments with float32 roundings after every product and sum (numpy float32 arrays)."""
    f = np.float32
    with np.errstate(all="ignore"):
        if grad_scale is not None:
            g = g * f(grad_scale)
        return m * f(betas[0]) + g * f(1 - betas[0]), v * f(betas[1]) + (g * g) * f(1 - betas[1])
