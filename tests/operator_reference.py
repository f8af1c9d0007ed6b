"""The operators of the quantized layers in 64 bits, on the CPU, straight from their definitions."""
import math

import numpy as np
import torch

LARGEST = torch.finfo(torch.float32).max
HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
SMALLEST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def route(logits, k, score="softmax", bias=None, groups=1, keep=None, group_score="max", renormalise=True, scale=1.0):
    """(ids, weights in fp64), one token at a time."""
    rows = logits.detach().double().cpu().numpy().reshape(-1, logits.shape[-1])
    E = rows.shape[1]
    b = np.zeros(E) if bias is None else bias.double().cpu().numpy()
    keep = groups if keep is None else keep
    ids, weights = np.full((len(rows), k), -1, dtype=np.int64), np.zeros((len(rows), k))
    for t, raw in enumerate(rows):
        l = np.minimum(np.where(np.isnan(raw), -math.inf, raw), LARGEST)
        real = [e for e in range(E) if l[e] > -math.inf]
        s = np.zeros(E)
        if score == "sigmoid":
            for e in real:
                s[e] = 1 / (1 + math.exp(-l[e])) if l[e] > -700 else 0.0
        elif real:
            top = max(l[e] for e in real)
            for e in real:
                s[e] = math.exp(l[e] - top)
            s /= s.sum()
        can = [e for e in real if not math.isnan(b[e]) and b[e] > -math.inf]
        value = {e: s[e] + b[e] for e in can}
        order = {e: (value[e] if bias is not None else l[e]) for e in can}
        if groups > 1:
            size = E // groups
            of = []
            # largest values without a bias: in the order of the logits, also where the scores are below the smallest number
            worth = order if group_score == "max" else value
            for g in range(groups):
                v = sorted((worth[e] for e in can if e // size == g), reverse=True)
                of.append(sum(v[:2] if group_score == "top2" else v[:1]) if v else -math.inf)
            kept = sorted(range(groups), key=lambda g: (-of[g], g))[:keep]
            can = [e for e in can if e // size in kept]
        chosen = sorted(can, key=lambda e: (-order[e], e))[:k]
        ids[t, : len(chosen)] = chosen
        if renormalise and chosen:
            # without the common factor, which may be below the smallest number
            if score == "softmax":
                top = max(l[e] for e in chosen)
                w = np.array([math.exp(l[e] - top) for e in chosen])
            else:
                m = min(0.0, max(l[e] for e in chosen))
                w = np.array([1 / (math.exp(m) + math.exp(m - l[e])) if m - l[e] < 700 else 0.0 for e in chosen])
            w = w / w.sum()
        else:
            w = s[chosen]
        weights[t, : len(chosen)] = w * scale
    return torch.from_numpy(ids.reshape(*logits.shape[:-1], k)), torch.from_numpy(weights.reshape(*logits.shape[:-1], k))


def plan(ids, n, first=0):
    flat = ids.cpu().numpy().reshape(-1).astype(np.int64) - first
    by_expert = [[i for i, e in enumerate(flat) if e == x] for x in range(n)]
    order = [i for group in by_expert for i in group]
    offsets = np.concatenate([[0], np.cumsum([len(g) for g in by_expert])])
    place = np.full(flat.size, -1)
    for at, i in enumerate(order):
        place[i] = at
    return offsets, np.array(order + [-1] * (flat.size - len(order)), dtype=np.int64), place.reshape(tuple(ids.shape))


def codes(x):
    """(codes, scale) of each row in fp64; rows with an infinity or a NaN: codes 0, scale NaN."""
    x = x.double()
    top = x.abs().amax(-1, keepdim=True)
    good = torch.isfinite(x).all(-1, keepdim=True)
    q = torch.round(127 * x / torch.where(top > 0, top, torch.ones_like(top)))
    q = torch.where(good, q, torch.zeros_like(q))
    return q, torch.where(good, top / 127, torch.full_like(top, math.nan))[..., 0]


def product_bound(y, product, dtype):
    """How far int8_matmul may be from y = product + bias: the sum of integers is exact; its conversion to fp32, the scale of
    the token, two products and the sum with the bias are one rounding each (2^-24 of what they give, the last of y), and the result's own."""
    return HALF_STEP[dtype] * 1.01 * y.abs() + 2.0 ** -24 * (4.1 * product.abs() + 1.1 * y.abs()) + SMALLEST[dtype]


def experts(x, ids, weights, gate_up, gate_up_scale, down, down_scale, first=0):
    """(y, bound) of int8_experts, both fp64.

    bound: h has a relative error of 4 roundings each for gate and up, the exponential (2 steps, and its argument's 4 roundings times
    |gate|), sum, division and two products: less than (16 + 5 |gate|) 2^-24.  Its code is then off by at most 127 times that relative error (plus as
    much again for the largest value's): where the exact quotient lies nearer to a middle, the code may differ by one, and the
    result by that times the weights' scales.  The sum of a pair's products may be kept in fp16 scaled by powers of two: to 2^-11, or,
    below fp16's normal range, to 2^-25 of 2^k p, with 2^k < I the power that brings 127 * 128 * I to 2^15 and p <= 2 max(scales of the
    32 columns), so to 2^-24 I max(scales); the rest are fp32 roundings and the result's own."""
    T, k = ids.shape
    E, I = gate_up.shape[0], gate_up.shape[1] // 2
    q, s = codes(x.cpu())
    ids, weights = ids.cpu(), weights.double().cpu()
    y, bound = torch.zeros(T, x.shape[-1], dtype=torch.float64), torch.zeros(T, x.shape[-1], dtype=torch.float64)
    for e in range(E):
        token, slot = torch.nonzero(ids == e + first, as_tuple=True)
        if not len(token):
            continue
        both = q[token] @ gate_up[e].double().cpu().t() * s[token, None] * gate_up_scale[e].double().cpu()
        g, u = both[:, :I], both[:, I:]
        h = g * torch.sigmoid(g) * u
        hq, hs = codes(h)
        top = 127 * hs[:, None]
        exact = 127 * h / torch.where(top > 0, top, torch.ones_like(top))
        near = (exact - exact.floor() - 0.5).abs() <= 127 * 2 * (16 + 5 * g.abs().clamp(max=200)) * 2.0 ** -24
        d, ds = down[e].double().cpu(), down_scale[e].double().cpu()
        w = weights[token, slot, None]
        part = hq @ d.t() * hs[:, None] * ds * w
        flips = near.double() @ d.abs().t() * hs[:, None] * ds.abs() * w.abs()
        near_scales = torch.nn.functional.pad(ds.abs(), (0, -len(ds) % 32)).view(-1, 32).amax(1).repeat_interleave(32)[: len(ds)]
        floor = 2.0 ** -24 * I * near_scales * hs[:, None] * w.abs()
        y.index_add_(0, token, part)
        bound.index_add_(0, token, flips + part.abs() * (2.0 ** -11 + (60 + 5 * 60) * 2.0 ** -24) + floor + 1e-40)
    return y, bound + HALF_STEP[x.dtype] * 1.01 * (y.abs() + bound) + SMALLEST[x.dtype]
