"""The operators of a quantized mixture-of-experts layer, as they are timed: routing tokens to experts with
the plan that groups them, the product in 8-bit integers, and the experts' gated MLPs in 8-bit integers.

`GPTQ(layer, None, ...).quantize(8)` leaves codes of 8 bits with one scale per output channel.  The integer
product multiplies them with activations that get 8-bit codes and one scale per token on the fly.  Definitions
(all of it in exact arithmetic, the result rounded once):

  codes of a token x       scale = max|x| / 127,  code_j = round_half_even(127 x_j / max|x|);  zeros for a zero token
  product                  y[t, n] = (sum_k code[t, k] w[n, k]) scale[t] w_scale[n] + bias[n]
  experts                  h[p] = silu(gate product) * up product of the pair's token, codes of h[p] as above,
                           y[t] = sum over the token's local pairs p of weight[p] * down product of h[p]
  routing                  score = sigmoid(logit) or softmax(logits);  value = score + bias;  groups of experts are
                           kept by the sum of their two largest values or by the largest, then the top_k largest values of
                           the kept groups, ties to the lowest index;  weights are the scores (without bias), divided by their
                           sum where asked, times a factor.  An expert whose logit is -inf or NaN, or whose bias is -inf, is
                           never chosen; where too few are left the expert is -1 and the weight 0
  plan                     pairs (token * top_k + slot) in the order of (expert, pair): offsets per expert, the pairs in
                           order, and the place of each pair (-1: not one of these experts)
"""
import math

import numpy as np
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
LARGEST = torch.finfo(torch.float32).max


def listed():
    return [
        # one decoded token: routing is all latency
        {"name": "route_one_token", "kind": "route", "tokens": 1, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "keep": 4, "group_score": "top2", "renormalise": True, "scale": 2.5, "dtype": "fp32", "left_out": 0, "padded": 0.0},
        # a calibration sequence with padding at its end, softmax scores in the model's type, some experts switched off
        {"name": "route_padded_softmax", "kind": "route", "tokens": 4093, "experts": 60, "top_k": 6, "score": "softmax", "bias": False, "groups": 1,
         "keep": 1, "group_score": "max", "renormalise": False, "scale": 1.0, "dtype": "bf16", "left_out": 0, "padded": 0.1},
        # sixteen sequences of 4096 tokens at once
        {"name": "route_65536_grouped", "kind": "route", "tokens": 65536, "experts": 256, "top_k": 8, "score": "sigmoid", "bias": True, "groups": 8,
         "keep": 4, "group_score": "top2", "renormalise": True, "scale": 2.5, "dtype": "fp32", "left_out": 3, "padded": 0.0},
        # decoding: one token through gate_proj of an expert, bound by its weights
        {"name": "int8_one_token", "kind": "matmul", "tokens": 1, "rows": 2048, "cols": 7168, "bias": False, "dtype": "bf16"},
        # a ragged handful of tokens through down_proj, sizes that fill no tile
        {"name": "int8_37_tokens", "kind": "matmul", "tokens": 37, "rows": 7168, "cols": 2048, "bias": True, "dtype": "fp16"},
        # an fp32 layer whose sizes divide nothing
        {"name": "int8_ragged_fp32", "kind": "matmul", "tokens": 1011, "rows": 1001, "cols": 1064, "bias": True, "dtype": "fp32"},
        # a calibration sequence through gate_proj
        {"name": "int8_4096_tokens", "kind": "matmul", "tokens": 4096, "rows": 2048, "cols": 7168, "bias": False, "dtype": "bf16"},
        # two sequences through o_proj, the widest layer of a block
        {"name": "int8_8192_wide", "kind": "matmul", "tokens": 8192, "rows": 7168, "cols": 16384, "bias": False, "dtype": "bf16"},
        # one decoded token whose eight experts are all here
        {"name": "experts_one_token", "kind": "experts", "tokens": 1, "experts": 32, "total": 32, "first": 0, "top_k": 8, "hidden": 7168,
         "inner": 2048, "dtype": "bf16"},
        # a decoding batch on one of eight ranks, which holds 32 of 256 experts
        {"name": "experts_64_tokens", "kind": "experts", "tokens": 64, "experts": 32, "total": 256, "first": 96, "top_k": 8, "hidden": 7168,
         "inner": 2048, "dtype": "bf16"},
        # a small block's experts
        {"name": "experts_small_block", "kind": "experts", "tokens": 333, "experts": 8, "total": 8, "first": 0, "top_k": 2, "hidden": 256,
         "inner": 128, "dtype": "fp16"},
        # four calibration sequences on one of eight ranks
        {"name": "experts_16384_tokens", "kind": "experts", "tokens": 16384, "experts": 32, "total": 256, "first": 32, "top_k": 8, "hidden": 7168,
         "inner": 2048, "dtype": "bf16"},
    ]


def _log_uniform(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    kind = rng.choice(["route", "matmul", "experts"])
    if kind == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * _log_uniform(rng, max(1, 8 // groups), 512 // groups)
        keep = rng.randint(max(1, groups // 2), groups)
        tokens = min(_log_uniform(rng, 1, 65536), 65536 * 256 // experts)
        return {"kind": kind, "tokens": tokens, "experts": experts, "top_k": rng.randint(1, min(8, experts // groups * keep)),
                "score": rng.choice(["sigmoid", "softmax"]), "bias": rng.random() < 0.5, "groups": groups, "keep": keep,
                "group_score": rng.choice(["top2", "max"]), "renormalise": rng.random() < 0.5, "scale": rng.choice([1.0, 2.5]),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "left_out": rng.choice([0, 0, 2]), "padded": rng.choice([0.0, 0.0, 0.2])}
    if kind == "matmul":
        rows, cols = _log_uniform(rng, 64, 16384), 8 * _log_uniform(rng, 8, 2048)
        tokens = max(1, min(_log_uniform(rng, 1, 16384), 8192 * 7168 * 16384 // (rows * cols)))
        return {"kind": kind, "tokens": tokens, "rows": rows, "cols": cols, "bias": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    experts, ranks = rng.randint(1, 32), rng.choice([1, 2, 4, 8])
    hidden, inner = 8 * _log_uniform(rng, 8, 896), 8 * _log_uniform(rng, 8, 256)
    total = experts * ranks
    top_k = rng.randint(1, min(8, total))
    fewest = 1 if ranks == 1 else -(-8 * ranks // top_k)      # some of them meet an expert of this rank
    tokens = max(fewest, min(_log_uniform(rng, 1, 16384), 16384 * ranks // top_k))
    return {"kind": kind, "tokens": tokens, "experts": experts, "total": total, "first": experts * rng.randrange(ranks), "top_k": top_k,
            "hidden": hidden, "inner": inner, "dtype": rng.choice(["bf16", "fp16"])}


def _device():
    return torch.device("cuda" if torch.cuda.is_available() else "cpu")


def _generator(seed):
    g = torch.Generator(device=_device())
    g.manual_seed(seed)
    return g


def _tokens(shape, dtype, g):
    """Activations: N(0,1) with a factor per channel, which gives outlier channels."""
    channels = torch.exp(0.5 * torch.randn(shape[-1], generator=g, device=_device()))
    return (torch.randn(shape, generator=g, device=_device()) * channels).to(dtype)


def _weights(shape, g):
    """8-bit codes of N(0,1) weights on an absmax grid (about 3.7 standard deviations to the border) in rows 16 bytes apart or a
    multiple of it, and their scales."""
    *lead, cols = shape
    codes = torch.zeros(*lead, -(-cols // 16) * 16, dtype=torch.int8, device=_device())
    for part in codes if len(lead) > 1 else [codes]:
        part[..., :cols] = (34.0 * torch.randn(*part.shape[:-1], cols, generator=g, device=_device())).round_().clamp_(-128, 127).to(torch.int8)
    scale = (0.02 * 3.7 / 127) * torch.exp(0.2 * torch.randn(lead, generator=g, device=_device()))
    return codes[..., :cols], scale


def prepare(case, seed):
    g, dev, kind = _generator(seed), _device(), case["kind"]
    dtype = DTYPES[case["dtype"]]
    if kind == "route":
        T, E = case["tokens"], case["experts"]
        logits = torch.randn(T, E, generator=g, device=dev) + 0.5 * torch.randn(E, generator=g, device=dev)
        bias = 0.1 * torch.randn(E, generator=g, device=dev) if case["bias"] else None
        if case["left_out"]:
            out = torch.randperm(E, generator=g, device=dev)[: min(case["left_out"], E - 1)]
            if bias is not None:
                bias[out] = -math.inf
            else:
                logits[:, out] = -math.inf
        n_padded = int(case["padded"] * T)
        if n_padded:
            logits[T - n_padded:] = -math.inf
        return {"case": case, "logits": logits.to(dtype), "bias": bias}
    if kind == "matmul":
        x = _tokens((case["tokens"], case["cols"]), dtype, g)
        codes, scale = _weights((case["rows"], case["cols"]), g)
        bias = torch.randn(case["rows"], generator=g, device=dev) if case["bias"] else None
        return {"case": case, "x": x, "codes": codes, "scale": scale, "bias": bias}
    T, E, k = case["tokens"], case["experts"], case["top_k"]
    x = _tokens((T, case["hidden"]), dtype, g)
    gate_up, gate_up_scale = _weights((E, 2 * case["inner"], case["hidden"]), g)
    down, down_scale = _weights((E, case["hidden"], case["inner"]), g)
    score = torch.sigmoid(torch.randn(T, case["total"], generator=g, device=dev) + 0.3 * torch.randn(case["total"], generator=g, device=dev))
    weights, ids = score.topk(k, dim=-1)
    return {"case": case, "x": x, "ids": ids.to(torch.int32), "weights": weights / weights.sum(-1, keepdim=True), "gate_up": gate_up,
            "gate_up_scale": gate_up_scale, "down": down, "down_scale": down_scale}


# ---------------------------------------------------------------- the plain form
def _plain_route(s):
    c, bias = s["case"], s["bias"]
    T, E, k, groups = c["tokens"], c["experts"], c["top_k"], c["groups"]
    # in 64 bits: values next to one another decide which expert is chosen
    logits = s["logits"].double().clamp(max=LARGEST)
    out = logits.isnan() | (logits == -math.inf)
    logits = logits.masked_fill(out, -math.inf)
    if c["score"] == "sigmoid":
        score = 1.0 / (1.0 + torch.exp(-logits))
    else:
        top = logits.amax(-1, keepdim=True)
        e = torch.exp(logits - top.masked_fill(top == -math.inf, 0.0))
        score = e / e.sum(-1, keepdim=True).clamp(min=1e-300)
    value = score
    if bias is not None:
        value = score + bias.double()
        out = out | (bias == -math.inf)
    value = value.masked_fill(out, -math.inf)
    by = value if bias is not None else logits      # without a bias the logits order the scores
    if groups > 1:
        v = value.view(T, groups, E // groups)
        best = torch.sort(v, dim=-1, descending=True)[0]
        of_group = best[..., 0]
        if c["group_score"] == "top2" and best.shape[-1] > 1:
            of_group = torch.where(best[..., 1] == -math.inf, best[..., 0], best[..., 0] + best[..., 1])
        kept = torch.sort(of_group, dim=-1, descending=True, stable=True)[1][:, : c["keep"]]
        keep = torch.zeros(T, groups, dtype=torch.bool, device=v.device).scatter_(1, kept, True)
        by = by.view(T, groups, -1).masked_fill(~keep[..., None], -math.inf).view(T, E)
    by, ids = torch.sort(by, dim=-1, descending=True, stable=True)
    none = by[:, :k] == -math.inf
    ids = ids[:, :k]
    w = score.gather(1, ids).masked_fill(none, 0.0)
    if c["renormalise"]:
        w = w / w.sum(-1, keepdim=True).clamp(min=1e-300)
    ids = ids.masked_fill(none, -1)
    # the plan: a stable sort by expert, those without one at the end
    P = T * k
    e = ids.reshape(-1)
    e = torch.where(e < 0, E, e)
    order = torch.sort(e, stable=True)[1]
    counts = torch.bincount(e, minlength=E + 1)
    offsets = torch.cat([counts.new_zeros(1), counts[:E].cumsum(0)])
    at = torch.arange(P, device=e.device)
    inside = at < offsets[E]
    place = torch.empty_like(at)
    place[order] = torch.where(inside, at, -1)
    return {"ids": ids.to(torch.int32), "weights": (w * c["scale"]).float(), "offsets": offsets.to(torch.int32),
            "order": torch.where(inside, order, -1).to(torch.int32), "place": place.view(T, k).to(torch.int32)}


def _plain_codes(x):
    x = x.float()
    top = x.abs().amax(-1, keepdim=True)
    safe = torch.where(top == 0, 1.0, top)
    # in 64 bits: whether a value lies above or below the middle of two codes
    return torch.round(127.0 * x.double() / safe.double()).float(), top / 127.0


def _plain_matmul(s):
    codes, x_scale = _plain_codes(s["x"])
    y = (codes @ s["codes"].float().t()) * x_scale * s["scale"]
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


def _plain_experts(s):
    x, ids = s["x"], s["ids"].long() - s["case"]["first"]
    (T, k), E = ids.shape, s["case"]["experts"]
    inner = s["case"]["inner"]
    codes, x_scale = _plain_codes(x)
    e = ids.reshape(-1)
    here = (e >= 0) & (e < E)
    pair = torch.nonzero(here)[:, 0]
    order = torch.sort(e[pair], stable=True)[1]
    pair = pair[order]
    e, token = e[pair], pair // k
    counts = torch.bincount(e, minlength=E)
    room = max(1, int(counts.max()))
    slot = torch.arange(pair.numel(), device=x.device) - (counts.cumsum(0) - counts)[e]
    # each expert's tokens in rows of their own
    rows = torch.zeros(E, room, x.shape[1], device=x.device)
    rows[e, slot] = codes[token]
    both = torch.bmm(rows, s["gate_up"].float().transpose(1, 2))[e, slot] * x_scale[token] * s["gate_up_scale"][e]
    gate, up = both[:, :inner], both[:, inner:]
    h_codes, h_scale = _plain_codes(gate / (1.0 + torch.exp(-gate)) * up)
    rows = torch.zeros(E, room, inner, device=x.device)
    rows[e, slot] = h_codes
    out = torch.bmm(rows, s["down"].float().transpose(1, 2))[e, slot] * h_scale * s["down_scale"][e]
    y = torch.zeros(T * k, x.shape[1], device=x.device)
    y[pair] = out * s["weights"].reshape(-1)[pair, None]
    return y.view(T, k, -1).sum(1).to(x.dtype)


def run(state):
    c = state["case"]
    if own:
        from moe_quant_b200 import ops

        if c["kind"] == "route":
            ids, weights = ops.route_tokens(state["logits"], c["top_k"], score=c["score"], bias=state["bias"], groups=c["groups"], keep_groups=c["keep"],
                                            group_score=c["group_score"], renormalise=c["renormalise"], scale=c["scale"])
            plan = ops.expert_plan(ids, c["experts"])
            return {"ids": ids, "weights": weights, "offsets": plan.offsets, "order": plan.order, "place": plan.place}
        if c["kind"] == "matmul":
            return ops.int8_matmul(state["x"], state["codes"], state["scale"], bias=state["bias"])
        return ops.int8_experts(state["x"], state["ids"], state["weights"], state["gate_up"], state["gate_up_scale"], state["down"],
                                state["down_scale"], first=c["first"])
    return {"route": _plain_route, "matmul": _plain_matmul, "experts": _plain_experts}[c["kind"]](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    T = case["tokens"]
    if case["kind"] == "route":
        E, k = case["experts"], case["top_k"]
        # logits in; experts and weights out; the plan reads the experts and writes the pairs' order and places
        return {"bytes": T * E * size + (4 * E if case["bias"] else 0) + T * k * (4 + 4) + T * k * (4 + 4) + 4 * (E + 1), "flops": 8 * T * E}
    if case["kind"] == "matmul":
        N, K = case["rows"], case["cols"]
        return {"bytes": T * K * size + N * K + 4 * N + (4 * N if case["bias"] else 0) + T * N * size, "flops": 2 * T * N * K}
    E, total, k, K, inner = case["experts"], case["total"], case["top_k"], case["hidden"], case["inner"]
    reached = E * (1.0 - (1.0 - k / total) ** T)      # experts that some token reaches, were they equally likely
    pairs = T * k * E / total
    return {"bytes": reached * 3 * K * inner + reached * 4 * (2 * inner + K) + 2 * T * K * size + T * k * 8, "flops": 2 * pairs * 3 * K * inner}


# ---------------------------------------------------------------- from the definitions, in 64 bits
def _exact_route(s):
    c = s["case"]
    T, E, k, groups = c["tokens"], c["experts"], c["top_k"], c["groups"]
    x = s["logits"].double().cpu().numpy()
    x = np.minimum(np.where(np.isnan(x), -np.inf, x), LARGEST)
    bias = np.zeros(E) if s["bias"] is None else s["bias"].double().cpu().numpy()
    possible = np.isfinite(x) & np.isfinite(bias)
    with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
        if c["score"] == "sigmoid":
            score = np.where(x >= 0, 1 / (1 + np.exp(-np.abs(x))), np.exp(-np.abs(x)) / (1 + np.exp(-np.abs(x))))
        else:
            shifted = np.exp(x - x.max(1, keepdims=True))
            score = np.nan_to_num(shifted / shifted.sum(1, keepdims=True))
        value = np.where(possible, score + bias, -np.inf)
        if groups > 1:
            size = E // groups
            best = -np.sort(-value.reshape(T, groups, size), axis=-1)
            total = best[..., 0].copy()
            if c["group_score"] == "top2" and size > 1:
                total += np.where(np.isfinite(best[..., 1]), best[..., 1], 0)
            rank = np.argsort(np.argsort(-total, axis=1, kind="stable"), axis=1, kind="stable")
            value = np.where(np.repeat(rank < c["keep"], size, axis=1), value, -np.inf)
    if s["bias"] is None:
        value = np.where(np.isfinite(value), x, -np.inf)
    chosen = np.argsort(-value, axis=1, kind="stable")[:, :k]
    got = np.isfinite(np.take_along_axis(value, chosen, 1))
    w = np.where(got, np.take_along_axis(score, chosen, 1), 0.0)
    if c["renormalise"]:
        total = w.sum(1, keepdims=True)
        w = np.divide(w, total, out=np.zeros_like(w), where=total > 0)
    ids = np.where(got, chosen, -1)
    flat = ids.reshape(-1)
    order = np.array([], dtype=np.int64) if not flat.size else np.argsort(np.where(flat < 0, E, flat), kind="stable")
    n = int((flat >= 0).sum())
    place = np.full(flat.size, -1)
    place[order[:n]] = np.arange(n)
    order[n:] = -1
    offsets = np.concatenate([[0], np.cumsum(np.bincount(flat[flat >= 0], minlength=E))])
    return {"ids": ids.astype(np.int32), "weights": w * c["scale"], "offsets": offsets.astype(np.int32), "order": order.astype(np.int32),
            "place": place.reshape(T, k).astype(np.int32)}


def _exact_codes(x):
    largest = x.abs().max(dim=1, keepdim=True).values
    return (127 * x / largest.clamp(min=5e-324)).round(), largest / 127


def _exact_matmul(s):
    codes, scale = _exact_codes(s["x"].double())
    y = codes.mm(s["codes"].double().t()).mul_(scale).mul_(s["scale"].double())
    return y if s["bias"] is None else y + s["bias"].double()


def _exact_experts(s):
    c, x = s["case"], s["x"].double()
    y = torch.zeros_like(x)
    codes, scale = _exact_codes(x)
    for e in range(c["experts"]):
        token, slot = torch.nonzero(s["ids"] == e + c["first"], as_tuple=True)
        if token.numel() == 0:
            continue
        both = codes[token].mm(s["gate_up"][e].double().t()) * scale[token] * s["gate_up_scale"][e].double()
        gate, up = both.split(c["inner"], dim=1)
        h, h_scale = _exact_codes(gate * torch.sigmoid(gate) * up)
        out = h.mm(s["down"][e].double().t()) * h_scale * s["down_scale"][e].double()
        y.index_add_(0, token, out * s["weights"][token, slot, None].double())
    return y


def exact(case, seed):
    if _device().type == "cpu" and work(case)["flops"] > 1e11:
        return None
    state = prepare(case, seed)
    return {"route": _exact_route, "matmul": _exact_matmul, "experts": _exact_experts}[case["kind"]](state)
