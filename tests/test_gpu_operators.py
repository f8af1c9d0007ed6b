"""Operators of the quantized layers against their definitions in 64 bits (operator_reference)."""
import copy
import math

import pytest
import torch
import torch.nn as nn

from moe_quant_b200 import GPTQ, Int8Experts, Int8Linear, int8_layout, ops
from moe_quant_b200._lib import MoeQuantError
from moe_quant_b200.block_driver import quantize_block
from moe_quant_b200.int8 import int8_block
from moe_quant_b200.synthetic_block import SyntheticMoEBlock
from tests import operator_reference as R

pytestmark = pytest.mark.gpu

BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _tokens(T, K, dtype, seed):
    g = _gen(seed)
    return (torch.randn(T, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))).to(dtype)


def _codes(shape, seed, pad=16):
    """int8 codes whose rows start `pad` bytes apart or a multiple of it, with other bytes between the rows."""
    g = _gen(seed)
    whole = torch.randint(-128, 128, (*shape[:-1], -(-shape[-1] // pad) * pad), dtype=torch.int8, generator=g)
    return whole, 0.001 * torch.exp(0.5 * torch.randn(*shape[:-1], generator=g))


# ------------------------------------------------------------------ routing
ROUTES = [
    dict(T=1, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4, group_score="top2", scale=2.5),
    dict(T=77, E=256, k=8, score="sigmoid", bias=True, groups=8, keep=4, group_score="top2", scale=2.5),
    dict(T=33, E=64, k=6, score="softmax", renormalise=False),
    dict(T=33, E=64, k=6, score="softmax"),
    dict(T=9, E=60, k=4, score="softmax", bias=True, renormalise=False),
    dict(T=40, E=160, k=6, score="softmax", groups=8, keep=3, group_score="max", renormalise=False, scale=16.0),
    dict(T=17, E=1, k=1, score="sigmoid"),
    dict(T=17, E=7, k=7, score="sigmoid", bias=True),
    dict(T=8, E=33, k=32, score="softmax"),
    dict(T=5, E=1024, k=32, score="sigmoid", bias=True, groups=32, keep=5, group_score="top2"),
    dict(T=21, E=1000, k=3, score="softmax", groups=4, keep=1, group_score="top2"),
    dict(T=30, E=32, k=2, score="sigmoid", groups=32, keep=16, group_score="top2"),
    dict(T=11, E=513, k=9, score="sigmoid", renormalise=False),
]


def _route_both(logits, bias, c, dev):
    kw = dict(score=c["score"], groups=c.get("groups", 1), group_score=c.get("group_score", "max"), renormalise=c.get("renormalise", True),
              scale=c.get("scale", 1.0))
    ids, w = ops.route_tokens(logits.to(dev), c["k"], bias=None if bias is None else bias.to(dev), keep_groups=c.get("keep"), **kw)
    want, ww = R.route(logits, c["k"], bias=bias, keep=c.get("keep"), **kw)
    assert ids.dtype == torch.int32 and w.dtype == FP32 and ids.shape == w.shape == (*logits.shape[:-1], c["k"])
    assert torch.equal(ids.cpu().long(), want)
    # exponentials of 2 steps each, their arguments rounded once (|l| up to `big`), sums of at most 1024 terms in a tree of 5 + 5 levels
    # per lane and warp (32 per lane at most: 31 roundings), a few products and quotients
    big = float(logits.double().nan_to_num(0, 0, 0).abs().amax()) if logits.numel() else 0.0
    tol = (2 * (2 + min(big, 200.0)) + 31 + 10 + 6) * 2.0 ** -24 * 2
    assert torch.all((w.cpu().double() - ww).abs() <= tol * ww.abs() + 2.0 ** -126)
    return ids, w


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("c", ROUTES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_route(cuda, c, dtype):
    g = _gen(c["E"] + c["T"])
    logits = (2 * torch.randn(c["T"], c["E"], generator=g)).to(dtype)
    _route_both(logits, 0.1 * torch.randn(c["E"], generator=g) if c.get("bias") else None, c, cuda)


@pytest.mark.parametrize("E", [32, 255, 256, 257, 500, 504, 508, 510, 511, 512, 1023])
def test_route_and_plan_of_every_size_of_scratch(cuda, E):
    """Numbers of experts around the borders of what a kernel may take of shared memory without asking, and of its variants."""
    g = _gen(E)
    ids, _ = _route_both(torch.randn(9, E, generator=g), 0.1 * torch.randn(E, generator=g), dict(k=4, score="sigmoid"), cuda)
    offsets, order, place = R.plan(ids, E)
    got = ops.expert_plan(ids, E)
    assert torch.equal(got.offsets.cpu().long(), torch.from_numpy(offsets)) and torch.equal(got.place.cpu().long(), torch.from_numpy(place))


@pytest.mark.parametrize("E", range(340, 372))
def test_plan_around_the_border_of_free_shared_memory(cuda, E):
    ids = torch.randint(0, E, (50, 2), dtype=torch.int32, generator=_gen(E))
    assert torch.equal(ops.expert_plan(ids.to(cuda), E).order.cpu().long(), torch.from_numpy(R.plan(ids, E)[1]))


@pytest.mark.parametrize("c", ROUTES, ids=lambda c: "-".join(str(v) for v in c.values()))
def test_route_masks(cuda, c):
    """-inf and NaN logits, rows that hold nothing else, experts switched off by their bias, logits of +inf and of the
    type's extremes."""
    g = _gen(5 + c["E"])
    T, E = c["T"] + 8, c["E"]
    logits = 2 * torch.randn(T, E, generator=g)
    logits[torch.rand(T, E, generator=g) < 0.5] = -math.inf
    logits[0] = -math.inf
    logits[1] = math.nan
    logits[2, 1:] = -math.inf
    logits[3, : (E + 1) // 2] = -R.LARGEST
    logits[4, E // 2] = math.inf
    logits[5, 0] = R.LARGEST
    logits[6, E // 3] = math.nan
    bias = None
    if c.get("bias"):
        bias = 0.1 * torch.randn(E, generator=g)
        bias[torch.rand(E, generator=g) < 0.2] = -math.inf
        if E > 20:
            bias[7], bias[11] = math.nan, -R.LARGEST
    ids, w = _route_both(logits, bias, c, cuda)
    assert torch.all(ids[:2] == -1) and torch.all(w[:2] == 0)
    assert torch.all((w == 0) | (ids >= 0)) and torch.all(torch.isfinite(w))


def test_route_ties_go_to_the_lowest_index(cuda):
    for E in (16, 64, 256):
        logits = torch.zeros(3, E)
        logits[1, E // 2:] = 1.0
        for c in (dict(k=5, score="sigmoid"), dict(k=5, score="softmax"), dict(k=5, score="sigmoid", groups=4, keep=2, group_score="top2"),
                  dict(k=5, score="sigmoid", groups=4, keep=2)):
            _route_both(logits, None, c, cuda)
            _route_both(logits, torch.full((E,), 0.25), c, cuda)


def test_route_values_next_to_one_another(cuda):
    """Scores that fp32 cannot tell apart: saturated sigmoids, biases that differ in the last place, sums of two that nearly agree."""
    g = _gen(9)
    E = 64
    logits = 15 + torch.rand(40, E, generator=g)          # 1 - sigmoid is 3e-7 and less
    c = dict(k=8, score="sigmoid", groups=8, keep=4, group_score="top2")
    _route_both(logits, None, c, cuda)
    _route_both(logits, 1.0 + 2.0 ** -23 * torch.randint(0, 3, (E,), generator=g), c, cuda)
    _route_both(1e-7 * torch.randn(40, E, generator=g), torch.zeros(E), c, cuda)
    _route_both(1e-7 * torch.randn(40, E, generator=g), 1e-8 * torch.randn(E, generator=g), dict(c, score="softmax"), cuda)
    # exact swaps: expert 2i + 1 has the logit of 2i, the biases are equal
    l = torch.randn(40, E // 2, generator=g).repeat_interleave(2, dim=1)
    _route_both(l, torch.zeros(E), c, cuda)
    # a large bias leaves few bits for the score
    _route_both(torch.randn(40, E, generator=g), torch.full((E,), 1000.0), c, cuda)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
def test_route_groups_whose_sums_lie_next_to_one_another(cuda, score, dtype):
    """Sums of two scores that differ by less than fp32 can tell: the group is the one of 64-bit sums, for logits of every type."""
    v = torch.arange(1.0, 4.0, 2.0 ** -6).to(dtype)
    i, j = torch.triu_indices(len(v), len(v), 1)
    s = torch.sigmoid(v.double()) if score == "sigmoid" else torch.exp(v.double() - 4)
    order = torch.argsort(s[i] + s[j])
    i, j, sums = i[order], j[order], (s[i] + s[j])[order]
    gap = (sums[1:] - sums[:-1]).where(sums[1:] - sums[:-1] > 1e-12, torch.tensor(1.0, dtype=torch.float64))     # (64 bits tell these apart)
    at = torch.argsort(gap)[:300]
    rows = torch.full((2, 300, 2, 4), -4.0, dtype=dtype)
    for n, (low, high) in enumerate([(at, at + 1), (at + 1, at)]):
        rows[n, :, 0, 1], rows[n, :, 0, 2] = v[i[low]], v[j[low]]
        rows[n, :, 1, 0], rows[n, :, 1, 3] = v[i[high]], v[j[high]]
    c = dict(T=600, E=8, k=2, score=score, groups=2, keep=1, group_score="top2")
    _route_both(rows.reshape(600, 8), None, c, cuda)


def test_route_sigmoid_weights_of_very_negative_logits(cuda):
    """Every score underflows, their ratios do not."""
    logits = -200 - 3 * torch.rand(6, 32, generator=_gen(2))
    _, w = _route_both(logits, None, dict(k=4, score="sigmoid"), cuda)
    assert torch.allclose(w.sum(-1), torch.ones(6, device=cuda), rtol=1e-6)


def test_route_takes_views_and_leading_dimensions(cuda):
    g = _gen(4)
    base = torch.randn(2, 9, 80, generator=g)
    for view in (base[..., 3:67], base.transpose(0, 1), base[:, ::2], base[0, :, ::2], base[0, 0]):
        c = dict(k=4, score="sigmoid")
        ids, w = ops.route_tokens(view.to(cuda) if view.is_contiguous() else _same_strides(view, cuda), 4, score="sigmoid")
        want, ww = R.route(view, 4, score="sigmoid")
        assert torch.equal(ids.cpu().long(), want), c
        assert torch.allclose(w.cpu().double(), ww, rtol=1e-5)
    ids, w = ops.route_tokens(torch.zeros(3, 0, 16, device=cuda), 2)
    assert ids.shape == w.shape == (3, 0, 2)


def _same_strides(view, dev):
    """The view on the device, with its strides and offset."""
    base = view._base.to(dev)
    return base.as_strided(view.shape, view.stride(), view.storage_offset())


def test_route_many_tokens_in_one_call(cuda):
    """More rows than one wave of blocks holds, against the torch form in fp64 on the device."""
    g = torch.Generator(device=cuda).manual_seed(1)
    logits = torch.randn(70001, 128, device=cuda, generator=g)
    bias = 0.1 * torch.randn(128, device=cuda, generator=g)
    ids, w = ops.route_tokens(logits, 4, score="sigmoid", bias=bias)
    s = torch.sigmoid(logits.double())
    want = torch.sort(s + bias.double(), descending=True, stable=True)[1][:, :4]
    assert torch.equal(ids.long(), want)
    ww = s.gather(1, want)
    assert torch.allclose(w.double(), ww / ww.sum(-1, keepdim=True), rtol=2e-6, atol=0)


# ------------------------------------------------------------------ the plan
@pytest.mark.parametrize("T, k, E, total, first", [(1, 8, 32, 32, 0), (0, 4, 8, 8, 0), (5, 1, 1, 1, 0), (33, 3, 7, 9, 1), (1000, 8, 32, 256, 64), (700, 6, 1024, 1024, 0),
                                                   (9001, 8, 60, 64, 3), (3, 2, 600, 600, 0)])
def test_expert_plan(cuda, T, k, E, total, first):
    ids = torch.randint(-1, total, (T, k), dtype=torch.int32, generator=_gen(T + E))
    offsets, order, place = R.plan(ids, E, first)
    got = ops.expert_plan(ids.to(cuda), E, first)
    assert torch.equal(got.offsets.cpu().long(), torch.from_numpy(offsets))
    assert torch.equal(got.order.cpu().long(), torch.from_numpy(order))
    assert got.place.shape == (T, k) and torch.equal(got.place.cpu().long(), torch.from_numpy(place))


def test_expert_plan_of_one_crowded_expert_and_of_none(cuda):
    ids = torch.full((5000, 2), 3, dtype=torch.int64, device=cuda)      # the same expert twice in every row
    p = ops.expert_plan(ids, 4)
    assert p.offsets.tolist() == [0, 0, 0, 0, 10000] and torch.equal(p.order, torch.arange(10000, dtype=torch.int32, device=cuda))
    for value in (-1, 4, 2 ** 31 - 1, -2 ** 31):
        p = ops.expert_plan(torch.full((5000, 2), value, dtype=torch.int32, device=cuda), 4)
        assert p.offsets.tolist() == [0] * 5 and torch.all(p.order == -1) and torch.all(p.place == -1)


# ------------------------------------------------------------------ codes
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("T, K", [(1, 1), (3, 8), (5, 100), (9, 1024), (4, 1025), (2, 7168), (3, 20001)])
def test_quantize_tokens(cuda, T, K, dtype):
    x = _tokens(T, K, dtype, K)
    x[T // 2, 0] = x[T // 2].abs().amax()
    if K > 3:   # quotients exactly between two codes, and the smallest steps beside them
        top = x[T // 2].abs().amax()
        x[T // 2, 1], x[T // 2, 2] = top / 2, -top / 2
        x[T // 2, 3] = torch.nextafter(top.float() / 2, torch.tensor(0.0)).to(dtype)
    codes, scale = ops.quantize_tokens(x.to(cuda))
    want, _ = R.codes(x)
    assert torch.equal(codes.cpu().double(), want)
    assert torch.equal(scale.cpu(), x.float().abs().amax(-1) / 127)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_quantize_tokens_extremes(cuda, dtype):
    x = torch.randn(9, 64, generator=_gen(1)).to(dtype)
    x[0] = 0
    x[1, 5] = math.inf
    x[2, 6] = math.nan
    x[3] *= 2.0 ** -125
    x[4] = x[4] * 2.0 ** -100 * 2.0 ** -30
    x[5] = torch.finfo(dtype).max
    x[6, 1:] = 0
    x[7] = torch.finfo(torch.float32).smallest_normal * 2.0 ** -7     # denormal
    x[8, 3] = -math.inf
    codes, scale = ops.quantize_tokens(x.to(cuda))
    want, s = R.codes(x)
    assert torch.equal(codes.cpu().double(), want)
    assert torch.equal(torch.isnan(scale.cpu()), torch.isnan(s)) and scale[0] == 0
    good = ~torch.isnan(s)
    assert torch.all((scale.cpu().double() - s)[good].abs() <= 2.0 ** -24 * s[good] + 2.0 ** -149)


def test_quantize_tokens_of_views(cuda):
    base = torch.randn(4, 6, 130, generator=_gen(3)).to(BF16)
    for view in (base[..., 1:129], base[:, 1:3, :64], base.transpose(0, 1), base[..., ::2], base[0, 0]):
        codes, scale = ops.quantize_tokens(_same_strides(view, cuda))
        want, s = R.codes(view)
        assert codes.shape == view.shape and scale.shape == view.shape[:-1]
        assert torch.equal(codes.cpu().double(), want) and torch.equal(scale.cpu(), view.float().abs().amax(-1) / 127)


# ------------------------------------------------------------------ the product
SHAPES = [(1, 1, 1), (1, 2048, 7168), (2, 300, 640), (3, 129, 48), (4, 64, 100), (5, 1000, 136), (8, 257, 520), (9, 128, 128), (16, 31, 77), (17, 384, 1000),
          (37, 512, 256), (64, 100, 3000), (127, 130, 64), (129, 256, 129), (200, 260, 896), (255, 33, 40), (257, 513, 128), (600, 700, 272), (1025, 70, 1160)]


def _matmul_bound(x, codes, scale, bias, out_dtype):
    q, s = R.codes(x.reshape(-1, x.shape[-1]).cpu())
    product = q @ codes.double().t() * s[:, None] * scale.double()
    y = product if bias is None else product + bias.double()
    return y, R.product_bound(y, product, out_dtype)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("T, N, K", SHAPES)
def test_int8_matmul(cuda, T, N, K, dtype):
    x = _tokens(T, K, dtype, T + K)
    whole, scale = _codes((N, K), N)
    w = whole.to(cuda)[:, :K]
    bias = torch.randn(N, generator=_gen(1)) if (T + N) % 2 else None
    y = ops.int8_matmul(x.to(cuda), w, scale.to(cuda), bias=None if bias is None else bias.to(cuda))
    want, bound = _matmul_bound(x, whole[:, :K], scale, bias, dtype)
    assert y.dtype == dtype and y.shape == (T, N)
    assert torch.all((y.cpu().double() - want).abs() <= bound)


@pytest.mark.parametrize("T", [1, 7, 40, 300])
@pytest.mark.parametrize("out_dtype", [FP32, BF16, FP16])
def test_int8_matmul_of_given_codes_is_exact_up_to_its_roundings(cuda, T, out_dtype):
    N, K = 200, 1500
    g = _gen(T)
    q = torch.zeros(T, 1504, dtype=torch.int8, device=cuda)[:, :K]
    q.copy_(torch.randint(-128, 128, (T, K), dtype=torch.int8, generator=g))
    whole, scale = _codes((N, K), 3)
    xs = torch.rand(T, generator=g)
    y = ops.int8_matmul(q, whole.to(cuda)[:, :K], scale.to(cuda), x_scale=xs.to(cuda), out_dtype=out_dtype)
    want = q.cpu().double() @ whole[:, :K].double().t() * xs.double()[:, None] * scale.double()
    assert y.dtype == out_dtype
    assert torch.all((y.cpu().double() - want).abs() <= R.product_bound(want, want, out_dtype))


def test_int8_matmul_of_the_largest_sums(cuda):
    """All codes at their ends over the longest row: the sum comes within 1 % of 2^31."""
    K = 131072
    w = torch.full((3, K), -128, dtype=torch.int8, device=cuda)
    w[1] = 127
    for T in (1, 20, 140):
        x = torch.ones(T, K, dtype=BF16, device=cuda)
        y = ops.int8_matmul(x, w, torch.full((3,), 1.0 / 128, device=cuda), out_dtype=FP32)
        want = torch.tensor([-float(K), 127 * K / 128, -float(K)], dtype=torch.float64) * 1.0
        assert torch.all((y.cpu().double() - want).abs() <= 5 * 2.0 ** -24 * want.abs())


def test_int8_matmul_of_the_lowest_codes(cuda):
    """-128 on both sides over the longest row that is allowed."""
    K = 131071
    w = torch.full((2, K + 1), -128, dtype=torch.int8, device=cuda)[:, :K]
    for T in (1, 20):
        q = torch.full((T, K + 1), -128, dtype=torch.int8, device=cuda)[:, :K]
        y = ops.int8_matmul(q, w, torch.ones(2, device=cuda), x_scale=torch.ones(T, device=cuda), out_dtype=FP32)
        assert torch.all((y.double() - 16384.0 * K).abs() <= 3 * 2.0 ** -24 * 16384.0 * K)


def test_offsets_beyond_32_bits(cuda):
    """More than 2^31 values in, and out: the last rows are as in a call of their own."""
    T, K = 300007, 7168
    x = torch.empty(T, K, dtype=BF16, device=cuda)
    x[:64] = 0.0
    x[64:].copy_(torch.randn(1, K, device=cuda).to(BF16).expand(T - 64, K))
    x[-64:] = torch.randn(64, K, device=cuda).to(BF16)
    codes, scale = ops.quantize_tokens(x)
    tail, tail_scale = ops.quantize_tokens(x[-64:].clone())
    assert torch.equal(codes[-64:], tail) and torch.equal(scale[-64:], tail_scale) and not torch.any(codes[:64])
    assert torch.equal(codes[T // 2], codes[64])
    del codes
    w = torch.randint(-128, 128, (8200, K), dtype=torch.int8, device=cuda)
    y = ops.int8_matmul(x, w, torch.ones(8200, device=cuda))
    assert y.numel() > 2 ** 31
    assert torch.equal(y[-64:], ops.int8_matmul(x[-64:].clone(), w, torch.ones(8200, device=cuda)))
    assert torch.equal(y[T // 2], y[64]) and not torch.any(y[:64])


@pytest.mark.parametrize("T", [2, 30, 200])
def test_int8_matmul_broken_and_zero_tokens(cuda, T):
    x = _tokens(T, 320, BF16, 1)
    x[0, 7] = math.inf
    x[1] = 0
    if T > 20:
        x[20, 3] = math.nan
    whole, scale = _codes((70, 320), 1)
    y = ops.int8_matmul(x.to(cuda), whole.to(cuda), scale.to(cuda)).cpu()
    broken = ~torch.isfinite(x).all(-1)
    assert torch.all(torch.isnan(y[broken])) and torch.all(y[1] == 0)
    want, bound = _matmul_bound(x[~broken], whole, scale, None, BF16)
    assert torch.all((y[~broken].double() - want).abs() <= bound)


@pytest.mark.parametrize("T", [1, 3, 50, 150])
def test_int8_matmul_of_views(cuda, T):
    """Rows that start on odd addresses, transposed leading dimensions, weights with bytes between their rows."""
    K, N = 200, 90
    base = torch.randn(2, T, 2 * K + 3, generator=_gen(T)).to(BF16)
    whole, scale = _codes((N, K), 2, pad=64)
    w = whole.to(cuda)[:, :K]
    assert w.stride(0) == 256
    for view in (base[..., 1:K + 1], base[..., ::2][..., :K], base.transpose(0, 1)[..., :K]):
        y = ops.int8_matmul(_same_strides(view, cuda), w, scale.to(cuda, torch.bfloat16))
        want, bound = _matmul_bound(view, whole[:, :K], scale.to(BF16), None, BF16)
        assert y.shape == (*view.shape[:-1], N)
        assert torch.all((y.cpu().double().reshape(want.shape) - want).abs() <= bound)
    # rows of weights of which every other one is used
    y = ops.int8_matmul(base[0, :, :K].to(cuda), whole.to(cuda)[::2, :K], scale.to(cuda)[::2])
    want, bound = _matmul_bound(base[0, :, :K], whole[::2, :K], scale[::2], None, BF16)
    assert torch.all((y.cpu().double() - want).abs() <= bound)


def test_int8_matmul_empty(cuda):
    w, s = torch.zeros(8, 32, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)
    assert ops.int8_matmul(torch.zeros(0, 32, device=cuda), w, s).shape == (0, 8)
    assert ops.int8_matmul(torch.zeros(4, 32, device=cuda), w[:0], s[:0]).shape == (4, 0)
    assert ops.int8_matmul(torch.zeros(2, 0, 32, device=cuda), w, s).shape == (2, 0, 8)


# ------------------------------------------------------------------ the experts
def _experts_case(T, k, E, total, first, K, I, dtype, seed):
    g = _gen(seed)
    x = _tokens(T, K, dtype, seed)
    ids = torch.rand(T, total, generator=g).topk(k).indices.to(torch.int32) if T else torch.zeros(0, k, dtype=torch.int32)
    weights = torch.rand(T, k, generator=g)
    gu, gus = _codes((E, 2 * I, K), seed + 1)
    d, ds = _codes((E, K, I), seed + 2)
    return dict(x=x, ids=ids, weights=weights, gate_up=gu[..., :K], gate_up_scale=gus, down=d[..., :I], down_scale=ds, first=first)


def _on(c, dev):
    out = {}
    for n, t in c.items():
        if not torch.is_tensor(t):
            out[n] = t
        elif t.dtype == torch.int8 and t._base is not None:
            out[n] = _same_strides(t, dev)
        else:
            out[n] = t.to(dev)
    return out


def _check_experts(y, c):
    want, bound = R.experts(**c)
    assert y.dtype == c["x"].dtype and y.shape == c["x"].shape
    off = (y.cpu().double() - want).abs()
    assert torch.all(off <= bound), float((off / bound).max())


EXPERTS = [(1, 1, 1, 1, 0, 16, 16), (1, 8, 8, 8, 0, 512, 256), (1, 4, 3, 12, 5, 264, 72), (2, 2, 4, 4, 0, 1000, 40), (7, 2, 4, 8, 4, 128, 64),
           (40, 8, 32, 32, 0, 128, 136), (64, 8, 4, 32, 8, 640, 256), (130, 2, 3, 3, 0, 256, 200), (333, 2, 8, 8, 0, 256, 128), (600, 1, 1, 1, 0, 320, 100),
           (700, 4, 2, 8, 3, 130, 130)]


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T, k, E, total, first, K, I", EXPERTS)
def test_int8_experts(cuda, T, k, E, total, first, K, I, dtype):
    c = _experts_case(T, k, E, total, first, K, I, dtype, T + K)
    _check_experts(ops.int8_experts(**_on(c, cuda)), c)


@pytest.mark.parametrize("T", [1, 6, 90, 400])
def test_int8_experts_without_pairs_and_with_crowded_ones(cuda, T):
    c = _experts_case(T, 2, 3, 3, 0, 192, 96, BF16, T)
    c["ids"] = torch.full((T, 2), -1, dtype=torch.int32)
    assert torch.all(ops.int8_experts(**_on(c, cuda)) == 0)
    c["ids"] = torch.full((T, 2), 1, dtype=torch.int32)          # the same expert twice
    _check_experts(ops.int8_experts(**_on(c, cuda)), c)
    c["ids"][T // 2:] = 7                                        # an expert of another rank
    _check_experts(ops.int8_experts(**_on(c, cuda)), c)


@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_int8_experts_of_the_largest_sums(cuda, dtype):
    """Every product of the down projection at its limit: h codes of 127 against weights of -128 and 127, scales that differ by 2^20."""
    T, K, I = 40, 64, 4096
    x = torch.ones(T, 16, dtype=dtype)
    gu, gus = torch.full((1, 2 * I, 16), 127, dtype=torch.int8), torch.full((1, 2 * I), 1.0 / 127 / 16)
    d = torch.full((1, 16, I), -128, dtype=torch.int8)
    d[0, 1::2] = 127
    ds = torch.full((1, 16), 1e-4)
    ds[0, 3], ds[0, 4] = 1e-4 * 2.0 ** -20, 3.9e-4
    c = dict(x=x, ids=torch.zeros(T, 1, dtype=torch.int32), weights=torch.ones(T, 1), gate_up=gu, gate_up_scale=gus, down=d, down_scale=ds, first=0)
    y = ops.int8_experts(**_on(c, cuda))
    assert torch.all(torch.isfinite(y))
    _check_experts(y, c)


def test_ids_outside_32_bits_are_no_expert(cuda):
    ids = torch.tensor([[2 ** 32 + 1, 1], [-2 ** 40, 0]], device=cuda)
    p = ops.expert_plan(ids, 2)
    assert p.offsets.tolist() == [0, 1, 2] and p.place.tolist() == [[-1, 1], [-1, 0]]


@pytest.mark.parametrize("T", [1, 5, 100])
def test_int8_experts_extremes(cuda, T):
    """A broken token breaks its own row alone; zero weights, zero and negative scales; large and tiny scales."""
    c = _experts_case(T, 2, 4, 4, 0, 256, 128, BF16, 3)
    c["down_scale"][:, 3] = 0
    c["down_scale"][:, 5] *= -1
    c["down_scale"][1] *= 2.0 ** 20
    c["down_scale"][2, ::2] *= 2.0 ** -12
    c["gate_up_scale"][3] *= 2.0 ** -20
    c["weights"][T // 2, 0] = 0
    _check_experts(ops.int8_experts(**_on(c, cuda)), c)
    c["x"][0, 9] = math.inf
    y = ops.int8_experts(**_on(c, cuda)).cpu()
    assert torch.all(torch.isnan(y[0]))
    rest = dict(c, x=c["x"][1:], ids=c["ids"][1:], weights=c["weights"][1:])
    if T > 1:
        _check_experts(y[1:], rest)


def test_int8_experts_empty_and_leading_dimensions(cuda):
    c = _experts_case(6, 2, 4, 4, 0, 128, 64, BF16, 3)
    d = _on(c, cuda)
    y = ops.int8_experts(**d)
    again = ops.int8_experts(**{**d, "x": d["x"].view(2, 3, -1), "ids": d["ids"].view(2, 3, 2).long(), "weights": d["weights"].view(2, 3, 2)})
    assert torch.equal(again.view(6, -1), y)
    none = ops.int8_experts(**{**d, "x": d["x"][:0], "ids": d["ids"][:0], "weights": d["weights"][:0]})
    assert none.shape == (0, 128)


# ------------------------------------------------------------------ calls as a program makes them
def test_results_do_not_depend_on_the_call(cuda):
    """Twice the same bits, also on another stream, in a graph, and with other calls under way."""
    c = _on(_experts_case(150, 4, 8, 8, 0, 384, 256, BF16, 8), cuda)
    x1 = c["x"][:3]
    w, ws = c["gate_up"][0], c["gate_up_scale"][0]
    logits = torch.randn(150, 8, device=cuda)

    def all_of_it():
        ids, weights = ops.route_tokens(logits, 4, score="sigmoid")
        return (ids, weights, ops.expert_plan(ids, 8).order, ops.int8_experts(**c), ops.int8_experts(**{**c, "x": x1, "ids": c["ids"][:3], "weights": c["weights"][:3]}),
                ops.int8_matmul(c["x"], w, ws), ops.int8_matmul(x1, w, ws), *ops.quantize_tokens(c["x"]))

    first = all_of_it()
    again = all_of_it()
    side = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    beside = []
    for s in side:
        with torch.cuda.stream(s):
            beside.append(all_of_it())
    torch.cuda.synchronize()
    for other in (again, *beside):
        assert all(torch.equal(a, b) for a, b in zip(first, other))


def test_graphs_replay_with_new_inputs(cuda):
    """Two graphs captured on one stream, replayed on two at once, each with inputs that changed after the capture."""
    cases = [_on(_experts_case(T, 2, 4, 4, 0, 256, 128, BF16, T), cuda) for T in (90, 1)]
    w = cases[0]["gate_up"][1]
    ws = cases[0]["gate_up_scale"][1]

    def run(c):
        ids, weights = ops.route_tokens(c["logits"], 2, score="sigmoid")
        return ids, weights, ops.int8_experts(c["x"], ids, weights, c["gate_up"], c["gate_up_scale"], c["down"], c["down_scale"]), ops.int8_matmul(c["x"], w, ws)

    for c in cases:
        c["logits"] = torch.randn(c["x"].shape[0], 4, device=cuda)
        run(c)
    stream = torch.cuda.Stream()
    graphs, outs = [], []
    for c in cases:
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append(run(c))
        graphs.append(graph)
    for c in cases:
        c["x"].copy_(torch.randn_like(c["x"]))
        c["logits"].copy_(torch.randn_like(c["logits"]))
    torch.cuda.synchronize()
    side = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for graph, s in zip(graphs, side):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for c, got in zip(cases, outs):
        assert all(torch.equal(a, b) for a, b in zip(run(c), got))


def test_gradients_are_refused(cuda):
    w, s = torch.zeros(8, 32, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)
    x = torch.zeros(4, 32, device=cuda, requires_grad=True)
    for call in (lambda: ops.int8_matmul(x, w, s), lambda: ops.route_tokens(x, 2), lambda: ops.quantize_tokens(x),
                 lambda: ops.int8_matmul(x.detach(), w, s.clone().requires_grad_())):
        with pytest.raises(MoeQuantError, match="no backward"):
            call()
        with torch.no_grad():
            call()


def test_wrapper_refusals(cuda):
    x, w, s = torch.zeros(4, 32, device=cuda), torch.zeros(8, 32, dtype=torch.int8, device=cuda), torch.ones(8, device=cuda)
    ids, weights = torch.zeros(4, 2, dtype=torch.int32, device=cuda), torch.ones(4, 2, device=cuda)
    gu, gus = torch.zeros(2, 32, 32, dtype=torch.int8, device=cuda), torch.ones(2, 32, device=cuda)
    d, ds = torch.zeros(2, 32, 16, dtype=torch.int8, device=cuda), torch.ones(2, 32, device=cuda)
    h = x.half()
    bad = [lambda: ops.int8_matmul(x[:, :31], w, s), lambda: ops.int8_matmul(x, w.int(), s), lambda: ops.int8_matmul(x, w, s[:7]),
           lambda: ops.int8_matmul(x.double(), w, s), lambda: ops.int8_matmul(x.to(torch.int8), w, s), lambda: ops.int8_matmul(x, w, s, x_scale=s[:4]),
           lambda: ops.int8_matmul(x.to(torch.int8), w, s, x_scale=s[:4]), lambda: ops.int8_matmul(x.to(torch.int8), w, s, x_scale=s[:3], out_dtype=FP32),
           lambda: ops.int8_matmul(x, w, s, bias=s[:4]), lambda: ops.int8_matmul(x, w.t()[:, :32].t(), s, out_dtype=torch.float64),
           lambda: ops.int8_matmul(x[:, 8:24], w[:, 8:24], s), lambda: ops.int8_matmul(x[:, :16], w.reshape(16, 16)[:8].t().contiguous().t(), s),
           lambda: ops.int8_matmul(x, w, s.cpu()), lambda: ops.int8_matmul(x[:, :20], torch.zeros(8, 20, dtype=torch.int8, device=cuda), s),
           lambda: ops.route_tokens(x, 0), lambda: ops.route_tokens(x, -1), lambda: ops.route_tokens(x, 33), lambda: ops.route_tokens(x, 2, score="tanh"), lambda: ops.route_tokens(x, 2, groups=5),
           lambda: ops.route_tokens(x, 2, bias=s), lambda: ops.route_tokens(x.to(torch.int8), 2), lambda: ops.route_tokens(x, 2, groups=4, keep_groups=5),
           lambda: ops.expert_plan(weights, 4), lambda: ops.expert_plan(ids, 0), lambda: ops.expert_plan(ids, 2000), lambda: ops.expert_plan(ids, 4, first=-1),
           lambda: ops.int8_experts(x, ids, weights, gu, gus, d, ds), lambda: ops.int8_experts(h, ids[:3], weights[:3], gu, gus, d, ds),
           lambda: ops.int8_experts(h, ids, weights, gu, gus, d.transpose(1, 2), ds), lambda: ops.int8_experts(h, ids, weights, gu[:, :31], gus, d, ds),
           lambda: ops.int8_experts(h, ids, weights, gu, gus[:, :31], d, ds), lambda: ops.int8_experts(h, ids, weights[:, :1], gu, gus, d, ds),
           lambda: ops.int8_experts(h, ids.float(), weights, gu, gus, d, ds)]
    for i, call in enumerate(bad):
        with pytest.raises(MoeQuantError):
            call()
            pytest.fail(f"call {i} was not refused")
    torch.cuda.synchronize()


# ------------------------------------------------------------------ together, on what the quantizer returns
def _quantized(R_, C, seed, dev):
    g = _gen(seed)
    layer = nn.Linear(C, R_, bias=False, dtype=BF16, device=dev)
    layer.weight.data = (0.05 * torch.randn(R_, C, generator=g)).to(dev, BF16)
    handle = GPTQ(layer, None, True, 1e-2, 128)
    handle.update(_tokens(2 * C, C, BF16, seed).to(dev))
    return handle.quantize(8)


def test_layer_runs_on_what_quantize_returns(cuda):
    q, s, z = _quantized(192, 256, 1, cuda)
    assert s.shape == (192, 1)
    layer = Int8Linear(q, s, z, bias=torch.linspace(-1, 1, 192, device=cuda))
    x = _tokens(70, 256, BF16, 2)
    codes, scale = int8_layout(q, s, z)
    want, bound = _matmul_bound(x, codes.cpu(), scale.cpu(), torch.linspace(-1, 1, 192), BF16)
    assert torch.all((layer(x.to(cuda)).cpu().double() - want).abs() <= bound)
    assert torch.equal(layer(x.to(cuda).view(2, 35, 256)).view(70, 192), layer(x.to(cuda)))


def test_router_plan_and_experts_together(cuda):
    """Route, group, run the quantized experts: as the chain of definitions gives it, and expert by expert as the plan lists them."""
    E, K, I, T, k = 6, 256, 128, 130, 3
    sides = {side: [_quantized(*((K, I) if side == "down" else (I, K)), 10 * e + i, cuda) for e in range(E)] for i, side in enumerate(("gate", "up", "down"))}
    experts = Int8Experts(sides["gate"], sides["up"], sides["down"])
    x = _tokens(T, K, BF16, 77)
    logits = torch.randn(T, E, generator=_gen(6))
    logits[T - 5:] = -math.inf                       # padding
    bias = torch.tensor([0.1, -0.2, 0.0, -math.inf, 0.3, 0.05])
    ids, weights = ops.route_tokens(logits.to(cuda), k, score="sigmoid", bias=bias.to(cuda), scale=2.5)
    want_ids, _ = R.route(logits, k, score="sigmoid", bias=bias, scale=2.5)
    assert torch.equal(ids.cpu().long(), want_ids) and not torch.any(ids == 3)
    y = experts(x.to(cuda), ids, weights)
    c = dict(x=x, ids=ids, weights=weights, gate_up=experts.gate_up, gate_up_scale=experts.gate_up_scale, down=experts.down, down_scale=experts.down_scale)
    _check_experts(y, c)
    assert torch.all(y[T - 5:] == 0)
    plan = ops.expert_plan(ids, E)
    offsets, order = plan.offsets.tolist(), plan.order.long()
    assert offsets[-1] == int((ids >= 0).sum())
    for e in range(E):
        mine = order[offsets[e]:offsets[e + 1]]
        assert torch.all(ids.reshape(-1)[mine] == e)
    # two ranks with half of the experts each: their sums are the whole, up to the roundings of the three results
    halves = [Int8Experts(*([r[i] for i in range(lo, lo + 3)] for r in sides.values()), first=lo)(x.to(cuda), ids, weights).double() for lo in (0, 3)]
    assert torch.all((sum(halves) - y.double()).abs() <= 2.0 ** -8 * 1.1 * (halves[0].abs() + halves[1].abs() + y.double().abs()) + 1e-6)


def test_block_driver_gives_the_outputs_of_the_served_block(cuda):
    torch.manual_seed(0)
    block = SyntheticMoEBlock(hidden=256, inter=128, n_experts=8, top_k=2, seed=3).to(BF16).to(cuda)
    block.mlp.gate.disabled_experts = [5]
    inputs = [_tokens(60, 256, BF16, i).to(cuda)[None] for i in range(3)]
    plain = copy.deepcopy(block)
    got = quantize_block(block, inputs, bits=8, group_size=None, int8_outputs=True)
    want = quantize_block(plain, inputs, bits=8, group_size=None)
    assert block.mlp.int8_experts is None and isinstance(block.mlp.shared_experts.up_proj, nn.Linear)
    for a, b in zip(block.parameters(), plain.parameters()):
        assert torch.equal(a, b)
    # activations of 8 bits: within a few steps of 1/127 of a token's largest value, averaged over a row
    for a, b, x in zip(got["outputs"], want["outputs"], inputs):
        assert a.shape == b.shape and bool(torch.isfinite(a).all())
        assert float((a - b).float().norm() / (b - x).float().norm()) < 0.1


def test_block_driver_of_an_fp32_block(cuda):
    block = SyntheticMoEBlock(hidden=64, inter=32, n_experts=4, top_k=2, q_rank=32, kv_rank=32, n_heads=2, nope_dim=16, rope_dim=16, v_dim=32, seed=1).to(cuda)
    x = _tokens(80, 64, FP32, 3).to(cuda)[None]
    plain = copy.deepcopy(block)
    a = quantize_block(block, [x], bits=8, group_size=None, int8_outputs=True)["outputs"][0]
    b = quantize_block(plain, [x], bits=8, group_size=None)["outputs"][0]
    assert a.dtype == FP32 and bool(torch.isfinite(a).all())
    assert float((a - b).norm() / (b - x).norm()) < 0.1


def test_block_runs_its_experts_by_the_operators(cuda):
    """The experts of a block inside the context are route_tokens and int8_experts; tokens that arrive one pair at a time, as over
    several ranks, go through the same operator."""
    block = SyntheticMoEBlock(hidden=128, inter=64, n_experts=4, top_k=2, seed=1).to(BF16).to(cuda)
    results = {}
    for i, (name, layer) in enumerate((n, l) for n, l in block.named_modules() if isinstance(l, nn.Linear) and ".experts." in n):
        results[name] = _quantized(*layer.weight.shape, i, cuda)
    x = _tokens(50, 128, BF16, 4).to(cuda)
    with torch.no_grad(), int8_block(block, results):
        moe = block.mlp
        ids, w = ops.route_tokens(x.float() @ moe.gate.weight.float().t(), 2, score="sigmoid")
        m = moe.int8_experts
        y = ops.int8_experts(x, ids, w, m.gate_up, m.gate_up_scale, m.down, m.down_scale)
        assert torch.equal(moe(x), y + moe.shared_experts(x))
        pairs = moe._run_experts(x.repeat_interleave(2, dim=0), ids.reshape(-1).long()).double().view(50, 2, 128)
        both = (pairs * w[..., None].double()).sum(1)
        # each pair's row was rounded to bf16 first
        assert torch.all((both - y.double()).abs() <= 2.0 ** -8 * 1.1 * ((pairs.abs() * w[..., None].double()).sum(1) + both.abs()) + 1e-6)
