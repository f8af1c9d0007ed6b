"""Operators of the quantized layers where their results could depend on what they should not."""
import threading

import pytest
import torch

from moe_quant_b200 import _lib, ops
from tests import operator_reference as R
from tests.test_gpu_operators import BF16, FP16, FP32, _codes, _experts_case, _gen, _on, _route_both, _tokens

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ the experts
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T", [1, 2, 40, 300])
def test_a_channel_keeps_its_digits_beside_larger_ones(cuda, T, dtype):
    """Scales that differ by up to 2^40 within 32 channels.  All codes of h are 127, so the sums are exact and the rest are roundings: h with up to
    (16 + 5 |gate|) 2^-24 (gate is 1 here), its scale, the factors and products one 2^-24 each, and the result's own half step."""
    K, I = 64, 1024
    x = torch.ones(T, 16, dtype=dtype)
    gate_up, gate_up_scale = torch.full((1, 2 * I, 16), 127, dtype=torch.int8), torch.full((1, 2 * I), 1.0 / 127 / 16)
    down = torch.randint(-128, 128, (1, K, I), dtype=torch.int8, generator=_gen(1))[:, :16]
    down_scale = 1e-2 * 2.0 ** -torch.linspace(0, 40, 16)[torch.randperm(16, generator=_gen(2))][None]
    if dtype == FP16:
        down_scale = down_scale * 2.0 ** 6      # (results of up to 3e5 * 0.73 / 127 * 0.64, 1e3; the smallest scales leave fp16's range)
    c = dict(x=x, ids=torch.zeros(T, 1, dtype=torch.int32), weights=torch.ones(T, 1), gate_up=gate_up, gate_up_scale=gate_up_scale, down=down,
             down_scale=down_scale)
    y = ops.int8_experts(**_on(c, cuda)).cpu().double()
    want, _ = R.experts(**c)
    assert torch.all((y - want).abs() <= want.abs() * (1.01 * R.HALF_STEP[dtype] + 60 * 2.0 ** -24) + R.SMALLEST[dtype])


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("T, k, E, K, I", [(9, 2, 4, 256, 128), (33, 4, 4, 264, 72), (300, 8, 8, 512, 520), (5, 3, 6, 130, 1000), (6, 2, 3, 7168, 2048)])
def test_a_token_gets_the_same_result_alone(cuda, T, k, E, K, I, dtype):
    c = _on(_experts_case(T, k, E, E, 0, K, I, dtype, T + K), cuda)
    c["gate_up_scale"] *= 8        # gates of some size
    c["ids"][T // 2, 0] = -1
    together = ops.int8_experts(**c)
    for t in range(0, T, max(1, T // 20)):
        alone = ops.int8_experts(**{**c, "x": c["x"][t:t + 1], "ids": c["ids"][t:t + 1], "weights": c["weights"][t:t + 1]})
        assert torch.equal(alone[0], together[t]), t


# ------------------------------------------------------------------ the product
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("N, K", [(520, 1024), (2048, 7168), (100, 300)])
def test_tokens_get_the_same_product_in_calls_of_any_size(cuda, N, K, dtype):
    """With a bias and without: few tokens, tiles whose k is shared, tiles of their own."""
    x = _tokens(2100, K, dtype, N).to(cuda)
    whole, scale = _codes((N, K), K)
    w, scale, bias = whole.to(cuda)[:, :K], scale.to(cuda), torch.randn(N, generator=_gen(2)).to(cuda)
    for b in (None, bias):
        full = ops.int8_matmul(x, w, scale, bias=b)
        for T in (1, 2, 4, 5, 37, 300, 1011):
            assert torch.equal(ops.int8_matmul(x[:T], w, scale, bias=b), full[:T]), T


# ------------------------------------------------------------------ routing
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("c", [
    dict(E=8, k=1, score="sigmoid"), dict(E=8, k=3, score="softmax"), dict(E=64, k=6, score="softmax", renormalise=False), dict(E=60, k=8, score="sigmoid"),
    dict(E=256, k=8, score="sigmoid"), dict(E=400, k=5, score="softmax"), dict(E=1000, k=30, score="sigmoid"),
    dict(E=64, k=4, score="sigmoid", groups=8, keep=3, group_score="top2"), dict(E=256, k=8, score="softmax", groups=8, keep=4),
    dict(E=60, k=4, score="sigmoid", groups=4, keep=2, group_score="top2"), dict(E=60, k=4, score="softmax", groups=4, keep=2)],
    ids=lambda c: "-".join(str(v) for v in c.values()))
def test_route_zeros_of_either_sign_are_a_tie(cuda, c, dtype):
    """-0.0 and +0.0 have one score: the lowest index comes first, at the cut behind the k-th too."""
    E = c["E"]
    g = _gen(E + c["k"])
    zeros = torch.where(torch.rand(40, E, generator=g) < 0.5, 0.0, -0.0)
    logits = torch.where(torch.rand(40, E, generator=g) < 0.3, -1.0, zeros)      # mostly zeros, more than k of them
    logits[:10] = zeros[:10]
    logits[10:20] = torch.where(torch.rand(10, E, generator=g) < 2.0 / E, zeros[10:20], -torch.rand(10, E, generator=g) - 0.5)     # a few
    logits[20:25] = torch.where(torch.rand(5, E, generator=g) < 0.1, 1.0, zeros[20:25])     # behind others
    logits = logits.to(dtype)
    assert torch.any(torch.signbit(logits) & (logits == 0)) and torch.any(~torch.signbit(logits) & (logits == 0))
    _route_both(logits, None, c, cuda)
    _route_both(logits, torch.where(torch.rand(E, generator=g) < 0.5, 0.0, -0.0), c, cuda)
    # one negative zero in front of a positive one
    logits = torch.full((1, E), -1.0, dtype=dtype)
    logits[0, 2], logits[0, E - 1] = -0.0, 0.0
    ids, _ = _route_both(logits, None, c, cuda)
    assert int(ids[0, 0]) == 2


def _choice_on_the_device(logits, k, score, bias, groups, keep, top2):
    """The choice by scores in 64 bits, in torch."""
    l = logits.double() + 0.0
    s = torch.sigmoid(l) if score == "sigmoid" else torch.softmax(l, -1)
    v = s if bias is None else s + bias.double()
    by = l if bias is None else v
    if groups > 1:
        worth = v if bias is not None or top2 else l
        best = worth.view(len(l), groups, -1).topk(2, -1).values
        kept = torch.sort(best.sum(-1) if top2 else best[..., 0], dim=-1, descending=True, stable=True)[1][:, :keep]
        stays = torch.zeros(len(l), groups, dtype=torch.bool, device=l.device).scatter_(1, kept, True)
        by = by.view(len(l), groups, -1).masked_fill(~stays[..., None], -float("inf")).view(l.shape)
    return torch.sort(by, dim=-1, descending=True, stable=True)[1][:, :k]


@pytest.mark.parametrize("grid", [False, True])
@pytest.mark.parametrize("E", [60, 256, 332, 900])
def test_route_many_random_rows(cuda, E, grid):
    """4000 rows each of 72 configurations; on a grid of values there are ties and zeros of either sign in every row."""
    g = torch.Generator(device=cuda).manual_seed(E)
    for score in ("sigmoid", "softmax"):
        for scale, dtype in ((0.01, FP32), (1.0, FP16), (40.0, BF16)):
            for bias_scale in (None, 0.0, 0.1):
                for groups, keep, top2 in ((1, 1, False), (4, 3, True), (2, 1, True), (4, 2, False)):
                    logits = scale * torch.randn(4000, E, device=cuda, generator=g)
                    logits = ((logits * (2 / scale)).round() * (scale / 2) if grid else logits).to(dtype)
                    bias = None if bias_scale is None else bias_scale * torch.randn(E, device=cuda, generator=g)
                    ids, _ = ops.route_tokens(logits, 8, score=score, bias=bias, groups=groups, keep_groups=keep, group_score="top2" if top2 else "max")
                    assert torch.equal(ids.long(), _choice_on_the_device(logits, 8, score, bias, groups, keep, top2)), (score, scale, bias_scale, groups)


# ------------------------------------------------------------------ calls of several threads
@pytest.mark.parametrize("what", ["plan", "route"])
@pytest.mark.parametrize("n_threads", [2, 6])
def test_threads_with_different_numbers_of_experts(cuda, what, n_threads):
    """What one thread's call lets a kernel take of shared memory must not take away what another's needs."""
    L, failures = _lib.lib(), []
    gate = threading.Barrier(n_threads)

    def work(i):
        E = (1024, 520)[i % 2]
        stream = torch.cuda.Stream()
        ids = torch.randint(0, E, (64,), dtype=torch.int32, generator=_gen(i)).to(cuda)
        order, place = torch.empty_like(ids), torch.empty_like(ids)
        offsets = torch.empty(E + 1, dtype=torch.int32, device=cuda)
        logits = torch.randn(16, E, device=cuda)
        chosen, weights = torch.empty(16, 4, dtype=torch.int32, device=cuda), torch.empty(16, 4, device=cuda)
        torch.cuda.synchronize()
        gate.wait()
        for _ in range(20000):
            if what == "plan":
                status = L.mq_expert_plan(ids.data_ptr(), 64, E, 0, offsets.data_ptr(), order.data_ptr(), place.data_ptr(), None, 0, stream.cuda_stream)
            else:
                status = L.mq_route_tokens(logits.data_ptr(), 0, 16, E, E, 4, 1, None, 1, 1, 0, 1, 1.0, chosen.data_ptr(), weights.data_ptr(),
                                           stream.cuda_stream)
            if status:
                failures.append((E, L.mq_last_error()))
        stream.synchronize()
        right = torch.equal(order.long(), torch.sort(ids, stable=True)[1]) if what == "plan" else torch.equal(
            chosen.long(), torch.sort(logits, descending=True, stable=True)[1][:, :4])
        if not right:
            failures.append((E, "wrong result"))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(n_threads)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failures, (len(failures), failures[0])
