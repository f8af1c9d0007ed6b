"""Operators of the quantized layers where their results could depend on what they should not."""
import pytest
import torch

from moe_quant_b200 import ops
from tests import operator_reference as R
from tests.test_gpu_operators import BF16, FP16, _experts_case, _gen, _on

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
