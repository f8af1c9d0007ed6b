"""Operators of the quantized layers: what needs no device.  Refusals are decided on the host, before any launch."""
import math
import os
import re

import pytest
import torch
import torch.nn as nn

from moe_quant_b200 import Int8Experts, Int8Linear, _lib, int8_layout, ops
from moe_quant_b200._lib import MoeQuantError
from moe_quant_b200.block_driver import quantize_block
from moe_quant_b200.int8 import int8_block
from moe_quant_b200.synthetic_block import SyntheticMoEBlock
from tests import operator_reference as R

P = 4096   # an address that is aligned and never read: every call here is refused on the host


def _status(name, *args):
    L = _lib.lib()
    return getattr(L, name)(*args), L.mq_last_error()


# ------------------------------------------------------------------ argument checks of the entry points
def _route(dtype=0, T=4, E=64, ld=64, k=8, score=1, bias=None, groups=8, keep=4, group_score=1, logits=P, ids=P, weights=P):
    return _status("mq_route_tokens", logits, dtype, T, E, ld, k, score, bias, groups, keep, group_score, 1, 1.0, ids, weights, None)


@pytest.mark.parametrize("change, status", [
    ({"dtype": 3}, 1), ({"T": -1}, 1), ({"E": 0}, 1), ({"ld": 63}, 1), ({"E": 1025, "ld": 1025, "groups": 1, "keep": 1}, 3), ({"k": 0}, 1), ({"k": 33}, 1),
    ({"E": 6, "groups": 1, "keep": 1, "k": 7}, 1), ({"score": 2}, 1), ({"group_score": -1}, 1), ({"groups": 0}, 1), ({"groups": 7}, 1),
    ({"groups": 64, "keep": 64}, 1), ({"keep": 0}, 1), ({"keep": 9}, 1), ({"logits": None}, 1), ({"ids": None}, 1), ({"weights": None}, 1)])
def test_route_refusals(change, status):
    assert _route(**change)[0] == status


def test_empty_calls_launch_nothing():
    assert _route(T=0, logits=None, ids=None, weights=None)[0] == 0
    assert _status("mq_quantize_tokens", None, 1, 0, 16, 16, None, 16, None, None)[0] == 0
    assert _status("mq_int8_matmul", None, 1, None, 0, 16, 16, P, 8, 16, P, None, 1, None, 8, None, 0, None)[0] == 0
    assert _status("mq_int8_matmul", P, 1, None, 4, 16, 16, None, 0, 16, None, None, 1, None, 0, None, 0, None)[0] == 0
    assert _experts(T=0)[0] == 0


@pytest.mark.parametrize("change, status", [
    ({"pairs": -1}, 1), ({"E": 0}, 1), ({"E": 1025}, 3), ({"pairs": 2 ** 31}, 3), ({"first": -1}, 1), ({"offsets": None}, 1), ({"ids": None}, 1),
    ({"pairs": 10 ** 6, "ws": None, "bytes": 0}, 4)])
def test_plan_refusals(change, status):
    a = {"ids": P, "pairs": 100, "E": 8, "first": 0, "offsets": P, "order": P, "place": P, "ws": P, "bytes": 1 << 30, **change}
    assert _status("mq_expert_plan", *a.values(), None)[0] == status


@pytest.mark.parametrize("change, status", [
    ({"dtype": 3}, 1), ({"dtype": -1}, 1), ({"T": -1}, 1), ({"K": 0}, 1), ({"ldx": 15}, 1), ({"ldc": 15}, 1), ({"x": None}, 1), ({"scale": None}, 1)])
def test_quantize_refusals(change, status):
    a = {"x": P, "dtype": 1, "T": 4, "K": 16, "ldx": 16, "codes": P, "ldc": 16, "scale": P, **change}
    assert _status("mq_quantize_tokens", *a.values(), None)[0] == status


@pytest.mark.parametrize("change, status", [
    ({"x_dtype": 4}, 1), ({"out_dtype": 3}, 1), ({"T": -1}, 1), ({"N": -1}, 1), ({"K": 0}, 1), ({"ldx": 60}, 1), ({"ldw": 60}, 1), ({"ldy": 7}, 1),
    ({"K": 131088, "ldx": 131088, "ldw": 131088}, 3), ({"T": 2 ** 31}, 3), ({"N": 2 ** 31, "ldy": 2 ** 31}, 3), ({"x": None}, 1), ({"w": None}, 1),
    ({"w_scale": None}, 1), ({"y": None}, 1), ({"x_dtype": 3}, 1), ({"w": P + 8}, 2), ({"ldw": 72}, 2), ({"x_dtype": 3, "x_scale": P, "x": P + 8}, 2),
    ({"x_dtype": 3, "x_scale": P, "ldx": 72}, 2), ({"x_dtype": 3, "x_scale": P, "K": 131072, "ldx": 131072, "ldw": 131072}, 3), ({"ws": None}, 4), ({"bytes": 16}, 4), ({"ws": P + 8}, 4)])
def test_matmul_refusals(change, status):
    a = {"x": P, "x_dtype": 1, "x_scale": None, "T": 40, "K": 64, "ldx": 64, "w": P, "N": 8, "ldw": 64, "w_scale": P, "bias": None, "out_dtype": 1,
         "y": P, "ldy": 8, "ws": P, "bytes": 1 << 30, **change}
    assert _status("mq_int8_matmul", *a.values(), None)[0] == status


def _experts(**change):
    a = {"x": P, "dtype": 1, "T": 40, "K": 64, "ldx": 64, "ids": P, "weights": P, "k": 2, "first": 0, "E": 4, "I": 32, "gate_up": P, "ld_gu": 64,
         "gu_expert": 4096, "gu_scale": P, "down": P, "ld_down": 32, "down_expert": 2048, "down_scale": P, "y": P, "ldy": 64, "ws": P, "bytes": 1 << 30, **change}
    return _status("mq_int8_experts", *a.values(), None)


@pytest.mark.parametrize("change, status", [
    ({"dtype": 0}, 1), ({"dtype": 3}, 1), ({"T": -1}, 1), ({"K": 0}, 1), ({"I": 0}, 1), ({"E": 0}, 1), ({"k": 0}, 1), ({"k": 33}, 1), ({"first": -1}, 1),
    ({"ldx": 63}, 1), ({"ldy": 63}, 1), ({"ld_gu": 48}, 1), ({"ld_down": 16}, 1), ({"gu_expert": -16}, 1), ({"E": 1025}, 3), ({"T": 2 ** 30}, 3),
    ({"K": 131088, "ldx": 131088, "ld_gu": 131088, "ldy": 131088}, 3), ({"I": 131088, "ld_down": 131088}, 3), ({"x": None}, 1), ({"ids": None}, 1),
    ({"weights": None}, 1), ({"gate_up": None}, 1), ({"down_scale": None}, 1), ({"y": None}, 1), ({"gate_up": P + 8}, 2), ({"down": P + 4}, 2),
    ({"ld_gu": 72}, 2), ({"ld_down": 40}, 2), ({"gu_expert": 4104}, 2), ({"down_expert": 2056}, 2), ({"ws": None}, 4), ({"bytes": 100}, 4)])
def test_experts_refusals(change, status):
    assert _experts(**change)[0] == status


def test_there_is_no_cpu_path():
    w, s = torch.zeros(8, 16, dtype=torch.int8), torch.ones(8)
    for call in (lambda: ops.route_tokens(torch.zeros(2, 8), 2), lambda: ops.expert_plan(torch.zeros(2, 2, dtype=torch.int32), 4),
                 lambda: ops.quantize_tokens(torch.zeros(2, 16)), lambda: ops.int8_matmul(torch.zeros(2, 16), w, s),
                 lambda: ops.int8_experts(torch.zeros(2, 16).half(), torch.zeros(2, 2, dtype=torch.int32), torch.ones(2, 2), w[None], s[None], w[None], s[None])):
        with pytest.raises(MoeQuantError, match="CUDA"):
            call()


# ------------------------------------------------------------------ layouts and modules
def test_int8_layout():
    q = torch.randint(0, 256, (5, 24), dtype=torch.uint8)
    codes, scale = int8_layout(q, torch.full((5, 1), 0.5, dtype=torch.bfloat16), torch.full((5, 1), 128.0))
    assert codes.dtype == torch.int8 and codes.shape == (5, 24) and codes.stride() == (32, 1)
    assert torch.equal(codes.int(), q.int() - 128)
    assert scale.dtype == torch.float32 and scale.shape == (5,)


def test_int8_layout_refusals():
    q, s = torch.zeros(4, 16, dtype=torch.uint8), torch.ones(4, 1)
    with pytest.raises(MoeQuantError, match="one group per row"):
        int8_layout(q, torch.ones(4, 2))
    with pytest.raises(MoeQuantError, match="128"):
        int8_layout(q, s, torch.full((4, 1), 8.0))
    with pytest.raises(MoeQuantError, match="uint8"):
        int8_layout(q.int(), s)
    with pytest.raises(MoeQuantError):
        Int8Experts([], [], [])


def test_int8_experts_stacks_gate_rows_before_up_rows():
    def layer(rows, cols, seed):
        return torch.randint(0, 256, (rows, cols), dtype=torch.uint8, generator=torch.Generator().manual_seed(seed)), torch.full((rows, 1), 1.0 + seed)
    m = Int8Experts([layer(8, 24, 0), layer(8, 24, 1)], [layer(8, 24, 2), layer(8, 24, 3)], [layer(24, 8, 4), layer(24, 8, 5)], first=6)
    assert m.gate_up.shape == (2, 16, 24) and m.down.shape == (2, 24, 8) and m.first == 6
    assert m.gate_up.stride(1) % 16 == 0 and m.down.stride(1) % 16 == 0
    assert torch.equal(m.gate_up[1, 8:].int(), layer(8, 24, 3)[0].int() - 128)
    assert m.gate_up_scale[1].tolist() == [2.0] * 8 + [4.0] * 8
    assert not list(m.parameters()) and not m.state_dict()


def _results(block):
    return {n: (torch.randint(0, 256, l.weight.shape, dtype=torch.uint8), torch.ones(l.weight.shape[0], 1, dtype=torch.bfloat16), torch.full((l.weight.shape[0], 1), 128.0))
            for n, l in block.named_modules() if isinstance(l, nn.Linear)}


def test_int8_block_swaps_layers_and_puts_them_back():
    block = SyntheticMoEBlock(hidden=32, inter=16, n_experts=4, top_k=2, q_rank=16, kv_rank=16, n_heads=2, nope_dim=8, rope_dim=8, v_dim=8)
    before = dict(block.named_modules())
    with int8_block(block, _results(block)):
        assert isinstance(block.self_attn.q_a_proj, Int8Linear) and isinstance(block.mlp.shared_experts.up_proj, Int8Linear)
        assert isinstance(block.mlp.int8_experts, Int8Experts) and block.mlp.int8_experts.gate_up.shape == (4, 32, 32)
        assert isinstance(block.mlp.experts[0].gate_proj, nn.Linear)      # not called
    assert dict(block.named_modules()) == before and block.mlp.int8_experts is None
    with int8_block(block, {}):
        assert dict(block.named_modules()) == before
    # an expert that was not quantized: the others become layers of their own
    results = _results(block)
    del results["mlp.experts.2.up_proj"]
    with int8_block(block, results):
        assert block.mlp.int8_experts is None and isinstance(block.mlp.experts[0].gate_proj, Int8Linear)
        assert isinstance(block.mlp.experts[2].up_proj, nn.Linear)
    assert dict(block.named_modules()) == before


def test_int8_block_of_fp32_layers_goes_layer_by_layer():
    block = SyntheticMoEBlock(hidden=32, inter=16, n_experts=2, top_k=1, q_rank=16, kv_rank=16, n_heads=2, nope_dim=8, rope_dim=8, v_dim=8)
    results = {n: (q, s.float(), z) for n, (q, s, z) in _results(block).items()}
    with int8_block(block, results):
        assert block.mlp.int8_experts is None and isinstance(block.mlp.experts[1].down_proj, Int8Linear)


def test_int8_block_puts_layers_back_after_an_error():
    block = SyntheticMoEBlock(hidden=32, inter=16, n_experts=2, top_k=1, q_rank=16, kv_rank=16, n_heads=2, nope_dim=8, rope_dim=8, v_dim=8)
    before = dict(block.named_modules())
    with pytest.raises(KeyError):
        with int8_block(block, _results(block)):
            raise KeyError
    assert dict(block.named_modules()) == before


def test_int8_outputs_need_eight_bits_per_channel():
    block = SyntheticMoEBlock(hidden=32, inter=16, n_experts=2, top_k=1, q_rank=16, kv_rank=16, n_heads=2, nope_dim=8, rope_dim=8, v_dim=8)
    for bits, group in ((4, None), (8, 128)):
        with pytest.raises(MoeQuantError, match="bits=8"):
            quantize_block(block, [], bits=bits, group_size=group, int8_outputs=True)


def test_only_elected_threads_wait_alone():
    """Waits of a single thread stand between its election and the point where its warp comes together again."""
    csrc = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "moe_quant_b200", "csrc")
    for name in sorted(n for n in os.listdir(csrc) if n.endswith((".cu", ".cuh")) and n != "mbarrier.cuh"):
        body = open(os.path.join(csrc, name)).read()
        for at in (m.start() for m in re.finditer(r"mbar_wait_elected\(", body)):
            elected, joined = body.rfind("elect_one())", 0, at), body.find("__syncwarp();", at)
            assert elected >= 0 and "__syncwarp" not in body[elected:at] and "_sync(" not in body[elected:joined], name


# ------------------------------------------------------------------ the reference itself
def test_reference_route_agrees_with_topk_where_that_is_defined():
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(50, 16, generator=g)
    ids, w = R.route(logits, 3, score="sigmoid")
    top, at = torch.sigmoid(logits.double()).topk(3)
    assert torch.equal(ids, at) and torch.allclose(w, top / top.sum(-1, keepdim=True), rtol=1e-12)
    ids, w = R.route(logits, 3, score="softmax", renormalise=False)
    top, at = torch.softmax(logits.double(), -1).topk(3)
    assert torch.equal(ids, at) and torch.allclose(w, top, rtol=1e-12)


def test_reference_codes():
    q, s = R.codes(torch.tensor([[127.0, 63.5, -0.5, 1.5], [0.0, 0.0, 0.0, 0.0], [1.0, math.inf, 0.0, 0.0]]))
    assert q.tolist() == [[127, 64, 0, 2], [0] * 4, [0] * 4]
    assert s[0] == 1 and s[1] == 0 and math.isnan(s[2])
