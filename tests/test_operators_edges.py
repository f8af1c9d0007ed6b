"""Operators of the quantized layers at the ends of what they take: what needs no device.  Refusals are decided on the host, before any launch."""
import copy

import numpy as np
import pytest
import torch
import torch.nn as nn
from torch.autograd import forward_ad

from moe_quant_b200 import Int8Experts, Int8Linear, _lib, block_driver, ops
from moe_quant_b200._lib import MoeQuantError
from moe_quant_b200.int8 import int8_block
from moe_quant_b200.synthetic_block import SyntheticMoEBlock
from tests.test_operators import P, _experts, _results, _status


@pytest.mark.parametrize("K", [2 ** 30 + 1, 2 ** 31 - 16384, 2 ** 31 - 1, 2 ** 31, 2 ** 40])
def test_rows_longer_than_the_kernel_counts_are_refused(K):
    """Columns are counted in 32 bits in steps of up to 16384, and looked at up to as many behind the last step: near 2^31 the count would wrap."""
    status, message = _status("mq_quantize_tokens", P, 1, 1, K, K, P, K, P, None)
    assert status == 3 and b"2^30" in message


@pytest.mark.parametrize("first, status", [(2 ** 31 - 9, 0), (2 ** 31 - 8, 1), (2 ** 31 - 1, 1), (2 ** 31, 1), (2 ** 62, 1)])
def test_experts_are_numbered_below_the_largest_id(first, status):
    """Ids of 64 bits that lie outside 32 are clamped to their ends, which must not be an expert's number.  (Accepted calls are refused for their workspace next: nothing is launched.)"""
    if status == 0:
        assert _status("mq_expert_plan", P, 10 ** 6, 8, first, P, P, P, None, 0, None)[0] == 4
        assert _experts(first=first, E=8, ws=None)[0] == 4
    else:
        assert _status("mq_expert_plan", P, 10 ** 6, 8, first, P, P, P, None, 0, None)[0] == status
        assert _experts(first=first, E=8, ws=None)[0] == status


# ------------------------------------------------------------------ codes of 16-bit values
@pytest.mark.parametrize("bits", [8, 11])
def test_codes_of_every_pair_of_significands(bits):
    """The kernel's arithmetic for bf16 (8 bits of significand) and fp16 (11), step by step in fp32: x * (127 / top), rounded to 20 bits, plus
    1.5 * 2^23.  Against round-half-even of 127 x / top in integers, for every significand of x and of the row's largest value, and every power of two
    between them up to the one from which all codes are zero.  (Powers of two that both share change no step.)"""
    half = 1 << bits - 1
    ties = 0
    for top in range(half, 2 * half):
        for down in range(9):
            x = np.arange(half, 2 * half, dtype=np.int64)
            x = x[x <= top << down]           # x / 2^down is at most top
            inv = np.float32(127.0) / np.float32(top)
            product = (x.astype(np.float32) * np.float32(2.0 ** -down)) * inv
            rounded = ((product.view(np.uint32) + np.uint32(8)) & ~np.uint32(15)).view(np.float32)
            code = (rounded + np.float32(12582912.0)) - np.float32(12582912.0)
            over, under = 127 * x, top << down
            whole, rest = over // under, over % under
            want = whole + ((2 * rest > under) | ((2 * rest == under) & (whole % 2 == 1)))
            ties += int((2 * rest == under).sum())
            assert np.array_equal(code.astype(np.int64), want), (top, down)
    assert ties > 0


# ------------------------------------------------------------------ the block driver
class _Handle:
    """Stands in for a GPTQ handle: keeps the layer's weight, with codes of one group per row."""

    issue_zero_samples = issue_nan_hessian = issue_non_invertible = False

    def __init__(self, layer, *args, **kwargs):
        self.layer = layer

    def update(self, x):
        pass

    def reset(self):
        pass


def _results_of(handles, bits, streams=8, want_error=False):
    out = []
    for h in handles:
        rows, cols = h.layer.weight.shape
        out.append((torch.full((rows, cols), 130, dtype=torch.uint8), torch.full((rows, 1), 0.01), torch.full((rows, 1), 128.0)))
    return (out, [None] * len(out)) if want_error else out


@pytest.mark.parametrize("code", [0, 94])
def test_block_driver_reports_a_wait_that_ran_out_in_the_integer_products(monkeypatch, code):
    """The kernels of the served block leave what memory held when a wait runs out, finite or not: outputs are given only after the word that waits
    record their codes in has been read."""
    monkeypatch.setattr(block_driver, "GPTQ", _Handle)
    monkeypatch.setattr(block_driver, "quantize_shared", _results_of)
    monkeypatch.setattr(block_driver, "quantize_many", _results_of)
    monkeypatch.setattr(block_driver.quant_utils, "dequantize_linear_weight", lambda q, s, z: (q.float() - z) * s)
    monkeypatch.setattr(ops, "int8_matmul", lambda x, w, s, bias=None: x @ (w.to(x.dtype) * s[:, None].to(x.dtype)).t())
    asked = []
    monkeypatch.setattr(_lib, "engine_fault", lambda: asked.append(1) or code)
    block = nn.Sequential(nn.Linear(32, 16, bias=False), nn.Linear(16, 32, bias=False))
    run = lambda **kw: block_driver.quantize_block(block, [torch.ones(4, 32)], bits=8, group_size=None, **kw)
    run()
    assert not asked
    if code:
        with pytest.raises(MoeQuantError, match="bounded wait .code 94"):
            run(int8_outputs=True)
    else:
        assert run(int8_outputs=True)["outputs"][0].shape == (4, 32)
    assert asked


# ------------------------------------------------------------------ the modules
def _layer(rows, cols, seed):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(0, 256, (rows, cols), dtype=torch.uint8, generator=g), 0.01 * torch.rand(rows, 1, generator=g) + 0.003


def _modules():
    experts = Int8Experts([_layer(12, 20, i) for i in range(3)], [_layer(12, 20, 10 + i) for i in range(3)], [_layer(20, 12, 20 + i) for i in range(3)])
    return Int8Linear(*_layer(9, 20, 5), bias=torch.linspace(-1, 1, 9) / 3), experts


@pytest.mark.parametrize("convert", [lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.double(), lambda m: nn.Sequential(m).bfloat16()[0],
                                     lambda m: m.to("cpu", torch.float16)])
def test_conversions_leave_scales_alone(convert):
    """They are fp32 numbers, whose rounding to fewer bits would go into every result."""
    for was, now in zip(_modules(), [convert(m) for m in _modules()]):
        for name, buffer in was.named_buffers():
            assert now.get_buffer(name).dtype == buffer.dtype and torch.equal(now.get_buffer(name), buffer), name


def test_scales_follow_their_module_to_other_devices():
    for m in _modules():
        assert {b.device.type for b in m.to("meta", torch.bfloat16).buffers()} == {"meta"}


@pytest.mark.parametrize("move", [lambda m: m.to("meta"), lambda m: m.to("meta", torch.float16), copy.deepcopy, lambda m: m._apply(torch.clone)])
def test_rows_of_codes_keep_their_padding_on_the_way(move):
    """Rows start 16 bytes apart or a multiple of it, also of a module that was built on one device and moved to another."""
    linear, experts = _modules()
    for codes in (linear.codes, experts.gate_up, experts.down):
        assert codes.stride()[-2:] == (-(-codes.shape[-1] // 16) * 16, 1)
    shapes = linear.codes.shape, experts.gate_up.shape, experts.down.shape
    strides = linear.codes.stride(), experts.gate_up.stride(), experts.down.stride()
    linear, experts = move(linear), move(experts)
    assert shapes == (linear.codes.shape, experts.gate_up.shape, experts.down.shape)
    assert strides == (linear.codes.stride(), experts.gate_up.stride(), experts.down.stride())


@pytest.mark.parametrize("side, expert, shape", [(0, 1, (12, 24)), (1, 2, (12, 24)), (1, 0, (16, 20)), (2, 1, (20, 14)), (2, slice(None), (20, 14)), (2, 0, (21, 12))])
def test_experts_of_unlike_sizes_are_refused(side, expert, shape):
    """Also where the padded rows have one length."""
    sides = [[_layer(12, 20, i) for i in range(3)], [_layer(12, 20, i) for i in range(3)], [_layer(20, 12, i) for i in range(3)]]
    Int8Experts(*sides)
    for i in range(3)[expert] if isinstance(expert, slice) else [expert]:
        sides[side][i] = _layer(*shape, i)
    with pytest.raises(MoeQuantError, match="Int8Experts"):
        Int8Experts(*sides)


def test_tangents_are_refused():
    """A result without its tangent would be taken for a constant."""
    x, w = torch.zeros(2, 16), torch.ones(3)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        for call in (lambda: ops._forward_only("op", dual, None), lambda: ops._forward_only("op", x, None, dual[:1])):
            with pytest.raises(MoeQuantError, match="tangents"):
                call()
            with torch.no_grad(), pytest.raises(MoeQuantError, match="tangents"):
                call()
        ops._forward_only("op", x, None, w, forward_ad.unpack_dual(dual).primal)
    ops._forward_only("op", x, None, w)


# ------------------------------------------------------------------ blocks whose layers are swapped
def _block():
    return SyntheticMoEBlock(hidden=32, inter=16, n_experts=4, top_k=2, q_rank=16, kv_rank=16, n_heads=2, nope_dim=8, rope_dim=8, v_dim=8)


def test_experts_with_biases_keep_them():
    block = _block()
    block.mlp.experts[1].up_proj.bias = nn.Parameter(torch.linspace(-1, 1, 16))
    with int8_block(block, _results(block)):
        assert block.mlp.int8_experts is None
        assert torch.equal(block.mlp.experts[1].up_proj.bias, torch.linspace(-1, 1, 16)) and block.mlp.experts[0].up_proj.bias is None
        assert all(isinstance(getattr(e, side), Int8Linear) for e in block.mlp.experts for side in ("gate_proj", "up_proj", "down_proj"))


def test_experts_that_were_there_before_come_back():
    block = _block()
    block.mlp.int8_experts = mine = Int8Experts(*([r] * 4 for r in (_layer(16, 32, 0), _layer(16, 32, 1), _layer(32, 16, 2))))
    with int8_block(block, _results(block)):
        assert isinstance(block.mlp.int8_experts, Int8Experts) and block.mlp.int8_experts is not mine
        with int8_block(block, _results(block)):
            pass
        assert block.mlp.int8_experts is not None and block.mlp.int8_experts is not mine
    assert block.mlp.int8_experts is mine


def test_experts_with_other_layers_run_layer_by_layer():
    """What int8_experts computes is a gated MLP of three projections; a fourth layer would be left out."""
    block = _block()
    block.mlp.experts[2].mix_proj = nn.Linear(16, 16, bias=False)
    with int8_block(block, _results(block)):
        assert block.mlp.int8_experts is None
        assert isinstance(block.mlp.experts[2].mix_proj, Int8Linear) and isinstance(block.mlp.experts[0].gate_proj, Int8Linear)
    assert isinstance(block.mlp.experts[2].mix_proj, nn.Linear)


def test_hooks_of_swapped_layers_fire(monkeypatch):
    monkeypatch.setattr(ops, "int8_matmul", lambda x, w, s, bias=None: x @ (w.to(x.dtype) * s[:, None].to(x.dtype)).t())
    block, seen = _block(), []
    layer = block.mlp.shared_experts.up_proj
    layer.register_forward_hook(lambda m, i, o: seen.append(("after", type(m))))
    layer.register_forward_pre_hook(lambda m, args, kwargs: seen.append(("before", type(m))), with_kwargs=True)
    x = torch.ones(2, 32)
    with int8_block(block, _results(block)):
        swapped = block.mlp.shared_experts.up_proj
        swapped(x)
        assert seen == [("before", Int8Linear), ("after", Int8Linear)]
        late = swapped.register_forward_hook(lambda m, i, o: seen.append("late"))
        swapped(x)
        assert seen.pop() == "late"
        late.remove()
    del seen[:]
    block.mlp.shared_experts.up_proj(x)
    assert seen == [("before", nn.Linear), ("after", nn.Linear)]


@pytest.mark.parametrize("where", ["", "down_proj"])
def test_experts_with_hooks_run_layer_by_layer(where):
    block = _block()
    handle = block.mlp.experts[3].get_submodule(where).register_forward_hook(lambda m, i, o: None)
    with int8_block(block, _results(block)):
        assert block.mlp.int8_experts is None and isinstance(block.mlp.experts[3].down_proj, Int8Linear)
    handle.remove()
    with int8_block(block, _results(block)):
        assert block.mlp.int8_experts is not None


@pytest.mark.parametrize("scale_type", [torch.float32, torch.bfloat16])
def test_experts_that_were_there_before_do_not_stand_in_for_new_ones(scale_type):
    """Experts that run layer by layer (here of fp32 layers, or with a hook) do so although the module had some of its own."""
    block = _block()
    block.mlp.int8_experts = mine = Int8Experts(*([r] * 4 for r in (_layer(16, 32, 0), _layer(16, 32, 1), _layer(32, 16, 2))))
    if scale_type != torch.float32:
        block.mlp.experts[0].register_forward_hook(lambda m, i, o: None)
    with int8_block(block, {n: (q, s.to(scale_type), z) for n, (q, s, z) in _results(block).items()}):
        assert block.mlp.int8_experts is None
    assert block.mlp.int8_experts is mine
    with int8_block(block, {n: r for n, r in _results(block).items() if "experts." not in n}):
        assert block.mlp.int8_experts is mine
    assert block.mlp.int8_experts is mine
