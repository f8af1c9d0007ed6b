"""Layers that run in 8-bit integers on what `GPTQ(layer, None, ...).quantize(8)` returns: codes of 8 bits with one scale per
output channel.  Activations get their codes token by token on the way in.  Forward only: the modules hold no
parameters, and their calls refuse inputs that ask for gradients.  Their buffers are not persistent: what is saved of a model is the
quantizer's codes, scales and zero points, from which the modules are built."""
from __future__ import annotations

import re
from contextlib import contextmanager
from typing import Mapping, Optional, Sequence, Tuple

import torch
import torch.nn as nn
from torch import Tensor

from . import ops
from ._lib import MoeQuantError


def int8_layout(qweight: Tensor, scale: Tensor, zero: Optional[Tensor] = None) -> Tuple[Tensor, Tensor]:
    """(int8 codes, fp32 scales) as ops.int8_matmul takes them, from the uint8 codes (R, C), the scales (R, 1) and the zero points of a
    symmetric 8-bit layer with one group per row.  Rows of the codes start 16 bytes apart or a multiple of it."""
    if qweight.dtype != torch.uint8 or qweight.dim() != 2:
        raise MoeQuantError("int8_layout: qweight must be a 2-D uint8 tensor")
    R, C = qweight.shape
    if scale.numel() != R:
        raise MoeQuantError(f"int8_layout: {scale.numel()} scales for {R} rows: quantize with one group per row (group_size None)")
    if zero is not None and not bool((zero == 128).all()):
        raise MoeQuantError("int8_layout: the zero point of 8-bit symmetric codes is 128")
    codes = torch.zeros(R, (C + 15) // 16 * 16, dtype=torch.uint8, device=qweight.device)[:, :C]
    torch.bitwise_xor(qweight, 128, out=codes)   # q - 128 in two's complement
    return codes.view(torch.int8), scale.reshape(R).to(torch.float32)


class _Int8Module(nn.Module):
    """Scales and biases stay in fp32 whatever type a module or the model around it is converted to: they follow it to other
    devices alone."""

    def _apply(self, fn, *args, **kwargs):
        kept = {n: b for n, b in self._buffers.items() if b is not None and b.is_floating_point()}
        super()._apply(fn, *args, **kwargs)
        for n, b in kept.items():
            if self._buffers[n].dtype != b.dtype:
                self._buffers[n] = b.to(self._buffers[n].device)
        return self


class Int8Linear(_Int8Module):
    """Stands in for an nn.Linear whose weight has been quantized to 8 bits per output channel."""

    def __init__(self, qweight: Tensor, scale: Tensor, zero: Optional[Tensor] = None, bias: Optional[Tensor] = None):
        super().__init__()
        codes, scale = int8_layout(qweight, scale, zero)
        self.out_features, self.in_features = codes.shape
        self.register_buffer("padded", _whole(codes), persistent=False)      # (a view would lose its row stride on the way to another device)
        self.register_buffer("scale", scale, persistent=False)
        self.register_buffer("bias", None if bias is None else bias.detach().to(torch.float32), persistent=False)

    @property
    def codes(self) -> Tensor:
        return _columns(self.padded, self.in_features)

    def forward(self, x: Tensor) -> Tensor:
        return ops.int8_matmul(x, self.codes, self.scale, bias=self.bias)


class Int8Experts(_Int8Module):
    """The gated MLPs of the experts first .. first + E - 1, one (qweight, scale, zero) per projection and expert."""

    def __init__(self, gate: Sequence, up: Sequence, down: Sequence, first: int = 0):
        super().__init__()
        if not len(gate) == len(up) == len(down) or not gate:
            raise MoeQuantError("Int8Experts: as many gate as up and down projections, and at least one")
        self.first = int(first)
        gates, ups, downs = ([int8_layout(*r) for r in side] for side in (gate, up, down))
        inner, hidden = gates[0][0].shape
        if any(c.shape != (inner, hidden) for c, _ in gates + ups) or any(c.shape != (hidden, inner) for c, _ in downs):
            raise MoeQuantError(f"Int8Experts: gate and up projections are not all {inner} x {hidden}, or down projections {hidden} x {inner}")
        both = [(torch.cat([_whole(g), _whole(u)]), torch.cat([gs, us])) for (g, gs), (u, us) in zip(gates, ups)]
        self.inner, self.hidden = inner, hidden
        self.register_buffer("padded_gate_up", torch.stack([c for c, _ in both]), persistent=False)
        self.register_buffer("gate_up_scale", torch.stack([s for _, s in both]), persistent=False)
        self.register_buffer("padded_down", torch.stack([_whole(c) for c, _ in downs]), persistent=False)
        self.register_buffer("down_scale", torch.stack([s for _, s in downs]), persistent=False)

    @property
    def gate_up(self) -> Tensor:
        return _columns(self.padded_gate_up, self.hidden)

    @property
    def down(self) -> Tensor:
        return _columns(self.padded_down, self.inner)

    def forward(self, x: Tensor, ids: Tensor, weights: Tensor) -> Tensor:
        return ops.int8_experts(x, ids, weights, self.gate_up, self.gate_up_scale, self.down, self.down_scale, first=self.first)


def _columns(padded: Tensor, n: int) -> Tensor:
    return padded if padded.shape[-1] == n else padded[..., :n]


def _whole(codes: Tensor) -> Tensor:
    """A view of the rows with their padding."""
    return codes.as_strided((codes.shape[0], codes.stride(0)), codes.stride())


_HOOKS = ("_forward_hooks", "_forward_hooks_with_kwargs", "_forward_hooks_always_called", "_forward_pre_hooks", "_forward_pre_hooks_with_kwargs")


@contextmanager
def int8_block(block: nn.Module, results: Mapping[str, Tuple[Tensor, Tensor, Tensor]]):
    """Within the context the block's quantized layers run in 8-bit integers: `results` maps their names to what quantize(8)
    returned.  A module whose experts are all among them, and which has a place for it (`int8_experts`), runs them through
    ops.int8_experts (in bf16 and fp16 blocks) if they are plain gated MLPs: three layers each, without biases or forward hooks.  Every
    other layer becomes an Int8Linear that keeps its bias and shares its forward hooks."""
    undo = []
    left = dict(results)
    try:
        for moe_name, moe in list(block.named_modules()):
            if not hasattr(moe, "int8_experts"):
                continue
            prefix = f"{moe_name}.experts." if moe_name else "experts."
            mine = {n[len(prefix):]: n for n in left if n.startswith(prefix)}
            ids = sorted({int(m.group(1)) for m in (re.fullmatch(r"(\d+)\.(gate|up|down)_proj", n) for n in mine) if m})
            sides = [[left.get(f"{prefix}{i}.{side}_proj") for i in ids] for side in ("gate", "up", "down")]
            local = [i for i, e in enumerate(moe.experts) if e is not None]
            if mine and moe.int8_experts is not None:      # of other weights
                undo.append((moe, "int8_experts", moe.int8_experts))
                moe.int8_experts = None
            if any(left[n][1].dtype == torch.float32 for n in mine.values()):
                continue
            biased = any(getattr(block.get_submodule(n), "bias", None) is not None for n in mine.values())     # (Int8Experts has none)
            others = len(mine) > 3 * len(ids)      # an expert with more layers than a gated MLP has
            hooked = any(m._forward_hooks or m._forward_pre_hooks for e in moe.experts if e is not None for m in e.modules())
            if biased or others or hooked or not ids or ids != local or ids != list(range(ids[0], ids[-1] + 1)) or any(r is None for side in sides for r in side):
                continue
            undo.append((moe, "int8_experts", None))
            moe.int8_experts = Int8Experts(*sides, first=ids[0])
            for n in mine.values():
                del left[n]
        for name, result in left.items():
            parent, _, leaf = name.rpartition(".")
            parent = block.get_submodule(parent)
            layer = getattr(parent, leaf)
            if not isinstance(layer, nn.Linear):
                raise MoeQuantError(f"int8_block: {name} is no nn.Linear")
            stand_in = Int8Linear(*result, bias=layer.bias)
            for hooks in _HOOKS:      # the same dicts: what is registered or removed meanwhile counts for both
                setattr(stand_in, hooks, getattr(layer, hooks))
            setattr(parent, leaf, stand_in)
            undo.append((parent, leaf, layer))
        yield block
    finally:
        for parent, leaf, was in reversed(undo):
            setattr(parent, leaf, was)
