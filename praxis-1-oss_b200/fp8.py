"""Routed and shared experts whose weights are held in block-scaled FP8.

``B200FP8RoutedExperts`` is the routed bank for checkpoints that store their
expert weights as E4M3 values with one fp32 scale per 128 x 128 block. It
implements the routed-bank protocol of :mod:`bank` (the one that
``MoEFeedForward._routed_tail`` calls, praxis/layers.py:2230-2270), so it
stands where ``B200NVFP4RoutedExperts`` does; ``FP8SharedExpert`` is the
shared expert (praxis/layers.py:1033-1089) in the same format. Activations are
quantized inside each call (``ops.fp8_quantize``); the forward runs on the
GPU through the C ABI, there is no CPU path.
"""

from __future__ import annotations

import math
from collections.abc import Mapping

import torch
from torch import Tensor, nn

from . import ops

_ROUTED_NAMES = frozenset(("gate_up_q", "gate_up_scale", "down_q", "down_scale"))


def _any_nan(codes: Tensor) -> bool:
    """Whether E4M3 codes hold a NaN; in pieces of 16 MB, since a bank may fill
    most of its device."""
    pieces = codes.view(torch.uint8).flatten().split(2**24)
    return bool(torch.stack([((piece & 0x7F) == 0x7F).any() for piece in pieces]).any())


def _validate(state: Mapping[str, Tensor], ndim: int) -> tuple[int, int, int]:
    """(E, C, F) of a gate/up and a down weight [.., 2F, C] and [.., C, F]."""
    if not isinstance(state, Mapping) or set(state) != _ROUTED_NAMES:
        raise ValueError("Unexpected FP8 packed buffer keys")
    if any(not isinstance(v, Tensor) or v.layout != torch.strided or not v.is_contiguous() or v.requires_grad
           for v in state.values()):
        raise ValueError("Reconstruction requires contiguous detached buffers")
    gu = state["gate_up_q"]
    if gu.ndim != ndim:
        raise ValueError("Expected grouped gate/up packed matrix" if ndim == 3 else "Expected a gate/up packed matrix")
    lead, (n, c) = tuple(gu.shape[:-2]), gu.shape[-2:]
    f = n // 2
    if 0 in gu.shape or n % 2 or c % 128 or f % 128:
        raise ValueError("Invalid FP8 expert dimensions: C and F must be multiples of 128")
    expected = {
        "gate_up_q": (lead + (2 * f, c), ops.F8),
        "gate_up_scale": (lead + (2 * f // 128, c // 128), torch.float32),
        "down_q": (lead + (c, f), ops.F8),
        "down_scale": (lead + (c // 128, f // 128), torch.float32),
    }
    for name, (shape, dtype) in expected.items():
        value = state[name]
        if tuple(value.shape) != shape or value.dtype != dtype:
            raise ValueError(f"Invalid FP8 buffer shape/dtype: {name}")
        if name.endswith("_scale") and not (torch.isfinite(value) & (value > 0)).all().item():
            raise ValueError(f"Invalid positive block scales: {name}")
        if name.endswith("_q") and _any_nan(value):
            raise ValueError(f"Invalid E4M3 values: {name}")
    return (lead[0] if lead else 1), c, f


class _FP8Experts(nn.Module):
    """The packed buffers: device moves, no dtype casts, inference only."""

    format = "fp8"

    def __init__(self, state: Mapping[str, Tensor], ndim: int) -> None:
        super().__init__()
        self.num_experts, self.in_features, self.hidden_features = _validate(state, ndim)
        for name in sorted(_ROUTED_NAMES):
            self.register_buffer(name, state[name].detach())
        super().train(False)

    def train(self, mode: bool = True):
        if mode:
            raise RuntimeError("FP8 experts support inference only")
        super().train(False)
        return self

    def _apply(self, fn, recurse: bool = True):
        moved = {name: fn(value) for name, value in self._buffers.items()}
        for name, value in self._buffers.items():
            if moved[name].dtype != value.dtype or moved[name].shape != value.shape:
                raise TypeError("FP8 buffers support device moves, not dtype/shape casts")
        self._buffers.update(moved)
        return self

    def weights(self) -> tuple[Tensor, Tensor, Tensor, Tensor]:
        """(gate_up_q, gate_up_scale, down_q, down_scale), as the kernels read them."""
        return self.gate_up_q, self.gate_up_scale, self.down_q, self.down_scale


class B200FP8RoutedExperts(_FP8Experts):
    """Routed experts on block-scaled FP8 weights: gate_up_q [E, 2F, C] (gate
    rows, then up rows), down_q [E, C, F], E4M3, with fp32 scales
    [E, 2F/128, C/128] and [E, C/128, F/128]. The kernels read the buffers as
    they are stored."""

    backend = "b200_sm100a_tcgen05_fp8"
    ACCEPTS_DISPATCH = False

    def __init__(self, state: Mapping[str, Tensor]) -> None:
        super().__init__(state, 3)

    @classmethod
    def from_packed(cls, state: Mapping[str, Tensor]) -> B200FP8RoutedExperts:
        return cls(state)

    def prepare(self) -> None:
        """Nothing to lay out (the NVFP4 bank interleaves its gate/up rows here)."""

    def routed_forward(self, x: Tensor, top_idx: Tensor, gate: Tensor, *, scaling: float, chunk_size: int,
                       dispatch=None) -> Tensor:
        """The scaled routed sum with the bf16 output boundary."""
        return self._routed_forward(x, top_idx, gate, scaling=scaling, chunk_size=chunk_size)

    def routed_forward_with_shared(self, x: Tensor, top_idx: Tensor, gate: Tensor, *, scaling: float,
                                   chunk_size: int, shared: Tensor, dispatch=None) -> Tensor:
        """Adds the shared expert after rounding the routed sum to bf16."""
        if (
            shared.shape != x.shape
            or shared.dtype != x.dtype
            or shared.device != x.device
            or not shared.is_contiguous()
            or (torch.is_grad_enabled() and shared.requires_grad)
        ):
            return self.routed_forward(x, top_idx, gate, scaling=scaling, chunk_size=chunk_size) + shared
        return self._routed_forward(x, top_idx, gate, scaling=scaling, chunk_size=chunk_size, shared=shared)

    def forward(self, x: Tensor, top_idx: Tensor, gate: Tensor, *, scaling: float, chunk_size: int) -> Tensor:
        return self.routed_forward(x, top_idx, gate, scaling=scaling, chunk_size=chunk_size)

    def _check(self, x, top_idx, gate, scaling, chunk_size) -> None:
        if torch.is_grad_enabled() and (x.requires_grad or gate.requires_grad):
            raise RuntimeError("FP8 routed experts support inference only")
        if type(chunk_size) is not int or chunk_size <= 0:
            raise ValueError("FP8 inference requires a positive dispatch chunk size")
        if isinstance(scaling, bool) or not isinstance(scaling, float | int) or not math.isfinite(scaling):
            raise ValueError("Routed scaling must be finite")
        # once for the whole call: a chunk's slices would hide rows of a longer tensor
        if x.ndim != 2 or top_idx.ndim != 2 or top_idx.shape[0] != x.shape[0] or gate.shape != top_idx.shape:
            raise ValueError("Expected routed activations [T, C] with expert indices and gates [T, k]")

    def _routed_forward(self, x: Tensor, top_idx: Tensor, gate: Tensor, *, scaling: float, chunk_size: int,
                        shared: Tensor | None = None) -> Tensor:
        self._check(x, top_idx, gate, scaling, chunk_size)
        if x.shape[0] <= chunk_size:
            return ops.fp8_moe_forward(x, top_idx, gate, *self.weights(), float(scaling), shared)
        out = torch.empty_like(x)
        for start in range(0, x.shape[0], chunk_size):
            end = min(start + chunk_size, x.shape[0])
            ops.fp8_moe_forward(x[start:end], top_idx[start:end], gate[start:end], *self.weights(), float(scaling),
                                None if shared is None else shared[start:end], out=out[start:end])
        return out

    def routed_forward_tail(self, x: Tensor, top_idx: Tensor, gate: Tensor, *, scaling: float, chunk_size: int,
                            tail: ops.Tail, shared: Tensor | None = None) -> tuple[Tensor, Tensor | None]:
        """:func:`bank.routed_forward_tail` for this bank."""
        self._check(x, top_idx, gate, scaling, chunk_size)
        if tail.residual.shape != x.shape:
            raise ValueError("Expected a contiguous BF16 residual shaped like the routed activations")
        if shared is not None and (shared.shape != x.shape or shared.dtype != x.dtype or not shared.is_contiguous()):
            raise ValueError("Expected a contiguous BF16 shared-expert output shaped like the activations")
        residual_out = torch.empty_like(x)
        normed = None if tail.norm_weight is None else torch.empty_like(x)
        for start in range(0, x.shape[0], chunk_size):
            end = min(start + chunk_size, x.shape[0])
            ops.fp8_moe_forward(
                x[start:end], top_idx[start:end], gate[start:end], *self.weights(), float(scaling),
                None if shared is None else shared[start:end], tail=tail.chunk(start, end),
                tail_out=(residual_out[start:end], None if normed is None else normed[start:end]))
        return residual_out, normed


class FP8SharedExpert(_FP8Experts):
    """The always-on dense SwiGLU expert on block-scaled FP8 weights:
    gate_up_q [2F, C], down_q [C, F]."""

    def __init__(self, state: Mapping[str, Tensor]) -> None:
        super().__init__(state, 2)

    @classmethod
    def from_weights(cls, gate_up: Tensor, down: Tensor) -> FP8SharedExpert:
        """From the bf16 matrices of ``SharedExpert``: gate_up [C, 2F], down [F, C]."""
        return cls(_pack(gate_up, down))

    def forward(self, x: Tensor, out: Tensor | None = None) -> Tensor:
        return ops.fp8_mlp(x, *self.weights(), out=out)


def _pack(gate_up: Tensor, down: Tensor) -> dict:
    with torch.no_grad():
        gate_up_q, gate_up_scale = ops.fp8_pack_weights(gate_up.detach().to(torch.bfloat16).contiguous())
        down_q, down_scale = ops.fp8_pack_weights(down.detach().to(torch.bfloat16).contiguous())
    return dict(gate_up_q=gate_up_q, gate_up_scale=gate_up_scale, down_q=down_q, down_scale=down_scale)


def pack_routed_experts_fp8(gate_up_weight: Tensor, down_weight: Tensor) -> B200FP8RoutedExperts:
    """Packs expert-first bf16 CUDA banks [E, C, 2F] / [E, F, C] (the layout of
    ``pack_routed_experts``) on their device."""
    for weight in (gate_up_weight, down_weight):
        if not isinstance(weight, Tensor) or weight.ndim != 3 or weight.dtype != torch.bfloat16:
            raise ValueError("Packing requires real BF16 expert-first banks")
    e, c, doubled = gate_up_weight.shape
    f = doubled // 2
    if e <= 0 or c <= 0 or f <= 0 or doubled % 2 or c % 128 or f % 128 or tuple(down_weight.shape) != (e, f, c):
        raise ValueError("Inconsistent routed banks; C and F must be multiples of 128")
    return B200FP8RoutedExperts(_pack(gate_up_weight, down_weight))
