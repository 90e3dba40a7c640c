"""Block-scaled FP8 linears: E4M3 codes with one power-of-two scale for each
block of 128 columns, next to the per-tensor FP8 linears of runtime.fp8
(recavsr_infer/runtime/fp8.py:13-55).

A matrix held in 8 bits is a pair (codes, scales): u8 E4M3 codes [rows, cols]
and u8 E8M0 scale bytes (2^(e-127), the smallest with amax <= 448 * scale) in
the flat 128x4 blocked order the tensor core reads (as operands also in torch's
float8_e4m3fn and float8_e8m0fnu); scale_bytes() gives them as [rows, blocks]. Activations have a scale for each row's block of 128 columns,
weights one for each 128 x 128 block.

    codes, scales, hidden = rms_norm_quantize(x, weight, eps, residual=hidden)
    qkv = mm(codes, w_codes, scales, w_scales, bias)
    codes, scales = quantize(attention)
    hidden = mm(codes, w_codes, scales, w_scales, bias, residual=hidden)
    codes, scales = swiglu_mm(codes, gu_codes, scales, gu_scales, gu_bias)

Every function runs on the current stream of its inputs' device and allocates
only what it returns. There is no CPU path. None has a backward pass: codes carry
no gradient, and a floating-point result of inputs that require one raises in
backward (mm into `out` refuses such inputs, as torch's functions do).

A call goes straight to the binding; under torch.compile, or where a gradient
would be asked for (the binding answers NotImplemented), through a custom op.
"""
from __future__ import annotations

import torch
from torch import nn

try:
    from .. import _fp8_block as _binding
except ImportError as error:
    raise ImportError("recavsr_b200/_fp8_block.so cannot be loaded: build it with `python -m recavsr_b200.build` "
                      "(there is no CPU fallback)") from error

BLOCK = 128


def scale_numel(rows: int, cols: int) -> int:
    """Bytes of the scales of a [rows, cols] matrix."""
    return -(-rows // BLOCK) * BLOCK * (-(-cols // (4 * BLOCK)) * 4)


def scale_bytes(scales: torch.Tensor, rows: int, cols: int) -> torch.Tensor:
    """The flat scale bytes of a [rows, cols] matrix as u8 [rows, ceil(cols / 128)]."""
    mb, kt = -(-rows // BLOCK), -(-cols // (4 * BLOCK))
    full = scales.view(torch.uint8).reshape(mb, kt, 32, 4, 4).permute(0, 3, 2, 1, 4)
    return full.reshape(mb * BLOCK, kt * 4)[:rows, :-(-cols // BLOCK)]


def dequantize(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """The fp32 values [rows, cols] that codes and scales stand for."""
    rows, cols = codes.shape
    e = scale_bytes(scales, rows, cols).to(torch.int32)
    power = torch.where(e == 0, 1 << 22, e << 23).view(torch.float32)      # 2^-127 is a subnormal
    power = torch.where(e == 255, torch.nan, power)
    values = codes.view(torch.float8_e4m3fn).to(torch.float32)
    return values * power.repeat_interleave(BLOCK, 1)[:, :cols]


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (fp32 / bf16 / fp16, K a multiple of 16) -> (codes, scales)."""
    if torch.compiler.is_compiling():
        return torch.ops.recavsr_b200.fp8_block_quantize(x, False)
    return _binding.quantize(x, False)


def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weight [N, K] -> (codes, scales), one scale for each 128 x 128 block."""
    if torch.compiler.is_compiling():
        return torch.ops.recavsr_b200.fp8_block_quantize(weight, True)
    return _binding.quantize(weight, True)


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """RMSNorm of x (+ residual) held in 8 bits: (codes, scales, hidden).

    h = x + residual is summed in fp32; hidden is h rounded to x's dtype (None
    without a residual) and the norm h * rsqrt(mean(h^2) + eps) * weight is
    quantized from fp32, without a rounding between. Rows of at most 16384
    columns, a multiple of 16."""
    if torch.compiler.is_compiling():
        if residual is None:
            return (*torch.ops.recavsr_b200.fp8_block_rms_norm(x, weight, eps), None)
        return torch.ops.recavsr_b200.fp8_block_add_rms_norm(x, weight, eps, residual)
    result = _binding.rms_norm_quantize(x, weight, eps, residual)
    if result is NotImplemented:
        return torch.ops.recavsr_b200.fp8_block_add_rms_norm(x, weight, eps, residual)
    return result


def mm(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, weight_scales: torch.Tensor,
       bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
       dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, N] = A [M, K] . W [N, K]^T + bias (+ residual), summed in fp32 and
    rounded once to dtype (bfloat16 by default, or float16; the residual has the
    same). `out` may be `residual` itself; it shares memory with no other input."""
    result = NotImplemented
    if not torch.compiler.is_compiling():
        result = _binding.mm(values, weights, scales, weight_scales, bias, residual, dtype, out)
    if result is not NotImplemented:
        return result
    if out is None:
        return torch.ops.recavsr_b200.fp8_block_mm(values, weights, scales, weight_scales, bias, residual, dtype)
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in (bias, residual, out)):
        raise ValueError("fp8_block.mm: with out there is no gradient, but an argument requires one.")
    torch.ops.recavsr_b200.fp8_block_mm_out(values, weights, scales, weight_scales, bias, residual, dtype, out)
    return out


def interleave_gate_up(gate: torch.Tensor, up: torch.Tensor) -> torch.Tensor:
    """Gate and up rows (or biases) [H, ...] in swiglu_mm's order: groups of 128
    gate then 128 up rows, the last group filled up with zeros."""
    if gate.shape != up.shape:
        raise ValueError("gate and up must have the same shape.")
    h = gate.shape[0]
    hp = -(-h // BLOCK) * BLOCK
    both = gate.new_zeros((2, hp, *gate.shape[1:]))
    both[0, :h], both[1, :h] = gate, up
    return both.reshape(2, hp // BLOCK, BLOCK, *gate.shape[1:]).transpose(0, 1).reshape(2 * hp, *gate.shape[1:])


def swiglu_mm(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, weight_scales: torch.Tensor,
              bias: torch.Tensor | None = None, *, features: int | None = None,
              ) -> tuple[torch.Tensor, torch.Tensor]:
    """silu(A . Wg^T + bg) * (A . Wu^T + bu) held in 8 bits: (codes, scales) of
    [M, features]. weights and bias come in interleave_gate_up's order;
    features (a multiple of 16) defaults to half the weight's rows."""
    if torch.compiler.is_compiling():
        return torch.ops.recavsr_b200.fp8_block_swiglu_mm(values, weights, scales, weight_scales, bias, features)
    return _binding.swiglu_mm(values, weights, scales, weight_scales, bias, features)


@torch.library.custom_op("recavsr_b200::fp8_block_quantize", mutates_args=())
def _quantize_op(x: torch.Tensor, weight: bool) -> tuple[torch.Tensor, torch.Tensor]:
    return _binding.quantize(x, weight)


@_quantize_op.register_fake
def _quantize_fake(x, weight):
    return (x.new_empty(x.shape, dtype=torch.uint8),
            x.new_empty((scale_numel(*x.shape),), dtype=torch.uint8))


@torch.library.custom_op("recavsr_b200::fp8_block_rms_norm", mutates_args=())
def _rms_norm_op(x: torch.Tensor, weight: torch.Tensor, eps: float) -> tuple[torch.Tensor, torch.Tensor]:
    return _binding.rms_norm_quantize(x, weight, eps, None)[:2]


@_rms_norm_op.register_fake
def _rms_norm_fake(x, weight, eps):
    return _quantize_fake(x, False)


@torch.library.custom_op("recavsr_b200::fp8_block_add_rms_norm", mutates_args=())
def _add_rms_norm_op(x: torch.Tensor, weight: torch.Tensor, eps: float,
                     residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    with torch.no_grad():
        return _binding.rms_norm_quantize(x, weight, eps, residual)


@_add_rms_norm_op.register_fake
def _add_rms_norm_fake(x, weight, eps, residual):
    return (*_quantize_fake(x, False), x.new_empty(x.shape))


@torch.library.custom_op("recavsr_b200::fp8_block_mm", mutates_args=())
def _mm_op(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, weight_scales: torch.Tensor,
           bias: torch.Tensor | None, residual: torch.Tensor | None, dtype: torch.dtype | None) -> torch.Tensor:
    with torch.no_grad():
        return _binding.mm(values, weights, scales, weight_scales, bias, residual, dtype, None)


@_mm_op.register_fake
def _mm_fake(values, weights, scales, weight_scales, bias, residual, dtype):
    dtype = dtype or (torch.bfloat16 if residual is None else residual.dtype)
    return values.new_empty((values.shape[0], weights.shape[0]), dtype=dtype)


@torch.library.custom_op("recavsr_b200::fp8_block_mm_out", mutates_args=("out",))
def _mm_out_op(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, weight_scales: torch.Tensor,
               bias: torch.Tensor | None, residual: torch.Tensor | None, dtype: torch.dtype | None,
               out: torch.Tensor) -> None:
    with torch.no_grad():
        _binding.mm(values, weights, scales, weight_scales, bias, residual, dtype, out)


@_mm_out_op.register_fake
def _mm_out_fake(values, weights, scales, weight_scales, bias, residual, dtype, out):
    return None


@torch.library.custom_op("recavsr_b200::fp8_block_swiglu_mm", mutates_args=())
def _swiglu_mm_op(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, weight_scales: torch.Tensor,
                  bias: torch.Tensor | None, features: int | None) -> tuple[torch.Tensor, torch.Tensor]:
    return _binding.swiglu_mm(values, weights, scales, weight_scales, bias, features)


@_swiglu_mm_op.register_fake
def _swiglu_mm_fake(values, weights, scales, weight_scales, bias, features):
    rows, h = values.shape[0], weights.shape[0] // 2 if features is None else features
    return (values.new_empty((rows, h), dtype=torch.uint8),
            values.new_empty((scale_numel(rows, h),), dtype=torch.uint8))


@torch.library.custom_op("recavsr_b200::fp8_block_linear", mutates_args=())
def _linear_op(x: torch.Tensor, weights: torch.Tensor, weight_scales: torch.Tensor,
               bias: torch.Tensor | None) -> torch.Tensor:
    with torch.no_grad():
        codes, scales = _binding.quantize(x, False)
        return _binding.mm(codes, weights, scales, weight_scales, bias, None, x.dtype, None)


@_linear_op.register_fake
def _linear_fake(x, weights, weight_scales, bias):
    return x.new_empty((x.shape[0], weights.shape[0]))


class BlockFP8Linear(nn.Module):
    """nn.Linear with block-scaled FP8 weights and activations: the form of
    runtime.fp8.FP8Linear whose scales follow blocks of 128, not the tensor."""

    @torch.inference_mode()
    def __init__(self, linear: nn.Linear):
        super().__init__()
        if linear.weight.device.type != "cuda" or linear.weight.dtype != torch.bfloat16:
            raise ValueError("FP8 conversion requires loaded CUDA BF16 linears.")
        if linear.in_features % 16:
            raise ValueError("Block FP8 linears need a multiple of 16 input features.")
        self.in_features, self.out_features = linear.in_features, linear.out_features
        codes, scales = quantize_weight(linear.weight.detach())
        self.register_buffer("weight_codes", codes)
        self.register_buffer("weight_scales", scales)
        self.register_buffer("bias", None if linear.bias is None else linear.bias.detach().float())

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.dtype not in (torch.bfloat16, torch.float16):
            raise ValueError("Block FP8 linears take BF16 or FP16 inputs and produce the same type.")
        rows = x.reshape(-1, self.in_features)
        if x.requires_grad and torch.is_grad_enabled():      # codes carry none: the op spans both steps
            out = torch.ops.recavsr_b200.fp8_block_linear(rows, self.weight_codes, self.weight_scales, self.bias)
        else:
            codes, scales = quantize(rows)
            out = mm(codes, self.weight_codes, scales, self.weight_scales, self.bias, dtype=x.dtype)
        return out.reshape(*x.shape[:-1], self.out_features)


def quantize_block_linears(block: nn.Module) -> None:
    """Replace every nn.Linear under `block` by a BlockFP8Linear."""
    for module in list(block.modules()):
        for name, child in list(module.named_children()):
            if isinstance(child, nn.Linear):
                setattr(module, name, BlockFP8Linear(child))
