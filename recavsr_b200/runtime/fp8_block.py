"""Block-scaled FP8 linears: E4M3 codes with one power-of-two scale for each
block of 128 columns, next to the per-tensor FP8 linears of runtime.fp8
(recavsr_infer/runtime/fp8.py:13-55).

A matrix held in 8 bits is a pair (codes, scales): u8 E4M3 codes [rows, cols]
and u8 E8M0 scale bytes (2^(e-127), the smallest with amax <= 448 * scale) in
the flat 128x4 blocked order the tensor core reads; scale_bytes() gives them as
[rows, blocks]. Activations have a scale for each row's block of 128 columns,
weights one for each 128 x 128 block.

    codes, scales, hidden = rms_norm_quantize(x, weight, eps, residual=hidden)
    qkv = mm(codes, w_codes, scales, w_scales, bias)
    codes, scales = quantize(attention)
    hidden = mm(codes, w_codes, scales, w_scales, bias, residual=hidden)
    codes, scales = swiglu_mm(codes, gu_codes, scales, gu_scales, gu_bias)

Every function runs on the current stream of its inputs' device and allocates
only what it returns. There is no CPU path.
"""
from __future__ import annotations

import torch
from torch import nn

from .. import _lib

BLOCK = 128
_DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_OUT = {torch.bfloat16: 1, torch.float16: 2}


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
    power = torch.where(e == 255, torch.nan, (e << 23).view(torch.float32))
    values = codes.view(torch.float8_e4m3fn).to(torch.float32)
    return values * power.repeat_interleave(BLOCK, 1)[:, :cols]


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """x as rows the kernels can read: unit column stride, 16-byte rows."""
    if not x.is_cuda:
        raise ValueError(f"{what}: the B200 kernels need CUDA tensors (got {x.device})")
    if x.dtype not in _DTYPES:
        raise ValueError(f"{what} takes float32 / bfloat16 / float16 rows (got {x.dtype}).")
    if x.dim() != 2:
        raise ValueError(f"{what} expects a 2-D matrix (got {x.dim()}-D).")
    n = x.shape[1]
    if n == 0 or n % 16:
        raise ValueError(f"{what}: columns must be a positive multiple of 16 (got {n}).")
    if not x.is_contiguous() and (x.stride(1) != 1 or x.stride(0) < n or (x.stride(0) * x.element_size()) % 16):
        return x.clone(memory_format=torch.contiguous_format)
    return x.clone(memory_format=torch.contiguous_format) if x.data_ptr() % 16 else x


def _row_stride(x: torch.Tensor) -> int:
    """Row stride in elements (that of a contiguous matrix for a single row)."""
    return x.shape[1] if x.is_contiguous() else x.stride(0)


def _held(rows: int, cols: int, device) -> tuple[torch.Tensor, torch.Tensor]:
    return (torch.empty((rows, cols), dtype=torch.uint8, device=device),
            torch.empty(scale_numel(rows, cols), dtype=torch.uint8, device=device))


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] (fp32 / bf16 / fp16, K a multiple of 16) -> (codes, scales)."""
    x = _rows(x, "fp8_block.quantize")
    m, k = x.shape
    codes, scales = _held(m, k, x.device)
    _lib.call_on(x.get_device(), "rc_fp8_block_quantize", x.data_ptr(), _DTYPES[x.dtype], m, k, _row_stride(x),
                 codes.data_ptr(), scales.data_ptr())
    return codes, scales


def quantize_weight(weight: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weight [N, K] -> (codes, scales), one scale for each 128 x 128 block."""
    w = _rows(weight, "fp8_block.quantize_weight")
    n, k = w.shape
    codes, scales = _held(n, k, w.device)
    _lib.call_on(w.get_device(), "rc_fp8_block_quantize_weight", w.data_ptr(), _DTYPES[w.dtype], n, k, _row_stride(w),
                 codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _vector(t: torch.Tensor, n: int, like: torch.Tensor, what: str) -> torch.Tensor:
    """A per-column vector (norm weight, bias) as 16-byte aligned fp32."""
    if t.shape != (n,) or t.get_device() != like.get_device():
        raise ValueError(f"{what} must have {n} elements on {like.device} (got {tuple(t.shape)} on {t.device}).")
    if t.dtype != torch.float32 or not t.is_contiguous():
        t = t.to(torch.float32).contiguous()
    return t.clone() if t.data_ptr() % 16 else t


def rms_norm_quantize(x: torch.Tensor, weight: torch.Tensor, eps: float, residual: torch.Tensor | None = None,
                      ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None]:
    """RMSNorm of x (+ residual) held in 8 bits: (codes, scales, hidden).

    h = x + residual is summed in fp32; hidden is h rounded to x's dtype (None
    without a residual) and the norm h * rsqrt(mean(h^2) + eps) * weight is
    quantized from fp32, without a rounding between."""
    x = _rows(x, "fp8_block.rms_norm_quantize")
    m, n = x.shape
    weight = _vector(weight, n, x, "fp8_block.rms_norm_quantize: weight")
    hidden, ldr = None, 0
    if residual is not None:
        if residual.shape != x.shape or residual.dtype != x.dtype or residual.get_device() != x.get_device():
            raise ValueError("fp8_block.rms_norm_quantize: residual must match x's shape, dtype and device.")
        residual = _rows(residual, "fp8_block.rms_norm_quantize")
        ldr = _row_stride(residual)
        hidden = torch.empty((m, n), dtype=x.dtype, device=x.device)
    codes, scales = _held(m, n, x.device)
    _lib.call_on(x.get_device(), "rc_fp8_block_rms_norm", x.data_ptr(), _row_stride(x), _lib.ptr(residual), ldr,
                 _DTYPES[x.dtype], m, n, weight.data_ptr(), eps, _lib.ptr(hidden), codes.data_ptr(),
                 scales.data_ptr())
    return codes, scales, hidden


def _operand(codes: torch.Tensor, scales: torch.Tensor, what: str) -> torch.Tensor:
    if not codes.is_cuda or scales.get_device() != codes.get_device():
        raise ValueError(f"{what}: codes and scales must be on one CUDA device (got {codes.device}, {scales.device}).")
    if codes.dim() != 2 or codes.element_size() != 1 or scales.element_size() != 1:
        raise ValueError(f"{what}: operands are 8-bit codes [rows, K] with 8-bit scales.")
    rows, k = codes.shape
    if k == 0 or k % 16:
        raise ValueError(f"{what}: K must be a positive multiple of 16 (got {k}).")
    if scales.numel() != scale_numel(rows, k) or not scales.is_contiguous() or scales.data_ptr() % 16:
        raise ValueError(f"{what}: a {rows} x {k} operand has {scale_numel(rows, k)} contiguous, 16-byte aligned "
                         "scale bytes.")
    if not codes.is_contiguous() and (codes.stride(1) != 1 or codes.stride(0) < k or codes.stride(0) % 16):
        return codes.clone(memory_format=torch.contiguous_format)
    return codes.clone(memory_format=torch.contiguous_format) if codes.data_ptr() % 16 else codes


def mm(values: torch.Tensor, weights: torch.Tensor, scales: torch.Tensor, weight_scales: torch.Tensor,
       bias: torch.Tensor | None = None, *, residual: torch.Tensor | None = None,
       dtype: torch.dtype | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """[M, N] = A [M, K] . W [N, K]^T + bias (+ residual), summed in fp32 and
    rounded once to dtype (bfloat16 by default, or float16). `out` may be
    `residual` itself."""
    values, weights = _operand(values, scales, "fp8_block.mm"), _operand(weights, weight_scales, "fp8_block.mm")
    (m, k), (n, kw), index = values.shape, weights.shape, values.get_device()
    if kw != k or weights.get_device() != index or n == 0:
        raise ValueError(f"fp8_block.mm: operands of {m} x {k} on {values.device} and {n} x {kw} on {weights.device}.")
    if dtype is None:
        dtype = out.dtype if out is not None else residual.dtype if residual is not None else torch.bfloat16
    if dtype not in _OUT:
        raise ValueError(f"fp8_block.mm produces bfloat16 or float16 (got {dtype}).")
    if bias is not None:
        bias = _vector(bias, n, values, "fp8_block.mm: bias")
    ldr = 0
    if residual is not None:
        if residual.shape != (m, n) or residual.dtype != dtype or residual.get_device() != index:
            raise ValueError(f"fp8_block.mm: residual must be {m} x {n} {dtype} on {values.device}.")
        if not residual.is_contiguous() and (residual.stride(1) != 1 or residual.stride(0) < n):
            residual = residual.clone(memory_format=torch.contiguous_format)
        ldr = _row_stride(residual)
    if out is None:
        out = torch.empty((m, n), dtype=dtype, device=values.device)
    elif out.shape != (m, n) or out.dtype != dtype or out.get_device() != index or (
            not out.is_contiguous() and (out.stride(1) != 1 or out.stride(0) < n)):
        raise ValueError(f"fp8_block.mm: out must be {m} x {n} {dtype} rows on {values.device}.")
    _lib.call_on(index, "rc_fp8_block_gemm", values.data_ptr(), _row_stride(values), scales.data_ptr(),
                 weights.data_ptr(), _row_stride(weights), weight_scales.data_ptr(), _lib.ptr(bias), m, n, k,
                 _OUT[dtype], _lib.ptr(residual), ldr, out.data_ptr(), _row_stride(out))
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
    values = _operand(values, scales, "fp8_block.swiglu_mm")
    weights = _operand(weights, weight_scales, "fp8_block.swiglu_mm")
    (m, k), (n, kw), index = values.shape, weights.shape, values.get_device()
    if kw != k or weights.get_device() != index:
        raise ValueError(f"fp8_block.swiglu_mm: operands of {m} x {k} on {values.device} and {n} x {kw} on "
                         f"{weights.device}.")
    h = n // 2 if features is None else features
    if h <= 0 or h % 16 or -(-h // BLOCK) * 2 * BLOCK != n:
        raise ValueError(f"fp8_block.swiglu_mm: {h} features need {-(-h // BLOCK) * 2 * BLOCK} interleaved weight "
                         f"rows (got {n}).")
    if bias is not None:
        bias = _vector(bias, n, values, "fp8_block.swiglu_mm: bias")
    codes, out_scales = _held(m, h, values.device)
    _lib.call_on(index, "rc_fp8_block_swiglu_gemm", values.data_ptr(), _row_stride(values), scales.data_ptr(),
                 weights.data_ptr(), _row_stride(weights), weight_scales.data_ptr(), _lib.ptr(bias), m, h, k,
                 codes.data_ptr(), out_scales.data_ptr())
    return codes, out_scales


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
        if x.dtype not in _OUT:
            raise ValueError("Block FP8 linears take BF16 or FP16 inputs and produce the same type.")
        codes, scales = quantize(x.reshape(-1, self.in_features))
        out = mm(codes, self.weight_codes, scales, self.weight_scales, self.bias, dtype=x.dtype)
        return out.reshape(*x.shape[:-1], self.out_features)


def quantize_block_linears(block: nn.Module) -> None:
    """Replace every nn.Linear under `block` by a BlockFP8Linear."""
    for module in list(block.modules()):
        for name, child in list(module.named_children()):
            if isinstance(child, nn.Linear):
                setattr(module, name, BlockFP8Linear(child))
