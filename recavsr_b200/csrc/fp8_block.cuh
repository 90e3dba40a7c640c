// Block-scaled FP8 values shared by the quantizers and the products.
//
// A matrix held in 8 bits is E4M3 codes [rows, cols] and one E8M0 scale byte e
// (the power of two 2^(e-127)) for each row's block of 128 columns: the
// smallest e >= 1 with amax <= 448 * 2^(e-127), so the largest code magnitude
// is at most 448 and no block saturates. A block with an infinity or a NaN has
// e = 255 (NaN) and NaN codes. The scale is a power of two because the tensor
// core applies E8M0 scales itself (kind::mxf8f6f4.block_scale): multiplying by
// one loses no bit and the product needs no scaling pass, while E4M3, a
// floating format, keeps its four significant bits at any scale.
//
// Scale bytes lie in the 128x4 blocked order of rc::sf_offset with the block of
// 128 columns as its k-block: one 512-byte atom is 128 rows x 512 columns.
#pragma once

#include <cuda_fp16.h>
#include <type_traits>

#include "common.cuh"

namespace fp8b {

constexpr int kBlock = 128;

enum DType : int { kF32 = 0, kBF16 = 1, kF16 = 2 };

__host__ __device__ __forceinline__ int blocks_of(int cols) { return (cols + kBlock - 1) / kBlock; }
__host__ __device__ __forceinline__ int atoms_of(int cols) { return (cols + 4 * kBlock - 1) / (4 * kBlock); }

// Scale byte from the bit pattern of amax >= 0 (or NaN). With amax =
// m * 2^(E-127), 1 <= m < 2, and 448 = 1.75 * 2^8, e is E - 8, one more when
// m > 1.75 (the add carries into the exponent field exactly then). Subnormal
// amax and zero give e = 1.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  if (amax_bits >= 0x7f800000u) return 255u;
  const int e = (int)((amax_bits + 0x1fffffu) >> 23) - 8;
  return (uint32_t)max(e, 1);
}
// 2^(127-e), which multiplies the values into codes; NaN for e = 255.
__device__ __forceinline__ float inverse_scale(uint32_t e) {
  return __uint_as_float(e == 255u ? 0x7fffffffu : (254u - e) << 23);
}
// Bit pattern of |v|: unsigned order is numeric order, NaN above infinity.
__device__ __forceinline__ uint32_t magnitude(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Four values -> four E4M3 codes, value j in byte j (round to nearest even;
// |v| <= 448 by the choice of the scale, NaN gives 0x7f).
__device__ __forceinline__ uint32_t e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}

// Eight consecutive values of a row as fp32 (16-byte aligned).
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    const float4 a = rc::ld_in(reinterpret_cast<const float4*>(p));
    const float4 b = rc::ld_in(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else {
    const uint4 w = rc::ld_in(reinterpret_cast<const uint4*>(p));
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 2 && alignof(T) == 2) {
        if constexpr (std::is_same<T, __half>::value) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[j]));
          v[2 * j] = f.x;
          v[2 * j + 1] = f.y;
        } else {
          v[2 * j] = __uint_as_float(u[j] << 16);
          v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
        }
      }
    }
  }
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __half*) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float a, float b, __nv_bfloat16*) { return rc::pack_bf16x2(a, b); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ __half from_float(float v, __half*) { return __float2half_rn(v); }
__device__ __forceinline__ __nv_bfloat16 from_float(float v, __nv_bfloat16*) { return __float2bfloat16_rn(v); }
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
  } else {
    T* tag = nullptr;
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2(v[0], v[1], tag), pack2(v[2], v[3], tag),
                                              pack2(v[4], v[5], tag), pack2(v[6], v[7], tag));
  }
}

// amax bits of the block that the 16 lanes of this lane's half-warp hold 8
// values each of.
__device__ __forceinline__ uint32_t block_amax(const float (&v)[8]) {
  uint32_t m = magnitude(v[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) m = max(m, magnitude(v[j]));
#pragma unroll
  for (int o = 8; o; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
__device__ __forceinline__ uint2 encode8(const float (&v)[8], float inv) {
  return make_uint2(e4m3x4(v[0] * inv, v[1] * inv, v[2] * inv, v[3] * inv),
                    e4m3x4(v[4] * inv, v[5] * inv, v[6] * inv, v[7] * inv));
}

}  // namespace fp8b
