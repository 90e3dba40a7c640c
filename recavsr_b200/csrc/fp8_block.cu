// Quantizers of block-scaled FP8 (fp8_block.cuh): rows, weights, and the rows
// an RMSNorm (with the residual's addition) produces. All are bound by the
// bytes they move: every input byte is read once, every output byte written
// once, and the scale of a block comes out of the registers of the 16 lanes
// that hold it. Measured (B200, device time, of the measured 6456 GB/s):
// rows 7040 x 14336 bf16 52.4 us = 0.90, 14080 x 512 bf16 4.0 us = 0.84 (from
// L2); weights 14336 x 3072 fp32 33.3 us = 1.0, bf16 31.6 us = 0.65 (half the
// bytes in flight); norm with residual 14081 x 2048 fp32 57.7 us = 1.0, 3520 x 512
// bf16 3.2 us, one row 2.2 us (launch and one round trip to memory), 7040 x 14336
// bf16 161 us = 0.68 (wide 16-bit rows wait for loads that stand behind stores).
#include <type_traits>

#include "fp8_block.cuh"

namespace {

using fp8b::kBlock;

// ---------------------------------------------------------------- rows
constexpr int kRowThreads = 256;
constexpr int kRowsPerCta = kRowThreads / 16;

// A half-warp takes one row's four blocks of a scale atom (512 columns), all
// four loads in flight before the first reduction, and writes the row's four
// scale bytes as one word. Rows past M (up to the atom's 128) get zero scales.
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
quantize_rows_kernel(const T* x, int M, int K, long long ldx, uint8_t* codes, uint8_t* scales) {
  rc::pdl_trigger();
  rc::pdl_wait();
  const int l = threadIdx.x & 15;
  const int row = blockIdx.x * kRowsPerCta + (threadIdx.x >> 4);
  const int col0 = blockIdx.y * 4 * kBlock + l * 8;
  const bool row_ok = row < M;
  float v[4][8];
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    if (row_ok && col0 + b * kBlock < K) {
      fp8b::load8(x + (size_t)row * ldx + col0 + b * kBlock, v[b]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[b][j] = 0.0f;
    }
  }
  uint32_t word = 0;
#pragma unroll
  for (int b = 0; b < 4; ++b) {
    const uint32_t e = fp8b::scale_byte(fp8b::block_amax(v[b]));
    if (row_ok && col0 + b * kBlock < K)
      *reinterpret_cast<uint2*>(codes + (size_t)row * K + col0 + b * kBlock) =
          fp8b::encode8(v[b], fp8b::inverse_scale(e));
    if (row_ok && (int)blockIdx.y * 4 + b < fp8b::blocks_of(K)) word |= e << (8 * b);
  }
  if (l == 0) *reinterpret_cast<uint32_t*>(scales + rc::sf_offset(row, blockIdx.y * 4, gridDim.y)) = word;
}

// ---------------------------------------------------------------- weights
// One CTA takes a 128 x 128 block: 16 lanes a row, 8 rows a thread, one scale
// byte stored for each of its 128 rows (the products read a scale per row).
template <typename T>
__global__ void __launch_bounds__(kRowThreads)
quantize_weight_kernel(const T* w, int N, int K, long long ldw, uint8_t* codes, uint8_t* scales) {
  __shared__ uint32_t s_max[kRowThreads / 32];
  rc::pdl_trigger();
  rc::pdl_wait();
  const int kb = blockIdx.x, col = kb * kBlock + (threadIdx.x & 15) * 8;
  const int row0 = blockIdx.y * kBlock + (threadIdx.x >> 4);
  constexpr int kSteps = kBlock / kRowsPerCta;
  float v[kSteps][8];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int row = row0 + i * kRowsPerCta;
    if (row < N && col < K) {
      fp8b::load8(w + (size_t)row * ldw + col, v[i]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, fp8b::magnitude(v[i][j]));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) s_max[threadIdx.x >> 5] = m;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kRowThreads / 32; ++i) m = max(m, s_max[i]);
  const uint32_t e = fp8b::scale_byte(m);
  const float inv = fp8b::inverse_scale(e);
#pragma unroll
  for (int i = 0; i < kSteps; ++i) {
    const int row = row0 + i * kRowsPerCta;
    if (row < N && col < K)
      *reinterpret_cast<uint2*>(codes + (size_t)row * K + col) = fp8b::encode8(v[i], inv);
  }
  if (threadIdx.x < kBlock) {
    const int row = blockIdx.y * kBlock + threadIdx.x;
    scales[rc::sf_offset(row, kb, fp8b::atoms_of(K))] = row < N && kb < fp8b::blocks_of(K) ? (uint8_t)e : 0;
  }
}

// ---------------------------------------------------------------- RMSNorm
// h = x + residual (fp32; rounded once into hidden when there is a residual),
// y = h * rsqrt(mean(h^2) + eps) * weight, quantized from fp32. TPR threads
// hold a row in registers, CH chunks of 8 columns each; 16 neighbouring
// threads of a chunk are one block of 128 columns.
template <int TPR>
constexpr int norm_threads() { return TPR < 256 ? 256 : TPR; }

template <typename T, int TPR, int CH>
__global__ void __launch_bounds__(norm_threads<TPR>())
rms_norm_kernel(const T* x, long long ldx, const T* residual, long long ldr, int M, int N, const float* weight,
                float eps, T* hidden, uint8_t* codes, uint8_t* scales) {
  constexpr int kThreads = norm_threads<TPR>();
  __shared__ float s_sum[kThreads / 32];
  rc::pdl_trigger();
  rc::pdl_wait();
  const int t = threadIdx.x % TPR;
  const int row = blockIdx.x * (kThreads / TPR) + threadIdx.x / TPR;
  const int katoms = fp8b::atoms_of(N);
  const bool row_ok = row < M;
  float v[CH][8];
  float sum = 0.0f;
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * TPR + t) * 8;
    if (row_ok && col < N) {
      fp8b::load8(x + (size_t)row * ldx + col, v[c]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = 0.0f;
    }
  }
  if (residual) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (c * TPR + t) * 8;
      if (row_ok && col < N) {
        float r[8];
        fp8b::load8(residual + (size_t)row * ldr + col, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[c][j] += r[j];
        fp8b::store8(hidden + (size_t)row * N + col, v[c]);
      }
    }
  }
#pragma unroll
  for (int c = 0; c < CH; ++c)
#pragma unroll
    for (int j = 0; j < 8; ++j) sum = fmaf(v[c][j], v[c][j], sum);
#pragma unroll
  for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if constexpr (TPR > 32) {
    constexpr int kWarps = TPR / 32;
    if ((threadIdx.x & 31) == 0) s_sum[threadIdx.x >> 5] = sum;
    __syncthreads();
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kWarps; ++i) sum += s_sum[threadIdx.x / TPR * kWarps + i];
  }
  const float rstd = rsqrtf(sum / (float)N + eps);
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (c * TPR + t) * 8;
    if (c * TPR * 8 >= katoms * 4 * kBlock) break;
    if (row_ok && col < N) {
      float w[8];
      fp8b::load8(weight + col, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[c][j] = v[c][j] * rstd * w[j];
    }
    const uint32_t e = fp8b::scale_byte(fp8b::block_amax(v[c]));
    if (row_ok && col < N)
      *reinterpret_cast<uint2*>(codes + (size_t)row * N + col) = fp8b::encode8(v[c], fp8b::inverse_scale(e));
    const int kb = col / kBlock;
    if ((t & 15) == 0 && kb < katoms * 4)
      scales[rc::sf_offset(row, kb, katoms)] = row_ok && kb < fp8b::blocks_of(N) ? (uint8_t)e : 0;
  }
  // Scale bytes past the columns this row's threads cover (the last atom's).
  for (int kb = CH * TPR / 16 + t; kb < katoms * 4; kb += TPR) scales[rc::sf_offset(row, kb, katoms)] = 0;
}

bool aligned16(const void* p) { return p && reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int dtype_size(int dtype) { return dtype == fp8b::kF32 ? 4 : 2; }

int check_rows(const char* what, const void* x, int dtype, int rows, int cols, long long ldx, const void* codes,
               const void* scales) {
  if (dtype < 0 || dtype > 2) return rc::set_error(RC_ERR_ARG, "%s: dtype must be 0 (fp32), 1 (bf16) or 2 (fp16)", what);
  if (rows < 0 || cols <= 0 || cols % 16)
    return rc::set_error(RC_ERR_ARG, "%s: columns must be a positive multiple of 16 (got %d x %d)", what, rows, cols);
  if (rows > INT32_MAX - kBlock) return rc::set_error(RC_ERR_ARG, "%s: too many rows (%d)", what, rows);
  if (!rows) return RC_OK;
  if (ldx < cols || (ldx * dtype_size(dtype)) % 16)
    return rc::set_error(RC_ERR_ARG, "%s: row stride %lld must hold %d columns and be a multiple of 16 bytes", what, ldx, cols);
  if (!aligned16(x) || !aligned16(codes) || !aligned16(scales))
    return rc::set_error(RC_ERR_ARG, "%s: pointers must be 16-byte aligned and not null", what);
  return RC_OK;
}

template <typename F>
int by_dtype(int dtype, F f) {
  switch (dtype) {
    case fp8b::kF32: return f((const float*)nullptr);
    case fp8b::kBF16: return f((const __nv_bfloat16*)nullptr);
    default: return f((const __half*)nullptr);
  }
}

}  // namespace

extern "C" {

long long rc_fp8_block_scales(long long rows, long long cols) {
  return (rows + kBlock - 1) / kBlock * kBlock * ((cols + 4 * kBlock - 1) / (4 * kBlock)) * 4;
}

int rc_fp8_block_quantize(const void* x, int dtype, int M, int K, long long ldx, uint8_t* codes, uint8_t* scales,
                          cudaStream_t stream) {
  const char* what = "rc_fp8_block_quantize";
  int r = check_rows(what, x, dtype, M, K, ldx, codes, scales);
  if (r || !M) return r;
  return by_dtype(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const dim3 grid((unsigned)((M + kBlock - 1) / kBlock * (kBlock / kRowsPerCta)), (unsigned)fp8b::atoms_of(K));
    if (grid.y > 65535u) return rc::set_error(RC_ERR_UNSUPPORTED, "%s: more than 33553920 columns", what);
    return rc::check_launch(rc::launch_pdl(quantize_rows_kernel<T>, grid, dim3(kRowThreads), 0, stream,
                                           static_cast<const T*>(x), M, K, ldx, codes, scales), what);
  });
}

int rc_fp8_block_quantize_weight(const void* w, int dtype, int N, int K, long long ldw, uint8_t* codes,
                                 uint8_t* scales, cudaStream_t stream) {
  const char* what = "rc_fp8_block_quantize_weight";
  int r = check_rows(what, w, dtype, N, K, ldw, codes, scales);
  if (r || !N) return r;
  return by_dtype(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const dim3 grid((unsigned)(fp8b::atoms_of(K) * 4), (unsigned)((N + kBlock - 1) / kBlock));
    if (grid.y > 65535u) return rc::set_error(RC_ERR_UNSUPPORTED, "%s: more than 8388480 rows", what);
    return rc::check_launch(rc::launch_pdl(quantize_weight_kernel<T>, grid, dim3(kRowThreads), 0, stream,
                                           static_cast<const T*>(w), N, K, ldw, codes, scales), what);
  });
}

int rc_fp8_block_rms_norm(const void* x, long long ldx, const void* residual, long long ldr, int dtype, int M, int N,
                          const float* weight, float eps, void* hidden, uint8_t* codes, uint8_t* scales,
                          cudaStream_t stream) {
  const char* what = "rc_fp8_block_rms_norm";
  int r = check_rows(what, x, dtype, M, N, ldx, codes, scales);
  if (r) return r;
  if (N > 16384) return rc::set_error(RC_ERR_UNSUPPORTED, "%s: rows of at most 16384 columns (got %d)", what, N);
  if (!M) return RC_OK;
  if (!aligned16(weight)) return rc::set_error(RC_ERR_ARG, "%s: weight must be 16-byte aligned and not null", what);
  if ((residual != nullptr) != (hidden != nullptr))
    return rc::set_error(RC_ERR_ARG, "%s: residual and hidden go together", what);
  if (residual && (!aligned16(residual) || !aligned16(hidden) || ldr < N || (ldr * dtype_size(dtype)) % 16))
    return rc::set_error(RC_ERR_ARG, "%s: residual and hidden must be 16-byte aligned rows", what);
  return by_dtype(dtype, [&](auto* tag) {
    using T = std::remove_const_t<std::remove_pointer_t<decltype(tag)>>;
    const int mpad = (M + kBlock - 1) / kBlock * kBlock;
    auto go = [&](auto kernel, int threads, int rows_per_cta) {
      return rc::check_launch(
          rc::launch_pdl(kernel, dim3((unsigned)(mpad / rows_per_cta)), dim3(threads), 0, stream,
                         static_cast<const T*>(x), ldx, static_cast<const T*>(residual), ldr, M, N, weight, eps,
                         static_cast<T*>(hidden), codes, scales), what);
    };
    if (N <= 256) return go(rms_norm_kernel<T, 32, 1>, 256, 8);
    if (N <= 512) return go(rms_norm_kernel<T, 32, 2>, 256, 8);
    if (N <= 1024) return go(rms_norm_kernel<T, 32, 4>, 256, 8);
    if (N <= 2048) return go(rms_norm_kernel<T, 128, 2>, 256, 2);
    if (N <= 4096) return go(rms_norm_kernel<T, 128, 4>, 256, 2);
    if (N <= 8192) return go(rms_norm_kernel<T, 512, 2>, 512, 1);
    return go(rms_norm_kernel<T, 512, 4>, 512, 1);
  });
}

}  // extern "C"
