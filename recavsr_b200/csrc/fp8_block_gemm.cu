// Products of block-scaled FP8 matrices (fp8_block.cuh) on tcgen05:
//   OUT     out = A . W^T + bias (+ residual), rounded once into bf16 / fp16
//   SWIGLU  y = silu(A . Wg^T + bg) * (A . Wu^T + bu), quantized again: E4M3
//           codes and a scale byte per block of 128 columns. W's rows (and the
//           bias) alternate 128 gate and 128 up rows, so a tile of 256 columns
//           is one block of 128 outputs with both of its factors.
//
// kind::mxf8f6f4.block_scale multiplies each row's 32 K elements by that row's
// E8M0 scales inside the tensor core. A block of 128 columns is one 128-byte
// k-tile, i.e. four MMAs of K = 32 with the same scale, and the instruction
// descriptor picks one of the four scale bytes of a tensor-memory word: an atom
// (128 rows x 4 blocks) is copied global -> smem (TMA) -> TMEM (tcgen05.cp)
// once per four k-tiles and needs no replication. Accumulation is fp32 in TMEM
// over the whole K.
//
// One CTA per SM (or CTA pair, PAIR: 256-row tiles over two SMs, each staging
// its own 128 rows of A and half of W's) walks the output tiles: warp 0 = TMA
// producer, warp 1 = MMA issuer, the other warps = epilogue, 64 columns of one
// accumulator row per thread. The accumulator is drained into registers and
// released before the epilogue's arithmetic; tiles of 128 and 192 columns have
// more than one accumulator, so the next tile's MMAs do not wait for that.
//
// Measured (B200, device time): 7040 x 3072 x 14336 + bias + residual 240-255
// us = 2.43-2.59 PFLOP/s, 0.72-0.77 of twice the measured bf16 rate, 274 us in a
// loop of seconds (the 1000 W cap holds the clock at 1.25 GHz); 1759 x 3072 x
// 3072 18.1 us; 3520 x 768 x 512 5.0 us; gated 14080 x 2048 x 512 33.1 us. What bounds
// them: 64 (256 x 256 tiles) to 128 (128 x 128) operand bytes per clock and SM
// that the MMAs take from L2, then the power cap; at short K the hand-over of
// the 256-column accumulator (a tile of CTA pairs at K = 512 takes 3100-3700
// cycles, 2048 of them MMAs) and, gated, two MUFU results per output.
#include <atomic>

#include "fp8_block.cuh"
#include "sm100.cuh"

namespace {

enum Epi : int { EPI_OUT = 0, EPI_SWIGLU = 1 };

constexpr int BM = 128;
constexpr int kRowBytes = 128;        // K elements (bytes) per k-tile: one scale block
constexpr int kSfAtom = 512;          // 128 rows x 4 scale bytes

struct Params {
  int M, N, K;                 // N: rows of W
  int k_tiles, m_blocks, n_blocks;
  int group_m;                 // row blocks per group of the raster
  uint32_t inv_group, inv_last;   // ceil(2^32 / rows) of a whole and of the last group
  int katoms;                  // scale atoms along K
  const float* bias;           // [N], nullable
  int staged;                  // OUT: rows of out (and residual) start on 16 bytes: they move by TMA
  int pairs;                   // or on 4 bytes
  void* out;                   // OUT
  long long ldo;
  const void* residual;        // OUT, nullable
  long long ldr;
  uint8_t* codes;              // SWIGLU: [M, H] codes and their scale atoms
  uint8_t* scales;
  int H;
};

struct Maps {
  CUtensorMap a, b, sfa, sfb, out, res;
};

template <int BN>
constexpr int epi_warps() { return BN / 16; }        // 4 lane quadrants x BN / 64 column shares
// Scale atoms (128 rows of W) under BN columns that start on a multiple of BN.
template <int BN>
constexpr int sfb_atoms() { return BN % 128 ? (BN + 64) / 128 : BN / 128; }
template <int BN>
constexpr int tile_threads() { return 64 + 32 * epi_warps<BN>(); }

template <int BN, int STAGES, int EPI, bool PAIR>
struct Smem {
  static constexpr int kA = BM * kRowBytes;
  static constexpr int kB = (PAIR ? BN / 2 : BN) * kRowBytes;    // a pair splits W's rows between its CTAs
  static constexpr int kSf = (1 + sfb_atoms<BN>()) * kSfAtom;
  static constexpr int offA = 0;
  static constexpr int offB = offA + STAGES * kA;
  static constexpr int offOut = offB + STAGES * kB;
  // Staging boxes of a warp's 32 rows, each a TMA store. OUT: 64 columns of 16
  // bits, or 32 twice where that buys a stage. SWIGLU: 32 codes.
  static constexpr int kBoxCols = EPI == EPI_SWIGLU ? 32 : BN == 128 ? 64 : 32;
  static constexpr int kBox = 32 * kBoxCols * (EPI == EPI_SWIGLU ? 1 : 2);
  static constexpr int kAmax = EPI == EPI_SWIGLU ? 2 * 4 * 4 * 32 * 4 : 0;      // the parts' amax, two tiles
  static constexpr int kOut = epi_warps<BN>() * kBox + kAmax;
  static constexpr int offBias = offOut + kOut;                     // 64 fp32 per epilogue warp
  static constexpr int offSf = offBias + epi_warps<BN>() * 64 * 4;
  static constexpr int offBar = offSf + STAGES * kSf;
  static constexpr int kBars = 2 * STAGES + 6 + 1 + epi_warps<BN>() + 2;
  static constexpr int kTotal = offBar + kBars * 8;
  static_assert(kTotal <= 232448, "shared memory");
};

__device__ __forceinline__ float4 ld_shared4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ uint4 ld_shared4u(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr));
  return v;
}
__device__ __forceinline__ void st_shared4(uint32_t addr, uint4 v) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
               : "memory");
}

template <typename Out>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<Out, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// silu(g) u of a pair as g / (1 + t) p u p with t = s^2 = exp(-|g|): p = 1 where
// g >= 0, and s below, where silu(g) = g t / (1 + t). The exponential of the half
// argument stays in range (s down to g = -174, silu under 2^-243) where exp(-g)
// would overflow, or its reciprocal flush, from g = -87 on; multiplied in one at
// a time, p keeps the product out of the subnormals until the last step. The MUFU
// evaluates exp2 and the reciprocal: the relative error is under 2^-19 + |g|
// 2^-23, the second part that of g rounded once more (the argument of exp2 is).
__device__ __forceinline__ float2 swiglu2(float2 g, float2 u) {
  constexpr float kHalfLog2e = 0.72134752044448170f;
  float2 s, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s.x) : "f"(fabsf(g.x) * -kHalfLog2e));
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(s.y) : "f"(fabsf(g.y) * -kHalfLog2e));
  const float2 d = __ffma2_rn(s, s, make_float2(1.0f, 1.0f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(d.x));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(d.y));
  const float2 p = make_float2(g.x < 0.0f ? s.x : 1.0f, g.y < 0.0f ? s.y : 1.0f);
  return __fmul2_rn(__fmul2_rn(__fmul2_rn(__fmul2_rn(g, r), p), u), p);
}

// Columns of this thread's accumulator row into registers, complete on return.
template <int COLS>
__device__ __forceinline__ void load_acc(uint32_t taddr, uint32_t (&r)[COLS]) {
#pragma unroll
  for (int c = 0; c < COLS; c += 32) sm100::tmem_ld32(taddr + c, r + c);
}
template <int COLS>
__device__ __forceinline__ void acc_ready(uint32_t (&r)[COLS]) {
  sm100::tmem_ld_wait();
#pragma unroll
  for (int c = 0; c < COLS; ++c) asm volatile("" : "+r"(r[c]));   // no use above the wait
}

// The tiles of one CTA (or pair), every step-th of the raster: groups of
// group_m row blocks, row block fastest within a group, then column block, so
// that one wave's tiles share few operand panels. Walked without a division:
// every epilogue warp follows it, and its instructions are the epilogue's.
struct Walk {
  int r, row0, rows;           // index within the group, the group's first row block and its row blocks
  __device__ __forceinline__ Walk(const Params& p, int tile) : r(tile), row0(0), rows(min(p.group_m, p.m_blocks)) { settle(p); }
  __device__ __forceinline__ void settle(const Params& p) {
    while (r >= rows * p.n_blocks && rows > 0) {
      r -= rows * p.n_blocks;
      row0 += rows;
      rows = min(p.group_m, p.m_blocks - row0);
    }
  }
  __device__ __forceinline__ bool more() const { return rows > 0; }
  __device__ __forceinline__ void next(const Params& p, int step) {
    r += step;
    settle(p);
  }
  __device__ __forceinline__ void coords(const Params& p, int& mb, int& nb) const {
    // r / rows: exact by the reciprocal's high product, as r * rows < 2^32 (checked on the host)
    nb = rows == 1 ? r : (int)__umulhi((uint32_t)r, rows == p.group_m ? p.inv_group : p.inv_last);
    mb = row0 + r - nb * rows;
  }
};

template <int BN, int STAGES, int EPI, bool PAIR, typename Out>
__global__ void __launch_bounds__(tile_threads<BN>(), 1)
tile_kernel(const __grid_constant__ Maps maps, const Params p) {
  using S = Smem<BN, STAGES, EPI, PAIR>;
  constexpr int kEpiWarps = epi_warps<BN>();
  constexpr int kAcc = BN == 128 ? 3 : BN == 192 ? 2 : 1;           // accumulators in TMEM
  constexpr int kSfaCols = 4, kSfbCols = 4 * sfb_atoms<BN>(), kSfCols = kSfaCols + kSfbCols;
  static_assert(EPI == EPI_OUT || BN == 256, "SWIGLU tiles are one block of 128 outputs");
  constexpr int kTmemCols = 512;
  static_assert(kAcc * BN + 2 * kSfCols <= kTmemCols, "TMEM budget");

  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::offBar);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;     // [3]
  uint64_t* acc_empty = acc_full + 3;      // [3]
  uint64_t* done = acc_empty + 3;
  uint64_t* res_full = done + 1;           // [kEpiWarps]
  volatile int* abort_flag = reinterpret_cast<volatile int*>(res_full + kEpiWarps);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(res_full + kEpiWarps + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int tiles = p.m_blocks * p.n_blocks;
  const uint32_t rank = PAIR ? sm100::cluster_ctarank() : 0u;
  const bool leader = rank == 0;
  const int tile0 = PAIR ? (int)(blockIdx.x >> 1) : (int)blockIdx.x;
  const int step = PAIR ? (int)(gridDim.x >> 1) : (int)gridDim.x;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 3; ++a) {
      sm100::mbar_init(&acc_full[a], 1);
      sm100::mbar_init(&acc_empty[a], PAIR ? 2 * kEpiWarps : kEpiWarps);   // one arrival per epilogue warp
    }
    sm100::mbar_init(done, 1);
    for (int w = 0; w < kEpiWarps; ++w) sm100::mbar_init(&res_full[w], 1);
    *abort_flag = 0;
    sm100::fence_mbar_init();
  }
  if (warp == 1) {
    if constexpr (PAIR) {
      sm100::tmem_alloc_pair(tmem_slot, kTmemCols);
      sm100::tmem_relinquish_pair();
    } else {
      sm100::tmem_alloc(tmem_slot, kTmemCols);
      sm100::tmem_relinquish();
    }
  }
  sm100::tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) sm100::cluster_sync();   // both CTAs' barriers initialised before any remote use
  sm100::tc_fence_after();
  rc::pdl_trigger();
  rc::pdl_wait();
  const uint32_t tmem = *tmem_slot;
  const uint32_t tmem_sf = tmem + kAcc * BN;   // 2 x (A's columns, W's columns)

  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int site) -> bool {
    if (sm100::mbar_wait(bar, parity, abort_flag)) return true;
    if (!*abort_flag) {
      rc::device_fail(kKernFp8Block, site);
      *abort_flag = 1;
    }
    return false;
  };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    if (sm100::elect_one_sync()) {
      sm100::tma_prefetch_desc(&maps.a);
      sm100::tma_prefetch_desc(&maps.b);
      sm100::tma_prefetch_desc(&maps.sfa);
      sm100::tma_prefetch_desc(&maps.sfb);
      int stage = 0;
      uint32_t phase = 0;
      long long issued = 0;
      bool ok = true;
      for (Walk walk(p, tile0); walk.more() && ok; walk.next(p, step)) {
        int mb, nb;
        walk.coords(p, mb, nb);
        const int rb = PAIR ? mb * 2 + (int)rank : mb;                          // this CTA's 128-row block of A
        const int brow = nb * BN + (PAIR ? (int)rank * (BN / 2) : 0);    // and its first row of W
        const int b_line = nb * BN / 128 * p.katoms * 4;
        for (int kt = 0; kt < p.k_tiles; ++kt) {
          if (!wait(&empty[stage], phase ^ 1, 1)) { ok = false; break; }
          uint8_t* a = smem + S::offA + stage * S::kA;
          uint8_t* b = smem + S::offB + stage * S::kB;
          uint8_t* sf = smem + S::offSf + stage * S::kSf;
          const bool atom = (kt & 3) == 0;
          const uint32_t bytes = S::kA + S::kB + (atom ? S::kSf : 0);
          const int line = (kt >> 2) * 4;
          if constexpr (PAIR) {
            const uint32_t bar = sm100::mapa(sm100::smem_u32(&full[stage]), 0);
            if (leader) sm100::mbar_arrive_expect_tx(&full[stage], 2 * bytes);
            sm100::tma_load_2d_pair(a, &maps.a, bar, kt * kRowBytes, rb * BM);
            sm100::tma_load_2d_pair(b, &maps.b, bar, kt * kRowBytes, brow);
            if (atom) {
              sm100::tma_load_2d_pair(sf, &maps.sfa, bar, 0, rb * p.katoms * 4 + line);
              for (int r = 0; r < sfb_atoms<BN>(); ++r)
                sm100::tma_load_2d_pair(sf + (1 + r) * kSfAtom, &maps.sfb, bar, 0, b_line + r * p.katoms * 4 + line);
            }
          } else {
            sm100::mbar_arrive_expect_tx(&full[stage], bytes);
            sm100::tma_load_2d(a, &maps.a, &full[stage], kt * kRowBytes, rb * BM);
            sm100::tma_load_2d(b, &maps.b, &full[stage], kt * kRowBytes, brow);
            if (atom) {
              sm100::tma_load_2d(sf, &maps.sfa, &full[stage], 0, rb * p.katoms * 4 + line);
              for (int r = 0; r < sfb_atoms<BN>(); ++r)
                sm100::tma_load_2d(sf + (1 + r) * kSfAtom, &maps.sfb, &full[stage], 0, b_line + r * p.katoms * 4 + line);
            }
          }
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // Every load this thread issued must land before the CTA exits. (A
      // pair's loads count on the leader's barriers: the leader drains for
      // both, and the final cluster barrier keeps the other CTA resident.)
      if (PAIR && !leader) issued = 0;
      for (int s = 0; s < STAGES && issued > 0; ++s, --issued) {
        if (stage == 0) { stage = STAGES; phase ^= 1; }
        --stage;
        sm100::mbar_wait(&full[stage], phase);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer
    if (leader && sm100::elect_one_sync()) {
      int stage = 0, sf_buf = 1, local = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint64_t da0 = sm100::desc_kmajor_sw128(sm100::smem_u32(smem + S::offA));
      const uint64_t db0 = sm100::desc_kmajor_sw128(sm100::smem_u32(smem + S::offB));
      const uint64_t dsf0 = sm100::desc_sf_rows(sm100::smem_u32(smem + S::offSf));
      auto commit = [&](uint64_t* bar) {
        if constexpr (PAIR) sm100::tc_commit_pair(bar);   // arrives in both CTAs
        else sm100::tc_commit(bar);
      };
      Walk walk(p, tile0);
      for (int tile = tile0; tile < tiles && ok; tile += step, ++local) {
        // The scale rows of a tile that starts in the middle of an atom begin
        // two columns (64 rows) into its copy.
        uint32_t shift = 0;
        if constexpr (BN % 128 != 0) {
          int mb, nb;
          walk.coords(p, mb, nb);
          shift = (uint32_t)(nb & 1) * 2;
          walk.next(p, step);
        }
        const int as = local % kAcc;
        if (!wait(&acc_empty[as], (uint32_t)((local / kAcc) & 1) ^ 1, 2)) { ok = false; break; }
        sm100::tc_fence_after();
        const uint32_t d = tmem + as * BN;
        uint32_t sfa = 0, sfb = 0;
        for (int kt = 0; kt < p.k_tiles; ++kt) {
          if (!wait(&full[stage], phase, 3)) { ok = false; break; }
          sm100::tc_fence_after();
          const uint64_t da = sm100::desc_add(da0, stage * S::kA);
          const uint64_t db = sm100::desc_add(db0, stage * S::kB);
          if ((kt & 3) == 0) {
            sf_buf ^= 1;
            sfa = tmem_sf + sf_buf * kSfCols;
            sfb = sfa + kSfaCols;
            const uint64_t dsf = sm100::desc_add(dsf0, stage * S::kSf);
#pragma unroll
            for (int r = 0; r < 1 + sfb_atoms<BN>(); ++r) {
              if constexpr (PAIR) sm100::tmem_cp_32x128b_warpx4_pair(sfa + 4 * r, sm100::desc_add(dsf, r * kSfAtom));
              else sm100::tmem_cp_32x128b_warpx4(sfa + 4 * r, sm100::desc_add(dsf, r * kSfAtom));
            }
          }
          const uint32_t idesc = sm100::idesc_mxf8(PAIR ? 2 * BM : BM, BN, 0) | ((kt & 3) << 4) | ((kt & 3) << 29);
          // Columns past K are zero in shared memory (TMA fills them), so a ragged
          // last k-tile may run whole MMAs.
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t a = sm100::desc_add(da, 32 * j), b = sm100::desc_add(db, 32 * j);
            if constexpr (PAIR) sm100::mma_mxf8_ss_pair(d, a, b, idesc, sfa, sfb + shift, (kt | j) != 0);
            else sm100::mma_mxf8_ss(d, a, b, idesc, sfa, sfb + shift, (kt | j) != 0);
          }
          commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        commit(&acc_full[as]);
      }
      // No MMA may still write TMEM when the CTA (pair) tears down.
      commit(done);
      sm100::mbar_wait(done, 0);
    } else if (PAIR && !leader && sm100::elect_one_sync()) {
      sm100::mbar_wait(done, 0);   // the leader's last commit also arrives here
    }
  } else {
    // ------------------------------------------------------------ epilogue
    const int w = warp - 2;
    const int quad = warp & 3;                 // TMEM lane quadrant of this warp
    const int part = w >> 2;                   // which 64 columns of the tile
    auto release = [&](int as) {
      sm100::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if constexpr (PAIR)
          sm100::mbar_arrive_cluster_relaxed(sm100::mapa(sm100::smem_u32(&acc_empty[as]), 0));
        else
          sm100::mbar_arrive(&acc_empty[as]);
      }
    };
    float* s_bias = reinterpret_cast<float*>(smem + S::offBias) + w * 64;
    const uint32_t bias_addr = sm100::smem_u32(s_bias);
    int local = 0;
    uint32_t res_phase = 0;
    // The bias of the warp's columns passes through shared memory (each lane
    // loads two of 64 and reads all); a tile's is loaded while the tile before
    // it is waited for, its latency out of the way. So are the coordinates.
    float bias0 = 0.0f, bias1 = 0.0f;
    Walk walk(p, tile0);
    int next_mb = 0, next_nb = 0;
    auto fetch = [&]() {
      if (!walk.more()) return;
      walk.coords(p, next_mb, next_nb);
      if (!p.bias) return;
      const int n = next_nb * BN + (EPI == EPI_OUT ? part * 64 : part * 32) + lane, n2 = n + (EPI == EPI_OUT ? 32 : 128);
      bias0 = n < p.N ? rc::ld_in(p.bias + n) : 0.0f;
      bias1 = n2 < p.N ? rc::ld_in(p.bias + n2) : 0.0f;
    };
    fetch();
    for (int tile = tile0; tile < tiles; tile += step, ++local) {
      const int mb = next_mb, nb = next_nb;
      const int rb = PAIR ? mb * 2 + (int)rank : mb;
      const int as = local % kAcc;
      const uint32_t parity = (uint32_t)((local / kAcc) & 1);
      const uint32_t tacc = tmem + as * BN + ((uint32_t)(quad * 32) << 16);
      const int row0 = rb * BM + quad * 32, row = row0 + lane;
      __syncwarp();                            // the last tile's bias has been read
      s_bias[lane] = bias0;
      s_bias[32 + lane] = bias1;
      walk.next(p, step);
      fetch();
      if constexpr (EPI == EPI_OUT) {
        const int col0 = nb * BN + part * 64;
        const bool inside = row0 < p.M && col0 < p.N;
        uint8_t* box = smem + S::offOut + w * S::kBox;
        constexpr int kCols = S::kBoxCols;
        const Out* res = static_cast<const Out*>(p.residual);
        Out* out = static_cast<Out*>(p.out);
        // The box's 128- or 64-byte swizzle: 8 lanes' 16-byte granules hit all banks.
        auto at = [&](int r, int c) {
          return box + r * (kCols * 2) + (((c >> 3) ^ (kCols == 64 ? r & 7 : (r >> 1) & 3)) << 4) + (c & 7) * 2;
        };
        // Rows that do not start on 16 bytes: the warp copies them between the
        // box and memory, lanes along the columns, in pairs where those are on
        // 4 bytes; kBatch loads are in flight at a time.
        const int across = p.pairs ? 2 : 1;
        constexpr int kBatch = 8;
        auto copy_in = [&](int h) {
          const int left = p.N - col0 - h, down = min(32, p.M - row0);
          const Out* from = res + (size_t)row0 * p.ldr + col0 + h;
          for (int c = lane * across; c < kCols; c += 32 * across)
            for (int r0 = 0; r0 < down; r0 += kBatch) {
              uint32_t v[kBatch];
#pragma unroll
              for (int r = 0; r < kBatch; ++r) {
                v[r] = 0;
                if (r0 + r < down && c < left) {
                  const Out* at_r = from + (size_t)(r0 + r) * p.ldr + c;
                  v[r] = across == 2 && c + 1 < left ? rc::ld_in(reinterpret_cast<const uint32_t*>(at_r))
                                                    : rc::ld_in(reinterpret_cast<const uint16_t*>(at_r));
                }
              }
#pragma unroll
              for (int r = 0; r < kBatch; ++r) {
                if (across == 2) *reinterpret_cast<uint32_t*>(at(r0 + r, c)) = v[r];
                else *reinterpret_cast<uint16_t*>(at(r0 + r, c)) = (uint16_t)v[r];
              }
            }
        };
        auto copy_out = [&](int h) {
          const int left = p.N - col0 - h, down = min(32, p.M - row0);
          Out* to = out + (size_t)row0 * p.ldo + col0 + h;
          for (int c = lane * across; c < kCols && c < left; c += 32 * across) {
#pragma unroll 8
            for (int r = 0; r < down; ++r) {
              Out* to_r = to + (size_t)r * p.ldo + c;
              if (across == 2 && c + 1 < left)
                *reinterpret_cast<uint32_t*>(to_r) = *reinterpret_cast<const uint32_t*>(at(r, c));
              else
                *reinterpret_cast<uint16_t*>(to_r) = *reinterpret_cast<const uint16_t*>(at(r, c));
            }
          }
        };
        auto load_residual = [&](int col) {      // one lane, once the last store has read the box
          sm100::mbar_arrive_expect_tx(&res_full[w], S::kBox);
          sm100::tma_load_2d(box, &maps.res, &res_full[w], col, row0);
        };
        if (inside) {
          if (p.staged && lane == 0) {
            sm100::bulk_wait_group_read0();
            if (res) load_residual(col0);
          }
          if (!p.staged && res) copy_in(0);
        }
        if (!__all_sync(0xffffffffu, wait(&acc_full[as], parity, 4))) {
          // Given up; the residual on its way into the box lands before the CTA leaves.
          if (inside && p.staged && res && lane == 0) sm100::mbar_wait(&res_full[w], res_phase);
          break;
        }
        sm100::tc_fence_after();
        uint32_t acc[64];
        load_acc(tacc + part * 64, acc);
        acc_ready(acc);
        release(as);
        if (!inside) continue;
        __syncwarp();
        bool ok = true;
#pragma unroll
        for (int h = 0; h < 64; h += kCols) {
          if (p.staged) {
            if (h) {
              if (lane == 0) {
                sm100::bulk_wait_group_read0();
                if (res) load_residual(col0 + h);
              }
              __syncwarp();
            }
            if (res) {
              if (!(ok = __all_sync(0xffffffffu, wait(&res_full[w], res_phase, 5)))) break;
              res_phase ^= 1;
            }
          } else if (res) {
            if (h) copy_in(h);
            __syncwarp();
          }
          // kStep columns at a time, their loads in flight together (as many as the registers hold).
          constexpr int kStep = BN == 128 ? 16 : 8;
#pragma unroll
          for (int c = 0; c < kCols; c += kStep) {
            float2 v[kStep / 2];
            uint4 r[kStep / 8];
            if (res) {
#pragma unroll
              for (int i = 0; i < kStep / 8; ++i) r[i] = ld_shared4u(sm100::smem_u32(at(lane, c + 8 * i)));
            }
#pragma unroll
            for (int i = 0; i < kStep / 4; ++i) {
              const float4 b = ld_shared4(bias_addr + (h + c + 4 * i) * 4);
              v[2 * i] = make_float2(b.x, b.y);
              v[2 * i + 1] = make_float2(b.z, b.w);
            }
#pragma unroll
            for (int i = 0; i < kStep / 2; ++i)
              v[i] = __fadd2_rn(make_float2(__uint_as_float(acc[h + c + 2 * i]),
                                            __uint_as_float(acc[h + c + 2 * i + 1])), v[i]);
#pragma unroll
            for (int i = 0; i < kStep / 8; ++i) {
              if (res) {
                v[4 * i] = __fadd2_rn(v[4 * i], unpack2<Out>(r[i].x));
                v[4 * i + 1] = __fadd2_rn(v[4 * i + 1], unpack2<Out>(r[i].y));
                v[4 * i + 2] = __fadd2_rn(v[4 * i + 2], unpack2<Out>(r[i].z));
                v[4 * i + 3] = __fadd2_rn(v[4 * i + 3], unpack2<Out>(r[i].w));
              }
              uint32_t o[4];
#pragma unroll
              for (int j = 0; j < 4; ++j) o[j] = fp8b::pack2(v[4 * i + j].x, v[4 * i + j].y, (Out*)nullptr);
              st_shared4(sm100::smem_u32(at(lane, c + 8 * i)), make_uint4(o[0], o[1], o[2], o[3]));
            }
          }
          if (p.staged) {
            sm100::fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0 && col0 + h < p.N) {
              sm100::tma_store_2d(&maps.out, box, col0 + h, row0);
              sm100::bulk_commit_group();
            }
          } else {
            __syncwarp();
            copy_out(h);
            __syncwarp();                        // the box is free again
          }
        }
        if (!ok) break;
      } else {
        uint32_t* s_amax = reinterpret_cast<uint32_t*>(smem + S::offOut + kEpiWarps * S::kBox) + ((local & 1) * 4 + quad) * 4 * 32;
        const bool ok = __all_sync(0xffffffffu, wait(&acc_full[as], parity, 4));
        uint32_t acc[64];                      // 32 gate, then the 32 up columns they pair with
        uint32_t m = 0;
        float y[32];
        if (ok) {
          sm100::tc_fence_after();
          sm100::tmem_ld32(tacc + part * 32, acc);
          sm100::tmem_ld32(tacc + 128 + part * 32, acc + 32);
          acc_ready(acc);
          release(as);
          __syncwarp();
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 bg = ld_shared4(bias_addr + c * 4), bu = ld_shared4(bias_addr + (32 + c) * 4);
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
              const float2 g = __fadd2_rn(make_float2(__uint_as_float(acc[c + i]), __uint_as_float(acc[c + i + 1])),
                                          i ? make_float2(bg.z, bg.w) : make_float2(bg.x, bg.y));
              const float2 u = __fadd2_rn(make_float2(__uint_as_float(acc[32 + c + i]), __uint_as_float(acc[33 + c + i])),
                                          i ? make_float2(bu.z, bu.w) : make_float2(bu.x, bu.y));
              const float2 v = swiglu2(g, u);
              y[c + i] = v.x;
              y[c + i + 1] = v.y;
            }
          }
          const int left = p.H - nb * 128 - part * 32;      // columns of this part that exist: none, 16 or 32
          if (left < 32) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (c >= 16 || left < 16) y[c] = 0.0f;
          }
          float top = 0.0f;
#pragma unroll
          for (int c = 0; c < 32; c += 2) top = rc::absmax3_nan(top, y[c], y[c + 1]);
          m = fp8b::magnitude(top);
          s_amax[part * 32 + lane] = m;
        }
        // The four warps of a lane quadrant share its rows' amax. (The buffer
        // of tile k is written again at tile k + 2, after the barrier of k + 1.)
        if (!sm100::bar_and(1 + quad, 128, ok)) break;
        m = max(max(s_amax[lane], s_amax[32 + lane]), max(s_amax[64 + lane], s_amax[96 + lane]));
        const uint32_t e = fp8b::scale_byte(m);
        const float inv = fp8b::inverse_scale(e);
        // A store from registers would touch 32 rows per instruction: the codes
        // leave by TMA from a box of 32 rows x 32 bytes.
        const int col0 = nb * 128 + part * 32;
        uint8_t* box = smem + S::offOut + w * S::kBox;
        if (lane == 0) sm100::bulk_wait_group_read0();     // the last tile's store has read it
        __syncwarp();
        uint32_t c[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
          c[j] = fp8b::e4m3x4(y[4 * j] * inv, y[4 * j + 1] * inv, y[4 * j + 2] * inv, y[4 * j + 3] * inv);
        const uint32_t dst = sm100::smem_u32(box) + lane * 32;
        st_shared4(dst, make_uint4(c[0], c[1], c[2], c[3]));
        st_shared4(dst + 16, make_uint4(c[4], c[5], c[6], c[7]));
        sm100::fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0 && row0 < p.M && col0 < p.H) {
          sm100::tma_store_2d(&maps.out, box, col0, row0);
          sm100::bulk_commit_group();
        }
        if (part == 0 && row < (p.M + 127) / 128 * 128) {
          const int atoms = fp8b::atoms_of(p.H);
          uint8_t* at = p.scales + ((size_t)rb * atoms + (nb >> 2)) * kSfAtom + lane * 16 + quad * 4;   // rc::sf_offset
          at[nb & 3] = row < p.M ? (uint8_t)e : 0;
          if (nb == p.n_blocks - 1)
            for (int kb = (nb & 3) + 1; kb < 4; ++kb) at[kb] = 0;
        }
      }
    }
    if (lane == 0) sm100::bulk_wait_group0();
  }
  sm100::tc_fence_before();
  __syncthreads();
  // A pair's CTAs leave together: the leader's MMAs read the other CTA's
  // shared memory and write its tensor memory until its `done` wait returns.
  if constexpr (PAIR) sm100::cluster_sync();
  if (warp == 1) {
    __syncwarp();
    sm100::tc_fence_after();
    if constexpr (PAIR) sm100::tmem_dealloc_pair(tmem, kTmemCols);
    else sm100::tmem_dealloc(tmem, kTmemCols);
  }
}

template <int BN, int STAGES, int EPI, bool PAIR, typename Out>
int launch(const Maps& maps, const Params& p, cudaStream_t stream, const char* what) {
  using S = Smem<BN, STAGES, EPI, PAIR>;
  auto kern = tile_kernel<BN, STAGES, EPI, PAIR, Out>;
  static rc::SmemAttrFlags flags = {};
  if (const int r = rc::ensure_smem_attr(flags, reinterpret_cast<const void*>(kern), S::kTotal, what)) return r;
  const int tiles = p.m_blocks * p.n_blocks, sms = rc::sm_count();
  if constexpr (PAIR) {
    const int pairs = tiles < sms / 2 ? tiles : sms / 2;
    return rc::check_launch(
        rc::launch_pdl_cluster(kern, dim3(2 * pairs), dim3(tile_threads<BN>()), S::kTotal, stream, 2, maps, p), what);
  }
  return rc::check_launch(
      rc::launch_pdl(kern, dim3(tiles < sms ? tiles : sms), dim3(tile_threads<BN>()), S::kTotal, stream, maps, p), what);
}

// Four columns n .. n+3 of an output row: its residual (zeros where there is
// none), and the rounded sum's store.
template <typename Out>
__device__ __forceinline__ void load_piece(const Params& p, int row, int n, float (&v)[4]) {
  const Out* res = static_cast<const Out*>(p.residual);
#pragma unroll
  for (int c = 0; c < 4; ++c) v[c] = 0.0f;
  if (!res || row >= p.M) return;
  res += (size_t)row * p.ldr + n;
  if (p.staged && n + 4 <= p.N) {
    const uint2 w = rc::ld_in(reinterpret_cast<const uint2*>(res));
    const float2 lo = unpack2<Out>(w.x), hi = unpack2<Out>(w.y);
    v[0] = lo.x;
    v[1] = lo.y;
    v[2] = hi.x;
    v[3] = hi.y;
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < p.N) v[c] = fp8b::to_float(rc::ld_in(res + c));
  }
}
template <typename Out>
__device__ __forceinline__ void store_piece(const Params& p, int row, int n, const float (&f)[4]) {
  if (row >= p.M) return;
  Out* out = static_cast<Out*>(p.out) + (size_t)row * p.ldo + n;
  if (p.staged && n + 4 <= p.N) {
    Out* tag = nullptr;
    *reinterpret_cast<uint2*>(out) = make_uint2(fp8b::pack2(f[0], f[1], tag), fp8b::pack2(f[2], f[3], tag));
  } else {
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (n + c < p.N) out[c] = fp8b::from_float(f[c], (Out*)nullptr);
  }
}

// ---------------------------------------------------------------- few rows
// The same products with the operands' roles exchanged, for up to 32 rows: W's
// 128 rows are the MMA's M side and all rows of A (BT = 16 or 32 with the zeros
// that fill them up) its N side, so a single row of A costs a 16-column MMA; and
// a cluster of up to 8 CTAs splits K. Each CTA accumulates its k-tiles
// in TMEM and pushes its fp32 partial, row of A by row, into the shared memory
// of the CTA that owns the row (stores do not wait for the other SM, reads
// would); after a cluster barrier each CTA sums its rows' partials in rank
// order (a fixed order: equal inputs give equal bits) and runs the epilogue,
// one warp per row, four columns per lane. SWIGLU runs a gate and an up tile
// side by side (kW = 2): a row's 128 outputs are one warp's, so the block's
// amax is one warp reduction. Measured: 1 x 3072 x 3072 4.0 us (2.35 TB/s of
// weight), 24 x 3072 x 14336 11.0 us (4.1 TB/s), 1 x 512 x 512 2.6 us; bound by
// the launch and the round trips before and after a CTA's k-tiles (4, 14 and 1 here).
constexpr int kRowsThreads = 192;     // producer, MMA issuer, 4 TMEM warps; all 6 in the epilogue

template <int BT, int EPI>
struct RowsSmem {
  static constexpr int kW = EPI == EPI_SWIGLU ? 2 : 1;
  static constexpr int kStage = (kW * BM + BT) * kRowBytes;
  static constexpr int kSf = (kW + 1) * kSfAtom;
  static constexpr int kStages = 98304 / (kStage + kSf);    // two CTAs per SM, but for gated tiles of 32 rows
  static constexpr int kPart = kW * (BT + 8) * BM * 4;      // the partials of the rows this CTA owns, by rank
  static constexpr int offPart = kStages * kStage;
  static constexpr int offSf = offPart + kPart;
  static constexpr int offBar = offSf + kStages * kSf;
  static constexpr int kTotal = offBar + (2 * kStages + 3) * 8;
  static constexpr int kTmem = kW * BT + 2 * 4 * (kW + 1);
  static constexpr int kTmemCols = kTmem <= 32 ? 32 : kTmem <= 64 ? 64 : kTmem <= 128 ? 128 : kTmem <= 256 ? 256 : 512;
  static constexpr int kPerSm = 2 * (kTotal + 1024) <= 233472 ? 2 : 1;    // of 228 KB an SM, 1 KB kept for each CTA
  static_assert(kTotal <= 232448, "shared memory");
};

// (The bounds' second argument tells the register allocator how many CTAs share an
// SM anyway; without it 24 x 3072 x 14336 takes 11.8 us, not 11.0.)
template <int BT, int EPI, typename Out>
__global__ void __launch_bounds__(kRowsThreads, RowsSmem<BT, EPI>::kPerSm)
rows_kernel(const __grid_constant__ Maps maps, const Params p, int split) {
  using S = RowsSmem<BT, EPI>;
  constexpr int kW = S::kW, STAGES = S::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::offBar);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  volatile int* abort_flag = reinterpret_cast<volatile int*>(acc_full + 1);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 2);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)sm100::cluster_ctarank();
  const int wt = blockIdx.x / split;                            // W's block of 128 rows, or of 128 gate and 128 up rows
  const int kt0 = (int)((long long)rank * p.k_tiles / split), kt1 = (int)((long long)(rank + 1) * p.k_tiles / split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    sm100::mbar_init(acc_full, 1);
    *abort_flag = 0;
    sm100::fence_mbar_init();
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, S::kTmemCols);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_arrive_relaxed();   // this CTA runs; waited for before the first store into a peer
  sm100::tc_fence_after();
  rc::pdl_trigger();
  rc::pdl_wait();
  const uint32_t tmem = *tmem_slot, tmem_sf = tmem + kW * BT;
  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int site) -> bool {
    if (sm100::mbar_wait(bar, parity, abort_flag)) return true;
    if (!*abort_flag) {
      rc::device_fail(kKernFp8Block, site);
      *abort_flag = 1;
    }
    return false;
  };

  if (warp == 0) {
    if (sm100::elect_one_sync()) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!wait(&empty[stage], phase ^ 1, 11)) break;
        uint8_t* a = smem + stage * S::kStage;
        uint8_t* sf = smem + S::offSf + stage * S::kSf;
        const bool atom = (kt & 3) == 0 || kt == kt0;
        const int line = (kt >> 2) * 4;
        sm100::mbar_arrive_expect_tx(&full[stage], S::kStage + (atom ? S::kSf : 0));
#pragma unroll
        for (int w = 0; w < kW; ++w)
          sm100::tma_load_2d(a + w * BM * kRowBytes, &maps.b, &full[stage], kt * kRowBytes, (wt * kW + w) * BM);
        sm100::tma_load_2d(a + kW * BM * kRowBytes, &maps.a, &full[stage], kt * kRowBytes, 0);
        if (atom) {
#pragma unroll
          for (int w = 0; w < kW; ++w)
            sm100::tma_load_2d(sf + w * kSfAtom, &maps.sfb, &full[stage], 0, (wt * kW + w) * p.katoms * 4 + line);
          sm100::tma_load_2d(sf + kW * kSfAtom, &maps.sfa, &full[stage], 0, line);
        }
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      for (int s = 0; s < STAGES && issued > 0; ++s, --issued) {   // loads land before the CTA goes on
        if (stage == 0) { stage = STAGES; phase ^= 1; }
        --stage;
        sm100::mbar_wait(&full[stage], phase);
      }
    }
  } else if (warp == 1) {
    if (sm100::elect_one_sync()) {
      int stage = 0, sf_buf = 1;
      uint32_t phase = 0, sfw = 0;
      const uint64_t d0 = sm100::desc_kmajor_sw128(sm100::smem_u32(smem));
      const uint64_t dsf0 = sm100::desc_sf_rows(sm100::smem_u32(smem + S::offSf));
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!wait(&full[stage], phase, 12)) break;
        sm100::tc_fence_after();
        if ((kt & 3) == 0 || kt == kt0) {
          sf_buf ^= 1;
          sfw = tmem_sf + sf_buf * 4 * (kW + 1);
#pragma unroll
          for (int w = 0; w <= kW; ++w)
            sm100::tmem_cp_32x128b_warpx4(sfw + 4 * w, sm100::desc_add(dsf0, stage * S::kSf + w * kSfAtom));
        }
        const uint32_t idesc = sm100::idesc_mxf8(BM, BT, 0) | ((kt & 3) << 4) | ((kt & 3) << 29);
        const uint64_t da = sm100::desc_add(d0, stage * S::kStage);
        const uint64_t db = sm100::desc_add(da, kW * BM * kRowBytes);
#pragma unroll
        for (int w = 0; w < kW; ++w)
#pragma unroll
          for (int j = 0; j < 4; ++j)
            sm100::mma_mxf8_ss(tmem + w * BT, sm100::desc_add(da, w * BM * kRowBytes + 32 * j),
                               sm100::desc_add(db, 32 * j), idesc, sfw + 4 * w, sfw + 4 * kW, kt != kt0 || j != 0);
        sm100::tc_commit(&empty[stage]);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      sm100::tc_commit(acc_full);
      sm100::mbar_wait(acc_full, 0);
    }
  }
  __syncwarp();
  // Every CTA of the cluster runs: their shared memory may be written. The TMEM
  // warps are here at once, so the barrier's latency is behind the main loop.
  sm100::cluster_wait();
  const int rows = p.M, per = (rows + split - 1) / split;       // at most BT; rank q owns rows q * per ...
  float* part = reinterpret_cast<float*>(smem + S::offPart);    // [rank][kW][per][128]
  bool ok = true;
  if (warp >= 2) {
    ok = __all_sync(0xffffffffu, wait(acc_full, 0, 13));
    sm100::tc_fence_after();
  }
  if (warp >= 2 && ok) {
    const int quad = warp & 3;
    constexpr int kChunk = BT < 32 ? BT : 32;
    const uint32_t mine = sm100::smem_u32(part) + (rank * kW * per * BM + quad * 32 + lane) * 4;
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      int owner = 0, i = 0;
      uint32_t to = sm100::mapa(mine + w * per * BM * 4, 0);
      for (int c = 0; c < BT; c += kChunk) {
        if (c >= rows) break;
        uint32_t acc[kChunk];
        const uint32_t addr = tmem + w * BT + c + ((uint32_t)(quad * 32) << 16);
        if constexpr (kChunk == 16) sm100::tmem_ld16(addr, acc);
        else sm100::tmem_ld32(addr, acc);
        acc_ready(acc);
#pragma unroll
        for (int j = 0; j < kChunk; ++j) {
          if (c + j >= rows) break;
          asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to), "r"(acc[j]) : "memory");
          to += BM * 4;
          if (++i == per) {
            i = 0;
            ++owner;
            to = sm100::mapa(mine + w * per * BM * 4, min(owner, split - 1));
          }
        }
      }
    }
    sm100::tc_fence_before();
  }
  sm100::cluster_sync();
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, S::kTmemCols);
  }
  // A warp takes kRows of this CTA's rows at a time, their loads in flight together.
  const int first = rank * per, mine = min(per, rows - first);
  constexpr int kRows = BT / 16;
  float4 bias[kW];
  if (p.bias) {
#pragma unroll
    for (int w = 0; w < kW; ++w) {
      const int n = (wt * kW + w) * BM + lane * 4;
      bias[w].x = n < p.N ? rc::ld_in(p.bias + n) : 0.0f;
      bias[w].y = n + 1 < p.N ? rc::ld_in(p.bias + n + 1) : 0.0f;
      bias[w].z = n + 2 < p.N ? rc::ld_in(p.bias + n + 2) : 0.0f;
      bias[w].w = n + 3 < p.N ? rc::ld_in(p.bias + n + 3) : 0.0f;
    }
  } else {
#pragma unroll
    for (int w = 0; w < kW; ++w) bias[w] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  for (int i = warp * kRows; i < mine; i += kRowsThreads / 32 * kRows) {
    float4 v[kRows][kW];
#pragma unroll
    for (int j = 0; j < kRows; ++j)
#pragma unroll
      for (int w = 0; w < kW; ++w) v[j][w] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float near[kRows][4];                                          // residual
    const int n = wt * BM + lane * 4;
    if constexpr (EPI == EPI_OUT) {
#pragma unroll
      for (int j = 0; j < kRows; ++j) load_piece<Out>(p, first + min(i + j, mine - 1), n, near[j]);
    }
    for (int q = 0; q < split; ++q) {
#pragma unroll
      for (int j = 0; j < kRows; ++j)
#pragma unroll
        for (int w = 0; w < kW; ++w) {
          // past the last row: the last once more, not stored
          const float4 x = ld_shared4(sm100::smem_u32(part) + (((q * kW + w) * per + min(i + j, mine - 1)) * BM + lane * 4) * 4);
          v[j][w].x += x.x;
          v[j][w].y += x.y;
          v[j][w].z += x.z;
          v[j][w].w += x.w;
        }
    }
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      if (i + j >= mine) break;
      const int row = first + i + j;
#pragma unroll
      for (int w = 0; w < kW; ++w) {
        v[j][w].x += bias[w].x;
        v[j][w].y += bias[w].y;
        v[j][w].z += bias[w].z;
        v[j][w].w += bias[w].w;
      }
      if constexpr (EPI == EPI_OUT) {
        const float f[4] = {v[j][0].x + near[j][0], v[j][0].y + near[j][1], v[j][0].z + near[j][2], v[j][0].w + near[j][3]};
        store_piece<Out>(p, row, n, f);
      } else {
        const float4 g = v[j][0], u = v[j][kW - 1];
        const float2 lo = swiglu2(make_float2(g.x, g.y), make_float2(u.x, u.y));
        const float2 hi = swiglu2(make_float2(g.z, g.w), make_float2(u.z, u.w));
        float y[4] = {lo.x, lo.y, hi.x, hi.y};
        const int col = wt * 128 + lane * 4;
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          if (col >= p.H) y[c] = 0.0f;                       // H is a multiple of 16
          m = max(m, fp8b::magnitude(y[c]));
        }
        const uint32_t e = fp8b::scale_byte(__reduce_max_sync(0xffffffffu, m));
        const float inv = fp8b::inverse_scale(e);
        if (col < p.H)
          *reinterpret_cast<uint32_t*>(p.codes + (size_t)row * p.H + col) =
              fp8b::e4m3x4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
        if (lane == 0) p.scales[rc::sf_offset(row, wt, fp8b::atoms_of(p.H))] = (uint8_t)e;
      }
    }
  }
  if constexpr (EPI == EPI_SWIGLU) {
    // Zero scales: rows past M of the atom's 128, and the last block's neighbours
    // up to the atom.
    const int atoms = fp8b::atoms_of(p.H);
    if (rank == 0)
      for (int row = threadIdx.x; row < 128; row += kRowsThreads) {
        if (row >= p.M) p.scales[rc::sf_offset(row, wt, atoms)] = 0;
        if (wt == p.n_blocks - 1)
          for (int kb = p.n_blocks; kb < 4 * atoms; ++kb) p.scales[rc::sf_offset(row, kb, atoms)] = 0;
      }
  }
}

// CTAs of a cluster along K: as many as every cluster of the launch finds room
// with at once, up to 8 and the k-tiles; one cluster too many is a second wave. A
// cluster stays within one group of SMs, so the room is less than the SMs', and
// the driver knows it for one CTA on each (clusters of 2 to 8 on a B200: 74, 45,
// 33, 26, 22, 15, 15). Gated tiles of 32 rows are alone on their SM. The others
// run two to an SM: twice the room, and clusters of 6 and 8 at least as many as
// of 3 and 4 (measured: 45 of 45, 33 of 33; of 4 not as many as of 2, 71 of 74).
// Measured (us) beside two CTAs for every SM: gated 32 x 8192 x 512 5.8 (10.4), 32
// x 2048 x 4096 6.9 (11.9), 16 x 4736 x 4096 11.4 (16.3), 1 x 6144 x 3072 5.3 (8.0).
template <int BT, int EPI, typename Out>
int rows_split(const Params& p) {
  using S = RowsSmem<BT, EPI>;
  static std::atomic<int> cache[rc::kMaxDevices][9] = {};    // clusters + 1, 0: not asked yet
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= rc::kMaxDevices) return 1;
  auto clusters = [&](int size) {
    int n = cache[dev][size].load(std::memory_order_relaxed) - 1;
    if (n < 0) {
      n = rc::resident_clusters(rows_kernel<BT, EPI, Out>, dim3(kRowsThreads), S::kTotal, (unsigned)size);
      cache[dev][size].store(n + 1, std::memory_order_relaxed);
    }
    return n;
  };
  for (int split = p.k_tiles < 8 ? p.k_tiles : 8; split > 1; --split) {
    int room = S::kPerSm * clusters(split);
    if (S::kPerSm == 2 && (split == 6 || split == 8) && room < clusters(split / 2)) room = clusters(split / 2);
    if (p.n_blocks <= room) return split;
  }
  return 1;
}

template <int BT, int EPI, typename Out>
int launch_rows(const Maps& maps, const Params& p, cudaStream_t stream, const char* what) {
  using S = RowsSmem<BT, EPI>;
  auto kern = rows_kernel<BT, EPI, Out>;
  static rc::SmemAttrFlags flags = {};
  if (const int r = rc::ensure_smem_attr(flags, reinterpret_cast<const void*>(kern), S::kTotal, what)) return r;
  const int split = rows_split<BT, EPI, Out>(p);
  return rc::check_launch(rc::launch_pdl_cluster(kern, dim3((unsigned)(p.n_blocks * split)),
                                                 dim3(kRowsThreads), S::kTotal, stream, (unsigned)split, maps, p, split),
                          what);
}

// ---------------------------------------------------------------- split K
// OUT for too few 128 x 128 tiles and too many rows for the rows kernel: a
// cluster of SPLIT CTAs takes one tile, each a range of k-tiles, and CTA q ends
// up with the tile's columns [q * 128 / SPLIT, ...): every CTA lays its fp32
// partial out by owner in the operands' stages and sends each owner its slice
// as one bulk copy between the two SMs' shared memory, counted on the owner's
// barrier (stores and loads of single values between SMs took 3 us longer);
// the owner sums the slices in rank order.
constexpr int kSplitThreads = 64 + 256;

template <int SPLIT>
struct SplitSmem {
  static constexpr int kStages = 4;
  static constexpr int kCols = BM / SPLIT;                  // columns per owner
  static constexpr int kStage = 2 * BM * kRowBytes, kSf = 2 * kSfAtom;
  static constexpr int kSlice = BM * kCols * 4;             // an owner's columns of one CTA's partial, [128][kCols] fp32
  static constexpr int offIn = kStages * kStage;            // the slices this CTA owns, by rank
  static constexpr int offSf = offIn + SPLIT * kSlice;
  static constexpr int offBar = offSf + kStages * kSf;
  static constexpr int kTotal = offBar + (2 * kStages + 4) * 8;
  static_assert(kTotal <= 232448 && SPLIT * kSlice <= kStages * kStage, "shared memory");
};

template <int SPLIT, typename Out>
__global__ void __launch_bounds__(kSplitThreads, 1)
split_kernel(const __grid_constant__ Maps maps, const Params p) {
  using S = SplitSmem<SPLIT>;
  constexpr int STAGES = S::kStages, kCols = S::kCols;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::offBar);
  uint64_t* empty = full + STAGES;
  uint64_t* acc_full = empty + STAGES;
  uint64_t* slices = acc_full + 1;               // the other CTAs' slices have arrived
  volatile int* abort_flag = reinterpret_cast<volatile int*>(acc_full + 2);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_full + 3);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = (int)sm100::cluster_ctarank();
  const int tile = blockIdx.x / SPLIT;
  const int mb = tile % p.m_blocks, nb = tile / p.m_blocks;
  const int kt0 = (int)((long long)rank * p.k_tiles / SPLIT), kt1 = (int)((long long)(rank + 1) * p.k_tiles / SPLIT);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      sm100::mbar_init(&full[s], 1);
      sm100::mbar_init(&empty[s], 1);
    }
    sm100::mbar_init(acc_full, 1);
    sm100::mbar_init(slices, 1);
    *abort_flag = 0;
    sm100::fence_mbar_init();
    sm100::mbar_arrive_expect_tx(slices, (SPLIT - 1) * S::kSlice);
  }
  if (warp == 1) {
    sm100::tmem_alloc(tmem_slot, 256);
    sm100::tmem_relinquish();
  }
  sm100::tc_fence_before();
  __syncthreads();
  sm100::cluster_sync();                         // every CTA's barriers are there before a slice is sent
  sm100::tc_fence_after();
  rc::pdl_trigger();
  rc::pdl_wait();
  const uint32_t tmem = *tmem_slot, tmem_sf = tmem + BM;
  auto wait = [&](uint64_t* bar, uint32_t parity, unsigned int site) -> bool {
    if (sm100::mbar_wait(bar, parity, abort_flag)) return true;
    if (!*abort_flag) {
      rc::device_fail(kKernFp8Block, site);
      *abort_flag = 1;
    }
    return false;
  };

  if (warp == 0) {
    if (sm100::elect_one_sync()) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!wait(&empty[stage], phase ^ 1, 21)) break;
        uint8_t* a = smem + stage * S::kStage;
        uint8_t* sf = smem + S::offSf + stage * S::kSf;
        const bool atom = (kt & 3) == 0 || kt == kt0;
        const int line = (kt >> 2) * 4;
        sm100::mbar_arrive_expect_tx(&full[stage], S::kStage + (atom ? S::kSf : 0));
        sm100::tma_load_2d(a, &maps.a, &full[stage], kt * kRowBytes, mb * BM);
        sm100::tma_load_2d(a + BM * kRowBytes, &maps.b, &full[stage], kt * kRowBytes, nb * BM);
        if (atom) {
          sm100::tma_load_2d(sf, &maps.sfa, &full[stage], 0, mb * p.katoms * 4 + line);
          sm100::tma_load_2d(sf + kSfAtom, &maps.sfb, &full[stage], 0, nb * p.katoms * 4 + line);
        }
        ++issued;
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      for (int s = 0; s < STAGES && issued > 0; ++s, --issued) {   // loads land before the CTA goes on
        if (stage == 0) { stage = STAGES; phase ^= 1; }
        --stage;
        sm100::mbar_wait(&full[stage], phase);
      }
    }
  } else if (warp == 1) {
    if (sm100::elect_one_sync()) {
      int stage = 0, sf_buf = 1;
      uint32_t phase = 0, sfa = 0;
      const uint64_t d0 = sm100::desc_kmajor_sw128(sm100::smem_u32(smem));
      const uint64_t dsf0 = sm100::desc_sf_rows(sm100::smem_u32(smem + S::offSf));
      for (int kt = kt0; kt < kt1; ++kt) {
        if (!wait(&full[stage], phase, 22)) break;
        sm100::tc_fence_after();
        if ((kt & 3) == 0 || kt == kt0) {
          sf_buf ^= 1;
          sfa = tmem_sf + sf_buf * 8;
          sm100::tmem_cp_32x128b_warpx4(sfa, sm100::desc_add(dsf0, stage * S::kSf));
          sm100::tmem_cp_32x128b_warpx4(sfa + 4, sm100::desc_add(dsf0, stage * S::kSf + kSfAtom));
        }
        const uint32_t idesc = sm100::idesc_mxf8(BM, BM, 0) | ((kt & 3) << 4) | ((kt & 3) << 29);
        const uint64_t da = sm100::desc_add(d0, stage * S::kStage), db = sm100::desc_add(da, BM * kRowBytes);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          sm100::mma_mxf8_ss(tmem, sm100::desc_add(da, 32 * j), sm100::desc_add(db, 32 * j), idesc, sfa, sfa + 4,
                             kt != kt0 || j != 0);
        sm100::tc_commit(&empty[stage]);
        if (++stage == STAGES) { stage = 0; phase ^= 1; }
      }
      sm100::tc_commit(acc_full);
      sm100::mbar_wait(acc_full, 0);
    }
  }
  __syncwarp();
  // 16-byte piece `c` (of kCols / 4) of row r of a slice: pieces are swizzled by
  // the row, so that 8 rows' (or one row's) pieces hit all banks.
  constexpr int kPieces = kCols / 4;
  auto piece = [&](int r, int c) {
    return (uint32_t)((r * kPieces + (c ^ (r & (kPieces < 8 ? kPieces - 1 : 7)))) * 16);
  };
  const uint32_t out_slices = sm100::smem_u32(smem), in_slices = sm100::smem_u32(smem + S::offIn);
  constexpr int kTasks = BM * kPieces / 256;                // 4-column pieces of the owned slice per thread
  const int t0 = (int)threadIdx.x - 64, n = nb * BM + rank * kCols + t0 % kPieces * 4;   // its columns: n .. n + 3
  float near[kTasks][4], bias[4];
  if (warp >= 2) {
    // Residual and bias, in flight over the main loop.
#pragma unroll
    for (int c = 0; c < 4; ++c) bias[c] = p.bias && n + c < p.N ? rc::ld_in(p.bias + n + c) : 0.0f;
#pragma unroll
    for (int i = 0; i < kTasks; ++i) {
      const int row = mb * BM + (t0 + i * 256) / kPieces;
      load_piece<Out>(p, row, n, near[i]);
    }
    const int quad = warp & 3, half = (warp - 2) >> 2, r = quad * 32 + lane;
    if (__all_sync(0xffffffffu, wait(acc_full, 0, 23))) {
      sm100::tc_fence_after();
      uint32_t acc[64];
      load_acc(tmem + half * 64 + ((uint32_t)(quad * 32) << 16), acc);
      acc_ready(acc);
#pragma unroll
      for (int c = 0; c < 64; c += 4) {
        const int col = half * 64 + c, q = col / kCols;
        const uint32_t to = (q == rank ? in_slices : out_slices) + q * S::kSlice + piece(r, col % kCols / 4);
        st_shared4(to, make_uint4(acc[c], acc[c + 1], acc[c + 2], acc[c + 3]));
      }
      sm100::tc_fence_before();
    }
    sm100::fence_proxy_async_smem();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (t0 < SPLIT && t0 != rank)                           // thread q sends rank q its slice
      asm volatile(
          "cp.async.bulk.shared::cluster.shared::cta.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
              sm100::mapa(in_slices + rank * S::kSlice, t0)),
          "r"(out_slices + t0 * S::kSlice), "r"((uint32_t)S::kSlice), "r"(sm100::mapa(sm100::smem_u32(slices), t0))
          : "memory");
    if (__all_sync(0xffffffffu, wait(slices, 0, 24))) {
#pragma unroll
      for (int i = 0; i < kTasks; ++i) {
        const int r = (t0 + i * 256) / kPieces, row = mb * BM + r;
        float f[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int q = 0; q < SPLIT; ++q) {
          const float4 x = ld_shared4(in_slices + q * S::kSlice + piece(r, t0 % kPieces));
          f[0] += x.x;
          f[1] += x.y;
          f[2] += x.z;
          f[3] += x.w;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) f[c] = f[c] + bias[c] + near[i][c];
        store_piece<Out>(p, row, n, f);
      }
    }
  }
  sm100::cluster_sync();      // no CTA leaves while its slices are on their way
  if (warp == 1) {
    sm100::tc_fence_after();
    sm100::tmem_dealloc(tmem, 256);
  }
}

template <int SPLIT, typename Out>
int launch_split(const Maps& maps, const Params& p, cudaStream_t stream, const char* what) {
  using S = SplitSmem<SPLIT>;
  auto kern = split_kernel<SPLIT, Out>;
  static rc::SmemAttrFlags flags = {};
  if (const int r = rc::ensure_smem_attr(flags, reinterpret_cast<const void*>(kern), S::kTotal, what)) return r;
  return rc::check_launch(rc::launch_pdl_cluster(kern, dim3((unsigned)(p.m_blocks * p.n_blocks * SPLIT)),
                                                 dim3(kSplitThreads), S::kTotal, stream, SPLIT, maps, p),
                          what);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// How a product runs.
struct Plan {
  int bt;        // rows kernel with BT rows of A per tile; 0: tile kernel
  int split;     // split kernel (bt 0, split > 1): CTAs per tile along K
  int bn;        // tile kernel: columns per tile
  bool pair;     // tile kernel: CTA pairs (256-row tiles)
};

// Up to 32 rows run on the rows kernel, which splits K itself (rows_split; us at
// split 1 / 2 / 4 / 8: 1 x 512 x 512 3.2 / 2.8 / 2.6 / -, 1 x 3072 x 3072 6.7 / 4.9 /
// 4.0 / 4.3, 24 x 3072 x 14336 - / - / 14.0 / 11.1; the tile kernel 4.1, 7.1 and
// 33). More rows take the tile kernel whose waves cost least: cycles of a k-tile
// and of a tile's hand-over with every SM busy, and of what comes before the first
// and after the last tile, fitted to measurements. What they decide (with a
// residual, us on 128 x 128 / pairs' 256 x 192 / 256 x
// 256): 3520 x 768 x 512 6.1 / 6.5 / 7.3, 880 x 3072 x 3072 14.6 / 11.7 /
// 13.9, 1759 x 3072 x 3072 22.1 / 18.3 / 22.0, 2500 x 4096 x 2048 27.0 / 21.6 /
// 25.4, 300 x 9216 x 3072 17.1 / 18.3 / 15.5, 7040 x 3072 x 14336 318 / 250 /
// 238. 128 x 128 tiles are bound by the operands' way into the SM (32 KB per
// 256 cycles of MMA); 256 columns leave tensor memory for one accumulator
// only, so their hand-over is not hidden.
Plan plan_for(int M, int N, int K, bool swiglu) {
  const int sms = rc::sm_count(), k_tiles = fp8b::blocks_of(K);
  auto up = [](long long a, long long b) { return (a + b - 1) / b; };
  Plan q{0, 1, 256, false};
  if (M <= 32) {
    q.bt = M <= 16 ? 16 : 32;
    return q;
  }
  struct Tile { int m, n, k_tile, tile, ends; };
  auto cost = [&](const Tile& t) {
    return up(up(M, t.m) * up(N, t.n), t.m == 256 ? sms / 2 : sms) * ((long long)t.k_tile * k_tiles + t.tile) + t.ends;
  };
  const long long pair = cost({256, 256, 520, 1300, 3000});
  if (swiglu) {
    q.pair = pair < cost({128, 256, 620, 1300, 3000});
    return q;
  }
  const long long narrow = cost({256, 192, 420, 200, 4100}), one = cost({128, 128, 400, 300, 1500});
  q.pair = pair < one || narrow < one;
  q.bn = !q.pair ? 128 : narrow < pair ? 192 : 256;
  // Few tiles and a long K: split while the clusters find room at once (of 8
  // CTAs, 12 do on 148 SMs). The exchange costs what about 9, 15 and 21
  // k-tiles do (us, split 1 / 2 / 4 / 8: 128 x 3072 x 3072 7.6 / 7.0 / 7.4 / -,
  // 500 x 500 x 5008 18.9 / 12.7 / 10.0 / -, 100 x 200 x 10000 30.5 / 18.0 /
  // 11.8 / 9.2, 300 x 3072 x 14336 31.3 / 24.0 / - / -; 128 x 768 x 512 4.2 /
  // 5.9).
  const long long tiles = up(M, 128) * up(N, 128);
  const struct { int split, ctas, exchange; } kSplits[] = {{2, sms, 3600}, {4, sms * 7 / 8, 6000}, {8, sms * 2 / 3, 8500}};
  long long best = q.pair ? (narrow < pair ? narrow : pair) : one;
  for (const auto& x : kSplits) {
    const long long with = 400 * up(k_tiles, x.split) + 1800 + x.exchange;
    if (tiles * x.split > x.ctas || k_tiles < x.split || with >= best) continue;
    best = with;
    q.pair = false;
    q.bn = 128;
    q.split = x.split;
  }
  return q;
}

// Tensor maps the two products share. N: rows of W.
int prepare(const char* what, const void* a, long long lda, const void* sa, const void* b, long long ldb,
            const void* sb, int M, int N, int K, bool swiglu, const Plan& q, Params& p, Maps& maps) {
  const int rows_a = q.bt ? q.bt : BM, rows_b = q.bt ? BM : q.pair ? q.bn / 2 : q.bn;   // TMA boxes
  const int tile_m = q.bt ? q.bt : q.pair ? 2 * BM : BM, tile_n = q.bt ? (swiglu ? 256 : 128) : q.bn;
  p.M = M;
  p.N = N;
  p.K = K;
  p.k_tiles = fp8b::blocks_of(K);
  p.katoms = fp8b::atoms_of(K);
  p.m_blocks = (M + tile_m - 1) / tile_m;
  p.n_blocks = (N + tile_n - 1) / tile_n;
  // A wave of (pairs of) SMs takes a group of row blocks times as many column
  // blocks as are left: near to square, it touches the fewest operand panels.
  p.group_m = q.pair ? 8 : 12;
  if (p.group_m > p.m_blocks) p.group_m = p.m_blocks;
  const int last = p.m_blocks % p.group_m ? p.m_blocks % p.group_m : p.group_m;
  p.inv_group = (uint32_t)((0x100000000ull + p.group_m - 1) / p.group_m);
  p.inv_last = (uint32_t)((0x100000000ull + last - 1) / last);
  const long long lines_a = 4LL * p.katoms * ((M + 127) / 128), lines_b = 4LL * p.katoms * ((N + 127) / 128);
  if ((long long)p.m_blocks * p.n_blocks * 8 > INT32_MAX || p.n_blocks > (1 << 24) || lines_a > INT32_MAX || lines_b > INT32_MAX)
    return rc::set_error(RC_ERR_UNSUPPORTED, "%s: %d x %d x %d is too large", what, M, N, K);
  const uint32_t box_a[2] = {kRowBytes, (uint32_t)rows_a}, box_b[2] = {kRowBytes, (uint32_t)rows_b}, box_s[2] = {128, 4};
  const uint64_t da[2] = {(uint64_t)K, (uint64_t)M}, db[2] = {(uint64_t)K, (uint64_t)N};
  const uint64_t sta[1] = {(uint64_t)lda}, stb[1] = {(uint64_t)ldb}, sts[1] = {128};
  const uint64_t dsa[2] = {128, (uint64_t)lines_a}, dsb[2] = {128, (uint64_t)lines_b};
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int r;
  if ((r = rc::encode_tmap(&maps.a, u8, 2, const_cast<void*>(a), da, sta, box_a, CU_TENSOR_MAP_SWIZZLE_128B, what)))
    return r;
  if ((r = rc::encode_tmap(&maps.b, u8, 2, const_cast<void*>(b), db, stb, box_b, CU_TENSOR_MAP_SWIZZLE_128B, what)))
    return r;
  if ((r = rc::encode_tmap(&maps.sfa, u8, 2, const_cast<void*>(sa), dsa, sts, box_s, CU_TENSOR_MAP_SWIZZLE_NONE, what)))
    return r;
  if ((r = rc::encode_tmap(&maps.sfb, u8, 2, const_cast<void*>(sb), dsb, sts, box_s, CU_TENSOR_MAP_SWIZZLE_NONE, what)))
    return r;
  maps.out = maps.res = maps.a;
  return RC_OK;
}

int check_operands(const char* what, const void* a, long long lda, const void* sa, const void* b, long long ldb,
                   const void* sb, const float* bias, int M, int N, int K) {
  if (M < 0 || N <= 0 || K <= 0 || K % 16)
    return rc::set_error(RC_ERR_ARG, "%s: K must be a positive multiple of 16 (got M %d, N %d, K %d)", what, M, N, K);
  if (lda < K || lda % 16 || ldb < K || ldb % 16)
    return rc::set_error(RC_ERR_ARG, "%s: row strides must hold K columns and be multiples of 16 bytes", what);
  if (!M) return RC_OK;
  if (!a || !sa || !b || !sb) return rc::set_error(RC_ERR_ARG, "%s: null operand", what);
  if (!aligned16(a) || !aligned16(sa) || !aligned16(b) || !aligned16(sb) || !aligned16(bias))
    return rc::set_error(RC_ERR_ARG, "%s: operands, scales and bias must be 16-byte aligned", what);
  return RC_OK;
}

template <int EPI, typename Out>
int run(const Maps& maps, const Params& p, const Plan& q, cudaStream_t stream, const char* what) {
  if (q.bt == 16) return launch_rows<16, EPI, Out>(maps, p, stream, what);
  if (q.bt == 32) return launch_rows<32, EPI, Out>(maps, p, stream, what);
  if constexpr (EPI == EPI_OUT) {
    if (q.split == 2) return launch_split<2, Out>(maps, p, stream, what);
    if (q.split == 4) return launch_split<4, Out>(maps, p, stream, what);
    if (q.split == 8) return launch_split<8, Out>(maps, p, stream, what);
  }
  if constexpr (EPI == EPI_OUT)
    if (q.bn == 192) return launch<192, 6, EPI, true, Out>(maps, p, stream, what);
  if (q.pair) return launch<256, EPI == EPI_OUT ? 5 : 6, EPI, true, Out>(maps, p, stream, what);
  if constexpr (EPI == EPI_OUT) return launch<128, 5, EPI, false, Out>(maps, p, stream, what);
  else return launch<256, 4, EPI, false, Out>(maps, p, stream, what);
}

}  // namespace

RC_DEVICE_ERROR_ACCESSOR(fp8_block)

extern "C" {

int rc_fp8_block_gemm(const uint8_t* a, long long lda, const uint8_t* a_scales, const uint8_t* b, long long ldb,
                      const uint8_t* b_scales, const float* bias, int M, int N, int K, int out_dtype,
                      const void* residual, long long ldr, void* out, long long ldo, cudaStream_t stream) {
  const char* what = "rc_fp8_block_gemm";
  if (out_dtype != fp8b::kBF16 && out_dtype != fp8b::kF16)
    return rc::set_error(RC_ERR_ARG, "%s: out_dtype must be 1 (bf16) or 2 (fp16)", what);
  int r = check_operands(what, a, lda, a_scales, b, ldb, b_scales, bias, M, N, K);
  if (r || !M) return r;
  if (!out || ldo < N || (residual && ldr < N) || reinterpret_cast<uintptr_t>(out) % 2 ||
      reinterpret_cast<uintptr_t>(residual) % 2)
    return rc::set_error(RC_ERR_ARG, "%s: out and residual must be rows of at least N columns", what);
  const Plan q = plan_for(M, N, K, false);
  Params p{};
  Maps maps;
  if ((r = prepare(what, a, lda, a_scales, b, ldb, b_scales, M, N, K, false, q, p, maps))) return r;
  p.bias = bias;
  p.out = out;
  p.ldo = ldo;
  p.residual = residual;
  p.ldr = ldr;
  // TMA moves the output (and the residual) where rows start on 16 bytes.
  p.staged = aligned16(out) && ldo % 8 == 0 && aligned16(residual) && (!residual || ldr % 8 == 0);
  p.pairs = ((reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(residual)) % 4 | ldo % 2 | (residual ? ldr % 2 : 0)) == 0;
  if (p.staged && !q.bt && q.split == 1) {
    const auto type = out_dtype == fp8b::kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const uint64_t dims[2] = {(uint64_t)N, (uint64_t)M};
    const bool wide = q.bn != 128;                       // the warp's staging box (Smem::kBoxCols)
    const uint32_t box[2] = {wide ? 32u : 64u, 32};
    const auto swizzle = wide ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B;
    const uint64_t so[1] = {(uint64_t)ldo * 2}, sr[1] = {(uint64_t)ldr * 2};
    if ((r = rc::encode_tmap(&maps.out, type, 2, out, dims, so, box, swizzle, what))) return r;
    if (residual && (r = rc::encode_tmap(&maps.res, type, 2, const_cast<void*>(residual), dims, sr, box,
                                         swizzle, what)))
      return r;
  }
  if (out_dtype == fp8b::kBF16) return run<EPI_OUT, __nv_bfloat16>(maps, p, q, stream, what);
  return run<EPI_OUT, __half>(maps, p, q, stream, what);
}

int rc_fp8_block_swiglu_gemm(const uint8_t* a, long long lda, const uint8_t* a_scales, const uint8_t* b,
                             long long ldb, const uint8_t* b_scales, const float* bias, int M, int H, int K,
                             uint8_t* codes, uint8_t* scales, cudaStream_t stream) {
  const char* what = "rc_fp8_block_swiglu_gemm";
  if (H <= 0 || H % 16 || H > (1 << 29)) return rc::set_error(RC_ERR_ARG, "%s: H must be a positive multiple of 16 (got %d)", what, H);
  const int N = (H + 127) / 128 * 256;
  int r = check_operands(what, a, lda, a_scales, b, ldb, b_scales, bias, M, N, K);
  if (r || !M) return r;
  if (!codes || !scales || !aligned16(codes) || !aligned16(scales))
    return rc::set_error(RC_ERR_ARG, "%s: codes and scales must be 16-byte aligned and not null", what);
  const Plan q = plan_for(M, N, K, true);
  Params p{};
  Maps maps;
  if ((r = prepare(what, a, lda, a_scales, b, ldb, b_scales, M, N, K, true, q, p, maps))) return r;
  p.bias = bias;
  p.codes = codes;
  p.scales = scales;
  p.H = H;
  if (!q.bt) {
    const uint64_t dims[2] = {(uint64_t)H, (uint64_t)M}, stride[1] = {(uint64_t)H};
    const uint32_t box[2] = {32, 32};
    if ((r = rc::encode_tmap(&maps.out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, codes, dims, stride, box,
                             CU_TENSOR_MAP_SWIZZLE_NONE, what)))
      return r;
  }
  return run<EPI_SWIGLU, __nv_bfloat16>(maps, p, q, stream, what);
}

}  // extern "C"
