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
// accumulator row per thread.
#include "fp8_block.cuh"
#include "sm100.cuh"

namespace {

enum Epi : int { EPI_OUT = 0, EPI_SWIGLU = 1 };

constexpr int BM = 128;
constexpr int kRowBytes = 128;        // K elements (bytes) per k-tile: one scale block
constexpr int kSfAtom = 512;          // 128 rows x 4 scale bytes
constexpr int kBox = 32 * 128;        // a warp's staging box: 32 rows x 64 16-bit columns

struct Params {
  int M, N, K;                 // N: rows of W
  int k_tiles, m_blocks, n_blocks, group_m;
  int katoms;                  // scale atoms along K
  const float* bias;           // [N], nullable
  int staged;                  // OUT: out (and residual) move by TMA
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
template <int BN>
constexpr int tile_threads() { return 64 + 32 * epi_warps<BN>(); }

template <int BN, int STAGES, int EPI, bool PAIR>
struct Smem {
  static constexpr int kA = BM * kRowBytes;
  static constexpr int kB = (PAIR ? BN / 2 : BN) * kRowBytes;    // a pair splits W's rows between its CTAs
  static constexpr int kSf = (1 + BN / 128) * kSfAtom;
  static constexpr int offA = 0;
  static constexpr int offB = offA + STAGES * kA;
  static constexpr int offOut = offB + STAGES * kB;
  static constexpr int kOut = EPI == EPI_OUT ? epi_warps<BN>() * kBox : 2 * 4 * 4 * 32 * 4;   // boxes | amax of parts
  static constexpr int offSf = offOut + kOut;
  static constexpr int offBar = offSf + STAGES * kSf;
  static constexpr int kBars = 2 * STAGES + 6 + 1 + epi_warps<BN>() + 2;
  static constexpr int kTotal = offBar + kBars * 8;
  static_assert(kTotal <= 232448, "shared memory");
};

template <typename Out>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (std::is_same<Out, __half>::value) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// silu(g) * u with the MUFU exp2 and reciprocal (relative error ~1e-6, far
// below the E4M3 rounding that follows).
__device__ __forceinline__ float swiglu(float g, float u) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(g * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return g * r * u;
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

__device__ __forceinline__ void tile_coords(const Params& p, int tile, int& mb, int& nb) {
  const int per_group = p.group_m * p.n_blocks;
  const int g = tile / per_group, r = tile - g * per_group;
  const int gm = min(p.group_m, p.m_blocks - g * p.group_m);
  mb = g * p.group_m + r % gm;
  nb = r / gm;
}

template <int BN, int STAGES, int EPI, bool PAIR, typename Out>
__global__ void __launch_bounds__(tile_threads<BN>(), 1)
tile_kernel(const __grid_constant__ Maps maps, const Params p) {
  using S = Smem<BN, STAGES, EPI, PAIR>;
  constexpr int kEpiWarps = epi_warps<BN>();
  constexpr int kAcc = BN == 128 ? 3 : 1;           // accumulators in TMEM
  constexpr int kSfaCols = 4, kSfbCols = 4 * (BN / 128), kSfCols = kSfaCols + kSfbCols;
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
      for (int tile = tile0; tile < tiles && ok; tile += step) {
        int mb, nb;
        tile_coords(p, tile, mb, nb);
        const int rb = PAIR ? mb * 2 + (int)rank : mb;                          // this CTA's 128-row block of A
        const int brow = PAIR ? nb * BN + (int)rank * (BN / 2) : nb * BN;       // and its first row of W
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
              for (int r = 0; r < BN / 128; ++r)
                sm100::tma_load_2d_pair(sf + (1 + r) * kSfAtom, &maps.sfb, bar, 0,
                                        (nb * (BN / 128) + r) * p.katoms * 4 + line);
            }
          } else {
            sm100::mbar_arrive_expect_tx(&full[stage], bytes);
            sm100::tma_load_2d(a, &maps.a, &full[stage], kt * kRowBytes, rb * BM);
            sm100::tma_load_2d(b, &maps.b, &full[stage], kt * kRowBytes, brow);
            if (atom) {
              sm100::tma_load_2d(sf, &maps.sfa, &full[stage], 0, rb * p.katoms * 4 + line);
              for (int r = 0; r < BN / 128; ++r)
                sm100::tma_load_2d(sf + (1 + r) * kSfAtom, &maps.sfb, &full[stage], 0,
                                   (nb * (BN / 128) + r) * p.katoms * 4 + line);
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
      for (int tile = tile0; tile < tiles && ok; tile += step, ++local) {
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
            for (int r = 0; r < 1 + BN / 128; ++r) {
              if constexpr (PAIR) sm100::tmem_cp_32x128b_warpx4_pair(sfa + 4 * r, sm100::desc_add(dsf, r * kSfAtom));
              else sm100::tmem_cp_32x128b_warpx4(sfa + 4 * r, sm100::desc_add(dsf, r * kSfAtom));
            }
          }
          const uint32_t idesc = sm100::idesc_mxf8(PAIR ? 2 * BM : BM, BN, 0) | ((kt & 3) << 4) | ((kt & 3) << 29);
          // Columns past K are zero in shared memory (TMA fills them), so a
          // ragged last k-tile may run whole MMAs.
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint64_t a = sm100::desc_add(da, 32 * j), b = sm100::desc_add(db, 32 * j);
            if constexpr (PAIR) sm100::mma_mxf8_ss_pair(d, a, b, idesc, sfa, sfb, (kt | j) != 0);
            else sm100::mma_mxf8_ss(d, a, b, idesc, sfa, sfb, (kt | j) != 0);
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
    int local = 0;
    uint32_t res_phase = 0;
    for (int tile = tile0; tile < tiles; tile += step, ++local) {
      int mb, nb;
      tile_coords(p, tile, mb, nb);
      const int rb = PAIR ? mb * 2 + (int)rank : mb;
      const int as = local % kAcc;
      const uint32_t parity = (uint32_t)((local / kAcc) & 1);
      const uint32_t tacc = tmem + as * BN + ((uint32_t)(quad * 32) << 16);
      const int row0 = rb * BM + quad * 32, row = row0 + lane;
      if constexpr (EPI == EPI_OUT) {
        const int col0 = nb * BN + part * 64;
        const bool inside = row0 < p.M && col0 < p.N;
        uint8_t* box = smem + S::offOut + w * kBox;
        const Out* res = static_cast<const Out*>(p.residual);
        Out* out = static_cast<Out*>(p.out);
        auto at = [&](int r, int c) { return box + sm100::sw128_offset(r, c >> 3) + (c & 7) * 2; };
        if (p.staged && inside && lane == 0) {
          sm100::bulk_wait_group_read0();      // the previous tile's store has read the box
          if (res) {
            sm100::mbar_arrive_expect_tx(&res_full[w], kBox);
            sm100::tma_load_2d(box, &maps.res, &res_full[w], col0, row0);
          }
        }
        if (!wait(&acc_full[as], parity, 4)) break;
        sm100::tc_fence_after();
        uint32_t acc[64];
        load_acc(tacc + part * 64, acc);
        acc_ready(acc);
        release(as);
        if (!inside) continue;
        if (res) {
          if (p.staged) {
            if (!wait(&res_full[w], res_phase, 5)) break;
            res_phase ^= 1;
          } else {
            for (int r = 0; r < 32 && row0 + r < p.M; ++r)
              for (int c = lane; c < 64 && col0 + c < p.N; c += 32)
                *reinterpret_cast<Out*>(at(r, c)) = rc::ld_in(res + (size_t)(row0 + r) * p.ldr + col0 + c);
            __syncwarp();
          }
        }
#pragma unroll
        for (int g = 0; g < 8; ++g) {
          const int n = col0 + 8 * g;
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(acc[8 * g + j]);
          if (p.bias) {
            if (n + 8 <= p.N) {
              float b[8];
              fp8b::load8(p.bias + n, b);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] += b[j];
            } else {
#pragma unroll
              for (int j = 0; j < 8; ++j)
                if (n + j < p.N) v[j] += rc::ld_in(p.bias + n + j);
            }
          }
          uint4* q = reinterpret_cast<uint4*>(at(lane, 8 * g));
          if (res) {
            const uint4 r4 = *q;
            const uint32_t rw[4] = {r4.x, r4.y, r4.z, r4.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float2 f = unpack2<Out>(rw[j]);
              v[2 * j] += f.x;
              v[2 * j + 1] += f.y;
            }
          }
          Out* tag = nullptr;
          *q = make_uint4(fp8b::pack2(v[0], v[1], tag), fp8b::pack2(v[2], v[3], tag), fp8b::pack2(v[4], v[5], tag),
                          fp8b::pack2(v[6], v[7], tag));
        }
        if (p.staged) {
          sm100::fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            sm100::tma_store_2d(&maps.out, box, col0, row0);
            sm100::bulk_commit_group();
          }
        } else {
          __syncwarp();
          for (int r = 0; r < 32 && row0 + r < p.M; ++r)
            for (int c = lane; c < 64 && col0 + c < p.N; c += 32)
              out[(size_t)(row0 + r) * p.ldo + col0 + c] = *reinterpret_cast<const Out*>(at(r, c));
          __syncwarp();                        // the box is free again
        }
      } else {
        uint32_t* s_amax = reinterpret_cast<uint32_t*>(smem + S::offOut) + ((local & 1) * 4 + quad) * 4 * 32;
        const bool ok = wait(&acc_full[as], parity, 4);
        uint32_t acc[64];                      // 32 gate, then the 32 up columns they pair with
        uint32_t m = 0;
        float y[32];
        if (ok) {
          sm100::tc_fence_after();
          sm100::tmem_ld32(tacc + part * 32, acc);
          sm100::tmem_ld32(tacc + 128 + part * 32, acc + 32);
          acc_ready(acc);
          release(as);
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            float bg[8] = {}, bu[8] = {};
            const int n = nb * BN + part * 32 + 8 * g;
            if (p.bias) {
              fp8b::load8(p.bias + n, bg);
              fp8b::load8(p.bias + n + 128, bu);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float v = swiglu(__uint_as_float(acc[8 * g + j]) + bg[j], __uint_as_float(acc[32 + 8 * g + j]) + bu[j]);
              y[8 * g + j] = nb * 128 + part * 32 + (8 * g & ~15) < p.H ? v : 0.0f;
              m = max(m, fp8b::magnitude(y[8 * g + j]));
            }
          }
          s_amax[part * 32 + lane] = m;
        }
        // The four warps of a lane quadrant share its rows' amax. (The buffer
        // of tile k is written again at tile k + 2, after the barrier of k + 1.)
        if (!sm100::bar_and(1 + quad, 128, ok)) break;
        m = max(max(s_amax[lane], s_amax[32 + lane]), max(s_amax[64 + lane], s_amax[96 + lane]));
        const uint32_t e = fp8b::scale_byte(m);
        const float inv = fp8b::inverse_scale(e);
        const int col0 = nb * 128 + part * 32;
        if (row < p.M) {
          uint32_t c[8];
#pragma unroll
          for (int j = 0; j < 8; ++j)
            c[j] = fp8b::e4m3x4(y[4 * j] * inv, y[4 * j + 1] * inv, y[4 * j + 2] * inv, y[4 * j + 3] * inv);
          uint4* dst = reinterpret_cast<uint4*>(p.codes + (size_t)row * p.H + col0);
          if (col0 < p.H) dst[0] = make_uint4(c[0], c[1], c[2], c[3]);
          if (col0 + 16 < p.H) dst[1] = make_uint4(c[4], c[5], c[6], c[7]);
        }
        if (part == 0 && row < (p.M + 127) / 128 * 128) {
          const int atoms = fp8b::atoms_of(p.H);
          p.scales[rc::sf_offset(row, nb, atoms)] = row < p.M ? (uint8_t)e : 0;
          if (nb == p.n_blocks - 1)
            for (int kb = p.n_blocks; kb < 4 * atoms; ++kb) p.scales[rc::sf_offset(row, kb, atoms)] = 0;
        }
      }
    }
    if (EPI == EPI_OUT && lane == 0) sm100::bulk_wait_group0();
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

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Checks and tensor maps the two products share. rows of W: N; its first
// 128-row block's scales start at sb.
int prepare(const char* what, const void* a, long long lda, const void* sa, const void* b, long long ldb,
            const void* sb, int M, int N, int K, int bn, bool pair, Params& p, Maps& maps) {
  p.M = M;
  p.N = N;
  p.K = K;
  p.k_tiles = fp8b::blocks_of(K);
  p.katoms = fp8b::atoms_of(K);
  p.m_blocks = (M + (pair ? 2 * BM : BM) - 1) / (pair ? 2 * BM : BM);
  p.n_blocks = (N + bn - 1) / bn;
  p.group_m = p.m_blocks;
  const long long lines_a = 4LL * p.katoms * ((M + 127) / 128), lines_b = 4LL * p.katoms * ((N + 127) / 128);
  if ((long long)p.m_blocks * p.n_blocks > INT32_MAX || lines_a > INT32_MAX || lines_b > INT32_MAX)
    return rc::set_error(RC_ERR_UNSUPPORTED, "%s: %d x %d x %d is too large", what, M, N, K);
  const uint32_t box[2] = {kRowBytes, BM}, box_b[2] = {kRowBytes, (uint32_t)(pair ? bn / 2 : bn)}, box_s[2] = {128, 4};
  const uint64_t da[2] = {(uint64_t)K, (uint64_t)M}, db[2] = {(uint64_t)K, (uint64_t)N};
  const uint64_t sta[1] = {(uint64_t)lda}, stb[1] = {(uint64_t)ldb}, sts[1] = {128};
  const uint64_t dsa[2] = {128, (uint64_t)lines_a}, dsb[2] = {128, (uint64_t)lines_b};
  const auto u8 = CU_TENSOR_MAP_DATA_TYPE_UINT8;
  int r;
  if ((r = rc::encode_tmap(&maps.a, u8, 2, const_cast<void*>(a), da, sta, box, CU_TENSOR_MAP_SWIZZLE_128B, what)))
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

template <typename Out>
int run_out(const Maps& maps, const Params& p, bool wide, cudaStream_t stream, const char* what) {
  if (wide) return launch<256, 3, EPI_OUT, false, Out>(maps, p, stream, what);
  return launch<128, 5, EPI_OUT, false, Out>(maps, p, stream, what);
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
  const bool wide = false;
  Params p{};
  Maps maps;
  if ((r = prepare(what, a, lda, a_scales, b, ldb, b_scales, M, N, K, wide ? 256 : 128, false, p, maps))) return r;
  p.bias = bias;
  p.out = out;
  p.ldo = ldo;
  p.residual = residual;
  p.ldr = ldr;
  // TMA moves the output (and the residual) where rows start on 16 bytes.
  p.staged = aligned16(out) && ldo % 8 == 0 && aligned16(residual) && (!residual || ldr % 8 == 0);
  if (p.staged) {
    const auto type = out_dtype == fp8b::kBF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    const uint64_t dims[2] = {(uint64_t)N, (uint64_t)M};
    const uint32_t box[2] = {64, 32};
    const uint64_t so[1] = {(uint64_t)ldo * 2}, sr[1] = {(uint64_t)ldr * 2};
    if ((r = rc::encode_tmap(&maps.out, type, 2, out, dims, so, box, CU_TENSOR_MAP_SWIZZLE_128B, what))) return r;
    if (residual && (r = rc::encode_tmap(&maps.res, type, 2, const_cast<void*>(residual), dims, sr, box,
                                         CU_TENSOR_MAP_SWIZZLE_128B, what)))
      return r;
  }
  if (out_dtype == fp8b::kBF16) return run_out<__nv_bfloat16>(maps, p, wide, stream, what);
  return run_out<__half>(maps, p, wide, stream, what);
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
  Params p{};
  Maps maps;
  if ((r = prepare(what, a, lda, a_scales, b, ldb, b_scales, M, N, K, 256, false, p, maps))) return r;
  p.bias = bias;
  p.codes = codes;
  p.scales = scales;
  p.H = H;
  return launch<256, 4, EPI_SWIGLU, false, __nv_bfloat16>(maps, p, stream, what);
}

}  // extern "C"
