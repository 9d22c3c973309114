// Product of two e4m3 matrices with a scale per group of 128 along the reduction (tcgen05 kind::f8f6f4, sm_100a):
//
//   C[m, n] = sum over blocks kb of 128:  sa[m, kb] * sb[n, kb] * (sum over k in kb of qa[m, k] * qb[n, k])
//
// The inner sums are exact products accumulated in fp32 in TMEM; scales differ from block to block, so an accumulator
// holds ONE block (four instructions of 128 or 256 x N x 32) and is then added, times its scales, to fp32 registers of
// the warps that later write the tile.  Two accumulators take turns: while the tensor core fills one, eight warps take
// up the other.  A lane holds a row of C: with sb per 128 columns (weights) both scales are one number per thread and
// block, and the whole addition is one packed multiply-add for two elements.  With a scale per row of B too (BROWS: weight
// gradients) the columns' scales go through shared memory.
//
// Both operands are K-major with 128-byte swizzle: a block of 128 is one swizzle row.  CG = 2: CTA pairs
// (cta_group::2), 256 x 256 tiles of which each CTA stages 128 rows of either operand, 32 KB per block where a CTA
// alone stages 48 for a tile of 128 x 256.
//
// Rows come as they are (`tile_expert` null: B matrices of M rows) or sorted by expert in the padded layout of the
// expert pass, an expert's tiles following each other with the row tile varying fastest.
//
// Every wait is bounded as in umma_gemm.cuh.  A warp whose wait gave up walks on through the remaining tiles without
// waiting, computing or storing, so that the named barriers of the epilogues are met by all that expect each other.
#pragma once
#include <algorithm>

#include "epilogues.cuh"
#include "fp8_quant.cuh"
#include "tcgen05.cuh"

namespace yb {

// Three warpgroups: the first issues copies (warp 0) and instructions (warp 1), the others hold 128 fp32 sums per thread.
// Registers go where they are needed: 384 threads start with 168 each, which is 40 + 2 x 232 for the three groups.
constexpr int kFp8EpiWarps = 8, kFp8FirstEpiWarp = 4;
constexpr int kFp8Threads = 32 * (kFp8FirstEpiWarp + kFp8EpiWarps);
constexpr int kFp8FewRegs = 40, kFp8ManyRegs = 232;

struct Fp8Params {
  int64_t M, N;                 // rows per matrix (not grouped), columns
  int K, B;                     // reduction length, matrices
  int MT, NT;                   // tiles of 128 * CG rows (not grouped), of BN columns
  const float* sa;              // scale of (matrix b, row m, block kb) at b * sa_b + m * sa_m + kb * sa_k
  const float* sb;              // of (matrix b, row or 128-row block n, block kb)
  int64_t sa_b, sa_m, sa_k, sb_b, sb_n, sb_k;
  // grouped
  const int32_t* tile_expert;   // expert of every tile of 128 * CG rows
  const int32_t* tile_first;    // [E + 1] prefix sums of those tiles; null: pad_off / 128
  const int32_t* pad_off;       // [E + 1]
  const int32_t* n_tiles;       // how many there are
  int32_t* status;              // device status word
  int clear_status;             // no earlier kernel of the call has set it to 0
};

template <int CG, int BN>
struct Fp8Smem {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = BN / CG * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  static constexpr int kStages = 196608 / kStageBytes;     // 4 (one CTA, 256 columns) or 6
  static constexpr int kTables = kStages * kStageBytes + 1024;
};
inline int fp8_smem_bytes(int tables, int experts) { return tables + (experts > 0 ? 2 * (experts + 1) * 4 : 0); }

template <int CG>
__device__ __forceinline__ void tc_mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if constexpr (CG == 1)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
__device__ __forceinline__ uint64_t pack_f32x2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void unpack_f32x2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma_f32x2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t mul_f32x2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// What an epilogue gets: the thread's row and the COLS columns from n0 on whose sums it holds (columns in pairs).
struct Fp8Tile {
  int b;               // matrix or expert
  int64_t row;         // row of the matrix, or padded row of the expert pass
  int64_t row_end;     // rows from here on are another's
  int n0, n_end;       // n_end: columns of the matrix
  int q, half, lane;   // lane quarter and column half of the warp
  bool ok;             // false: take part in barriers only
};

template <int CG, int BN, bool BROWS, bool GROUPED, class Epi>
__global__ void __launch_bounds__(kFp8Threads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const Fp8Params p,
                const Epi epi) {
  using SM = Fp8Smem<CG, BN>;
  constexpr int kStages = SM::kStages, kCols = BN / 2, kChunks = kCols / 32;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kStages];       // CG = 2: used in the leader CTA
  __shared__ __align__(8) uint64_t bar_empty[kStages];      // per CTA
  __shared__ __align__(8) uint64_t bar_tmem_full[2];        // per CTA
  __shared__ __align__(8) uint64_t bar_tmem_empty[2];       // CG = 2: used in the leader CTA
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ __align__(16) float s_sb[BROWS ? 2 : 1][BROWS ? BN : 1];
  __shared__ typename Epi::Shared s_epi;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 2 ? cluster_ctarank() : 0;
  const bool leader = rank == 0;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  int32_t* s_first = reinterpret_cast<int32_t*>(smem_raw + SM::kTables);   // grouped: first tile of each expert
  int32_t* s_pad = s_first + p.B + 1;                                      // first padded row of each expert

  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), CG);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bar_tmem_full[a]), 1);
      mbar_init(smem_u32(&bar_tmem_empty[a]), CG * kFp8EpiWarps);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                   ::"r"(smem_u32(&tmem_base_slot)), "r"(2u * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                   ::"r"(smem_u32(&tmem_base_slot)), "r"(2u * BN) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync_all();     // the peer's barriers exist before any remote signal is sent
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  pdl_trigger();
  pdl_wait();
  if constexpr (GROUPED) {
    for (int i = threadIdx.x; i <= p.B; i += kFp8Threads) {
      s_pad[i] = p.pad_off[i];
      s_first[i] = p.tile_first != nullptr ? p.tile_first[i] : p.pad_off[i] / kTileM;
    }
    __syncthreads();
  }
  if (p.clear_status && blockIdx.x == 0 && threadIdx.x == 0) *p.status = kStatusOk;   // waits give up after seconds at the earliest
  const int64_t total = GROUPED ? (int64_t)*after_wait(p.n_tiles) * p.NT : (int64_t)p.B * p.MT * p.NT;
  const int64_t first_id = blockIdx.x / CG, n_workers = gridDim.x / CG;
  const int kblocks = (p.K + kFp8Group - 1) / kFp8Group;

  // work item -> matrix or expert, first row of the tile, first column
  auto decode = [&](int64_t id, int& b, int64_t& m0, int& n0) {
    if constexpr (GROUPED) {
      const int tile = (int)(id / p.NT);
      int lo = 0, hi = p.B;                      // the last expert whose first tile is not behind this one
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_first[mid] <= tile) lo = mid; else hi = mid;
      }
      b = lo;
      const int cnt = s_first[b + 1] - s_first[b];
      const int local = (int)(id - (int64_t)s_first[b] * p.NT);
      const int nt = local / cnt;
      m0 = s_pad[b] + (int64_t)(local - nt * cnt) * (kTileM * CG);
      n0 = nt * BN;
    } else {
      const int64_t per = (int64_t)p.MT * p.NT;
      b = (int)(id / per);
      const int64_t local = id - b * per;
      const int nt = (int)(local / p.MT);
      m0 = (local - (int64_t)nt * p.MT) * (kTileM * CG);
      n0 = nt * BN;
    }
  };

  if (warp < kFp8FirstEpiWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp8FewRegs));
    if (warp == 0) {
      // =========================== TMA producer (of each CTA) ==================================
      const bool elected = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t id = first_id; id < total && ok; id += n_workers) {
        int b, n0;
        int64_t m0;
        decode(id, b, m0, n0);
        const int width = min(BN, ((int)p.N - n0 + 15) & ~15);
        const int am = (int)m0 + (int)rank * 128, bn = n0 + (int)rank * (width / CG);
        for (int kb = 0; kb < kblocks; ++kb) {
          ok = mbar_wait_warp(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag);
          if (!ok) break;
          if (elected) {
            const uint32_t sa = smem_base + stage * SM::kStageBytes;
            if constexpr (CG == 1) {
              const uint32_t full = smem_u32(&bar_full[stage]);
              mbar_expect_tx(full, SM::kStageBytes);
              tma_load_3d(sa, &tmA, kb * kFp8Group, am, GROUPED ? 0 : b, full);
              tma_load_3d(sa + SM::kABytes, &tmB, kb * kFp8Group, bn, b, full);
            } else {
              const uint32_t full = mapa_u32(smem_u32(&bar_full[stage]), 0);
              mbar_expect_tx_cluster(full, SM::kStageBytes);
              tma2_load_3d(sa, &tmA, kb * kFp8Group, am, GROUPED ? 0 : b, full);
              tma2_load_3d(sa + SM::kABytes, &tmB, kb * kFp8Group, bn, b, full);
            }
          }
          __syncwarp();
          if (++stage == kStages) { stage = 0; phase ^= 1u; }
        }
      }
      // the commits that free the last stages must have arrived here before this CTA ends
      for (int s = 0; s < kStages && ok; ++s)
        ok = mbar_wait_warp(smem_u32(&bar_empty[s]), s < stage ? phase : phase ^ 1u, &abort_flag);
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicMax(p.status, (int)kStatusProducerTimeout);
      }
      __syncwarp();
    } else if (warp == 1) {
      // =========================== MMA issuer (of the leader) ==================================
      if (leader) {
        const uint32_t idesc_base = (1u << 4) | ((uint32_t)(128 * CG >> 4) << 24);   // e4m3 x e4m3 -> fp32, both K-major
        const uint64_t adesc0 = make_smem_desc(smem_base, 16, 1024);
        const uint64_t bdesc0 = make_smem_desc(smem_base + SM::kABytes, 16, 1024);
        const bool elected = elect_one();
        int stage = 0, acc = 0;
        uint32_t phase = 0, acc_phase = 0;
        bool ok = true;
        for (int64_t id = first_id; id < total && ok; id += n_workers) {
          int b, n0;
          int64_t m0;
          decode(id, b, m0, n0);
          const uint32_t width = min(BN, ((int)p.N - n0 + 15) & ~15);
          const uint32_t idesc = idesc_base | ((width >> 3) << 17);
          for (int kb = 0; kb < kblocks; ++kb) {
            ok = mbar_wait_warp(smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, &abort_flag);
            if (ok) ok = mbar_wait_warp(smem_u32(&bar_full[stage]), phase, &abort_flag);
            if (!ok) break;
            tc_fence_after();
            if (elected) {
              const uint64_t adesc = adesc0 + (uint64_t)(stage * (SM::kStageBytes >> 4));
              const uint64_t bdesc = bdesc0 + (uint64_t)(stage * (SM::kStageBytes >> 4));
  #pragma unroll
              for (int k = 0; k < kFp8Group / 32; ++k)
                tc_mma_fp8<CG>(tmem_base + acc * BN, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc, (uint32_t)(k != 0));
              if constexpr (CG == 1) {
                tc_commit(smem_u32(&bar_empty[stage]));
                tc_commit(smem_u32(&bar_tmem_full[acc]));
              } else {
                tc2_commit_pair(smem_u32(&bar_empty[stage]));
                tc2_commit_pair(smem_u32(&bar_tmem_full[acc]));
              }
            }
            __syncwarp();
            if (++stage == kStages) { stage = 0; phase ^= 1u; }
            acc ^= 1;
            if (acc == 0) acc_phase ^= 1u;
          }
        }
        if (!ok && lane == 0) {
          abort_flag = 1;
          atomicMax(p.status, (int)kStatusMmaTimeout);
        }
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp8ManyRegs));
    // =========================== scaled sums and epilogue (warps 4 .. 11 of each CTA) ========
    const int q = warp & 3;                      // TMEM lane quarter this warp may read
    const int half = (warp - kFp8FirstEpiWarp) >> 2;            // its columns: kCols from half * kCols on
    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + half * kCols;
    int acc = 0;
    uint32_t acc_phase = 0, parity = 0;
    bool ok = true;
    for (int64_t id = first_id; id < total; id += n_workers, parity ^= 1u) {
      Fp8Tile t;
      int n0;
      int64_t m0;
      decode(id, t.b, m0, n0);
      t.row = m0 + rank * 128 + q * 32 + lane;
      t.row_end = GROUPED ? (int64_t)s_pad[t.b + 1] : p.M;
      t.n0 = n0 + half * kCols;
      t.n_end = (int)p.N;
      t.q = q; t.half = half; t.lane = lane;
      const int width = min(BN, ((int)p.N - n0 + 15) & ~15) - half * kCols;    // columns computed; may be <= 0
      const bool row_ok = t.row < t.row_end;
      const auto pre = epi.begin(t, row_ok);
      const float* sa = p.sa + (GROUPED ? 0 : t.b * p.sa_b) + (row_ok ? t.row : 0) * p.sa_m;
      const float* sb;
      const bool col_mine = BROWS && t.n0 + q * 32 + lane < p.N && (kCols == 128 || q * 32 < kCols);
      if constexpr (BROWS) sb = p.sb + t.b * p.sb_b + (col_mine ? (int64_t)(t.n0 + q * 32 + lane) : 0) * p.sb_n;
      else sb = p.sb + t.b * p.sb_b + (int64_t)(min(t.n0, (int)p.N - 1) / kFp8Group) * p.sb_n;
      float sa_next = *sa, sb_next = *sb;
      uint64_t sum[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) sum[i] = 0;
      for (int kb = 0; kb < kblocks; ++kb) {
        const float sa_now = sa_next, sb_now = sb_next;
        if (kb + 1 < kblocks) {
          sa_next = sa[(kb + 1) * p.sa_k];
          sb_next = sb[(kb + 1) * p.sb_k];
        }
        if constexpr (BROWS) {
          // the columns' scales of this half; of the other buffer the warps of this half are done once they meet here
          if (kCols == 128 || q * 32 < kCols) s_sb[acc][half * kCols + q * 32 + lane] = col_mine ? sb_now : 0.f;
          named_sync(1 + half, 128);
        }
        if (ok) ok = mbar_wait_warp(smem_u32(&bar_tmem_full[acc]), acc_phase, &abort_flag);
        if (ok) {
          tc_fence_after();
          const uint64_t s2 = BROWS ? pack_f32x2(sa_now, sa_now) : pack_f32x2(sa_now * sb_now, sa_now * sb_now);
          // 32 columns at a time, the next ones on their way while these are added
          uint32_t r[2][32];
          if (width > 0) {
            tc_ld_32x32_issue(t_row + acc * BN, r[0]);
#pragma unroll
            for (int c = 0; c < kChunks; ++c) {
              if (c * 32 < width) {
                tc_ld_wait(r[c & 1]);
                if (c + 1 < kChunks && (c + 1) * 32 < width) tc_ld_32x32_issue(t_row + acc * BN + (c + 1) * 32, r[(c + 1) & 1]);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                  const uint64_t v = pack_f32x2(__uint_as_float(r[c & 1][2 * i]), __uint_as_float(r[c & 1][2 * i + 1]));
                  if constexpr (BROWS) {
                    const float2 s = *reinterpret_cast<const float2*>(&s_sb[acc][half * kCols + c * 32 + 2 * i]);
                    sum[c * 16 + i] = fma_f32x2(v, mul_f32x2(s2, pack_f32x2(s.x, s.y)), sum[c * 16 + i]);
                  } else {
                    sum[c * 16 + i] = fma_f32x2(v, s2, sum[c * 16 + i]);
                  }
                }
              }
            }
          }
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if constexpr (CG == 1) mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
            else mbar_arrive_cluster(mapa_u32(smem_u32(&bar_tmem_empty[acc]), 0));
          }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      t.ok = ok;
      epi.template finish<kCols>(t, row_ok, pre, sum, s_epi, parity);
    }
    if (!ok) {
      abort_flag = 1;
      atomicMax(p.status, (int)kStatusEpilogueTimeout);
    }
  }

  // ---- teardown ---------------------------------------------------------------------------
  tc_fence_before();
  __syncthreads();
  if (abort_flag != 0) {
    // give copies that may still be in flight time to land before the shared memory is released
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 2000000ull) __nanosleep(1000);
    __syncthreads();
  }
  if constexpr (CG == 2) cluster_sync_all();     // neither CTA releases what the pair may still use
  if (warp == 1) {
    tc_fence_after();
    if constexpr (CG == 1)
      asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * BN) : "memory");
    else
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(2u * BN) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------
// Epilogues
// ---------------------------------------------------------------------------------------------

// C[b, m, n] rounded to T
template <typename T>
struct Fp8Store {
  struct Shared {};
  struct Pre {};
  T* C;
  int64_t ld, batch;
  int vec;                 // rows start on 16-byte boundaries

  __device__ __forceinline__ Pre begin(const Fp8Tile&, bool) const { return {}; }
  template <int COLS>
  __device__ __forceinline__ void finish(const Fp8Tile& t, bool row_ok, const Pre&, const uint64_t (&sum)[COLS / 2], Shared&,
                                         uint32_t) const {
    if (!t.ok || !row_ok) return;
    T* c = C + t.b * batch + t.row * ld + t.n0;
    constexpr int VE = 16 / (int)sizeof(T);
    const int cols = t.n_end - t.n0;
#pragma unroll
    for (int i = 0; i < COLS; i += VE) {
      float v[VE];
#pragma unroll
      for (int j = 0; j < VE; j += 2) unpack_f32x2(sum[(i + j) / 2], v[j], v[j + 1]);
      if (vec && i + VE <= cols) {
        if constexpr (sizeof(T) == 2)
          *reinterpret_cast<uint4*>(c + i) = make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                                                        pack_bf16x2(v[6], v[7]));
        else
          *reinterpret_cast<float4*>(c + i) = make_float4(v[0], v[1], v[2], v[3]);
      } else {
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (i + j < cols) DT<T>::st(c + i + j, v[j]);
      }
    }
  }
};

// gate_up of the expert pass: + bias, clamped SwiGLU of the interleaved (gate, up) columns, quantised in groups of 128
// activations.  A tile of 256 columns holds one group of each of its rows, half of it in either of two warps, which
// tell each other their largest magnitudes.
template <typename T>
struct Fp8GluQuant {
  struct Shared { uint32_t most[2][2][128]; };
  struct Pre {};
  const T* bias;           // [E, 2H]
  uint8_t* act;            // [rows, ld]
  float* scale;            // (row, group) at group * scale_group + row
  int64_t ld, scale_group;

  __device__ __forceinline__ Pre begin(const Fp8Tile&, bool) const { return {}; }
  template <int COLS>
  __device__ __forceinline__ void finish(const Fp8Tile& t, bool row_ok, const Pre&, const uint64_t (&sum)[COLS / 2], Shared& s,
                                         uint32_t parity) const {
    static_assert(COLS == 128, "a group of 128 activations is a tile of 256 columns");
    float a[COLS / 2];
    uint32_t most = 0;
    const T* bs = bias + (int64_t)t.b * t.n_end + t.n0;
#pragma unroll
    for (int i = 0; i < COLS / 2; ++i) {
      float g, u;
      unpack_f32x2(sum[i], g, u);
      a[i] = 0.f;
      if (t.n0 + 2 * i < t.n_end) a[i] = glu_act(g + DT<T>::ld(bs + 2 * i), u + DT<T>::ld(bs + 2 * i + 1));
      most = max(most, abs_bits(a[i]));
    }
    const int r = t.q * 32 + t.lane;
    s.most[parity][t.half][r] = most;
    named_sync(4 + t.q, 64);
    if (!t.ok || !row_ok || t.n0 >= t.n_end) return;
    const float top = fp8_group_max(max(most, s.most[parity][t.half ^ 1][r])), inv = fp8_inverse(top);
    const int64_t col = t.n0 / 2;
    uint8_t* dst = act + t.row * ld + col;
#pragma unroll
    for (int i = 0; i < COLS / 2; i += 16)
      if (col + i < ld) {
        uint4 c;
        c.x = e4m3x4(a[i] * inv, a[i + 1] * inv, a[i + 2] * inv, a[i + 3] * inv);
        c.y = e4m3x4(a[i + 4] * inv, a[i + 5] * inv, a[i + 6] * inv, a[i + 7] * inv);
        c.z = e4m3x4(a[i + 8] * inv, a[i + 9] * inv, a[i + 10] * inv, a[i + 11] * inv);
        c.w = e4m3x4(a[i + 12] * inv, a[i + 13] * inv, a[i + 14] * inv, a[i + 15] * inv);
        *reinterpret_cast<uint4*>(dst + i) = c;
      }
    if (t.half == 0) scale[(t.n0 / (2 * kFp8Group)) * scale_group + t.row] = fp8_scale(top);
  }
};

// down of the expert pass: y = w_row * (v + bias) in fp32 at the flat position of the row, or (fp32 calls) at the padded row
// itself, as combine_padded_kernel wants the K rows of a token that it sums.  Padding rows have no position and no weight.
template <typename T>
struct Fp8WeightedRows {
  static constexpr bool kFlat = sizeof(T) != sizeof(float);
  struct Shared {};
  struct Pre { float w; int64_t at; };
  const T* bias;           // [E, N]
  float* y;                // [S, N] or [rows, N]
  const int32_t* row_token;
  const int32_t* row_flat;
  const float* row_weight;
  int64_t N;

  __device__ __forceinline__ Pre begin(const Fp8Tile& t, bool row_ok) const {
    Pre p{0.f, -1};
    if (row_ok && row_token[t.row] >= 0) {
      p.at = kFlat ? (int64_t)row_flat[t.row] : t.row;
      p.w = row_weight[t.row];
    }
    return p;
  }
  template <int COLS>
  __device__ __forceinline__ void finish(const Fp8Tile& t, bool, const Pre& p, const uint64_t (&sum)[COLS / 2], Shared&,
                                         uint32_t) const {
    if (!t.ok || p.at < 0) return;
    float* dst = y + p.at * N + t.n0;
    const T* bs = bias + t.b * N + t.n0;
    const int cols = t.n_end - t.n0;                   // a multiple of 8
#pragma unroll
    for (int i = 0; i < COLS; i += 4)
      if (i < cols) {
        float v[4];
        unpack_f32x2(sum[i / 2], v[0], v[1]);
        unpack_f32x2(sum[i / 2 + 1], v[2], v[3]);
        *reinterpret_cast<float4*>(dst + i) = make_float4(p.w * (v[0] + DT<T>::ld(bs + i)), p.w * (v[1] + DT<T>::ld(bs + i + 1)),
                                                          p.w * (v[2] + DT<T>::ld(bs + i + 2)), p.w * (v[3] + DT<T>::ld(bs + i + 3)));
      }
  }
};

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// CTAs (CG = 1) or CTA pairs that run at the same time, asked once per kernel and device
template <int CG, typename... KArgs>
inline int fp8_resident(void (*kern)(KArgs...), PerDevice<int>& known) {
  const int dev = current_device_index();
  int n = known.get(dev);
  if (n > 0) return n;
  constexpr int kMost = 227 * 1024 - 8192;     // static shared memory beside it
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost) != cudaSuccess) return 0;
  if (CG == 1) {
    n = umma_sm_count();
  } else {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(umma_sm_count() & ~1);
    cfg.blockDim = dim3(kFp8Threads);
    cfg.dynamicSmemBytes = kMost;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = CG;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
      (void)cudaGetLastError();
      n = umma_sm_count() / CG;
    }
  }
  known.set(dev, n);
  return n;
}

struct Fp8Operand {
  const void* q;
  int64_t rows, ld, batch;      // rows per matrix, pitch, distance of matrices (bytes)
};

// `max_tiles`: row tiles of 128 * CG rows in all
template <int CG, int BN, bool BROWS, bool GROUPED, class Epi>
inline int launch_fp8_gemm(const Fp8Operand& a, const Fp8Operand& b, Fp8Params p, const Epi& epi, int64_t max_tiles, bool pdl,
                           cudaStream_t st) {
  if (!umma_available()) return YAMOE_ERR_UNSUPPORTED;
  using SM = Fp8Smem<CG, BN>;
  CUtensorMap tmA, tmB;
  const uint64_t na = GROUPED ? 1 : (uint64_t)p.B;
  const uint64_t da[3] = {(uint64_t)p.K, (uint64_t)a.rows, na}, db[3] = {(uint64_t)p.K, (uint64_t)b.rows, (uint64_t)p.B};
  const uint64_t ga[2] = {(uint64_t)a.ld, (uint64_t)(na > 1 ? a.batch : a.ld)};
  const uint64_t gb[2] = {(uint64_t)b.ld, (uint64_t)(p.B > 1 ? b.batch : b.ld)};
  const uint32_t boxa[3] = {128, 128, 1}, boxb[3] = {128, BN / CG, 1};
  if (!encode_map(&tmA, a.q, 3, da, ga, boxa, kMapU8) || !encode_map(&tmB, b.q, 3, db, gb, boxb, kMapU8)) return YAMOE_ERR_CUDA;
  auto kern = fp8_gemm_kernel<CG, BN, BROWS, GROUPED, Epi>;
  static PerDevice<int> resident;    // per template instantiation and device
  const int workers = fp8_resident<CG>(kern, resident);
  if (workers <= 0) return YAMOE_ERR_CUDA;
  p.NT = (int)ceil_div(p.N, BN);
  const int64_t total = max_tiles * p.NT;
  if (total <= 0) return YAMOE_OK;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * std::min<int64_t>(total, workers)));
  cfg.blockDim = dim3(kFp8Threads);
  cfg.dynamicSmemBytes = (size_t)fp8_smem_bytes(SM::kTables, GROUPED ? p.B : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled(pdl) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, tmA, tmB, p, epi) != cudaSuccess) return YAMOE_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

}  // namespace yb
