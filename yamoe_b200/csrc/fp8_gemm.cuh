// Product of two e4m3 matrices with a scale per group of 128 along the reduction (tcgen05 kind::f8f6f4, sm_100a):
//
//   C[m, n] = sum over blocks kb of 128:  sa[m, kb] * sb[n, kb] * (sum over k in kb of qa[m, k] * qb[n, k])
//
// The inner sums are exact products accumulated in fp32 in TMEM; scales differ from block to block, so an accumulator
// holds ONE block (four instructions of 128 x 256 x 32) and is then added, times its scales, to fp32 registers of
// the warps that later write the tile.  A lane holds a row of C: with sb per 128 columns (weights) both scales are one
// number per thread and accumulator, and the whole addition is one packed multiply-add for two elements.  With a scale per
// row of B too (BROWS: weight gradients) the columns' scales go through shared memory.
//
// What bounds it, in clocks per block of a 128 x 256 tile (8192 x 5760 x 2880; its four instructions need 512): the
// instructions alone 623, with the copies of their operands (48 KB) 735, with the additions 930, of which a third is
// waiting for loads from TMEM; a tile's end and beginning take another 90.  So an accumulator has the whole width of the
// tile (one wait and one arrival per block and warp), a load of 32 columns is always on its way while those before it are
// added, across blocks too (64 columns at a time, refilled half by half, took 5 % longer), the scales are brought to
// shared memory by a warp of their own, four blocks at a time, and a tile leaves by TMA while the next one is begun.
// That size takes 167 us among calls like it, 1.63 PFLOP/s at the 1560 MHz that the power cap leaves (170 alone); a bf16 product of
// that size by cuBLAS 209 us at 1400 MHz (196 to 269 alone).
//
// Both operands are K-major with 128-byte swizzle: a block of 128 is one swizzle row.  A CTA has tiles of 128 x 256 (CTA pairs
// with tiles of 256 x 256 were no faster, 150.5 and 151.2 us at that size when additions and stores took longer, and tiles
// of 256 rows fit experts' rows less well).  Few tiles: 128 x 128, and a cluster of up to four CTAs shares a tile's blocks
// (split); each CTA ends with a share of the columns, to whose sums the others send theirs, added in order.
//
// Rows come as they are (B matrices of M rows) or (GROUPED) sorted by expert in the padded layout of the
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

// Three warpgroups: the first issues copies (warp 0), instructions (warp 1) and fetches scales (warp 2), the others hold 128 fp32
// sums per thread.
// Registers go where they are needed: 384 threads start with 168 each, which is 40 + 2 x 232 for the three groups.
constexpr int kFp8EpiWarps = 8, kFp8FirstEpiWarp = 4;
constexpr int kFp8Threads = 32 * (kFp8FirstEpiWarp + kFp8EpiWarps);
constexpr int kFp8FewRegs = 40, kFp8ManyRegs = 232;

struct Fp8Params {
  int64_t M, N;                 // rows per matrix (not grouped), columns
  int K, B;                     // reduction length, matrices
  int MT, NT;                   // tiles of 128 rows (not grouped), of BN columns
  const float* sa;              // scale of (matrix b, row m, block kb) at b * sa_b + m * sa_m + kb * sa_k
  const float* sb;              // of (matrix b, row or 128-row block n, block kb)
  int64_t sa_b, sa_m, sa_k, sb_b, sb_n, sb_k;
  // grouped
  const int32_t* pad_off;       // [E + 1] first padded row of each expert, in tiles of 128 rows
  const int32_t* n_tiles;       // how many there are
  int32_t* status;              // device status word
  int clear_status;             // no earlier kernel of the call has set it to 0
  int splits;                   // CTAs of a cluster that share a tile's blocks (BN = 128); each cluster has one tile then
};
constexpr int kFp8MaxSplits = 4;

constexpr int kFp8ScaleBlocks = 4, kFp8ScaleSlots = 2;     // blocks of 128 whose scales come together, such groups on their way

constexpr int kFp8BoxBytes = 32 * 128;
constexpr int kFp8ShareBytes = 128 * 64 * 4;               // the most that a CTA of a cluster has of a tile's sums in the end

template <int BN, bool BROWS>
struct Fp8Smem {
  static constexpr int kABytes = 128 * 128;
  static constexpr int kBBytes = BN * 128;
  static constexpr int kStageBytes = kABytes + kBBytes;
  // 128 columns: the last of the six stages is where rows park, unless a cluster shares the tile, whose CTAs have one each
  // and park when the stages are done with
  static constexpr int kStages = BN == 256 ? 3 : 6;
  static constexpr int kBoxes = BN / 128;                  // of 32 rows of 128 bytes, of a warp, on their way out
  static constexpr int kParkBytes = kBoxes * kFp8BoxBytes;
  static constexpr int kScaleFloats = 128 + (BROWS ? BN : 4);                    // of a block: rows, columns or column blocks
  static constexpr int kPark = (BN == 256 ? kStages : kStages - 1) * kStageBytes;     // from the 1024-byte boundary on
  static constexpr int kScales = kPark + kFp8EpiWarps * kParkBytes;
  static_assert(kScales >= kStages * kStageBytes, "a stage is as large as what the warps park");
  static_assert(BN != 128 || kPark >= kFp8MaxSplits * kFp8ShareBytes, "the sums of a cluster's parts");
  static constexpr int kTables = kScales + kFp8ScaleSlots * kFp8ScaleBlocks * kScaleFloats * 4 + 1024;
};
inline int fp8_smem_bytes(int tables, int experts) { return tables + (experts > 0 ? (experts + 1) * 4 : 0); }

__device__ __forceinline__ void tc_mma_fp8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
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

__device__ __forceinline__ void copy_float(uint32_t dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}

// What an epilogue gets: the thread's row and the COLS columns from n0 on whose sums it holds, in pairs.
struct Fp8Tile {
  int b;               // matrix or expert
  int64_t row;         // row of the matrix, or padded row of the expert pass
  int64_t row_end;     // rows from here on are another's
  int n0, n_end;       // n_end: columns of the matrix
  int q, half, lane;   // lane quarter and column half of the warp
  uint32_t park;       // shared memory of the warp's own (kParkBytes)
  bool ok;             // false: take part in barriers only
  const CUtensorMap* out;      // where boxes of 32 rows of 128 bytes go
};
// The four groups of 16 columns of a half of a tile of 128, shared out to `splits` CTAs
__device__ __forceinline__ int fp8_owner(int g, int splits) { return g * splits / 4; }
__device__ __forceinline__ int fp8_first_group(int part, int splits) { return (4 * part + splits - 1) / splits; }

template <int BN, bool BROWS, bool GROUPED, class Epi>
__global__ void __launch_bounds__(kFp8Threads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                const __grid_constant__ CUtensorMap tmOut, const Fp8Params p,
                const Epi epi) {
  using SM = Fp8Smem<BN, BROWS>;
  constexpr int kAccs = 512 / BN, kCols = BN / 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[SM::kStages], bar_empty[SM::kStages], bar_tmem_full[kAccs], bar_tmem_empty[kAccs];
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;
  __shared__ __align__(8) uint64_t bar_scale_full[kFp8ScaleSlots], bar_scale_empty[kFp8ScaleSlots];
  __shared__ typename Epi::Shared s_epi;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int splits = BN == 128 && !GROUPED ? p.splits : 1;
  const int stages = BN == 256 || splits > 1 ? SM::kStages : SM::kStages - 1;
  const int part = splits > 1 ? (int)cluster_ctarank() : 0;       // of the tile's blocks
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  uint8_t* const aligned = smem_raw + (smem_base - smem_u32(smem_raw));
  float* const s_scale = reinterpret_cast<float*>(aligned + SM::kScales);
  int32_t* s_pad = reinterpret_cast<int32_t*>(smem_raw + SM::kTables);     // grouped: first padded row of each expert

  if (threadIdx.x == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 1);
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int a = 0; a < kAccs; ++a) {
      mbar_init(smem_u32(&bar_tmem_full[a]), 1);
      mbar_init(smem_u32(&bar_tmem_empty[a]), kFp8EpiWarps);
    }
    for (int i = 0; i < kFp8ScaleSlots; ++i) {
      mbar_init(smem_u32(&bar_scale_full[i]), 32);
      mbar_init(smem_u32(&bar_scale_empty[i]), kFp8EpiWarps);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  pdl_trigger();
  pdl_wait();
  if constexpr (GROUPED) {
    for (int i = threadIdx.x; i <= p.B; i += kFp8Threads) s_pad[i] = p.pad_off[i];
    __syncthreads();
  }
  if (p.clear_status && blockIdx.x == 0 && threadIdx.x == 0) *p.status = kStatusOk;   // waits give up after seconds at the earliest
  const int64_t total = GROUPED ? (int64_t)*after_wait(p.n_tiles) * p.NT : (int64_t)p.B * p.MT * p.NT;
  const int64_t first_id = blockIdx.x / splits, n_workers = gridDim.x / splits;
  const int kblocks_all = (p.K + kFp8Group - 1) / kFp8Group;
  const int kb_first = part * kblocks_all / splits, kb_end = (part + 1) * kblocks_all / splits;

  // work item -> matrix or expert, first row of the tile, first column
  auto decode = [&](int64_t id, int& b, int64_t& m0, int& n0) {
    if constexpr (GROUPED) {
      const int row = (int)((uint32_t)id / (uint32_t)p.NT) * kTileM;
      int lo = 0, hi = p.B;                      // the last expert whose first tile is not behind this one
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_pad[mid] <= row) lo = mid; else hi = mid;
      }
      b = lo;
      const int first = s_pad[b] / kTileM, cnt = s_pad[b + 1] / kTileM - first;
      const int local = (int)id - first * p.NT;
      const int nt = local / cnt;
      m0 = s_pad[b] + (int64_t)(local - nt * cnt) * kTileM;
      n0 = nt * BN;
    } else {
      const int64_t per = (int64_t)p.MT * p.NT;
      b = (int)(id / per);
      const int64_t local = id - b * per;
      const int nt = (int)(local / p.MT);
      m0 = (local - (int64_t)nt * p.MT) * kTileM;
      n0 = nt * BN;
    }
  };

  if (warp < kFp8FirstEpiWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kFp8FewRegs));
    if (warp == 0) {
      // =========================== TMA producer ================================================
      const bool elected = elect_one();
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t id = first_id; id < total && ok; id += n_workers) {
        int b, n0;
        int64_t m0;
        decode(id, b, m0, n0);
        for (int kb = kb_first; kb < kb_end; ++kb) {
          ok = mbar_wait_warp(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag);
          if (!ok) break;
          if (elected) {
            const uint32_t sa = smem_base + stage * SM::kStageBytes;
            const uint32_t full = smem_u32(&bar_full[stage]);
            mbar_expect_tx(full, SM::kStageBytes);
            tma_load_3d(sa, &tmA, kb * kFp8Group, (int)m0, GROUPED ? 0 : b, full);
            tma_load_3d(sa + SM::kABytes, &tmB, kb * kFp8Group, n0, b, full);
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1u; }
        }
      }
      // the commits that free the last stages must have arrived here before this CTA ends
      for (int s = 0; s < stages && ok; ++s)
        ok = mbar_wait_warp(smem_u32(&bar_empty[s]), s < stage ? phase : phase ^ 1u, &abort_flag);
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicMax(p.status, (int)kStatusProducerTimeout);
      }
      __syncwarp();
    } else if (warp == 1) {
      // =========================== MMA issuer ==================================================
      const uint32_t idesc_base = (1u << 4) | ((uint32_t)(128 >> 4) << 24);   // e4m3 x e4m3 -> fp32, both K-major
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
        const uint32_t idesc = idesc_base | ((uint32_t)(min(BN, ((int)p.N - n0 + 15) & ~15) >> 3) << 17);
        for (int kb = kb_first; kb < kb_end; ++kb) {
          ok = mbar_wait_warp(smem_u32(&bar_full[stage]), phase, &abort_flag);
          if (ok) ok = mbar_wait_warp(smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, &abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (elected) {
            const uint64_t adesc = adesc0 + (uint64_t)(stage * (SM::kStageBytes >> 4));
            const uint64_t bdesc = bdesc0 + (uint64_t)(stage * (SM::kStageBytes >> 4));
#pragma unroll
            for (int k = 0; k < kFp8Group / 32; ++k)
              tc_mma_fp8(tmem_base + acc * BN, adesc + (uint64_t)(2 * k), bdesc + (uint64_t)(2 * k), idesc, (uint32_t)(k != 0));
            tc_commit(smem_u32(&bar_tmem_full[acc]));
            tc_commit(smem_u32(&bar_empty[stage]));
          }
          __syncwarp();
          if (++stage == stages) { stage = 0; phase ^= 1u; }
          if (++acc == kAccs) { acc = 0; acc_phase ^= 1u; }
        }
      }
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicMax(p.status, (int)kStatusMmaTimeout);
      }
      __syncwarp();
    } else if (warp == 2) {
      // =========================== scales ======================================================
      // Four bytes at a time, each on its way by itself; rows and columns that do not exist are 0.
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t id = first_id; id < total && ok; id += n_workers) {
        int b, n0;
        int64_t m0;
        decode(id, b, m0, n0);
        const int64_t row0 = m0, row_end = GROUPED ? (int64_t)s_pad[b + 1] : p.M;
        const float* sa = p.sa + (GROUPED ? 0 : b * p.sa_b);
        const float* sb = p.sb + b * p.sb_b;
        for (int kb = kb_first; kb < kb_end; kb += kFp8ScaleBlocks) {
          ok = mbar_wait_warp(smem_u32(&bar_scale_empty[slot]), phase ^ 1u, &abort_flag);
          if (!ok) break;
          for (int i = 0; i < kFp8ScaleBlocks && kb + i < kb_end; ++i) {
            const uint32_t dst = smem_u32(s_scale + (slot * kFp8ScaleBlocks + i) * SM::kScaleFloats);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int64_t row = row0 + j * 32 + lane;
              copy_float(dst + (j * 32 + lane) * 4, sa + (row < row_end ? row : 0) * p.sa_m + (kb + i) * p.sa_k, row < row_end);
            }
            if constexpr (BROWS) {
#pragma unroll
              for (int j = 0; j < BN / 32; ++j) {
                const int col = n0 + j * 32 + lane;
                copy_float(dst + (128 + j * 32 + lane) * 4, sb + (int64_t)(col < p.N ? col : 0) * p.sb_n + (kb + i) * p.sb_k, col < p.N);
              }
            } else if (lane < BN / 128) {
              const bool there = n0 + lane * 128 < p.N;
              copy_float(dst + (128 + lane) * 4, sb + (int64_t)(n0 / kFp8Group + (there ? lane : 0)) * p.sb_n + (kb + i) * p.sb_k, there);
            }
          }
          asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(&bar_scale_full[slot])) : "memory");
          if (++slot == kFp8ScaleSlots) { slot = 0; phase ^= 1u; }
        }
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicMax(p.status, (int)kStatusProducerTimeout);
      }
      __syncwarp();
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kFp8ManyRegs));
    // =========================== scaled sums and epilogue (warps 4 .. 11) ====================
    const int q = warp & 3;                      // TMEM lane quarter this warp may read
    const int half = (warp - kFp8FirstEpiWarp) >> 2;      // its columns: kCols from half * kCols on
    const uint32_t t_row = tmem_base + ((uint32_t)(q * 32) << 16) + half * kCols;
    int acc = 0, slot = 0;
    uint32_t acc_phase = 0, slot_phase = 0, parity = 0;
    bool ok = true;
    for (int64_t id = first_id; id < total; id += n_workers, parity ^= 1u) {
      Fp8Tile t;
      int n0;
      int64_t m0;
      decode(id, t.b, m0, n0);
      t.row = m0 + q * 32 + lane;
      t.row_end = GROUPED ? (int64_t)s_pad[t.b + 1] : p.M;
      t.n0 = n0 + half * kCols;
      t.n_end = (int)p.N;
      t.q = q; t.half = half; t.lane = lane;
      t.out = &tmOut;
      t.park = smem_base + SM::kPark + (warp - kFp8FirstEpiWarp) * SM::kParkBytes;
      const bool row_ok = t.row < t.row_end;
      const auto pre = epi.begin(t, row_ok);
      uint64_t sum[kCols / 2];
#pragma unroll
      for (int i = 0; i < kCols / 2; ++i) sum[i] = 0;
      // (Columns behind the matrix are loaded and added like others; nobody reads their sums.)
      uint32_t r[2][32];
      if (ok) ok = mbar_wait_warp(smem_u32(&bar_tmem_full[acc]), acc_phase, &abort_flag);
      if (ok) {
        tc_fence_after();
        tc_ld_32x32_issue(t_row + acc * BN, r[0]);
      }
      for (int kb = kb_first; kb < kb_end; ++kb) {
        const int in_slot = (kb - kb_first) % kFp8ScaleBlocks;
        if (in_slot == 0 && ok) ok = mbar_wait_warp(smem_u32(&bar_scale_full[slot]), slot_phase, &abort_flag);
        const float* scale = s_scale + (slot * kFp8ScaleBlocks + in_slot) * SM::kScaleFloats;
        const float sa = scale[q * 32 + lane], s = BROWS ? sa : sa * scale[128 + half * kCols / 128];
        const uint64_t s2 = pack_f32x2(s, s);
        const bool last = kb + 1 == kb_end;
        const int next = acc + 1 == kAccs ? 0 : acc + 1;
        const uint32_t next_phase = acc_phase ^ (next == 0 ? 1u : 0u);
        uint32_t early = 0;
        if (ok) {
#pragma unroll
          for (int c = 0; c < kCols / 32; ++c) {
            uint32_t (&now)[32] = r[c & 1], (&then)[32] = r[(c + 1) & 1];
            tc_ld_wait(now);
            if (c + 1 < kCols / 32) {
              tc_ld_32x32_issue(t_row + acc * BN + (c + 1) * 32, then);
              if (c + 2 == kCols / 32) early = last ? 1u : mbar_try_wait(smem_u32(&bar_tmem_full[next]), next_phase);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) {
                mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
              }
              if (!last) {
                if (!__all_sync(0xffffffffu, early != 0)) ok = mbar_wait_warp(smem_u32(&bar_tmem_full[next]), next_phase, &abort_flag);
                if (ok) {
                  tc_fence_after();
                  tc_ld_32x32_issue(t_row + next * BN, then);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) {
              const uint64_t v = pack_f32x2(__uint_as_float(now[2 * i]), __uint_as_float(now[2 * i + 1]));
              const uint64_t x = pack_f32x2(__uint_as_float(now[2 * i + 2]), __uint_as_float(now[2 * i + 3]));
              uint64_t f = s2, g = s2;
              if constexpr (BROWS) {
                const float4 cols = *reinterpret_cast<const float4*>(scale + 128 + half * kCols + c * 32 + 2 * i);
                f = mul_f32x2(s2, pack_f32x2(cols.x, cols.y));
                g = mul_f32x2(s2, pack_f32x2(cols.z, cols.w));
              }
              sum[c * 16 + i] = fma_f32x2(v, f, sum[c * 16 + i]);
              sum[c * 16 + i + 1] = fma_f32x2(x, g, sum[c * 16 + i + 1]);
            }
          }
        }
        acc = next;
        acc_phase = next_phase;
        if (in_slot == kFp8ScaleBlocks - 1 || last) {
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_u32(&bar_scale_empty[slot]));
          if (++slot == kFp8ScaleSlots) { slot = 0; slot_phase ^= 1u; }
        }
      }
      t.ok = ok;
      if constexpr (BN == 128 && !GROUPED) {
        if (splits > 1) {
          // Each CTA gets all parts' sums of its own share of the columns, its own among them, so that no register is
          // picked by part: [part][half][four columns][row], a warp stores 512 contiguous bytes.
          const uint32_t at = (uint32_t)(half * (kFp8ShareBytes / 2) + (q * 32 + lane) * 16);
          cluster_sync_all();                    // everyone's copies and instructions are done with their shared memory
          if (row_ok) {
#pragma unroll
            for (int g = 0; g < kCols / 16; ++g) {
              const int owner = fp8_owner(g, splits);
              const uint32_t dst = mapa_u32(smem_base, owner) + part * kFp8ShareBytes + at + (g - fp8_first_group(owner, splits)) * 8192;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                float v[4];
                unpack_f32x2(sum[8 * g + 2 * i], v[0], v[1]);
                unpack_f32x2(sum[8 * g + 2 * i + 1], v[2], v[3]);
                asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)i * 2048u), "f"(v[0]), "f"(v[1]),
                             "f"(v[2]), "f"(v[3]) : "memory");
              }
            }
          }
          cluster_sync_all();
          if (ok && t.row - lane < t.row_end) {
            const int g0 = fp8_first_group(part, splits), g1 = fp8_first_group(part + 1, splits);
#pragma unroll 1
            for (int g = g0; g < g1 && t.n0 + 16 * g < t.n_end; ++g) {
              float v[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = 0.f;
#pragma unroll 1
              for (int o = 0; o < splits; ++o) {
                const uint32_t src = smem_base + o * kFp8ShareBytes + at + (g - g0) * 8192;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                  float x[4];
                  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(x[0]), "=f"(x[1]), "=f"(x[2]), "=f"(x[3])
                               : "r"(src + (uint32_t)i * 2048u) : "memory");
#pragma unroll
                  for (int j = 0; j < 4; ++j) v[4 * i + j] += x[j];
                }
              }
              epi.store_group(t, v, 16 * g);
            }
          }
          break;
        }
      }
      epi.template finish<kCols, SM::kBoxes>(t, row_ok, pre, sum, s_epi, parity);
    }
    tma_store_wait_all();
    if (!ok) {
      abort_flag = 1;
      atomicMax(p.status, (int)kStatusEpilogueTimeout);
    }
  }

  if (splits > 1 && warp < kFp8FirstEpiWarp) {     // what the other warps do between their sums and their epilogue
    cluster_sync_all();
    cluster_sync_all();
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
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---------------------------------------------------------------------------------------------
// Epilogues
// ---------------------------------------------------------------------------------------------

// 64 bytes of each of the warp's 32 rows (a lane's own, in `v`) to `dst` (null: nowhere), of which `pieces` of 16 bytes
// exist.  By way of shared memory, so that four lanes write a row's bytes side by side.
__device__ __forceinline__ void store_rows_64(uint32_t park, int lane, const uint4 (&v)[4], char* dst, int pieces) {
#pragma unroll
  for (int k = 0; k < 4; ++k)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(park + lane * 64 + ((k ^ ((lane >> 1) & 3)) << 4)), "r"(v[k].x),
                 "r"(v[k].y), "r"(v[k].z), "r"(v[k].w) : "memory");
  __syncwarp();
  const int k = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = i * 8 + (lane >> 2);
    char* to = reinterpret_cast<char*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
    uint4 x;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                 : "r"(park + r * 64 + ((k ^ ((r >> 1) & 3)) << 4)) : "memory");
    if (to != nullptr && k < pieces) *reinterpret_cast<uint4*>(to + 16 * k) = x;
  }
  __syncwarp();
}

// 16 bytes (piece k) of the lane's row of a box, as TMA with 128-byte swizzle wants them
__device__ __forceinline__ void park_row(const Fp8Tile& t, int box, int k, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(t.park + box * kFp8BoxBytes + t.lane * 128 + ((k ^ (t.lane & 7)) << 4)),
               "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}
// The warp's boxes on their way; rows and columns that do not exist are cut off by the tensor map.  While a tile is stored no
// accumulator is taken up: 128 x 256 values of bf16 took 6000 clocks by 16-byte stores straight from the lanes that hold
// the rows, 3450 with four lanes to a row, as long with a bulk copy per row (95 clocks apiece to issue), 1300 as boxes.
template <int BOXES>
__device__ __forceinline__ void send_boxes(const Fp8Tile& t, int col, int box_cols) {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  __syncwarp();
  if (t.lane == 0 && t.row < t.row_end) {
#pragma unroll
    for (int x = 0; x < BOXES; ++x)
      if (col + x * box_cols < t.n_end)
        tma_store_3d(t.out, col + x * box_cols, (int)t.row, t.b, t.park + x * kFp8BoxBytes);
    tma_store_commit();
  }
}
__device__ __forceinline__ void boxes_free(int lane) {
  if (lane == 0) tma_store_wait_read();
  __syncwarp();
}

// C[b, m, n] rounded to T
template <typename T>
struct Fp8Store {
  struct Shared {};
  struct Pre {};
  T* C;
  int64_t ld, batch;
  int vec;                 // rows start on 16-byte boundaries

  __device__ __forceinline__ Pre begin(const Fp8Tile&, bool) const { return {}; }

  // 16 columns of the warp's rows from n0 + i on, the lane's in `v`, as far as they exist
  __device__ __forceinline__ void store_group(const Fp8Tile& t, const float (&v)[16], int i) const {
    constexpr int kPieces = (int)sizeof(T), kPitch = 16 * kPieces + 16;      // 16-byte pieces of a row
    const uint32_t mine = t.park + t.lane * kPitch;
#pragma unroll
    for (int k = 0; k < kPieces; ++k) {
      uint4 w;
      if constexpr (sizeof(T) == 2)
        w = make_uint4(pack_bf16x2(v[8 * k], v[8 * k + 1]), pack_bf16x2(v[8 * k + 2], v[8 * k + 3]),
                       pack_bf16x2(v[8 * k + 4], v[8 * k + 5]), pack_bf16x2(v[8 * k + 6], v[8 * k + 7]));
      else
        w = make_uint4(__float_as_uint(v[4 * k]), __float_as_uint(v[4 * k + 1]), __float_as_uint(v[4 * k + 2]),
                       __float_as_uint(v[4 * k + 3]));
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(mine + 16 * k), "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w) : "memory");
    }
    __syncwarp();
    const int rows = (int)min((int64_t)32, t.row_end - (t.row - t.lane));
    const int cols = min(16, t.n_end - t.n0 - i);
    T* const first = C + t.b * batch + (t.row - t.lane) * ld + t.n0 + i;      // the warp's first row
    if (vec) {
      constexpr int kRows = 32 / kPieces;              // at a time
      const int k = t.lane % kPieces;
#pragma unroll
      for (int p = 0; p < kPieces; ++p) {
        const int r = p * kRows + t.lane / kPieces;
        uint4 x;
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x.x), "=r"(x.y), "=r"(x.z), "=r"(x.w)
                     : "r"(t.park + r * kPitch + 16 * k) : "memory");
        if (r < rows && k * (16 / kPieces) < cols) *reinterpret_cast<uint4*>(first + r * ld + k * (16 / kPieces)) = x;
      }
    } else {
      using U = typename std::conditional<sizeof(T) == 2, uint16_t, uint32_t>::type;
      const int j = t.lane & 15;
      U x[16];
#pragma unroll
      for (int p = 0; p < 16; ++p) {
        const uint32_t at = t.park + (2 * p + (t.lane >> 4)) * kPitch + j * (int)sizeof(T);
        if constexpr (sizeof(T) == 2) asm volatile("ld.shared.b16 %0, [%1];" : "=h"(x[p]) : "r"(at) : "memory");
        else asm volatile("ld.shared.b32 %0, [%1];" : "=r"(x[p]) : "r"(at) : "memory");
      }
#pragma unroll
      for (int p = 0; p < 16; ++p) {
        const int r = 2 * p + (t.lane >> 4);
        if (r < rows && j < cols) reinterpret_cast<U*>(first + r * ld)[j] = x[p];
      }
    }
    __syncwarp();
  }

  template <int COLS, int BOXES>
  __device__ __forceinline__ void finish(const Fp8Tile& t, bool, const Pre&, const uint64_t (&sum)[COLS / 2], Shared&, uint32_t) const {
    if (!t.ok) return;
    if (vec) {
      constexpr int kBoxCols = 128 / (int)sizeof(T);
#pragma unroll
      for (int i = 0; i < COLS; i += BOXES * kBoxCols) {
        if (t.n0 + i >= t.n_end) break;
        boxes_free(t.lane);
#pragma unroll
        for (int k = 0; k < 8 * BOXES; ++k) {
          constexpr int VE = 16 / (int)sizeof(T);
          float v[VE];
#pragma unroll
          for (int j = 0; j < VE; j += 2) unpack_f32x2(sum[(i + k * VE + j) / 2], v[j], v[j + 1]);
          if constexpr (sizeof(T) == 2)
            park_row(t, k / 8, k % 8, pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
          else
            park_row(t, k / 8, k % 8, __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        }
        send_boxes<BOXES>(t, t.n0 + i, kBoxCols);
      }
      return;
    }
#pragma unroll
    for (int i = 0; i < COLS; i += 16) {
      if (t.n0 + i >= t.n_end) break;
      float v[16];
#pragma unroll
      for (int j = 0; j < 16; j += 2) unpack_f32x2(sum[(i + j) / 2], v[j], v[j + 1]);
      store_group(t, v, i);
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
  template <int COLS, int BOXES>
  __device__ __forceinline__ void finish(const Fp8Tile& t, bool row_ok, const Pre&, const uint64_t (&sum)[COLS / 2], Shared& s,
                                         uint32_t parity) const {
    static_assert(COLS == 128, "a group of 128 activations is a tile of 256 columns");
    float a[64];
    uint32_t most = 0;
    const T* bs = bias + (int64_t)t.b * t.n_end + t.n0;
#pragma unroll
    for (int i = 0; i < 64; i += 4) {
      float b[8];                                  // eight columns: n_end is a multiple of 16, and so is n0
      if (t.n0 + 2 * i < t.n_end) load_vec<T, 8>(bs + 2 * i, b);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float g, v;
        unpack_f32x2(sum[i + j], g, v);
        a[i + j] = t.n0 + 2 * i < t.n_end ? glu_act(g + b[2 * j], v + b[2 * j + 1]) : 0.f;
        most = max(most, abs_bits(a[i + j]));
      }
    }
    const int r = t.q * 32 + t.lane;
    s.most[parity][t.half][r] = most;
    named_sync(4 + t.q, 64);
    if (!t.ok || t.n0 >= t.n_end) return;
    const float top = fp8_group_max(max(most, s.most[parity][t.half ^ 1][r])), inv = fp8_inverse(top);
    uint4 w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k)
      w[k] = make_uint4(e4m3x4(a[16 * k] * inv, a[16 * k + 1] * inv, a[16 * k + 2] * inv, a[16 * k + 3] * inv),
                        e4m3x4(a[16 * k + 4] * inv, a[16 * k + 5] * inv, a[16 * k + 6] * inv, a[16 * k + 7] * inv),
                        e4m3x4(a[16 * k + 8] * inv, a[16 * k + 9] * inv, a[16 * k + 10] * inv, a[16 * k + 11] * inv),
                        e4m3x4(a[16 * k + 12] * inv, a[16 * k + 13] * inv, a[16 * k + 14] * inv, a[16 * k + 15] * inv));
    const int64_t col = t.n0 / 2;
    store_rows_64(t.park, t.lane, w, row_ok ? reinterpret_cast<char*>(act + t.row * ld + col) : nullptr, (int)(ld - col) / 16);
    if (row_ok && t.half == 0) scale[(t.n0 / (2 * kFp8Group)) * scale_group + t.row] = fp8_scale(top);
  }
};

// down of the expert pass: y = w_row * (v + bias) in fp32 at the padded row, as combine_padded_kernel wants the K rows of a
// token that it sums.  What padding rows get is not read.
template <typename T>
struct Fp8WeightedRows {
  struct Shared {};
  struct Pre { float w; };
  const T* bias;           // [E, N]
  const int32_t* row_token;
  const float* row_weight;
  int64_t N;

  __device__ __forceinline__ Pre begin(const Fp8Tile& t, bool row_ok) const {
    const int token = row_ok ? row_token[t.row] : -1;
    const float w = row_ok ? row_weight[t.row] : 0.f;          // (padding rows have none)
    return Pre{token >= 0 ? w : 0.f};
  }
  template <int COLS, int BOXES>
  __device__ __forceinline__ void finish(const Fp8Tile& t, bool, const Pre& p, const uint64_t (&sum)[COLS / 2], Shared&,
                                         uint32_t) const {
    if (!t.ok) return;
    const T* bs = bias + t.b * N + t.n0;
    Fp8Tile o = t;
    o.b = 0;                                         // the rows of all experts are one matrix
#pragma unroll
    for (int i = 0; i < COLS; i += 32 * BOXES) {
      const int cols = t.n_end - t.n0 - i;           // a multiple of 8
      if (cols <= 0) break;
      boxes_free(t.lane);
#pragma unroll
      for (int k = 0; k < 4 * BOXES; ++k) {
        float b[8] = {}, v[8];
        if (8 * k < cols) load_vec<T, 8>(bs + i + 8 * k, b);
#pragma unroll
        for (int j = 0; j < 8; j += 2) unpack_f32x2(sum[(i + 8 * k + j) / 2], v[j], v[j + 1]);
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = p.w * (v[j] + b[j]);
        park_row(t, k / 4, 2 * (k % 4), __float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
        park_row(t, k / 4, 2 * (k % 4) + 1, __float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7]));
      }
      send_boxes<BOXES>(o, t.n0 + i, 32);
    }
  }
};

// ---------------------------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------------------------

// Prepares a kernel for its shared memory, once per kernel and device
template <class Epi>
constexpr int kFp8MostSmem = 227 * 1024 - 1024 - (int)sizeof(typename Epi::Shared);     // static shared memory lies beside it
template <class Epi, typename... KArgs>
inline bool fp8_configure(void (*kern)(KArgs...), PerDevice<int>& done) {
  const int dev = current_device_index();
  if (done.get(dev)) return true;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFp8MostSmem<Epi>) != cudaSuccess) return false;
  done.set(dev, 1);
  return true;
}

struct Fp8Operand {
  const void* q;
  int64_t rows, ld, batch;      // rows per matrix, pitch, distance of matrices (bytes)
};
// Where the boxes of a tile go; null: the epilogue sends none
struct Fp8Out {
  void* c;
  int64_t rows, cols, batch;    // rows of a matrix; matrices
  int size;                     // of a value: 2 bf16, 4 fp32
};

// Clusters of `splits` CTAs that are on the GPU at the same time
template <bool BROWS, class Epi>
inline int fp8_clusters(int splits) {
  static PerDevice<int> most[kFp8MaxSplits + 1], configured;
  const int dev = current_device_index();
  int n = most[splits].get(dev);
  if (n > 0) return n;
  auto kern = fp8_gemm_kernel<128, BROWS, false, Epi>;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits);
  cfg.blockDim = dim3(kFp8Threads);
  cfg.dynamicSmemBytes = (size_t)fp8_smem_bytes(Fp8Smem<128, BROWS>::kTables, 0);
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (!fp8_configure<Epi>(kern, configured) || cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = umma_sm_count() / splits;
  }
  most[splits].set(dev, n);
  return n;
}

// `max_tiles`: row tiles of 128 rows in all
template <int BN, bool BROWS, bool GROUPED, class Epi>
inline int launch_fp8_gemm(const Fp8Operand& a, const Fp8Operand& b, const Fp8Out& o, Fp8Params p, const Epi& epi, int64_t max_tiles,
                           cudaStream_t st) {
  if (!umma_available()) return YAMOE_ERR_UNSUPPORTED;
  using SM = Fp8Smem<BN, BROWS>;
  static_assert(SM::kTables + (GROUPED ? 1025 * 4 : 0) <= kFp8MostSmem<Epi>, "up to 1024 experts");
  CUtensorMap tmA, tmB, tmOut{};
  const uint64_t na = GROUPED ? 1 : (uint64_t)p.B;
  const uint64_t da[3] = {(uint64_t)p.K, (uint64_t)a.rows, na}, db[3] = {(uint64_t)p.K, (uint64_t)b.rows, (uint64_t)p.B};
  const uint64_t ga[2] = {(uint64_t)a.ld, (uint64_t)(na > 1 ? a.batch : a.ld * a.rows)};
  const uint64_t gb[2] = {(uint64_t)b.ld, (uint64_t)(p.B > 1 ? b.batch : b.ld * b.rows)};
  const uint32_t boxa[3] = {128, 128, 1}, boxb[3] = {128, BN, 1};
  if (!encode_map(&tmA, a.q, 3, da, ga, boxa, kMapU8) || !encode_map(&tmB, b.q, 3, db, gb, boxb, kMapU8)) return YAMOE_ERR_CUDA;
  if (o.c != nullptr) {
    const uint64_t dim[3] = {(uint64_t)o.cols, (uint64_t)o.rows, (uint64_t)o.batch};
    const uint64_t pitch[2] = {(uint64_t)(o.cols * o.size), (uint64_t)(o.cols * o.size * o.rows)};
    const uint32_t box[3] = {128u / o.size, 32, 1};
    if (!encode_map(&tmOut, o.c, 3, dim, pitch, box, o.size == 2 ? kMapBf16 : kMapF32Swizzled)) return YAMOE_ERR_CUDA;
  }
  auto kern = fp8_gemm_kernel<BN, BROWS, GROUPED, Epi>;
  static PerDevice<int> configured;    // per template instantiation and device
  if (!fp8_configure<Epi>(kern, configured)) return YAMOE_ERR_CUDA;
  p.NT = (int)ceil_div(p.N, BN);
  const int64_t total = max_tiles * p.NT;
  if (total <= 0) return YAMOE_OK;
  const bool split = BN == 128 && !GROUPED && p.splits > 1;
  if (!split) p.splits = 1;
  // Clusters that start early, on SMs that the launch before leaves free, take places from those that cannot: 45 clusters of three
  // took 16.6 us instead of 12.6.
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(split ? p.splits * total : std::min<int64_t>(total, umma_sm_count())));
  cfg.blockDim = dim3(kFp8Threads);
  cfg.dynamicSmemBytes = (size_t)fp8_smem_bytes(SM::kTables, GROUPED ? p.B : 0);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = p.splits;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled(true) && !split ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (cudaLaunchKernelEx(&cfg, kern, tmA, tmB, tmOut, p, epi) != cudaSuccess) return YAMOE_ERR_CUDA;
  return cudaGetLastError() == cudaSuccess ? YAMOE_OK : YAMOE_ERR_CUDA;
}

}  // namespace yb
