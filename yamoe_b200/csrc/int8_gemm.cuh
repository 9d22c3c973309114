// Product of two matrices of 8-bit integers with a scale per row of either (tcgen05 kind::i8, cta_group::2, sm_100a):
//
//   C[m, n] = sa[m] * sb[n] * (sum over k of qa[m, k] * qb[n, k])
//
// The sum is exact in 32 bits (K < 2^17), so neither tiles nor splits change a result; it is brought to fp32 once, then times sa, times sb
// (a product of the two scales first could leave the range), and rounded once to the output's type.
//
// Three arrangements: one or several pairs of matrices, and rows sorted by expert (offsets[e] .. offsets[e + 1] - 1 times matrix e).
//
// int8_pair_kernel.  As in umma_pair.cuh, CTA pairs with the weights' rows (output columns) in the instruction's M dimension, 256 to a pair, and
// the tokens' rows in its N dimension, any multiple of 32 up to 256: an expert's rows are cut into tiles of equal width wherever they
// begin, so nothing is padded in memory, and few rows cost few clocks.  A k-block is 128 bytes wide, one swizzle row, up to 32 KB per CTA;
// two accumulators, so that a tile is scaled and stored while the next is multiplied.  Scales are met in the epilogue alone, unlike the
// e4m3 products with a scale per 128 (fp8_gemm.cuh), whose sums leave TMEM after every block.  8192 x 5760 x 2880: 88 us on a cool GPU, 3.1
// PFLOP/s, 111 for seconds on end under the power cap; 2048 rows of 32 experts, 5760 x 2880 each: 98 us alone behind a flushed L2, 5.7 TB/s, 93 among its
// like; 32 matrices of 64 rows 90 and 87 us, of 512 rows 189 and 211 (power).
// Few tiles: a cluster of up to four pairs shares a tile's k-blocks; the chunks of 32 rows are dealt out among the pairs, each of which gets
// the others' sums of its chunks through distributed shared memory.
//
// int8_rows_kernel.  A handful of rows: bound by the bytes of the weights and by latency.  A CTA has 16 output columns and all rows, its eight
// warps take 64-byte blocks of k in turn, straight from global memory to mma.sync m16n8k32; their sums meet in shared memory.
//
// Every wait is bounded as in umma_gemm.cuh.
#pragma once
#include <algorithm>

#include "tcgen05.cuh"

namespace yb {

// A k-block: this CTA's 128 rows of weights and half of the tile's rows of tokens in boxes of 32, 128 bytes each.  Blocks come, are multiplied and
// are given back in groups: two at a time, which spares the warps every other wait (64 x 5760 x 2880: one at a time 9.3 us, two 8.3; the widest tiles of
// 2048 rows of 32 experts, which wait for HBM: 92, 93), but for the widest tiles of products that are not grouped, whose instructions take longer than
// the waits and of which the ring holds three groups of two (8192 x 5760 x 2880, alone: 94, 98).
constexpr int int8_block_bytes(int width) { return 128 * 128 + (width + 63) / 64 * 4096; }
constexpr int int8_depth(int width, bool grouped) { return width > 192 && !grouped ? 1 : 2; }
constexpr int kInt8Ring = 10 * int8_block_bytes(64), kInt8MaxGroups = 6;
constexpr int int8_groups(int width, int depth) { return kInt8Ring / (depth * int8_block_bytes(width)); }
static_assert(int8_groups(32, 2) == 5 && int8_groups(128, 2) == 4 && int8_groups(192, 2) == 3 && int8_groups(256, 1) == kInt8MaxGroups, "");
constexpr int kInt8EpiWarps = 8, kInt8Threads = 32 * (3 + kInt8EpiWarps);
constexpr int kInt8ParkBytes = 32 * 64;                  // 32 rows of an epilogue warp's 32 columns on their way out
constexpr int kInt8RingBytes = kInt8Ring + 1024;         // + slack for 1024-byte alignment
constexpr int kInt8MaxSplits = 4;
constexpr int kInt8ChunkBytes = 128 * 32 * 4;            // sums of 128 columns and 32 rows
// Chunks of 32 rows are dealt out to the pairs.  Where the sums of chunk c of pair `part` wait at its owner: a slot for each pair.
__host__ __device__ constexpr int int8_owner(int c, int splits) { return c % splits; }
__host__ __device__ constexpr int int8_exchange_slot(int c, int splits, int part) { return c / splits * splits + part; }
constexpr int int8_exchange_slots(int splits) { return (8 + splits - 1) / splits * splits; }
static_assert(int8_exchange_slots(2) * kInt8ChunkBytes <= kInt8Ring && int8_exchange_slots(3) * kInt8ChunkBytes <= kInt8Ring &&
              int8_exchange_slots(4) * kInt8ChunkBytes <= kInt8Ring, "the exchange takes the ring's place");
constexpr int kInt8MaxExperts = 1024;
// Rows of a tile where `rows` are cut into `tiles`, a multiple of 32; the last tile has the rest.
__host__ __device__ constexpr int int8_tile_rows(int rows, int tiles) { return ((rows + tiles - 1) / tiles + 31) & ~31; }

template <typename T>
struct Int8Params {
  int64_t M;                    // rows per matrix, or of all experts
  int N, K, B;                  // columns, reduction length, matrices (experts)
  int width;                    // rows of a tile at most, a multiple of 32
  int groups, depth, block_bytes;       // of the ring: groups of `depth` k-blocks, for tiles of that width
  int MT, NT;                   // tiles of `width` rows per matrix (not grouped), of 256 columns
  const float* sa;              // scale of (matrix b, row m) at b * sa_b + m * sa_m
  const float* sb;
  int64_t sa_b, sa_m, sb_b, sb_n;
  const int32_t* offsets;       // grouped: [B + 1]
  T* out;                       // rows N apart, matrices M * N
  int wide;                     // bf16 in rows of 16-byte multiples
  int32_t* status;
  int splits;                   // pairs of a cluster that share a tile's k-blocks; a cluster has one tile then
};

__device__ __forceinline__ void tc2_mma_int8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the barrier at this shared-memory offset in the CTAs of `mask` once every MMA issued so far is done
__device__ __forceinline__ void tc2_commit_to(uint32_t bar, uint16_t mask) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
               ::"r"(bar), "h"(mask) : "memory");
}

// Row `e` of the experts' table, kept within the rows that there are
__device__ __forceinline__ int int8_offset(const int32_t* offsets, int e, int64_t M) {
  return (int)max((int64_t)0, min((int64_t)offsets[e], M));
}

template <typename T>
__device__ __forceinline__ void int8_zero_row(T* row, int N, int first, int step) {
  for (int n = first; n < N; n += step) DT<T>::st(row + n, 0.f);
}

// Sums of 32 columns and 32 rows as a warp loads them.  `wide`: by tc_ld_16x256_issue, v[16 (h >> 1) + 4 j + 2 (h & 1) + o] is column 8 h + lane / 4, row
// 8 j + 2 (lane % 4) + o; else by tc_ld_32x32_issue, v[i] is this lane's column, row i.
__device__ __forceinline__ void int8_load_sums(bool wide, uint32_t taddr, uint32_t (&v)[32]) {
  if (wide) tc_ld_16x256_issue(taddr, v);
  else tc_ld_32x32_issue(taddr, v);
  tc_ld_wait(v);
}

// Such sums scaled and stored: the columns from `col` on, rows `row` .. row + nvalid - 1 of `out`; lane i has the scales of row i, sb those of the lane's
// columns.  bf16 in rows of 16-byte multiples (`wide`) is turned around by stmatrix in 2 KB of the warp's own and leaves in 16-byte pieces,
// four to a row; the 16-byte pieces of a parked row are permuted so that eight rows of a matrix fall on different banks.
template <typename T>
__device__ __forceinline__ void int8_store(const Int8Params<T>& p, T* out, bool wide, float sa_lane, const float (&sb)[4], int col, int64_t row,
                                           int nvalid, int lane, uint32_t park, const uint32_t (&v)[32]) {
  if (sizeof(T) == 2 && wide) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float a0 = __shfl_sync(0xffffffffu, sa_lane, 8 * j + 2 * (lane & 3)), a1 = __shfl_sync(0xffffffffu, sa_lane, 8 * j + 2 * (lane & 3) + 1);
      uint32_t two[4];
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int i = 16 * (h >> 1) + 4 * j + 2 * (h & 1);
        const __nv_bfloat162 b = __floats2bfloat162_rn((float)(int)v[i] * a0 * sb[h], (float)(int)v[i + 1] * a1 * sb[h]);
        two[h] = *reinterpret_cast<const uint32_t*>(&b);
      }
      const int r = 8 * j + (lane & 7), piece = (lane >> 3) ^ ((r >> 1) & 3);
      stmatrix_x4_trans(park + r * 64 + piece * 16, two[0], two[1], two[2], two[3]);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 8 * i + (lane >> 2), c = col + 8 * (lane & 3);
      uint4 q;
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w)
                   : "r"(park + r * 64 + (((lane & 3) ^ ((r >> 1) & 3)) << 4)) : "memory");
      if (r < nvalid && c < p.N) *reinterpret_cast<uint4*>(out + (row + r) * p.N + c) = q;
    }
    __syncwarp();
  } else {
    T* at = out + row * p.N + col + lane;
#pragma unroll
    for (int i = 0; i < 32; ++i) {
      const float x = (float)(int)v[i] * __shfl_sync(0xffffffffu, sa_lane, i) * sb[0];
      if (i < nvalid && col + lane < p.N) DT<T>::st(at, x);
      at += p.N;
    }
  }
}

template <typename T, bool GROUPED>
__global__ void __launch_bounds__(kInt8Threads, 1)
int8_pair_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                 const __grid_constant__ CUtensorMap tmXsmall, const Int8Params<T> p) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t bar_full[kInt8MaxGroups];       // used in the leader CTA of the pair
  __shared__ __align__(8) uint64_t bar_empty[kInt8MaxGroups];      // per CTA
  __shared__ __align__(8) uint64_t bar_tmem_full[2];            // per CTA
  __shared__ __align__(8) uint64_t bar_tmem_empty[2];           // used in the leader CTA
  __shared__ uint32_t tmem_base_slot;
  __shared__ int abort_flag;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t cta = cluster_ctarank(), rank = cta & 1, lead = cta & ~1u;
  const bool leader = rank == 0;
  const uint16_t pair_mask = (uint16_t)(3u << lead);
  const int splits = GROUPED ? 1 : p.splits, part = (int)(cta >> 1);
  const int groups = p.groups, depth = p.depth, block_bytes = p.block_bytes;
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  int32_t* s_row = reinterpret_cast<int32_t*>(smem_raw + kInt8RingBytes + kInt8EpiWarps * kInt8ParkBytes);      // grouped: [B + 1] first row of each expert
  int32_t* s_tile = s_row + p.B + 1;                                           // grouped: [B + 1] row tiles before each expert's

  if (threadIdx.x == 0) {
    for (const CUtensorMap* map : {&tmW, &tmX, &tmXsmall}) asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
    for (int s = 0; s < groups; ++s) {
      mbar_init(smem_u32(&bar_full[s]), 2);    // arrive.expect_tx of both CTAs
      mbar_init(smem_u32(&bar_empty[s]), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(smem_u32(&bar_tmem_full[a]), 1);
      mbar_init(smem_u32(&bar_tmem_empty[a]), 2 * kInt8EpiWarps);
    }
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&tmem_base_slot)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();          // the peers' barriers exist before any remote signal is sent
  tc_fence_after();
  const uint32_t tmem_base = tmem_base_slot;
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0 && threadIdx.x == 0) *p.status = kStatusOk;        // waits give up after seconds at the earliest
  if constexpr (GROUPED) {
    const int32_t* offsets = after_wait(p.offsets);
    for (int i = threadIdx.x; i <= p.B; i += kInt8Threads) s_row[i] = int8_offset(offsets, i, p.M);
    __syncthreads();
    if (warp == 0) {
      // first rows, none below one before it (which keeps whatever the table holds within the rows), and the numbers of tiles
      int before = 0, top = s_row[0];
      for (int e0 = 0; e0 < p.B; e0 += 32) {
        const int e = e0 + lane;
        int end = max(top, e < p.B ? s_row[e + 1] : 0);
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, end, o);
          if (lane >= o) end = max(end, up);
        }
        int first = __shfl_up_sync(0xffffffffu, end, 1);
        if (lane == 0) first = top;
        int tiles = (end - first + p.width - 1) / p.width;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int up = __shfl_up_sync(0xffffffffu, tiles, o);
          if (lane >= o) tiles += up;
        }
        if (e < p.B) {
          s_row[e + 1] = end;
          s_tile[e + 1] = before + tiles;
        }
        before += __shfl_sync(0xffffffffu, tiles, 31);
        top = __shfl_sync(0xffffffffu, end, 31);
      }
      if (lane == 0) s_tile[0] = 0;
    }
    __syncthreads();
  }
  const int total = (GROUPED ? s_tile[p.B] : p.B * p.MT) * p.NT;             // (the host keeps them below 2^30)
  const int first_id = blockIdx.x / (2 * splits), n_workers = gridDim.x / (2 * splits);
  const int kblocks_all = (p.K + 127) >> 7;
  const int kb_first = part * kblocks_all / splits, kb_end = (part + 1) * kblocks_all / splits;

  // work item -> matrix or expert, first column, first row, its end, width (a multiple of 32)
  auto decode = [&](int id, int& b, int& m0, int& row0, int& row_end, int& width) {
    int local, tiles, first, rows;
    if constexpr (GROUPED) {
      const int tile = id / p.NT;                       // experts' tiles follow each other, NT items to each
      int lo = 0, hi = p.B;                             // the last expert whose first tile is not behind this one
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_tile[mid] <= tile) lo = mid; else hi = mid;
      }
      b = lo;
      tiles = s_tile[b + 1] - s_tile[b];
      local = id - s_tile[b] * p.NT;
      first = s_row[b];
      rows = s_row[b + 1] - first;
    } else {
      const int per = p.MT * p.NT;
      b = id / per;
      local = id - b * per;
      tiles = p.MT;
      first = 0;
      rows = (int)p.M;
    }
    // the row tile varies fastest, so that the pairs running at a time share weights in L2
    const int nt = local / tiles;
    const int step = int8_tile_rows(rows, tiles);
    m0 = nt * 256;
    row0 = first + (local - nt * tiles) * step;
    row_end = min(first + rows, row0 + step);
    width = (row_end - row0 + 31) & ~31;                 // (tiles of at most 256 rows, rounded up to 32: none is left without rows)
  };

  if (warp == 0 || warp == 2 + kInt8EpiWarps) {
    // =========================== TMA producers (both CTAs) ===================================
    // one warp for the weights, which also announces the bytes of both, and one for the tokens
    const bool for_w = warp == 0;
    const bool elected = elect_one();
    int group = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int id = first_id; id < total && ok; id += n_workers) {
      int b, m0, row0, row_end, width;
      decode(id, b, m0, row0, row_end, width);
      const int half = width >> 1, my_m = m0 + (int)rank * 128, my_row = row0 + (int)rank * half;
      const bool load_w = my_m < p.N;      // nothing of this CTA's columns exists: its results are not read
      const bool big = half > 96;
      const int small = (half + 31) >> 5;
      const uint32_t bytes = (load_w ? 128 * 128 : 0) + (big ? 128 * 128 : small * 4096);
      for (int kb = kb_first; kb < kb_end; kb += depth) {
        ok = mbar_wait_warp(smem_u32(&bar_empty[group]), phase ^ 1u, &abort_flag);
        if (!ok) break;
        const int blocks = min(depth, kb_end - kb);
        if (elected) {
          const uint32_t full = mapa_u32(smem_u32(&bar_full[group]), lead);
          if (for_w) mbar_expect_tx_cluster(full, blocks * bytes);
          for (int k = 0; k < blocks; ++k) {
            const uint32_t sw = smem_base + (depth * group + k) * block_bytes, sx = sw + 128 * 128;
            const int k0 = (kb + k) * 128;
            if (for_w) {
              if (load_w) tma2_load_3d(sw, &tmW, k0, my_m, b, full);
            } else if (big) {
              tma2_load_3d(sx, &tmX, k0, my_row, GROUPED ? 0 : b, full);
            } else {
              for (int i = 0; i < small; ++i) tma2_load_3d(sx + i * 4096, &tmXsmall, k0, my_row + 32 * i, GROUPED ? 0 : b, full);
            }
          }
        }
        __syncwarp();
        if (++group == groups) { group = 0; phase ^= 1u; }
      }
    }
    // the commits that free the last groups must have arrived here before this CTA ends
    for (int g = 0; g < groups && ok; ++g)
      ok = mbar_wait_warp(smem_u32(&bar_empty[g]), g < group ? phase : phase ^ 1u, &abort_flag);
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicMax(p.status, (int)kStatusProducerTimeout);
    }
    __syncwarp();
  } else if (warp == 1) {
    // =========================== MMA issuer (leader CTA only) ================================
    if (leader) {
      // s8 x s8 -> s32, both K-major; without its N field (bits 17..22 = N / 8), which depends on the tile
      constexpr uint32_t idesc_base = (2u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(256 >> 4) << 24);
      const uint64_t wdesc0 = make_smem_desc(smem_base, 16, 1024), xdesc0 = make_smem_desc(smem_base + 128 * 128, 16, 1024);
      const bool elected = elect_one();
      int group = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int id = first_id; id < total && ok; id += n_workers) {
        int b, m0, row0, row_end, width;
        decode(id, b, m0, row0, row_end, width);
        const uint32_t idesc = idesc_base | ((uint32_t)(width >> 3) << 17);
        ok = mbar_wait_warp(smem_u32(&bar_tmem_empty[acc]), acc_phase ^ 1u, &abort_flag);
        if (!ok) break;
        tc_fence_after();
        for (int kb = kb_first; kb < kb_end; kb += depth) {
          ok = mbar_wait_warp(smem_u32(&bar_full[group]), phase, &abort_flag);
          if (!ok) break;
          tc_fence_after();
          if (elected) {
            const int blocks = min(depth, kb_end - kb);
            for (int i = 0; i < blocks; ++i) {
              const uint64_t at = (uint64_t)((depth * group + i) * (block_bytes >> 4));
#pragma unroll
              for (int k = 0; k < 4; ++k)
                tc2_mma_int8(tmem_base + acc * 256, wdesc0 + at + (uint64_t)(2 * k), xdesc0 + at + (uint64_t)(2 * k), idesc,
                             (uint32_t)(kb + i != kb_first || k != 0));
            }
            tc2_commit_to(smem_u32(&bar_empty[group]), pair_mask);
            if (kb + depth >= kb_end) tc2_commit_to(smem_u32(&bar_tmem_full[acc]), pair_mask);
          }
          __syncwarp();
          if (++group == groups) { group = 0; phase ^= 1u; }
        }
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicMax(p.status, (int)kStatusMmaTimeout);
      }
    }
    __syncwarp();
  } else {
    // =========================== epilogue (warps 2 .. 9 of both CTAs) ========================
    const int q = warp & 3;                    // TMEM lane quarter this warp may read
    const int turn = (warp - 2) >> 2;          // takes every other chunk of 32 rows
    const bool wide = sizeof(T) == 2 && p.wide;
    const uint32_t park = smem_u32(smem_raw + kInt8RingBytes) + (warp - 2) * kInt8ParkBytes;
    const float* sa = after_wait(p.sa);
    const float* sb = after_wait(p.sb);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int id = first_id; id < total; id += n_workers) {
      int b, m0, row0, row_end, width;
      decode(id, b, m0, row0, row_end, width);
      const int col = m0 + (int)rank * 128 + q * 32;
      const bool mine = col < p.N;
      const int chunks = width >> 5;
      float scale[4];                          // of the lane's columns, see int8_load_sums
#pragma unroll
      for (int h = 0; h < 4; ++h) {
        const int m = wide ? col + 8 * h + (lane >> 2) : col + lane;
        scale[h] = m < p.N ? sb[b * p.sb_b + m * p.sb_n] : 0.f;
      }
      const float* sa_b = sa + (GROUPED ? 0 : b * p.sa_b);
      T* out = p.out + (GROUPED ? 0 : (int64_t)b * p.M * p.N);
      auto row_scale = [&](int c) {
        const int row = row0 + c * 32 + lane;
        return row < row_end ? sa_b[row * p.sa_m] : 0.f;
      };
      float sa_next = row_scale(turn);         // a chunk ahead
      const bool ok = mbar_wait_warp(smem_u32(&bar_tmem_full[acc]), acc_phase, &abort_flag);
      if (!ok) {
        abort_flag = 1;
        atomicMax(p.status, (int)kStatusEpilogueTimeout);
      }
      const uint32_t t_row = tmem_base + acc * 256 + ((uint32_t)(q * 32) << 16);
      if (splits > 1) {
        const uint32_t at = (uint32_t)(q * 32 + lane) * 16;
        tc_fence_after();
        cluster_sync_all();                    // everyone's copies and instructions are done with their shared memory
        if (ok && mine) {
          for (int c = turn; c < chunks; c += 2) {
            const int owner = int8_owner(c, splits);
            if (owner == part) continue;
            uint32_t v[32];
            int8_load_sums(wide, t_row + c * 32, v);
            const uint32_t dst = mapa_u32(smem_base, 2 * owner + rank) + int8_exchange_slot(c, splits, part) * kInt8ChunkBytes + at;
#pragma unroll
            for (int i = 0; i < 8; ++i)
              asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (uint32_t)i * 2048u), "r"(v[4 * i]), "r"(v[4 * i + 1]),
                           "r"(v[4 * i + 2]), "r"(v[4 * i + 3]) : "memory");
          }
        }
        cluster_sync_all();
        if (ok && mine) {
          for (int c = turn; c < chunks; c += 2) {
            if (int8_owner(c, splits) != part) continue;
            uint32_t v[32];
            int8_load_sums(wide, t_row + c * 32, v);
            for (int o = 0; o < splits; ++o) {
              if (o == part) continue;
              const uint32_t src = smem_base + int8_exchange_slot(c, splits, o) * kInt8ChunkBytes + at;
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                uint32_t x[4];
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                             : "r"(src + (uint32_t)i * 2048u) : "memory");
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * i + j] += x[j];
              }
            }
            int8_store(p, out, wide, row_scale(c), scale, col, row0 + c * 32, min(32, row_end - row0 - c * 32), lane, park, v);
          }
        }
        break;
      }
      if (!ok) break;
      tc_fence_after();
      if (mine) {
#pragma unroll 1
        for (int c = turn; c < chunks; c += 2) {
          const float sa_lane = sa_next;
          sa_next = row_scale(c + 2);
          uint32_t v[32];
          int8_load_sums(wide, t_row + c * 32, v);
          int8_store(p, out, wide, sa_lane, scale, col, row0 + c * 32, min(32, row_end - row0 - c * 32), lane, park, v);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(mapa_u32(smem_u32(&bar_tmem_empty[acc]), lead));
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
    if constexpr (GROUPED) {                   // rows of no expert
      const int64_t step = (int64_t)gridDim.x * kInt8EpiWarps;
      for (int64_t r = (int64_t)blockIdx.x * kInt8EpiWarps + warp - 2; r < p.M; r += step) {
        if (r >= s_row[0] && r < s_row[p.B]) {
          r += (s_row[p.B] - 1 - r) / step * step;         // on to the last one of its own among the experts' rows
          continue;
        }
        int8_zero_row(p.out + r * p.N, p.N, lane, 32);
      }
    }
  }
  if (splits > 1 && (warp < 2 || warp >= 2 + kInt8EpiWarps)) {      // what the epilogue's warps meet in
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
  cluster_sync_all();          // no CTA releases shared memory or TMEM that another may still use
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512u) : "memory");
  }
}

// ---- a handful of rows ----------------------------------------------------------------------------------------------------
constexpr int kInt8RowsThreads = 256;

__device__ __forceinline__ void mma_int8(int (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// the first `n` bytes of a word
__device__ __forceinline__ uint32_t first_bytes(uint32_t w, int n) { return n >= 4 ? w : n <= 0 ? 0u : w & ((1u << (8 * n)) - 1u); }

struct Int8Rows {
  const uint8_t* x;             // codes of the tokens [B, M, ldx]
  const uint8_t* w;             // of the weights [B, N, ldw]
  int64_t ldx, x_batch, ldw, w_batch;
};

// blockIdx.x: 16 columns; blockIdx.y: matrix, or (GROUPED) the experts that have rows, one after the other.  8 * NT rows at a time; U blocks
// of 64 bytes of each row are on their way together.
//
// A sum does not depend on the order of its terms: lane (g, t) takes 16 neighbouring bytes of rows g and g + 8, words 0 and 1 of which are one
// instruction's k, 2 and 3 the next one's, of weights and tokens alike.
template <typename T, int NT, int U, bool GROUPED>
__global__ void __launch_bounds__(kInt8RowsThreads, NT == 1 ? 4 : 3)
int8_rows_kernel(const Int8Rows d, const Int8Params<T> p) {
  constexpr int kRows = 8 * NT;
  __shared__ int s_sum[8][kRows][17];
  __shared__ int s_count[8], s_expert;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * 16;
  pdl_trigger();
  pdl_wait();
  if (blockIdx.x == 0 && blockIdx.y == 0 && threadIdx.x == 0) *p.status = kStatusOk;
  int b = blockIdx.y;
  int64_t row0 = 0, row_end = p.M;
  if constexpr (GROUPED) {
    const int32_t* offsets = after_wait(p.offsets);
    unsigned have[4];
    int count = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {              // 128 experts to a warp
      const int e = warp * 128 + i * 32 + lane;
      have[i] = __ballot_sync(0xffffffffu, e < p.B && int8_offset(offsets, min(e, p.B - 1) + 1, p.M) > int8_offset(offsets, min(e, p.B - 1), p.M));
      count += __popc(have[i]);
    }
    if (lane == 0) s_count[warp] = count;
    if (threadIdx.x == 0) s_expert = -1;
    __syncthreads();
    int index = b;
    for (int w = 0; w < warp; ++w) index -= s_count[w];
    if (index >= 0 && index < count) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = __popc(have[i]);
        if (index >= 0 && index < c && lane == 0) s_expert = warp * 128 + i * 32 + (int)__fns(have[i], 0, index + 1);
        index -= c;
      }
    }
    __syncthreads();
    if (blockIdx.y == 0) {                     // rows of no expert
      const int first = int8_offset(offsets, 0, p.M), end = int8_offset(offsets, p.B, p.M), n = n0 + (threadIdx.x & 15);
      if (n < p.N)
        for (int64_t r = threadIdx.x >> 4; r < p.M; r += kInt8RowsThreads / 16)
          if (r < first || r >= end) DT<T>::st(p.out + r * p.N + n, 0.f);
    }
    b = s_expert;
    if (b < 0) return;
    row0 = int8_offset(offsets, b, p.M);
    row_end = int8_offset(offsets, b + 1, p.M);
  }
  const uint8_t* w = after_wait(d.w) + b * d.w_batch + 16 * t;
  const uint8_t* x = after_wait(d.x) + (GROUPED ? 0 : b * d.x_batch) + 16 * t;
  const float* sa = after_wait(p.sa) + (GROUPED ? 0 : b * p.sa_b);
  const float* sb = after_wait(p.sb) + b * p.sb_b;
  T* out = p.out + (GROUPED ? 0 : (int64_t)b * p.M * p.N);
  const uint8_t* w0 = w + (int64_t)min(n0 + g, p.N - 1) * d.ldw;           // columns that do not exist: computed and not stored
  const uint8_t* w1 = w + (int64_t)min(n0 + g + 8, p.N - 1) * d.ldw;
  const int blocks = (p.K + 63) >> 6;
  for (; row0 < row_end; row0 += kRows) {
    int c[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) c[j][i] = 0;
    const uint8_t* xr[NT];
    bool there[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      there[j] = row0 + 8 * j + g < row_end;
      xr[j] = x + (there[j] ? row0 + 8 * j + g : row0) * d.ldx;
    }
    for (int blk = warp; blk < blocks; blk += 8 * U) {
      uint4 a0[U], a1[U], v[U][NT];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        // bytes of this lane's sixteen that exist; those of a row's end are read with it, as pitches are multiples of 16, and masked
        const int k = (blk + 8 * u) * 64, left = p.K - k - 16 * t;
        a0[u] = a1[u] = make_uint4(0, 0, 0, 0);
        if (left > 0) {
          a0[u] = ld_written(reinterpret_cast<const uint4*>(w0 + k));
          a1[u] = ld_written(reinterpret_cast<const uint4*>(w1 + k));
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          v[u][j] = make_uint4(0, 0, 0, 0);
          if (left > 0 && there[j]) v[u][j] = ld_written(reinterpret_cast<const uint4*>(xr[j] + k));
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int left = p.K - (blk + 8 * u) * 64 - 16 * t;
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint4 z = v[u][j];
          if (left < 16) z = make_uint4(first_bytes(z.x, left), first_bytes(z.y, left - 4), first_bytes(z.z, left - 8), first_bytes(z.w, left - 12));
          mma_int8(c[j], a0[u].x, a1[u].x, a0[u].y, a1[u].y, z.x, z.y);
          mma_int8(c[j], a0[u].z, a1[u].z, a0[u].w, a1[u].w, z.z, z.w);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) s_sum[warp][8 * j + 2 * t + (i & 1)][g + 8 * (i >> 1)] = c[j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < kRows * 16; i += kInt8RowsThreads) {
      const int r = i >> 4, n = n0 + (i & 15);
      if (row0 + r < row_end && n < p.N) {
        int sum = 0;
#pragma unroll
        for (int v = 0; v < 8; ++v) sum += s_sum[v][r][i & 15];
        DT<T>::st(out + (row0 + r) * p.N + n, (float)sum * sa[(row0 + r) * p.sa_m] * sb[n * p.sb_n]);
      }
    }
    __syncthreads();
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
struct Int8Operand {
  const void* q;
  int64_t rows, ld, batch;
};

inline bool int8_map(CUtensorMap* m, const Int8Operand& o, int K, int B, uint32_t box_rows) {
  const uint64_t dims[3] = {(uint64_t)K, (uint64_t)o.rows, (uint64_t)B};
  const uint64_t strides[2] = {(uint64_t)o.ld, B > 1 ? (uint64_t)o.batch : (uint64_t)(o.ld * o.rows)};
  const uint32_t box[3] = {128, box_rows, 1};
  return encode_map(m, o.q, 3, dims, strides, box, kMapU8);
}

inline int int8_pair_smem(int experts) { return kInt8RingBytes + kInt8EpiWarps * kInt8ParkBytes + (experts > 0 ? 2 * (experts + 1) * 4 : 0); }

// Clusters of `cluster` CTAs of a kernel that run at the same time (asked once per kernel, size and device).
template <auto kern>
inline int int8_resident(int cluster, int smem) {
  static PerDevice<int> known[2 * kInt8MaxSplits + 1];
  const int dev = current_device_index();
  int n = known[cluster].get(dev);
  if (n > 0) return n;
  if (taken(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)) != cudaSuccess) return 0;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(umma_sm_count() / cluster * cluster));
  cfg.blockDim = dim3(kInt8Threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)cluster;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) {
    (void)cudaGetLastError();
    n = std::max(1, umma_sm_count() / cluster);
  }
  known[cluster].set(dev, n);
  return n;
}

// Tiles of a product that is not grouped: the least of the estimated clocks, fitted to 130 measurements of 15 products at all widths and splits
// (6 % off on average; what it picks is within 2 % of the best, but for 700 x 700 x 700, 6.5 instead of 5.8 us).  A k-block takes some 370 at
// any width that its copies bound, or its instructions, 2 per row and a tenth; a tile 1400 besides; the last tile's epilogue 28 per
// row, shared out where a cluster shares the tile, for which it meets twice and moves sums.
struct Int8Choice { int width, splits; };
template <auto kern>
inline Int8Choice int8_choose(int64_t B, int64_t M, int64_t N, int64_t K, int smem) {
  const int64_t kb = ceil_div(K, 128), NT = ceil_div(N, 256);
  Int8Choice best{256, 1};
  double least = 1e30;
  for (int width = 32; width <= 256; width += 32) {
    const int64_t MT = ceil_div(M, width);
    const int even = (int)round_up(ceil_div(M, MT), 32);           // what the tiles come to
    if (even != width) continue;
    for (int s = 1; s <= kInt8MaxSplits && s <= kb; ++s) {
      const int64_t tiles = B * MT * NT, room = std::max(1, int8_resident<kern>(2 * s, smem));
      if (s > 1 && tiles > room) break;                            // a cluster has one tile
      const double t = (double)ceil_div(tiles, room) * ((double)ceil_div(kb, s) * std::max(370.0, 2.2 * width) + 1400) + 28.0 * width / s +
                       (s > 1 ? 2900 + 31 * width : 0);
      if (t < least) { least = t; best = Int8Choice{width, s}; }
    }
  }
  return best;
}

template <typename T, bool GROUPED>
inline int launch_int8_pair(const Int8Operand& X, const Int8Operand& W, Int8Params<T> p, cudaStream_t st) {
  if (!umma_available()) return YAMOE_ERR_UNSUPPORTED;
  CUtensorMap tmW, tmX, tmXs;
  if (!int8_map(&tmW, W, p.K, p.B, 128) || !int8_map(&tmX, X, p.K, GROUPED ? 1 : p.B, 128) || !int8_map(&tmXs, X, p.K, GROUPED ? 1 : p.B, 32))
    return YAMOE_ERR_CUDA;
  constexpr auto kern = int8_pair_kernel<T, GROUPED>;
  const int most = int8_pair_smem(GROUPED ? kInt8MaxExperts : 0), smem = int8_pair_smem(GROUPED ? p.B : 0);
  p.NT = (int)ceil_div(p.N, 256);
  const int pairs = int8_resident<kern>(2, most);
  if (pairs <= 0) return YAMOE_ERR_CUDA;
  if constexpr (GROUPED) {
    // Narrow tiles, and with them more k-blocks on their way, where experts have few rows (5760 x 2880 each of 32 experts, rows dealt out at random, among
    // launches of its like, mean rows per expert and us with tiles of 64 / 128 / 256: 0.5 39 / 40 / 44; 16 84 / 83 / 89; 64 92 / 87 / 93; 128
    // 147 / 110 / 101: the border between the wider two lies between 64 and 128 rows since k-blocks come in groups, higher than it is set).
    p.width = p.M <= 8 * (int64_t)p.B ? 64 : p.M <= 32 * (int64_t)p.B ? 128 : 256;
    p.splits = 1;
    p.depth = int8_depth(p.width, GROUPED);
    p.groups = int8_groups(p.width, p.depth);
    p.block_bytes = int8_block_bytes(p.width);
    const int64_t tiles = (ceil_div(p.M, p.width) + std::min<int64_t>(p.B, p.M)) * p.NT;       // at most
    if (tiles >= (int64_t)1 << 30) return YAMOE_ERR_UNSUPPORTED;
    return launch_clusters(kern, 2, true, dim3((unsigned)(2 * std::min<int64_t>(tiles, pairs))), dim3(kInt8Threads), smem, st, tmW, tmX, tmXs, p);
  } else {
    const Int8Choice c = int8_choose<kern>(p.B, p.M, p.N, p.K, most);
    p.width = c.width;
    p.splits = c.splits;
    p.depth = int8_depth(p.width, GROUPED);
    p.groups = int8_groups(p.width, p.depth);
    p.block_bytes = int8_block_bytes(p.width);
    p.MT = (int)ceil_div(p.M, c.width);
    const int64_t tiles = (int64_t)p.B * p.MT * p.NT;
    if (tiles >= (int64_t)1 << 30) return YAMOE_ERR_UNSUPPORTED;
    const int64_t grid = c.splits > 1 ? 2 * c.splits * tiles : 2 * std::min<int64_t>(tiles, pairs);
    return launch_clusters(kern, 2 * c.splits, true, dim3((unsigned)grid), dim3(kInt8Threads), smem, st, tmW, tmX, tmXs, p);
  }
}

// U: with it four CTAs of eight rows fit an SM (1 x 5760 x 2880: 5.1 us; six blocks on their way, two CTAs, 6.7), three of up to 32 (16 rows 6.0,
// 32 rows 9.1).  Blocks that a warp has come out even with U = 2 or 3.
template <typename T, bool GROUPED>
inline int launch_int8_rows(const Int8Rows& d, const Int8Params<T>& p, cudaStream_t st) {
  const dim3 grid((unsigned)ceil_div(p.N, 16), (unsigned)(GROUPED ? std::min<int64_t>(p.B, p.M) : p.B));
  const int64_t blocks = ceil_div(ceil_div(p.K, 64), 8);
  auto kern = round_up(blocks, 2) < round_up(blocks, 3) ? int8_rows_kernel<T, 1, 2, GROUPED> : int8_rows_kernel<T, 1, 3, GROUPED>;
  if constexpr (!GROUPED) {
    if (p.M > 16) kern = int8_rows_kernel<T, 4, 1, GROUPED>;
    else if (p.M > 8) kern = int8_rows_kernel<T, 2, 2, GROUPED>;
  }
  return launch_behind(kern, grid, dim3(kInt8RowsThreads), 0, st, d, p);
}

// Few rows go by int8_rows_kernel: up to 32 (rows kernel / pairs, us: 32 x 5760 x 2880 9.1 / 9.2, 32 x 2048 x 1024 4.0 / 7.5; 64 x 5760 x 2880
// 20 / 9.4), and up to eight of experts, which share weights no more than their number (one token of four experts, 5760 x 2880 each:
// 12.9 / 16.4; sixteen rows of sixteen experts 89 / 44).
inline bool int8_few_rows(int64_t M, int64_t B, bool grouped) { return B <= 65535 && M <= (grouped ? 8 : 32); }

template <typename T>
inline int launch_int8_mm(const Int8Operand& X, const Int8Operand& W, const Int8Params<T>& p, cudaStream_t st) {
  const bool grouped = p.offsets != nullptr;
  if (int8_few_rows(p.M, p.B, grouped)) {
    const Int8Rows d{reinterpret_cast<const uint8_t*>(X.q), reinterpret_cast<const uint8_t*>(W.q), X.ld, X.batch, W.ld, W.batch};
    return grouped ? launch_int8_rows<T, true>(d, p, st) : launch_int8_rows<T, false>(d, p, st);
  }
  return grouped ? launch_int8_pair<T, true>(X, W, p, st) : launch_int8_pair<T, false>(X, W, p, st);
}

}  // namespace yb
