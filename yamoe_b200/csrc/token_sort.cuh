// Tokens sorted by expert and back, as operators of their own.
//
//   sort      row_of[t, k] = first row of expert e + number of assignments p' < p = t K + k of the same expert e
//             rows[row_of[t, k]] = hidden[t]; rows without an assignment are zero
//   combine   out[t] = sum over k of w[t, k] rows[row_of[t, k]]
//   its gradients   d_rows[r] = sum over p with row_of[p] = r of w[p] d_out[t(p)],   d_w[t, k] = <d_out[t], rows[row_of[t, k]]>
//
// Without a capacity an expert's rows follow those of the expert before it; with one, expert e has rows e C .. e C + C - 1 and
// assignments behind its first C are dropped (row_of = -1), as are ids outside [0, E).
//
// Bound by HBM for a prompt and by latency for a batch of single tokens.  A token's row is read once and written K times (a warp per
// 512-byte piece of a token, the pieces of a token side by side in the grid).  Up to kSortSmallMax assignments every CTA ranks all of them
// for itself and goes on to copy: one launch.  Above, blocks count, rank and copy in three launches; a block takes what lies before it from the
// table of all blocks' counts, so that no CTA waits for another and nothing has to be zeroed.
#pragma once
#include <algorithm>

#include "common.cuh"

namespace yb {

constexpr int kSortMaxExperts = 1024;
constexpr int kSortSmallRounds = 4;
constexpr int kSortSmallMax = 1024 * kSortSmallRounds;
constexpr int kSortThreads = 256, kSortWarps = 8, kSortRounds = 4;
constexpr int kSortPart = kSortThreads * kSortRounds;         // assignments that a block ranks at a time
constexpr int kSortMaxBlocks = 256;

struct SortArgs {
  const int64_t* indices;       // [S]
  const uint8_t* hidden;        // [T, row_bytes]
  uint8_t* rows;                // [R, row_bytes]
  int32_t* row_of;              // [S]
  int32_t* offsets;             // [E + 1] rows kept before each expert's
  int64_t T, R, row_bytes;
  int S, E, K;
  int bits;                     // of an expert's number
  int capacity;                 // -1: none
  int32_t* counts;              // [blocks, E] (large sorts)
  int parts;                    // of kSortPart assignments that a block takes
};

__device__ __forceinline__ int sort_kept(int total, int capacity) { return capacity < 0 ? total : min(total, capacity); }

// Inclusive scan of one number per thread over a CTA of whole warps; `part` has a place for each warp.
template <int WARPS>
__device__ __forceinline__ int block_scan(int v, int* part) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += up;
  }
  if (lane == 31) part[w] = v;
  __syncthreads();
  int before = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) before += i < w ? part[i] : 0;
  __syncthreads();
  return v + before;
}

// Places of the warp's items among those of their keys that it has taken before, whose numbers are `base`.  Keys are below 2^bits, or negative: no item.
// Lanes of the same key are found by a ballot per bit, which takes less than match.any where a warp has many keys (300 tokens, 4 of 128 experts each:
// 6.8 -> 6.1 us, 64 tokens among 1024 experts 5.7 -> 5.3).
__device__ __forceinline__ int take_places(int key, int bits, int32_t* base, int lane) {
  unsigned mask = __ballot_sync(0xffffffffu, key >= 0);
#pragma unroll
  for (int b = 0; b < 10; ++b)
    if (b < bits) {
      const bool set = (key >> b) & 1;
      const unsigned have = __ballot_sync(0xffffffffu, set);
      mask &= set ? have : ~have;
    }
  int place = 0;
  if (key >= 0) place = base[key] + __popc(mask & ((1u << lane) - 1u));
  __syncwarp();
  if (key >= 0 && (__ffs(mask) - 1) == lane) base[key] += __popc(mask);
  __syncwarp();
  return place;
}

// Row of the assignment that is `place`-th of expert e's, -1 behind the capacity
__device__ __forceinline__ int sorted_row(const SortArgs& a, int e, int place, const int32_t* offsets) {
  if (a.capacity < 0) return offsets[e] + place;
  return place < a.capacity ? e * a.capacity + place : -1;
}

__device__ __forceinline__ int load_expert(const int64_t* indices, int j, int end, int E) {
  if (j < end) {
    const int64_t v = indices[j];
    if (v >= 0 && v < E) return (int)v;
  }
  return -1;
}

// One 32-lane piece of a token's row to the rows of its K assignments, the first four of which are looked up while it is on its way.
template <typename P>
__device__ __forceinline__ void copy_piece(const SortArgs& a, int64_t t, int i, int n, const int32_t* row_of) {
  if (i >= n) return;
  const P v = reinterpret_cast<const P*>(a.hidden + t * a.row_bytes)[i];
  for (int k0 = 0; k0 < a.K; k0 += 4) {
    int r[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) r[k] = k0 + k < a.K ? row_of[k0 + k] : -1;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      if (r[k] >= 0) reinterpret_cast<P*>(a.rows + r[k] * a.row_bytes)[i] = v;
  }
}
template <typename P>
__device__ __forceinline__ void zero_row(const SortArgs& a, int64_t r, int n, int lane) {
  P* d = reinterpret_cast<P*>(a.rows + r * a.row_bytes);
  for (int i = lane; i < n; i += 32) d[i] = P{};
}
// Rows without an assignment, eight to a warp: lanes look, the warp writes.
constexpr int kZeroRows = 8;
template <typename P>
__device__ __forceinline__ void zero_unused(const SortArgs& a, int64_t first, int n, int lane, const int32_t* offsets) {
  const int64_t r = first + lane;
  bool unused = false;
  if (lane < kZeroRows && r < a.R) {
    if (a.capacity < 0) {
      unused = r >= offsets[a.E];
    } else {
      const int e = (int)(r / a.capacity);
      unused = r - (int64_t)e * a.capacity >= offsets[e + 1] - offsets[e];
    }
  }
  for (unsigned todo = __ballot_sync(0xffffffffu, unused); todo != 0; todo &= todo - 1) zero_row<P>(a, first + (__ffs(todo) - 1), n, lane);
}

// ---- small: everything in one launch ------------------------------------------------------------------------------------
// CTAs of 32 warps, or of eight where they are enough for the assignments and the experts (16 tokens of 2880, 4 of 128 experts each: 5.3 / 2.5 us).
constexpr size_t sort_small_smem(int warps, int S, int E) { return ((size_t)warps * E + E + 1 + S) * sizeof(int32_t); }
// With eight warps it fits what every launch may have, static arrays (a number per warp) included; with 32 a launch has to be allowed more.
constexpr size_t kAnyLaunchSmem = 48 * 1024;
constexpr int kSortFewMax = 256 * kSortSmallRounds, kSortFewExperts = 256;      // eight warps: assignments, experts
static_assert(sort_small_smem(8, kSortFewMax, kSortFewExperts) + 8 * sizeof(int) <= kAnyLaunchSmem, "");

template <typename P, int WARPS>
__global__ void __launch_bounds__(32 * WARPS)
sort_small_kernel(SortArgs a, int rounds) {
  extern __shared__ int32_t smem_i[];
  int32_t* base = smem_i;                              // [warps][E] counts, then first row of a warp's assignments of an expert
  int32_t* offsets = smem_i + WARPS * a.E;   // [E + 1]
  int32_t* row_of = offsets + a.E + 1;                 // [S]
  __shared__ int s_part[WARPS];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int used = (a.S + 32 * rounds - 1) / (32 * rounds);      // warps that have assignments
  for (int i = tid; i < used * a.E; i += 32 * WARPS) base[i] = 0;
  pdl_trigger();
  pdl_wait();
  const int64_t* indices = after_wait(a.indices);
  a.hidden = after_wait(a.hidden);
  const int first = w * 32 * rounds;
  int ex[kSortSmallRounds];
#pragma unroll
  for (int i = 0; i < kSortSmallRounds; ++i) ex[i] = i < rounds ? load_expert(indices, first + i * 32 + lane, a.S, a.E) : -1;
  __syncthreads();
  int32_t* mine = base + w * a.E;
  int place[kSortSmallRounds];
#pragma unroll
  for (int i = 0; i < kSortSmallRounds; ++i) place[i] = i < rounds ? take_places(ex[i], a.bits, mine, lane) : 0;
  __syncthreads();
  int total = 0;
  if (tid < a.E) {
#pragma unroll 4
    for (int v = 0; v < used; ++v) {
      const int c = base[v * a.E + tid];
      base[v * a.E + tid] = total;
      total += c;
    }
  }
  const int kept = sort_kept(total, a.capacity);
  const int end = block_scan<WARPS>(kept, s_part);
  if (tid == 0) offsets[0] = 0;
  if (tid < a.E) offsets[tid + 1] = end;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= a.E; e += 32 * WARPS) a.offsets[e] = offsets[e];
#pragma unroll
  for (int i = 0; i < kSortSmallRounds; ++i)
    if (i < rounds) {
      const int e = ex[i], j = first + i * 32 + lane;
      const int r = e >= 0 ? sorted_row(a, e, mine[e] + place[i], offsets) : -1;
      if (j < a.S) {
        row_of[j] = r;
        if (blockIdx.x == 0) a.row_of[j] = r;
      }
    }
  __syncthreads();
  const int n = (int)(a.row_bytes / sizeof(P));
  const unsigned chunks = (unsigned)(n + 31) / 32;
  const unsigned warps = gridDim.x * WARPS, at = blockIdx.x * WARPS + w;
  for (unsigned u = at; u < (unsigned)a.T * chunks; u += warps) {
    const unsigned t = u / chunks;
    copy_piece<P>(a, t, (int)(u - t * chunks) * 32 + lane, n, row_of + t * a.K);
  }
  for (int64_t r = at * kZeroRows; r < a.R; r += warps * kZeroRows) zero_unused<P>(a, r, n, lane, offsets);
}

// ---- large: count, rank, copy -------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(kSortThreads)
sort_count_kernel(SortArgs a) {
  extern __shared__ int32_t smem_i[];                  // [E]
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) smem_i[e] = 0;
  pdl_trigger();
  pdl_wait();
  const int64_t* indices = after_wait(a.indices);
  __syncthreads();
  const int64_t first = (int64_t)blockIdx.x * a.parts * kSortPart;
  const int64_t end = min((int64_t)a.S, first + (int64_t)a.parts * kSortPart);
  for (int64_t j = first + threadIdx.x; j < end; j += kSortThreads) {
    const int64_t v = indices[j];
    if (v >= 0 && v < a.E) atomicAdd(&smem_i[v], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < a.E; e += kSortThreads) a.counts[(size_t)blockIdx.x * a.E + e] = smem_i[e];
}

constexpr size_t sort_rank_smem(int E) { return ((size_t)kSortWarps * E + 3 * E + 1) * sizeof(int32_t); }
static_assert(sort_rank_smem(kSortMaxExperts) + kSortWarps * sizeof(int) <= kAnyLaunchSmem, "");

__global__ void __launch_bounds__(kSortThreads)
sort_rank_kernel(SortArgs a) {
  extern __shared__ int32_t smem_i[];
  int32_t* base = smem_i;                        // [warps][E]
  int32_t* next = smem_i + kSortWarps * a.E;     // [E] place of this block's next assignment of an expert
  int32_t* kept = next + a.E;                    // [E]
  int32_t* offsets = kept + a.E;                 // [E + 1]
  __shared__ int s_part[kSortWarps];
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  pdl_trigger();
  pdl_wait();
  const int64_t* indices = after_wait(a.indices);
  const int32_t* counts = after_wait(a.counts);
  for (int e = tid; e < a.E; e += kSortThreads) {
    int lower = 0, total = 0;
#pragma unroll 8
    for (int b = 0; b < (int)gridDim.x; ++b) {
      const int c = counts[(size_t)b * a.E + e];
      total += c;
      lower += b < (int)blockIdx.x ? c : 0;
    }
    next[e] = lower;
    kept[e] = sort_kept(total, a.capacity);
  }
  __syncthreads();
  // four neighbouring experts to a thread
  int v[kSortMaxExperts / kSortThreads], sum = 0;
#pragma unroll
  for (int i = 0; i < kSortMaxExperts / kSortThreads; ++i) {
    const int e = tid * (kSortMaxExperts / kSortThreads) + i;
    v[i] = e < a.E ? kept[e] : 0;
    sum += v[i];
  }
  int end = block_scan<kSortWarps>(sum, s_part) - sum;
  if (tid == 0) offsets[0] = 0;
#pragma unroll
  for (int i = 0; i < kSortMaxExperts / kSortThreads; ++i) {
    const int e = tid * (kSortMaxExperts / kSortThreads) + i;
    end += v[i];
    if (e < a.E) offsets[e + 1] = end;
  }
  __syncthreads();
  if (blockIdx.x == 0)
    for (int e = tid; e <= a.E; e += kSortThreads) a.offsets[e] = offsets[e];
  for (int part = 0; part < a.parts; ++part) {
    const int64_t part0 = ((int64_t)blockIdx.x * a.parts + part) * kSortPart;
    if (part0 >= a.S) break;
    const int first = (int)part0 + w * 32 * kSortRounds;
    for (int i = tid; i < kSortWarps * a.E; i += kSortThreads) base[i] = 0;
    int ex[kSortRounds];
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) ex[i] = load_expert(indices, first + i * 32 + lane, a.S, a.E);
    __syncthreads();
    int32_t* mine = base + w * a.E;
    int place[kSortRounds];
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) place[i] = take_places(ex[i], a.bits, mine, lane);
    __syncthreads();
    for (int e = tid; e < a.E; e += kSortThreads) {
      int run = next[e];
#pragma unroll
      for (int u = 0; u < kSortWarps; ++u) {
        const int c = base[u * a.E + e];
        base[u * a.E + e] = run;
        run += c;
      }
      next[e] = run;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kSortRounds; ++i) {
      const int e = ex[i], j = first + i * 32 + lane;
      if (j < a.S) a.row_of[j] = e >= 0 ? sorted_row(a, e, mine[e] + place[i], offsets) : -1;
    }
    __syncthreads();
  }
}

constexpr int kCopyWarps = 8;

// CTAs below `zero_ctas` zero rows without an assignment, the others copy.
template <typename P>
__global__ void __launch_bounds__(kCopyWarps * 32)
sort_copy_kernel(SortArgs a, unsigned zero_ctas) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int n = (int)(a.row_bytes / sizeof(P));
  const unsigned chunks = (unsigned)(n + 31) / 32;
  pdl_trigger();
  pdl_wait();
  a.hidden = after_wait(a.hidden);
  const int32_t* row_of = after_wait(a.row_of);
  if (blockIdx.x < zero_ctas) {
    const int64_t first = ((int64_t)blockIdx.x * kCopyWarps + w) * kZeroRows;
    if (first < a.R) zero_unused<P>(a, first, n, lane, after_wait(a.offsets));
  } else {
    const unsigned u = (blockIdx.x - zero_ctas) * kCopyWarps + w, t = u / chunks;
    if (t < a.T) copy_piece<P>(a, t, (int)(u - t * chunks) * 32 + lane, n, row_of + t * a.K);
  }
}

// Blocks of a large sort and the parts that each takes.
struct SortBlocks { int blocks, parts; };
inline SortBlocks sort_blocks(int64_t S) {
  const int64_t all = ceil_div(S, kSortPart), parts = std::max<int64_t>(1, ceil_div(all, kSortMaxBlocks));
  return SortBlocks{(int)ceil_div(all, parts), (int)parts};
}
inline size_t sort_counts_bytes(int64_t S, int E) {
  return S <= kSortSmallMax ? 0 : (size_t)sort_blocks(S).blocks * E * sizeof(int32_t);
}

template <typename P, int WARPS>
inline int launch_sort_small(const SortArgs& a, int64_t chunks, cudaStream_t st) {
  const size_t smem = sort_small_smem(WARPS, a.S, a.E);
  if constexpr (WARPS > 8) {                 // allowed once, for the largest call
    static PerDevice<size_t> allowed;        // per template instantiation and device
    YB_CUDA_OK(allow_smem(sort_small_kernel<P, WARPS>, sort_small_smem(WARPS, kSortSmallMax, kSortMaxExperts), allowed));
  }
  const int rounds = std::max(1, (int)ceil_div(a.S, 32 * WARPS));
  const int64_t work = std::max(ceil_div(a.T * chunks, WARPS), ceil_div(a.R, WARPS * kZeroRows));
  const int64_t grid = std::max<int64_t>(1, std::min<int64_t>(work, kSMs * (32 / WARPS)));
  return launch_behind(sort_small_kernel<P, WARPS>, dim3((unsigned)grid), dim3(32 * WARPS), smem, st, a, rounds);
}

template <typename P>
inline int launch_sort(SortArgs a, cudaStream_t st) {
  const int64_t n = a.row_bytes / (int64_t)sizeof(P), chunks = ceil_div(n, 32);
  if (n > 0x7fffffff || a.T * chunks > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;      // 2^31 pieces of 512 bytes are 1 TB
  if (a.S <= kSortSmallMax)
    return a.S <= kSortFewMax && a.E <= kSortFewExperts ? launch_sort_small<P, 8>(a, chunks, st) : launch_sort_small<P, 32>(a, chunks, st);
  const SortBlocks b = sort_blocks(a.S);
  a.parts = b.parts;
  int rc = launch_behind(sort_count_kernel, dim3(b.blocks), dim3(kSortThreads), a.E * sizeof(int32_t), st, a);
  if (rc) return rc;
  if ((rc = launch_behind(sort_rank_kernel, dim3(b.blocks), dim3(kSortThreads), sort_rank_smem(a.E), st, a))) return rc;
  const int64_t copy = ceil_div(a.T * chunks, kCopyWarps), zero = ceil_div(a.R, kCopyWarps * kZeroRows);
  if (copy + zero == 0) return YAMOE_OK;
  return launch_behind(sort_copy_kernel<P>, dim3((unsigned)(copy + zero)), dim3(kCopyWarps * 32), 0, st, a, (unsigned)zero);
}

// ---- combine --------------------------------------------------------------------------------------------------------------
template <typename T, typename TW>
struct CombineArgs {
  const T* rows;                // [n_rows, H]
  const int32_t* row_of;        // [T, K]; outside [0, n_rows): nothing
  const TW* weights;            // [T, K], or [T, E] with indices; null: 1
  const int64_t* indices;       // [T, K] columns of the weights; null: the slots
  int64_t Tn, n_rows;
  int H, K, E;
  __device__ __forceinline__ void behind_wait() {
    rows = after_wait(rows);
    row_of = after_wait(row_of);
    weights = after_wait(weights);
    indices = after_wait(indices);
  }
  // row of assignment p, -1 for none
  __device__ __forceinline__ int row(int64_t p) const {
    const int r = row_of[p];
    return r >= 0 && r < n_rows ? r : -1;
  }
  // weight of slot k of token t; 0 for a column that does not exist
  __device__ __forceinline__ float weight(int64_t t, int k) const {
    if (weights == nullptr) return 1.f;
    if (indices == nullptr) return DT<TW>::ld(weights + t * K + k);
    const int64_t c = indices[t * K + k];
    return c >= 0 && c < E ? DT<TW>::ld(weights + t * E + c) : 0.f;
  }
};

// VE neighbouring values: a 16-byte piece, one of four bytes (bf16 rows that are multiples of those only), or one value.  4096 tokens of 2878, 4 rows each:
// in single values 70 us, in pairs 48; of 2880, in eights, 23.
template <typename T, int VE> struct Piece {
  uint4 q;
  __device__ __forceinline__ void clear() { q = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const T* p) { q = ld_written(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&v)[VE]) const {
    const uint32_t u[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        v[j] = __uint_as_float(u[j]);
      } else {
        v[2 * j] = __uint_as_float(u[j] << 16);
        v[2 * j + 1] = __uint_as_float(u[j] & 0xffff0000u);
      }
    }
  }
  static __device__ __forceinline__ void put(T* p, const float (&v)[VE]) {
    uint32_t u[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if constexpr (sizeof(T) == 4) {
        u[j] = __float_as_uint(v[j]);
      } else {
        const __nv_bfloat162 two = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        u[j] = *reinterpret_cast<const uint32_t*>(&two);
      }
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(u[0], u[1], u[2], u[3]);
  }
};
template <> struct Piece<__nv_bfloat16, 2> {
  uint32_t q;
  __device__ __forceinline__ void clear() { q = 0; }
  __device__ __forceinline__ void load(const __nv_bfloat16* p) { q = *reinterpret_cast<const uint32_t*>(p); }
  __device__ __forceinline__ void get(float (&v)[2]) const {
    v[0] = __uint_as_float(q << 16);
    v[1] = __uint_as_float(q & 0xffff0000u);
  }
  static __device__ __forceinline__ void put(__nv_bfloat16* p, const float (&v)[2]) {
    *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(v[0], v[1]);
  }
};
template <typename T> struct Piece<T, 1> {
  T q;
  __device__ __forceinline__ void clear() { DT<T>::st(&q, 0.f); }
  __device__ __forceinline__ void load(const T* p) { q = *p; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = DT<T>::ld(&q); }
  static __device__ __forceinline__ void put(T* p, const float (&v)[1]) { DT<T>::st(p, v[0]); }
};

// One warp per 32 pieces of a token; the rows of KB slots are on their way together.  Sums in fp32 in the order of the slots.
template <typename T, typename TW, int VE, int KB>
__global__ void __launch_bounds__(kCopyWarps * 32, KB > 4 ? 4 : 5)
combine_tokens_kernel(CombineArgs<T, TW> a, T* out) {
  pdl_trigger();
  pdl_wait();
  a.behind_wait();
  const unsigned pieces = (unsigned)a.H / VE, chunks = (pieces + 31) / 32;
  const unsigned u = blockIdx.x * kCopyWarps + (threadIdx.x >> 5);
  const int64_t t = u / chunks;
  const int lane = threadIdx.x & 31;
  const unsigned i = (u - (unsigned)t * chunks) * 32 + lane;
  if (t >= a.Tn) return;
  const bool there = i < pieces;
  float acc[VE];
#pragma unroll
  for (int j = 0; j < VE; ++j) acc[j] = 0.f;
  for (int k0 = 0; k0 < a.K; k0 += KB) {
    // lane k looks up slot k0 + k for all
    const int slot = k0 + lane;
    const int mine = lane < KB && slot < a.K ? a.row(t * a.K + slot) : -1;
    Piece<T, VE> q[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const int r = __shfl_sync(0xffffffffu, mine, k);
      q[k].clear();                        // what is left out adds 0 * 0
      if (r >= 0 && there) q[k].load(a.rows + (int64_t)r * a.H + i * VE);
    }
    const float weight = mine >= 0 ? a.weight(t, slot) : 0.f;
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      const float w = __shfl_sync(0xffffffffu, weight, k);
      float v[VE];
      q[k].get(v);
#pragma unroll
      for (int j = 0; j < VE; ++j) acc[j] = fmaf(w, v[j], acc[j]);
    }
  }
  if (there) Piece<T, VE>::put(out + t * a.H + i * VE, acc);
}

// ---- gradients of the combine -----------------------------------------------------------------------------------------------
// Whose row a row is: head[r] is one of its assignments (-1: none), next[p] the one behind p (-1: none).  The rows of sort_tokens
// have one assignment or none, but row_of may name a row as often as it likes.
__global__ void __launch_bounds__(256)
link_rows_kernel(const int32_t* row_of, int64_t S, int64_t n_rows, int32_t* head, int32_t* next) {
  pdl_trigger();
  pdl_wait();
  const int64_t p = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (p >= S) return;
  const int r = after_wait(row_of)[p];
  if (r >= 0 && r < n_rows) next[p] = atomicExch(head + r, (int32_t)p);
}

// The gradient of a row that several assignments name, by one warp, for 32 pieces from i0 on of every `step`.  Atomics made the links of its assignments,
// so their order is not that of the assignments; the sum's is.  Up to 32 links are ranked; for more the warp goes through row_of, once while they fit
// its list, again and again where they do not.
constexpr int kListed = 256;
template <typename T, typename TW, int VE>
__device__ __forceinline__ void sum_shared_row(const CombineArgs<T, TW>& a, const T* d_out, T* d_rows, const int32_t* next, int64_t row, int p0,
                                            unsigned i0, unsigned step, int32_t* list) {
  const int lane = threadIdx.x & 31;
  const unsigned pieces = (unsigned)a.H / VE;
  const int64_t S = a.Tn * a.K;
  // assignments from s on into the list, at most kListed, 128 looked at together; s: the first that was not looked at
  const auto fill = [&](int64_t& s) {
    int m = 0;
    __syncwarp();
    for (; s < S && m <= kListed - 128; s += 128) {
      int32_t r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) r[u] = s + 32 * u + lane < S ? a.row_of[s + 32 * u + lane] : -1;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const unsigned hit = __ballot_sync(0xffffffffu, r[u] == row);
        if (r[u] == row) list[m + __popc(hit & ((1u << lane) - 1u))] = (int32_t)(s + 32 * u + lane);
        m += __popc(hit);
      }
    }
    __syncwarp();
    return m;
  };
  int n = 0, held = 0;                          // links of the row, lane's one
  for (int p = p0; p >= 0 && n <= 32; p = next[p]) held = n++ == lane ? p : held;
  int64_t s = S;                                // what the list does not have begins here
  if (n <= 32) {
    int place = 0;
    for (int k = 0; k < n; ++k) place += __shfl_sync(0xffffffffu, held, k) < held;
    if (lane < n) list[place] = held;
    __syncwarp();
  } else {
    s = 0;
    n = fill(s);
  }
  const bool whole = s >= S;
  for (; i0 < pieces; i0 += step) {
    const unsigned i = i0 + lane;
    float acc[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[j] = 0.f;
    if (!whole) {
      s = 0;
      n = fill(s);
    }
    while (true) {
      for (int k0 = 0; k0 < n; k0 += 4) {
        Piece<T, VE> q[4];
        float wgt[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          q[k].clear();
          wgt[k] = 0.f;
          if (k0 + k < n) {
            const int p = list[k0 + k], t = p / a.K;
            wgt[k] = a.weight(t, p - t * a.K);
            if (i < pieces) q[k].load(d_out + (int64_t)t * a.H + i * VE);
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          float v[VE];
          q[k].get(v);
#pragma unroll
          for (int j = 0; j < VE; ++j) acc[j] = fmaf(wgt[k], v[j], acc[j]);
        }
      }
      if (s >= S) break;
      n = fill(s);
    }
    if (i < pieces) Piece<T, VE>::put(d_rows + row * a.H + i * VE, acc);
  }
}

// From the tokens' side, so that d_out is read once: `wpt` warps (1, 2, 4 or 8) share a token, write the rows that only it has and add up
// the products with all its rows, each warp its pieces, the warps in order.  The first `row_ctas` CTAs look for the other rows: those
// of no assignment become zero, those of several the sum over them.  A warp looks at eight rows, or at one, or a CTA at one, where that is no more
// than a CTA per SM: few rows may have many assignments each (8192 tokens of 2880, whose 4 rows each are any of 1000: eight to a warp
// 1569 us, one 397; any of 149, one to a warp: 1602, any of 148, one to a CTA: 465).
//
// The rows of four slots are on their way together, of more one four after the other, with d_out from L1 or L2 again: eight at once leave too few warps to an SM
// (8192 tokens of 2880, 8 rows each: 143 / 155 us; 32 tokens 10.3 / 9.7).
struct RowShare {
  int rows, warps;       // that a warp looks at, that share a row
  __host__ __device__ explicit RowShare(int64_t n_rows) : rows(n_rows <= kSMs * kCopyWarps ? 1 : kZeroRows), warps(n_rows <= kSMs ? kCopyWarps : 1) {}
};
template <typename T, typename TW, int VE>
__global__ void __launch_bounds__(kCopyWarps * 32)
combine_backward_kernel(CombineArgs<T, TW> a, const T* d_out, T* d_rows, TW* d_weights, const int32_t* head, const int32_t* next,
                        int wpt, unsigned row_ctas) {
  constexpr int KB = 4;
  extern __shared__ float s_dot[];              // [warps][K], or a list per warp
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const unsigned pieces = (unsigned)a.H / VE;
  pdl_trigger();
  pdl_wait();
  a.behind_wait();
  d_out = after_wait(d_out);
  head = after_wait(head);
  next = after_wait(next);
  if (blockIdx.x < row_ctas) {
    const RowShare share(a.n_rows);
    const unsigned unit = blockIdx.x * kCopyWarps + w, step = 32 * share.warps, i0 = unit % share.warps * 32;
    const int64_t first = (int64_t)(unit / share.warps) * share.rows;
    int h = 0;
    bool nobody = false, shared = false;
    if (lane < share.rows && first + lane < a.n_rows) {
      h = head[first + lane];
      nobody = h < 0;
      shared = h >= 0 && next[h] >= 0;
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, nobody); todo != 0; todo &= todo - 1) {
      const float zero[VE] = {};
      for (unsigned i = i0 + lane; i < pieces; i += step) Piece<T, VE>::put(d_rows + (first + __ffs(todo) - 1) * a.H + i * VE, zero);
    }
    for (unsigned todo = __ballot_sync(0xffffffffu, shared); todo != 0; todo &= todo - 1) {
      const int l = __ffs(todo) - 1;
      sum_shared_row<T, TW, VE>(a, d_out, d_rows, next, first + l, __shfl_sync(0xffffffffu, h, l), i0, step,
                                reinterpret_cast<int32_t*>(s_dot) + w * kListed);
    }
    return;
  }
  const int64_t t = (int64_t)(blockIdx.x - row_ctas) * (kCopyWarps / wpt) + w / wpt;
  const int part = w % wpt;
  for (int k0 = 0; k0 < a.K && t < a.Tn; k0 += KB) {
    int r[KB];
    float wgt[KB], dot[KB];
    bool own[KB];
#pragma unroll
    for (int k = 0; k < KB; ++k) {
      r[k] = k0 + k < a.K ? a.row(t * a.K + k0 + k) : -1;
      wgt[k] = r[k] >= 0 ? a.weight(t, k0 + k) : 0.f;
      dot[k] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < KB; ++k)
      own[k] = d_rows != nullptr && r[k] >= 0 && head[r[k]] == (int)(t * a.K + k0 + k) && next[t * a.K + k0 + k] < 0;
    for (unsigned i = lane + 32 * part; i < pieces; i += 32 * wpt) {
      Piece<T, VE> g, q[KB];
      g.load(d_out + t * a.H + i * VE);
      if (d_weights != nullptr) {
#pragma unroll
        for (int k = 0; k < KB; ++k)
          if (r[k] >= 0) q[k].load(a.rows + (int64_t)r[k] * a.H + i * VE);
      }
      float d[VE];
      g.get(d);
#pragma unroll
      for (int k = 0; k < KB; ++k) {
        if (r[k] < 0) continue;
        float v[VE];
        if (d_weights != nullptr) {
          q[k].get(v);
#pragma unroll
          for (int j = 0; j < VE; ++j) dot[k] = fmaf(d[j], v[j], dot[k]);
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) v[j] = wgt[k] * d[j];
        if (own[k]) Piece<T, VE>::put(d_rows + (int64_t)r[k] * a.H + i * VE, v);
      }
    }
    if (d_weights != nullptr) {
#pragma unroll
      for (int k = 0; k < KB; ++k) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) dot[k] += __shfl_xor_sync(0xffffffffu, dot[k], o);
        if (lane == 0 && k0 + k < a.K) s_dot[w * a.K + k0 + k] = dot[k];
      }
    }
  }
  if (d_weights == nullptr) return;
  __syncthreads();
  if (part != 0 || t >= a.Tn) return;
  // of each slot the sum over the token's warps, by its first one
  for (int k = lane; k < a.K; k += 32) {
    float sum = 0.f;
    for (int o = 0; o < wpt; ++o) sum += s_dot[(w + o) * a.K + k];
    s_dot[w * a.K + k] = sum;
    if (a.indices == nullptr) DT<TW>::st(d_weights + t * a.K + k, sum);
  }
  if (a.indices == nullptr) return;
  __syncwarp();
  for (int c = lane; c < a.E; c += 32) {        // every column of the dense weights, also where two slots have the same
    float sum = 0.f;
    for (int k = 0; k < a.K; ++k)
      if (a.indices[t * a.K + k] == c) sum += s_dot[w * a.K + k];
    DT<TW>::st(d_weights + t * a.E + c, sum);
  }
}

template <typename T, typename TW, int VE>
inline int launch_combine_tokens_ve(const CombineArgs<T, TW>& a, T* out, cudaStream_t st) {
  const int64_t chunks = a.Tn * ceil_div(a.H / VE, 32), ctas = ceil_div(chunks, kCopyWarps);
  if (chunks > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
  auto kern = a.K <= 4 ? combine_tokens_kernel<T, TW, VE, 4> : combine_tokens_kernel<T, TW, VE, 8>;
  return launch_behind(kern, dim3((unsigned)ctas), dim3(kCopyWarps * 32), 0, st, a, out);
}

template <typename T, typename TW, int VE>
inline int launch_combine_backward_ve(const CombineArgs<T, TW>& a, const T* d_out, T* d_rows, TW* d_weights, int32_t* head, int32_t* next,
                                      cudaStream_t st) {
  const RowShare share(a.n_rows);
  // at least 32 warps per SM, while each has pieces of the token
  int wpt = 1;
  while (wpt < kCopyWarps && a.Tn * wpt < kSMs * 32 && a.H / VE > 32 * wpt) wpt *= 2;
  const int64_t S = a.Tn * a.K, token = ceil_div(a.Tn * wpt, kCopyWarps), row = d_rows == nullptr ? 0 : ceil_div(a.n_rows * share.warps, kCopyWarps * share.rows);
  if (token + row > 0x7fffffff || ceil_div(S, 256) > 0x7fffffff) return YAMOE_ERR_UNSUPPORTED;
  if (d_rows != nullptr && a.n_rows > 0) {
    YB_CUDA_OK(cudaMemsetAsync(head, 0xFF, (size_t)a.n_rows * sizeof(int32_t), st));
    const int rc = S == 0 ? YAMOE_OK
                          : launch_behind(link_rows_kernel, dim3((unsigned)ceil_div(S, 256)), dim3(256), 0, st, a.row_of, S, a.n_rows, head, next);
    if (rc) return rc;
  }
  if (token + row == 0) return YAMOE_OK;
  auto kern = combine_backward_kernel<T, TW, VE>;
  return launch_behind(kern, dim3((unsigned)(token + row)), dim3(kCopyWarps * 32), kCopyWarps * std::max(a.K, kListed) * sizeof(float), st, a, d_out, d_rows,
                       d_weights, (const int32_t*)head, (const int32_t*)next, wpt, (unsigned)row);
}

inline bool pieces_of(uintptr_t bytes, int64_t row_bytes, std::initializer_list<const void*> at) {
  uintptr_t bits = (uintptr_t)row_bytes;
  for (const void* p : at) bits |= reinterpret_cast<uintptr_t>(p);
  return (bits & (bytes - 1)) == 0;
}

}  // namespace yb
