// Host code around launches and what kernels and launchers share of index arithmetic, with the runtime's calls replaced: runs without a GPU.  One argument names the check.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <atomic>
#include <chrono>
#include <condition_variable>
#include <cstdio>
#include <cstring>
#include <mutex>
#include <thread>

namespace fake {

std::mutex mutex;
std::condition_variable changed;
int largest = 0, calls = 0;           // the attribute as the runtime holds it
bool meet = false;                    // a call waits, but not for long, until another one is over
cudaError_t result = cudaSuccess, last = cudaSuccess;

template <typename Kern>
cudaError_t set_attribute(Kern, cudaFuncAttribute, int value) {
  std::unique_lock<std::mutex> lock(mutex);
  if (result != cudaSuccess) return last = result;
  largest = value;
  const int mine = ++calls;
  changed.notify_all();
  if (meet && mine == 1) changed.wait_for(lock, std::chrono::milliseconds(500), [] { return calls > 1; });
  return cudaSuccess;
}
cudaError_t get_device(int* device) {
  *device = 0;
  return cudaSuccess;
}
template <typename... K, typename... A>
cudaError_t launch(const cudaLaunchConfig_t*, void (*)(K...), A&&...) {
  return result == cudaSuccess ? cudaSuccess : last = result;
}
cudaError_t memset_async(void*, int, size_t, cudaStream_t) { return result == cudaSuccess ? cudaSuccess : last = result; }
cudaError_t get_last_error() {
  const cudaError_t e = last;
  last = cudaSuccess;
  return e;
}

}  // namespace fake

#define cudaFuncSetAttribute fake::set_attribute
#define cudaGetDevice fake::get_device
#define cudaLaunchKernelEx fake::launch
#define cudaMemsetAsync fake::memset_async
#define cudaGetLastError fake::get_last_error
#include "int8_gemm.cuh"
#include "int8_quant.cuh"
#include "token_sort.cuh"

using namespace yb;

static void kernel(int) {}

#define EXPECT(x)                                        \
  do {                                                   \
    if (!(x)) {                                          \
      std::printf("line %d: %s\n", __LINE__, #x);        \
      return 1;                                          \
    }                                                    \
  } while (0)

// Two threads ask for different sizes at the same time, whoever comes first: what the kernel may have is at least what is remembered of it.
static int two_threads(size_t first, size_t second) {
  static PerDevice<size_t> allowed[2];
  PerDevice<size_t>& mine = allowed[first > second];
  fake::largest = fake::calls = 0;
  fake::meet = true;
  std::thread a([&] { (void)allow_smem(kernel, first, mine); });
  {
    std::unique_lock<std::mutex> lock(fake::mutex);
    fake::changed.wait_for(lock, std::chrono::seconds(5), [] { return fake::calls > 0; });
  }
  std::thread b([&] { (void)allow_smem(kernel, second, mine); });
  a.join();
  b.join();
  EXPECT(fake::largest == 150000);
  EXPECT(mine.get(0) == 150000);
  // and a later call of either size finds it done
  const int before = fake::calls;
  EXPECT(allow_smem(kernel, 150000, mine) == 0 && allow_smem(kernel, 100000, mine) == 0 && fake::calls == before);
  return 0;
}

static int memset_status() {
  YB_CUDA_OK(cudaMemsetAsync(nullptr, 0, 4, nullptr));
  return YAMOE_OK;
}

// A call that was refused leaves nothing for the check behind the next launch.
static int refused() {
  static PerDevice<size_t> allowed;
  const auto calls = {+[] { return launch_behind(kernel, dim3(1), dim3(32), 0, nullptr, 0); },
                      +[] { return launch_clusters(kernel, 2, true, dim3(2), dim3(32), 0, nullptr, 0); },
                      +[] { return launch_pdl_opt(true, kernel, dim3(1), dim3(32), 0, nullptr, 0) == cudaSuccess ? (int)YAMOE_OK : (int)YAMOE_ERR_CUDA; },
                      +[] { return launch_early(kernel, dim3(1), dim3(32), nullptr, 0) == cudaSuccess ? (int)YAMOE_OK : (int)YAMOE_ERR_CUDA; },
                      +[] { return allow_smem(kernel, 100000, allowed) == cudaSuccess ? (int)YAMOE_OK : (int)YAMOE_ERR_CUDA; }, +[] { return memset_status(); }};
  for (const auto& call : calls) {
    fake::result = cudaErrorInvalidValue;
    EXPECT(call() == YAMOE_ERR_CUDA);
    fake::result = cudaSuccess;
    EXPECT(fake::last == cudaSuccess);
    EXPECT(call() == YAMOE_OK);
  }
  return 0;
}

// An expert's rows are cut into tiles of one height, a multiple of 32 and no more than asked for; none is left without rows.
static int tiles() {
  for (int width = 32; width <= 256; width += 32)
    for (int rows = 1; rows < 200000; rows += rows < 3000 ? 1 : 997) {
      const int n = (rows + width - 1) / width, step = int8_tile_rows(rows, n);
      EXPECT(step % 32 == 0 && step <= width);
      EXPECT((int64_t)(n - 1) * step < rows && rows <= (int64_t)n * step);
    }
  return 0;
}

// The parts of a strip are multiples of 16 rows; none is left without rows, but for an x without any.
static int parts() {
  EXPECT(int8_parts(0) == 1 && int8_part_rows(0, 1) == 0);
  for (int64_t M = 1; M < ((int64_t)1 << 31); M += M < 5000 ? 1 : M / 7) {
    const int n = int8_parts(M);
    const int64_t rows = int8_part_rows(M, n);
    EXPECT(n >= 1 && n <= kInt8MaxParts && rows % 16 == 0);
    EXPECT((n - 1) * rows < M && M <= n * rows);
  }
  return 0;
}

// What the product's ring holds at every width, in groups of one or two k-blocks; the exchange of a shared tile in its place; all of a CTA's shared memory.
static int ring() {
  for (int grouped = 0; grouped < 2; ++grouped)
    for (int width = 32; width <= 256; width += 32) {
      const int depth = int8_depth(width, grouped), groups = int8_groups(width, depth), half = width / 2;
      EXPECT(groups >= 3 && groups <= kInt8MaxGroups && groups * depth * int8_block_bytes(width) <= kInt8Ring);
      // tokens come by boxes of 32 rows, or by one of 128
      EXPECT(128 * 128 + (half > 96 ? 4 : (half + 31) / 32) * 4096 <= int8_block_bytes(width));
    }
  for (int splits = 2; splits <= kInt8MaxSplits; ++splits)
    for (int c = 0; c < 8; ++c)
      for (int part = 0; part < splits; ++part) {
        EXPECT(int8_exchange_slot(c, splits, part) < int8_exchange_slots(splits));
        for (int d = 0; d < c; ++d)           // no slot of an owner serves twice
          for (int other = 0; other < splits; ++other)
            EXPECT(int8_owner(c, splits) != int8_owner(d, splits) || int8_exchange_slot(c, splits, part) != int8_exchange_slot(d, splits, other));
      }
  EXPECT(int8_pair_smem(kInt8MaxExperts) + 512 <= 227 * 1024);
  // every sort of up to kSortSmallMax assignments, statics included
  EXPECT(sort_small_smem(32, kSortSmallMax, kSortMaxExperts) + 32 * sizeof(int) <= 227 * 1024);
  return 0;
}

int main(int, char** argv) {
  if (!std::strcmp(argv[1], "tiles")) return tiles();
  if (!std::strcmp(argv[1], "parts")) return parts();
  if (!std::strcmp(argv[1], "ring")) return ring();
  if (!std::strcmp(argv[1], "refused")) return refused();
  if (!std::strcmp(argv[1], "threads")) return two_threads(150000, 100000) || two_threads(100000, 150000);
  return 2;
}
