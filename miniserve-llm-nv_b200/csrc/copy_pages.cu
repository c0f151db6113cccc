// Copies of whole cache pages: pool[run][destination[i]] = pool[run][source[i]] for every run (layer) of a pool, several pools at once.
//
// A page of a pool [runs, pages, ...] is one contiguous piece of memory, so this is a copy of n x runs x pools pieces of a few to a few
// hundred kilobytes; it reads every source and writes every destination once, and memory bandwidth bounds it (one page: the launch).  The
// page numbers are host-side bookkeeping: they travel as kernel arguments, with the launch, so that no copy to the device precedes it and a
// captured launch keeps them.  The caller has checked that no destination is a source or is named twice, so the blocks need no order.
// 256 pages of 32 KB in 16 layers of keys and of values: 81.4 us, 6.6 TB/s read and written together, the rate of a plain copy; one page in 28 layers, replayed: 1.7 us.
#include "common.cuh"

#include <string.h>

namespace ms {
namespace pages {

constexpr int kPools = 8;               // pools of one launch
constexpr int kThreads = 256, kDeep = 4;            // every thread has kDeep units on their way

struct Pool {
  unsigned char* base;
  long long page_bytes, run_bytes;      // of one page, and of one run's pages
  int first;                            // runs of the pools before this one
  int unit;                             // bytes that a thread moves at once: what the address and a page's size are multiples of
};

template <int N>
struct Copies {
  Pool pool[kPools];
  int pools;
  int source[N], destination[N];
};

template <typename Unit>
__device__ __forceinline__ void copy_piece(const unsigned char* from, unsigned char* to, long long bytes, long long first, long long step) {
  const Unit* src = reinterpret_cast<const Unit*>(from);
  Unit* dst = reinterpret_cast<Unit*>(to);
  const long long units = bytes / (long long)sizeof(Unit);
  for (long long base = first; base < units; base += step * kDeep) {
    Unit held[kDeep];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      if (base + j * kThreads < units) held[j] = src[base + j * kThreads];
#pragma unroll
    for (int j = 0; j < kDeep; ++j)
      if (base + j * kThreads < units) dst[base + j * kThreads] = held[j];
  }
}

// Block (piece of a page, copy, run of a pool).
template <int N>
__global__ void __launch_bounds__(kThreads) copy_pages_kernel(const __grid_constant__ Copies<N> copies) {
  grid_dependency_wait();
  grid_dependency_launch();
  int p = 0;
  while (p + 1 < copies.pools && (int)blockIdx.z >= copies.pool[p + 1].first) ++p;
  const Pool& pool = copies.pool[p];
  unsigned char* run = pool.base + (long long)((int)blockIdx.z - pool.first) * pool.run_bytes;
  const unsigned char* from = run + copies.source[blockIdx.y] * pool.page_bytes;
  unsigned char* to = run + copies.destination[blockIdx.y] * pool.page_bytes;
  const long long first = (long long)blockIdx.x * (kThreads * kDeep) + threadIdx.x, step = (long long)gridDim.x * kThreads;
  if (pool.unit == 16) copy_piece<uint4>(from, to, pool.page_bytes, first, step);
  else if (pool.unit == 8) copy_piece<uint2>(from, to, pool.page_bytes, first, step);
  else if (pool.unit == 4) copy_piece<unsigned>(from, to, pool.page_bytes, first, step);
  else copy_piece<unsigned short>(from, to, pool.page_bytes, first, step);
}

template <int N>
int launch_copies(const Pool* pool, int pools, int runs, long long pieces, const int* sources, const int* destinations, int n, cudaStream_t stream) {
  Copies<N> copies;
  memcpy(copies.pool, pool, sizeof(Pool) * pools);
  copies.pools = pools;
  memcpy(copies.source, sources, sizeof(int) * n);
  memcpy(copies.destination, destinations, sizeof(int) * n);
  ms::launch(copy_pages_kernel<N>, dim3((unsigned)pieces, n, runs), dim3(kThreads), 0, stream, copies);
  MS_CHECK_LAUNCH("copy_pages");
  return 0;
}

}  // namespace pages
}  // namespace ms

using namespace ms;

// described: for each pool its address, runs, pages and bytes of a page (64-bit integers, on the host); sources, destinations [n]: page
// numbers, on the host, the same for every pool.  Every destination is written once and is no source.
MS_EXPORT int ms_copy_pages(const long long* described, int n_pools, const int* sources, const int* destinations, int n, cudaStream_t stream) {
  using namespace ms::pages;
  if (n == 0 || n_pools == 0) return 0;
  MS_REQUIRE(n > 0 && n_pools > 0 && n_pools <= kPools, "copy_pages: %d copies in %d pools (1..%d)", n, n_pools, kPools);
  Pool pool[kPools];
  long long runs = 0, pieces = 1;
  for (int p = 0; p < n_pools; ++p) {
    const long long* d = described + 4 * p;
    MS_REQUIRE(d[1] > 0 && d[2] > 0 && d[3] > 0, "copy_pages: pool %d has %lld runs of %lld pages of %lld bytes", p, d[1], d[2], d[3]);
    for (int i = 0; i < n; ++i)
      MS_REQUIRE(sources[i] >= 0 && sources[i] < d[2] && destinations[i] >= 0 && destinations[i] < d[2],
                 "copy_pages: page %d to %d of a pool of %lld", sources[i], destinations[i], d[2]);
    int unit = 16;
    while (unit > 2 && ((unsigned long long)d[0] % unit || d[3] % unit)) unit /= 2;
    MS_REQUIRE((unsigned long long)d[0] % unit == 0 && d[3] % unit == 0, "copy_pages: pages of %lld bytes at an odd address or of odd size", d[3]);
    pool[p] = Pool{reinterpret_cast<unsigned char*>(d[0]), d[3], d[2] * d[3], (int)runs, unit};
    runs += d[1];
    const long long of_pool = (d[3] / unit + kThreads * kDeep - 1) / (kThreads * kDeep);
    if (of_pool > pieces) pieces = of_pool;
  }
  MS_REQUIRE(runs <= 65535, "copy_pages: %lld runs in one call are too many", runs);
  if (pieces > 1024) pieces = 1024;      // (a block then walks over its page)
  constexpr int few = 32, many = 900;
  for (int at = 0; at < n; at += many) {
    const int part = n - at < many ? n - at : many;
    const int code = part <= few ? launch_copies<few>(pool, n_pools, (int)runs, pieces, sources + at, destinations + at, part, stream)
                                 : launch_copies<many>(pool, n_pools, (int)runs, pieces, sources + at, destinations + at, part, stream);
    if (code != 0) return code;
  }
  return 0;
}
