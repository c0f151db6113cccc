// What the kernels of attention behind a shared prefix have in common: the batch, its units of work and where their parts of the result go.
#pragma once

#include "common.cuh"

#include <atomic>

namespace ms {
namespace prefix {

constexpr float kLog2e = 1.4426950408889634f;

struct Batch {
  const int* block_tables;
  int table_stride;
  const int* positions;
  const int* query_start;
  const int* context_lens;
  const int* group_start;
  const int* prefix_lens;
  int page_size, n_q, n_kv, n_requests, n_groups, n_tokens, n_pages;
};

// Whatever the index arrays hold, no kernel reads or writes outside the tensors: tokens, requests and keys are cut to what there is, and a page that is not
// in the pool reads as zeros.

// Results of parts: o [items][count][d] and lse [items][count] in base 2, item = token * n_q + head; a unit's split i of a prefix is part i, of a
// request's own keys part prefix + i.
struct Parts {
  float* o;
  float* lse;
  int prefix, own, count;
};

// The pool's row of a key in the page `page`, one behind the last (which a tensor map fills with zeros) for a page that is not there.
__device__ __forceinline__ int pool_row_of(const Batch& b, int page, int kv_head, int key) {
  return (unsigned)page < (unsigned)b.n_pages ? (page * b.n_kv + kv_head) * b.page_size + key % b.page_size : b.n_pages * b.n_kv * b.page_size;
}

struct Unit {
  int token, token_end;      // the rows' tokens
  int key, key_end;          // all of the unit's keys
  const int* table;
  int split, splits, part;
};

// The last group that starts at or before the request; called by whole warps, whose lanes look at 32 groups at once.
__device__ __forceinline__ int group_of(const Batch& b, int request) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int first = 1; first < b.n_groups; first += 32) {
    const bool starts = first + lane < b.n_groups && b.group_start[first + lane] <= request;
    const int here = __popc(__ballot_sync(0xffffffffu, starts));
    before += here;
    if (here < 32) break;
  }
  return before;
}

__device__ __forceinline__ int within(int value, int most) { return min(max(value, 0), most); }
// The keys of a request: never more than its table's row has room for.
__device__ __forceinline__ int keys_of(const Batch& b, int request) { return (int)min((long long)b.context_lens[request], (long long)b.table_stride * b.page_size); }

__device__ __forceinline__ Unit prefix_unit(const Batch& b, int group, int split, const Parts& parts) {
  Unit u;
  const int first = within(b.group_start[group], b.n_requests), last = within(b.group_start[group + 1], b.n_requests);
  u.token = within(b.query_start[first], b.n_tokens), u.token_end = max(u.token, within(b.query_start[last], b.n_tokens));
  // (never more than its first request, whose table is read, has)
  u.key = 0, u.key_end = first < b.n_requests ? max(0, min(b.prefix_lens[group], keys_of(b, first))) : 0;
  u.table = b.block_tables + (size_t)first * b.table_stride;
  u.split = split, u.splits = parts.prefix, u.part = split;
  return u;
}

__device__ __forceinline__ Unit own_unit(const Batch& b, int request, int split, const Parts& parts) {
  Unit u;
  u.token = within(b.query_start[request], b.n_tokens), u.token_end = max(u.token, within(b.query_start[request + 1], b.n_tokens));
  u.key = max(0, b.prefix_lens[group_of(b, request)]), u.key_end = max(u.key, keys_of(b, request));
  u.table = b.block_tables + (size_t)request * b.table_stride;
  u.split = split, u.splits = parts.own, u.part = parts.prefix + split;
  return u;
}

// Units in the order: every group's prefix with its splits, then every request's own keys with theirs.
__device__ __forceinline__ Unit unit_of(const Batch& b, int index, const Parts& parts) {
  const int shared = b.n_groups * parts.prefix;
  if (index < shared) return prefix_unit(b, index / parts.prefix, index % parts.prefix, parts);
  return own_unit(b, (index - shared) / parts.own, (index - shared) % parts.own, parts);
}

// Own keys run beside the prefixes of the same call, the kernel before theirs on the stream, which lets them start after its own wait for what came before.
// What follows them waits for them alone: one of their blocks, the last, ends no sooner than the prefixes' kernel has.  (Where every block did,
// each kept its place on the multiprocessor until then.)
__device__ __forceinline__ bool last_block() {
  return blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1 && blockIdx.z == gridDim.z - 1;
}

// All of a multiprocessor's memory as shared memory while the kernel runs there, so that blocks of the prefixes and of the own keys, which need not wait for one
// another, find room side by side.
// Asked of the driver once for each kernel and device (`asked`: a bit for each of the first 64 devices; asking twice does no harm).
template <typename... Params>
cudaError_t share_multiprocessor(void (*kernel)(Params...), std::atomic<unsigned long long>& asked) {
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  const unsigned long long bit = device < 64 ? 1ull << device : 0;
  if (e != cudaSuccess || (asked.load(std::memory_order_relaxed) & bit)) return e;
  e = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel), cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
  if (e == cudaSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// Launches of the parts on the tensor cores (attention_prefix_tcgen05.cu: prefixes; attention_prefix_own.cu: own keys; attention_prefix_mma.cu: both) and whether they take
// the sizes; `beside`: see there.
bool prefix_tcgen05_takes(int d, int group, int page_size, long long pool_rows);
int launch_prefix_tcgen05(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int d, int n_tokens,
                          int max_group_tokens, float scale, float softcap, int* error_flag, cudaStream_t stream);
bool own_tma_takes(int d, int page_size, long long pool_rows);
int launch_own_tma(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int d, int most_tokens,
                   float scale, float softcap, bool all_units, bool beside, int* error_flag, cudaStream_t stream);
bool prefix_mma_takes(int d);
int launch_part_mma(const void* q, const void* k_pool, const void* v_pool, const Batch& b, const Parts& parts, int d, int most_tokens, float scale,
                    float softcap, bool own, bool beside, cudaStream_t stream);

}  // namespace prefix
}  // namespace ms
