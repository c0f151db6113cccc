// Attention of a batch whose requests share the pages of a long prefix.
//
// The requests stand in groups of consecutive ones; the first `prefix` tokens of a group's requests lie in the same pages.  A token at position p
// sees the keys 0 .. p of its request.  With s_t = scale q . k_t (under a soft cap c tanh(s / c)) the softmax over all t is joined from parts:
//   part i:   m_i = max s_t,  l_i = sum 2^(s_t' - m_i'),  o_i = sum 2^(s_t' - m_i') v_t / l_i,  lse_i = m_i' + log2 l_i      (s' = s log2 e)
//   whole:    o = sum_i 2^(lse_i - M) o_i / (sum_i 2^(lse_i - M) + 2^(sink' - M))
// The keys before the prefix's end are parts of the group: all its tokens and all heads of a key head are rows against one read of the keys and
// values.  What lies behind the prefix are parts of each request.  Both kinds are cut further along the keys where the rows are few.
//
// This file holds the kernel for any head size and type in float32 arithmetic, and the join.
#include "attention_prefix.cuh"

namespace ms {
namespace prefix {

// Thread block: sixteen rows of one unit (a group's prefix or a request's own keys) and key head, over its share of the keys; a warp holds four rows, a
// lane one key of a tile of 32 for the scores and every 32nd column for the values.
constexpr int kRows = 16, kKeys = 32, kThreads = 128;

__device__ __forceinline__ float4 load_four(const float* p) { return *reinterpret_cast<const float4*>(p); }
__device__ __forceinline__ float4 load_four(const __nv_bfloat16* p) {
  const uint2 two = *reinterpret_cast<const uint2*>(p);
  return make_float4(__uint_as_float(two.x << 16), __uint_as_float(two.x & 0xffff0000u), __uint_as_float(two.y << 16), __uint_as_float(two.y & 0xffff0000u));
}

// COLUMNS: columns of the values to a lane, ceil(d / 32) or more.
template <typename T, int COLUMNS>
__global__ void __launch_bounds__(kThreads) general_kernel(const T* __restrict__ q, const T* __restrict__ k_pool, const T* __restrict__ v_pool, Batch b,
                                                           int d, float scale, float softcap, Parts parts) {
  grid_dependency_wait();
  grid_dependency_launch();
  extern __shared__ __align__(16) float smem[];
  const int dp = (d + 3) / 4 * 4, ks_stride = dp + 4;
  const bool wide = d % 4 == 0 && ((reinterpret_cast<uintptr_t>(k_pool) | reinterpret_cast<uintptr_t>(v_pool)) & 15) == 0;
  float* q_s = smem;                                 // [kRows][dp]
  float* k_s = q_s + kRows * dp;                     // [kKeys][dp + 4]
  float* v_s = k_s + kKeys * ks_stride;              // [kKeys][dp]
  float* p_s = v_s + kKeys * dp;                     // [kRows][kKeys]
  const Unit u = unit_of(b, (int)blockIdx.z, parts);
  const int kv_head = blockIdx.y, group = b.n_q / b.n_kv;
  const int rows_total = (u.token_end - u.token) * group, row0 = (int)blockIdx.x * kRows;
  if (row0 >= rows_total) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = (u.key_end - u.key + kKeys - 1) / kKeys, share = (tiles + u.splits - 1) / u.splits;
  const int tile_lo = u.split * share, tile_hi = min(tiles, tile_lo + share);
  for (int i = threadIdx.x; i < kRows * dp; i += kThreads) {
    const int r = i / dp, c = i % dp, row = row0 + r;
    float v = 0.f;
    if (row < rows_total && c < d) v = to_float(q[((size_t)(u.token + row / group) * b.n_q + kv_head * group + row % group) * d + c]);
    q_s[i] = v;
  }
  int limit[4];                                      // the last position that the row sees
  float top[4], sum[4], acc[4][COLUMNS];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = row0 + warp * 4 + r;
    limit[r] = row < rows_total ? b.positions[u.token + row / group] : -1;
    top[r] = -INFINITY, sum[r] = 0.f;
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c) acc[r][c] = 0.f;
  }
  for (int tile = tile_lo; tile < tile_hi; ++tile) {
    const int key0 = u.key + tile * kKeys, live = min(kKeys, u.key_end - key0);
    __syncthreads();
    {
      // four threads to a key, four numbers at a time where the head size allows it; keys behind the last are zeros: whatever their memory holds is not read
      const int r = (int)threadIdx.x / 4, key = key0 + r;
      const int page = r < live ? u.table[key / b.page_size] : -1;
      const bool there = (unsigned)page < (unsigned)b.n_pages;
      const size_t at = there ? (((size_t)page * b.n_kv + kv_head) * b.page_size + key % b.page_size) * d : 0;
      if (wide) {
#pragma unroll 4
        for (int c = (int)threadIdx.x % 4 * 4; c < d; c += 16) {
          float4 k = make_float4(0.f, 0.f, 0.f, 0.f), v = k;
          if (there) k = load_four(k_pool + at + c), v = load_four(v_pool + at + c);
          *reinterpret_cast<float4*>(k_s + r * ks_stride + c) = k;
          *reinterpret_cast<float4*>(v_s + r * dp + c) = v;
        }
      } else {
        for (int c = (int)threadIdx.x % 4; c < dp; c += 4) {
          k_s[r * ks_stride + c] = there && c < d ? to_float(k_pool[at + c]) : 0.f;
          v_s[r * dp + c] = there && c < d ? to_float(v_pool[at + c]) : 0.f;
        }
      }
    }
    __syncthreads();
    float s[4] = {};
    for (int c = 0; c < dp; c += 4) {
      const float4 k = *reinterpret_cast<const float4*>(k_s + lane * ks_stride + c);
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float4 a = *reinterpret_cast<const float4*>(q_s + (warp * 4 + r) * dp + c);
        s[r] = fmaf(a.x, k.x, fmaf(a.y, k.y, fmaf(a.z, k.z, fmaf(a.w, k.w, s[r]))));
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      float x = s[r] * scale;
      if (softcap > 0.f) x = softcap * tanhf(x / softcap);
      x *= kLog2e;
      if (lane >= live || key0 + lane > limit[r]) x = -INFINITY;
      const float updated = fmaxf(top[r], warp_max(x));
      const float base = updated == -INFINITY ? 0.f : updated;
      const float factor = exp2f(top[r] - base);     // (0 where nothing was seen)
      const float p = exp2f(x - base);
      sum[r] = sum[r] * factor + p;                  // of this lane's keys
      top[r] = updated;
      p_s[(warp * 4 + r) * kKeys + lane] = p;
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c) acc[r][c] *= factor;
    }
    __syncwarp();
    for (int key = 0; key < live; ++key) {
      float p[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) p[r] = p_s[(warp * 4 + r) * kKeys + key];
#pragma unroll
      for (int c = 0; c < COLUMNS; ++c)
        if (lane + 32 * c < d) {
          const float v = v_s[key * dp + lane + 32 * c];
#pragma unroll
          for (int r = 0; r < 4; ++r)
            if (p[r] != 0.f) acc[r][c] = fmaf(p[r], v, acc[r][c]);           // (a value that no row sees may be anything)
        }
    }
    __syncwarp();
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = row0 + warp * 4 + r;
    const float total = warp_sum(sum[r]);
    if (row >= rows_total) continue;
    const size_t item = (size_t)(u.token + row / group) * b.n_q + kv_head * group + row % group, at = item * parts.count + u.part;
    const float inv = total == 0.f ? 0.f : 1.f / total;          // (NaN stays NaN)
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
      if (lane + 32 * c < d) parts.o[at * d + lane + 32 * c] = acc[r][c] * inv;
    if (lane == 0) parts.lse[at] = total == 0.f ? -INFINITY : top[r] + log2f(total);
  }
}

// Warp: one (token, head).  A part without keys has weight 0 and its numbers are not read.
template <typename T, int COLUMNS>
__global__ void __launch_bounds__(128) join_kernel(Parts parts, int d, int n_q, const int* __restrict__ tokens, const float* __restrict__ sink,
                                                  int has_sink, T* __restrict__ out) {
  grid_dependency_wait();
  grid_dependency_launch();
  const int item = (int)blockIdx.x * 4 + (int)(threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (item / n_q >= *tokens) return;                // (rows behind the last request stay as they are)
  const float* lse = parts.lse + (size_t)item * parts.count;
  const float* o = parts.o + (size_t)item * parts.count * d;
  float top = -INFINITY;
  for (int i = lane; i < parts.count; i += 32) top = fmaxf(top, __ldcg(lse + i));
  top = warp_max(top);
  float sink2 = -INFINITY;
  if (has_sink) sink2 = sink != nullptr ? sink[item % n_q] * kLog2e : 0.f;
  top = fmaxf(top, sink2);
  const float base = top == -INFINITY ? 0.f : top;
  float total = exp2f(sink2 - base), acc[COLUMNS] = {};
  for (int i = 0; i < parts.count; ++i) {
    const float w = exp2f(__ldcg(lse + i) - base);
    if (w == 0.f) continue;
    total += w;
#pragma unroll
    for (int c = 0; c < COLUMNS; ++c)
      if (lane + 32 * c < d) acc[c] = fmaf(w, __ldcg(o + (size_t)i * d + lane + 32 * c), acc[c]);
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
#pragma unroll
  for (int c = 0; c < COLUMNS; ++c)
    if (lane + 32 * c < d) out[(size_t)item * d + lane + 32 * c] = from_float<T>(acc[c] * inv);
}

// Block: one (token, head) of a head size that is a multiple of four.  Groups of d / 4 lanes take a part each, four numbers a lane, kDeep parts on their way
// before their weights are known; the groups' sums meet in shared memory, in a fixed order.  One trip to the second-level cache for up to
// 4 x 32 / (d / 4) x kDeep parts (a warp that took part after part waited for each: 19.5 us for 1,024 rows of 19 parts, 5.3 so).
constexpr int kMostParts = 128, kDeep = 5, kMostGroups = 64;
template <typename T>
__global__ void __launch_bounds__(128) join_wide_kernel(Parts parts, int d, int n_q, const int* __restrict__ tokens, const float* __restrict__ sink,
                                                       int has_sink, T* __restrict__ out) {
  grid_dependency_wait();
  grid_dependency_launch();
  extern __shared__ __align__(16) float sums[];      // [groups][d]
  __shared__ float weights[kMostParts];
  const int item = blockIdx.x;
  if (item / n_q >= *tokens) return;                // (rows behind the last request stay as they are)
  const int lanes = d / 4, groups = min(kMostGroups, 128 / lanes), group = (int)threadIdx.x / lanes, lane = (int)threadIdx.x % lanes;
  const float4* o = reinterpret_cast<const float4*>(parts.o + (size_t)item * parts.count * d) + lane;
  float4 held[kDeep];
#pragma unroll
  for (int j = 0; j < kDeep; ++j) {
    const int i = group + j * groups;
    if (group < groups && i < parts.count) held[j] = __ldcg(o + (size_t)i * lanes);
  }
  // every warp forms all weights, so that all have the sum
  const float* lse = parts.lse + (size_t)item * parts.count;
  const int l = threadIdx.x & 31;
  float mine[kMostParts / 32], top = -INFINITY;
#pragma unroll
  for (int j = 0; j < kMostParts / 32; ++j) {
    mine[j] = l + 32 * j < parts.count ? __ldcg(lse + l + 32 * j) : -INFINITY;
    top = fmaxf(top, mine[j]);
  }
  float sink2 = -INFINITY;
  if (has_sink) sink2 = sink != nullptr ? sink[item % n_q] * kLog2e : 0.f;
  top = fmaxf(warp_max(top), sink2);
  const float base = top == -INFINITY ? 0.f : top;
  float total = 0.f;
#pragma unroll
  for (int j = 0; j < kMostParts / 32; ++j) {
    mine[j] = exp2f(mine[j] - base);
    total += mine[j];
    if (threadIdx.x < 32) weights[l + 32 * j] = mine[j];
  }
  total = warp_sum(total) + exp2f(sink2 - base);
  __syncthreads();
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int first = group; group < groups && first < parts.count; first += kDeep * groups) {
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int i = first + j * groups;
      const float w = i < parts.count ? weights[i] : 0.f;
      if (w != 0.f) {                              // (a part without keys: its numbers are not read as such)
        const float4 v = held[j];
        acc.x = fmaf(w, v.x, acc.x), acc.y = fmaf(w, v.y, acc.y), acc.z = fmaf(w, v.z, acc.z), acc.w = fmaf(w, v.w, acc.w);
      }
    }
#pragma unroll
    for (int j = 0; j < kDeep; ++j) {
      const int i = first + (kDeep + j) * groups;
      if (i < parts.count) held[j] = __ldcg(o + (size_t)i * lanes);
    }
  }
  if (group < groups) reinterpret_cast<float4*>(sums)[group * lanes + lane] = acc;
  __syncthreads();
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int c = threadIdx.x; c < d; c += 128) {
    float sum = 0.f;
    for (int g = 0; g < groups; ++g) sum += sums[g * d + c];
    out[(size_t)item * d + c] = from_float<T>(sum * inv);
  }
}

template <typename T, int COLUMNS>
int launch_join(const Parts& parts, int d, int n_q, const int* tokens, int items, const float* sink_scores, int sink, void* out, cudaStream_t stream) {
  if (d % 4 == 0 && parts.count <= kMostParts) {
    const int groups = 128 / (d / 4) < kMostGroups ? 128 / (d / 4) : kMostGroups;
    ms::launch(join_wide_kernel<T>, dim3(items), dim3(128), (size_t)groups * d * sizeof(float), stream, parts, d, n_q, tokens, sink_scores, sink, (T*)out);
  } else {
    ms::launch(join_kernel<T, COLUMNS>, dim3((items + 3) / 4), dim3(128), 0, stream, parts, d, n_q, tokens, sink_scores, sink, (T*)out);
  }
  MS_CHECK_LAUNCH("prefix attention (join)");
  return 0;
}

template <typename T, int COLUMNS>
int launch_general(const void* q, const void* k_pool, const void* v_pool, const Batch& b, int d, float scale, float softcap, const Parts& parts, dim3 grid,
                   cudaStream_t stream) {
  const int dp = (d + 3) / 4 * 4;
  const size_t smem = (size_t)(kRows * dp + kKeys * (2 * dp + 4) + kRows * kKeys) * sizeof(float);
  MS_REQUIRE(allow_shared(general_kernel<T, COLUMNS>, smem) == cudaSuccess, "prefix attention: cannot reserve %zu bytes of shared memory", smem);
  ms::launch(general_kernel<T, COLUMNS>, grid, dim3(kThreads), smem, stream, (const T*)q, (const T*)k_pool, (const T*)v_pool, b, d, scale, softcap, parts);
  MS_CHECK_LAUNCH("prefix attention");
  return 0;
}

template <typename T, int COLUMNS>
int attend(const void* q, const void* k_pool, const void* v_pool, const Batch& b, int d, float scale, float softcap, const Parts& parts, dim3 grid, int items,
           const float* sink_scores, int sink, void* out, cudaStream_t stream) {
  const int code = launch_general<T, COLUMNS>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, stream);
  return code != 0 ? code : launch_join<T, COLUMNS>(parts, d, b.n_q, b.query_start + b.n_requests, items, sink_scores, sink, out, stream);
}

template <typename T>
int attend_any(const void* q, const void* k_pool, const void* v_pool, const Batch& b, int d, float scale, float softcap, const Parts& parts, dim3 grid,
               int items, const float* sink_scores, int sink, void* out, cudaStream_t stream) {
  if (d <= 64) return attend<T, 2>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, items, sink_scores, sink, out, stream);
  if (d <= 128) return attend<T, 4>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, items, sink_scores, sink, out, stream);
  if (d <= 256) return attend<T, 8>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, items, sink_scores, sink, out, stream);
  return attend<T, 16>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, items, sink_scores, sink, out, stream);
}

}  // namespace prefix
}  // namespace ms

using namespace ms;



// Whether all units, prefixes too, go through the kernel of the own keys: where a group's rows are those of one warp.  (Two requests of two heads to a
// key head behind 512 keys: 8.0 us a call so, 10.1 with the prefixes on tcgen05.)
static bool one_kernel(int tensor, int d, int n_q, int n_kv, int page_size, int max_group_tokens) {
  return tensor && (long long)max_group_tokens * (n_q / n_kv) <= 16 && prefix::own_tma_takes(d, page_size, 0);
}

// Into how many parts, 1 to 64, a unit's keys are cut.  own: the units are n_requests requests with up to max_query_len tokens and max_suffix_len keys of their own,
// else n_groups groups and their prefixes.  tensor: on the tensor cores.
static int parts_of(int own, int tensor, int d, int n_q, int n_kv, int page_size, int n_groups, int max_group_tokens, int max_prefix_len,
                    int n_requests, int max_query_len, int max_suffix_len) {
  const int units = own ? n_requests : n_groups, most_tokens = own ? max_query_len : max_group_tokens, most_keys = own ? max_suffix_len : max_prefix_len;
  if (units < 1 || n_kv < 1 || most_keys < 1 || most_tokens < 1) return 1;
  const int group = n_q / n_kv;
  const long long rows = (long long)most_tokens * group;
  int parts = 1, most = 64;
  if (!own && one_kernel(tensor, d, n_q, n_kv, page_size, max_group_tokens)) own = 1;          // (the same kernel)
  if (tensor && !own && prefix::prefix_tcgen05_takes(d, group, page_size, 0)) {
    // Blocks with a multiprocessor each for the prefixes: 6.5 us to start and to end, then 1 us a key tile (1.3 a row and key tile where there are two row
    // tiles).  The multiprocessors that they leave, and a twelfth of theirs, work at the own keys meanwhile, which alone take the time of their
    // reads at 5.5 TB/s (half of the most that they can be), 7 us at least; when the prefixes are done, all do.
    const int tokens = 128 / group;
    const long long row_tiles = (most_tokens + tokens - 1) / tokens, base = (long long)units * n_kv * ((row_tiles + 1) / 2), tiles = (most_keys + 127) / 128;
    const double bytes = 0.5 * 4.0 * n_requests * (double)max_suffix_len * n_kv * d, own_us = bytes / 5.5e6 > 7.0 ? bytes / 5.5e6 : 7.0;
    double least = 1e30;
    for (int s = 1; s <= most && s <= tiles; ++s) {
      const long long blocks = base * s, rounds = (blocks + 147) / 148;
      const double us = (double)rounds * (6.5 + (row_tiles > 1 ? 2.6 : 1.0) * (double)((tiles + s - 1) / s));
      const double left = blocks < 148 ? (double)(148 - blocks) / 148.0 + 1.0 / 12.0 : 1.0 / 12.0;
      const double rest = own_us - us * left, cost = us + (rest > 0.0 ? rest : 0.0) + 0.1 * s;
      if (cost < least) least = cost, parts = s;
    }
    return parts;
  }
  // small blocks: so many that they fill the multiprocessors, a part keeping some tiles
  const bool few = rows <= 16, ring = tensor && own && prefix::own_tma_takes(d, page_size, 0);
  const long long base = (long long)units * n_kv * (ring ? (rows <= 32 ? 1 : (rows + 63) / 64) : tensor ? (few ? 1 : (rows + 63) / 64) : (rows + 15) / 16);
  const long long slots = 148 * (ring ? (few ? 12 : 6) : tensor ? (few ? 5 : 2) : 3);
  const int keep = ring ? (few ? 48 : 128) : tensor ? (few ? 64 : 128) : 64;
  parts = (int)((slots + base - 1) / base);
  if (most > (most_keys + keep - 1) / keep) most = (most_keys + keep - 1) / keep;
  if (parts > most) parts = most;
  return parts < 1 ? 1 : parts;
}

// What ms_prefix_attention is to be given for these sizes: whether the tensor-core kernels run (bfloat16 tensors at multiples of 16 bytes, a head size that
// they take) times 65,536, the parts of a prefix (none where no group has one) times 256, the parts of a request's own keys.
MS_EXPORT int ms_prefix_attention_plan(int dtype, int aligned, int d, int n_q, int n_kv, int page_size, int n_groups, int max_group_tokens, int max_prefix_len,
                                       int n_requests, int max_query_len, int max_suffix_len) {
  const int tensor = dtype == MS_BF16 && aligned && prefix::prefix_mma_takes(d) ? 1 : 0;
  const int shared = max_prefix_len > 0 ? parts_of(0, tensor, d, n_q, n_kv, page_size, n_groups, max_group_tokens, max_prefix_len, n_requests, max_query_len, max_suffix_len) : 0;
  const int own = parts_of(1, tensor, d, n_q, n_kv, page_size, n_groups, max_group_tokens, max_prefix_len, n_requests, max_query_len, max_suffix_len);
  return tensor << 16 | shared << 8 | own;
}

// q, out [n_tokens, n_q, d] of type dtype; pools [pages, n_kv, page_size, d] of one layer; block_tables [requests, table_stride]; positions [n_tokens];
// query_start [requests + 1]; context_lens [requests] (lengths after this step's tokens); group_start [groups + 1] (requests; the first is 0, the last
// the number of requests); prefix_lens [groups].  part_o [n_tokens n_q (prefix_parts + own_parts) d] and part_lse (without d) are float32 scratch.
// max_query_len, max_group_tokens: upper bounds of a request's and a group's tokens.  sink != 0: one more term of the denominator, e^0 or
// e^sink_scores[head].  tensor: the tensor-core kernels are to run (bfloat16, addresses that are multiples of 16 bytes, sizes that they take).
MS_EXPORT int ms_prefix_attention(int tensor, const void* q, int dtype, const void* k_pool, const void* v_pool, int n_pages, const int* block_tables, int table_stride,
                                  const int* positions, const int* query_start, const int* context_lens, const int* group_start,
                                  const int* prefix_lens, int page_size, int n_q, int n_kv, int d, float scale, float softcap, int sink,
                                  const float* sink_scores, void* out, float* part_o, float* part_lse, int prefix_parts, int own_parts, int n_requests,
                                  int n_groups, int n_tokens, int max_query_len, int max_group_tokens, int* error_flag, cudaStream_t stream) {
  using namespace ms::prefix;
  if (n_tokens == 0) return 0;
  MS_REQUIRE(n_kv > 0 && n_q % n_kv == 0, "prefix attention: %d query heads are not a multiple of %d key/value heads", n_q, n_kv);
  MS_REQUIRE(d >= 1 && d <= 512 && page_size > 0, "prefix attention: head size %d, page size %d", d, page_size);
  MS_REQUIRE(prefix_parts >= 0 && own_parts >= 1 && part_o && part_lse, "prefix attention: %d + %d parts need scratch", prefix_parts, own_parts);
  const long long units = (long long)n_groups * prefix_parts + (long long)n_requests * own_parts;
  const int group = n_q / n_kv, most = max_query_len > max_group_tokens ? max_query_len : max_group_tokens;
  const long long tiles = ((long long)most * group + kRows - 1) / kRows;
  MS_REQUIRE(units <= 65535 && n_kv <= 65535 && tiles <= 2147483647LL, "prefix attention: grid %lld x %d x %lld exceeds the launch limits", tiles, n_kv, units);
  const Batch b{block_tables, table_stride, positions, query_start, context_lens, group_start, prefix_lens, page_size, n_q, n_kv, n_requests, n_groups, n_tokens, n_pages};
  const Parts parts{part_o, part_lse, prefix_parts, own_parts, prefix_parts + own_parts};
  const dim3 grid((unsigned)tiles, n_kv, (unsigned)units);
  const int items = n_tokens * n_q;
  if (tensor) {
    MS_REQUIRE(dtype == MS_BF16 && prefix_mma_takes(d) && error_flag != nullptr, "prefix attention: head size %d is not the tensor-core kernels'", d);
    int code = 0;
    const bool shared = prefix_parts > 0 && n_groups > 0, pool_fits = (long long)n_pages * n_kv * page_size < 2147483648LL;
    const bool together = shared && pool_fits && one_kernel(tensor, d, n_q, n_kv, page_size, max_group_tokens);
    if (together)
      code = launch_own_tma(q, k_pool, v_pool, n_pages, b, parts, d, max_group_tokens, scale, softcap, true, false, error_flag, stream);
    else if (shared && prefix_tcgen05_takes(d, group, page_size, (long long)n_pages * n_kv * page_size))
      code = launch_prefix_tcgen05(q, k_pool, v_pool, n_pages, b, parts, d, n_tokens, max_group_tokens, scale, softcap, error_flag, stream);
    else if (shared)
      code = launch_part_mma(q, k_pool, v_pool, b, parts, d, max_group_tokens, scale, softcap, false, false, stream);
    if (code == 0 && !together && own_tma_takes(d, page_size, (long long)n_pages * n_kv * page_size))
      code = launch_own_tma(q, k_pool, v_pool, n_pages, b, parts, d, max_query_len, scale, softcap, false, shared, error_flag, stream);
    else if (code == 0 && !together)
      code = launch_part_mma(q, k_pool, v_pool, b, parts, d, max_query_len, scale, softcap, true, shared, stream);
    if (code != 0) return code;
    if (d <= 64) return launch_join<__nv_bfloat16, 2>(parts, d, n_q, query_start + n_requests, items, sink_scores, sink, out, stream);
    return launch_join<__nv_bfloat16, 4>(parts, d, n_q, query_start + n_requests, items, sink_scores, sink, out, stream);
  }
  if (dtype == MS_F32) return attend_any<float>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, items, sink_scores, sink, out, stream);
  return attend_any<__nv_bfloat16>(q, k_pool, v_pool, b, d, scale, softcap, parts, grid, items, sink_scores, sink, out, stream);
}
