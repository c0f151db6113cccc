// Every request's own keys behind a shared prefix, on mma.sync with TMA-fed tiles (bfloat16, head sizes 64 and 128, pages of a multiple of eight tokens).
//
// Thread block: W warps of 16 rows (token, query head of the key head's group) of one request and key head, over its share of the keys.  Tiles of keys
// and values come page by page through TMA, in boxes of 8 rows and more with the 128-byte swizzle: one instruction a box where gathering the same rows
// took a warp 32 asynchronous copies and their addresses a tile.  S = Q K^T, running maximum and sum in float32, O += P V with P rounded to
// bfloat16 (V's type: a weight off by at most 2^-8 of itself).  Keys behind the context's end are masked, their rows of V zeroed.
//
// A step of single tokens has one warp's rows a request.  What such a warp waits for is itself - the fixed latencies of its own instructions, with one warp
// on a scheduler - so blocks are small: one warp, two tiles of 8 KB, no shared memory for the rows, and twelve blocks share a multiprocessor.  The reads
// bound it: 134 MB of 64 requests' own keys take about 27 us (5 TB/s), most of them while the prefixes' products run.  Waits are bounded: one that runs out sets the error flag, the copies in flight land, and the block returns.
#include "attention_prefix.cuh"
#include "mma_common.cuh"
#include "tcgen05.cuh"

namespace ms {
namespace prefix {
namespace own {

using namespace ms::t5;

template <int W> constexpr int kStages = W == 1 ? 2 : 4;
template <int D, int W> constexpr int kKeys = (D == 128 ? 16 : 32) * (W == 1 ? 1 : 2);          // of a tile

template <int D, int W>
constexpr size_t smem_bytes() { return (size_t)kStages<W> * 2 * kKeys<D, W> * D * 2 + 1024; }

__device__ __forceinline__ float fast_exp2(float x) {       // ex2.approx: relative error about 2^-22, -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Address of the 16-byte chunk c (0 .. D / 8 - 1) of row r of a tile of `rows` rows in shared memory: column blocks of 128 bytes, swizzled.
__device__ __forceinline__ const unsigned char* chunk(const unsigned char* tile, int rows, int r, int c) {
  return tile + (size_t)(c >> 3) * (rows * 128) + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

// all_units: the groups' prefixes too, in the order of unit_of.
template <int D, int W>
__global__ void __launch_bounds__(W * 32)
own_kernel(const __nv_bfloat16* __restrict__ q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Batch b, Parts parts,
           int box_rows, float scale_log2, float cap_log2, int all_units, int beside, int* __restrict__ error_flag) {
  constexpr int ROWS = 16 * W, THREADS = 32 * W, CHUNKS = D / 8, BN = kKeys<D, W>, TILE = BN * D * 2, STAGES = kStages<W>;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  auto k_tile = [&](int s) { return smem + (size_t)s * 2 * TILE; };
  auto v_tile = [&](int s) { return smem + (size_t)s * 2 * TILE + TILE; };
  __shared__ uint64_t full[STAGES];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 0) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) mbar_init(&full[s], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  if (!beside) grid_dependency_wait();
  grid_dependency_launch();

  const int kv_head = blockIdx.y, group = b.n_q / b.n_kv;
  const Unit u = all_units ? unit_of(b, (int)blockIdx.z, parts) : own_unit(b, (int)blockIdx.z / parts.own, (int)blockIdx.z % parts.own, parts);
  const int rows_total = (u.token_end - u.token) * group, row0 = (int)blockIdx.x * ROWS;
  // tiles from a multiple of BN on, so that a box never leaves its page; keys before the first own one are masked
  const int base = u.key / BN * BN, tiles = u.key_end > u.key ? (u.key_end - base + BN - 1) / BN : 0, share = (tiles + u.splits - 1) / u.splits;
  const int tile_lo = u.split * share, n_tiles = row0 < rows_total ? max(0, min(tiles, tile_lo + share) - tile_lo) : 0;
  const int key_lo = base + tile_lo * BN;

  auto send = [&](int j) {                           // warp 0: tile j of this block's share
    const int key0 = key_lo + j * BN, live = min(BN / box_rows, (u.key_end - key0 + box_rows - 1) / box_rows), stage = j % STAGES;
    if (lane == 0) mbar_expect_tx(&full[stage], (unsigned)(live * box_rows * D * 2 * 2));
    __syncwarp();
    for (int i = lane; i < live * (D / 64) * 2; i += 32) {
      const int values = i & 1, db = (i >> 1) % (D / 64), box = (i >> 1) / (D / 64), key = key0 + box * box_rows;
      const int pool_row = pool_row_of(b, u.table[key / b.page_size], kv_head, key);
      unsigned char* to = (values ? v_tile(stage) : k_tile(stage)) + (size_t)db * (BN * 128) + (size_t)(box * box_rows) * 128;
      tma_load_2d(to, values ? &map_v : &map_k, &full[stage], db * 64, pool_row);
    }
  };
  if (warp == 0)
    for (int j = 0; j < min(STAGES - 1, n_tiles); ++j) send(j);

  const int quad_row = lane >> 2, quad_col = lane & 3;
  int limit[2];                                      // the last key that the row sees
  unsigned q_frag[D / 16][4];
  float acc_o[D / 8][4], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
  if (n_tiles > 0) {
    // the rows straight into the fragments of the products: rows lane / 4 and 8 behind, columns 2 (lane % 4) and 8 behind of every sixteen
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int row = row0 + warp * 16 + quad_row + half * 8;
      const bool valid = row < rows_total;
      limit[half] = valid ? min(b.positions[u.token + row / group], u.key_end - 1) : -1;
      const unsigned* src = reinterpret_cast<const unsigned*>(q) + (valid ? ((size_t)(u.token + row / group) * b.n_q + kv_head * group + row % group) * (D / 2) + quad_col : 0);
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        q_frag[kk][half] = valid ? src[kk * 8] : 0u;
        q_frag[kk][half + 2] = valid ? src[kk * 8 + 4] : 0u;
      }
    }
  }
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc_o[n][e] = 0.f;

  bool ok = true;
  for (int j = 0; j < n_tiles; ++j) {
    const int stage = j % STAGES;
    // (the stage of tile j - 1 is free: all warps are past it)
    if (W > 1) __syncthreads(); else __syncwarp();
    if (warp == 0 && j + STAGES - 1 < n_tiles) send(j + STAGES - 1);
    ok = mbar_wait(&full[stage], (unsigned)(j / STAGES) & 1, error_flag, 51);
    if (W > 1) ok = __syncthreads_and(ok); else ok = __all_sync(0xffffffffu, ok);
    if (!ok) {
      if (warp == 0) let_copies_land(full, STAGES, min(n_tiles, j + STAGES), error_flag);
      break;
    }
    const unsigned char* ks = k_tile(stage);
    unsigned char* vs = v_tile(stage);
    const int key0 = key_lo + j * BN;
    if (key0 + BN > u.key_end) {
      // the last tile: rows of V behind the context are zeros (a weight of 0 times whatever lies there would not be 0)
      const int live = u.key_end - key0;
      for (int i = tid; i < (BN - live) * CHUNKS; i += THREADS)
        *reinterpret_cast<uint4*>(const_cast<unsigned char*>(chunk(vs, BN, live + i / CHUNKS, i % CHUNKS))) = make_uint4(0, 0, 0, 0);
      if (W > 1) __syncthreads(); else __syncwarp();
    }

    float acc_s[BN / 8][4];
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc_s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
      for (int np = 0; np < BN / 16; ++np) {
        unsigned f[4];
        ldmatrix_x4(f, chunk(ks, BN, np * 16 + (lane & 7) + (lane >> 4) * 8, kk * 2 + ((lane >> 3) & 1)));
        mma_bf16(acc_s[2 * np], q_frag[kk], f[0], f[1]);
        mma_bf16(acc_s[2 * np + 1], q_frag[kk], f[2], f[3]);
      }
    if (cap_log2 > 0.f) {
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc_s[n][e] = capped_score(acc_s[n][e], cap_log2);
    }
    if (key0 < u.key || !__all_sync(0xffffffffu, key0 + BN - 1 <= min(limit[0], limit[1]))) {
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = key0 + n * 8 + quad_col * 2 + (e & 1);
          if (key > limit[e >> 1] || key < u.key) acc_s[n][e] = -INFINITY;
        }
    }
    float from[2], sum[2] = {0.f, 0.f}, corr[2];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float v = acc_s[0][2 * half];
#pragma unroll
      for (int n = 0; n < BN / 8; ++n) v = fmaxf(v, fmaxf(acc_s[n][2 * half], acc_s[n][2 * half + 1]));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
      const float updated = fmaxf(m_run[half], v);
      from[half] = updated == -INFINITY ? 0.f : updated * scale_log2;
      corr[half] = exp2f(m_run[half] * scale_log2 - from[half]);      // m == -inf gives 0
      m_run[half] = updated;
    }
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc_s[n][e] = fast_exp2(fmaf(acc_s[n][e], scale_log2, -from[e >> 1]));
        sum[e >> 1] += acc_s[n][e];
      }
#pragma unroll
    for (int half = 0; half < 2; ++half) l_run[half] = l_run[half] * corr[half] + sum[half];
    if (!__all_sync(0xffffffffu, corr[0] == 1.f && corr[1] == 1.f)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n) {
        acc_o[n][0] *= corr[0], acc_o[n][1] *= corr[0];
        acc_o[n][2] *= corr[1], acc_o[n][3] *= corr[1];
      }
    }
#pragma unroll
    for (int kp = 0; kp < BN / 16; ++kp) {
      unsigned p[4];
      p[0] = pack_bf16(acc_s[2 * kp][0], acc_s[2 * kp][1]);
      p[1] = pack_bf16(acc_s[2 * kp][2], acc_s[2 * kp][3]);
      p[2] = pack_bf16(acc_s[2 * kp + 1][0], acc_s[2 * kp + 1][1]);
      p[3] = pack_bf16(acc_s[2 * kp + 1][2], acc_s[2 * kp + 1][3]);
#pragma unroll
      for (int np = 0; np < D / 16; ++np) {
        unsigned f[4];
        ldmatrix_x4_trans(f, chunk(vs, BN, kp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, np * 2 + (lane >> 4)));
        mma_bf16(acc_o[2 * np], p, f[0], f[1]);
        mma_bf16(acc_o[2 * np + 1], p, f[2], f[3]);
      }
    }
  }

  if (ok && row0 < rows_total) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float l = l_run[half];
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      const int row = row0 + warp * 16 + quad_row + half * 8;
      if (row >= rows_total) continue;
      const size_t at = ((size_t)(u.token + row / group) * b.n_q + kv_head * group + row % group) * parts.count + u.part;
      const float inv = l == 0.f ? 0.f : 1.f / l;          // (NaN stays NaN)
      if (n_tiles > 0) {
        float* dst = parts.o + at * D;
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
          *reinterpret_cast<float2*>(dst + n * 8 + quad_col * 2) = make_float2(acc_o[n][2 * half] * inv, acc_o[n][2 * half + 1] * inv);
      }
      if (quad_col == 0) parts.lse[at] = l == 0.f ? -INFINITY : m_run[half] * scale_log2 + log2f(l);
    }
  }
  if (beside && last_block()) grid_dependency_wait();
}

// Rows of a page that one box takes, 0 where these pages are not taken: a power of two up to a tile that divides the page.
static int box_rows_of(int page_size, int keys) {
  int rows = keys;
  while (rows >= 8 && page_size % rows != 0) rows /= 2;
  return rows >= 8 ? rows : 0;
}

template <int D, int W>
int launch(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int most_tokens, float scale,
           float softcap, bool all_units, bool beside, int* error_flag, cudaStream_t stream) {
  EncodeTiled fn = encode_tiled();
  MS_REQUIRE(fn != nullptr, "prefix attention: the driver offers no tensor maps");
  const int box_rows = box_rows_of(b.page_size, kKeys<D, W>);
  CUtensorMap map_k, map_v;
  const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)n_pages * b.n_kv * b.page_size};
  const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
  const cuuint32_t box[2] = {64, (cuuint32_t)box_rows}, elem[2] = {1, 1};
  auto encode = [&](CUtensorMap* map, const void* base) {
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  MS_REQUIRE(encode(&map_k, k_pool) && encode(&map_v, v_pool), "prefix attention: tensor map of the pools failed");
  auto kernel = own_kernel<D, W>;
  const size_t smem = smem_bytes<D, W>();
  static std::atomic<unsigned long long> asked{0};
  MS_REQUIRE(allow_shared(kernel, smem) == cudaSuccess && share_multiprocessor(kernel, asked) == cudaSuccess, "prefix attention: cannot reserve %zu bytes of shared memory", smem);
  const long long tiles = ((long long)most_tokens * (b.n_q / b.n_kv) + 16 * W - 1) / (16 * W), units = (long long)b.n_requests * parts.own + (all_units ? (long long)b.n_groups * parts.prefix : 0);
  MS_REQUIRE(tiles <= 2147483647LL && units <= 65535 && b.n_kv <= 65535, "prefix attention: grid %lld x %d x %lld exceeds the launch limits", tiles, b.n_kv, units);
  const float scale_log2 = (softcap > 0.f ? softcap : scale) * kLog2e, twice = softcap > 0.f ? 2.f * scale / softcap * kLog2e : 0.f;
  const cudaError_t e = ms::launch(kernel, dim3((unsigned)tiles, b.n_kv, (unsigned)units), dim3(W * 32), smem, stream, (const __nv_bfloat16*)q, map_k, map_v, b,
                                   parts, box_rows, scale_log2, twice, all_units ? 1 : 0, beside ? 1 : 0, error_flag);
  if (e != cudaSuccess) MS_FAIL("prefix attention: launch failed: %s", cudaGetErrorString(e));
  return 0;
}

template <int D>
int launch_rows(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int most_tokens, float scale,
                float softcap, bool all_units, bool beside, int* error_flag, cudaStream_t stream) {
  const long long rows = (long long)most_tokens * (b.n_q / b.n_kv);
  if (rows <= 16) return launch<D, 1>(q, k_pool, v_pool, n_pages, b, parts, most_tokens, scale, softcap, all_units, beside, error_flag, stream);
  if (rows <= 32) return launch<D, 2>(q, k_pool, v_pool, n_pages, b, parts, most_tokens, scale, softcap, all_units, beside, error_flag, stream);
  return launch<D, 4>(q, k_pool, v_pool, n_pages, b, parts, most_tokens, scale, softcap, all_units, beside, error_flag, stream);
}

}  // namespace own

bool own_tma_takes(int d, int page_size, long long pool_rows) {
  return (d == 128 || d == 64) && own::box_rows_of(page_size, 16) > 0 && pool_rows < 2147483648LL;
}

int launch_own_tma(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int d, int most_tokens,
                   float scale, float softcap, bool all_units, bool beside, int* error_flag, cudaStream_t stream) {
  return d == 128 ? own::launch_rows<128>(q, k_pool, v_pool, n_pages, b, parts, most_tokens, scale, softcap, all_units, beside, error_flag, stream)
                  : own::launch_rows<64>(q, k_pool, v_pool, n_pages, b, parts, most_tokens, scale, softcap, all_units, beside, error_flag, stream);
}

}  // namespace prefix
}  // namespace ms
