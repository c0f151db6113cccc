// Parts of attention behind a shared prefix on mma.sync (bfloat16, head sizes that are multiples of 8 up to 128, pages of any size): every request's own
// keys, and the prefixes where the tcgen05 kernel does not take the sizes.
//
// Thread block: W warps of 16 rows (token, query head of the key head's group) of one unit and key head, over its share of the keys; a step of single
// tokens has few rows a request, so one warp (W = 1) and many small blocks hide the latencies.  Tiles of BN keys are gathered from the pages with
// 16-byte asynchronous copies, two in shared memory; a row there is 16 bytes longer than a multiple of 32 bytes, so that eight rows of a fragment lie
// in different banks.  S = Q K^T, running maximum and sum (float32), O += P V with P rounded to bfloat16 (V's type: a weight off by at most 2^-8 of
// itself).  The reads of keys and values bound it.
#include "attention_prefix.cuh"
#include "mma_common.cuh"

namespace ms {
namespace prefix {
namespace mm {

template <int DP> constexpr int kStride = DP + 8;            // elements of a row in shared memory

template <int DP, int W, int BN, int STAGES>
constexpr size_t smem_bytes() {
  return (size_t)(16 * W + 2 * STAGES * BN) * kStride<DP> * 2 + (size_t)STAGES * BN * sizeof(long long);
}

// own: the units are the requests' own keys, else the groups' prefixes.  beside: the kernel before this one on the stream is the prefixes' of the same
// call, which let this one start after its own wait for what came before: nothing here depends on it but the order in which the join may start.
template <int DP, int W, int BN, int STAGES>
__global__ void __launch_bounds__(W * 32)
part_kernel(const __nv_bfloat16* __restrict__ q, const __nv_bfloat16* __restrict__ k_pool, const __nv_bfloat16* __restrict__ v_pool, Batch b, Parts parts,
            int d, float scale_log2, float cap_log2, int own, int beside) {
  constexpr int ROWS = 16 * W, THREADS = 32 * W, CHUNKS = DP / 8, STRIDE = kStride<DP>;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  __nv_bfloat16* q_s = reinterpret_cast<__nv_bfloat16*>(smem_raw);               // [ROWS][STRIDE]
  __nv_bfloat16* k_s = q_s + ROWS * STRIDE;                                      // [STAGES][BN][STRIDE]
  __nv_bfloat16* v_s = k_s + STAGES * BN * STRIDE;                               // [STAGES][BN][STRIDE]
  long long* row_offset = reinterpret_cast<long long*>(v_s + STAGES * BN * STRIDE);   // [STAGES][BN] pool offset of a key row, -1: none
  if (!beside) grid_dependency_wait();
  grid_dependency_launch();

  const int splits = own ? parts.own : parts.prefix;
  const Unit u = own ? own_unit(b, (int)blockIdx.z / splits, (int)blockIdx.z % splits, parts) : prefix_unit(b, (int)blockIdx.z / splits, (int)blockIdx.z % splits, parts);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kv_head = blockIdx.y, group = b.n_q / b.n_kv;
  const int rows_total = (u.token_end - u.token) * group, row0 = (int)blockIdx.x * ROWS;
  if (row0 >= rows_total) {
    if (beside && last_block()) grid_dependency_wait();
    return;
  }
  const int tiles = (u.key_end - u.key + BN - 1) / BN, share = (tiles + u.splits - 1) / u.splits;
  const int tile_lo = u.split * share, tile_hi = min(tiles, tile_lo + share);

  auto find_rows = [&](int tile, int buffer) {
    const int key0 = u.key + tile * BN;
    for (int r = tid; r < BN; r += THREADS) {
      const int key = key0 + r;
      long long offset = -1;
      if (tile < tile_hi && key < u.key_end) {
        const int page = u.table[key / b.page_size];
        if ((unsigned)page < (unsigned)b.n_pages) offset = (((long long)page * b.n_kv + kv_head) * b.page_size + key % b.page_size) * d;
      }
      row_offset[buffer * BN + r] = offset;
    }
  };
  auto load_tile = [&](int stage) {
    __nv_bfloat16* ks = k_s + stage * BN * STRIDE;
    __nv_bfloat16* vs = v_s + stage * BN * STRIDE;
#pragma unroll 4
    for (int i = tid; i < BN * CHUNKS; i += THREADS) {
      const int r = i / CHUNKS, c = i % CHUNKS;
      const long long offset = row_offset[stage * BN + r];
      const bool valid = offset >= 0 && c * 8 < d;           // (zeros elsewhere)
      const long long at = valid ? offset + c * 8 : 0;
      cp_async_16(ks + r * STRIDE + c * 8, k_pool + at, valid);
      cp_async_16(vs + r * STRIDE + c * 8, v_pool + at, valid);
    }
  };

#pragma unroll
  for (int s = 0; s < STAGES; ++s) find_rows(tile_lo + s, s);
  __syncthreads();
  for (int i = tid; i < ROWS * CHUNKS; i += THREADS) {
    const int r = i / CHUNKS, c = i % CHUNKS, row = row0 + r;
    const bool valid = row < rows_total && c * 8 < d;
    const __nv_bfloat16* src = q;
    if (valid) src = q + ((size_t)(u.token + row / group) * b.n_q + kv_head * group + row % group) * d + c * 8;
    cp_async_16(q_s + r * STRIDE + c * 8, src, valid);
  }
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) {
    if (tile_lo + s < tile_hi) load_tile(s);
    cp_async_commit();
  }

  const int quad_row = lane >> 2, quad_col = lane & 3;
  int limit[2];                                      // the last key that the row sees
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int row = row0 + warp * 16 + quad_row + half * 8;
    limit[half] = row < rows_total ? min(b.positions[u.token + row / group], u.key_end - 1) : -1;
  }
  unsigned q_frag[DP / 16][4];
  float acc_o[DP / 8][4], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll
  for (int n = 0; n < DP / 8; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc_o[n][e] = 0.f;

  for (int tile = tile_lo; tile < tile_hi; ++tile) {
    const int stage = (tile - tile_lo) % STAGES;
    if (tile + STAGES - 1 < tile_hi) load_tile((stage + STAGES - 1) % STAGES);
    cp_async_commit();
    cp_async_wait<STAGES - 1>();
    __syncthreads();
    if (tile == tile_lo) {
#pragma unroll
      for (int kk = 0; kk < DP / 16; ++kk)
        ldmatrix_x4(q_frag[kk], q_s + (warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * STRIDE + kk * 16 + (lane >> 4) * 8);
    }
    find_rows(tile + STAGES, stage);     // this tile's copies have landed; its offsets are no longer needed
    const __nv_bfloat16* ks = k_s + stage * BN * STRIDE;
    const __nv_bfloat16* vs = v_s + stage * BN * STRIDE;
    const int key0 = u.key + tile * BN;

    float acc_s[BN / 8][4];
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc_s[n][e] = 0.f;
#pragma unroll
    for (int kk = 0; kk < DP / 16; ++kk)
#pragma unroll
      for (int np = 0; np < BN / 16; ++np) {
        unsigned f[4];
        ldmatrix_x4(f, ks + (np * 16 + (lane & 7) + (lane >> 4) * 8) * STRIDE + kk * 16 + ((lane >> 3) & 1) * 8);
        mma_bf16(acc_s[2 * np], q_frag[kk], f[0], f[1]);
        mma_bf16(acc_s[2 * np + 1], q_frag[kk], f[2], f[3]);
      }
    if (cap_log2 > 0.f) {
#pragma unroll
      for (int n = 0; n < BN / 8; ++n)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc_s[n][e] = capped_score(acc_s[n][e], cap_log2);
    }
    float tile_max[2] = {-INFINITY, -INFINITY};
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (key0 + n * 8 + quad_col * 2 + (e & 1) > limit[e >> 1]) acc_s[n][e] = -INFINITY;
        tile_max[e >> 1] = fmaxf(tile_max[e >> 1], acc_s[n][e]);
      }
    float base[2], corr[2], sum[2] = {0.f, 0.f};
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float v = tile_max[half];
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
      v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
      const float updated = fmaxf(m_run[half], v);
      base[half] = updated == -INFINITY ? 0.f : updated * scale_log2;
      corr[half] = exp2f(m_run[half] * scale_log2 - base[half]);      // m == -inf gives 0
      m_run[half] = updated;
    }
#pragma unroll
    for (int n = 0; n < BN / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        acc_s[n][e] = exp2f(acc_s[n][e] * scale_log2 - base[e >> 1]);
        sum[e >> 1] += acc_s[n][e];
      }
#pragma unroll
    for (int half = 0; half < 2; ++half) l_run[half] = l_run[half] * corr[half] + sum[half];
#pragma unroll
    for (int n = 0; n < DP / 8; ++n) {
      acc_o[n][0] *= corr[0], acc_o[n][1] *= corr[0];
      acc_o[n][2] *= corr[1], acc_o[n][3] *= corr[1];
    }
#pragma unroll
    for (int kp = 0; kp < BN / 16; ++kp) {
      unsigned p[4];
      p[0] = pack_bf16(acc_s[2 * kp][0], acc_s[2 * kp][1]);
      p[1] = pack_bf16(acc_s[2 * kp][2], acc_s[2 * kp][3]);
      p[2] = pack_bf16(acc_s[2 * kp + 1][0], acc_s[2 * kp + 1][1]);
      p[3] = pack_bf16(acc_s[2 * kp + 1][2], acc_s[2 * kp + 1][3]);
#pragma unroll
      for (int np = 0; np < DP / 16; ++np) {
        unsigned f[4];
        ldmatrix_x4_trans(f, vs + (kp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8) * STRIDE + np * 16 + (lane >> 4) * 8);
        mma_bf16(acc_o[2 * np], p, f[0], f[1]);
        mma_bf16(acc_o[2 * np + 1], p, f[2], f[3]);
      }
    }
    __syncthreads();       // all warps are done with this stage before it is refilled
  }
  cp_async_wait<0>();

#pragma unroll
  for (int half = 0; half < 2; ++half) {
    float l = l_run[half];
    l += __shfl_xor_sync(0xffffffffu, l, 1);
    l += __shfl_xor_sync(0xffffffffu, l, 2);
    const int row = row0 + warp * 16 + quad_row + half * 8;
    if (row >= rows_total) continue;
    const size_t at = ((size_t)(u.token + row / group) * b.n_q + kv_head * group + row % group) * parts.count + u.part;
    const float inv = l == 0.f ? 0.f : 1.f / l;          // (NaN stays NaN)
    float* dst = parts.o + at * d;
#pragma unroll
    for (int n = 0; n < DP / 8; ++n)
      if (n * 8 < d) *reinterpret_cast<float2*>(dst + n * 8 + quad_col * 2) = make_float2(acc_o[n][2 * half] * inv, acc_o[n][2 * half + 1] * inv);
    if (quad_col == 0) parts.lse[at] = l == 0.f ? -INFINITY : m_run[half] * scale_log2 + log2f(l);
  }
  if (beside && last_block()) grid_dependency_wait();
}

template <int DP, int W, int BN, int STAGES>
int launch_part(const void* q, const void* k_pool, const void* v_pool, const Batch& b, const Parts& parts, int d, int most_tokens, float scale, float softcap,
                bool own, bool beside, cudaStream_t stream) {
  auto kernel = part_kernel<DP, W, BN, STAGES>;
  const size_t smem = smem_bytes<DP, W, BN, STAGES>();
  MS_REQUIRE(allow_shared(kernel, smem) == cudaSuccess, "prefix attention: cannot reserve %zu bytes of shared memory", smem);
  const long long tiles = ((long long)most_tokens * (b.n_q / b.n_kv) + 16 * W - 1) / (16 * W);
  const long long units = own ? (long long)b.n_requests * parts.own : (long long)b.n_groups * parts.prefix;
  MS_REQUIRE(tiles <= 2147483647LL && units <= 65535 && b.n_kv <= 65535, "prefix attention: grid %lld x %d x %lld exceeds the launch limits", tiles, b.n_kv, units);
  const float scale_log2 = (softcap > 0.f ? softcap : scale) * kLog2e;
  const float twice = softcap > 0.f ? 2.f * scale / softcap * kLog2e : 0.f;
  ms::launch(kernel, dim3((unsigned)tiles, b.n_kv, (unsigned)units), dim3(W * 32), smem, stream, (const __nv_bfloat16*)q, (const __nv_bfloat16*)k_pool,
             (const __nv_bfloat16*)v_pool, b, parts, d, scale_log2, twice, own ? 1 : 0, beside ? 1 : 0);
  MS_CHECK_LAUNCH("prefix attention (parts)");
  return 0;
}

template <int DP>
int launch_part_rows(const void* q, const void* k_pool, const void* v_pool, const Batch& b, const Parts& parts, int d, int most_tokens, float scale,
                     float softcap, bool own, bool beside, cudaStream_t stream) {
  if (most_tokens * (b.n_q / b.n_kv) <= 16)
    return launch_part<DP, 1, 32, 2>(q, k_pool, v_pool, b, parts, d, most_tokens, scale, softcap, own, beside, stream);
  return launch_part<DP, 4, 64, 2>(q, k_pool, v_pool, b, parts, d, most_tokens, scale, softcap, own, beside, stream);
}

}  // namespace mm

bool prefix_mma_takes(int d) { return d >= 8 && d <= 128 && d % 8 == 0; }

int launch_part_mma(const void* q, const void* k_pool, const void* v_pool, const Batch& b, const Parts& parts, int d, int most_tokens, float scale,
                    float softcap, bool own, bool beside, cudaStream_t stream) {
#define MS_PART_CASE(DP) \
  if (d <= DP) return mm::launch_part_rows<DP>(q, k_pool, v_pool, b, parts, d, most_tokens, scale, softcap, own, beside, stream)
  MS_PART_CASE(32);
  MS_PART_CASE(48);
  MS_PART_CASE(64);
  MS_PART_CASE(80);
  MS_PART_CASE(96);
  MS_PART_CASE(112);
  MS_PART_CASE(128);
#undef MS_PART_CASE
  MS_FAIL("prefix attention: head size %d", d);
}

}  // namespace prefix
}  // namespace ms
