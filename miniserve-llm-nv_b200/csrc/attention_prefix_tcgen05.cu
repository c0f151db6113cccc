// The shared prefix's part of attention on the fifth-generation tensor cores (bfloat16, head sizes 64 and 128).
//
// One thread block: up to 128 rows of a group and key head - rows are (token, query head of the key head's group), token-major, floor(128 / group)
// whole tokens - against its share of the prefix's key tiles.  A tile is as many whole pages as 128 keys hold.
//   warp 0      TMA: the rows once (a box over tokens x heads x head size), then per tile a box a page of K and of V into a ring in
//               shared memory (128-byte swizzle)
//   warp 1      tcgen05.mma: S = Q K^T into one of two score buffers in tensor memory, a tile ahead; O += P V with P from tensor memory
//   warps 2..9  two threads per row, a half of the tile's keys each: S from tensor memory, mask, maximum, 2^(s - m), P as bfloat16 back over S.
//               The output stays in tensor memory and is rescaled only where a maximum grew by more than 2^8.
// P is rounded to bfloat16, V's type (a product takes operands of one type): a weight is off by at most 2^-8 of itself, the sum under it is of the
// unrounded weights, in float32.  Keys behind the prefix's end are not loaded; the tile's rows of V there are zeroed, so that whatever
// memory holds is never multiplied.  Warps whose rows hold no token do nothing between their arrivals.
//
// Few rows: the reads bound it (one tile of 64 KB per block and turn, 148 blocks); from 256 rows a key head on the products and the exponentials.
// All mbarrier waits are bounded; a wait that runs out sets the error flag and every role drains and returns.
#include "attention_prefix.cuh"
#include "tcgen05.cuh"

namespace ms {
namespace prefix {

using namespace ms::t5;

namespace tc {

constexpr int ROWS = 128, BN = 128, THREADS = 320, TMEM_COLUMNS = 512;
constexpr int HALF = BN / 2;               // keys of a tile per softmax thread
template <int D> constexpr int kv_stages() { return D == 128 ? 3 : 4; }

__device__ __forceinline__ float fast_exp2(float x) {       // ex2.approx: relative error about 2^-22, -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <int D>
struct Layout {
  static constexpr int STAGES = kv_stages<D>();
  static constexpr int DBLOCKS = D / 64;                 // 128-byte column blocks of a row
  static constexpr int Q_BYTES = ROWS * D * 2;
  static constexpr int TILE_BYTES = BN * D * 2;          // one K or V tile
  static constexpr size_t TOTAL = (size_t)Q_BYTES + (size_t)STAGES * 2 * TILE_BYTES + 1024;
};

template <int D>
__global__ void __launch_bounds__(THREADS, 1)
prefix_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Batch b,
              Parts parts, int box_rows, float scale_log2, float cap_log2, int* __restrict__ error_flag) {
  using L = Layout<D>;
  constexpr int STAGES = L::STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  unsigned char* q_s = smem;
  auto k_stage = [&](int s) { return smem + L::Q_BYTES + (size_t)s * 2 * L::TILE_BYTES; };
  auto v_stage = [&](int s) { return k_stage(s) + L::TILE_BYTES; };
  __shared__ uint64_t q_full, k_full[STAGES], v_full[STAGES], kv_empty[STAGES];
  __shared__ uint64_t s_full[2], p_full[2], pv_done[2];      // pv_done[j & 1]: the output is complete up to key tile j
  __shared__ unsigned tmem_base_s;
  // [tile parity][half][row]: the two threads of a row agree on its maximum, as bfloat16 rounded up (any bound above the true maximum serves);
  // the same bytes carry the two row sums at the end.
  __shared__ __align__(16) __nv_bfloat16 half_max_s[2][2][ROWS];

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_head = blockIdx.y, group = b.n_q / b.n_kv, tokens_per_tile = ROWS / group;

  if (warp == 0 && lane == 0) {
    mbar_init(&q_full, 1);
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&v_full[s], 1);
      mbar_init(&kv_empty[s], 1);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 2 * ROWS);
      mbar_init(&pv_done[i], 1);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int boxes = BN / box_rows, tile_keys = boxes * box_rows;
  if (tile_keys < BN) {
    // rows of V that no page fills: zeros once and for all
    const int chunks = (BN - tile_keys) * 8 * L::DBLOCKS * STAGES;
    for (int i = threadIdx.x; i < chunks; i += THREADS) {
      const int c = i % 8, r = i / 8 % (BN - tile_keys), rest = i / (8 * (BN - tile_keys));
      *reinterpret_cast<uint4*>(v_stage(rest / L::DBLOCKS) + (size_t)(rest % L::DBLOCKS) * (BN * 128) + (size_t)(tile_keys + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
    }
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  tmem_fence_before();
  __syncthreads();
  tmem_fence_after();
  const unsigned tmem_base = tmem_base_s;
  auto s_column = [&](int i) { return (unsigned)(i * BN); };
  const unsigned o_column = 2 * BN;

  grid_dependency_wait();
  grid_dependency_launch();

  const Unit u = prefix_unit(b, (int)blockIdx.z / parts.prefix, (int)blockIdx.z % parts.prefix, parts);
  const int token0 = u.token + (int)blockIdx.x * tokens_per_tile;
  const int live_rows = max(0, min(u.token_end - token0, tokens_per_tile)) * group;
  const int all_tiles = (u.key_end + tile_keys - 1) / tile_keys, share = (all_tiles + u.splits - 1) / u.splits;
  const int first_tile = u.split * share;
  const int n_tiles = live_rows > 0 ? max(0, min(all_tiles, first_tile + share) - first_tile) : 0;

  if (n_tiles > 0) {
    if (warp == 0) {
      // ---------------- producer: lane 0 announces the bytes, all lanes issue the page loads
      if (lane == 0) {
        mbar_expect_tx(&q_full, (unsigned)(tokens_per_tile * group * D * 2));
#pragma unroll
        for (int db = 0; db < L::DBLOCKS; ++db) tma_load_3d(q_s + db * (ROWS * 128), &map_q, &q_full, db * 64, kv_head * group, token0);
      }
      bool ok = true;
      int sent = 0;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int stage = j % STAGES;
        const int key0 = (first_tile + j) * tile_keys;
        const int live_boxes = min(boxes, (u.key_end - key0 + box_rows - 1) / box_rows);
        if (lane == 0) {
          ok = mbar_wait(&kv_empty[stage], ((unsigned)(j / STAGES) & 1) ^ 1, error_flag, 31);
          if (ok) {
            mbar_expect_tx(&k_full[stage], (unsigned)(live_boxes * box_rows * D * 2));
            mbar_expect_tx(&v_full[stage], (unsigned)(live_boxes * box_rows * D * 2));
          }
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        sent = j + 1;
        for (int i = lane; i < live_boxes * L::DBLOCKS; i += 32) {
          const int p = i / L::DBLOCKS, db = i % L::DBLOCKS;
          const int key = key0 + p * box_rows;
          const int pool_row = (u.table[key / b.page_size] * b.n_kv + kv_head) * b.page_size + key % b.page_size;
          const size_t at = (size_t)db * (BN * 128) + (size_t)(p * box_rows) * 128;
          tma_load_2d(k_stage(stage) + at, &map_k, &k_full[stage], db * 64, pool_row);
          tma_load_2d(v_stage(stage) + at, &map_v, &v_full[stage], db * 64, pool_row);
        }
      }
      if (!ok) {
        // a wait ran out: the copies in flight land before the block may exit
        mbar_wait(&q_full, 0, error_flag, 32);
        let_copies_land(k_full, STAGES, sent, error_flag);
        let_copies_land(v_full, STAGES, sent, error_flag);
      }
    } else if (warp == 1) {
      if (lane == 0) {
        // ---------------- MMA issue
        constexpr unsigned idesc_s = umma_idesc(ROWS, BN, false);
        constexpr unsigned idesc_pv = umma_idesc(ROWS, D, true);
        auto issue_scores = [&](int j) {
          const int stage = j % STAGES, i = j & 1;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            const uint64_t a_desc = umma_desc(q_s + (kk / 4) * (ROWS * 128)) + 2 * (kk % 4);
            const uint64_t b_desc = umma_desc(k_stage(stage) + (kk / 4) * (BN * 128)) + 2 * (kk % 4);
            umma_bf16(tmem_base + s_column(i), a_desc, b_desc, idesc_s, kk != 0 ? 1u : 0u);
          }
          umma_commit(&s_full[i]);
        };
        bool ok = mbar_wait(&q_full, 0, error_flag, 33) && mbar_wait(&k_full[0], 0, error_flag, 34);
        if (ok) {
          tmem_fence_after();
          issue_scores(0);
        }
        for (int j = 0; j < n_tiles && ok; ++j) {
          const int stage = j % STAGES, i = j & 1;
          if (j + 1 < n_tiles) {
            ok = mbar_wait(&k_full[(j + 1) % STAGES], (unsigned)((j + 1) / STAGES) & 1, error_flag, 35);
            if (!ok) break;
            tmem_fence_after();
            issue_scores(j + 1);
          }
          ok = mbar_wait(&p_full[i], (unsigned)(j / 2) & 1, error_flag, 36) && mbar_wait(&v_full[stage], (unsigned)(j / STAGES) & 1, error_flag, 37);
          if (!ok) break;
          tmem_fence_after();
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk) {
            const uint64_t b_desc = umma_desc_mn_major(v_stage(stage) + kk * (16 * 128), BN * 128);
            umma_bf16_a_tmem(tmem_base + o_column, tmem_base + s_column(i) + kk * 8, b_desc, idesc_pv, (j | kk) != 0 ? 1u : 0u);
          }
          umma_commit(&pv_done[j & 1]);
          umma_commit(&kv_empty[stage]);
        }
      }
    } else {
      // ---------------- softmax and result: two threads per row, one per half of the tile's keys
      const int quarter = warp & 3, half = warp >= 6 ? 1 : 0;
      const int row = quarter * 32 + lane;
      const bool mine = row < live_rows, any = quarter * 32 < live_rows;
      const int token = token0 + (mine ? row / group : 0);
      const int limit = mine ? min(b.positions[token], u.key_end - 1) : -1;        // the last key that the row sees
      const unsigned lane_field = (unsigned)(quarter * 32) << 16;
      const unsigned o_addr = tmem_base + lane_field + o_column + half * (D / 2);   // this thread's half of the row's output
      // All 256 threads pass this barrier together; it also tells everyone whether anyone gave up a wait.
      auto all_ok = [](bool mine_ok) {
        unsigned result;
        asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.and.pred q, 1, 256, p;\nselp.u32 %0, 1, 0, q;\n}"
                     : "=r"(result) : "r"((unsigned)mine_ok) : "memory");
        return result != 0;
      };
      float m_used = -INFINITY;      // the maximum that the exponents and the output are relative to
      float l = 0.f;                 // the sum over this thread's half of the keys
      bool ok = true;
      for (int j = 0; j < n_tiles; ++j) {
        const int i2 = j & 1;
        const unsigned phase = (unsigned)(j / 2) & 1;
        const int tile_key = (first_tile + j) * tile_keys, key0 = tile_key + half * HALF;
        const int live = min(tile_keys, u.key_end - tile_key);       // keys of the tile that are the prefix's
        ok = ok && mbar_wait(&s_full[i2], phase, error_flag, 38);
        ok = __all_sync(0xffffffffu, ok);
        const unsigned s_addr = tmem_base + lane_field + s_column(i2) + half * HALF;
        float v[HALF];
        float tile_max = -INFINITY;
        if (ok && any) {
          tmem_fence_after();
          tmem_load_32_nowait(s_addr, *reinterpret_cast<float(*)[32]>(&v[0]));
          tmem_load_32_nowait(s_addr + 32, *reinterpret_cast<float(*)[32]>(&v[32]));
          tmem_load_wait();
          if (cap_log2 > 0.f) {
#pragma unroll
            for (int i = 0; i < HALF; ++i) v[i] = capped_score(v[i], cap_log2);
          }
          float part_max[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) part_max[e] = -INFINITY;
          const int seen = min(limit - key0, tile_key + live - 1 - key0);      // keys 0 .. seen of this half are visible
          if (seen >= HALF - 1) {
#pragma unroll
            for (int i = 0; i < HALF; ++i) part_max[i & 7] = fmaxf(part_max[i & 7], v[i]);
          } else {
#pragma unroll
            for (int i = 0; i < HALF; ++i) {
              if (i > seen) v[i] = -INFINITY;
              part_max[i & 7] = fmaxf(part_max[i & 7], v[i]);
            }
          }
          tile_max = fmaxf(fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3])),
                           fmaxf(fmaxf(part_max[4], part_max[5]), fmaxf(part_max[6], part_max[7])));
        }
        const __nv_bfloat16 bound = __float2bfloat16_ru(tile_max);
        half_max_s[i2][half][row] = bound;
        if (ok && live < tile_keys) {
          // the last tile's rows of V behind the prefix: zeros (weights of 0 times whatever lies there would not be 0)
          ok = mbar_wait(&v_full[j % STAGES], (unsigned)(j / STAGES) & 1, error_flag, 39);
          if (ok) {
            const int dead = tile_keys - live;
            for (int i = threadIdx.x - 64; i < dead * 8 * L::DBLOCKS; i += 2 * ROWS) {
              const int c = i % 8, r = i / 8 % dead, db = i / (8 * dead);
              *reinterpret_cast<uint4*>(v_stage(j % STAGES) + (size_t)db * (BN * 128) + (size_t)(live + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          }
        }
        if (!all_ok(ok)) {
          ok = false;
          break;
        }
        tile_max = fmaxf(__bfloat162float(bound), __bfloat162float(half_max_s[i2][half ^ 1][row]));
        const float candidate = fmaxf(m_used, tile_max);
        const bool grow = candidate != -INFINITY && (m_used == -INFINITY || (candidate - m_used) * scale_log2 > 8.f);
        if (__any_sync(0xffffffffu, grow)) {
          const float factor = grow ? (m_used == -INFINITY ? 0.f : exp2f((m_used - candidate) * scale_log2)) : 1.f;
          if (grow) m_used = candidate;
          l *= factor;
          if (j > 0) {
            ok = mbar_wait(&pv_done[(j - 1) & 1], (unsigned)((j - 1) / 2) & 1, error_flag, 40);     // the output must be complete up to tile j - 1
            ok = __all_sync(0xffffffffu, ok);
            if (ok) {
              tmem_fence_after();
#pragma unroll
              for (int c = 0; c < D / 2; c += 32) {
                float o[32];
                tmem_load_32(o_addr + c, o);
                unsigned scaled[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) scaled[i] = __float_as_uint(o[i] * factor);
                tmem_store_32(o_addr + c, scaled);
              }
              tmem_store_wait();
            }
          }
        }
        if (ok) {
          if (any) {
            const float base = m_used == -INFINITY ? 0.f : m_used * scale_log2;
            float part_sum[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) part_sum[e] = 0.f;
#pragma unroll
            for (int c = 0; c < HALF; c += 32) {
              unsigned packed[16];
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const float p0 = fast_exp2(v[c + i] * scale_log2 - base);
                const float p1 = fast_exp2(v[c + i + 1] * scale_log2 - base);
                part_sum[(i >> 1) & 7] += p0 + p1;
                const __nv_bfloat162 pair = __floats2bfloat162_rn(p0, p1);
                packed[i / 2] = *reinterpret_cast<const unsigned*>(&pair);
              }
              tmem_store_16(tmem_base + lane_field + s_column(i2) + (half * HALF + c) / 2, packed);
            }
            l += ((part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3])) + ((part_sum[4] + part_sum[5]) + (part_sum[6] + part_sum[7]));
            tmem_store_wait();
          }
          tmem_fence_before();
          mbar_arrive(&p_full[i2]);
        }
      }
      if (ok && n_tiles > 1) ok = mbar_wait(&pv_done[(n_tiles - 2) & 1], (unsigned)((n_tiles - 2) / 2) & 1, error_flag, 41);
      if (ok) ok = mbar_wait(&pv_done[(n_tiles - 1) & 1], (unsigned)((n_tiles - 1) / 2) & 1, error_flag, 41);
      ok = __all_sync(0xffffffffu, ok);
      ok = all_ok(ok);                                 // nobody reads the maxima any more
      float* half_sum_s = reinterpret_cast<float*>(&half_max_s[0][0][0]);      // [half][row]
      half_sum_s[half * ROWS + row] = l;
      if (all_ok(ok) && any) {
        tmem_fence_after();
        l = half_sum_s[row] + half_sum_s[ROWS + row];
        const float inv = l == 0.f ? 0.f : 1.f / l;          // (NaN stays NaN)
        const size_t at = mine ? ((size_t)token * b.n_q + kv_head * group + row % group) * parts.count + u.part : 0;
        float* dst = parts.o + at * D + half * (D / 2);
#pragma unroll
        for (int c = 0; c < D / 2; c += 32) {
          float o[32];
          tmem_load_32(o_addr + c, o);
          if (mine) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              *reinterpret_cast<float4*>(dst + c + i) = make_float4(o[i] * inv, o[i + 1] * inv, o[i + 2] * inv, o[i + 3] * inv);
          }
        }
        if (mine && half == 0) parts.lse[at] = l == 0.f ? -INFINITY : m_used * scale_log2 + log2f(l);
      }
    }
  } else if (live_rows > 0) {
    // no keys for this part: weight 0
    for (int row = threadIdx.x; row < live_rows; row += THREADS)
      parts.lse[((size_t)(token0 + row / group) * b.n_q + kv_head * group + row % group) * parts.count + u.part] = -INFINITY;
  }

  tmem_fence_before();
  __syncthreads();
  if (warp == 1) {
    tmem_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(TMEM_COLUMNS) : "memory");
  }
}

static bool encode(CUtensorMap* map, int rank, const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
  EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return false;
  const cuuint32_t elem[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of a page that one box takes (0: these pages are not taken): whole pages of a multiple of eight up to 128, or 128 of larger ones.
static int box_rows_of(int page_size) {
  if (page_size >= 8 && page_size <= BN && page_size % 8 == 0) return page_size;
  return page_size > BN && page_size % BN == 0 ? BN : 0;
}

template <int D>
int launch_prefix(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int n_tokens, int row_tiles,
                  float scale, float softcap, int* error_flag, cudaStream_t stream) {
  const int group = b.n_q / b.n_kv, box_rows = box_rows_of(b.page_size);
  CUtensorMap map_q, map_k, map_v;
  {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)b.n_q, (cuuint64_t)n_tokens};
    const cuuint64_t strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)b.n_q * D * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)group, (cuuint32_t)(ROWS / group)};
    MS_REQUIRE(encode(&map_q, 3, q, dims, strides, box), "prefix attention: tensor map of the queries failed");
  }
  {
    const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)n_pages * b.n_kv * b.page_size};
    const cuuint64_t strides[1] = {(cuuint64_t)D * 2};
    const cuuint32_t box[2] = {64, (cuuint32_t)box_rows};
    MS_REQUIRE(encode(&map_k, 2, k_pool, dims, strides, box) && encode(&map_v, 2, v_pool, dims, strides, box), "prefix attention: tensor map of the pools failed");
  }
  auto kernel = prefix_kernel<D>;
  const size_t smem = Layout<D>::TOTAL;
  MS_REQUIRE(allow_shared(kernel, smem) == cudaSuccess, "prefix attention: cannot reserve %zu bytes of shared memory", smem);
  const float scale_log2 = (softcap > 0.f ? softcap : scale) * kLog2e;
  const float twice = softcap > 0.f ? 2.f * scale / softcap * kLog2e : 0.f;
  const cudaError_t e = ms::launch(kernel, dim3((unsigned)row_tiles, b.n_kv, (unsigned)(b.n_groups * parts.prefix)), dim3(THREADS), smem, stream, map_q,
                                   map_k, map_v, b, parts, box_rows, scale_log2, twice, error_flag);
  if (e != cudaSuccess) MS_FAIL("prefix attention: launch failed: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace tc

int launch_prefix_tcgen05(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int d, int n_tokens,
                          int max_group_tokens, float scale, float softcap, int* error_flag, cudaStream_t stream) {
  const int tokens_per_tile = tc::ROWS / (b.n_q / b.n_kv), row_tiles = (max_group_tokens + tokens_per_tile - 1) / tokens_per_tile;
  return d == 128 ? tc::launch_prefix<128>(q, k_pool, v_pool, n_pages, b, parts, n_tokens, row_tiles, scale, softcap, error_flag, stream)
                  : tc::launch_prefix<64>(q, k_pool, v_pool, n_pages, b, parts, n_tokens, row_tiles, scale, softcap, error_flag, stream);
}

bool prefix_tcgen05_takes(int d, int group, int page_size, long long pool_rows) {
  return (d == 64 || d == 128) && group <= tc::ROWS && tc::box_rows_of(page_size) > 0 && pool_rows < 2147483648LL;
}

}  // namespace prefix
}  // namespace ms
