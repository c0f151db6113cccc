// The shared prefix's part of attention on the fifth-generation tensor cores (bfloat16, head sizes 64 and 128).
//
// One thread block: one or two row tiles of a group and key head against its share of the prefix's key tiles; a row tile is up to 128 rows (token, query
// head of the key head's group), token-major, floor(128 / group) whole tokens; a key tile is as many whole pages as 128 keys hold.  Two streams of work
// share the tensor cores and the exponential units, so that one's products run beside the other's softmax:
//   two row tiles (groups of more than 128 rows): stream s is row tile s; both read every key tile
//   one row tile:                                   stream s takes the key tiles s, s + 2, ...; the two results are joined at the end
//   warp 0       TMA: the rows once (a box over tokens x heads x head size), then K tile after tile, one box a page (128-byte swizzle)
//   warp 1       tcgen05.mma: S_s = Q K^T into tensor memory, O_s += P_s V with P from tensor memory over the scores that it came from
//   warps 2..5   stream 0, warps 6..9 stream 1: a thread to a row: S from tensor memory, mask, maximum, 2^(s - m), P as bfloat16 back.  The output stays
//                in tensor memory and is rescaled only where a maximum grew by more than 2^8.
//   warp 10      TMA: V tile after tile
// P is rounded to bfloat16, V's type (a product takes operands of one type): a weight is off by at most 2^-8 of itself; the sum under it is of the
// unrounded weights, in float32.  Keys behind the prefix's end are not loaded; the tile's rows of V there are zeroed, so that whatever
// memory holds is never multiplied.  Warps whose rows hold no token do nothing between their arrivals.
//
// A row tile and key tile of head size 128 are 8.4 MFLOP and 16,384 exponentials: 0.75 us of a multiprocessor's share of the measured rate of products, 0.54
// of its exponential units; reading the key tile takes its share of the memory rate 1.45 us.  So the reads bound one row tile, the products two.
// Measured: a step of two row tiles takes 3,950 cycles of which the products take 3,300 (104 a 128 x 128 x 16 product); 64 requests behind 32,768 keys, own
// keys and join with them, 71 us replayed; 32 behind 4,096, where setting up, results and join (about 12 us) are most of it, 19.5.
// All mbarrier waits are bounded; a wait that runs out sets the error flag and every role drains and returns.
#include "attention_prefix.cuh"
#include "tcgen05.cuh"

namespace ms {
namespace prefix {

using namespace ms::t5;

namespace tc {

constexpr int ROWS = 128, BN = 128, THREADS = 352, TMEM_COLUMNS = 512;

// True in one thread of the warp.
__device__ __forceinline__ bool elect_one() {
  unsigned chosen;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(chosen));
  return chosen != 0;
}

__device__ __forceinline__ float fast_exp2(float x) {       // ex2.approx: relative error about 2^-22, -inf gives 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// tanh(x), x = v pre, of a row's scores (twice_pre_log2 = 2 pre log2 e).  Where all of a warp's |x| are 0.35 or less, as scores well below their cap are, by
// the series x - x^3 / 3 + 2 x^5 / 15 - 17 x^7 / 315 + 62 x^9 / 2835, which is off by less than 2^-23 there, two numbers an instruction: the
// exponential and the reciprocal of capped_score keep the special-function units busy twice as long as the softmax itself (a tile took
// 3,000 to 5,000 cycles for them).  Columns behind the row's last key, `seen` (`whole`: no row of the warp has any), have no say in it, nor has
// a row without a token (not `mine`): they may hold products of whatever shared memory held before.
__device__ __forceinline__ void cap_scores(float (&v)[BN], float twice_pre_log2, bool whole, int seen, bool mine) {
  const float pre = twice_pre_log2 * 0.34657359027997264f;          // ln 2 / 2
  float most = 0.f;
  if (whole) {
#pragma unroll
    for (int i = 0; i < BN; ++i) most = fmaxf(most, fabsf(v[i]));
  } else {
#pragma unroll
    for (int i = 0; i < BN; ++i) most = i <= seen ? fmaxf(most, fabsf(v[i])) : most;
  }
  if (!mine) most = 0.f;
  if (__all_sync(0xffffffffu, most * pre <= 0.35f)) {
    const unsigned long long pre2 = pack2(pre, pre);
#pragma unroll
    for (int i = 0; i < BN; i += 2) {
      const unsigned long long x = mul2(pack2(v[i], v[i + 1]), pre2), y = mul2(x, x);
      unsigned long long p = pack2(62.f / 2835.f, 62.f / 2835.f);
      p = fma2(p, y, pack2(-17.f / 315.f, -17.f / 315.f));
      p = fma2(p, y, pack2(2.f / 15.f, 2.f / 15.f));
      p = fma2(p, y, pack2(-1.f / 3.f, -1.f / 3.f));
      p = fma2(p, y, pack2(1.f, 1.f));
      unpack2(mul2(p, x), v[i], v[i + 1]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < BN; ++i) v[i] = capped_score(v[i], twice_pre_log2);
  }
}

template <int D, bool TWO>
struct Layout {
  static constexpr int K_STAGES = 2, V_STAGES = 2;
  static constexpr int DBLOCKS = D / 64;                 // 128-byte column blocks of a row
  static constexpr int Q_BYTES = ROWS * D * 2;           // of a row tile
  static constexpr int TILE_BYTES = BN * D * 2;          // one K or V tile
  static constexpr int K_AT = (TWO ? 2 : 1) * Q_BYTES, V_AT = K_AT + K_STAGES * TILE_BYTES;
  static constexpr size_t TOTAL = (size_t)V_AT + (size_t)V_STAGES * TILE_BYTES + 1024;
  static constexpr int STRIDE = D + 4;                   // floats of a row of the results on their way out, over the rows and tiles
  static_assert((TWO ? 2 : 1) * ROWS * STRIDE * 4 + ROWS * 8 <= V_AT + V_STAGES * TILE_BYTES, "the results fit over rows and tiles");
};

template <int D, bool TWO, bool CAP>
__global__ void __launch_bounds__(THREADS, 1)
prefix_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, Batch b,
              Parts parts, int box_rows, float scale_log2, float cap_log2, int* __restrict__ error_flag) {
  using L = Layout<D, TWO>;
  constexpr int K_STAGES = L::K_STAGES, V_STAGES = L::V_STAGES;
  extern __shared__ unsigned char smem_raw[];
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  auto q_tile = [&](int s) { return smem + (TWO ? (size_t)s * L::Q_BYTES : 0); };
  auto k_stage = [&](int i) { return smem + L::K_AT + (size_t)i * L::TILE_BYTES; };
  auto v_stage = [&](int i) { return smem + L::V_AT + (size_t)i * L::TILE_BYTES; };
  __shared__ uint64_t q_full, k_full[K_STAGES], k_empty[K_STAGES], v_full[V_STAGES], v_empty[V_STAGES];
  __shared__ uint64_t s_full[2], p_full[2], o_full[2];
  __shared__ unsigned tmem_base_s;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int kv_head = blockIdx.y, group = b.n_q / b.n_kv, tokens_per_tile = ROWS / group;

  if (warp == 0 && lane == 0) {
    mbar_init(&q_full, 1);
#pragma unroll
    for (int i = 0; i < K_STAGES; ++i) mbar_init(&k_full[i], 1), mbar_init(&k_empty[i], 1);
#pragma unroll
    for (int i = 0; i < V_STAGES; ++i) mbar_init(&v_full[i], 1), mbar_init(&v_empty[i], 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) mbar_init(&s_full[i], 1), mbar_init(&p_full[i], ROWS), mbar_init(&o_full[i], 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(TMEM_COLUMNS) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  const int boxes = BN / box_rows, tile_keys = boxes * box_rows;
  if (tile_keys < BN) {
    // rows of V that no page fills: zeros once and for all
    const int chunks = (BN - tile_keys) * 8 * L::DBLOCKS * V_STAGES;
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
  auto s_column = [&](int s) { return (unsigned)(s * BN); };
  auto o_column = [&](int s) { return (unsigned)(2 * BN + s * D); };

  grid_dependency_wait();
  grid_dependency_launch();

  const Unit u = prefix_unit(b, (int)blockIdx.z / parts.prefix, (int)blockIdx.z % parts.prefix, parts);
  const int token0 = u.token + (int)blockIdx.x * (TWO ? 2 : 1) * tokens_per_tile;
  auto rows_of = [&](int s) { return max(0, min(u.token_end - token0 - (TWO ? s * tokens_per_tile : 0), tokens_per_tile)) * group; };
  const int all_tiles = (u.key_end + tile_keys - 1) / tile_keys, share = (all_tiles + u.splits - 1) / u.splits;
  const int first_tile = u.split * share;
  const int n_tiles = rows_of(0) > 0 ? max(0, min(all_tiles, first_tile + share) - first_tile) : 0;
  // stream s goes steps_of(s) steps; its step t is the tile tile_of(s, t) of this block
  auto steps_of = [&](int s) { return TWO ? (rows_of(s) > 0 ? n_tiles : 0) : (n_tiles + 1 - s) / 2; };
  auto tile_of = [](int s, int t) { return TWO ? t : 2 * t + s; };

  if (n_tiles > 0) {
    if (warp == 0 || warp == 10) {
      // ---------------- producers of K (and the rows) and of V: lane 0 announces the bytes, all lanes issue the page loads
      const bool keys = warp == 0;
      const int stages = keys ? K_STAGES : V_STAGES;
      uint64_t* full = keys ? k_full : v_full;
      uint64_t* empty = keys ? k_empty : v_empty;
      const CUtensorMap* map = keys ? &map_k : &map_v;
      if (keys && lane == 0) {
        const int row_tiles = TWO && rows_of(1) > 0 ? 2 : 1;
        mbar_expect_tx(&q_full, (unsigned)(row_tiles * tokens_per_tile * group * D * 2));
        for (int s = 0; s < row_tiles; ++s)
#pragma unroll
          for (int db = 0; db < L::DBLOCKS; ++db)
            tma_load_3d(q_tile(s) + db * (ROWS * 128), &map_q, &q_full, db * 64, kv_head * group, token0 + s * tokens_per_tile);
      }
      bool ok = true;
      int sent = 0;
      for (int j = 0; j < n_tiles && ok; ++j) {
        const int stage = j % stages;
        const int key0 = (first_tile + j) * tile_keys;
        const int live_boxes = min(boxes, (u.key_end - key0 + box_rows - 1) / box_rows);
        if (lane == 0) {
          ok = mbar_wait(&empty[stage], ((unsigned)(j / stages) & 1) ^ 1, error_flag, 31);
          if (ok) mbar_expect_tx(&full[stage], (unsigned)(live_boxes * box_rows * D * 2));
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        sent = j + 1;
        unsigned char* to = keys ? k_stage(stage) : v_stage(stage);
        for (int i = lane; i < live_boxes * L::DBLOCKS; i += 32) {
          const int p = i / L::DBLOCKS, db = i % L::DBLOCKS, key = key0 + p * box_rows;
          const int pool_row = pool_row_of(b, u.table[key / b.page_size], kv_head, key);
          tma_load_2d(to + (size_t)db * (BN * 128) + (size_t)(p * box_rows) * 128, map, &full[stage], db * 64, pool_row);
        }
      }
      if (!ok) {
        // a wait ran out: the copies in flight land before the block may exit
        if (keys) mbar_wait(&q_full, 0, error_flag, 32);
        let_copies_land(full, stages, sent, error_flag);
      }
    } else if (warp == 1) {
      // ---------------- MMA issue: the whole warp goes along and one elected thread issues, so that descriptors are the warp's and lie in its uniform
      // registers (formed by one thread alone, eight products took 900 to 1,200 cycles to issue, twice what they take to run)
      constexpr unsigned idesc_s = umma_idesc(ROWS, BN, false);
      constexpr unsigned idesc_pv = umma_idesc(ROWS, D, true);
      const int steps0 = steps_of(0), steps1 = steps_of(1);
      const int last_reader = TWO && steps1 > 0 ? 1 : 0;          // of a tile that both streams read
      const bool leader = elect_one();
      // (S of the next step goes where P of this one lay: products run in the order of their issue)
      auto scores = [&](int s, int t) {
        const int j = tile_of(s, t), stage = j % K_STAGES;
        if (!__all_sync(0xffffffffu, mbar_wait(&k_full[stage], (unsigned)(j / K_STAGES) & 1, error_flag, 34))) return false;
        tmem_fence_after();
        const uint64_t a_desc = umma_desc(q_tile(s)), b_desc = umma_desc(k_stage(stage));
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma_bf16(tmem_base + s_column(s), a_desc + (kk / 4) * (ROWS * 128 / 16) + 2 * (kk % 4), b_desc + (kk / 4) * (BN * 128 / 16) + 2 * (kk % 4), idesc_s,
                      kk != 0 ? 1u : 0u);
          umma_commit(&s_full[s]);
          if (!TWO || s == last_reader) umma_commit(&k_empty[stage]);
        }
        __syncwarp();
        return true;
      };
      auto output = [&](int s, int t) {
        const int j = tile_of(s, t), stage = j % V_STAGES;
        const bool ready = mbar_wait(&p_full[s], (unsigned)t & 1, error_flag, 36) && mbar_wait(&v_full[stage], (unsigned)(j / V_STAGES) & 1, error_flag, 37);
        if (!__all_sync(0xffffffffu, ready)) return false;
        tmem_fence_after();
        const uint64_t b_desc = umma_desc_mn_major(v_stage(stage), BN * 128);
        if (leader) {
#pragma unroll
          for (int kk = 0; kk < BN / 16; ++kk)
            umma_bf16_a_tmem(tmem_base + o_column(s), tmem_base + s_column(s) + kk * 8, b_desc + kk * (16 * 128 / 16), idesc_pv, (t | kk) != 0 ? 1u : 0u);
          if (!TWO || s == last_reader) umma_commit(&v_empty[stage]);
          if (t + 1 == (s == 0 ? steps0 : steps1)) umma_commit(&o_full[s]);
        }
        __syncwarp();
        return true;
      };
      bool ok = __all_sync(0xffffffffu, mbar_wait(&q_full, 0, error_flag, 33)) && scores(0, 0) && (steps1 == 0 || scores(1, 0));
      for (int t = 0; t < steps0 && ok; ++t) {
        ok = output(0, t) && (t + 1 >= steps0 || scores(0, t + 1));
        if (ok && t < steps1) ok = output(1, t) && (t + 1 >= steps1 || scores(1, t + 1));
      }
    } else {
      // ---------------- softmax and result: a thread to a row
      const int s = warp >= 6 ? 1 : 0, quarter = warp & 3;
      const int row = quarter * 32 + lane, live_rows = rows_of(s), steps = steps_of(s);
      const bool mine = row < live_rows, any = quarter * 32 < live_rows;
      const int token = token0 + (TWO ? s * tokens_per_tile : 0) + (mine ? row / group : 0);
      // the last key that the row sees (a row without a token sees all: its numbers go nowhere, and a warp that it is in need not mask for it)
      const int limit = mine ? min(b.positions[token], u.key_end - 1) : u.key_end - 1;
      const unsigned lane_field = (unsigned)(quarter * 32) << 16;
      const unsigned s_addr = tmem_base + lane_field + s_column(s), o_addr = tmem_base + lane_field + o_column(s);
      float m_used = -INFINITY;      // the maximum that the exponents and the output are relative to
      float l = 0.f;
      bool ok = true;
      for (int t = 0; t < steps && ok; ++t) {
        const int j = tile_of(s, t), key0 = (first_tile + j) * tile_keys;
        const int live = min(tile_keys, u.key_end - key0);           // keys of the tile that are the prefix's
        // (the products behind these scores were issued after those of the step before: the output is complete up to it)
        ok = mbar_wait(&s_full[s], (unsigned)t & 1, error_flag, 38);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        tmem_fence_after();
        if (any) {
          float v[BN];
#pragma unroll
          for (int c = 0; c < BN; c += 32) tmem_load_32_nowait(s_addr + c, *reinterpret_cast<float(*)[32]>(&v[c]));
          tmem_load_wait();
          const int seen = min(limit, key0 + live - 1) - key0;       // keys 0 .. seen of the tile are visible
          const bool whole = __all_sync(0xffffffffu, seen >= BN - 1);
          if (CAP) cap_scores(v, cap_log2, whole, seen, mine);
          if (!whole) {
#pragma unroll
            for (int i = 0; i < BN; ++i)
              if (i > seen) v[i] = -INFINITY;
          }
          float part_max[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) part_max[e] = v[e];
#pragma unroll
          for (int i = 8; i < BN; ++i) part_max[i & 7] = fmaxf(part_max[i & 7], v[i]);
          const float tile_max = fmaxf(fmaxf(fmaxf(part_max[0], part_max[1]), fmaxf(part_max[2], part_max[3])),
                                       fmaxf(fmaxf(part_max[4], part_max[5]), fmaxf(part_max[6], part_max[7])));
          const float candidate = fmaxf(m_used, tile_max);
          const bool grow = candidate != -INFINITY && (m_used == -INFINITY || (candidate - m_used) * scale_log2 > 8.f);
          if (__any_sync(0xffffffffu, grow)) {
            const float factor = grow ? (m_used == -INFINITY ? 0.f : exp2f((m_used - candidate) * scale_log2)) : 1.f;
            if (grow) m_used = candidate;
            l *= factor;
            if (t > 0) {
#pragma unroll 1
              for (int c = 0; c < D; c += 16) {
                float o[16];
                tmem_load_16_nowait(o_addr + c, o);
                tmem_load_wait();
                unsigned scaled[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) scaled[i] = __float_as_uint(o[i] * factor);
                tmem_store_16(o_addr + c, scaled);
              }
              tmem_store_wait();
            }
          }
          const float base = m_used == -INFINITY ? 0.f : m_used * scale_log2;
          float part_sum[8];
#pragma unroll
          for (int e = 0; e < 8; ++e) part_sum[e] = 0.f;
#pragma unroll
          for (int c = 0; c < BN; c += 32) {
            unsigned packed[16];
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float p0 = fast_exp2(fmaf(v[c + i], scale_log2, -base));
              const float p1 = fast_exp2(fmaf(v[c + i + 1], scale_log2, -base));
              part_sum[(i >> 1) & 7] += p0 + p1;
              const __nv_bfloat162 pair = __floats2bfloat162_rn(p0, p1);
              packed[i / 2] = *reinterpret_cast<const unsigned*>(&pair);
            }
            tmem_store_16(s_addr + c / 2, packed);
          }
          l += ((part_sum[0] + part_sum[1]) + (part_sum[2] + part_sum[3])) + ((part_sum[4] + part_sum[5]) + (part_sum[6] + part_sum[7]));
          tmem_store_wait();
        }
        if (live < tile_keys && (!TWO || s == 0)) {
          // the last tile's rows of V behind the prefix: zeros (weights of 0 times whatever lies there would not be 0).  Of a tile that both streams
          // read stream 0 writes them: the products of its step come first.
          const int stage = j % V_STAGES;
          ok = mbar_wait(&v_full[stage], (unsigned)(j / V_STAGES) & 1, error_flag, 39);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          const int dead = tile_keys - live, thread = (int)threadIdx.x - 64 - s * ROWS;
          for (int i = thread; i < dead * 8 * L::DBLOCKS; i += ROWS) {
            const int c = i % 8, r = i / 8 % dead, db = i / (8 * dead);
            *reinterpret_cast<uint4*>(v_stage(stage) + (size_t)db * (BN * 128) + (size_t)(live + r) * 128 + c * 16) = make_uint4(0, 0, 0, 0);
          }
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        tmem_fence_before();
        mbar_arrive(&p_full[s]);
      }
      // no product reads the rows and tiles any more once both streams are through: they hold the results on their way out, a row to a thread
      if (ok) ok = mbar_wait(&o_full[0], 0, error_flag, 41);
      if (ok && steps_of(1) > 0) ok = mbar_wait(&o_full[1], 0, error_flag, 41);
      ok = __all_sync(0xffffffffu, ok);
      float* own_row = reinterpret_cast<float*>(smem) + (size_t)((TWO ? s * ROWS : 0) + row) * L::STRIDE;
      float joined_m = -INFINITY, joined_l = 0.f;                 // stream 1's, for stream 0
      const bool joined = !TWO && n_tiles > 1;
      if (joined) {
        // one row tile: stream 1's result passes to stream 0
        float* ends = reinterpret_cast<float*>(smem) + ROWS * L::STRIDE;
        if (s == 1) {
          ends[2 * row] = m_used, ends[2 * row + 1] = l;
          if (ok && any) {
            tmem_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
              float o[32];
              tmem_load_32(o_addr + c, o);
#pragma unroll
              for (int i = 0; i < 32; i += 4) *reinterpret_cast<float4*>(own_row + c + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
            }
          }
        }
        // all 256 threads pass this barrier, which also tells everyone whether anyone gave up a wait
        unsigned all;
        asm volatile("{\n.reg .pred p, q;\nsetp.ne.u32 p, %1, 0;\nbar.red.and.pred q, 1, 256, p;\nselp.u32 %0, 1, 0, q;\n}"
                     : "=r"(all) : "r"((unsigned)ok) : "memory");
        ok = all != 0;
        joined_m = ends[2 * row], joined_l = ends[2 * row + 1];
      }
      if (ok && any && steps > 0 && (TWO || s == 0)) {
        tmem_fence_after();
        // relative to the larger of the two maxima
        const float top = fmaxf(m_used, joined_m), zero = top == -INFINITY ? 0.f : top;
        const float mine_share = exp2f((m_used - zero) * scale_log2), other_share = exp2f((joined_m - zero) * scale_log2);
        l = l * mine_share + joined_l * other_share;
        const float inv = l == 0.f ? 0.f : 1.f / l;          // (NaN stays NaN)
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          float o[32];
          tmem_load_32(o_addr + c, o);
#pragma unroll
          for (int i = 0; i < 32; i += 4) {
            float4 v = make_float4(o[i] * mine_share, o[i + 1] * mine_share, o[i + 2] * mine_share, o[i + 3] * mine_share);
            float4* place = reinterpret_cast<float4*>(own_row + c + i);
            if (joined) {
              const float4 w = *place;
              v.x = fmaf(w.x, other_share, v.x), v.y = fmaf(w.y, other_share, v.y), v.z = fmaf(w.z, other_share, v.z), v.w = fmaf(w.w, other_share, v.w);
            }
            *place = make_float4(v.x * inv, v.y * inv, v.z * inv, v.w * inv);
          }
        }
        const size_t at = mine ? ((size_t)token * b.n_q + kv_head * group + row % group) * parts.count + u.part : 0;
        if (mine) parts.lse[at] = l == 0.f ? -INFINITY : zero * scale_log2 + log2f(l);
        // a warp's rows one after the other, a row by the whole warp: a thread's own row at a time went out in sixteen bytes of each line (8 us at the end of
        // two row tiles of head size 128)
        __syncwarp();
        const float* warp_rows = own_row - (size_t)lane * L::STRIDE;
        const int rows = min(32, live_rows - quarter * 32);
        constexpr int LANES = D / 4;                         // of a row
#pragma unroll 4
        for (int first = 0; first < rows; first += 32 / LANES) {
          const int r = first + lane / LANES;
          const size_t to = __shfl_sync(0xffffffffu, (unsigned long long)at, r);
          if (r < rows)
            *reinterpret_cast<float4*>(parts.o + to * D + lane % LANES * 4) = *reinterpret_cast<const float4*>(warp_rows + (size_t)r * L::STRIDE + lane % LANES * 4);
        }
      }
    }
  } else {
    // no keys for this part: weight 0
    for (int s = 0; s < (TWO ? 2 : 1); ++s)
      for (int row = threadIdx.x; row < rows_of(s); row += THREADS)
        parts.lse[((size_t)(token0 + s * tokens_per_tile + row / group) * b.n_q + kv_head * group + row % group) * parts.count + u.part] = -INFINITY;
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

template <int D, bool TWO>
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
  const bool cap = softcap > 0.f;
  auto kernel = cap ? prefix_kernel<D, TWO, true> : prefix_kernel<D, TWO, false>;
  const size_t smem = Layout<D, TWO>::TOTAL;
  static std::atomic<unsigned long long> asked_of[2];
  std::atomic<unsigned long long>& asked = asked_of[cap ? 1 : 0];
  MS_REQUIRE(allow_shared(kernel, smem) == cudaSuccess && share_multiprocessor(kernel, asked) == cudaSuccess, "prefix attention: cannot reserve %zu bytes of shared memory", smem);
  const float scale_log2 = (softcap > 0.f ? softcap : scale) * kLog2e;
  const float twice = softcap > 0.f ? 2.f * scale / softcap * kLog2e : 0.f;
  const cudaError_t e = ms::launch(kernel, dim3((unsigned)(TWO ? (row_tiles + 1) / 2 : row_tiles), b.n_kv, (unsigned)(b.n_groups * parts.prefix)), dim3(THREADS), smem, stream, map_q,
                                   map_k, map_v, b, parts, box_rows, scale_log2, twice, error_flag);
  if (e != cudaSuccess) MS_FAIL("prefix attention: launch failed: %s", cudaGetErrorString(e));
  return 0;
}

}  // namespace tc

int launch_prefix_tcgen05(const void* q, const void* k_pool, const void* v_pool, int n_pages, const Batch& b, const Parts& parts, int d, int n_tokens,
                          int max_group_tokens, float scale, float softcap, int* error_flag, cudaStream_t stream) {
  const int tokens_per_tile = tc::ROWS / (b.n_q / b.n_kv), row_tiles = (max_group_tokens + tokens_per_tile - 1) / tokens_per_tile;
#define MS_PREFIX_CASE(D, TWO) \
  return tc::launch_prefix<D, TWO>(q, k_pool, v_pool, n_pages, b, parts, n_tokens, row_tiles, scale, softcap, error_flag, stream)
  if (d == 128) { if (row_tiles > 1) { MS_PREFIX_CASE(128, true); } else { MS_PREFIX_CASE(128, false); } }
  if (row_tiles > 1) { MS_PREFIX_CASE(64, true); } else { MS_PREFIX_CASE(64, false); }
#undef MS_PREFIX_CASE
}

bool prefix_tcgen05_takes(int d, int group, int page_size, long long pool_rows) {
  return (d == 64 || d == 128) && group <= tc::ROWS && tc::box_rows_of(page_size) > 0 && pool_rows < 2147483648LL;
}

}  // namespace prefix
}  // namespace ms
