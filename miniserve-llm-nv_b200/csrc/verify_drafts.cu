// Verification of drafted tokens against the target's probabilities, with the random numbers given.
//
// A request brings D drafted tokens and D + 1 rows of target logits.  p, the distribution that `sample` draws from: w_i = e^((x_i - max) /
// temperature) over the kept entries (the top_k largest, of equal ones the lower index first; of those the nucleus: in descending order an
// entry stays while the mass before it is at most top_p), divided by their sum; temperature 0: one at the argmax.  Draft i with the draft's
// probabilities q_i (one at the drafted token where there are none) passes iff u_i q_i(d_i) < p_i(d_i).  At the first that does not, the next
// token is argmax max(p - q, 0) / e with given exponential variates e, which draws from the normed residual; where all pass, argmax p / e
// of the last row.  No running sum over the vocabulary has to be inverted: a token's choice hangs on the two best quotients, not on the
// last bits of a sum of 150,000.
//
// Two kernels, both bound by the reads: of all rows of logits, then of one row of logits, draft probabilities and variates per request.  A
// cluster of eight blocks works on a row: a block's eighth (76 KB of a vocabulary of 151,936) is read from memory once and stays in the
// first-level cache for the passes that the filters take; counts, masses and candidates meet in distributed shared memory.
#include "common.cuh"

#include <cooperative_groups.h>

namespace ms {
namespace verify {

namespace cg = cooperative_groups;

constexpr int kRanks = 8, kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;              // of one round of a search over 32-bit keys: eleven, eleven and ten bits

struct Record {  // one per state slot, as `sample` reads it
  float temperature;
  float top_p;
  int top_k;
  int reserved[5];
};

struct Row {      // what the second kernel needs to know of a row
  float top, inverse;      // the largest logit, and 1 / the kept sum of e^((x - top) / temperature)
  unsigned thr;            // kept: order_key > thr, or equal to it and an index below bound
  int bound;
  int best;                // argmax
  int passes;              // its draft passes
  int reserved[2];
};

__device__ __forceinline__ unsigned order_key(float f) {
  const unsigned u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

struct Best {
  float value;
  int index;
};
__device__ __forceinline__ Best better(Best a, Best b) {
  return b.value > a.value || (b.value == a.value && b.index < a.index) ? b : a;
}

// NaN counts as an entry that is masked, and -0 as 0 (their keys would differ).
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.f : -INFINITY; }
// (x - top) / temperature, 0 at x = top also where both are infinite.
__device__ __forceinline__ float exponent(float x, float top, float temperature) { return x == top ? 0.f : (x - top) / temperature; }

// This block's part of a row, in index order over the ranks; the parts start at 16-byte boundaries.
struct Part {
  const float* row;
  int begin, end, vocab;
  __device__ Part(const float* r, int v, int rank) : row(r), vocab(v) {
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / 4;
    const int per = ((v + kRanks - 1) / kRanks + 3) / 4 * 4;
    begin = rank == 0 ? 0 : min(v, rank * per + lead);
    end = rank == kRanks - 1 ? v : min(v, (rank + 1) * per + lead);
  }
  template <typename F> __device__ __forceinline__ void each(F f) const {
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(row + begin) & 15)) & 15) / 4;
    const int first = min(end, begin + lead), quads = (end - first) / 4;
    if (begin + (int)threadIdx.x < first) f(begin + (int)threadIdx.x, clean(row[begin + threadIdx.x]));
    const float4* wide = reinterpret_cast<const float4*>(row + first);
    for (int g = threadIdx.x; g < quads; g += 4 * kThreads) {
      float4 v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (g + j * kThreads < quads) v[j] = wide[g + j * kThreads];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (g + j * kThreads < quads) {
          const int i = first + 4 * (g + j * kThreads);
          f(i, clean(v[j].x)), f(i + 1, clean(v[j].y)), f(i + 2, clean(v[j].z)), f(i + 3, clean(v[j].w));
        }
    }
    const int tail = first + 4 * quads + (int)threadIdx.x;
    if (tail < end) f(tail, clean(row[tail]));
  }
};

struct Shared {
  unsigned long long bins[2][kBins];       // this block's, in one of two buffers in turn: a rank may still read the last round's
  unsigned long long scan[kWarps];
  double sums[2][kRanks];
  Best bests[2][kRanks];
  float tops[2][kRanks];
  int counts[2][kRanks];
  float warp_float[kWarps];
  double warp_double[kWarps];
  Best warp_best[kWarps];
  int warp_int[kWarps];
  int found;
  unsigned long long above;
};

// Values of all threads of the cluster, joined in a fixed order: every rank writes its block's into slot `rank` of every rank's array.  `turn`
// alternates, so that no rank's next value overtakes a slower rank's reads.
__device__ Best cluster_best(Shared& s, cg::cluster_group& cluster, int rank, Best v, int turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    Best other;
    other.value = __shfl_xor_sync(0xffffffffu, v.value, o);
    other.index = __shfl_xor_sync(0xffffffffu, v.index, o);
    v = better(v, other);
  }
  if (lane == 0) s.warp_best[warp] = v;
  __syncthreads();
  if (threadIdx.x < kRanks) {
    Best b = s.warp_best[0];
    for (int w = 1; w < kWarps; ++w) b = better(b, s.warp_best[w]);
    cluster.map_shared_rank(&s, threadIdx.x)->bests[turn][rank] = b;
  }
  cluster.sync();
  Best b = s.bests[turn][0];
  for (int r = 1; r < kRanks; ++r) b = better(b, s.bests[turn][r]);
  return b;
}

__device__ double cluster_sum(Shared& s, cg::cluster_group& cluster, int rank, double v, int turn) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) s.warp_double[warp] = v;
  __syncthreads();
  if (threadIdx.x < kRanks) {
    double b = 0.0;
    for (int w = 0; w < kWarps; ++w) b += s.warp_double[w];
    cluster.map_shared_rank(&s, threadIdx.x)->sums[turn][rank] = b;
  }
  cluster.sync();
  double b = 0.0;
  for (int r = 0; r < kRanks; ++r) b += s.sums[turn][r];
  return b;
}

// One round of a search from the largest key down: with this round's bins filled on every rank, the highest bin at which the sum over it and
// all higher ones exceeds `limit` (bin 0 where none does); `above`: the sum over the higher ones.
__device__ int find_bin(Shared& s, cg::cluster_group& cluster, int buffer, unsigned long long limit, unsigned long long& above) {
  cluster.sync();
  constexpr int kEach = kBins / kThreads;
  unsigned long long mine[kEach] = {};
  // thread t holds the bins kBins - 1 - (t kEach + j): the largest keys first
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    for (int r = 0; r < kRanks; ++r) mine[j] += cluster.map_shared_rank(&s, r)->bins[buffer][kBins - 1 - (threadIdx.x * kEach + j)];
  unsigned long long sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) sum += mine[j];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += other;
  }
  if (threadIdx.x == 0) s.found = -1;
  if (lane == 31) s.scan[warp] = before;
  __syncthreads();
  before -= sum;
  for (int w = 0; w < warp; ++w) before += s.scan[w];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (before <= limit && before + mine[j] > limit) {          // true at one bin at most
      s.found = kBins - 1 - (threadIdx.x * kEach + j);
      s.above = before;
    }
    before += mine[j];
  }
  if (threadIdx.x == kThreads - 1 && before <= limit) {
    s.found = 0;
    s.above = before - mine[kEach - 1];
  }
  __syncthreads();
  above = s.above;
  return s.found;
}

// The largest index bound with at most `need` entries below it for which `is` holds, over the whole row: ranks hold its parts in order.
template <typename F>
__device__ int index_bound(Shared& s, cg::cluster_group& cluster, int rank, const Part& part, int need, F is) {
  int count = 0;
  part.each([&](int i, float x) { count += is(i, x) ? 1 : 0; });
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) count += __shfl_xor_sync(0xffffffffu, count, o);
  cluster.sync();                                   // (the slots below may still be read)
  if (lane == 0) s.warp_int[warp] = count;
  __syncthreads();
  if (threadIdx.x < kRanks) {
    int all = 0;
    for (int w = 0; w < kWarps; ++w) all += s.warp_int[w];
    cluster.map_shared_rank(&s, threadIdx.x)->counts[0][rank] = all;
  }
  cluster.sync();
  int before = 0, owner = kRanks - 1;
  for (int r = 0; r < kRanks; ++r) {
    if (before + s.counts[0][r] > need) {
      owner = r;
      break;
    }
    if (r + 1 < kRanks) before += s.counts[0][r];
  }
  if (rank == owner) {
    // the entry number `need` (from 0) of those for which `is` holds is the first that is not taken
    if (threadIdx.x == 0) s.found = part.vocab;
    __syncthreads();
    for (int base = part.begin; base < part.end; base += kThreads) {
      const int i = base + (int)threadIdx.x;
      const bool mine = i < part.end && is(i, clean(part.row[i]));
      const unsigned votes = __ballot_sync(0xffffffffu, mine);
      if (lane == 0) s.warp_int[warp] = __popc(votes);
      __syncthreads();
      int place = before + __popc(votes & ((1u << lane) - 1u));
      for (int w = 0; w < warp; ++w) place += s.warp_int[w];
      if (mine && place == need) s.found = i;
      for (int w = 0; w < kWarps; ++w) before += s.warp_int[w];
      __syncthreads();
      if (before > need) break;
    }
    if (threadIdx.x < kRanks) cluster.map_shared_rank(&s, threadIdx.x)->counts[1][0] = s.found;
  }
  cluster.sync();
  return s.counts[1][0];
}

__device__ __forceinline__ int request_of(const int* draft_start, int requests, int row) {
  int low = 0, high = requests - 1;               // the last request whose first row is not behind `row`
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (draft_start[mid] + mid <= row) low = mid; else high = mid - 1;
  }
  return low;
}

// Cluster: a row of logits.
__global__ void __cluster_dims__(kRanks, 1, 1) __launch_bounds__(kThreads)
verify_rows_kernel(const float* __restrict__ logits, int vocab, const int* __restrict__ drafts, const int* __restrict__ draft_start, int requests,
                   int total, const float* __restrict__ uniforms, const float* __restrict__ draft_probs, const Record* __restrict__ records,
                   const int* __restrict__ slots, Row* __restrict__ out, float* __restrict__ target_probs, int shift) {
  __shared__ Shared s;
  grid_dependency_wait();
  grid_dependency_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), r = (int)(blockIdx.x / kRanks);
  const int request = request_of(draft_start, requests, r);
  const int draft = r - request;                               // (the row's place among all drafts, if it has one)
  const bool drafted = draft >= 0 && draft < draft_start[request + 1] && draft < total;
  Record rec{0.f, 1.f, 0};
  if (records != nullptr) rec = records[slots[request]];
  const bool greedy = !(rec.temperature > 0.f);
  const bool top_k = rec.top_k > 0 && rec.top_k < vocab, top_p = rec.top_p < 1.f;
  const Part part(logits + (size_t)r * vocab, vocab, rank);

  Best best{-INFINITY, 0x7fffffff};
  double sum = 0.0;
  // without filters one pass gives the sum too: relative to the thread's own running maximum
  const bool one_pass = !greedy && !top_k && !top_p;
  float partial = 0.f;
  part.each([&](int i, float x) {
    if (x > best.value) {
      if (one_pass && best.value > -INFINITY) partial *= expf(exponent(best.value, x, rec.temperature));
      best = Best{x, i};
    }
    if (one_pass && x > -INFINITY) partial += expf(exponent(x, best.value, rec.temperature));
  });
  const float mine = best.value;
  best = cluster_best(s, cluster, rank, best, 0);
  const float top = best.value;
  const bool nothing = top == -INFINITY;            // every entry is masked: no token has a probability
  Row row{};
  row.top = top;
  row.best = best.index == 0x7fffffff ? 0 : best.index;
  row.bound = vocab;
  const int token = drafted ? drafts[draft] : 0;
  const bool known = drafted && token >= 0 && token < vocab;
  float p = 0.f;
  if (greedy) {
    p = known && !nothing && token == row.best ? 1.f : 0.f;
    row.passes = p > 0.f;
  } else if (!nothing) {
    const float temperature = rec.temperature;
    // of the entries near the largest, which make up most of a mass, the exponential in float64: which entry a border falls on then does not hang
    // on the rounding of the largest terms
    auto weight = [&](float x) {
      const float e = exponent(x, top, temperature);
      return e > -7.f ? exp(x == top ? 0.0 : ((double)x - (double)top) / (double)temperature) : (double)expf(e);
    };
    if (one_pass) {
      sum = mine == -INFINITY ? 0.0 : (double)(partial * expf(exponent(mine, top, temperature)));
      sum = cluster_sum(s, cluster, rank, sum, 0);
    } else {
      int buffer = 0;
      auto clear = [&](int b) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) s.bins[b][i] = 0;
        __syncthreads();
      };
      if (top_k) {
        unsigned prefix = 0;
        unsigned long long rest = (unsigned long long)rec.top_k - 1, above = 0;
#pragma unroll 1
        for (int round = 0; round < 3; ++round) {
          const int low = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
          clear(buffer);
          part.each([&](int, float x) {
            const unsigned key = order_key(x);
            if (round == 0 || (key >> (low + bits)) == prefix) atomicAdd(&s.bins[buffer][(key >> low) & ((1u << bits) - 1u)], 1ull);
          });
          const int bin = find_bin(s, cluster, buffer, rest, above);
          rest -= above;
          prefix = (prefix << bits) | (unsigned)bin;
          buffer ^= 1;
        }
        row.thr = prefix;
        // rest: how many of the entries equal to the threshold stand before the last kept one
        const unsigned thr = row.thr;
        row.bound = index_bound(s, cluster, rank, part, (int)rest + 1, [&](int, float x) { return order_key(x) == thr; });
      }
      const unsigned thr_k = row.thr;
      const int bound_k = row.bound;
      auto kept = [&](unsigned key, int i) { return key > thr_k || (key == thr_k && i < bound_k); };
      if (top_p) {
        const double unit = (double)(1ull << shift);
        auto fixed = [&](float x) { return (unsigned long long)__double2ll_rn(weight(x) * unit); };
        double all = 0.0;
        unsigned prefix = 0;
        unsigned long long limit = 0, above = 0, so_far = 0;
        {
          double z = 0.0;
          part.each([&](int i, float x) {
            if (kept(order_key(x), i)) z += (double)fixed(x);
          });
          all = cluster_sum(s, cluster, rank, z, 0);
        }
        limit = (unsigned long long)floor((double)rec.top_p * all);
#pragma unroll 1
        for (int round = 0; round < 3; ++round) {
          const int low = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
          clear(buffer);
          part.each([&](int i, float x) {
            const unsigned key = order_key(x);
            if ((round == 0 || (key >> (low + bits)) == prefix) && kept(key, i)) {
              const unsigned long long w = fixed(x);
              if (w != 0) atomicAdd(&s.bins[buffer][(key >> low) & ((1u << bits) - 1u)], w);
            }
          });
          const int bin = find_bin(s, cluster, buffer, limit - so_far, above);
          so_far += above;
          prefix = (prefix << bits) | (unsigned)bin;
          buffer ^= 1;
        }
        if (prefix >= thr_k) {
          // of the entries equal to the threshold those stay whose mass before is at most the limit
          const float x = __uint_as_float((prefix & 0x80000000u) ? (prefix & 0x7fffffffu) : ~prefix);
          const unsigned long long each = fixed(x);
          const unsigned long long room = each > 0 ? (limit - so_far) / each + 1 : 1;
          const int most = room > (unsigned long long)vocab ? vocab : (int)room;
          row.thr = prefix;
          const int outer = prefix == thr_k ? bound_k : vocab;
          const unsigned thr = prefix;
          row.bound = min(outer, index_bound(s, cluster, rank, part, most, [&](int i, float v) { return order_key(v) == thr && i < outer; }));
        }
      }
      const unsigned thr = row.thr;
      const int bound = row.bound;
      part.each([&](int i, float x) {
        const unsigned key = order_key(x);
        if (key > thr || (key == thr && i < bound)) sum += weight(x);
      });
      sum = cluster_sum(s, cluster, rank, sum, 1);
    }
    row.inverse = sum > 0.0 ? (float)(1.0 / sum) : 0.f;
    if (known) {
      const float x = clean(part.row[token]);
      const unsigned key = order_key(x);
      if (x > -INFINITY && (key > row.thr || (key == row.thr && token < row.bound))) p = expf(exponent(x, top, temperature)) * row.inverse;
      const float q = draft_probs != nullptr ? draft_probs[(size_t)draft * vocab + token] : 1.f;
      row.passes = uniforms[draft] * q < p;
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    out[r] = row;
    if (drafted && target_probs != nullptr) target_probs[draft] = p;
  }
  cluster.sync();                    // no block leaves while another may reach into its shared memory
}

// Cluster: a request.
__global__ void __cluster_dims__(kRanks, 1, 1) __launch_bounds__(kThreads)
verify_choose_kernel(const float* __restrict__ logits, int vocab, const int* __restrict__ drafts, const int* __restrict__ draft_start,
                     const float* __restrict__ noise, const float* __restrict__ draft_probs, const Record* __restrict__ records,
                     const int* __restrict__ slots, const Row* __restrict__ rows, int total, int* __restrict__ accepted,
                     int* __restrict__ next_token) {
  __shared__ Shared s;
  grid_dependency_wait();
  grid_dependency_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), request = (int)(blockIdx.x / kRanks);
  const int first = min(max(draft_start[request], 0), total), count = min(max(draft_start[request + 1], first), total) - first;
  int passed = count;
  for (int base = 0; base < count && passed == count; base += 32) {          // (every warp for itself)
    const int i = base + (int)(threadIdx.x & 31);
    const unsigned failed = __ballot_sync(0xffffffffu, i < count && rows[first + request + i].passes == 0);
    if (failed != 0) passed = base + __ffs((int)failed) - 1;
  }
  const int r = first + request + passed;
  const Row row = rows[r];
  Record rec{0.f, 1.f, 0};
  if (records != nullptr) rec = records[slots[request]];
  const bool greedy = !(rec.temperature > 0.f);
  int chosen = row.best;
  if (!greedy && row.inverse > 0.f) {
    const bool rejected = passed < count;
    const float* q = rejected && draft_probs != nullptr ? draft_probs + (size_t)(first + passed) * vocab : nullptr;
    const int token = rejected ? drafts[first + passed] : -1;
    const float* e = noise + (size_t)request * vocab;
    const Part part(logits + (size_t)r * vocab, vocab, rank);
    auto race = [&](bool residual) {
      Best best{-INFINITY, 0x7fffffff};
      for (int i = part.begin + (int)threadIdx.x; i < part.end; i += kThreads) {
        const float x = clean(part.row[i]);
        const unsigned key = order_key(x);
        if (!(x > -INFINITY) || !(key > row.thr || (key == row.thr && i < row.bound))) continue;
        float left = expf(exponent(x, row.top, rec.temperature)) * row.inverse;
        if (residual) left = q != nullptr ? left - q[i] : i == token ? 0.f : left;
        if (!(left > 0.f)) continue;
        const float value = left / e[i];
        if (value > best.value) best = Best{value, i};
      }
      return best;
    };
    Best best = cluster_best(s, cluster, rank, race(rejected), 0);
    // nothing of the target is left where the draft's probabilities cover it but for rounding: then the target itself is drawn from
    if (rejected && best.index == 0x7fffffff) best = cluster_best(s, cluster, rank, race(false), 1);
    if (best.index != 0x7fffffff) chosen = best.index;
  }
  if (rank == 0 && threadIdx.x == 0) {
    accepted[request] = passed;
    next_token[request] = chosen;
  }
  cluster.sync();
}

}  // namespace verify
}  // namespace ms

using namespace ms;

// Bytes of scratch that ms_verify_drafts needs for a row of logits.
MS_EXPORT int ms_verify_row_bytes() { return (int)sizeof(verify::Row); }

// logits [n_drafts + requests, vocab] float32: request r's rows are draft_start[r] + r .. draft_start[r + 1] + r.  drafts, uniforms [n_drafts];
// draft_start [requests + 1]; draft_probs [n_drafts, vocab] or null; noise [requests, vocab]; records [slots, 8] 32-bit words (temperature,
// top_p as float, top_k) or null for argmax, slot_of_request [requests].  accepted, next_token [requests]; target_probs [n_drafts] or null.
MS_EXPORT int ms_verify_drafts(const float* logits, int vocab, const int* drafts, const int* draft_start, int requests, int n_drafts,
                               const float* uniforms, const float* noise, const float* draft_probs, const void* records,
                               const int* slot_of_request, int* accepted, int* next_token, float* target_probs, void* scratch,
                               cudaStream_t stream) {
  using namespace ms::verify;
  if (requests == 0) return 0;
  MS_REQUIRE(requests > 0 && n_drafts >= 0 && vocab > 0 && vocab <= (1 << 26), "verify_drafts: %d requests, %d drafts, vocabulary %d", requests, n_drafts, vocab);
  MS_REQUIRE((long long)requests + n_drafts <= 2147483647LL / kRanks, "verify_drafts: %d drafts of %d requests in one call are too many", n_drafts, requests);
  MS_REQUIRE(records == nullptr || (slot_of_request != nullptr && noise != nullptr && (uniforms != nullptr || n_drafts == 0)),
             "verify_drafts: sampling records need slots, uniforms and noise");
  MS_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 8 == 0, "verify_drafts: scratch is missing or not aligned");
  int shift = 62;              // masses are sums of up to `vocab` weights of at most one, in units of 2^-shift
  while (shift > 0 && ((long long)vocab >> (62 - shift)) != 0) --shift;
  ms::launch(verify_rows_kernel, dim3((unsigned)((n_drafts + requests) * kRanks)), dim3(kThreads), 0, stream, logits, vocab, drafts, draft_start,
             requests, n_drafts, uniforms, draft_probs, (const Record*)records, slot_of_request, (Row*)scratch, target_probs, shift);
  MS_CHECK_LAUNCH("verify_drafts (rows)");
  ms::launch(verify_choose_kernel, dim3((unsigned)(requests * kRanks)), dim3(kThreads), 0, stream, logits, vocab, drafts, draft_start, noise,
             draft_probs, (const Record*)records, slot_of_request, (const Row*)scratch, n_drafts, accepted, next_token);
  MS_CHECK_LAUNCH("verify_drafts (choice)");
  return 0;
}
