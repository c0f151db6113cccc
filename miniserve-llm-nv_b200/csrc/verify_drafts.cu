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
//
// The filters' borders are found in two passes: counts and masses in 2,048 bins of 1/64 of (max - x) / temperature (equal steps in the exponent spread the
// entries; the bits of the numbers would put most into a few bins, whose atomics wait for one another), then the entries of the bin that holds the border,
// ranked one by one.  Masses are sums of integers (units of 2^-44 of the largest weight at 151,936 entries), so that their order changes nothing.  Where
// a bin holds more than the list takes (equal logits) or the border lies behind the bins, three rounds over the bits of the numbers find it.
#include "common.cuh"

#include <cooperative_groups.h>

namespace ms {
namespace verify {

namespace cg = cooperative_groups;

constexpr int kRanks = 8, kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 2048;              // also of one round of a search over 32-bit keys: eleven, eleven and ten bits
constexpr float kBinsToOne = 64.f;
constexpr int kListed = 1024;            // entries of a border's bin that are ranked one by one

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
  int best;                // argmax (temperature 0)
  int passes;              // its draft passes
  int reserved[2];
};

__device__ __forceinline__ unsigned order_key(float f) {
  const unsigned u = __float_as_uint(f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float number_of(unsigned key) { return __uint_as_float((key & 0x80000000u) ? (key & 0x7fffffffu) : ~key); }

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
// e^((x - top) / temperature) with per = log2 e / temperature: of the sums and the quotients, where a weight that is off by 2^-21 of itself (e^-10 and
// below; the large ones are off by 2^-22) changes nothing but a choice between two quotients that near.
__device__ __forceinline__ float quick_weight(float x, float top, float per) {
  float w;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(x == top ? 0.f : (x - top) * per));
  return w;
}

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
  // f(x, first): sixteen entries; number 4 j + e has the index first + 4 kThreads j + e, and is -inf where there is none.
  template <typename F> __device__ __forceinline__ void sixteen(F f) const {
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(row + begin) & 15)) & 15) / 4;
    const int first = min(end, begin + lead), quads = (end - first) / 4;
    const float4* wide = reinterpret_cast<const float4*>(row + first);
    for (int g = threadIdx.x; g < quads; g += 4 * kThreads) {
      float x[16];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (g + j * kThreads < quads) v = wide[g + j * kThreads];
        x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = clean(x[j]);
      f(x, first + 4 * g);
    }
    // the ragged ends: up to three entries before the first boundary and behind the last
    const int ends = first - begin + (end - first - 4 * quads);
    if ((int)threadIdx.x < ends) {
      const int i = (int)threadIdx.x < first - begin ? begin + (int)threadIdx.x : first + 4 * quads + (int)threadIdx.x - (first - begin);
      float x[16];
#pragma unroll
      for (int j = 1; j < 16; ++j) x[j] = -INFINITY;
      x[0] = clean(row[i]);
      f(x, i);
    }
  }
  template <typename F> __device__ __forceinline__ void each(F f) const {      // f(index, x) of every entry that is not masked
    sixteen([&](const float (&x)[16], int first) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (x[j] > -INFINITY) f(first + (j / 4) * 4 * kThreads + j % 4, x[j]);
    });
  }
};

struct Entry {
  float x;
  int index;
  unsigned long long mass;
};

struct Joined {
  Best bests[2][kRanks];
  Best warp_best[kWarps];
};

struct Shared : Joined {
  unsigned long long mass[kBins];
  unsigned count[kBins];
  Entry list[kListed];
  int listed;
  unsigned long long scan[kWarps];
  double sums[kRanks];
  int counts[kRanks];
  double warp_double[kWarps];
  int warp_int[kWarps];
  int found, bin, bound;
  unsigned thr;
  unsigned long long above, kept;
};

// Values of all threads of the cluster, joined in a fixed order: every rank writes its block's into slot `rank` of every rank's array.  `turn`
// alternates where it is called twice, so that no rank's next value overtakes a slower rank's reads.
__device__ Best cluster_best(Joined& s, cg::cluster_group& cluster, int rank, Best v, int turn) {
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

__device__ double cluster_sum(Shared& s, cg::cluster_group& cluster, int rank, double v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) s.warp_double[warp] = v;
  __syncthreads();
  if (threadIdx.x < kRanks) {
    double b = 0.0;
    for (int w = 0; w < kWarps; ++w) b += s.warp_double[w];
    cluster.map_shared_rank(&s, threadIdx.x)->sums[rank] = b;
  }
  cluster.sync();
  double b = 0.0;
  for (int r = 0; r < kRanks; ++r) b += s.sums[r];
  return b;
}

// Over this block's bins from the first on: the first at which the running sum exceeds `limit` (kBins where none does); `above`: the sum before it.
template <typename T>
__device__ int first_over(Shared& s, const T* bins, unsigned long long limit, unsigned long long& above) {
  constexpr int kEach = kBins / kThreads;
  unsigned long long mine[kEach], sum = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    mine[j] = bins[threadIdx.x * kEach + j];
    sum += mine[j];
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long before = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += other;
  }
  __syncthreads();
  if (lane == 31) s.scan[warp] = before;
  if (threadIdx.x == 0) s.found = kBins;
  __syncthreads();
  before -= sum;
  for (int w = 0; w < warp; ++w) before += s.scan[w];
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    if (before <= limit && before + mine[j] > limit) {          // true at one bin at most
      s.found = (int)threadIdx.x * kEach + j;
      s.above = before;
    }
    before += mine[j];
  }
  if (threadIdx.x == kThreads - 1 && before <= limit) s.above = before;
  __syncthreads();
  above = s.above;
  return s.found;
}

// All ranks' bins added up in rank 0's, which calls this.
template <typename T>
__device__ void gather_bins(cg::cluster_group& cluster, T* bins) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) {
    T sum = bins[i];
#pragma unroll
    for (int r = 1; r < kRanks; ++r) sum += *cluster.map_shared_rank(bins + i, r);
    bins[i] = sum;
  }
  __syncthreads();
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
    cluster.map_shared_rank(&s, threadIdx.x)->counts[rank] = all;
  }
  cluster.sync();
  int before = 0, owner = kRanks - 1;
  for (int r = 0; r < kRanks; ++r) {
    if (before + s.counts[r] > need) {
      owner = r;
      break;
    }
    if (r + 1 < kRanks) before += s.counts[r];
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
    if (threadIdx.x < kRanks) cluster.map_shared_rank(&s, threadIdx.x)->bound = s.found;
  }
  cluster.sync();
  return s.bound;
}

__device__ __forceinline__ int request_of(const int* draft_start, int requests, int row) {
  int low = 0, high = requests - 1;               // the last request whose first row is not behind `row`
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (draft_start[mid] + mid <= row) low = mid; else high = mid - 1;
  }
  return low;
}

// A row's weights as sums of integers: units of 2^-shift of the largest.  Of the entries near the largest, which make up most of a mass, the exponential in
// float64: which entry a border falls on then does not hang on the rounding of the largest terms.
struct Weights {
  float top, temperature, to_bin;
  double unit;
  __device__ Weights(float t, float heat, int shift) : top(t), temperature(heat), to_bin(kBinsToOne / heat), unit((double)(1ull << shift)) {}
  __device__ __forceinline__ unsigned long long of(float x) const {
    const float e = exponent(x, top, temperature);
    if (e > -7.f) return (unsigned long long)__double2ll_rn(exp(x == top ? 0.0 : ((double)x - (double)top) / (double)temperature) * unit);
    return (unsigned long long)__float2ll_rn(expf(e) * (float)unit);
  }
  // (entries of one bin have a higher number than those of the bins before it are smaller than they; behind the last bin: kBins)
  __device__ __forceinline__ int bin(float x) const {
    const float t = x == top ? 0.f : (top - x) * to_bin;
    return t < (float)kBins ? (int)t : kBins;
  }
};

// The kept set of a row with filters by two passes; false on every rank where the border's bin is too full or the border lies behind the bins.  On
// rank 0 row.thr, row.bound and `total`, the kept mass, are set.
__device__ bool filter_by_bins(Shared& s, cg::cluster_group& cluster, int rank, const Part& part, const Weights& weights, const Record& rec, bool top_k,
                               bool top_p, Row& row, unsigned long long& total) {
  for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0, s.count[i] = 0;
  if (threadIdx.x == 0) s.listed = 0;
  __syncthreads();
  part.each([&](int, float x) {
    const int bin = weights.bin(x);
    if (bin >= kBins) return;                   // (less than e^-32 of the largest: no mass)
    const unsigned long long w = weights.of(x);
    if (w != 0) atomicAdd(&s.mass[bin], w);
    if (top_k) atomicAdd(&s.count[bin], 1u);
  });
  cluster.sync();
  // rank 0 alone searches; `bin` says which bin's entries all ranks are to send it: -1 none, -2 give up
  unsigned long long limit = 0, above = 0, before = 0;       // of the mass
  int need = 0;                                               // top_k: how many of the bin's entries stay
  if (rank == 0) {
    gather_bins(cluster, s.mass);
    if (top_k) gather_bins(cluster, s.count);
    int bin;
    if (top_k) {
      bin = first_over(s, s.count, (unsigned long long)rec.top_k - 1, before);
      need = rec.top_k - (int)before;
      if (bin == kBins) bin = -2;
    } else {
      first_over(s, s.mass, ~0ull - 1, total);                // (all of it)
      limit = (unsigned long long)floor((double)rec.top_p * (double)total);
      bin = first_over(s, s.mass, limit, above);
      if (bin == kBins) bin = -2;
    }
    if (threadIdx.x < kRanks) cluster.map_shared_rank(&s, threadIdx.x)->bin = bin;
  }
#pragma unroll 1
  for (int round = 0; round < 2; ++round) {
    cluster.sync();
    const int bin = s.bin;
    if (bin < 0) break;
    Shared* first = cluster.map_shared_rank(&s, 0);
    part.each([&](int i, float x) {
      if (weights.bin(x) != bin) return;
      const int at = atomicAdd(&first->listed, 1);
      if (at < kListed) first->list[at] = Entry{x, i, weights.of(x)};
    });
    cluster.sync();
    if (rank == 0) {
      const int listed = s.listed;
      int next = listed > kListed ? -2 : -1;
      if (next == -1) {
        const bool by_count = top_k && round == 0;
        if (by_count) {
          // the mass before this bin, then that of the entries that stay
          unsigned long long part_mass = 0;
          for (int i = threadIdx.x; i < bin; i += kThreads) part_mass += s.mass[i];
          if (threadIdx.x == 0) s.above = 0, s.kept = 0;
          __syncthreads();
          if (part_mass != 0) atomicAdd(&s.above, part_mass);
          __syncthreads();
          above = s.above;
        }
        // an entry's place in the bin, and the mass of those before it; of those that stay the last one is the border
        auto solve = [&](bool count, bool mass, int most) {
          __syncthreads();
          if (threadIdx.x == 0) s.found = -1, s.kept = 0;
          __syncthreads();
          constexpr int kEach = kListed / kThreads;
          int place[kEach];
#pragma unroll
          for (int j = 0; j < kEach; ++j) {
            const int a = (int)threadIdx.x + j * kThreads;
            place[j] = -2;
            if (a >= listed) continue;
            const Entry mine = s.list[a];
            unsigned long long sum = 0;
            int ahead = 0;
            for (int c = 0; c < listed; ++c) {
              const Entry other = s.list[c];
              if (other.x > mine.x || (other.x == mine.x && other.index < mine.index)) ++ahead, sum += other.mass;
            }
            place[j] = ahead;
            if ((!count || ahead < most) && (!mass || above + sum <= limit)) {
              atomicAdd(&s.kept, mine.mass);
              atomicMax(&s.found, ahead);
            }
          }
          __syncthreads();
#pragma unroll
          for (int j = 0; j < kEach; ++j)
            if (place[j] == s.found) {
              const Entry mine = s.list[threadIdx.x + j * kThreads];
              s.thr = order_key(mine.x), s.bound = mine.index + 1;
            }
          __syncthreads();
          total = above + s.kept;
        };
        if (by_count) {
          solve(true, false, need);
          if (top_p) {
            limit = (unsigned long long)floor((double)rec.top_p * (double)total);
            if (limit >= above) {
              solve(true, true, need);              // the nucleus ends in this bin
            } else {
              unsigned long long in_front;
              next = first_over(s, s.mass, limit, in_front);
              above = in_front;
            }
          }
        } else {
          solve(false, true, 0);
        }
      }
      __syncthreads();
      if (threadIdx.x == 0) s.listed = 0;
      if (threadIdx.x < kRanks) cluster.map_shared_rank(&s, threadIdx.x)->bin = next;
      row.thr = s.thr, row.bound = s.bound;
    }
  }
  cluster.sync();
  return s.bin != -2;
}

// The same by three rounds over the bits of the numbers, the largest first, which takes any row.
__device__ void filter_by_bits(Shared& s, cg::cluster_group& cluster, int rank, const Part& part, const Weights& weights, const Record& rec, bool top_k,
                               bool top_p, Row& row, unsigned long long& total) {
  row.thr = 0, row.bound = part.vocab;
  unsigned prefix = 0;
  int most = 0;
  if (top_k) {
    unsigned long long rest = (unsigned long long)rec.top_k - 1;
#pragma unroll 1
    for (int round = 0; round < 3; ++round) {
      const int low = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
      for (int i = threadIdx.x; i < kBins; i += kThreads) s.count[i] = 0;
      __syncthreads();
      part.each([&](int, float x) {
        const unsigned key = order_key(x);
        if (round == 0 || (key >> (low + bits)) == prefix) atomicAdd(&s.count[kBins - 1 - ((key >> low) & ((1u << bits) - 1u))], 1u);
      });
      cluster.sync();
      if (rank == 0) {
        gather_bins(cluster, s.count);
        unsigned long long before;
        const int bin = first_over(s, s.count, rest, before);
        rest -= before;
        if (threadIdx.x < kRanks) {
          Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
          other->bin = bin, other->bound = (int)rest + 1;
        }
      }
      cluster.sync();
      if (s.bin == kBins) break;                     // fewer entries than top_k: all stay
      prefix = (prefix << bits) | (unsigned)(kBins - 1 - s.bin);
      most = s.bound;
    }
    if (s.bin != kBins) {
      const unsigned thr = prefix;
      row.thr = thr;
      row.bound = index_bound(s, cluster, rank, part, most, [&](int, float x) { return order_key(x) == thr; });
    }
  }
  const unsigned thr_k = row.thr;
  const int bound_k = row.bound;
  auto kept = [&](unsigned key, int i) { return key > thr_k || (key == thr_k && i < bound_k); };
  if (!top_p) {
    double sum = 0.0;
    part.each([&](int i, float x) {
      if (kept(order_key(x), i)) sum += (double)weights.of(x);
    });
    total = (unsigned long long)cluster_sum(s, cluster, rank, sum);
    return;
  }
  unsigned long long limit = 0, above = 0;           // (rank 0's)
  prefix = 0;
#pragma unroll 1
  for (int round = 0; round < 3; ++round) {
    const int low = round == 0 ? 21 : round == 1 ? 10 : 0, bits = round == 2 ? 10 : 11;
    cluster.sync();                                  // (rank 0 may still read)
    for (int i = threadIdx.x; i < kBins; i += kThreads) s.mass[i] = 0;
    __syncthreads();
    part.each([&](int i, float x) {
      const unsigned key = order_key(x);
      if ((round == 0 || (key >> (low + bits)) == prefix) && kept(key, i)) {
        const unsigned long long w = weights.of(x);
        if (w != 0) atomicAdd(&s.mass[kBins - 1 - ((key >> low) & ((1u << bits) - 1u))], w);
      }
    });
    cluster.sync();
    if (rank == 0) {
      gather_bins(cluster, s.mass);
      if (round == 0) {
        first_over(s, s.mass, ~0ull - 1, total);
        limit = (unsigned long long)floor((double)rec.top_p * (double)total);
      }
      unsigned long long before;
      const int bin = min(first_over(s, s.mass, limit - above, before), kBins - 1);
      above += before;
      if (round == 2) {
        // of the equal entries at the border those stay whose mass before is at most the limit
        const unsigned long long each = weights.of(number_of((prefix << bits) | (unsigned)(kBins - 1 - bin)));
        const unsigned long long room = each > 0 ? (limit - above) / each + 1 : 1, there = each > 0 ? s.mass[bin] / each : 0;
        const unsigned long long stay = room < there ? room : there;
        total = above + stay * each;
        most = room < (unsigned long long)part.vocab ? (int)room : part.vocab;
      }
      if (threadIdx.x < kRanks) {
        Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
        other->bin = bin, other->bound = most;
      }
    }
    cluster.sync();
    prefix = (prefix << bits) | (unsigned)(kBins - 1 - s.bin);
    most = s.bound;
  }
  if (prefix >= thr_k) {
    const unsigned thr = prefix;
    const int outer = thr == thr_k ? bound_k : part.vocab;
    row.thr = thr;
    row.bound = min(outer, index_bound(s, cluster, rank, part, most, [&](int i, float x) { return order_key(x) == thr && i < outer; }));
  }
}

// Cluster: a row of logits.
__global__ void __cluster_dims__(kRanks, 1, 1) __launch_bounds__(kThreads, 2)
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
  const int token = drafted ? drafts[draft] : 0;
  const bool known = drafted && token >= 0 && token < vocab;
  Row row{};
  row.bound = vocab;
  float p = 0.f;
  Best best{-INFINITY, 0x7fffffff};
  if (greedy) {
    part.sixteen([&](const float (&x)[16], int first) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (x[j] > -INFINITY) best = better(best, Best{x[j], first + (j / 4) * 4 * kThreads + j % 4});
    });
    best = cluster_best(s, cluster, rank, best, 0);
    row.best = best.index == 0x7fffffff ? 0 : best.index;
    p = known && best.index == token ? 1.f : 0.f;
    row.passes = p > 0.f;
  } else {
    // the largest, and without filters in the same pass the sum relative to this thread's running maximum
    const bool one_pass = !top_k && !top_p;
    const float per = 1.4426950408889634f / rec.temperature;
    float partial = 0.f;
    part.sixteen([&](const float (&x)[16], int) {
      float m = x[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) m = fmaxf(m, x[j]);
      if (m > best.value) {
        if (one_pass && best.value > -INFINITY) partial *= quick_weight(best.value, m, per);
        best.value = m;
      }
      if (one_pass && best.value > -INFINITY) {
        float sum[4] = {};
#pragma unroll
        for (int j = 0; j < 16; ++j) sum[j & 3] += quick_weight(x[j], best.value, per);
        partial += (sum[0] + sum[1]) + (sum[2] + sum[3]);
      }
    });
    const float mine = best.value;
    row.top = cluster_best(s, cluster, rank, best, 0).value;
    if (row.top > -INFINITY) {                   // (else every entry is masked: no token has a probability)
      double sum = 0.0;                          // (rank 0's)
      if (one_pass) {
        sum = cluster_sum(s, cluster, rank, mine == -INFINITY ? 0.0 : (double)(partial * quick_weight(mine, row.top, per)));
      } else {
        const Weights weights(row.top, rec.temperature, shift);
        unsigned long long mass = 0;
        if (!filter_by_bins(s, cluster, rank, part, weights, rec, top_k, top_p, row, mass))
          filter_by_bits(s, cluster, rank, part, weights, rec, top_k, top_p, row, mass);
        sum = (double)mass / weights.unit;
      }
      row.inverse = sum > 0.0 ? (float)(1.0 / sum) : 0.f;
      if (known) {
        const float x = clean(part.row[token]);
        const unsigned key = order_key(x);
        if (x > -INFINITY && (key > row.thr || (key == row.thr && token < row.bound))) p = expf(exponent(x, row.top, rec.temperature)) * row.inverse;
        const float q = draft_probs != nullptr ? draft_probs[(size_t)draft * vocab + token] : 1.f;
        row.passes = uniforms[draft] * q < p;
      }
    }
  }
  if (rank == 0 && threadIdx.x == 0) {
    out[r] = row;
    if (drafted && target_probs != nullptr) target_probs[draft] = p;
  }
  cluster.sync();                    // no block leaves while another may reach into its shared memory
}

// Cluster: a request.
__global__ void __cluster_dims__(kRanks, 1, 1) __launch_bounds__(kThreads, 2)
verify_choose_kernel(const float* __restrict__ logits, int vocab, const int* __restrict__ drafts, const int* __restrict__ draft_start,
                     const float* __restrict__ noise, const float* __restrict__ draft_probs, const Record* __restrict__ records,
                     const int* __restrict__ slots, const Row* __restrict__ rows, int total, int* __restrict__ accepted,
                     int* __restrict__ next_token) {
  __shared__ Joined s;
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
    const float* x_row = logits + (size_t)r * vocab;
    const float* q_row = rejected && draft_probs != nullptr ? draft_probs + (size_t)(first + passed) * vocab : nullptr;
    const float* e_row = noise + (size_t)request * vocab;
    const int token = rejected ? drafts[first + passed] : -1;
    const float per = 1.4426950408889634f / rec.temperature;
    // (rows of a vocabulary that is no multiple of four start at other boundaries each: numbers one by one)
    const bool wide = vocab % 4 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(draft_probs) | reinterpret_cast<uintptr_t>(noise)) & 15) == 0;
    const int quads = (vocab + 3) / 4, share = (quads + kRanks - 1) / kRanks, quad_end = min(quads, (rank + 1) * share);
    auto race = [&](bool residual) {
      Best best{-INFINITY, 0x7fffffff};
      constexpr int kDeep = 2;
      for (int g = rank * share + (int)threadIdx.x; g < quad_end; g += kDeep * kThreads) {
        float x[kDeep][4], q[kDeep][4], e[kDeep][4];
#pragma unroll
        for (int j = 0; j < kDeep; ++j) {
          const int quad = g + j * kThreads, i = 4 * quad;
#pragma unroll
          for (int c = 0; c < 4; ++c) x[j][c] = -INFINITY, q[j][c] = 0.f, e[j][c] = 1.f;
          if (quad >= quad_end) continue;
          if (wide) {
            *reinterpret_cast<float4*>(x[j]) = *reinterpret_cast<const float4*>(x_row + i);
            *reinterpret_cast<float4*>(e[j]) = *reinterpret_cast<const float4*>(e_row + i);
            if (residual && q_row != nullptr) *reinterpret_cast<float4*>(q[j]) = *reinterpret_cast<const float4*>(q_row + i);
          } else {
#pragma unroll
            for (int c = 0; c < 4; ++c)
              if (i + c < vocab) {
                x[j][c] = x_row[i + c], e[j][c] = e_row[i + c];
                if (residual && q_row != nullptr) q[j][c] = q_row[i + c];
              }
          }
        }
#pragma unroll
        for (int j = 0; j < kDeep; ++j)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int i = 4 * (g + j * kThreads) + c;
            const float v = clean(x[j][c]);
            const unsigned key = order_key(v);
            if (!(v > -INFINITY) || !(key > row.thr || (key == row.thr && i < row.bound))) continue;
            float left = quick_weight(v, row.top, per) * row.inverse;
            if (residual) left = q_row != nullptr ? left - q[j][c] : i == token ? 0.f : left;
            if (!(left > 0.f)) continue;
            const float value = left / e[j][c];
            if (value > best.value || (value == best.value && i < best.index)) best = Best{value, i};
          }
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
