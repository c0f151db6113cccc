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
// Two kernels: over all rows of logits, then over one row of logits, draft probabilities and variates per request.  A cluster of one to eight
// blocks works on a row; counts, masses and candidates meet in distributed shared memory.  Rows without filters and the second kernel are
// bound by their reads (72 rows of 151,936 and 16 requests: 30 us replayed), rows with filters by their passes over the row and the barriers between them
// (272 rows of 64 requests: about 113 us; the second kernel 25).
//
// The filters' borders.  Of up to 256 entries (top_k): the k-th largest of the threads' own largest entries is not above the k-th largest of all; what is not
// below it is a list of little more than k, whose entries are ranked one by one.  Otherwise masses (for top_k counts too) in 256 bins of an eighth
// of (max - x) / temperature, a column of bins to each lane (equal steps in the exponent and columns of their own keep atomic additions from
// waiting for one another), then in 256 parts of the bin that holds the border, then the list of that part; a bin of few entries is listed at once.
// Masses are sums of integers (units of 2^-44 of the largest weight at 151,936 entries), so that their order changes nothing.  Where a part
// holds more than the list takes (equal logits) or the border lies behind the bins, rounds over the bits of the numbers find it.
// Flat rows, of whose bin at the border a block has more entries than it keeps: the row is read once more for the counts of the bin's parts and once for the
// list (408 rows of 151,936 normally distributed logits, temperature 1, top_p 0.95: deviation 1 1,134 us, 2 331, peaked ones 278; by
// the bits of the numbers 6,200 for deviation 1).
#include "common.cuh"

#include <cooperative_groups.h>

namespace ms {
namespace verify {

namespace cg = cooperative_groups;

constexpr int kMostRanks = 8, kThreads = 512, kWarps = kThreads / 32;
constexpr int kBins = 256, kBinsToOne = 8;           // bins of (max - x) / temperature
constexpr int kExactBins = 4 * kBinsToOne;          // those whose masses are sums of every entry's own
constexpr int kFine = 256;                           // parts of a bin
constexpr int kListed = 512, kShort = 128;          // entries that are ranked one by one; those of a whole bin (their comparisons grow with the square)
constexpr int kNear = 4096;                          // a block's entries of the bin that holds the border, as far as they are kept
constexpr int kFewKept = 256;                        // top_k up to which the threads' largest entries give the list
constexpr int kDigit = 256;                          // of a round over the bits of the numbers

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
  __device__ Part(const float* r, int v, int rank, int ranks) : row(r), vocab(v) {
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(r) & 15)) & 15) / 4;
    const int per = ((v + ranks - 1) / ranks + 3) / 4 * 4;
    begin = rank == 0 ? 0 : min(v, rank * per + lead);
    end = rank == ranks - 1 ? v : min(v, (rank + 1) * per + lead);
  }
  // f(x, first): sixteen entries; number 4 j + e has the index first + 4 kThreads j + e, and is -inf where there is none.
  template <typename F> __device__ __forceinline__ void sixteen(F f) const {
    const int lead = (int)((16 - (reinterpret_cast<uintptr_t>(row + begin) & 15)) & 15) / 4;
    const int first = min(end, begin + lead), quads = (end - first) / 4, ends = end - begin - 4 * quads;
    const float4* wide = reinterpret_cast<const float4*>(row + first);
    const int rounds = (quads + 4 * kThreads - 1) / (4 * kThreads);
#pragma unroll 1
    for (int round = 0; round < rounds + (ends > 0 ? 1 : 0); ++round) {
      float x[16];
      int at = first + 4 * (round * 4 * kThreads + (int)threadIdx.x);
      if (round < rounds) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int g = (round * 4 + j) * kThreads + (int)threadIdx.x;
          float4 v = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
          if (g < quads) v = wide[g];
          x[4 * j] = v.x, x[4 * j + 1] = v.y, x[4 * j + 2] = v.z, x[4 * j + 3] = v.w;
        }
      } else {                                       // the ragged ends: up to three entries before the first boundary and behind the last
        const int t = (int)threadIdx.x;
        at = t < first - begin ? begin + t : first + 4 * quads + t - (first - begin);
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = -INFINITY;
        if (t < ends) x[0] = row[at];
      }
#pragma unroll
      for (int j = 0; j < 16; ++j) x[j] = clean(x[j]);
      f(x, at);
    }
  }
  // f(index, x) of every entry that is not masked, with small code: for the rare passes.
  template <typename F> __device__ __forceinline__ void each(F f) const {
#pragma unroll 1
    for (int i = begin + (int)threadIdx.x; i < end; i += kThreads) {
      const float x = clean(row[i]);
      if (x > -INFINITY) f(i, x);
    }
  }
};

// x[j], where indexing would put the sixteen into local memory (reading the entry again took 500 cycles).
__device__ __forceinline__ float pick(const float (&x)[16], int j) {
  float v = x[0];
#pragma unroll
  for (int c = 1; c < 16; ++c) v = j == c ? x[c] : v;
  return v;
}

struct Entry {
  float x;
  int index;
  unsigned long long mass;
};

struct Near {
  float x;
  int index;
};

struct Joined {
  Best bests[2][kMostRanks];
  Best warp_best[kWarps];
};

struct Shared : Joined {
  union {
    unsigned cells[kBins][32];                                 // this block's counts, then masses, a column to each lane
    Near near[kNear];                                          // afterwards: this block's entries of the bin that holds the border
  };
  unsigned limbs[3][kExactBins][32];                           // sixteen bits of each weight
  unsigned long long bin_count[kBins], bin_mass[kBins];        // this block's, then on rank 0 all ranks'
  unsigned fine_count[kFine], fine_low[kFine], fine_high[kFine];
  unsigned long long fine_mass[kFine], fine_counts[kFine];
  unsigned long long digit[kDigit];
  Entry list[kListed];
  int listed;
  unsigned long long scan[kWarps];
  double sums[kMostRanks];
  int counts[kMostRanks];
  double warp_double[kWarps];
  int warp_int[kWarps];
  unsigned long long warp_mass[kWarps];
  int found, bound, command, bin, part, held;
  unsigned thr, border, lower[kMostRanks];
  unsigned long long above;
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
  if (threadIdx.x < cluster.num_blocks()) {
    Best b = s.warp_best[0];
    for (int w = 1; w < kWarps; ++w) b = better(b, s.warp_best[w]);
    cluster.map_shared_rank(&s, threadIdx.x)->bests[turn][rank] = b;
  }
  cluster.sync();
  Best b = s.bests[turn][0];
  for (int r = 1; r < (int)cluster.num_blocks(); ++r) b = better(b, s.bests[turn][r]);
  return b;
}

__device__ double cluster_sum(Shared& s, cg::cluster_group& cluster, int rank, double v) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lane == 0) s.warp_double[warp] = v;
  __syncthreads();
  if (threadIdx.x < cluster.num_blocks()) {
    double b = 0.0;
    for (int w = 0; w < kWarps; ++w) b += s.warp_double[w];
    cluster.map_shared_rank(&s, threadIdx.x)->sums[rank] = b;
  }
  cluster.sync();
  double b = 0.0;
  for (int r = 0; r < (int)cluster.num_blocks(); ++r) b += s.sums[r];
  return b;
}

// Over `bins` (up to one for each thread) from the first on: the first at which the running sum exceeds `limit` (n where none does); `above`: the sum
// before it.
__device__ __noinline__ int first_over(Shared& s, const unsigned long long* bins, int n, unsigned long long limit, unsigned long long& above) {
  const unsigned long long mine = (int)threadIdx.x < n ? bins[threadIdx.x] : 0;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  unsigned long long before = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += other;
  }
  __syncthreads();
  if (lane == 31) s.scan[warp] = before;
  if (threadIdx.x == 0) s.found = n;
  __syncthreads();
  before -= mine;
#pragma unroll 1
  for (int w = 0; w < warp; ++w) before += s.scan[w];
  if (before <= limit && before + mine > limit) s.found = (int)threadIdx.x, s.above = before;          // one thread at most
  if (threadIdx.x == kThreads - 1 && before + mine <= limit) s.above = before + mine;
  __syncthreads();
  above = s.above;
  return s.found;
}

// The sum over this block of one number a thread.
__device__ unsigned long long block_mass(Shared& s, unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.warp_mass[threadIdx.x >> 5] = v;
  __syncthreads();
  unsigned long long sum = 0;
  for (int w = 0; w < kWarps; ++w) sum += s.warp_mass[w];
  return sum;
}

// Numbers of all ranks added up in rank 0's, which calls this.
__device__ __noinline__ void gather(cg::cluster_group& cluster, unsigned long long* numbers, int n) {
  if ((int)threadIdx.x < n) {
    unsigned long long sum = numbers[threadIdx.x];
    const int ranks = (int)cluster.num_blocks();
#pragma unroll
    for (int r = 1; r < kMostRanks; ++r)
      if (r < ranks) sum += *cluster.map_shared_rank(numbers + threadIdx.x, r);
    numbers[threadIdx.x] = sum;
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
  if (threadIdx.x < cluster.num_blocks()) {
    int all = 0;
    for (int w = 0; w < kWarps; ++w) all += s.warp_int[w];
    cluster.map_shared_rank(&s, threadIdx.x)->counts[rank] = all;
  }
  cluster.sync();
  const int ranks = (int)cluster.num_blocks();
  int before = 0, owner = ranks - 1;
  for (int r = 0; r < ranks; ++r) {
    if (before + s.counts[r] > need) {
      owner = r;
      break;
    }
    if (r + 1 < ranks) before += s.counts[r];
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
    if ((int)threadIdx.x < ranks) cluster.map_shared_rank(&s, threadIdx.x)->bound = s.found;
  }
  cluster.sync();
  return s.bound;
}

// A request's record; argmax where there are none, or none in its slot.
__device__ __forceinline__ Record record_of(const Record* records, int n_records, const int* slots, int request) {
  Record rec{0.f, 1.f, 0};
  if (records != nullptr && (unsigned)slots[request] < (unsigned)n_records) rec = records[slots[request]];
  rec.top_p = fmaxf(rec.top_p, 0.f);
  return rec;
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
  __device__ Weights(float t, float heat, int shift) : top(t), temperature(heat), to_bin((float)kBinsToOne / heat), unit((double)(1ull << shift)) {}
  __device__ __noinline__ unsigned long long of(float x) const {
    const float e = exponent(x, top, temperature);
    if (e > -7.f) return (unsigned long long)__double2ll_rn(exp(x == top ? 0.0 : ((double)x - (double)top) / (double)temperature) * unit);
    return (unsigned long long)__float2ll_rn(expf(e) * (float)unit);
  }
  // (max - x) / temperature in bins; bin b is what rounds to b, and its entries are larger than those of the bins behind it.  (The rounding is an addition:
  // a conversion takes the pipe that the exponentials need.  Products and additions are rounded one by one wherever this is used: an entry that one
  // use puts into another bin or part than the next would be counted in one and looked for in the other.)
  __device__ __forceinline__ float place(float x) const { return __fmul_rn(top - x, to_bin); }
  static __device__ __forceinline__ int bin(float place) { return __float_as_int(__fadd_rn(place, 12582912.f)) - __float_as_int(12582912.f); }
  static __device__ __forceinline__ float middle(float place) { return __fadd_rn(place, 12582912.f) - 12582912.f; }
  // Numbers not above, and not below, every x whose place is `t` (which is off by 2^-21 of itself): to look closely at few entries.
  __device__ __forceinline__ float under(float t) const { return edge(t) - 1e-5f * (fabsf(edge(t)) + fabsf(top)) - 1e-30f; }
  __device__ __forceinline__ float over(float t) const { return edge(t) + 1e-5f * (fabsf(edge(t)) + fabsf(top)) + 1e-30f; }
  __device__ __forceinline__ float edge(float t) const { return top - t * (temperature / (float)kBinsToOne); }
  // the part of its bin, 0 .. kFine - 1
  static __device__ __forceinline__ int fine(float place) { return min(kFine - 1, max(0, (int)(__fadd_rn(place - middle(place), 0.5f) * (float)kFine))); }
  // w / W of an entry `u` bins behind the upper edge of its bin
  static __device__ __forceinline__ float share(float u) {
    float w;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(w) : "f"(u * (-1.4426950408889634f / kBinsToOne)));
    return w;
  }
  // W of bin b, times `unit`
  __device__ __forceinline__ double edge_weight(int b) const { return exp(((double)-b + 0.5) / kBinsToOne) * unit; }
};

// An entry's place among the `listed` and the mass of those before it; of those that stay (the first `most` of them, those with above + the mass before
// them <= limit) the last one is the border, s.thr and s.bound.  Returns their mass.  `lanes` neighbouring threads share an entry's comparisons.
__device__ __noinline__ unsigned long long rank_list(Shared& s, int listed, int most, unsigned long long above, unsigned long long limit) {
  int lanes = 32;
  while (lanes > 1 && listed * lanes > kThreads) lanes /= 2;
  const int sub = (int)threadIdx.x % lanes, step = kThreads / lanes;
  int last = -1, border = -1;
  unsigned long long kept = 0;
#pragma unroll 1
  for (int base = 0; base < listed; base += step) {          // (once, or twice beyond kThreads entries)
    const int a = base + (int)threadIdx.x / lanes;
    unsigned long long sum = 0;
    int ahead = 0;
    const Entry mine = s.list[min(a, listed - 1)];
    if (a < listed) {
#pragma unroll 2
      for (int c = sub; c < listed; c += lanes) {
        const Entry other = s.list[c];
        const bool larger = other.x > mine.x || (other.x == mine.x && other.index < mine.index);
        ahead += larger ? 1 : 0;
        sum += larger ? other.mass : 0;
      }
    }
#pragma unroll 1
    for (int o = lanes / 2; o > 0; o >>= 1) {
      ahead += __shfl_xor_sync(0xffffffffu, ahead, o);
      sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (a < listed && sub == 0 && ahead < most && above + sum <= limit) {
      kept += mine.mass;
      if (ahead > last) last = ahead, border = a;
    }
  }
  const int best = __reduce_max_sync(0xffffffffu, last);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s.warp_int[threadIdx.x >> 5] = best;
  kept = block_mass(s, kept);
  int over_all = -1;
#pragma unroll 1
  for (int w = 0; w < kWarps; ++w) over_all = max(over_all, s.warp_int[w]);
  if (last >= 0 && last == over_all) s.thr = order_key(s.list[border].x), s.bound = s.list[border].index + 1;
  __syncthreads();
  return kept;
}

// The kept set of a row with a top_k of up to kFewKept from a list of little more than top_k entries; false on every rank where the list is too long.
// `largest`: this thread's.  On rank 0 row.thr, row.bound and `total`, the kept mass, are set.
__device__ __noinline__ bool filter_by_largest(Shared& s, cg::cluster_group& cluster, int rank, const Part& part, const Weights& weights, const Record& rec,
                                               bool top_p, float largest, Row& row, unsigned long long& total) {
  // the top_k-th largest of this block's threads', to sixteen bits, downwards
  const unsigned mine = order_key(largest);
  unsigned lower = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 16; --bit) {
    const unsigned candidate = lower | (1u << bit);
    if (__syncthreads_count(mine >= candidate) >= rec.top_k) lower = candidate;
  }
  if (threadIdx.x == 0) s.listed = 0;
  if (threadIdx.x < cluster.num_blocks()) cluster.map_shared_rank(&s, threadIdx.x)->lower[rank] = lower;
  cluster.sync();
  for (int r = 0; r < (int)cluster.num_blocks(); ++r) lower = max(lower, s.lower[r]);
  const float from = number_of(lower) == number_of(lower) && lower > 0x007fffffu ? number_of(lower) : -INFINITY;          // (keys below that of -inf are no number's)
  Shared* first = cluster.map_shared_rank(&s, 0);
  part.sixteen([&](const float (&x)[16], int at) {
    unsigned inside = 0;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (x[j] >= from && x[j] > -INFINITY) inside |= 1u << j;
#pragma unroll 1
    for (; inside != 0; inside &= inside - 1) {
      const int j = __ffs((int)inside) - 1, i = at + (j / 4) * 4 * kThreads + j % 4;
      const float v = pick(x, j);
      const int slot = atomicAdd(&first->listed, 1);
      if (slot < kListed) first->list[slot] = Entry{v, i, weights.of(v)};
    }
  });
  cluster.sync();
  if (rank == 0) {
    const int listed = s.listed;
    const bool fits = listed <= kListed && listed > 0;
    if (fits) {
      total = rank_list(s, listed, rec.top_k, 0, ~0ull);
      if (top_p) total = rank_list(s, listed, rec.top_k, 0, (unsigned long long)floor((double)rec.top_p * (double)total));
      row.thr = s.thr, row.bound = s.bound;
    }
    if (threadIdx.x < cluster.num_blocks()) cluster.map_shared_rank(&s, threadIdx.x)->command = fits ? 0 : -1;
  }
  cluster.sync();
  return s.command == 0;
}

// The kept set of a row with filters by bins, their parts and a list; false on every rank where a list is too long or the border lies behind the bins.  On
// rank 0 row.thr, row.bound and `total`, the kept mass, are set.
//
// A bin's mass: of the first eight bins (the weights from e^-4 up) the sum of its entries' own; of the others W sum w / W, W the weight at the bin's upper
// edge, w / W in steps of 2^-19 where 151,936 entries are one block's (finer for fewer): those weights are e^-4 and less of the largest each, and
// their roundings cancel, so that a border moves by less than 2^-23 of the mass.  Additions are of 32 bits: one of 64 bits in shared memory took the
// multiprocessor 1.3 cycles for every entry.
enum : int { kDone = 0, kGiveUp = -1, kFill = 1, kList = 2 };

__device__ __noinline__ bool filter_by_bins(Shared& s, cg::cluster_group& cluster, int rank, const Part& part, const Weights& weights, const Record& rec,
                                            bool top_k, bool top_p, Row& row, unsigned long long& total) {
  const int lane = threadIdx.x & 31, ranks = (int)cluster.num_blocks();
  for (int i = threadIdx.x; i < 3 * kExactBins * 32; i += kThreads) (&s.limbs[0][0][0])[i] = 0;
  int bits = 32;                                     // of w / W: so many that a lane's entries cannot overflow 32 bits
  for (int most = (part.vocab / ranks) / 32 + 80; most > 0; most >>= 1) --bits;
  bits = min(bits, 22);
  const float steps = (float)(1 << bits);
#pragma unroll 1
  for (int masses = top_k ? 0 : 1; masses < (top_p ? 2 : 1); ++masses) {          // (without top_p only the kept sum is needed, at the end)
    __syncthreads();
    for (int i = threadIdx.x; i < kBins * 32; i += kThreads) (&s.cells[0][0])[i] = 0;
    __syncthreads();
    part.sixteen([&](const float (&x)[16], int) {
      unsigned large = 0;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float t = weights.place(x[j]);
        if (!(t < (float)kBins - 1.f)) continue;          // (masked, or less than e^-31 of the largest: no mass)
        const int bin = Weights::bin(t);
        if (bin < kExactBins) large |= 1u << j;
        const unsigned share = __float_as_uint(fmaf(Weights::share(t - Weights::middle(t) + 0.5f), steps, 8388608.f)) & 0x7fffffu;
        atomicAdd(&s.cells[bin][lane], masses ? share : 1u);
      }
      if (!masses) large = 0;
#pragma unroll 1
      for (; large != 0; large &= large - 1) {
        const float v = pick(x, __ffs((int)large) - 1);
        const unsigned long long w = weights.of(v);
        const int bin = Weights::bin(weights.place(v));
        atomicAdd(&s.limbs[0][bin][lane], (unsigned)w & 0xffffu);
        atomicAdd(&s.limbs[1][bin][lane], (unsigned)(w >> 16) & 0xffffu);
        atomicAdd(&s.limbs[2][bin][lane], (unsigned)(w >> 32));
      }
    });
    __syncthreads();
    // this block's columns: two threads to a bin
    const int bin = (int)threadIdx.x / 2;
    const bool exact = masses && bin < kExactBins;
    unsigned long long w = 0;
#pragma unroll 4
    for (int c = 0; c < 16; ++c) {
      const int column = (c * 2 + (int)threadIdx.x + bin) & 31;          // (even ones to one thread, odd ones to the other; neighbours at other banks)
      w += exact ? s.limbs[0][bin][column] + ((unsigned long long)s.limbs[1][bin][column] << 16) + ((unsigned long long)s.limbs[2][bin][column] << 32)
                 : s.cells[bin][column];
    }
    w += __shfl_xor_sync(0xffffffffu, w, 1);
    if (threadIdx.x % 2 == 0) (masses ? s.bin_mass : s.bin_count)[bin] = w;
  }
  static_assert(kThreads == 2 * kBins && kThreads >= kFine && kThreads >= kDigit, "a thread to a bin");
  cluster.sync();

  // rank 0 alone searches and says what all ranks are to do next
  bool by_count = top_k;
  int bin = 0, fine = -1, need = 0;                          // fine: the part of the bin that is listed, -1: all of it
  unsigned long long limit = ~0ull, above = 0, before = 0;       // masses
  auto tell = [&](int command) {
    if ((int)threadIdx.x < ranks) {
      Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
      other->command = command, other->bin = bin, other->part = fine;
    }
  };
  auto mass_before = [&](const unsigned long long* masses, int n) { return block_mass(s, (int)threadIdx.x < n ? masses[threadIdx.x] : 0); };
  auto entries_of = [&](int b) {     // at most: the mass over the weight at the lower edge
    return top_k ? (double)s.bin_count[b] : (double)s.bin_mass[b] / weights.edge_weight(b + 1);
  };
  auto look_into = [&]() {           // (the bin as a whole where it is short)
    fine = -1;
    if (threadIdx.x == 0) s.listed = 0;
    if (bin >= kBins) tell(kGiveUp);
    else tell(entries_of(bin) <= (double)kShort ? kList : kFill);
  };
  if (rank == 0) {
    if (top_k) gather(cluster, s.bin_count, kBins);
    if (top_p) gather(cluster, s.bin_mass, kBins);
    if ((int)threadIdx.x >= kExactBins && (int)threadIdx.x < kBins)
      s.bin_mass[threadIdx.x] = (unsigned long long)__double2ll_rn(weights.edge_weight((int)threadIdx.x) / (double)steps * (double)s.bin_mass[threadIdx.x]);
    __syncthreads();
    if (by_count) {
      bin = first_over(s, s.bin_count, kBins, (unsigned long long)rec.top_k - 1, before);
      need = rec.top_k - (int)before;
      if (top_p) above = mass_before(s.bin_mass, bin);
    } else {
      total = mass_before(s.bin_mass, kBins);
      limit = (unsigned long long)floor((double)rec.top_p * (double)total);
      bin = first_over(s, s.bin_mass, kBins, limit, above);
    }
    look_into();
  }
  int command;
#pragma unroll 1
  for (;;) {
    cluster.sync();
    command = s.command;
    if (command <= 0) break;
    const int of_bin = s.bin, of_part = s.part;
    Shared* first = cluster.map_shared_rank(&s, 0);
    auto list = [&](float v, int i) {
      const int slot = atomicAdd(&first->listed, 1);
      if (slot < kListed) first->list[slot] = Entry{v, i, weights.of(v)};
    };
    auto take = [&](float v, int i) {
      const float t = weights.place(v);
      if (Weights::bin(t) != of_bin) return;
      const int f = Weights::fine(t);
      if (command == kList) {
        if (of_part < 0 || f == of_part) list(v, i);
        return;
      }
      // w / W in steps of 2^-26 as two halves of thirteen bits: no part of 2^19 entries overflows 32 bits
      const unsigned q = (unsigned)(Weights::share(t - Weights::middle(t) + 0.5f) * 67108863.f);
      atomicAdd(&s.fine_count[f], 1u);
      atomicAdd(&s.fine_low[f], q & 8191u);
      atomicAdd(&s.fine_high[f], q >> 13);
    };
    if (command == kFill || of_part < 0) {               // (else a part of the bin whose entries this block holds)
      if (threadIdx.x == 0) s.held = 0;
      if (command == kFill)
        for (int i = threadIdx.x; i < kFine; i += kThreads) s.fine_count[i] = 0, s.fine_low[i] = 0, s.fine_high[i] = 0;
      __syncthreads();
      const float least = weights.under((float)of_bin + 0.5f), most = weights.over((float)of_bin - 0.5f);
      part.sixteen([&](const float (&x)[16], int at) {
        unsigned inside = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (x[j] >= least && x[j] <= most) inside |= 1u << j;          // (and a few beside the bin's edges)
        // room for all of the warp's at once
        const int mine = __popc(inside);
        int before_me = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int other = __shfl_up_sync(0xffffffffu, before_me, o);
          if (lane >= o) before_me += other;
        }
        const int all = __shfl_sync(0xffffffffu, before_me, 31);
        if (all == 0) return;
        int base = 0;
        if (lane == 0) base = atomicAdd(&s.held, all);
        int slot = __shfl_sync(0xffffffffu, base, 0) + before_me - mine;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (inside >> j & 1) {
            if (slot < kNear) s.near[slot] = Near{x[j], at + (j / 4) * 4 * kThreads + j % 4};
            ++slot;
          }
      });
      __syncthreads();
    }
    if (s.held <= kNear) {
      for (int a = threadIdx.x; a < s.held; a += kThreads) take(s.near[a].x, s.near[a].index);
    } else {
      // more than there is room for (flat rows, of which a block has more than about 100,000 entries): from the row
      part.sixteen([&](const float (&x)[16], int at) {
        unsigned inside = 0;
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (Weights::bin(weights.place(x[j])) == of_bin) inside |= 1u << j;
#pragma unroll 1
        for (; inside != 0; inside &= inside - 1) {
          const int j = __ffs((int)inside) - 1;
          take(pick(x, j), at + (j / 4) * 4 * kThreads + j % 4);
        }
      });
    }
    if (command == kFill) {
      __syncthreads();
      for (int i = threadIdx.x; i < kFine; i += kThreads) s.fine_counts[i] = s.fine_count[i], s.fine_mass[i] = s.fine_low[i] + ((unsigned long long)s.fine_high[i] << 13);
    }
    cluster.sync();
    if (rank != 0) continue;
    if (command == kFill) {
      gather(cluster, s.fine_counts, kFine);
      gather(cluster, s.fine_mass, kFine);
      for (int i = threadIdx.x; i < kFine; i += kThreads)
        s.fine_mass[i] = (unsigned long long)__double2ll_rn(weights.edge_weight(bin) / 67108863.0 * (double)s.fine_mass[i]);
      __syncthreads();
      if (by_count) {
        fine = first_over(s, s.fine_counts, kFine, (unsigned long long)need - 1, before);
        need -= (int)before;
        above += mass_before(s.fine_mass, fine);
      } else {
        fine = first_over(s, s.fine_mass, kFine, limit - above, before);
        above += before;
      }
      tell(fine < kFine && s.fine_counts[fine] <= kListed ? kList : kGiveUp);
      continue;
    }
    const int listed = s.listed;
    if (listed > kListed || listed == 0) {
      tell(kGiveUp);
      continue;
    }
    const unsigned long long stay = rank_list(s, listed, by_count ? need : listed, above, by_count ? ~0ull : limit);
    total = above + stay;
    if (by_count && top_p) {
      by_count = false;
      limit = (unsigned long long)floor((double)rec.top_p * (double)total);
      if (limit >= above) {                              // the nucleus ends in this list
        total = above + rank_list(s, listed, need, above, limit);
      } else {
        const int old_bin = bin, old_fine = fine;
        bin = first_over(s, s.bin_mass, kBins, limit, above);
        if (bin == old_bin && old_fine >= 0) {           // in an earlier part of the same bin
          fine = first_over(s, s.fine_mass, kFine, limit - above, before);
          above += before;
          if (threadIdx.x == 0) s.listed = 0;
          tell(fine < kFine && s.fine_counts[fine] <= kListed ? kList : kGiveUp);
        } else {
          look_into();
        }
        continue;
      }
    }
    row.thr = s.thr, row.bound = s.bound;
    tell(kDone);
  }
  if (command == kDone && !top_p) {
    // the kept sum: large weights as they are, the others as float32 sums of a thread's
    if (rank == 0 && (int)threadIdx.x < ranks) {
      Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
      other->border = row.thr, other->bound = row.bound;
    }
    cluster.sync();
    const unsigned thr = s.border;
    const int bound = s.bound;
    const float per = 1.4426950408889634f / weights.temperature;
    unsigned long long large_sum = 0;
    float small_sum = 0.f;
    part.sixteen([&](const float (&x)[16], int at) {
      unsigned large = 0;
      float sum = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const unsigned key = order_key(x[j]);
        if (!(key > thr || (key == thr && at + (j / 4) * 4 * kThreads + j % 4 < bound))) continue;
        if (weights.place(x[j]) < (float)kExactBins) large |= 1u << j;
        else sum += quick_weight(x[j], weights.top, per);
      }
      small_sum += sum;
#pragma unroll 1
      for (; large != 0; large &= large - 1) large_sum += weights.of(pick(x, __ffs((int)large) - 1));
    });
    total = (unsigned long long)cluster_sum(s, cluster, rank, (double)large_sum + (double)small_sum * weights.unit);
  }
  return command == kDone;
}

// The same by four rounds over the bits of the numbers, the largest first, which takes any row.
__device__ __noinline__ void filter_by_bits(Shared& s, cg::cluster_group& cluster, int rank, const Part& part, const Weights& weights, const Record& rec,
                                            bool top_k, bool top_p, Row& row, unsigned long long& total) {
  row.thr = 0, row.bound = part.vocab;
  const int ranks = (int)cluster.num_blocks();
  // fills this round's digits with what `amount` gives for the entries under the prefix, the largest digit first
  auto fill = [&](int low, unsigned prefix, auto amount) {
    cluster.sync();                                  // (rank 0 may still read)
    for (int i = threadIdx.x; i < kDigit; i += kThreads) s.digit[i] = 0;
    __syncthreads();
    part.each([&](int i, float x) {
      const unsigned key = order_key(x);
      if (low != 24 && (key >> (low + 8)) != prefix) return;
      const unsigned long long a = amount(key, i, x);
      if (a != 0) atomicAdd(&s.digit[255 - ((key >> low) & 255u)], a);
    });
    cluster.sync();
    if (rank == 0) gather(cluster, s.digit, kDigit);
  };
  auto tell = [&](int digit, int bound) {
    if ((int)threadIdx.x < ranks) {
      Shared* other = cluster.map_shared_rank(&s, threadIdx.x);
      other->bin = digit, other->bound = bound;
    }
  };
  unsigned prefix = 0;
  int most = 0;
  bool all = false;
  if (top_k) {
    unsigned long long rest = (unsigned long long)rec.top_k - 1, before;
#pragma unroll 1
    for (int low = 24; low >= 0 && !all; low -= 8) {
      fill(low, prefix, [](unsigned, int, float) { return 1ull; });
      if (rank == 0) {
        const int digit = first_over(s, s.digit, kDigit, rest, before);
        rest -= before;
        tell(digit, (int)rest + 1);
      }
      cluster.sync();
      all = s.bin == kDigit;                         // fewer entries than top_k: all stay
      prefix = (prefix << 8) | (unsigned)(255 - s.bin);
      most = s.bound;
    }
    if (!all) {
      const unsigned thr = prefix;
      row.thr = thr;
      row.bound = index_bound(s, cluster, rank, part, most, [&](int, float x) { return order_key(x) == thr; });
    }
  }
  const unsigned thr_k = row.thr;
  const int bound_k = row.bound;
  auto kept = [&](unsigned key, int i) { return key > thr_k || (key == thr_k && i < bound_k); };
  unsigned long long limit = ~0ull - 1, above = 0, before = 0;           // (rank 0's)
  prefix = 0;
#pragma unroll 1
  for (int low = 24; low >= 0; low -= 8) {
    fill(low, prefix, [&](unsigned key, int i, float x) { return kept(key, i) ? weights.of(x) : 0ull; });
    if (rank == 0) {
      if (low == 24) {
        first_over(s, s.digit, kDigit, ~0ull - 1, total);
        limit = (unsigned long long)floor((double)rec.top_p * (double)total);
      }
      const int digit = min(first_over(s, s.digit, kDigit, limit - above, before), kDigit - 1);
      above += before;
      if (low == 0) {
        // of the equal entries at the border those stay whose mass before is at most the limit
        const unsigned long long each = weights.of(number_of((prefix << 8) | (unsigned)(255 - digit)));
        const unsigned long long room = each > 0 ? (limit - above) / each + 1 : 1, there = each > 0 ? s.digit[digit] / each : 0;
        if (top_p) total = above + (room < there ? room : there) * each;
        most = room < (unsigned long long)part.vocab ? (int)room : part.vocab;
      }
      tell(digit, most);
    }
    cluster.sync();
    prefix = (prefix << 8) | (unsigned)(255 - s.bin);
    most = s.bound;
    if (!top_p) return;                              // (the kept mass is known)
  }
  if (prefix >= thr_k) {
    const unsigned thr = prefix;
    const int outer = thr == thr_k ? bound_k : part.vocab;
    row.thr = thr;
    row.bound = min(outer, index_bound(s, cluster, rank, part, most, [&](int i, float x) { return order_key(x) == thr && i < outer; }));
  }
}

// Row number `place` of all in the order of what their filters cost, the dearest first: those that bins take, those that a list takes, those without
// filters; inside of each in the order of the requests, which are as many as a block has threads, at most.
__device__ __noinline__ void row_by_work(Shared& s, const int* draft_start, int requests, int total, int vocab, const Record* records, int n_records, const int* slots,
                                         int place, int& request, int& r) {
  const int t = (int)threadIdx.x, lane = t & 31, warp = t >> 5;
  constexpr int kField = 21;                       // bits of a count of rows
  int cost = 0, rows = 0;
  if (t < requests) {
    const Record rec = record_of(records, n_records, slots, t);
    const bool top_k = rec.top_k > 0 && rec.top_k < vocab, filters = rec.temperature > 0.f && (top_k || rec.top_p < 1.f);
    cost = !filters ? 2 : top_k && rec.top_k <= kFewKept ? 1 : 0;
    rows = max(0, min(total, draft_start[t + 1] - draft_start[t]) + 1);
  }
  const unsigned long long mine = (unsigned long long)rows << (kField * cost);
  unsigned long long before = mine, all = 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned long long other = __shfl_up_sync(0xffffffffu, before, o);
    if (lane >= o) before += other;
  }
  if (lane == 31) s.scan[warp] = before;
  if (t == 0) s.found = requests - 1, s.bound = 0;
  __syncthreads();
  before -= mine;
#pragma unroll 1
  for (int w = 0; w < kWarps; ++w) {
    if (w == warp) before += all;
    all += s.scan[w];
  }
  auto field = [](unsigned long long v, int c) { return (int)(v >> (kField * c)) & ((1 << kField) - 1); };
  const int start = field(before, cost) + (cost > 0 ? field(all, 0) : 0) + (cost > 1 ? field(all, 1) : 0);
  if (place >= start && place < start + rows) s.found = t, s.bound = place - start;          // one thread
  __syncthreads();
  request = s.found;
  r = max(0, min(draft_start[request] + request + s.bound, total + requests - 1));
}

// Cluster: a row of logits; by_work: the rows that take longest first.
__global__ void __launch_bounds__(kThreads, 2)
verify_rows_kernel(const float* __restrict__ logits, int vocab, const int* __restrict__ drafts, const int* __restrict__ draft_start, int requests,
                   int total, const float* __restrict__ uniforms, const float* __restrict__ draft_probs, const Record* __restrict__ records,
                   int n_records, const int* __restrict__ slots, Row* __restrict__ out, float* __restrict__ target_probs, int shift, int by_work) {
  extern __shared__ __align__(16) unsigned char smem[];
  Shared& s = *reinterpret_cast<Shared*>(smem);
  grid_dependency_wait();
  grid_dependency_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  cluster.barrier_arrive();          // (waited for before the first number goes into another block's shared memory: that block runs by then)
  int r = (int)blockIdx.x / ranks, request;
  if (by_work)
    row_by_work(s, draft_start, requests, total, vocab, records, n_records, slots, r, request, r);
  else
    request = request_of(draft_start, requests, r);
  const int draft = r - request;                               // (the row's place among all drafts, if it has one)
  const bool drafted = draft >= 0 && draft < draft_start[request + 1] && draft < total;
  const Record rec = record_of(records, n_records, slots, request);
  const bool greedy = !(rec.temperature > 0.f);
  const bool top_k = rec.top_k > 0 && rec.top_k < vocab, top_p = rec.top_p < 1.f;
  const Part part(logits + (size_t)r * vocab, vocab, rank, ranks);
  const int token = drafted ? drafts[draft] : 0;
  const bool known = drafted && token >= 0 && token < vocab;
  Row row{};
  row.bound = vocab;
  float p = 0.f;
  Best best{-INFINITY, 0x7fffffff};
  if (greedy) {
    // the largest of sixteen and where they start; then which of them it is
    int start = -1;
    part.sixteen([&](const float (&x)[16], int at) {
      float m = x[0];
#pragma unroll
      for (int j = 1; j < 16; ++j) m = fmaxf(m, x[j]);
      if (m > best.value || (m == best.value && at < start)) best.value = m, start = at;
    });
    if (start >= 0 && best.value > -INFINITY) {
      float again[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int i = start + (j / 4) * 4 * kThreads + j % 4;
        again[j] = i < part.end ? part.row[i] : -INFINITY;
      }
#pragma unroll
      for (int j = 15; j >= 0; --j)
        if (again[j] == best.value) best.index = start + (j / 4) * 4 * kThreads + j % 4;
    }
    cluster.barrier_wait();
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
    cluster.barrier_wait();
    row.top = cluster_best(s, cluster, rank, best, 0).value;
    if (row.top > -INFINITY) {                   // (else every entry is masked: no token has a probability)
      double sum = 0.0;                          // (rank 0's)
      if (one_pass) {
        sum = cluster_sum(s, cluster, rank, mine == -INFINITY ? 0.0 : (double)(partial * quick_weight(mine, row.top, per)));
      } else {
        const Weights weights(row.top, rec.temperature, shift);
        unsigned long long mass = 0;
        const bool finite = row.top < INFINITY;          // (else the bins have no meaning)
        if (!(finite && top_k && rec.top_k <= kFewKept && filter_by_largest(s, cluster, rank, part, weights, rec, top_p, mine, row, mass)) &&
            !(finite && filter_by_bins(s, cluster, rank, part, weights, rec, top_k, top_p, row, mass)))
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
__global__ void __launch_bounds__(kThreads, 2)
verify_choose_kernel(const float* __restrict__ logits, int vocab, const int* __restrict__ drafts, const int* __restrict__ draft_start,
                     const float* __restrict__ noise, const float* __restrict__ draft_probs, const Record* __restrict__ records,
                     int n_records, const int* __restrict__ slots, const Row* __restrict__ rows, int total, int* __restrict__ accepted,
                     int* __restrict__ next_token) {
  __shared__ Joined s;
  grid_dependency_wait();
  grid_dependency_launch();
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks(), request = (int)blockIdx.x / ranks;
  cluster.barrier_arrive();          // (as above)
  const int first = min(max(draft_start[request], 0), total), count = min(max(draft_start[request + 1], first), total) - first;
  int passed = count;
  for (int base = 0; base < count && passed == count; base += 32) {          // (every warp for itself)
    const int i = base + (int)(threadIdx.x & 31);
    const unsigned failed = __ballot_sync(0xffffffffu, i < count && rows[first + request + i].passes == 0);
    if (failed != 0) passed = base + __ffs((int)failed) - 1;
  }
  const int r = first + request + passed;
  const Row row = rows[r];
  const Record rec = record_of(records, n_records, slots, request);
  const bool greedy = !(rec.temperature > 0.f);
  int chosen = row.best;
  cluster.barrier_wait();
  if (!greedy && row.inverse > 0.f) {
    const bool rejected = passed < count;
    const float* x_row = logits + (size_t)r * vocab;
    const float* q_row = rejected && draft_probs != nullptr ? draft_probs + (size_t)(first + passed) * vocab : nullptr;
    const float* e_row = noise + (size_t)request * vocab;
    const int token = rejected ? drafts[first + passed] : -1;
    const float per = 1.4426950408889634f / rec.temperature;
    // (rows of a vocabulary that is no multiple of four start at other boundaries each: numbers one by one)
    const bool wide = vocab % 4 == 0 && ((reinterpret_cast<uintptr_t>(logits) | reinterpret_cast<uintptr_t>(draft_probs) | reinterpret_cast<uintptr_t>(noise)) & 15) == 0;
    const int quads = (vocab + 3) / 4, share = (quads + ranks - 1) / ranks, quad_end = min(quads, (rank + 1) * share);
    const float border = row.thr == 0 ? -INFINITY : number_of(row.thr);
    auto race = [&](bool residual) {
      const int out_of = residual && q_row == nullptr ? token : -1;          // (a draft that was not drawn: its own token has nothing left)
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
            // (indices grow along this thread's way, so that the first of equal ones stays; NaN is no candidate)
            const int i = 4 * (g + j * kThreads) + c;
            const float v = x[j][c];
            const bool kept = v > border || (v == border && i < row.bound);
            const float left = quick_weight(v, row.top, per) * row.inverse - q[j][c], value = __fdividef(left, e[j][c]);
            if (kept && left > 0.f && i != out_of && value > best.value) best = Best{value, i};
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

namespace ms {
namespace verify {

// Blocks to a row: many for few rows, whose latency counts, and fewer for more, so that no more clusters are asked for than find room at once (two blocks a
// multiprocessor, a cluster's within one of the GPU's parts).  Up to 400 rows of a large vocabulary keep two, which even out what the filters of different
// rows take; beyond, one block's rows fill the multiprocessors and there is less to exchange.  us of both kernels with 1, 2, 4 and 8 blocks for every row and
// request, 151,936 logits: 4 rows, greedy 14.8, 11.3, 9.3, 8.3; 72 rows without filters 53, 33, 33, 40; 272 rows with four kinds of filters 195, 140, 177, 369.
// With 1 and 2: 408 rows 226, 203, 510 rows 237, 242, 600 rows 253, 273; of 64,000 logits 272 rows 99, 78, 408 rows 115, 113, 510 rows 122, 135; of 32,768
// logits 272 rows 65, 62, 408 rows 71, 83; 36 rows of 32,011 44, 33.  (Where all rows cost the same, one is 2 to 20 % ahead from 170 rows on: 63, 72 for 272
// without filters.  What they cost only the GPU knows.)
static int ranks_for(int rows, int vocab) {
  if (rows <= 32) return kMostRanks;
  if (rows <= 64) return 4;
  return rows <= 148 || (rows <= 400 && vocab >= 32768) ? 2 : 1;
}

// Whether the rows that take longest go first: where not all blocks run at once (two to a multiprocessor) and rows differ.  Otherwise the last to start may be
// a slow one, and the others' multiprocessors wait for it: 272 rows of 64 requests with four kinds of filters, replayed: 168 us in the rows' order, 141 so; the order itself costs
// 2 to 4 us.
static int by_work_for(int rows, int ranks, int requests, const void* records) {
  return (long long)rows * ranks > 2 * 148 && records != nullptr && requests <= kThreads && rows < (1 << 21) ? 1 : 0;
}

template <typename... Params, typename... Args>
cudaError_t launch_clusters(void (*kernel)(Params...), int rows, int ranks, size_t smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(rows * ranks));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attribute[2];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = ranks, attribute[0].val.clusterDim.y = 1, attribute[0].val.clusterDim.z = 1;
  attribute[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attribute[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attribute;
  config.numAttrs = dependent_launch_enabled() ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

}  // namespace verify
}  // namespace ms

// Bytes of scratch that ms_verify_drafts needs for a row of logits.
MS_EXPORT int ms_verify_row_bytes() { return (int)sizeof(verify::Row); }

// logits [n_drafts + requests, vocab] float32: request r's rows are draft_start[r] + r .. draft_start[r + 1] + r.  drafts, uniforms [n_drafts];
// draft_start [requests + 1]; draft_probs [n_drafts, vocab] or null; noise [requests, vocab]; records [slots, 8] 32-bit words (temperature,
// top_p as float, top_k) or null for argmax, slot_of_request [requests].  accepted, next_token [requests]; target_probs [n_drafts] or null.
MS_EXPORT int ms_verify_drafts(const float* logits, int vocab, const int* drafts, const int* draft_start, int requests, int n_drafts,
                               const float* uniforms, const float* noise, const float* draft_probs, const void* records, int n_records,
                               const int* slot_of_request, int* accepted, int* next_token, float* target_probs, void* scratch,
                               cudaStream_t stream) {
  using namespace ms::verify;
  if (requests == 0) return 0;
  MS_REQUIRE(requests > 0 && n_drafts >= 0 && vocab > 0 && vocab <= (1 << 19), "verify_drafts: %d requests, %d drafts, vocabulary %d", requests, n_drafts, vocab);
  MS_REQUIRE((long long)requests + n_drafts <= 2147483647LL / kMostRanks, "verify_drafts: %d drafts of %d requests in one call are too many", n_drafts, requests);
  MS_REQUIRE(records == nullptr || (slot_of_request != nullptr && noise != nullptr && (uniforms != nullptr || n_drafts == 0)),
             "verify_drafts: sampling records need slots, uniforms and noise");
  MS_REQUIRE(scratch != nullptr && reinterpret_cast<uintptr_t>(scratch) % 8 == 0, "verify_drafts: scratch is missing or not aligned");
  int shift = 62;              // masses are sums of up to `vocab` weights of at most one, in units of 2^-shift
  while (shift > 0 && ((long long)vocab >> (62 - shift)) != 0) --shift;
  const int rows = n_drafts + requests, ranks = ranks_for(rows, vocab);
  cudaError_t e = allow_shared(verify_rows_kernel, sizeof(Shared));
  if (e == cudaSuccess)
    e = launch_clusters(verify_rows_kernel, rows, ranks, sizeof(Shared), stream, logits, vocab, drafts, draft_start, requests, n_drafts, uniforms,
                                  draft_probs, (const Record*)records, n_records, slot_of_request, (Row*)scratch, target_probs, shift, by_work_for(rows, ranks, requests, records));
  if (e == cudaSuccess)
    e = launch_clusters(verify_choose_kernel, requests, ranks_for(requests, vocab), 0, stream, logits, vocab, drafts, draft_start, noise, draft_probs, (const Record*)records, n_records,
                        slot_of_request, (const Row*)scratch, n_drafts, accepted, next_token);
  if (e != cudaSuccess) cudaGetLastError();
  MS_REQUIRE(e == cudaSuccess, "verify_drafts: launch failed: %s", cudaGetErrorString(e));
  return 0;
}
