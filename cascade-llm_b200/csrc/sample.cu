// Sampling of one token per row of logits with temperature, top-k, top-p and
// min-p from a given uniform number.
//
//   e_i = exp((x_i - m) / T), m = max_i x_i;  w_i = floor(2^40 e_i), an integer.
// Order: larger logit first, then smaller index; every filter keeps a prefix
// of it: the first K tokens (mass W_K); those with a mass of less than
// ceil(p W_K) before them; those with e_i >= min_p. With the kept tokens' mass
// W the answer is the first token, in index order, whose cumulated kept mass
// exceeds floor(u W).
//
// Why integers: 32-bit sums of 128,000 weights depend on their order and are off
// by about 1e-6 of the mass, which moves answers between grids and runs. The
// weights' integer sums are exact whatever the order, atomics included; the
// 2^-40 cut leaves out tokens below 1e-12 of the most likely one. p and u are
// taken as 24-bit fixed point, which is exact for a 32-bit uniform number.
//
// Bound: one read of the logits from HBM; after that it is the barriers between
// the steps. A row belongs to a cluster of 1 to 8 CTAs (few rows: more of
// them), which read their slices from HBM once and from L2 afterwards, and
// talk through distributed shared memory:
//   1. m, from each thread's largest logit;
//   2. a bound on the logits that can be kept. With top-k: the K-th largest of
//      the threads' maxima is at most the K-th largest logit, so one
//      histogram entry per thread is enough. With top-p alone: the same for about
//      800 tokens, whose mass is compared with the mass of all in the pass that
//      gathers them. With min-p alone: the bound itself;
//   3. the tokens above the bound, usually a little more than are kept, go to the
//      first CTA as (logit, index) words: cut by every filter and searched in
//      index order there, while the other CTAs leave the SM.
// Where the bounded tokens do not hold the top-p mass, a histogram of rounded masses
// tells an interval of depths with a few hundred tokens, and one more pass sums what
// is above it exactly and gathers it. Where lists of 1024 tokens do not suffice (a
// large K, ties), histograms in exact integers get finer by 512 and then, when ties
// fill that, by 8-bit digits of the logits' ordered bits. Both leave an exact cut
// (a logit, and how many that equal it), and the cluster searches its slices in index
// order, as it does where nothing filters.
//
// Measured with logits from HBM (in L2): one row of 128256 fp32 logits 6.0 us (4.6)
// greedy, 14 (13) with top-k 50, 17 to 40 with top-p 0.9, by the number of tokens that it
// keeps; 256 bf16 rows 15 (11) greedy, 33 (28) with top-k 50, 53 (47) unfiltered, 66 (59)
// with mixed filters, where one read from HBM takes 10. Times beside the choices below
// are with the logits in L2. Registers: 64, the most for two CTAs per SM, with 256 to 316
// bytes of spill stores: one kernel holds every path.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "cascade_b200.h"
#include "internal.h"
#include "paged_device.cuh"

namespace cb {

struct SampleParams {
  const char* logits;
  int64_t row_bytes;
  int vocab, rows;
  bool by_cost;  // rows in the order of their cost
  const float *temperature, *top_p, *min_p, *uniform;
  const int32_t* top_k;
  int64_t* tokens;
  float* logprobs;
};

constexpr int kSampleThreads = 512;
constexpr int kSampleWarps = kSampleThreads / 32;
constexpr int kBins = kSampleThreads;
constexpr int kListMax = 2 * kSampleThreads;  // tokens that the first CTA can hold
constexpr int kFew = kSampleThreads / 4;      // tokens that it compares with one another
// Tokens that top-p alone is tried on. One peaked row 18 us with 700 and 37 with 200,
// which do not hold the boundary; lists end at 1024.
constexpr float kTopPList = 800.0f;
constexpr int kFewTied = 64;         // tokens in the boundary's bin that are compared with one another
constexpr int kPieces = 64;          // of a warp's range, in the search by index
constexpr int kClusterMax = 8;
constexpr int kSliceMax = 260000;    // logits of a CTA: that many limbs of 14 bits (and a vector more) fit 32 bits
constexpr float kReach = 41.0f;      // no weight beyond: 2^-41
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// Top-p alone: mass is summed up to the bound of the tokens that are tried first and
// to this much deeper, and where they do not hold the boundary its band's histogram
// follows.
constexpr int kBands = 2;
constexpr float kBandWidth = 7.0f;

// Element types: value of one, and the largest of a 16-byte vector (NaN never wins).
template <typename T>
struct HalfLogits;
template <>
struct HalfLogits<Bf16> {
  using Raw = uint16_t;
  static constexpr uint16_t kLowest = 0xFF80;
  static __device__ __forceinline__ float value(uint16_t r) { return bf16f(r); }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w);
    const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
template <>
struct HalfLogits<Fp16> {
  using Raw = uint16_t;
  static constexpr uint16_t kLowest = 0xFC00;
  static __device__ __forceinline__ float value(uint16_t r) { return __half2float(__ushort_as_half(r)); }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const __half2* h = reinterpret_cast<const __half2*>(&w);
    const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
    return fmaxf(__low2float(m), __high2float(m));
  }
};
struct F32Logits {
  using Raw = float;
  static constexpr float kLowest = -INFINITY;
  static __device__ __forceinline__ float value(float r) { return r; }
  static __device__ __forceinline__ float largest(const uint4& w) {
    const float* x = reinterpret_cast<const float*>(&w);
    return fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
  }
};

// Unsigned integer with the order of the float (-0 counts as 0).
__device__ __forceinline__ uint32_t ordered(float x) {
  const uint32_t u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float from_ordered(uint32_t k) {
  return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k);
}
// floor(2^40 odds) of odds in [0, 1]: the mantissa shifted by the exponent. (A
// conversion to a 64-bit integer is slow and holds up the exponentials, which
// go through the same unit.)
__device__ __forceinline__ uint64_t weight(float odds) {
  const uint32_t bits = __float_as_uint(odds);
  const uint64_t mantissa = uint64_t((bits & 0x7FFFFFu) | 0x800000u) << 17;
  return mantissa >> min(127u - (bits >> 23), 63u);
}

// A sum of such weights of up to 4095 odds: 8 + e and 2^-17 + rest, rounded down,
// hold bits 39 to 20 and 19 to 0 of 2^40 e as their mantissas' ends. Six instructions of
// 32 bits, where shifting the mantissa and a 64-bit sum take a dozen: 256 unfiltered
// rows 92 -> 72 us.
struct WeightSum {
  uint32_t high = 0, low = 0;
  __device__ __forceinline__ void add(const WeightSum& other) {
    high += other.high;
    low += other.low;
  }
  __device__ __forceinline__ void add(float e) {
    const float a = __fadd_rz(e, 8.0f), b = __fadd_rz(__fsub_rn(e, __fsub_rn(a, 8.0f)), 0x1p-17f);
    high += __float_as_uint(a) - 0x41000000u;
    low += __float_as_uint(b) - 0x37000000u;
  }
  __device__ __forceinline__ uint64_t value() const { return (uint64_t(high) << 20) + low; }
};

// floor(a * b / 2^24) (round = 2^24 - 1: its ceiling) for a <= 2^24, b < 2^60
__device__ __forceinline__ uint64_t part24(uint64_t a, uint64_t b, uint64_t round) {
  return a * (b >> 24) + ((a * (b & 0xFFFFFFu) + round) >> 24);
}

__device__ __forceinline__ uint64_t max64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t shfl_xor64(uint64_t v, int o) { return __shfl_xor_sync(0xFFFFFFFFu, v, o); }
__device__ __forceinline__ uint64_t warp_sum64(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += shfl_xor64(v, o);
  return v;
}
__device__ __forceinline__ uint64_t warp_scan64(uint64_t v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint64_t x = __shfl_up_sync(0xFFFFFFFFu, v, o);
    if (lane >= o) v += x;
  }
  return v;
}
// Inclusive scan over the CTA; `part` may be used again after it.
__device__ __forceinline__ uint64_t block_scan64(uint64_t v, uint64_t* part, uint64_t& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  v = warp_scan64(v);
  if (lane == 31) part[warp] = v;
  __syncthreads();
  uint64_t before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kSampleWarps; ++w) {
    if (w < warp) before += part[w];
    total += part[w];
  }
  __syncthreads();
  return v + before;
}

// One CTA's shared state. `lists` and `found` are the first CTA's; `bins` and
// `below` are read by all; the rest is local, or sent to all.
struct SampleShared {
  unsigned int hist[3][kBins];    // tokens, or their mass in limbs of `limb` bits
  uint64_t bins[kBins];           // the same in one word
  uint64_t staged[2][kListMax];   // this CTA's tokens for the lists
  unsigned int staged_count[2];
  unsigned int staged_at[2];      // their place in the lists
  union {
    uint64_t lists[2][kListMax];  // tokens above the boundary's bin, and in it
    struct {
      uint64_t piece_mass[kSampleWarps][kPieces];
      unsigned int piece_ties[kSampleWarps][kPieces];
    };
  };
  uint4 ends[3];                  // the row's first and last vector, and one of -inf
  uint64_t sums[kBands + 1][kSampleWarps];
  unsigned int found[2];
  uint64_t part[kSampleWarps];
  unsigned int warp_ties[kSampleWarps];
  uint64_t top[kClusterMax];      // every CTA's best (ordered logit, ~vector)
  uint64_t slice_mass[kClusterMax], slice_sums[kBands + 1][kClusterMax];
  unsigned int slice_ties[kClusterMax];
  int bin, past_bin;              // of the current histogram
  uint64_t left;                  // of the target, from this bin on
  float cut_x;
  uint64_t cut_ties;
};

namespace cg = cooperative_groups;

template <typename L>
struct Sampler {
  using Raw = typename L::Raw;
  static constexpr int kVector = 16 / sizeof(Raw);
  static constexpr int kBatch = 4;  // vectors of a thread in flight

  const SampleParams& p;
  SampleShared& s;
  cg::cluster_group cluster;
  int rank, ranks, tid, lane, warp;
  const char* at;     // the row
  int lead;           // vector v holds logits v * kVector - lead on
  int from, to;       // this CTA's vectors
  float top, inverse;
  int limb;           // bits of a limb: a sum over the slice fits 32
  float listed_depth = kReach;  // no token in the lists is deeper

  __device__ Sampler(const SampleParams& p_, SampleShared& s_) : p(p_), s(s_), cluster(cg::this_cluster()) {
    rank = int(cluster.block_rank());
    ranks = int(cluster.num_blocks());
    tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  }

  __device__ __forceinline__ void sync_all() {
    if (ranks == 1)
      __syncthreads();
    else
      cluster.sync();
  }
  template <typename V>
  __device__ __forceinline__ V* of(V* x, int r) {
    return r == rank ? x : cluster.map_shared_rank(x, r);
  }

  // -log2 of a logit's odds: falls as the logit grows; NaN for a NaN.
  __device__ __forceinline__ float depth(float x) const { return (top - x) * inverse; }
  __device__ __forceinline__ float odds(float x) const { return x == top ? 1.0f : ex2(-depth(x)); }

  // Vector v of the row; places outside of it are -inf. The vectors at the row's
  // ends, which are not read whole, and one of -inf lie in shared memory.
  __device__ __forceinline__ uint4 vector(int v) const {
    const int i = v * kVector - lead;
    const char* from_row = at + int64_t(i) * int(sizeof(Raw));
    const void* p0 = v >= to ? &s.ends[2] : i < 0 ? &s.ends[0] : i > p.vocab - kVector ? &s.ends[1] : (const void*)from_row;
    return *reinterpret_cast<const uint4*>(p0);
  }
  __device__ __forceinline__ void keep_ends(int vectors) {
    if (tid < 3 * kVector) {
      const int end = tid / kVector, j = tid - end * kVector;
      const int i = (end == 0 ? 0 : vectors - 1) * kVector - lead + j;
      reinterpret_cast<Raw*>(s.ends)[tid] =
          end < 2 && i >= 0 && i < p.vocab ? reinterpret_cast<const Raw*>(at)[i] : L::kLowest;
    }
    __syncthreads();
  }
  // f(vector, its number) over the slice, in no particular order; Rolled: one
  // copy of f, for what few vectors pass (the kernel's code has to be fetched too)
  template <bool Rolled, typename F>
  __device__ __forceinline__ void each_vector(F f) const {
    for (int v = from + tid; v < to; v += kBatch * kSampleThreads) {
      uint4 w[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) w[b] = vector(v + b * kSampleThreads);
      if (Rolled) {
#pragma unroll 1
        for (int b = 0; b < kBatch; ++b) {
          f(w[0], v + b * kSampleThreads);
#pragma unroll
          for (int i = 1; i < kBatch; ++i) w[i - 1] = w[i];
        }
      } else {
#pragma unroll
        for (int b = 0; b < kBatch; ++b) f(w[b], v + b * kSampleThreads);
      }
    }
  }
  // f(logit, index) over a vector whose first index is i
  template <typename F>
  static __device__ __forceinline__ void each_of(const uint4& w, int i, F f) {
    const Raw* e = reinterpret_cast<const Raw*>(&w);
#pragma unroll
    for (int j = 0; j < kVector; ++j) f(L::value(e[j]), i + j);
  }
  // f(logit, index) over vectors with a token less deep than `deepest`
  template <typename F>
  __device__ __forceinline__ void each(float deepest, F f) const {
    each_vector<true>([&](const uint4& w, int v) {
      if (depth(L::largest(w)) < deepest) each_of(w, v * kVector - lead, f);
    });
  }

  __device__ void answer(int row, uint32_t index, float x, uint64_t kept) const {
    p.tokens[row] = index;
    if (p.logprobs) p.logprobs[row] = (x == top ? 0.0f : -depth(x) * kLn2) - logf(float(kept) * 9.094947017729282e-13f);
  }

  // Bins of [low, low + kBins / scale), and of one of them. The same roundings
  // in every pass (no contraction), so that each puts a token into the same bin.
  struct Bins {
    float low, high, scale;
    __device__ __forceinline__ float place(float d) const { return __fmul_rn(__fsub_rn(d, low), scale); }
    __device__ __forceinline__ bool has(float d) const { return d >= low && d < high; }
    __device__ __forceinline__ int of(float d) const { return min(max(int(place(d)), 0), kBins - 1); }
    __device__ __forceinline__ int within(float d, int bin) const {
      return min(max(int(__fmul_rn(__fsub_rn(place(d), float(bin)), float(kBins))), 0), kBins - 1);
    }
    // one bin's, or (fine >= 0) one part's
    __device__ __forceinline__ Bins part(int bin, int fine) const {
      const float from = low + float(bin) / scale;
      if (fine < 0) return {from, high, scale * float(kBins)};
      return {from + float(fine) / (scale * float(kBins)), high, scale * float(kBins) * float(kBins)};
    }
    // The least depth in the bin, or (fine >= 0) in the part of it: the estimate moved to
    // where the bins of the other passes change, a few steps.
    __device__ __forceinline__ float first(int bin, int fine) const {
      if (bin >= kBins || (bin == kBins - 1 && fine >= kBins)) return high;
      if (bin == 0 && fine <= 0) return low;
      auto there = [&](float d) {
        const int b = of(d);
        return b > bin || (b == bin && (fine < 0 || (fine < kBins && within(d, bin) >= fine)));
      };
      float d = low + (float(bin) + (fine < 0 ? 0.0f : float(fine) * (1.0f / kBins))) / scale;
      while (d > low && there(d)) d = __uint_as_float(__float_as_uint(d) - 1);
      while (d < high && !there(d)) d = __uint_as_float(__float_as_uint(d) + 1);
      return d;
    }
    __device__ __forceinline__ float end(int bin) const { return low + (float(bin + 1) + 0.01f) / scale; }
  };
  __device__ __forceinline__ void add_mass(int bin, float d) { add_to(bin, weight(ex2(-d))); }
  __device__ __forceinline__ void add_to(int bin, uint64_t m) {
    const unsigned mask = (1u << limb) - 1u;
    const unsigned low = unsigned(m) & mask, middle = unsigned(m >> limb) & mask, high = unsigned(m >> (2 * limb));
    atomicAdd(&s.hist[0][bin], low);
    if (middle) atomicAdd(&s.hist[1][bin], middle);
    if (high) atomicAdd(&s.hist[2][bin], high);
  }
  __device__ __forceinline__ uint64_t bin_mass() const {
    return s.hist[0][tid] + (uint64_t(s.hist[1][tid]) << limb) + (uint64_t(s.hist[2][tid]) << (2 * limb));
  }
  // Not while another CTA may still read it: `fresh` is the first use.
  __device__ __forceinline__ void clear_hist(bool fresh) {
    if (!fresh) sync_all();
#pragma unroll
    for (int k = 0; k < 3; ++k) s.hist[k][tid] = 0;
    __syncthreads();
  }
  enum { kTokens, kMass, kCopies };
  // Behind a histogram of every CTA (of tokens, of mass in limbs, or three copies of
  // one whose sums fit 32 bits): each adds up all of them and finds the bin in which the
  // running sum reaches target(sum of all), into s.bin and s.left (what of it is left
  // there); -1 if it never does. Into s.past_bin goes the bin in which it passes target +
  // margin (the last one if none). All of them do the same work, which saves the cluster
  // a barrier.
  template <typename F>
  __device__ __forceinline__ void find_bin(int what, F target, uint64_t margin = 0) {
    __syncthreads();
    const uint64_t counted = s.hist[0][tid];
    s.bins[tid] = what == kMass ? bin_mass() : what == kCopies ? counted + s.hist[1][tid] + s.hist[2][tid] : counted;
    sync_all();
    // loads that do not wait for one another
    uint64_t x[kClusterMax], here = 0;
#pragma unroll
    for (int r = 0; r < kClusterMax; ++r) x[r] = of(&s, r < ranks ? r : rank)->bins[tid];
#pragma unroll
    for (int r = 0; r < kClusterMax; ++r) here += r < ranks ? x[r] : 0;
    uint64_t total;
    const uint64_t upto = block_scan64(here, s.part, total), before = upto - here, left = target(total);
    const bool hit = before < left && left <= upto;
    if (hit || (tid == 0 && total < left)) {
      s.bin = hit ? tid : -1;
      s.left = left - (hit ? before : total);
    }
    if ((before <= left + margin || tid == 0) && (left + margin < upto || tid == kBins - 1)) s.past_bin = tid;
    __syncthreads();
  }

  struct Cut {
    float x;        // logits above it stay, and
    uint64_t ties;  // this many of those equal to it, in index order
  };

  static constexpr int kWhole = -1;  // all parts of a bin
  struct Ends {
    float at[kBands + 1];
  };
  // The tokens less deep than `to_first` go to the first CTA's first list (bit 0 of
  // Lists), those from there to `to_second` to its second (bit 1). Sums: also the mass
  // less deep than each of that many ends, for every CTA in `sums`.
  template <int Lists, int Sums = 0>
  __device__ __forceinline__ void gather(float to_first, float to_second, Ends ends = {}) {
    // The tokens' indexes are staged in this CTA first: its tokens would queue at the
    // first CTA's counters.
    if (tid < 2) s.staged_count[tid] = 0;
    WeightSum part[Sums > 0 ? Sums : 1];
    __syncthreads();
    auto stage = [&](int which, unsigned hits, int v) {  // bit j of hits: token j of the vector
      const volatile unsigned* so_far = &s.staged_count[which];
      if (hits == 0 || *so_far > kListMax) return;
      unsigned place = atomicAdd(&s.staged_count[which], unsigned(__popc(hits)));
      uint32_t* index = reinterpret_cast<uint32_t*>(s.staged[which]);
      for (; hits; hits &= hits - 1, ++place)
        if (place < kListMax) index[place] = v * kVector - lead + __ffs(hits) - 1;
    };
    auto take = [&](const uint4& w, int v) {
      if (!(depth(L::largest(w)) < to_second)) return;
      unsigned hits[2] = {0, 0};
      each_of(w, 0, [&](float x, int j) {
        const float d = depth(x);
        const bool first = d < to_first;
        hits[0] |= unsigned(first) << j;
        hits[1] |= unsigned(!first && d < to_second) << j;
      });
      if (Lists & 1) stage(0, hits[0], v);
      if (Lists & 2) stage(1, hits[1], v);
    };
    if (Sums) {
      each_vector<true>([&](const uint4& w, int v) {
        each_of(w, 0, [&](float x, int) {
          const float d = depth(x);
          WeightSum one;
          one.add(fmaxf(ex2(-d), 0.0f));  // a NaN has no weight
#pragma unroll
          for (int k = 0; k < Sums; ++k)
            if (d < ends.at[k]) part[k].add(one);
        });
        take(w, v);
      });
#pragma unroll
      for (int k = 0; k < Sums; ++k) {
        const uint64_t x = warp_sum64(part[k].value());
        if (lane == 0) s.sums[k][warp] = x;
      }
    } else {
      each_vector<true>(take);
    }
    __syncthreads();
    unsigned int* found = of(&s.found[0], 0);
    if (tid < 2) s.staged_at[tid] = s.staged_count[tid] ? atomicAdd(found + tid, s.staged_count[tid]) : 0;
    if (Sums && warp >= 4 && warp < 4 + Sums) {
      const uint64_t x = warp_sum64(lane < kSampleWarps ? s.sums[warp - 4][lane] : 0);
      if (lane < ranks) of(&s, lane)->slice_sums[warp - 4][rank] = x;
    }
    __syncthreads();
    uint64_t* lists = of(&s.lists[0][0], 0);
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const unsigned count = min(s.staged_count[which], unsigned(kListMax)), place = s.staged_at[which];
      for (unsigned i = tid; i < count && place + i < kListMax; i += kSampleThreads) {
        const uint32_t index = reinterpret_cast<const uint32_t*>(s.staged[which])[i];
        const float x = L::value(reinterpret_cast<const Raw*>(at)[index]);
        lists[which * kListMax + place + i] = (uint64_t(ordered(x)) << 32) | uint32_t(~index);
      }
    }
    sync_all();
    const volatile unsigned int* count = found;
    listed[0] = count[0];
    listed[1] = count[1];
#pragma unroll
    for (int k = 0; k < Sums; ++k) {
      sums[k] = 0;
      for (int r = 0; r < ranks; ++r) sums[k] += s.slice_sums[k][r];
    }
    if (ranks > 1) cluster.barrier_arrive();
  }
  // Behind every gather: everybody has read the counts, so the first CTA may
  // end or empty its lists.
  __device__ __forceinline__ void gathered() {
    if (ranks > 1)
      cluster.barrier_wait();
    else
      __syncthreads();
  }
  unsigned int listed[2];
  uint64_t sums[kBands + 1];  // mass less deep than each of a gather's Ends
  __device__ __forceinline__ bool one_list() const { return listed[0] + listed[1] <= kListMax; }
  __device__ __forceinline__ void forget() {
    gathered();
    if (tid == 0) s.found[0] = s.found[1] = 0;
    sync_all();
  }

  // A histogram of the tokens, or of their mass, over bins; over the parts
  // of one bin (fine == kWhole); or over the next 8 bits, below `prefix`, of the
  // ordered logits in one part. Leaves the bin that holds the target in s.bin,
  // what is left of the target there in s.left.
  template <typename F>
  __device__ __forceinline__ void count(bool by_mass, F target, float deepest, Bins bins, int bin, int fine, int shift,
                                        uint32_t prefix) {
    clear_hist(fresh);
    fresh = false;
    each(deepest, [&](float x, int) {
      const float d = depth(x);
      if (!bins.has(d)) return;
      int b = bins.of(d);
      if (bin >= 0) {
        if (b != bin) return;
        b = bins.within(d, bin);
        if (fine >= 0) {
          const uint32_t k = ordered(x);
          if (b != fine || (shift < 24 && (k >> (shift + 8)) != prefix)) return;
          b = 255 - int((k >> shift) & 255);
        }
      }
      if (by_mass)
        add_mass(b, d);
      else
        atomicAdd(&s.hist[0][b], 1u);
    });
    find_bin(by_mass ? kMass : kTokens, target);
  }

  // Boundary of the first target() tokens, or of the least prefix with a mass of
  // target(sum over the bins). True: the first CTA holds every token down to it in
  // its lists, those in the boundary's bin in the second. False: `cut` is the
  // exact boundary.
  template <typename F>
  __device__ __forceinline__ bool boundary(bool by_mass, Bins bins, F target, Cut& cut) {
    uint64_t left = 0;
    float deepest = bins.high;
    int bin = -1, part = kWhole;
    uint32_t prefix = 0;
    // bins, the parts of one bin, then (ties fill that part) four digits
#pragma unroll 1
    for (int level = 0; level < 6; ++level) {
      const int shift = 40 - 8 * level;
      count(by_mass, [&](uint64_t sum) { return level == 0 ? target(sum) : left; }, deepest, bins, bin, part, shift, prefix);
      left = s.left;
      if (level >= 2) {
        prefix = (prefix << 8) | uint32_t(255 - s.bin);
        continue;
      }
      if (s.bin < 0) {  // fewer tokens with weight than the target: all stay
        cut = {-INFINITY, 0};
        return false;
      }
      if (level == 0) {
        bin = s.bin;
        deepest = bins.end(bin);
      } else {
        part = s.bin;
      }
      if (level == 0)
        gather<3>(bins.first(bin, kWhole), bins.first(bin + 1, kWhole));
      else
        gather<2>(bins.first(bin, part), bins.first(bin, part + 1));
      if (level == 0 && one_list()) {
        listed_depth = deepest;
        return true;
      }
      if (listed[1] <= kListMax) {
        cut = settle(by_mass, left, bins.part(bin, part));
        return false;
      }
      forget();
    }
    cut.x = from_ordered(prefix);
    const uint64_t one = weight(odds(cut.x));
    cut.ties = by_mass ? (one ? (left + one - 1) / one : 1) : left;
    return false;
  }
  // The cut with a mass of `wanted`, `before` of it less deep than low, in [low, high).
  // Where it falls is read from a histogram of rounded masses, of one 32-bit addition
  // per token, with a margin; sums and the tokens listed there make it exact, or
  // narrow the interval. False: ties fill it. Over flat logits one fp32 row takes 39 us, 42
  // with exact histograms (two or three additions a token, and a pass more), 256
  // mixed bf16 rows 64 and 70.
  __device__ __forceinline__ bool estimated(float low, float high, uint64_t before, uint64_t wanted, Cut& cut) {
#pragma unroll 1
    for (int tries = 0; tries < 3; ++tries) {
      const Bins bins = {low, high, kBins / (high - low)};
      clear_hist(fresh);
      fresh = false;
      const float lift = low + float(limb);
      unsigned int* mine = s.hist[lane % 3];  // three copies: bf16 logits crowd into few bins
      each(high, [&](float x, int) {
        const float d = depth(x);
        if (bins.has(d)) atomicAdd(mine + bins.of(d), __float2uint_rn(ex2(lift - d)));
      });
      // 2^-40 units to 2^-lift
      const uint64_t target = uint64_t(float(wanted - before) * ex2(lift - 40.0f)), margin = target >> 11;
      find_bin(kCopies, [&](uint64_t) { return max64(target - margin, 1); }, 2 * margin);
      const float from = bins.first(max(s.bin, 0), kWhole), end = bins.first(s.past_bin + 1, kWhole);
      gather<2, 2>(from, end, Ends{{from, end}});
      if (sums[0] < wanted && wanted <= sums[1]) {
        if (listed[1] <= kListMax) {
          cut = settle(true, wanted - sums[0], {from, end, kBins / (end - from)});
          return true;
        }
        low = from, high = end, before = sums[0];
      } else if (sums[0] < wanted) {
        low = end, before = sums[1];
      } else {
        high = from;
      }
      forget();
    }
    return false;
  }
  bool fresh = true;  // the histogram has not been used yet
  static __device__ __forceinline__ Bins all_depths() { return {0.0f, kReach, kBins / kReach}; }

  // The cut inside the second list, for all. Empties the lists.
  __device__ __forceinline__ Cut settle(bool by_mass, uint64_t left, Bins bins) {
    const int n = int(listed[1]);
    if (rank == 0) {
      __syncthreads();
      uint64_t w[2], mass[2], last = ~uint64_t(0);
      bool in[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int i = tid + h * kSampleThreads;
        in[h] = i < n;
        w[h] = in[h] ? s.lists[1][i] : 0;
        mass[h] = in[h] ? weight(odds(from_ordered(uint32_t(w[h] >> 32)))) : 0;
      }
      keep_first(w, mass, in, bins, by_mass, left);
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (in[h]) last = min(last, w[h]);  // the smallest word that stays
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) last = min(last, shfl_xor64(last, o));
      if (lane == 0) s.part[warp] = last;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < kSampleWarps; ++k) last = min(last, s.part[k]);
      const uint32_t key = uint32_t(last >> 32);
      int ties = 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) ties += __syncthreads_count(in[h] && uint32_t(w[h] >> 32) == key);
      if (tid < ranks) {
        SampleShared* to_cta = of(&s, tid);
        to_cta->cut_x = from_ordered(key);
        to_cta->cut_ties = uint64_t(ties);
      }
    }
    forget();  // a barrier behind the sending
    return {s.cut_x, s.cut_ties};
  }

  // Kept mass of a vector's tokens above a cut, and how many equal it.
  __device__ __forceinline__ void look(const uint4& w, Cut cut, float min_p, uint64_t& mass, unsigned& ties) const {
    WeightSum sum;
    ties = 0;
    each_of(w, 0, [&](float x, int) {
      const float o = ex2(-depth(x));  // NaN where the largest logit is infinite: its equals are ties
      sum.add(x > cut.x && o >= min_p ? o : 0.0f);
      ties += x == cut.x;
    });
    mass = sum.value();
  }

  // How many logits equal x; for every CTA.
  __device__ __forceinline__ uint64_t count_equal(float x) {
    uint64_t sum = 0;
    each_vector<true>([&](const uint4& w, int) {
      each_of(w, 0, [&](float y, int) { sum += y == x; });
    });
    return cluster_sum(sum);
  }
  // Mass of the tokens that a cut keeps; for every CTA.
  __device__ __forceinline__ uint64_t kept_mass(Cut cut) {
    uint64_t sum = 0;
    each_vector<true>([&](const uint4& w, int) {
      uint64_t m;
      unsigned ties;
      look(w, cut, 0.0f, m, ties);
      sum += m;
    });
    return cluster_sum(sum) + (cut.ties ? cut.ties * weight(odds(cut.x)) : 0);
  }
  __device__ uint64_t cluster_sum(uint64_t sum) {
    sum = warp_sum64(sum);
    if (lane == 0) s.part[warp] = sum;
    __syncthreads();
    sum = 0;
    for (int w = 0; w < kSampleWarps; ++w) sum += s.part[w];
    if (tid < ranks) of(&s, tid)->slice_mass[rank] = sum;
    sync_all();
    sum = 0;
    for (int r = 0; r < ranks; ++r) sum += s.slice_mass[r];
    sync_all();  // slice_mass is free again
    return sum;
  }

  // The cut's tokens in index order: each warp owns a contiguous range of
  // vectors in kPieces pieces, a lane a vector at a time.
  __device__ __forceinline__ void search(int row, Cut cut, float min_p) {
    const float tie_odds = cut.ties ? odds(cut.x) : 0.0f;
    const uint64_t one = weight(tie_odds), most_ties = tie_odds >= min_p ? cut.ties : 0;
    const int steps = (to - from + kSampleThreads - 1) / kSampleThreads;  // of a warp, 32 vectors each
    const int per = (steps + kPieces - 1) / kPieces;                      // steps of a piece
    const int first = min(from + warp * steps * 32, to), end = min(first + steps * 32, to);
    uint64_t sum = 0;
    unsigned ties = 0;
    for (int piece = 0, v = first; v < end; piece += kBatch) {
      uint64_t mass[kBatch] = {};
      unsigned equal[kBatch] = {};
      for (int k = 0; k < per; ++k) {
        uint4 w[kBatch];
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          const int at_v = v + (b * per + k) * 32 + lane;
          w[b] = vector(at_v < end ? at_v : to);
        }
#pragma unroll
        for (int b = 0; b < kBatch; ++b) {
          uint64_t m;
          unsigned n;
          look(w[b], cut, min_p, m, n);
          mass[b] += m;
          equal[b] += n;
        }
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        mass[b] = warp_sum64(mass[b]);
        equal[b] = __reduce_add_sync(0xFFFFFFFFu, equal[b]);
        if (lane == 0 && piece + b < kPieces)
          s.piece_mass[warp][piece + b] = mass[b], s.piece_ties[warp][piece + b] = equal[b];
        sum += mass[b];
        ties += equal[b];
      }
      v += kBatch * per * 32;
    }
    if (lane == 0) s.part[warp] = sum, s.warp_ties[warp] = ties;
    __syncthreads();
    uint64_t slice_sum = 0, sum_before = 0, slice_ties = 0, ties_before = 0;
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) {
      if (w == warp) sum_before = slice_sum, ties_before = slice_ties;
      slice_sum += s.part[w];
      slice_ties += s.warp_ties[w];
    }
    if (tid < ranks) {
      SampleShared* there = of(&s, tid);
      there->slice_mass[rank] = slice_sum;
      there->slice_ties[rank] = unsigned(slice_ties);
    }
    sync_all();
    uint64_t all = 0, seen = 0;
    for (int r = 0; r < ranks; ++r) {
      if (r == rank) sum_before += all, ties_before += seen;
      all += s.slice_mass[r];
      seen += s.slice_ties[r];
    }
    auto kept_ties = [&](uint64_t n) { return min(n, most_ties) * one; };
    const uint64_t kept = all + kept_ties(seen);
    const uint64_t target = part24(uniform24(row), kept, 0);
    if (target < sum_before + kept_ties(ties_before) || target >= sum_before + sum + kept_ties(ties_before + ties)) return;
    // this warp holds the answer: its piece, then 32 vectors, then the vector
    int v = first;
    for (int piece = 0; piece < kPieces; ++piece) {
      const uint64_t s1 = sum_before + s.piece_mass[warp][piece], t1 = ties_before + s.piece_ties[warp][piece];
      if (target < s1 + kept_ties(t1)) break;
      sum_before = s1;
      ties_before = t1;
      v += per * 32;
    }
    for (; v < end; v += 32) {
      uint64_t m;
      unsigned n;
      const uint4 w = vector(v + lane < end ? v + lane : to);
      look(w, cut, min_p, m, n);
      unsigned upto = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned y = __shfl_up_sync(0xFFFFFFFFu, upto, o);
        if (lane >= o) upto += y;
      }
      const uint64_t run = sum_before + warp_scan64(m), t1 = ties_before + upto;
      const unsigned past = __ballot_sync(0xFFFFFFFFu, run + kept_ties(t1) > target);
      if (past) {
        if (lane != __ffs(past) - 1) return;
        uint64_t s0 = run - m, t0 = t1 - n;
        bool done = false;
        each_of(w, (v + lane) * kVector - lead, [&](float x, int i) {
          const float o = ex2(-depth(x));
          if (x > cut.x && o >= min_p) s0 += weight(o);
          t0 += x == cut.x;
          if (!done && s0 + kept_ties(t0) > target) {
            done = true;
            answer(row, i, x, kept);
          }
        });
        return;
      }
      sum_before = __shfl_sync(0xFFFFFFFFu, run, 31);
      ties_before = __shfl_sync(0xFFFFFFFFu, t1, 31);
    }
  }

  // Which of n threads' largest logits bounds about kTopPList tokens: with m tokens spread
  // evenly above a bound, n (1 - exp(-m / n)) threads hold one.
  static __device__ __forceinline__ int likely(int n) {
    return max(1, int(float(n) * (1.0f - ex2(-kTopPList * kLog2e / float(n)))));
  }
  __device__ __forceinline__ uint64_t uniform24(int row) const {
    return min(16777215u, __float2uint_rz(fmaxf(p.uniform[row], 0.0f) * 16777216.0f));
  }
  static __device__ __forceinline__ uint64_t need(float top_p, uint64_t total) {
    return max64(part24(__float2uint_rn(fmaxf(top_p, 0.0f) * 16777216.0f), total, 0xFFFFFFu), 1);
  }

  // First CTA: its lists hold every kept token. total: W_K, unless top-k
  // filters here (then it is the first `most` tokens' mass).
  __device__ __forceinline__ void finish(int row, int most, float top_p, float min_p, uint64_t total) {
    const int a = int(listed[0]), n = a + int(listed[1]);
    uint64_t w[2], mass[2];
    bool in[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = tid + h * kSampleThreads;
      in[h] = i < n;
      w[h] = !in[h] ? 0 : i < a ? s.lists[0][i] : s.lists[1][i - a];
      mass[h] = in[h] ? weight(odds(from_ordered(uint32_t(w[h] >> 32)))) : 0;
    }
    const Bins bins = {0.0f, listed_depth, kBins / listed_depth};
    if (most < n) keep_first(w, mass, in, bins, false, most);
    if (most < p.vocab) block_scan64((in[0] ? mass[0] : 0) + (in[1] ? mass[1] : 0), s.part, total);
    if (top_p < 1.0f) keep_first(w, mass, in, bins, true, need(top_p, total));
#pragma unroll
    for (int h = 0; h < 2; ++h)
      if (!in[h] || odds(from_ordered(uint32_t(w[h] >> 32))) < min_p) mass[h] = 0;
    choose(row, w, mass);
  }

  // First CTA, two words per thread (`in`: still kept) and their masses: takes out
  // those with `target` or more ahead of them in tokens, or in mass. A histogram,
  // and the words of the boundary's bin against one another.
  __device__ __forceinline__ void keep_first(const uint64_t (&w)[2], const uint64_t (&mass)[2], bool (&in)[2],
                                             Bins bins, bool by_mass, uint64_t target) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) s.hist[k][tid] = 0;
    if (tid == 0) s.staged_count[0] = 0, s.bin = kBins;
    __syncthreads();
    int bin[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bin[h] = -1;
      if (!in[h]) continue;
      bin[h] = bins.of(depth(from_ordered(uint32_t(w[h] >> 32))));
      if (by_mass)
        add_to(bin[h], mass[h]);
      else
        atomicAdd(&s.hist[0][bin[h]], 1u);
    }
    __syncthreads();
    uint64_t sum;
    const uint64_t here = by_mass ? bin_mass() : s.hist[0][tid], upto = block_scan64(here, s.part, sum);
    if (upto - here < target && target <= upto) {
      s.bin = tid;
      s.left = target - (upto - here);
    }
    __syncthreads();
    const int edge = s.bin;
    const uint64_t left = s.left;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!in[h]) continue;
      in[h] = bin[h] <= edge;
      if (bin[h] != edge) continue;
      const unsigned place = atomicAdd(&s.staged_count[0], 1u);
      s.staged[0][place] = w[h];
      s.staged[1][place] = by_mass ? mass[h] : 1;
    }
    __syncthreads();
    const unsigned count = s.staged_count[0];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!in[h] || bin[h] != edge) continue;
      uint64_t before = 0;
      for (unsigned j = 0; j < count; ++j) before += s.staged[0][j] > w[h] ? s.staged[1][j] : 0;
      in[h] = before < left;
    }
  }

  // First CTA, a token of every kept word (its mass; 0: none) per thread and half:
  // the answer in index order. The masses by 512 ranges of indexes, then the
  // tokens of the range that holds the target.
  __device__ __forceinline__ void choose(int row, const uint64_t (&w)[2], const uint64_t (&mass)[2]) {
    const uint32_t range = uint32_t(p.vocab + kBins - 1) / kBins;
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 3; ++k) s.hist[k][tid] = 0;
    if (tid == 0) s.staged_count[0] = 0;
    __syncthreads();
    int bin[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bin[h] = mass[h] ? int(~uint32_t(w[h]) / range) : -1;
      if (bin[h] >= 0) add_to(bin[h], mass[h]);
    }
    __syncthreads();
    uint64_t total;
    const uint64_t here = bin_mass(), upto = block_scan64(here, s.part, total);
    const uint64_t target = part24(uniform24(row), total, 0);
    if (upto - here <= target && target < upto) {
      s.bin = tid;
      s.left = target - (upto - here);
    }
    __syncthreads();
    const int wanted = s.bin;
    const uint64_t left = s.left;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (bin[h] != wanted) continue;
      const unsigned place = atomicAdd(&s.staged_count[0], 1u);
      s.staged[0][place] = w[h];
      s.staged[1][place] = mass[h];
    }
    __syncthreads();
    const unsigned count = s.staged_count[0];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (bin[h] != wanted) continue;
      uint64_t before = 0;
      for (unsigned j = 0; j < count; ++j)
        before += uint32_t(s.staged[0][j]) > uint32_t(w[h]) ? s.staged[1][j] : 0;  // ~index: a smaller index
      if (before <= left && left < before + mass[h])
        answer(row, ~uint32_t(w[h]), from_ordered(uint32_t(w[h] >> 32)), total);
    }
  }

  // First CTA, behind boundary(): the first list is kept whole, and of the
  // second the tokens with less than s.left (tokens, or mass) before them.
  __device__ __forceinline__ void finish_bounded(int row, bool by_mass, float min_p) {
    const int a = int(listed[0]), n = a + int(listed[1]);
    const uint64_t left = s.left;
    uint64_t w[2], mass[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = tid + h * kSampleThreads;
      w[h] = i < a ? s.lists[0][i] : i < n ? s.lists[1][i - a] : 0;
      const float o = i < n ? odds(from_ordered(uint32_t(w[h] >> 32))) : -1.0f;
      mass[h] = o >= min_p ? weight(o) : 0;
      if (i >= a && i < n) s.bins[i - a] = by_mass ? weight(o) : 1;
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = tid + h * kSampleThreads;
      if (i < a || i >= n) continue;
      uint64_t before = 0;
      for (int j = 0; j < n - a; ++j) before += s.lists[1][j] > w[h] ? s.bins[j] : 0;
      if (before >= left) mass[h] = 0;
    }
    choose(row, w, mass);
  }

  // The same for up to kFew tokens, each against all: the four threads of a token
  // look at a part of the others each and add up what is ahead of it. Top-k 50 12.9 us
  // for a row, 13.6 with histograms; for 183 tokens these are faster.
  __device__ __forceinline__ void finish_few(int row, int most, float top_p, float min_p, uint64_t total) {
    const int a = int(listed[0]), n = a + int(listed[1]);
    const int i = tid >> 2, part = tid & 3;
    const bool mine = i < n;
    const uint64_t word = !mine ? 0 : i < a ? s.lists[0][i] : s.lists[1][i - a];
    const float o = mine ? odds(from_ordered(uint32_t(word >> 32))) : 0.0f;
    const uint64_t mass = mine ? weight(o) : 0;
    __syncthreads();
    ulonglong2* pairs = reinterpret_cast<ulonglong2*>(s.lists[0]);  // (word, mass)
    if (part == 0 && mine) pairs[i] = make_ulonglong2(word, mass);
    uint64_t sum;
    block_scan64(part == 0 ? mass : 0, s.part, sum);  // and a barrier
    auto joined = [&](uint64_t v) {
      v += shfl_xor64(v, 1);
      return v + shfl_xor64(v, 2);
    };
    uint64_t ahead = 0, before = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 4) {
      const ulonglong2 other = pairs[j];
      if (other.x > word) {
        ++ahead;
        before += other.y;
      }
    }
    ahead = joined(ahead);
    before = joined(before);
    if (most < p.vocab) {  // the first `most` tokens' mass
      if (mine && ahead + 1 == uint64_t(most)) s.left = before + mass;
      __syncthreads();
      total = n < most ? sum : s.left;
    }
    const uint64_t limit = top_p < 1.0f ? need(top_p, total) : ~uint64_t(0);
    const bool keep = mine && ahead < uint64_t(most) && before < limit && o >= min_p;
    __syncthreads();
    if (part == 0 && mine && !keep) pairs[i].y = 0;
    block_scan64(part == 0 && keep ? mass : 0, s.part, sum);
    before = 0;
#pragma unroll 4
    for (int j = part; j < n; j += 4) {
      const ulonglong2 other = pairs[j];
      before += uint32_t(other.x) > uint32_t(word) ? other.y : 0;  // ~index: a smaller index
    }
    before = joined(before);
    const uint64_t target = part24(uniform24(row), sum, 0);
    if (part == 0 && keep && before <= target && target < before + mass)
      answer(row, ~uint32_t(word), from_ordered(uint32_t(word >> 32)), sum);
  }

  // Where a batch makes more CTAs than run at once: the rows that are dear (top-p
  // alone, or a large K) come first, the y-th of them for cluster y; behind
  // them every CTA of a cluster takes one of the other rows by itself, without the
  // cluster's barriers. Returns the row, or -1: none is left. Without it 256
  // rows took 58 us instead of 31 with top-k 50, 20 instead of 11 greedy; unfiltered ones
  // take 47 us as cheap rows, 72 as dear ones; 256 mixed ones 200 if all were cheap, 60.
  __device__ __forceinline__ int assign(int y) {
    auto dear = [&](int r) {
      const float t = p.temperature ? p.temperature[r] : 1.0f;
      const int k = p.top_k ? p.top_k[r] : 0;
      const float top_p = p.top_p ? p.top_p[r] : 1.0f;
      return t > 0.0f && (k > kListMax / 2 || (k <= 0 && top_p < 1.0f));
    };
    int all = 0;
    for (int r = tid; r - tid < p.rows; r += kSampleThreads) all += __syncthreads_count(r < p.rows && dear(r));
    const bool wanted = y < all;
    int skip = y;  // rows of this kind before the one looked for
    if (!wanted) {
      skip = (y - all) * ranks + rank;
      if (skip >= p.rows - all) return -1;
      rank = 0;
      ranks = 1;
    }
    for (int r = tid; r - tid < p.rows; r += kSampleThreads) {
      const bool is = r < p.rows && dear(r) == wanted;
      const unsigned lanes = __ballot_sync(0xFFFFFFFFu, is);
      if (lane == 0) s.warp_ties[warp] = __popc(lanes);
      const int here = __syncthreads_count(is);
      if (skip < here) {
        int before = __popc(lanes & ((1u << lane) - 1u));
        for (int w = 0; w < warp; ++w) before += s.warp_ties[w];
        if (is && before == skip) s.bin = r;
        __syncthreads();
        return s.bin;
      }
      skip -= here;
      __syncthreads();  // warp_ties is free again
    }
    return -1;
  }

  __device__ void run(int row) {
    at = p.logits + row * p.row_bytes;
    lead = int(reinterpret_cast<uintptr_t>(at) & 15) / int(sizeof(Raw));
    const int vectors = (p.vocab + lead + kVector - 1) / kVector;
    from = int(int64_t(vectors) * rank / ranks);
    to = int(int64_t(vectors) * (rank + 1) / ranks);
    limb = __clz(max((to - from) * kVector, 2 * kSampleThreads));
    const float t = p.temperature ? p.temperature[row] : 1.0f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    float min_p = p.min_p ? p.min_p[row] : 0.0f;
    if (tid == 0) s.found[0] = s.found[1] = 0;
    keep_ends(vectors);
    if (ranks > 1) cluster.barrier_arrive();
    float mine = -INFINITY;  // this thread's largest logit
    int where = from;
    each_vector<false>([&](const uint4& w, int v) {
      const float x = L::largest(w);
      if (x > mine) mine = x, where = v;
    });
    uint64_t best = (uint64_t(ordered(mine)) << 32) | uint32_t(~where);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) best = max64(best, shfl_xor64(best, o));
    if (lane == 0) s.part[warp] = best;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kSampleWarps; ++w) best = max64(best, s.part[w]);
    if (ranks > 1) {
      cluster.barrier_wait();  // every CTA of the cluster runs: its shared memory may be written
      if (tid < ranks) of(&s, tid)->top[rank] = best;
      sync_all();
      for (int r = 0; r < ranks; ++r) best = max64(best, s.top[r]);
    } else {
      __syncthreads();  // every warp has read s.part: a search without a filter writes it next
    }
    top = from_ordered(uint32_t(best >> 32));
    inverse = kLog2e / t;
    const bool greedy = !(t > 0.0f);
    const int most = greedy ? 1 : k > 0 ? min(k, p.vocab) : p.vocab;
    if (top == -INFINITY) {  // nothing to choose from
      if (rank == 0 && tid == 0) {
        p.tokens[row] = -1;
        if (p.logprobs) p.logprobs[row] = -INFINITY;
      }
      return;
    }
    if (most == 1) {
      const int v = int(~uint32_t(best));
      if (tid == 0 && v >= from && v < to) {
        int first = p.vocab;
        each_of(vector(v), v * kVector - lead, [&](float x, int i) {
          if (x == top) first = min(first, i);
        });
        p.tokens[row] = first;
        if (p.logprobs) p.logprobs[row] = 0.0f;
      }
      return;
    }
    min_p = min_p > 0.0f ? fminf(min_p, 1.0f) : 0.0f;  // the most likely token always stays; NaN: off
    const bool by_count = most < p.vocab, by_mass = top_p < 1.0f;
    Cut cut = {-INFINITY, 0};
    bool complete = false;  // the first CTA's lists hold every kept token
    bool bounded = false;   // and s.left of the second list's count or mass is kept
    uint64_t total = 0;
    if (isinf(top) || isinf(inverse)) {
      // only the largest logit's equals have odds, of 1 each
      inverse = 0.0f;
      const uint64_t one = weight(1.0f), ties = min(count_equal(top), uint64_t(most));
      cut = {top, by_mass ? min(ties, (need(top_p, ties * one) + one - 1) / one) : ties};
    } else {
      Bins bins = all_depths();
      const bool summed = by_mass && !by_count;
      if (by_count || by_mass || min_p > 0.0f) {
        // min-p cuts the gathered tokens unless top-p needs the mass of all K
        float deepest = min_p > 0.0f && !by_mass ? fminf(kReach, -log2f(min_p) * 1.00001f + 1e-4f) : kReach;
        if (by_count || by_mass) {
          clear_hist(true);
          fresh = false;
          const float d = depth(mine);
          if (bins.has(d)) atomicAdd(&s.hist[0][bins.of(d)], 1u);
          const int aim = by_count ? most : likely(min(vectors, ranks * kSampleThreads));
          find_bin(kTokens, [&](uint64_t) { return uint64_t(aim); });
          if (s.bin >= 0) deepest = fminf(deepest, bins.end(s.bin));  // otherwise whatever has weight can be kept
        }
        if (summed) {
          gather<1, 3>(deepest, deepest, Ends{{deepest, deepest + kBandWidth, kReach}});
          total = sums[2];
          complete = one_list() && sums[0] >= need(top_p, total);
        } else {
          gather<1>(deepest, deepest);
          complete = one_list();
        }
        if (!complete) forget();
        listed_depth = deepest;
      }
      // the exact cuts, by count and then by mass
#pragma unroll 1
      for (int pass = by_count ? 0 : 1; pass < (by_mass ? 2 : 1) && !complete; ++pass) {
        if (pass == 1 && by_count) total = kept_mass(cut);
        uint64_t before = 0;
        Cut next = cut;
        if (summed) {
          const float ends[] = {0.0f, listed_depth, listed_depth + kBandWidth, kReach};
          int band = 0;
          while (band < kBands && sums[band] < need(top_p, total)) before = sums[band++];
          bins = {ends[band], fminf(ends[band + 1], kReach), 0.0f};
          bins.scale = kBins / (bins.high - bins.low);
          if (estimated(bins.low, bins.high, before, need(top_p, total), cut)) break;
        }
        complete = boundary(pass == 1, bins, [&](uint64_t) {
          if (pass == 0) return uint64_t(most);
          return need(top_p, total) - before;
        }, next);
        if (cut.ties == 0 || next.x > cut.x || (next.x == cut.x && next.ties < cut.ties)) cut = next;
        bounded = complete && !(pass == 0 && by_mass);
      }
    }
    if (!complete) return search(row, cut, min_p);
    if (rank == 0) {
      if (ranks == 1) __syncthreads();
      const unsigned n = listed[0] + listed[1];
      // a mass W_K that is known replaces the first K tokens' mass
      const int first = total ? p.vocab : most;
      if (bounded && listed[1] <= kFewTied)
        finish_bounded(row, by_mass, min_p);
      else if (n <= kFew)
        finish_few(row, first, top_p, min_p, total);
      else
        finish(row, first, top_p, min_p, total);
    }
    if (ranks > 1) cluster.barrier_wait();  // the other CTAs have read the first one's counts
  }
};

template <typename L>
__global__ void __launch_bounds__(kSampleThreads, 2) sample_kernel(const __grid_constant__ SampleParams p) {
  __shared__ SampleShared shared;
  grid_dep_wait();
  Sampler<L> sampler(p, shared);
  const int row = p.by_cost ? sampler.assign(blockIdx.y) : int(blockIdx.y);
  if (row >= 0) sampler.run(row);
}

template <typename L>
static int run_sample(const char* what, SampleParams p, int rows, cudaStream_t stream) {
  // CTAs of a row: more than run at once in all, since rows differ by ten times in
  // work, with 8192 logits each at least. 256 rows of 128256 bf16 logits with mixed
  // filters take 85 / 60 / 78 us with 2 / 4 / 8 CTAs a row, 500 200 / 100 / 112, 150 84 / 61 / 50.
  int ranks = 1;
  while (ranks < kClusterMax && ((rows * ranks < 4 * sm_count() && p.vocab > ranks * 8192) || p.vocab > ranks * kSliceMax))
    ranks <<= 1;
  CB_REQUIRE(p.vocab <= ranks * kSliceMax, "%s: vocab=%d (at most %d)", what, p.vocab, kClusterMax * kSliceMax);
  p.rows = rows;
  p.by_cost = ranks > 1 && rows * ranks > 2 * sm_count() && p.vocab <= kSliceMax;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ranks, rows);
  cfg.blockDim = dim3(kSampleThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ranks;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.numAttrs = 1;
  if (pdl_enabled()) {
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 2;
  }
  cfg.attrs = attr;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, sample_kernel<L>, p);
  if (e != cudaSuccess) return fail(kErrCuda, "%s: launch failed: %s", what, cudaGetErrorString(e));
  return check_launch(what);
}

}  // namespace cb

using namespace cb;

extern "C" int cb_sample(const void* logits, int dtype, int64_t row_stride, int rows, int vocab,
                         const float* temperature, const int32_t* top_k, const float* top_p, const float* min_p,
                         const float* uniform, int64_t* tokens, float* logprobs, void* stream) {
  const char* what = "cb_sample";
  CB_REQUIRE(dtype == CB_BF16 || dtype == CB_FP16 || dtype == CB_FP32, "%s: dtype=%d", what, dtype);
  CB_REQUIRE(rows >= 0 && rows <= 65535 && vocab >= 1, "%s: rows=%d vocab=%d", what, rows, vocab);
  if (rows == 0) return kOk;
  CB_REQUIRE(logits && uniform && tokens, "%s: null pointer", what);
  SampleParams p = {};
  p.logits = static_cast<const char*>(logits);
  p.row_bytes = row_stride * (dtype == CB_FP32 ? 4 : 2);
  p.vocab = vocab;
  p.temperature = temperature, p.top_p = top_p, p.min_p = min_p, p.uniform = uniform;
  p.top_k = top_k;
  p.tokens = tokens, p.logprobs = logprobs;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == CB_FP32   ? run_sample<F32Logits>(what, p, rows, s)
         : dtype == CB_BF16 ? run_sample<HalfLogits<Bf16>>(what, p, rows, s)
                            : run_sample<HalfLogits<Fp16>>(what, p, rows, s);
}
