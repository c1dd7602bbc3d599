// Attention of one new token per sequence over a paged key-value cache.
//
//   s_j = scale * q . k_j,  o = sum_j exp(s_j - m) v_j / l,
//   m = max_j s_j, l = sum_j exp(s_j - m), lse = m + log l,
// over the positions j < lengths[b] of sequence b, whose page is
// table[b][j / page_size]. A sequence of length 0 gives o = 0, lse = -inf.
//
// Bound: a position's K and V are read once for q_heads / kv_heads flop per byte
// (1 to 16), so HBM bounds it and the kernel keeps HBM busy:
//
// * The work of a launch is cut into units of 64 positions of one (sequence,
//   KV head), in that order, and every CTA takes an equal contiguous share of
//   all units (two CTAs per SM; a segment's beginning counts as two units).
//   Ragged batches balance by themselves, nothing is known on the host, and a
//   captured launch serves any lengths. A CTA's share covers whole (sequence, head) segments except at its two ends; such
//   an end is a partial (m, l, o) in the workspace and the last CTA of the
//   segment to finish (ticket) joins the parts in CTA order, so the result
//   does not depend on which that is.
// * The 4 warps of a CTA take 16 positions of a unit each and never wait for
//   one another inside a segment: every warp has its own ring of cp.async
//   stages, which runs ahead over the ends of segments. The gather is by row,
//   so pages may have any size and may end inside a tile. Rows behind the
//   length (or on a page that does not exist) are zero-filled, not read.
// * All query heads of a KV head share one read of its rows. Scores and outputs
//   are computed transposed, S^T = K Q^T and O^T = V^T P^T, so that the 16
//   rows of mma.m16n8k16 are cache positions (or head dimensions) and the 8
//   columns are query heads: a group of 4 fills half of an MMA, not a quarter.
//   mma.sync rather than tcgen05: the latter's smallest tile has 64 rows, and at
//   these ratios the tensor pipe is idle most of the time either way.
// * Softmax statistics and sums are fp32. P enters the second product as the
//   sum of two 16-bit values (rounded, and the rest): weights to 2^-16 (bf16) or
//   2^-22 (fp16), where one value leaves 2^-8 or 2^-11. The output's own rounding
//   hides that but for 1 to 3 in 1000 outputs, which differ in their last place.
//
// Measured: 858,000 positions of 8 KV heads x 128 in 523 us = 6.8 TB/s (a plain copy
// moves 6.5); 32 sequences of 1 to 4096 positions 19.8 us (17.5 with the pages in L2);
// one of 77 4.5 us.
#include "cascade_b200.h"
#include "internal.h"
#include "paged_device.cuh"

namespace cb {

int32_t* error_word();

struct PagedParams {
  const uint16_t *q, *k, *v;
  int64_t q_token, q_head, table_stride;
  const int32_t *table, *lengths;
  uint16_t* out;
  float* lse;
  unsigned int* tickets;  // one per CTA
  float* parts;           // two slots per CTA: kMaxRows rows of D outputs, then (m, l) pairs
  int sequences, kv_heads, group, row_tiles, pages, page_size;
  int capacity;  // positions of a table row
  uint32_t page_mul, page_shift;  // j / page_size = j * page_mul >> (31 + page_shift) for j < 2^31
  float scale_log2;
  int* err;
};

constexpr int kPagedWarps = 4;
constexpr int kPagedThreads = kPagedWarps * 32;
constexpr int kTile = 16;                   // positions of a warp's step
constexpr int kUnit = kTile * kPagedWarps;  // positions of a CTA's step
constexpr int kStages = 3;
constexpr int kPagedCtas = 2;               // per SM
constexpr int kMaxRows = 16;                // query heads of a CTA's segment
// Beginning and ending a segment (its queries, the join of the warps) takes about as
// long as this many units. With 0 / 1 / 2 / 3: 32 sequences of 1 to 4096 positions
// 21.4 / 19.9 / 19.7 / 20.2 us, 100 of 10 to 800 26.0 / 22.7 / 23.8 / 25.4, one of 77
// 7.3 / 8.9 / 4.5 / 6.4.
constexpr int kSegmentCost = 2;
// A CTA's share at least, in places: parts cost 2 us for the ticket and 0.1 to
// 0.2 us each for the join, the units of a share follow one another. With 1 / 2 / 4 /
// 8: one sequence of 77 positions (32 query and 8 KV heads of 128) 6.4 / 4.6 / 4.6 /
// 7.3 us, of 2048 12.0 / 10.4 / 10.9 / 14.1, of 32,000 32 with each; of 8 and 2 heads of
// 64 5.9 / 4.1 / 4.1 / 6.4, 7.8 / 7.3 / 8.7 / 11.5 and 24.3 / 24.4 / 22.2 / 17.7; 12 of
// 100 to 20,000, 8 heads over one of 64, 20.1 / 20.2 / 17.4 / 15.9. Short sequences
// want less, long ones of few KV heads more.
constexpr int kShareMin = 4;
constexpr int kTicketBytes = 4096;

template <int D>
struct PagedSmem {
  static constexpr int kStageBytes = kTile * D * 2 * 2;  // K rows, then V rows
  static constexpr int kBytes = kPagedWarps * kStages * kStageBytes;
};
template <int D>
constexpr int64_t kPartFloats = kMaxRows * (D + 2);

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool read) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(read ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma(Bf16, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma(Fp16, float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Weights are held as exp2(s - m + kLift): fp16 ends at 2^-24, so lifting the
// largest weight to 2^10 keeps weights down to 2^-34 of it.
template <typename T>
constexpr float kLift = 0.0f;
template <>
constexpr float kLift<Fp16> = 10.0f;

__device__ __forceinline__ int paged_length(const PagedParams& p, int b) {
  return max(0, min(p.lengths[b], p.capacity));
}
// Units of a sequence per head; an empty one has one, which writes its zeros.
__device__ __forceinline__ int unit_count(int length) { return max(1, (length + kUnit - 1) / kUnit); }

// A unit in the launch's order: sequence b, head tile h, unit j. Its place counts
// the units before it and kSegmentCost for every segment up to its own. Place is
// int where the tables' widths keep every place below 2^30: the plan is a chain
// that each CTA walks before its first copy (smallest call 4.5 against 5.0 us, one
// sequence of 2048 positions 10.2 against 10.9), int64_t where they do not.
template <typename Place>
struct Cursor {
  Place place;
  int b, h, j, units, length;
  __device__ __forceinline__ void enter(const PagedParams& p) {
    length = paged_length(p, b);
    units = unit_count(length);
  }
  __device__ __forceinline__ void next(const PagedParams& p, int heads) {
    ++place;
    if (++j < units) return;
    j = 0;
    place += kSegmentCost;
    if (++h == heads) {
      h = 0;
      if (++b < p.sequences) enter(p);
    }
  }
  __device__ __forceinline__ Place first_place() const { return place - j; }
};

__device__ __forceinline__ int quotient(int a, int b) { return uint32_t(a) / uint32_t(b); }
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) { return uint64_t(a) / uint64_t(b); }
// Equal shares of `total` places for `ctas` CTAs; the first ones take one more.
template <typename Place>
struct Shares {
  Place each, more;
  __device__ __forceinline__ Shares(Place total, Place ctas) : each(quotient(total, ctas)), more(total - each * ctas) {}
  __device__ __forceinline__ Place begin(int cta) const { return each * cta + min(Place(cta), more); }
  __device__ __forceinline__ int owner(Place place) const {
    const Place big = more * (each + 1);
    return int(place < big ? quotient(place, each + 1) : more + quotient(place - big, each));
  }
};

// NT: 8-column tiles of query heads (1: groups up to 8, else 2; a group of more
// than 16 heads takes several head tiles, which read K and V again, from L2)
template <typename T, int D, int NT, typename Place>
__global__ void __launch_bounds__(kPagedThreads, kPagedCtas) paged_attention_kernel(const __grid_constant__ PagedParams p) {
  using Smem = PagedSmem<D>;
  constexpr int kChunks = D / 8;              // 16-byte chunks of a row
  constexpr int kRowsPerCopy = 32 / kChunks;  // rows that one warp-wide copy covers
  constexpr int kCopies = kTile / kRowsPerCopy;
  extern __shared__ __align__(1024) uint8_t smem[];
  __shared__ Place s_scan[kPagedWarps];
  __shared__ Place s_first;
  __shared__ int s_b;
  __shared__ uint32_t s_valid[kPagedWarps][kStages];
  __shared__ float2 s_ml[kPagedWarps][kMaxRows];
  __shared__ unsigned int s_ticket;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int heads = p.kv_heads * p.row_tiles;
  grid_dep_wait();

  // ---- this CTA's share of the units
  const int per = (p.sequences + kPagedThreads - 1) / kPagedThreads;
  const int own0 = min(tid * per, p.sequences), own1 = min(own0 + per, p.sequences);
  Place own = 0;
  for (int b = own0; b < own1; ++b) {
    if (blockIdx.x == 0) {
      const int length = p.lengths[b];
      if ((length < 0 || length > p.capacity) && p.err) atomicExch(p.err, kErrPagedLength);
    }
    own += unit_count(paged_length(p, b)) + kSegmentCost;
  }
  Place sum = own;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const Place x = __shfl_up_sync(0xFFFFFFFFu, sum, o);
    if (lane >= o) sum += x;
  }
  if (lane == 31) s_scan[warp] = sum;
  __syncthreads();
  Place total = 0, before = sum - own;
#pragma unroll
  for (int w = 0; w < kPagedWarps; ++w) {
    if (w < warp) before += s_scan[w];
    total += s_scan[w];
  }
  // places: kSegmentCost of them and then the units, for every head of every sequence
  total *= heads;
  before *= heads;
  own *= heads;
  const int ctas = int(min(Place(gridDim.x), (total + kShareMin - 1) / kShareMin));
  if (int(blockIdx.x) >= ctas) return;
  const Shares<Place> shares(total, ctas);
  const Place v0 = shares.begin(blockIdx.x), v1 = shares.begin(blockIdx.x + 1);
  if (v0 >= before && v0 < before + own) {
    int b = own0;
    for (;; ++b) {
      const Place here = Place(unit_count(paged_length(p, b)) + kSegmentCost) * heads;
      if (v0 < before + here) break;
      before += here;
    }
    s_b = b;
    s_first = before;
  }
  __syncthreads();
  Cursor<Place> at;
  at.b = s_b;
  at.enter(p);
  {
    const Place offset = v0 - s_first;
    const int size = at.units + kSegmentCost;
    at.h = int(quotient(offset, Place(size)));
    const Place segment = s_first + Place(at.h) * size;
    at.j = max(0, int(v0 - segment) - kSegmentCost);
    at.place = segment + kSegmentCost + at.j;
  }
  if (at.place >= v1) return;  // a share may end before a segment's first unit

  // ---- the warp's ring
  const uint32_t ring = smem_u32(smem) + warp * (kStages * Smem::kStageBytes);
  const int copy_row = lane / kChunks, copy_chunk = lane % kChunks;
  // `ahead` is the next unit to copy, `probe` the one after it; the page of this
  // lane's row (lane & 15) is looked up two units before its copy, since short
  // sequences would otherwise wait for the table at every unit
  Cursor<Place> ahead = at, probe = at;
  auto look_up = [&]() {
    if (probe.place >= v1) return -1;
    const int j = probe.j * kUnit + warp * kTile + (lane & 15);
    const uint32_t column = uint32_t((uint64_t(uint32_t(j)) * p.page_mul) >> (31 + p.page_shift));
    return j < probe.length ? p.table[probe.b * p.table_stride + column] : -1;
  };
  int page = look_up();
  probe.next(p, heads);
  int next_page = look_up();
  auto issue = [&](int stage) {
    if (ahead.place < v1) {
      const int j = ahead.j * kUnit + warp * kTile + (lane & 15);
      const uint32_t column = uint32_t((uint64_t(uint32_t(j)) * p.page_mul) >> (31 + p.page_shift));
      const bool live = j < ahead.length;
      const bool valid = live && uint32_t(page) < uint32_t(p.pages);
      if (live && !valid && p.err) atomicExch(p.err, kErrPagedPage);
      const int kv = ahead.h / p.row_tiles;
      const uint32_t row = valid ? (uint32_t(page) * p.kv_heads + kv) * p.page_size + (j - column * p.page_size) : 0;
      const unsigned mask = __ballot_sync(0xFFFFFFFFu, valid) & 0xFFFFu;
      if (lane == 0) s_valid[warp][stage] = mask;
      const uint32_t base = ring + stage * Smem::kStageBytes;
      if (mask) {
#pragma unroll
        for (int i = 0; i < kCopies; ++i) {
          const int r = i * kRowsPerCopy + copy_row;
          const int64_t offset = int64_t(__shfl_sync(0xFFFFFFFFu, row, r)) * D + copy_chunk * 8;
          const uint32_t dst = base + r * (D * 2) + ((copy_chunk ^ (r & 7)) << 4);
          const bool read = (mask >> r) & 1;
          cp_async16(dst, p.k + offset, read);
          cp_async16(dst + kTile * D * 2, p.v + offset, read);
        }
      }
      ahead.next(p, heads);
      probe.next(p, heads);
      page = next_page;
      next_page = look_up();
    }
    cp_async_commit();
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) issue(s);

  // ---- the units, segment by segment
  uint32_t qf[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2];
  auto first_head = [&](const Cursor<Place>& c) {
    const int kv = c.h / p.row_tiles;
    return kv * p.group + (c.h - kv * p.row_tiles) * (8 * NT);
  };
  auto row_count = [&](const Cursor<Place>& c) { return min(8 * NT, p.group - (c.h % p.row_tiles) * (8 * NT)); };
  auto load_queries = [&](const Cursor<Place>& c) {
    const int head0 = first_head(c), rows = row_count(c);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int head = n * 8 + (lane >> 2);
      const uint16_t* src = p.q + c.b * p.q_token + (head0 + head) * p.q_head + (lane & 3) * 2;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        qf[n][kk][0] = head < rows ? __ldcg(reinterpret_cast<const unsigned int*>(src + kk * 16)) : 0u;
        qf[n][kk][1] = head < rows ? __ldcg(reinterpret_cast<const unsigned int*>(src + kk * 16 + 8)) : 0u;
      }
    }
  };
  auto clear_state = [&]() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[n][kk][e] = 0.0f;
      m[n][0] = m[n][1] = -INFINITY;
      l[n][0] = l[n][1] = 0.0f;
    }
  };
  const int a_row = (lane & 7) + ((lane >> 3) & 1) * 8, a_chunk = lane >> 4;  // K as the A operand
  const int t_row = (lane & 7) + (lane >> 4) * 8, t_chunk = (lane >> 3) & 1;  // V, transposed
  auto compute = [&](int stage) {
    const unsigned mask = s_valid[warp][stage];
    if (mask == 0) return;
    const uint32_t base = ring + stage * Smem::kStageBytes;
    float s[NT][4] = {};
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      uint32_t a[4];
      ldsm4(a, base + a_row * (D * 2) + (((kk * 2 + a_chunk) ^ (a_row & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) mma(T(), s[n], a, qf[n][kk][0], qf[n][kk][1]);
    }
    const bool low = (mask >> (lane >> 2)) & 1, high = (mask >> ((lane >> 2) + 8)) & 1;
    uint32_t hi[NT][2], rest[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      float grow[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        s[n][c] = low ? s[n][c] * p.scale_log2 : -INFINITY;
        s[n][c + 2] = high ? s[n][c + 2] * p.scale_log2 : -INFINITY;
        float top = fmaxf(s[n][c], s[n][c + 2]);
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, x));
        top = fmaxf(top, m[n][c]);
        const float base_m = (top == -INFINITY ? 0.0f : top) - kLift<T>;
        grow[c] = ex2(m[n][c] - kLift<T> - base_m);
        m[n][c] = top;
        s[n][c] = ex2(s[n][c] - base_m);
        s[n][c + 2] = ex2(s[n][c + 2] - base_m);
        l[n][c] = l[n][c] * grow[c] + s[n][c] + s[n][c + 2];
      }
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const uint32_t w = T::pack(s[n][2 * half], s[n][2 * half + 1]);
        const uint32_t r = T::pack(s[n][2 * half] - T::lo(w), s[n][2 * half + 1] - T::hi(w));
        hi[n][half] = transpose8x8(w);
        rest[n][half] = transpose8x8(r);
      }
#pragma unroll
      for (int t = 0; t < D / 16; ++t) {
        o[n][t][0] *= grow[0];
        o[n][t][1] *= grow[1];
        o[n][t][2] *= grow[0];
        o[n][t][3] *= grow[1];
      }
    }
#pragma unroll
    for (int t = 0; t < D / 16; ++t) {
      uint32_t a[4];
      ldsm4_trans(a, base + kTile * D * 2 + t_row * (D * 2) + (((t * 2 + t_chunk) ^ (t_row & 7)) << 4));
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        mma(T(), o[n][t], a, hi[n][0], hi[n][1]);
        mma(T(), o[n][t], a, rest[n][0], rest[n][1]);
      }
    }
  };

  // Four outputs of a row from their unnormalised sums.
  auto write_row = [&](int64_t row, int d, const float4& z, float top, float sum) {
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<uint2*>(p.out + row * D + d) =
        make_uint2(T::pack(z.x * inv, z.y * inv), T::pack(z.z * inv, z.w * inv));
    if (d == 0 && p.lse)
      p.lse[row] = sum == 0.0f ? -INFINITY : (top - kLift<T>) * 0.6931471805599453f + logf(sum);
  };
  // Joins the four warps' states and writes the segment's rows: to `out`, or as
  // a partial. Each warp leaves its outputs in the stage that it has just
  // consumed, which nothing refills before the next unit.
  auto slot = [&](int w, int stage) {
    return reinterpret_cast<float*>(smem + (w * kStages + stage) * Smem::kStageBytes);
  };
  // float d of row h; the exclusive or keeps the four heads of a store in different banks
  auto place = [&](int h, int d) { return h * D + (d ^ (((h >> 1) & 3) << 3)); };
  auto end_segment = [&](int stage, bool starts_here, bool ends_here) {
    const int head0 = first_head(at), rows = row_count(at);
    const bool whole = starts_here && ends_here;
    float* part = p.parts + (int64_t(blockIdx.x) * 2 + (starts_here ? 1 : 0)) * kPartFloats<D>;
    const int64_t row0 = int64_t(at.b) * (p.kv_heads * p.group) + head0;
    float* mine = slot(warp, stage);
    __syncwarp();  // every lane has read the stage
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float sum = l[n][c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, x);
        const int h = n * 8 + (lane & 3) * 2 + c;
        if (lane < 4) s_ml[warp][h] = make_float2(m[n][c], sum);
#pragma unroll
        for (int t = 0; t < D / 16; ++t) {
          mine[place(h, t * 16 + (lane >> 2))] = o[n][t][c];
          mine[place(h, t * 16 + 8 + (lane >> 2))] = o[n][t][c + 2];
        }
      }
    }
    __syncthreads();
    for (int i = tid; i < rows * (D / 4); i += kPagedThreads) {
      const int h = i / (D / 4), d = (i - h * (D / 4)) * 4;
      float2 ml[kPagedWarps];
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        ml[w] = s_ml[w][h];
        top = fmaxf(top, ml[w].x);
      }
      float4 z = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
      for (int w = 0; w < kPagedWarps; ++w) {
        const float f = ml[w].y == 0.0f ? 0.0f : ex2(ml[w].x - top);
        const float4 x = *reinterpret_cast<const float4*>(slot(w, stage) + place(h, d));
        sum = fmaf(ml[w].y, f, sum);
        z.x = fmaf(x.x, f, z.x);
        z.y = fmaf(x.y, f, z.y);
        z.z = fmaf(x.z, f, z.z);
        z.w = fmaf(x.w, f, z.w);
      }
      if (whole) {
        write_row(row0 + h, d, z, top, sum);
      } else {
        *reinterpret_cast<float4*>(part + h * D + d) = z;
        if (d == 0) *reinterpret_cast<float2*>(part + kMaxRows * D + h * 2) = make_float2(top, sum);
      }
    }
    __syncthreads();  // the stages may be filled again
    if (whole) return;
    // the last CTA of the segment joins the parts, in their order
    const int first = shares.owner(at.first_place()), last = shares.owner(at.first_place() + at.units - 1);
    if (tid == 0) s_ticket = atom_add_acq_rel_gpu(&p.tickets[first], 1u);
    __syncthreads();
    if (s_ticket != unsigned(last - first)) return;
    if (tid == 0) p.tickets[first] = 0;
    // Parts by the chunk: their (m, l) into a consumed stage, one warp per row for
    // the common maximum and the parts' factors, then the outputs, whose loads
    // wait for nothing but the factors.
    constexpr int kItems = NT * D / 64;                         // float4 outputs of a thread
    constexpr int kParts = 16 / kItems;                         // parts in flight together
    constexpr int kChunk = Smem::kStageBytes / (8 * 8 * NT);    // parts of a chunk
    auto part_of = [&](int c) { return p.parts + (int64_t(c) * 2 + (c == first ? 1 : 0)) * kPartFloats<D>; };
    float2* ml = reinterpret_cast<float2*>(slot(0, stage));
    float4 z[kItems];
    float top[kItems], sum[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) z[k] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), top[k] = -INFINITY, sum[k] = 0.0f;
    for (int c0 = first; c0 <= last; c0 += kChunk) {
      const int n = min(kChunk, last - c0 + 1);
      for (int i = tid; i < n * rows; i += kPagedThreads) {
        const int c = i / rows, h = i - c * rows;
        ml[c * 8 * NT + h] = __ldcg(reinterpret_cast<const float2*>(part_of(c0 + c) + kMaxRows * D + h * 2));
      }
      __syncthreads();
      for (int h = warp; h < rows; h += kPagedWarps) {
        float most = -INFINITY, all = 0.0f;
        for (int c = lane; c < n; c += 32) {
          const float2 x = ml[c * 8 * NT + h];
          if (x.y != 0.0f) most = fmaxf(most, x.x);
        }
        most = warp_max(most);
        for (int c = lane; c < n; c += 32) {
          const float2 x = ml[c * 8 * NT + h];
          const float f = x.y == 0.0f ? 0.0f : ex2(x.x - most);
          all = fmaf(x.y, f, all);
          ml[c * 8 * NT + h].x = f;
        }
        all = warp_sum(all);
        if (lane == 0) s_ml[0][h] = make_float2(most, all);
      }
      __syncthreads();
      float scale[kItems];
      int row[kItems];
#pragma unroll
      for (int k = 0; k < kItems; ++k) {
        row[k] = min((tid + k * kPagedThreads) / (D / 4), rows - 1);
        const float2 chunk = s_ml[0][row[k]];
        const float grown = fmaxf(top[k], chunk.x);
        const float f = sum[k] == 0.0f ? 0.0f : ex2(top[k] - grown);
        scale[k] = chunk.y == 0.0f ? 0.0f : ex2(chunk.x - grown);
        top[k] = grown;
        sum[k] = sum[k] * f + chunk.y * scale[k];
        z[k].x *= f;
        z[k].y *= f;
        z[k].z *= f;
        z[k].w *= f;
      }
      for (int b = 0; b < n; b += kParts) {
        float4 x[kParts][kItems];
#pragma unroll
        for (int c = 0; c < kParts; ++c) {
          const float* from = part_of(c0 + min(b + c, n - 1));
#pragma unroll
          for (int k = 0; k < kItems; ++k)
            x[c][k] = __ldcg(reinterpret_cast<const float4*>(from + row[k] * D + ((tid + k * kPagedThreads) % (D / 4)) * 4));
        }
#pragma unroll
        for (int c = 0; c < kParts; ++c) {
#pragma unroll
          for (int k = 0; k < kItems; ++k) {
            const float g = b + c < n ? ml[(b + c) * 8 * NT + row[k]].x * scale[k] : 0.0f;
            z[k].x = fmaf(x[c][k].x, g, z[k].x);
            z[k].y = fmaf(x[c][k].y, g, z[k].y);
            z[k].z = fmaf(x[c][k].z, g, z[k].z);
            z[k].w = fmaf(x[c][k].w, g, z[k].w);
          }
        }
      }
      __syncthreads();  // the chunk's factors have been read
    }
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const int i = tid + k * kPagedThreads, h = i / (D / 4);
      if (h < rows) write_row(row0 + h, (i - h * (D / 4)) * 4, z[k], top[k], sum[k]);
    }
  };

  load_queries(at);
  clear_state();
  bool starts_here = at.j == 0;
  int stage = 0;
  while (true) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    issue(stage == 0 ? kStages - 1 : stage - 1);
    compute(stage);
    Cursor<Place> following = at;
    following.next(p, heads);
    const bool last_unit = at.j + 1 == at.units, done = following.place >= v1;
    if (last_unit || done) {
      if (!done) load_queries(following);  // in flight while this segment's states are joined
      end_segment(stage, starts_here, last_unit);
      if (done) break;
      clear_state();
      starts_here = true;
    }
    at = following;
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
}

static int paged_grid() { return kPagedCtas * sm_count(); }

template <typename T, int D, int NT, typename Place>
static int run_paged(const char* what, const PagedParams& p, cudaStream_t stream) {
  const auto kernel = paged_attention_kernel<T, D, NT, Place>;
  const int rc = configure_smem(what, kernel, PagedSmem<D>::kBytes);
  if (rc != kOk) return rc;
  return launch(what, kernel, dim3(paged_grid()), dim3(kPagedThreads), PagedSmem<D>::kBytes, stream, p);
}
template <typename T, int D, int NT>
static int run_paged(const char* what, const PagedParams& p, cudaStream_t stream) {
  const int64_t segments = int64_t(p.sequences) * p.kv_heads * p.row_tiles;
  const int64_t longest = (p.capacity + kUnit - 1) / kUnit + 1 + kSegmentCost;
  return segments <= (int64_t(1) << 30) / longest ? run_paged<T, D, NT, int>(what, p, stream)
                                                  : run_paged<T, D, NT, int64_t>(what, p, stream);
}
template <typename T>
static int run_paged(const char* what, const PagedParams& p, int head_dim, int tiles, cudaStream_t stream) {
  if (head_dim == 64) return tiles == 1 ? run_paged<T, 64, 1>(what, p, stream) : run_paged<T, 64, 2>(what, p, stream);
  return tiles == 1 ? run_paged<T, 128, 1>(what, p, stream) : run_paged<T, 128, 2>(what, p, stream);
}

}  // namespace cb

using namespace cb;

extern "C" int64_t cb_paged_attention_workspace_bytes(void) {
  return kTicketBytes + int64_t(paged_grid()) * 2 * kPartFloats<128> * 4;
}

extern "C" int cb_paged_attention(const void* q, int64_t q_token, int64_t q_head, const void* k_pages,
                                  const void* v_pages, int dtype, int sequences, int q_heads, int kv_heads,
                                  int head_dim, int pages, int page_size, const int32_t* table, int64_t table_stride,
                                  int table_width, const int32_t* lengths, float scale, void* out, float* lse,
                                  void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "cb_paged_attention";
  CB_REQUIRE(dtype == CB_BF16 || dtype == CB_FP16, "%s: dtype must be bf16 or fp16", what);
  CB_REQUIRE(sequences >= 0, "%s: sequences=%d", what, sequences);
  CB_REQUIRE(kv_heads >= 1 && q_heads >= kv_heads && q_heads % kv_heads == 0,
             "%s: q_heads=%d must be a multiple of kv_heads=%d", what, q_heads, kv_heads);
  CB_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head_dim=%d (64 or 128)", what, head_dim);
  CB_REQUIRE(pages >= 1 && page_size >= 1 && table_width >= 1 && table_stride >= table_width,
             "%s: pages, page_size and the table's width must be positive", what);
  CB_REQUIRE(int64_t(table_width) * page_size < (int64_t(1) << 31) - kUnit,
             "%s: a table row of %d pages of %d passes 2^31 positions", what, table_width, page_size);
  CB_REQUIRE(int64_t(pages) * kv_heads < (int64_t(1) << 32) / page_size, "%s: the pool has more than 2^32 rows", what);
  if (sequences == 0) return kOk;
  CB_REQUIRE(q && k_pages && v_pages && table && lengths && out && workspace, "%s: null pointer", what);
  CB_REQUIRE(aligned16(q) && aligned16(k_pages) && aligned16(v_pages) && aligned16(out) && aligned16(workspace),
             "%s: q/pages/out/workspace must be 16-byte aligned", what);
  CB_REQUIRE((q_token | q_head) % 8 == 0, "%s: strides must be multiples of 8 elements", what);
  CB_REQUIRE(workspace_bytes >= cb_paged_attention_workspace_bytes(), "%s: the workspace is too small", what);
  CB_REQUIRE(paged_grid() * 4 <= kTicketBytes, "%s: %d CTAs", what, paged_grid());
  PagedParams p = {};
  p.q = static_cast<const uint16_t*>(q);
  p.k = static_cast<const uint16_t*>(k_pages);
  p.v = static_cast<const uint16_t*>(v_pages);
  p.q_token = q_token, p.q_head = q_head, p.table_stride = table_stride;
  p.table = table, p.lengths = lengths;
  p.out = static_cast<uint16_t*>(out), p.lse = lse;
  p.tickets = static_cast<unsigned int*>(workspace);
  p.parts = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + kTicketBytes);
  p.sequences = sequences, p.kv_heads = kv_heads, p.group = q_heads / kv_heads;
  p.pages = pages, p.page_size = page_size, p.capacity = table_width * page_size;
  p.scale_log2 = scale * 1.4426950408889634f;
  while ((int64_t(1) << p.page_shift) < page_size) ++p.page_shift;
  p.page_mul = uint32_t(((uint64_t(1) << (31 + p.page_shift)) + page_size - 1) / page_size);
  p.err = error_word();
  const int tiles = p.group <= 8 ? 1 : 2;
  p.row_tiles = (p.group + 8 * tiles - 1) / (8 * tiles);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return dtype == CB_BF16 ? run_paged<Bf16>(what, p, head_dim, tiles, s) : run_paged<Fp16>(what, p, head_dim, tiles, s);
}
