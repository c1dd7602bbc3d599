// Page bookkeeping of a paged key-value cache on the device: fork, reserve,
// free and compact, without a host round trip.
//
// State: table int32 [sequences, width] (the pages of a sequence in order, -1
// behind them), lengths int32 [sequences], ref int32 [pages] (how many table
// entries name the page; 0: free), storage [outer, pages, page_bytes] (outer =
// layers x {K, V}). Pages are taken lowest index first, in the order of the
// request, so that every result is determined by the state alone.
//
// Two kinds of kernel. A plan kernel is one CTA: it validates, counts the free
// pages and picks them (each warp owns a contiguous range of `ref`: a counting
// pass, one scan over the warps, an assigning pass), all or nothing. An apply
// kernel moves the pages' bytes (HBM-bound: read + write of outer x page_bytes
// per page) and edits table rows; it reads the plan's outcome on the device.
//
// Measured: half of 1024 pages of 2 MB compacted in 183 us = 5.8 TB/s read and
// written (a plain copy: 6.5); a fork of 7 children with their tails 9 us, a free
// 1.1, a reserve 3.0: one chain of loads and a few barriers each.
#include "cascade_b200.h"
#include "internal.h"
#include "paged_device.cuh"

namespace cb {

int32_t* error_word();

constexpr int kPlanThreads = 1024;  // of a plan kernel at most
constexpr int kPlanWarps = kPlanThreads / 32;
constexpr int kSmallPool = 4096;    // pages that 256 threads plan: their barriers take a third of 1024 threads'
constexpr int kPicks = 4096;        // picked pages kept in shared memory
constexpr int kMoveThreads = 256;
constexpr int kMaxPages = 2000000;
constexpr int kMaxForkSlots = 65536;

// Exclusive scan of one value per thread over the CTA; returns the prefix and
// the total. Ends behind a barrier, so `part` can be used again.
__device__ __forceinline__ int block_scan(int v, int* part, int& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) part[warp] = x;
  __syncthreads();
  int w = lane < int(blockDim.x >> 5) ? part[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, w, o);
    if (lane >= o) w += y;
  }
  total = __shfl_sync(0xFFFFFFFFu, w, 31);
  const int before = __shfl_sync(0xFFFFFFFFu, w, warp) - __shfl_sync(0xFFFFFFFFu, x, 31);
  __syncthreads();
  return before + x - v;
}

// Sum of one value per thread over the CTA, for every thread.
__device__ __forceinline__ int64_t block_sum(int64_t v, int64_t* part) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < int(blockDim.x >> 5); ++w) v += part[w];
  return v;
}

// The pages [first, last) that this warp owns.
__device__ __forceinline__ void warp_pages(int pages, int& first, int& last) {
  const int per = ((pages + int(blockDim.x) - 1) / int(blockDim.x)) * 32, warp = threadIdx.x >> 5;
  first = int(min(int64_t(warp) * per, int64_t(pages)));
  last = min(first + per, pages);
}
// How many of the warp's pages this lane sees free.
__device__ __forceinline__ int count_free(const int32_t* ref, int pages) {
  int first, last, mine = 0;
  warp_pages(pages, first, last);
#pragma unroll 8
  for (int i = first + int(threadIdx.x & 31); i < last; i += 32) mine += ref[i] == 0;
  return mine;
}

// Picks the `need` lowest free pages in ascending order, into shared memory or,
// when they are too many, the workspace. `mine` is count_free's answer. Returns how
// many pages are free (nothing is picked when they are fewer than need).
struct Picks {
  int near[kPicks];
  int32_t* far;
  int need;
  __device__ __forceinline__ int& at(int i) { return need <= kPicks ? near[i] : far[i]; }
};
__device__ __forceinline__ int pick_free(const int32_t* ref, int pages, int need, int mine, Picks& picks,
                                         int32_t* workspace, int* part) {
  const int lane = threadIdx.x & 31;
  int first, last, free;
  warp_pages(pages, first, last);
  int rank = block_scan(mine, part, free);
  rank = __shfl_sync(0xFFFFFFFFu, rank, 0);  // free pages before this warp's range
  if (threadIdx.x == 0) picks.far = workspace, picks.need = need;
  __syncthreads();
  if (free >= need) {
    for (int i = first; i < last && rank < need; i += 32) {
      const bool open = i + lane < last && ref[i + lane] == 0;
      const unsigned mask = __ballot_sync(0xFFFFFFFFu, open);
      const int place = rank + __popc(mask & ((1u << lane) - 1u));
      if (open && place < need) picks.at(place) = i + lane;
      rank += __popc(mask);
    }
  }
  __syncthreads();
  return free;
}

__device__ __forceinline__ int page_count(int64_t length, int page_size) {
  return int((length + page_size - 1) / page_size);
}

// ------------------------------------------------------------------ free
// One CTA per entry. Taking the length with an exchange makes a slot that is
// listed twice (or empty) a no-op the second time.
__global__ void __launch_bounds__(kMoveThreads) pages_free_kernel(const int32_t* slots, int sequences, int width,
                                                                 int32_t* table, int32_t* lengths, int32_t* ref,
                                                                 int pages, int* err) {
  __shared__ int held;
  grid_dep_wait();
  const int slot = slots[blockIdx.x];
  if (slot < 0 || slot >= sequences) {
    if (threadIdx.x == 0 && err) atomicExch(err, kErrPagesSlot);
    return;
  }
  if (threadIdx.x == 0) held = atomicExch(&lengths[slot], 0);
  __syncthreads();
  if (held == 0) return;
  int32_t* row = table + int64_t(slot) * width;
  for (int j = threadIdx.x; j < width; j += kMoveThreads) {
    const int page = row[j];
    if (page < 0) continue;
    row[j] = -1;
    bool held_page = page < pages;
    if (held_page && atomicSub(&ref[page], 1) <= 0) {
      atomicAdd(&ref[page], 1);
      held_page = false;
    }
    if (!held_page && err) atomicExch(err, kErrPagesRef);
  }
}

// ------------------------------------------------------------------ fork
struct ForkParams {
  const int32_t *parents, *children;
  int n, sequences, width, pages, page_size;
  int32_t *table, *lengths, *ref, *status, *workspace;
  uint8_t* storage;
  int64_t outer, page_bytes;
  int* err;
};

__global__ void __launch_bounds__(kPlanThreads) pages_fork_plan_kernel(const __grid_constant__ ForkParams p) {
  __shared__ int part[kPlanWarps];
  __shared__ Picks picks;
  __shared__ unsigned int listed[kMaxForkSlots / 32];  // the children, a bit each
  __shared__ int bad;
  grid_dep_wait();
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) bad = 0;
  for (int i = tid; i < (p.sequences + 31) / 32; i += threads) listed[i] = 0;
  const int open = count_free(p.ref, p.pages);
  __syncthreads();
  bool wrong = false;
  for (int i = tid; i < p.n; i += threads) {
    const int parent = p.parents[i], child = p.children[i];
    if (parent < 0 || parent >= p.sequences || child < 0 || child >= p.sequences ||
        (atomicOr(&listed[child >> 5], 1u << (child & 31)) >> (child & 31) & 1u) || p.lengths[child] != 0)
      wrong = true;
  }
  if (wrong) bad = 1;
  __syncthreads();
  int tails = 0;
  for (int base = 0; base < p.n; base += threads) {
    const int i = base + tid;
    int tail = 0;
    if (i < p.n && !bad) {
      const int parent = p.parents[i], length = p.lengths[parent];
      if ((listed[parent >> 5] >> (parent & 31) & 1u) || length < 0 || page_count(length, p.page_size) > p.width)
        wrong = true;
      tail = length > 0 && length % p.page_size != 0;
    }
    int total;
    block_scan(tail, part, total);
    tails += total;
  }
  if (wrong) bad = 1;
  __syncthreads();
  const bool stop = bad != 0;
  const int free = pick_free(p.ref, p.pages, stop ? 0 : tails, open, picks, p.workspace, part);
  if (stop || free < tails) {
    if (tid == 0) p.status[0] = stop ? -1 : tails - free;
    return;
  }
  int before = 0;
  for (int base = 0; base < p.n; base += threads) {
    const int i = base + tid;
    int length = 0, tail = 0, source = 0, total;
    if (i < p.n) {
      const int parent = p.parents[i];
      length = p.lengths[parent];
      tail = length % p.page_size != 0;
      if (tail) source = p.table[int64_t(parent) * p.width + length / p.page_size];
    }
    const int rank = before + block_scan(tail, part, total);
    before += total;
    if (i < p.n) {
      const int child = p.children[i];
      p.lengths[child] = length;
      if (tail) {
        const int page = picks.at(rank);
        p.workspace[rank] = page;
        p.workspace[p.pages + rank] = source;
        p.table[int64_t(child) * p.width + length / p.page_size] = page;
        p.ref[page] = 1;
      }
    }
  }
  if (tid == 0) {
    p.status[0] = 0;
    p.workspace[2 * int64_t(p.pages)] = tails;
  }
}

// Eight 16-byte vectors of a thread in flight.
__device__ __forceinline__ void copy_bytes(uint8_t* dst, const uint8_t* src, int64_t bytes) {
  constexpr int kBatch = 8, kStep = kMoveThreads * 16;
  for (int64_t at = int64_t(threadIdx.x) * 16; at < bytes; at += kBatch * kStep) {
    uint4 x[kBatch];
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (at + k * kStep < bytes) x[k] = __ldcs(reinterpret_cast<const uint4*>(src + at + k * kStep));
#pragma unroll
    for (int k = 0; k < kBatch; ++k)
      if (at + k * kStep < bytes) __stcs(reinterpret_cast<uint4*>(dst + at + k * kStep), x[k]);
  }
}

// The first n CTAs write a child's table row and count the shares each; the
// others copy one block of a tail page, of which the plan left target and source
// at workspace[rank] and workspace[pages + rank] and the number behind them.
__global__ void __launch_bounds__(kMoveThreads) pages_fork_apply_kernel(const __grid_constant__ ForkParams p) {
  grid_dep_wait();
  if (int(blockIdx.x) < p.n) {
    if (p.status[0] != 0) return;
    const int parent = p.parents[blockIdx.x], child = p.children[blockIdx.x];
    const int full = p.lengths[parent] / p.page_size;
    const int32_t* from = p.table + int64_t(parent) * p.width;
    int32_t* to = p.table + int64_t(child) * p.width;
    for (int j = threadIdx.x; j < full; j += kMoveThreads) {
      const int page = from[j];
      to[j] = page;
      if (page >= 0 && page < p.pages)
        atomicAdd(&p.ref[page], 1);
      else if (p.err)
        atomicExch(p.err, kErrPagesRef);
    }
    return;
  }
  const int64_t item = int64_t(blockIdx.x) - p.n, rank = item / p.outer, o = item - rank * p.outer;
  if (rank >= p.pages) return;
  // four loads that do not wait for one another
  const int status = p.status[0], tails = p.workspace[2 * int64_t(p.pages)];
  const int dst = p.workspace[rank], src = p.workspace[p.pages + rank];
  if (status != 0 || rank >= tails) return;
  if (src < 0 || src >= p.pages) {
    if (threadIdx.x == 0 && p.err) atomicExch(p.err, kErrPagesRef);
    return;
  }
  uint8_t* base = p.storage + o * p.pages * p.page_bytes;
  copy_bytes(base + dst * p.page_bytes, base + src * p.page_bytes, p.page_bytes);
}

// --------------------------------------------------------------- reserve
struct ReserveParams {
  const int32_t* extra;
  int sequences, width, pages, page_size;
  int32_t *table, *lengths, *ref, *status, *workspace;
};

__global__ void __launch_bounds__(kPlanThreads) pages_reserve_kernel(const __grid_constant__ ReserveParams p) {
  __shared__ int part[kPlanWarps];
  __shared__ int64_t sums[kPlanWarps];
  __shared__ int first[kPlanThreads], held[kPlanThreads], want[kPlanThreads];
  __shared__ Picks picks;
  __shared__ int bad;
  grid_dep_wait();
  const int tid = threadIdx.x, threads = blockDim.x;
  if (tid == 0) bad = 0;
  const int open = count_free(p.ref, p.pages);
  __syncthreads();
  int64_t need = 0;
  bool wrong = false;
  for (int s = tid; s < p.sequences; s += threads) {
    const int64_t length = p.lengths[s], grown = length + p.extra[s];
    if (length < 0 || p.extra[s] < 0 || grown > int64_t(p.width) * p.page_size)
      wrong = true;
    else
      need += page_count(grown, p.page_size) - page_count(length, p.page_size);
  }
  need = block_sum(need, sums);
  if (wrong) bad = 1;
  __syncthreads();
  const bool stop = bad != 0;
  // (more than all pages can never be picked: the exact need is only told)
  const int wanted = int(min(need, int64_t(p.pages) + 1));
  const int free = pick_free(p.ref, p.pages, stop ? 0 : wanted, open, picks, p.workspace, part);
  if (stop || free < wanted) {
    if (tid == 0) p.status[0] = stop ? -1 : int(min(need - free, int64_t(INT32_MAX)));
    return;
  }
  int before = 0;
  for (int base = 0; base < p.sequences; base += threads) {
    const int s = base + tid;
    int more = 0, old = 0, total;
    if (s < p.sequences) {
      const int length = p.lengths[s], grown = length + p.extra[s];
      old = page_count(length, p.page_size);
      more = page_count(grown, p.page_size) - old;
      p.lengths[s] = grown;
    }
    first[tid] = before + block_scan(more, part, total);
    held[tid] = old;
    want[tid] = more;
    before += total;
    __syncthreads();
    const int count = min(threads, p.sequences - base);
    for (int r = tid >> 5; r < count; r += threads >> 5) {
      int32_t* row = p.table + int64_t(base + r) * p.width + held[r];
      for (int j = tid & 31; j < want[r]; j += 32) {
        const int page = picks.at(first[r] + j);
        row[j] = page;
        p.ref[page] = 1;
      }
    }
    __syncthreads();
  }
  if (tid == 0) p.status[0] = 0;
}

// --------------------------------------------------------------- compact
struct CompactParams {
  const int32_t *table, *ref;
  int sequences, width, pages;
  int32_t *table_out, *ref_out, *live, *workspace;
  uint8_t* storage;
  int64_t outer, page_bytes;
  int* err;
};

// workspace: [0] the moves' count, then their sources, targets (half of the
// pages each) and the new index of every page beyond the dense prefix.
__device__ __forceinline__ int32_t* move_source(const CompactParams& p) { return p.workspace + 2; }
__device__ __forceinline__ int32_t* move_target(const CompactParams& p) {
  return p.workspace + 2 + (p.pages + 1) / 2;
}
__device__ __forceinline__ int32_t* move_index(const CompactParams& p) {
  return p.workspace + 2 + 2 * ((p.pages + 1) / 2);
}

__global__ void __launch_bounds__(kPlanThreads) pages_compact_plan_kernel(const __grid_constant__ CompactParams p) {
  __shared__ int part[kPlanWarps];
  __shared__ int2 pairs[kPicks / 2];  // (source, target)
  grid_dep_wait();
  const int tid = threadIdx.x, lane = tid & 31, threads = blockDim.x;
  int first, last, free, moves;
  warp_pages(p.pages, first, last);
  block_scan(count_free(p.ref, p.pages), part, free);
  const int live = p.pages - free;
  // holes below `live` and live pages from it on: as many of one as of the other
  int holes = 0, movers = 0;
  for (int i = first + lane; i < last; i += 32) {
    const bool used = p.ref[i] != 0;
    holes += i < live && !used;
    movers += i >= live && used;
  }
  int hole = __shfl_sync(0xFFFFFFFFu, block_scan(holes, part, moves), 0);
  int mover = __shfl_sync(0xFFFFFFFFu, block_scan(movers, part, moves), 0);
  const bool near = moves <= kPicks / 2;  // the lists are read again here: from shared memory if they fit
  int32_t *source = move_source(p), *target = move_target(p), *index = move_index(p);
  for (int i = first; i < last; i += 32) {
    const int page = i + lane;
    const bool in = page < last, used = in && p.ref[page] != 0;
    const bool is_hole = in && !used && page < live, is_mover = used && page >= live;
    const unsigned below = (1u << lane) - 1u;
    const unsigned h = __ballot_sync(0xFFFFFFFFu, is_hole), m = __ballot_sync(0xFFFFFFFFu, is_mover);
    if (is_hole) {
      const int j = hole + __popc(h & below);
      target[j] = page;
      if (near) pairs[j].y = page;
    }
    if (is_mover) {
      const int j = mover + __popc(m & below);
      source[j] = page;
      if (near) pairs[j].x = page;
    }
    hole += __popc(h);
    mover += __popc(m);
  }
  __syncthreads();
  for (int j = tid; j < moves; j += threads) {
    const int2 move = near ? pairs[j] : make_int2(source[j], target[j]);
    index[move.x] = move.y;
    p.ref_out[move.y] = p.ref[move.x];  // targets are free: nobody reads their count any more
  }
  __syncthreads();
  for (int i = tid; i < p.pages; i += threads) {
    const int r = p.ref[i];
    if (i >= live) {
      if (r == 0) index[i] = -1;
      p.ref_out[i] = 0;
    } else if (r != 0) {
      p.ref_out[i] = r;
    }
  }
  if (tid == 0) {
    p.workspace[0] = moves;
    p.live[0] = live;
  }
}

__global__ void __launch_bounds__(kMoveThreads) pages_compact_apply_kernel(const __grid_constant__ CompactParams p) {
  grid_dep_wait();
  const int64_t moves = p.workspace[0], items = moves * p.outer;
  const int live = p.live[0];
  const int32_t *source = move_source(p), *target = move_target(p), *index = move_index(p);
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t o = it / moves, j = it - o * moves;
    uint8_t* base = p.storage + o * p.pages * p.page_bytes;
    copy_bytes(base + target[j] * p.page_bytes, base + source[j] * p.page_bytes, p.page_bytes);
  }
  const int64_t entries = int64_t(p.sequences) * p.width;
  for (int64_t e = int64_t(blockIdx.x) * kMoveThreads + threadIdx.x; e < entries; e += int64_t(gridDim.x) * kMoveThreads) {
    int page = p.table[e];
    if (page >= p.pages) {
      if (p.err) atomicExch(p.err, kErrPagesRef);
      page = -1;
    } else if (page >= live) {
      page = index[page];
      if (page < 0 && p.err) atomicExch(p.err, kErrPagesRef);
    } else if (page < 0) {
      page = -1;
    }
    p.table_out[e] = page;
  }
}

}  // namespace cb

using namespace cb;

static int plan_threads(int pages, int requests) {
  return pages <= kSmallPool && requests <= 256 ? 256 : kPlanThreads;
}
static int check_state(const char* what, const void* table, int sequences, int width, const void* ref, int pages) {
  CB_REQUIRE(sequences >= 1 && width >= 1 && pages >= 1, "%s: sequences, table width and pages must be positive", what);
  // the plan kernels' 32-bit scans add up to 1024 counts of at most pages
  CB_REQUIRE(pages <= kMaxPages, "%s: pages=%d (at most %d)", what, pages, kMaxPages);
  CB_REQUIRE(table && ref, "%s: null pointer", what);
  return kOk;
}
static int check_storage(const char* what, const void* storage, int64_t outer, int64_t page_bytes) {
  CB_REQUIRE(storage && aligned16(storage), "%s: storage must be a 16-byte aligned device pointer", what);
  CB_REQUIRE(outer >= 1 && outer < (1 << 20), "%s: outer=%lld", what, (long long)outer);
  CB_REQUIRE(page_bytes >= 16 && page_bytes % 16 == 0, "%s: page_bytes=%lld must be a multiple of 16", what,
             (long long)page_bytes);
  return kOk;
}

extern "C" int64_t cb_pages_workspace_ints(int pages) { return pages < 1 ? 0 : 2 * int64_t(pages) + 64; }

extern "C" int cb_pages_free(const int32_t* slots, int n, int32_t* table, int sequences, int width, int32_t* lengths,
                             int32_t* ref, int pages, void* stream) {
  const char* what = "cb_pages_free";
  CB_REQUIRE(n >= 0, "%s: n=%d", what, n);
  if (n == 0) return kOk;
  int rc = check_state(what, table, sequences, width, ref, pages);
  if (rc != kOk) return rc;
  CB_REQUIRE(slots && lengths, "%s: null pointer", what);
  return launch(what, pages_free_kernel, dim3(n), dim3(kMoveThreads), 0, static_cast<cudaStream_t>(stream), slots,
                sequences, width, table, lengths, ref, pages, reinterpret_cast<int*>(error_word()));
}

extern "C" int cb_pages_fork(const int32_t* parents, const int32_t* children, int n, int32_t* table, int sequences,
                             int width, int32_t* lengths, int32_t* ref, int pages, int page_size, void* storage,
                             int64_t outer, int64_t page_bytes, int32_t* status, int32_t* workspace, void* stream) {
  const char* what = "cb_pages_fork";
  int rc = check_state(what, table, sequences, width, ref, pages);
  if (rc == kOk) rc = check_storage(what, storage, outer, page_bytes);
  if (rc != kOk) return rc;
  CB_REQUIRE(sequences <= kMaxForkSlots, "%s: sequences=%d (at most %d)", what, sequences, kMaxForkSlots);
  CB_REQUIRE(n >= 0 && int64_t(n) * (outer + 1) < (int64_t(1) << 31), "%s: n=%d x outer=%lld", what, n, (long long)outer);
  CB_REQUIRE(page_size >= 1, "%s: page_size=%d", what, page_size);
  CB_REQUIRE(lengths && status && workspace && (n == 0 || (parents && children)), "%s: null pointer", what);
  ForkParams p = {parents, children, n,      sequences, width,     pages,
                  page_size, table,  lengths, ref,      status,    workspace,
                  static_cast<uint8_t*>(storage), outer, page_bytes, error_word()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch(what, pages_fork_plan_kernel, dim3(1), dim3(plan_threads(pages, n)), 0, s, p);
  if (rc != kOk || n == 0) return rc;
  return launch(what, pages_fork_apply_kernel, dim3(unsigned(n * (outer + 1))), dim3(kMoveThreads), 0, s, p);
}

extern "C" int cb_pages_reserve(const int32_t* extra, int32_t* table, int sequences, int width, int32_t* lengths,
                                int32_t* ref, int pages, int page_size, int32_t* status, int32_t* workspace,
                                void* stream) {
  const char* what = "cb_pages_reserve";
  int rc = check_state(what, table, sequences, width, ref, pages);
  if (rc != kOk) return rc;
  CB_REQUIRE(page_size >= 1 && int64_t(width) * page_size < (int64_t(1) << 31), "%s: page_size=%d", what, page_size);
  CB_REQUIRE(extra && lengths && status && workspace, "%s: null pointer", what);
  ReserveParams p = {extra, sequences, width, pages, page_size, table, lengths, ref, status, workspace};
  return launch(what, pages_reserve_kernel, dim3(1), dim3(plan_threads(pages, sequences)), 0, static_cast<cudaStream_t>(stream), p);
}

extern "C" int cb_pages_compact(const int32_t* table, int sequences, int width, const int32_t* ref, int pages,
                                void* storage, int64_t outer, int64_t page_bytes, int32_t* table_out,
                                int32_t* ref_out, int32_t* live, int32_t* workspace, void* stream) {
  const char* what = "cb_pages_compact";
  int rc = check_state(what, table, sequences, width, ref, pages);
  if (rc == kOk) rc = check_storage(what, storage, outer, page_bytes);
  if (rc != kOk) return rc;
  CB_REQUIRE(table_out && ref_out && live && workspace, "%s: null pointer", what);
  CompactParams p = {table,     ref,     sequences, width,     pages, table_out,
                     ref_out,   live,    workspace, static_cast<uint8_t*>(storage), outer, page_bytes, error_word()};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  rc = launch(what, pages_compact_plan_kernel, dim3(1), dim3(plan_threads(pages, 0)), 0, s, p);
  if (rc != kOk) return rc;
  return launch(what, pages_compact_apply_kernel, dim3(8 * sm_count()), dim3(kMoveThreads), 0, s, p);
}
