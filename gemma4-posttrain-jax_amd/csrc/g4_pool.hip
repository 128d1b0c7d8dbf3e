// Pages of a pool taken, shared, copied, given back and moved together: g4_paged_reserve, g4_paged_fork, g4_paged_copy,
// g4_paged_free, g4_paged_compact. No reference counterpart (its caches are dense arrays). refs[p] counts the table
// entries that hold page p; a page is free where it is 0 or below. Everything is on the device and ordered by
// the stream, so a captured step can take and give back pages.
//
// Which fresh page goes to which entry is fixed: the i-th entry that wants one, row by row, gets the i-th lowest free
// page. A first launch turns refs into a bitmap of free pages with a count per group of 256 and counts what each
// row wants; in the second each workgroup sums the counts before its own (they are few: 4096 groups are a million
// pages), and each entry finds its page by its rank: a binary search among the groups in LDS, then bits.
#include <type_traits>

#include "g4_paged.h"

namespace g4 {
namespace {

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr int kGroup = 256;       // pages per count: four words of the bitmap
constexpr int kSpans = 4096;      // counts held in LDS; beyond a million pages one for several groups

struct PoolWorkspace {
  uint64_t* bits;   // [groups * 4] free pages
  int32_t* counts;  // [groups]
  int32_t* wants;   // [rows]
  int32_t* src;     // [pairs] pages to copy from, to (-1: none), and how many slots
  int32_t* dst;
  int32_t* slots;
  int32_t* map;     // [pages] where a page went
  int32_t* moved;   // [1]
};

__host__ __device__ inline int64_t groups_of(int32_t pages) { return ((int64_t)pages + kGroup - 1) / kGroup; }

// Carves the workspace; returns its bytes.
size_t carve(PoolWorkspace& w, void* base, int32_t pages, int64_t rows, int64_t pairs, bool map) {
  const int64_t g = groups_of(pages);
  size_t at = 0;
  const auto take = [&](int64_t bytes) {
    void* p = base ? static_cast<char*>(base) + at : nullptr;
    at += ((size_t)bytes + 15) / 16 * 16;
    return p;
  };
  w.bits = static_cast<uint64_t*>(take(g * 32));
  w.counts = static_cast<int32_t*>(take(g * 4));
  w.wants = static_cast<int32_t*>(take(rows * 4));
  w.src = static_cast<int32_t*>(take(pairs * 4));
  w.dst = static_cast<int32_t*>(take(pairs * 4));
  w.slots = static_cast<int32_t*>(take(map ? 0 : pairs * 4));
  w.map = static_cast<int32_t*>(take(map ? (int64_t)pages * 4 : 0));
  w.moved = static_cast<int32_t*>(take(map ? 4 : 0));
  return at;
}

// --- what a row wants ----------------------------------------------------------------------------------------

struct Reserve {
  G4PageTable table;
  const int32_t* lengths;
  int32_t num_pages, page_size;

  __device__ __forceinline__ bool page(int32_t p) const { return (uint32_t)p < (uint32_t)num_pages; }
  __device__ __forceinline__ int rows() const { return table.rows; }
  __device__ __forceinline__ int width() const { return table.max_pages; }
  struct Row {
    int32_t* entries;
    int upto;  // entries below that get a page
  };
  __device__ __forceinline__ Row row(int b) const {
    const int n = lengths[b], ps = __builtin_ctz(page_size);
    const int upto = n <= 0 ? 0 : (int)(((uint32_t)n + page_size - 1u) >> ps);
    return Row{table.entries + b * table.stride, min(upto, table.max_pages)};
  }
  __device__ __forceinline__ bool wants(const Row& r, int e) const { return e < r.upto && !page(r.entries[e]); }
  __device__ __forceinline__ int last(const Row& r) const { return r.upto; }  // no entry from there on is looked at
  __device__ __forceinline__ void settle(const Row& r, int, int e, bool wanted, int32_t fresh, int32_t* refs) const {
    if (!wanted || fresh < 0) return;
    r.entries[e] = fresh;
    refs[fresh] = 1;
  }
};

struct Fork {
  G4PageTable table, out;
  const int32_t* parents;
  const int32_t* lengths;
  int32_t num_pages, page_size;
  int32_t *src, *dst, *slots;

  __device__ __forceinline__ bool page(int32_t p) const { return (uint32_t)p < (uint32_t)num_pages; }
  __device__ __forceinline__ int rows() const { return out.rows; }
  struct Row {
    const int32_t* from;
    int32_t* to;
    int whole, rest;  // pages that are shared, slots of the one that is copied
  };
  __device__ __forceinline__ Row row(int i) const {
    Row r{nullptr, out.entries + i * out.stride, 0, 0};
    const int a = parents[i];
    if ((uint32_t)a >= (uint32_t)table.rows) return r;
    r.from = table.entries + a * table.stride;
    const int n = min(max(lengths[a], 0), min(table.max_pages, out.max_pages) * page_size);
    r.whole = n >> __builtin_ctz(page_size);
    r.rest = n & (page_size - 1);
    return r;
  }
  __device__ __forceinline__ bool wants(const Row& r, int e) const { return r.rest > 0 && e == r.whole && page(r.from[e]); }
  __device__ __forceinline__ int last(const Row&) const { return out.max_pages; }
  __device__ __forceinline__ void settle(const Row& r, int i, int e, bool wanted, int32_t fresh, int32_t* refs) const {
    int32_t entry = -1;
    if (e < r.whole) {
      entry = r.from[e];
      if (page(entry)) atomicAdd(refs + entry, 1);
      else entry = -1;
    } else if (wanted && fresh >= 0) {
      entry = fresh;
      refs[fresh] = 1;
    }
    r.to[e] = entry;
    if (e == min(r.whole, out.max_pages - 1)) {  // the row's one pair
      const bool copy = e == r.whole && entry >= 0;
      src[i] = copy ? r.from[e] : -1;
      dst[i] = copy ? entry : -1;
      slots[i] = r.rest;
    }
  }
};

// --- the free pages ------------------------------------------------------------------------------------------

// The bitmap and count of one group of 256 pages by one wave.
__device__ __forceinline__ void scan_group(const int32_t* refs, int32_t pages, int64_t g, const PoolWorkspace& w, int lane) {
  int32_t v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t p = g * kGroup + i * 64 + lane;
    v[i] = p < pages ? refs[p] : 1;
  }
  int count = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint64_t free = __ballot(v[i] <= 0);
    count += __popcll(free);
    if (lane == 0) w.bits[g * 4 + i] = free;
  }
  if (lane == 0) w.counts[g] = count;
}

// What row b wants, by one wave.
template <typename Op>
__device__ __forceinline__ void count_wants(const Op& op, int b, const PoolWorkspace& w, int lane) {
  const auto row = op.row(b);
  int n = 0;
  for (int e0 = 0; e0 < op.last(row); e0 += 64)
    n += __popcll(__ballot(e0 + lane < op.last(row) && op.wants(row, e0 + lane)));
  if (lane == 0) w.wants[b] = n;
}

// Groups of pages in the first `group_blocks` workgroups, rows in the others; a wave each.
template <typename Op>
__global__ __launch_bounds__(kThreads) void scan_kernel(Op op, const int32_t* refs, int32_t pages, PoolWorkspace w,
                                                        int group_blocks) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x < group_blocks) {
    const int64_t g = (int64_t)blockIdx.x * kWaves + wave;
    if (g * kGroup < pages) scan_group(refs, pages, g, w, lane);
    return;
  }
  if constexpr (!std::is_same_v<Op, int>) {
    const int b = ((int)blockIdx.x - group_blocks) * kWaves + wave;
    if (b < op.rows()) count_wants(op, b, w, lane);
  }
}

// The free pages by rank, in LDS per workgroup of THREADS.
template <int THREADS>
struct FreePages {
  int32_t before[kSpans + 1];  // free pages below a span's first
  int32_t partial[2][THREADS / 64];
  int spans, per;              // groups per span

  // The sum of v over the threads below this one; `total` over all. (The caller's next use of `partial` is behind a barrier.)
  __device__ __forceinline__ int exclusive(int v, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(x, d, 64);
      x += lane >= d ? y : 0;
    }
    if (lane == 63) partial[0][wave] = x;
    __syncthreads();
    int below = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) {
      below += i < wave ? partial[0][i] : 0;
      total += partial[0][i];
    }
    __syncthreads();
    return below + x - v;
  }
  // Over all threads.
  __device__ __forceinline__ void sums(int& u, int& v) {
#pragma unroll
    for (int d = 32; d; d >>= 1) u += __shfl_xor(u, d, 64), v += __shfl_xor(v, d, 64);
    if ((threadIdx.x & 63) == 0) partial[0][threadIdx.x >> 6] = u, partial[1][threadIdx.x >> 6] = v;
    __syncthreads();
    u = v = 0;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) u += partial[0][i], v += partial[1][i];
    __syncthreads();
  }

  __device__ __forceinline__ void load(const PoolWorkspace& w, int64_t groups) {
    per = (int)((groups + kSpans - 1) / kSpans);  // (the same in every thread)
    spans = (int)((groups + per - 1) / per);
    const int each = (spans + THREADS - 1) / THREADS;
    const int from = min((int)threadIdx.x * each, spans), to = min(from + each, spans);
    int sum = 0;
    for (int s = from; s < to; ++s) {
      int n = 0;
      for (int64_t g = (int64_t)s * per; g < min((int64_t)(s + 1) * per, groups); ++g) n += w.counts[g];
      before[s] = n;
      sum += n;
    }
    int total;
    int at = exclusive(sum, total);
    for (int s = from; s < to; ++s) {
      const int n = before[s];
      before[s] = at;
      at += n;
    }
    if (threadIdx.x == 0) before[spans] = total;
    __syncthreads();
  }
  __device__ __forceinline__ int total() const { return before[spans]; }

  // the page of a rank in [0, total())
  __device__ __forceinline__ int32_t select(const PoolWorkspace& w, int rank) const {
    int lo = 0, hi = spans;  // before[lo] <= rank < before[hi]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (before[mid] <= rank) lo = mid;
      else hi = mid;
    }
    rank -= before[lo];
    int64_t g = (int64_t)lo * per;
    for (int n; per > 1 && rank >= (n = w.counts[g]); ++g) rank -= n;
    uint64_t word[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) word[i] = w.bits[g * 4 + i];
    int i = 0;
#pragma unroll
    for (int j = 0; j < 3; ++j) {
      const int n = __popcll(word[j]);
      if (i == j && rank >= n) rank -= n, i = j + 1;
    }
    uint64_t x = i == 0 ? word[0] : i == 1 ? word[1] : i == 2 ? word[2] : word[3];
    int at = 0;
#pragma unroll
    for (int half = 32; half; half >>= 1) {
      const int n = __popcll(x & ((1ull << half) - 1));
      if (rank >= n) rank -= n, x >>= half, at += half;
    }
    return (int32_t)(g * kGroup + i * 64 + at);
  }

  // free pages below p, 0 <= p <= pages
  __device__ __forceinline__ int rank(const PoolWorkspace& w, int64_t groups, int64_t p) const {
    const int64_t g = p / kGroup;
    if (g >= groups) return total();
    int n = before[g / per];
    for (int64_t i = g / per * per; i < g; ++i) n += w.counts[i];
    const int word = (int)(p % kGroup) >> 6;
    for (int i = 0; i < word; ++i) n += __popcll(w.bits[g * 4 + i]);
    return n + __popcll(w.bits[g * 4 + word] & ((1ull << (p & 63)) - 1));
  }
};

// The fresh pages of rows row0 .. row0 + per - 1, per <= THREADS. shortage (of all rows): how many entries got none.
template <int THREADS, typename Op>
__device__ __forceinline__ void assign_rows(const Op& op, int32_t* refs, int32_t pages, const PoolWorkspace& w, int row0, int per,
                                            int32_t* shortage) {
  __shared__ FreePages<THREADS> free;
  __shared__ int32_t base[THREADS];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, rows = op.rows();
  int before = 0, all = 0;
  for (int i = threadIdx.x; i < (row0 == 0 ? rows : row0); i += THREADS) {
    const int n = w.wants[i];
    before += i < row0 ? n : 0;
    all += n;
  }
  const int mine = row0 + (int)threadIdx.x;
  const int wanted_here = (int)threadIdx.x < per && mine < rows ? w.wants[mine] : 0;
  free.load(w, groups_of(pages));
  free.sums(before, all);
  if (row0 == 0 && threadIdx.x == 0) *shortage = max(0, all - free.total());
  int total;
  base[threadIdx.x] = before + free.exclusive(wanted_here, total);
  __syncthreads();
  for (int i = wave; i < per && row0 + i < rows; i += THREADS / 64) {
    const auto row = op.row(row0 + i);
    int rank = base[i];
    for (int e0 = 0; e0 < op.last(row); e0 += 64) {
      const int e = e0 + lane;
      const bool wanted = e < op.last(row) && op.wants(row, e);
      const uint64_t who = __ballot(wanted);
      const int mine_rank = rank + __popcll(who & ((1ull << lane) - 1));
      const int32_t fresh = wanted && mine_rank < free.total() ? free.select(w, mine_rank) : -1;
      if (e < op.last(row)) op.settle(row, row0 + i, e, wanted, fresh, refs);
      rank += __popcll(who);
    }
  }
}

template <typename Op>
__global__ __launch_bounds__(kThreads) void assign_kernel(Op op, int32_t* refs, int32_t pages, PoolWorkspace w, int per,
                                                          int32_t* shortage) {
  assign_rows<kThreads>(op, refs, pages, w, blockIdx.x * per, per, shortage);
}

// Both launches in one, of one workgroup, whose waves take the groups and the rows in turns and keep what the launches hand over
// in LDS: for few rows of a small pool. (One prompt of 701 positions to 4 rows in a pool of 77 pages, fork, free and reserve
// replayed from a graph: 25.9 -> 21.0 us. 64 rows are four turns of 16 waves, and the two launches as fast.)
constexpr int kFewRows = 32, kFewPages = 16384, kFewThreads = 1024;
template <typename Op>
__global__ __launch_bounds__(kFewThreads) void few_kernel(Op op, int32_t* refs, int32_t pages, int32_t* shortage) {
  __shared__ uint64_t bits[kFewPages / 64];
  __shared__ int32_t counts[kFewPages / kGroup], wants[kFewRows];
  PoolWorkspace w = {};
  w.bits = bits, w.counts = counts, w.wants = wants;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int b = wave; b < op.rows(); b += kFewThreads / 64) count_wants(op, b, w, lane);
  for (int g = wave; g < groups_of(pages); g += kFewThreads / 64) scan_group(refs, pages, g, w, lane);
  __syncthreads();
  assign_rows<kFewThreads>(op, refs, pages, w, 0, op.rows(), shortage);
}

// --- copies ----------------------------------------------------------------------------------------------------

constexpr int kMaxLayers = 32;      // per launch (they ride in the kernel's arguments)
constexpr int kUnitBytes = 16384;   // of keys or values that a workgroup copies at a time (8 KiB 86, 16 and 32 KiB 67 us below)

struct Layer {
  uint8_t* data[2];   // key, value
  uint8_t* scale[2];  // NULL in bf16
  int32_t heads, chunk_bytes;  // of 32 slots of one head
  int32_t per, units;          // chunks per unit, units per page and array
};
struct Copies {
  Layer layers[kMaxLayers];
  int32_t n_layers, num_pages, chunks;  // 32-slot chunks per page and head
};

// Where entries of a table go: nothing where map is NULL.
struct Remap {
  G4PageTable table;
  const int32_t* map;
};

// Pairs of pages (their number on the device where `moved` is given) in every layer: a workgroup per layer and array (which
// change fastest), pair and unit of `per` chunks, or several units one after the other. Of a page those chunks that
// hold its first slots[i] slots, or all. Bound by HBM: 576 e4m3 pages of 32 KiB from 144, 8 layers, in 67 us (5.7 TB/s; a plain copy
// of as many bytes 5.7, with non-temporal loads 6.4, which here lose what the sources' readers share: 108 us). With the layers
// slowest instead of fastest 87 us.
__global__ __launch_bounds__(kThreads) void copy_kernel(Copies c, const int32_t* src, const int32_t* dst, const int32_t* slots,
                                                        int pairs, const int32_t* moved, Remap remap) {
  if (moved) pairs = *moved;
  if (remap.map) {
    const G4PageTable& t = remap.table;
    for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (int64_t)t.rows * t.max_pages;
         i += (int64_t)gridDim.x * kThreads) {
      const int b = (int)(i / t.max_pages), e = (int)(i - (int64_t)b * t.max_pages);
      int32_t& entry = t.entries[b * t.stride + e];
      const int32_t p = entry;
      if ((uint32_t)p < (uint32_t)c.num_pages && remap.map[p] != p) entry = remap.map[p];
    }
  }
  const int arrays = 2 * c.n_layers, la = (int)(blockIdx.x % (unsigned)arrays);
  const Layer& layer = c.layers[la >> 1];
  const int array = la & 1, units = layer.units, chunks = layer.heads * c.chunks;  // of a page
  const int shift = __builtin_ctz(layer.chunk_bytes / 16), tid = threadIdx.x;              // 16-byte pieces of a chunk
  const int64_t page_bytes = (int64_t)chunks * layer.chunk_bytes;
  uint8_t* const data = layer.data[array];
  uint8_t* const scale = layer.scale[array];
  for (int64_t u = blockIdx.x / (unsigned)arrays; u < (int64_t)pairs * units; u += gridDim.x / (unsigned)arrays) {
    const int i = (int)(u / units), j0 = (int)(u - (int64_t)i * units) * layer.per;
    const int32_t from = src[i], to = dst[i];
    if ((uint32_t)from >= (uint32_t)c.num_pages || (uint32_t)to >= (uint32_t)c.num_pages || from == to) continue;
    const int n = min(layer.per, chunks - j0), live = slots ? (slots[i] + 31) >> 5 : c.chunks;
    const u32x4* const s = reinterpret_cast<const u32x4*>(data + from * page_bytes + (int64_t)j0 * layer.chunk_bytes);
    u32x4* const d = reinterpret_cast<u32x4*>(data + to * page_bytes + (int64_t)j0 * layer.chunk_bytes);
    constexpr int kAtOnce = 4;
    for (int p0 = tid; p0 < n << shift; p0 += kAtOnce * kThreads) {
      u32x4 v[kAtOnce];
      bool go[kAtOnce];
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k) {
        const int p = p0 + k * kThreads;
        go[k] = p < n << shift && ((j0 + (p >> shift)) & (c.chunks - 1)) < live;
        if (go[k]) v[k] = s[p];
      }
#pragma unroll
      for (int k = 0; k < kAtOnce; ++k)
        if (go[k]) __builtin_nontemporal_store(v[k], d + p0 + k * kThreads);
    }
    if (scale) {  // 32 bytes per chunk
      for (int p = tid; p < n * 4; p += kThreads) {
        if (((j0 + p / 4) & (c.chunks - 1)) >= live) continue;
        const int64_t at = (int64_t)j0 * 32 + p * 8;
        *reinterpret_cast<uint64_t*>(scale + (int64_t)to * chunks * 32 + at) =
            *reinterpret_cast<const uint64_t*>(scale + (int64_t)from * chunks * 32 + at);
      }
    }
  }
}

// --- free and compact --------------------------------------------------------------------------------------------

__global__ __launch_bounds__(kThreads) void free_kernel(G4PageTable t, const int32_t* keep, int32_t num_pages, int32_t page_size,
                                                        int32_t* refs) {
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < (int64_t)t.rows * t.max_pages;
       i += (int64_t)gridDim.x * kThreads) {
    const int b = (int)(i / t.max_pages), e = (int)(i - (int64_t)b * t.max_pages);
    const int64_t kept = ((int64_t)max(keep[b], 0) + page_size - 1) / page_size;
    if (e < kept) continue;
    int32_t& entry = t.entries[b * t.stride + e];
    const int32_t p = entry;
    if ((uint32_t)p < (uint32_t)num_pages) atomicSub(refs + p, 1);
    if (p != -1) entry = -1;
  }
}

// Where every page goes: with n pages in use, the i-th in use at n or behind it to the i-th free one below n. Pages first,
// first + step, ... by this thread.
template <int THREADS>
__device__ __forceinline__ void move_pages(int32_t* refs, int32_t pages, const PoolWorkspace& w, int32_t* live, int64_t first, int64_t step) {
  __shared__ FreePages<THREADS> free;
  const int64_t groups = groups_of(pages);
  free.load(w, groups);
  const int n = pages - free.total();
  const int holes = free.rank(w, groups, n);  // free pages below n, as many as pages in use from n on
  if (first == 0) *live = n, *w.moved = holes;
  for (int64_t p = first; p < pages; p += step) {
    int32_t to = (int32_t)p;
    if (p >= n && !(w.bits[p >> 6] >> (p & 63) & 1)) {
      const int i = (int)(p - n) - (free.rank(w, groups, p) - holes);
      to = free.select(w, i);
      w.src[i] = (int32_t)p;
      w.dst[i] = to;
      refs[to] = refs[p];
      refs[p] = 0;
    }
    w.map[p] = to;
  }
}
__global__ __launch_bounds__(kThreads) void move_kernel(int32_t* refs, int32_t pages, PoolWorkspace w, int32_t* live) {
  move_pages<kThreads>(refs, pages, w, live, (int64_t)blockIdx.x * kThreads + threadIdx.x, (int64_t)gridDim.x * kThreads);
}
// The scan and this in one launch of one workgroup, as few_kernel (replayed from a graph, 300 pages 13.3 -> 12.1 us with the copies, 2200
// 35.7 -> 34.9; 4200 17.7 -> 18.9, of one head of 64).
constexpr int kMovePages = 2560;
__global__ __launch_bounds__(kFewThreads) void few_move_kernel(int32_t* refs, int32_t pages, PoolWorkspace w, int32_t* live) {
  __shared__ uint64_t bits[kMovePages / 64];
  __shared__ int32_t counts[kMovePages / kGroup];
  w.bits = bits, w.counts = counts;
  for (int g = threadIdx.x >> 6; g < groups_of(pages); g += kFewThreads / 64) scan_group(refs, pages, g, w, threadIdx.x & 63);
  __syncthreads();
  move_pages<kFewThreads>(refs, pages, w, live, threadIdx.x, kFewThreads);
}

// --- host ----------------------------------------------------------------------------------------------------------

int check_table(const G4PageTable& t, const char* who) {
  if (t.rows <= 0 || t.max_pages <= 0 || t.stride < t.max_pages || !t.entries)
    return fail(G4_ERR_INVALID, "%s: page table of %d x %d entries, stride %lld%s", who, t.rows, t.max_pages, (long long)t.stride,
                t.entries ? "" : ", NULL");
  if ((int64_t)t.rows * t.max_pages > 0x7fffffffLL) return fail(G4_ERR_UNSUPPORTED, "%s: 2^31 table entries and more", who);
  return G4_OK;
}

int check_pool(int32_t num_pages, int32_t page_size, const int32_t* refs, const char* who) {
  if (num_pages <= 0 || num_pages > 0x7fffffff - kGroup)
    return fail(G4_ERR_INVALID, "%s: num_pages %d (positive, below 2^31 - 256)", who, num_pages);
  if (page_size < 32 || page_size > 1024 || (page_size & (page_size - 1)))
    return fail(G4_ERR_INVALID, "%s: page_size %d (a power of two, 32 .. 1024)", who, page_size);
  if (!refs) return fail(G4_ERR_INVALID, "%s: refs is NULL", who);
  return G4_OK;
}

int check_workspace(const void* p, size_t have, size_t need, const char* who) {
  if (!p || have < need) return fail(G4_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, p ? have : 0, need);
  if (reinterpret_cast<uintptr_t>(p) % 16) return fail(G4_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  return G4_OK;
}

int check_layers(const G4PagedCache* layers, int32_t n, const char* who) {
  if (!layers || n <= 0 || n > 4096) return fail(G4_ERR_INVALID, "%s: %d layers%s", who, n, layers ? "" : ", NULL");
  for (int32_t i = 0; i < n; ++i) {
    const int rc = check_paged_cache(layers[i], who);
    if (rc != G4_OK) return rc;
    if (layers[i].num_pages != layers[0].num_pages || layers[i].page_size != layers[0].page_size)
      return fail(G4_ERR_INVALID, "%s: layer %d has %d pages of %d, layer 0 %d of %d", who, i, layers[i].num_pages,
                  layers[i].page_size, layers[0].num_pages, layers[0].page_size);
    if ((int64_t)layers[i].kv_heads * layers[i].page_size > 0x7fffffff / 2048)
      return fail(G4_ERR_UNSUPPORTED, "%s: %d heads", who, layers[i].kv_heads);
  }
  return G4_OK;
}

unsigned blocks_for(int64_t n, int64_t most) { return (unsigned)(n < 1 ? 1 : n > most ? most : n); }

// `pairs`: their number, or where `moved` is given the most there can be.
int launch_copies(const G4PagedCache* layers, int32_t n, const int32_t* src, const int32_t* dst, const int32_t* slots,
                  int64_t pairs, const int32_t* moved, Remap remap, hipStream_t st, const char* who) {
  for (int32_t l0 = 0; l0 < n; l0 += kMaxLayers) {
    Copies c = {};
    const int32_t here = n - l0 < kMaxLayers ? n - l0 : kMaxLayers;
    c.n_layers = here;
    int64_t units = 0;
    c.num_pages = layers[0].num_pages;
    c.chunks = layers[0].page_size / 32;
    for (int32_t l = 0; l < here; ++l) {
      const G4PagedCache& x = layers[l0 + l];
      Layer& y = c.layers[l];
      y.data[0] = static_cast<uint8_t*>(x.key);
      y.data[1] = static_cast<uint8_t*>(x.value);
      y.scale[0] = x.format == G4_PAGES_E4M3 ? x.key_scale : nullptr;
      y.scale[1] = x.format == G4_PAGES_E4M3 ? x.value_scale : nullptr;
      y.heads = x.kv_heads;
      y.chunk_bytes = 32 * x.head_dim * (x.format == G4_PAGES_E4M3 ? 1 : 2);
      y.per = kUnitBytes / y.chunk_bytes > 0 ? kUnitBytes / y.chunk_bytes : 1;
      y.units = (y.heads * c.chunks + y.per - 1) / y.per;
      if (y.units > units) units = y.units;
    }
    const int64_t blocks = pairs * units, most = (moved ? 4096 : 1 << 23) / (2 * here) + 1;
    hipLaunchKernelGGL(copy_kernel, dim3(blocks_for(blocks, most) * 2u * (unsigned)here), dim3(kThreads), 0, st, c, src, dst, slots,
                       (int)pairs, moved, remap);
    remap.map = nullptr;  // once
    const int rc = check_launch(who);
    if (rc != G4_OK) return rc;
  }
  return G4_OK;
}

template <typename Op>
int launch_assign(const Op& op, int32_t rows, int32_t pages, int32_t* refs, const PoolWorkspace& w, int32_t* shortage,
                  hipStream_t st, const char* who) {
  if (rows <= kFewRows && pages <= kFewPages) {
    hipLaunchKernelGGL(few_kernel<Op>, dim3(1), dim3(kFewThreads), 0, st, op, refs, pages, shortage);
    return check_launch(who);
  }
  const int64_t groups = groups_of(pages), group_blocks = (groups + kWaves - 1) / kWaves;
  hipLaunchKernelGGL(scan_kernel<Op>, dim3((unsigned)(group_blocks + (rows + (int64_t)kWaves - 1) / kWaves)), dim3(kThreads), 0, st, op,
                     refs, pages, w, (int)group_blocks);
  int rc = check_launch(who);
  if (rc != G4_OK) return rc;
  int64_t per = (rows + 255LL) / 256;  // rows per workgroup: up to 256 workgroups, each of which reads the wants before its own
  per = (per + kWaves - 1) / kWaves * kWaves;
  if (per > kThreads) per = kThreads;
  hipLaunchKernelGGL(assign_kernel<Op>, dim3((unsigned)((rows + per - 1) / per)), dim3(kThreads), 0, st, op, refs, pages, w, (int)per,
                     shortage);
  return check_launch(who);
}

}  // namespace
}  // namespace g4

extern "C" int g4_paged_copy(const G4PagedCache* layers, int32_t n_layers, int32_t pairs, const int32_t* src, const int32_t* dst,
                             void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_copy";
  const int rc = check_layers(layers, n_layers, who);
  if (rc != G4_OK) return rc;
  if (pairs <= 0 || !src || !dst) return fail(G4_ERR_INVALID, "%s: %d pairs%s", who, pairs, src && dst ? "" : ", NULL");
  return launch_copies(layers, n_layers, src, dst, nullptr, pairs, nullptr, Remap{}, reinterpret_cast<hipStream_t>(stream), who);
}

extern "C" size_t g4_paged_reserve_workspace_size(const G4PagedReserveArgs* a) {
  g4::PoolWorkspace w;
  return !a || a->num_pages <= 0 || a->table.rows <= 0 ? 0 : g4::carve(w, nullptr, a->num_pages, a->table.rows, 0, false);
}

extern "C" int g4_paged_reserve(const G4PagedReserveArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_reserve";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedReserveArgs& a = *args;
  int rc = check_pool(a.num_pages, a.page_size, a.refs, who);
  if (rc == G4_OK) rc = check_table(a.table, who);
  if (rc == G4_OK && (!a.lengths || !a.shortage)) rc = fail(G4_ERR_INVALID, "%s: lengths / shortage is NULL", who);
  if (rc == G4_OK) rc = check_workspace(a.workspace, a.workspace_bytes, g4_paged_reserve_workspace_size(args), who);
  if (rc != G4_OK) return rc;
  PoolWorkspace w;
  carve(w, a.workspace, a.num_pages, a.table.rows, 0, false);
  const Reserve op{a.table, a.lengths, a.num_pages, a.page_size};
  return launch_assign(op, a.table.rows, a.num_pages, a.refs, w, a.shortage, reinterpret_cast<hipStream_t>(stream), who);
}

extern "C" size_t g4_paged_fork_workspace_size(const G4PagedForkArgs* a) {
  g4::PoolWorkspace w;
  return !a || !a->layers || a->layers[0].num_pages <= 0 || a->out.rows <= 0
             ? 0 : g4::carve(w, nullptr, a->layers[0].num_pages, a->out.rows, a->out.rows, false);
}

extern "C" int g4_paged_fork(const G4PagedForkArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_fork";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedForkArgs& a = *args;
  int rc = check_layers(a.layers, a.n_layers, who);
  if (rc == G4_OK) rc = check_pool(a.layers[0].num_pages, a.layers[0].page_size, a.refs, who);
  if (rc == G4_OK) rc = check_table(a.table, who);
  if (rc == G4_OK) rc = check_table(a.out, who);
  if (rc != G4_OK) return rc;
  if (!a.parents || !a.lengths || !a.shortage) return fail(G4_ERR_INVALID, "%s: parents / lengths / shortage is NULL", who);
  const int32_t ps = a.layers[0].page_size;
  const int32_t width = a.table.max_pages < a.out.max_pages ? a.table.max_pages : a.out.max_pages;
  if ((int64_t)width * ps > 0x7fffffffLL) return fail(G4_ERR_UNSUPPORTED, "%s: %d pages of %d positions pass 2^31", who, width, ps);
  const auto end = [](const G4PageTable& t) { return t.entries + (t.rows - 1) * t.stride + t.max_pages; };
  if (a.table.entries < end(a.out) && a.out.entries < end(a.table))
    return fail(G4_ERR_INVALID, "%s: the children's table overlaps the parents'", who);
  rc = check_workspace(a.workspace, a.workspace_bytes, g4_paged_fork_workspace_size(args), who);
  if (rc != G4_OK) return rc;
  PoolWorkspace w;
  carve(w, a.workspace, a.layers[0].num_pages, a.out.rows, a.out.rows, false);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const Fork op{a.table, a.out, a.parents, a.lengths, a.layers[0].num_pages, ps, w.src, w.dst, w.slots};
  rc = launch_assign(op, a.out.rows, a.layers[0].num_pages, a.refs, w, a.shortage, st, who);
  if (rc != G4_OK) return rc;
  return launch_copies(a.layers, a.n_layers, w.src, w.dst, w.slots, a.out.rows, nullptr, Remap{}, st, who);
}

extern "C" int g4_paged_free(const G4PagedFreeArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_free";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedFreeArgs& a = *args;
  int rc = check_pool(a.num_pages, a.page_size, a.refs, who);
  if (rc == G4_OK) rc = check_table(a.table, who);
  if (rc != G4_OK) return rc;
  if (!a.keep) return fail(G4_ERR_INVALID, "%s: keep is NULL", who);
  const int64_t n = (int64_t)a.table.rows * a.table.max_pages;
  hipLaunchKernelGGL(free_kernel, dim3(blocks_for((n + kThreads - 1) / kThreads, 1 << 16)), dim3(kThreads), 0,
                     reinterpret_cast<hipStream_t>(stream), a.table, a.keep, a.num_pages, a.page_size, a.refs);
  return check_launch(who);
}

extern "C" size_t g4_paged_compact_workspace_size(const G4PagedCompactArgs* a) {
  g4::PoolWorkspace w;
  return !a || !a->layers || a->layers[0].num_pages <= 0
             ? 0 : g4::carve(w, nullptr, a->layers[0].num_pages, 0, a->layers[0].num_pages / 2 + 1, true);
}

extern "C" int g4_paged_compact(const G4PagedCompactArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_compact";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedCompactArgs& a = *args;
  int rc = check_layers(a.layers, a.n_layers, who);
  if (rc == G4_OK) rc = check_pool(a.layers[0].num_pages, a.layers[0].page_size, a.refs, who);
  if (rc == G4_OK) rc = check_table(a.table, who);
  if (rc == G4_OK && !a.live) rc = fail(G4_ERR_INVALID, "%s: live is NULL", who);
  if (rc == G4_OK) rc = check_workspace(a.workspace, a.workspace_bytes, g4_paged_compact_workspace_size(args), who);
  if (rc != G4_OK) return rc;
  const int32_t pages = a.layers[0].num_pages;
  PoolWorkspace w;
  carve(w, a.workspace, pages, 0, pages / 2 + 1, true);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  if (pages <= kMovePages) {
    hipLaunchKernelGGL(few_move_kernel, dim3(1), dim3(kFewThreads), 0, st, a.refs, pages, w, a.live);
    if ((rc = check_launch(who)) != G4_OK) return rc;
  } else {
    const int64_t group_blocks = (groups_of(pages) + kWaves - 1) / kWaves;
    hipLaunchKernelGGL(scan_kernel<int>, dim3((unsigned)group_blocks), dim3(kThreads), 0, st, 0, a.refs, pages, w, (int)group_blocks);
    if ((rc = check_launch(who)) != G4_OK) return rc;
    hipLaunchKernelGGL(move_kernel, dim3(blocks_for((pages + (int64_t)kThreads - 1) / kThreads, 256)), dim3(kThreads), 0, st, a.refs,
                       pages, w, a.live);
    if ((rc = check_launch(who)) != G4_OK) return rc;
  }
  return launch_copies(a.layers, a.n_layers, w.src, w.dst, nullptr, pages / 2, w.moved, Remap{a.table, w.map}, st, who);
}
