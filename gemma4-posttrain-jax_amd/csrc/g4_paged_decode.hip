// One-token attention over a paged cache (g4_paged_decode_attention).
//
// Per (row, kv head): scores s = q . k on MFMA with the keys as the A operand, so that a lane holds the
// scores of keys 8 g .. 8 g + 7 (g = lane / 16) of its query column lane % 16 -- which is the B operand of
// the value product, V^T as A. Neither scores nor probabilities leave the registers. One pass over
// the keys: per wave a running maximum m and sum l in f32, o rescaled where m grows.
//
// A (row, head) is one workgroup's work, or, where rows are long or few, pieces of at most `per` chunks of 32
// slots: `per` follows from the sum of all rows' chunks, so that ragged rows, few long ones and many short
// ones fill the chip alike. The lengths stand on the device, so each workgroup finds its piece from them
// itself, or in a large batch from what one workgroup has made of them before. A (row, head) of one piece is
// finished by it; the others leave (m, l, o) per piece, which a last launch joins in the pieces' order.
//
// Bound by HBM where there is enough to read: 16 rows x 2 heads of 1024 .. 32768 keys of 256 dims, 553 MB in bf16 in
// 87.8 us (6.3 TB/s; a plain non-temporal read reaches 7.1), 277 MB in e4m3 in 45.6 us (6.1), and 3 - 4 us more for the
// join; 256 rows of 200 .. 767 keys, 256 MB, in 47 us (5.4). By latency where there is little: 2 (row, head)s of 512 keys 9.6 us.
#include <type_traits>

#include "g4_paged.h"

namespace g4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kCus = 256, kXcds = 8;

// 16 bytes by the caches' usual way, or past them.
template <bool NT>
__device__ __forceinline__ u32x4 load_piece(std::bool_constant<NT>, __amdgpu_buffer_rsrc_t r, uint32_t voffset, uint32_t soffset) {
  if constexpr (NT)
    return buffer_load16_nt(r, voffset, soffset);
  else
    return buffer_load16(r, voffset, soffset);
}

template <int D, int WAVES_>
struct Groups {
  static constexpr int WAVES = WAVES_;                  // per workgroup
  static constexpr int SIMD_WAVES = D >= 256 ? 2 : 4;   // resident, by registers
  static constexpr int PARTS = D == 512 ? 2 : 1;        // waves that share a chunk, a half of the dims each
  static constexpr int KEYS = WAVES / PARTS;            // chunks in work at a time
  static constexpr int THREADS = 64 * WAVES;
};
constexpr int split_waves(int D) { return D == 512 ? 8 : 4; }
// Workgroups of the split kernel that are resident at once.
constexpr int resident(int D) { return kCus * (D == 512 ? 1 : (D == 256 ? 2 : 4)); }
// elements between q rows (bf16) and between o rows (f32) in LDS: 16 rows' accesses fall on different banks
constexpr int q_stride(int D) { return D + 8; }
constexpr int o_stride(int D) { return D + 4; }

// Floats of LDS for the waves' o; with two parts the scores of two turns are exchanged there before.
template <int D, int WAVES>
__host__ __device__ constexpr int o_floats(int R) {
  using G = Groups<D, WAVES>;
  const int o = G::KEYS * R * o_stride(D), scores = G::PARTS == 2 ? 2 * G::WAVES * 64 * 8 : 0;
  return o > scores ? o : scores;
}

struct Workspace {
  float* o;      // [slots][R][D] o of each piece of a split (row, head)
  float* ml;     // [slots][R][2] their m and l
  int2* ranges;  // [pairs] first slot and number of slots of a (row, head), {0, 0}: not split
  int2* plan;    // [batch + 1] pieces and slots before each row; NULL up to kRows rows
};

// The two MFMA A operands (keys: 8 dims each; values: 8 slots of a dim each) in 16 bytes of e4m3.
__device__ __forceinline__ bf16x8 e4m3_operand(uint32_t w0, uint32_t w1) {
  u32x4 o;
  uint32_t lo, hi;
  unpack_e4m3(w0, lo, hi);
  o[0] = lo, o[1] = hi;
  unpack_e4m3(w1, lo, hi);
  o[2] = lo, o[3] = hi;
  return as_bf16x8(o);
}

// What one wave holds of a chunk: DW dims.
template <int DW, bool F8>
struct Shape {
  static constexpr int KRUNS = F8 ? DW / 64 : DW / 32;  // 16-byte key loads per lane, chunk and half
  static constexpr int VLOADS = F8 ? DW / 32 : DW / 16;  // 16-byte value loads per lane and chunk
  static constexpr int BYTES = F8 ? 1 : 2;
};

struct RowKeys {
  int lo, hi;  // attended positions [lo, hi)
  __device__ __forceinline__ int first() const { return lo >> 5; }
  __device__ __forceinline__ int chunks() const { return hi > lo ? ((hi + 31) >> 5) - (lo >> 5) : 0; }
};

__device__ __forceinline__ RowKeys row_keys(const G4PagedDecodeArgs& a, int length) {
  const int cap = a.max_pages * a.cache.page_size;
  const int hi = length < 0 ? 0 : (length > cap ? cap : length);
  return RowKeys{a.window > 0 && hi > a.window ? hi - a.window : 0, hi};
}

// Sums over the wave's lanes 0 .. own (every lane active), and over all lanes, by lane moves in the vector
// pipeline: shifts within the rows of 16, then row ends broadcast to the rows after them.
__device__ __forceinline__ int scan_incl(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);  // row_shr:2
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);  // row_shr:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);  // row_shr:8
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return v;
}
__device__ __forceinline__ int sum_lanes(int v) { return __builtin_amdgcn_readlane(scan_incl(v), 63); }

// A workgroup's part of a (row, head): piece `index` of `count`.
struct Piece {
  int b, h, index, count, slot;  // slot: its place in the workspace (count > 1)
  RowKeys keys;                  // of row b
};

// How long the pieces are: the least of kTries lengths `per` whose pieces are all resident at once. The rows' ends add
// at most one piece per (row, head) to total / per, so the last of them does where there are fewer of those than room.
// Where there are more, rows of up to twice the mean share of a workgroup stay whole.
// The host bounds the chunks of all (row, head) pairs by 2^30 and a row's by 2^22, which the f32 division needs.
constexpr int kTries = 5;
__device__ __forceinline__ float try_share(int i, int total, int pairs, int room, int min_per) {  // 1 / per
  const int target = pairs < room ? room - (int)((int64_t)pairs * i / (kTries - 1)) : room / 2;
  const int per = (int)((float)total * __builtin_amdgcn_rcpf((float)target)) + 1;
  return __builtin_amdgcn_rcpf((float)(per > min_per ? per : min_per));
}
// ceil(n / per), 1 of a row without chunks: floor((n - 1) / per) + 1, the quotient off a whole number by 1 / per at
// least where it is not one
__device__ __forceinline__ int pieces_of(int n, float share) { return (n > 0 ? (int)((float)(n - 1) * share) : 0) + 1; }

// Consecutive pieces on one XCD (workgroup i runs on XCD i % 8): rows that share pages read them from its L2. False:
// none for this workgroup.
__device__ __forceinline__ bool my_piece(int count, int& want) {
  const int xcd_share = (count + kXcds - 1) / kXcds, y = blockIdx.x / kXcds;
  want = (int)(blockIdx.x % kXcds) * xcd_share + y;
  return y < xcd_share && want < count;
}

// Piece blockIdx of a cut call of up to kRows rows. Every wave finds it by itself: the rows' chunk counts are summed over the
// wave, then the pieces and the workspace slots before each row.
constexpr int kRowRegs = 8, kRows = 64 * kRowRegs;

__device__ __forceinline__ bool find_piece(const G4PagedDecodeArgs& a, int room, int min_per, int lane, Piece& out) {
  const int H = a.cache.kv_heads, B = a.batch;
  RowKeys rows[kRowRegs] = {};  // of rows 64 i + lane; no positions behind the last row
  int length[kRowRegs];
  const bool upper = B > kRows / 2;  // one branch for the upper half: the loads are on their way together
#pragma unroll
  for (int i = 0; i < kRowRegs; ++i) {
    if (i == kRowRegs / 2 && !upper) break;
    const int b = 64 * i + lane;
    length[i] = a.lengths[b < B ? b : B - 1];
  }
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kRowRegs; ++i) {
    if (i == kRowRegs / 2 && !upper) break;
    rows[i] = row_keys(a, 64 * i + lane < B ? length[i] : 0);
    sum += rows[i].chunks();
  }
  const int total = sum_lanes(sum) * H;
  float share[kTries];
  int n_pieces[kTries];
#pragma unroll
  for (int i = 0; i < kTries; ++i) {
    share[i] = try_share(i, total, B * H, room, min_per);
    n_pieces[i] = 0;
  }
#pragma unroll
  for (int j = 0; j < kRowRegs; ++j) {
    if (64 * j >= B) break;
#pragma unroll
    for (int i = 0; i < kTries; ++i) n_pieces[i] += 64 * j + lane < B ? pieces_of(rows[j].chunks(), share[i]) : 0;
  }
  float cut = share[kTries - 1];
  int count = 0, want;
#pragma unroll
  for (int i = kTries - 1; i >= 0; --i) {
    n_pieces[i] = sum_lanes(n_pieces[i]) * H;
    if (i == kTries - 1 || n_pieces[i] <= room) cut = share[i], count = n_pieces[i];
  }
  if (!my_piece(count, want)) return false;
  int before = 0, slots = 0;  // pieces and slots of the rows before these 64
#pragma unroll
  for (int j = 0; j < kRowRegs; ++j) {
    if (64 * j >= B) break;
    const int k = 64 * j + lane < B ? pieces_of(rows[j].chunks(), cut) : 0, used = k > 1 ? k * H : 0;
    const int incl = scan_incl(k * H), sincl = scan_incl(used);
    const int end = before + __builtin_amdgcn_readlane(incl, 63);
    if (want < end) {
      const int at = __builtin_popcountll(__ballot(before + incl <= want));  // the row's lane
      const int kk = __builtin_amdgcn_readlane(k, at);
      const int local = want - before - (__builtin_amdgcn_readlane(incl, at) - kk * H);
      out.b = 64 * j + at;
      out.h = __builtin_amdgcn_readfirstlane(local / kk);
      out.index = local - out.h * kk;
      out.count = kk;
      out.slot = slots + __builtin_amdgcn_readlane(sincl, at) - (kk > 1 ? kk * H : 0) + local;
      out.keys = RowKeys{__builtin_amdgcn_readlane(rows[j].lo, at), __builtin_amdgcn_readlane(rows[j].hi, at)};
      return true;
    }
    before = end;
    slots += __builtin_amdgcn_readlane(sincl, 63);
  }
  return false;
}

// Of more rows a launch of one workgroup writes the pieces and slots before each row and before their end, [batch + 1],
// and a wave looks its piece up: reading all lengths in every workgroup of a grid that grows with the rows would take
// time with their square. us per call of rows of 20 - 199 keys in a table of 4096, e4m3, found by each wave (1024 rows and
// more: in turns of 256) / planned:
//     rows                     257        384        512        1024       4096
//     2 heads of 256 dims   16.4/19.5  21.0/23.1  25.8/25.2  64.0/39.9   541/134
//     1 head of 64 dims     11.7/15.0  13.3/15.5  15.4/16.3  26.7/16.1   206/33
// Beyond 512 rows their lengths would take more registers than the loop leaves.
constexpr int kPlanThreads = 1024, kPlanWaves = kPlanThreads / 64;

// Over the workgroup: the sum of v, and of the threads before this one.
__device__ __forceinline__ int scan_workgroup(int v, int& before, int (&waves)[kPlanWaves]) {
  const int incl = scan_incl(v), wave = threadIdx.x >> 6;
  __syncthreads();  // what was read from `waves` before
  if ((threadIdx.x & 63) == 63) waves[wave] = incl;
  __syncthreads();
  int total = 0;
  before = incl - v;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    before += w < wave ? waves[w] : 0;
    total += waves[w];
  }
  return total;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(G4PagedDecodeArgs a, int2* plan, int room, int min_per) {
  __shared__ int waves[kPlanWaves];
  const int H = a.cache.kv_heads, B = a.batch;
  // this thread's rows
  const int b0 = (int)((int64_t)B * threadIdx.x / kPlanThreads), b1 = (int)((int64_t)B * (threadIdx.x + 1) / kPlanThreads);
  auto chunks_of = [&](int b) { return row_keys(a, a.lengths[b]).chunks(); };
  int sum = 0, before, slots;
  for (int b = b0; b < b1; ++b) sum += chunks_of(b);
  const int total = scan_workgroup(sum, before, waves) * H;
  float share[kTries], cut = 0.f;
  int n_pieces[kTries];
#pragma unroll
  for (int i = 0; i < kTries; ++i) {
    share[i] = try_share(i, total, B * H, room, min_per);
    n_pieces[i] = 0;
  }
  for (int b = b0; b < b1; ++b) {
    const int n = chunks_of(b);
#pragma unroll
    for (int i = 0; i < kTries; ++i) n_pieces[i] += pieces_of(n, share[i]);
  }
#pragma unroll
  for (int i = kTries - 1; i >= 0; --i) {
    const int count = scan_workgroup(n_pieces[i], before, waves) * H;
    if (i == kTries - 1 || count <= room) cut = share[i];
  }
  int pieces = 0, used = 0;
  for (int b = b0; b < b1; ++b) {
    const int k = pieces_of(chunks_of(b), cut) * H;
    pieces += k;
    used += k > H ? k : 0;
  }
  const int count = scan_workgroup(pieces, before, waves), all_slots = scan_workgroup(used, slots, waves);
  for (int b = b0; b < b1; ++b) {
    const int k = pieces_of(chunks_of(b), cut) * H;
    plan[b] = make_int2(before, slots);
    before += k;
    slots += k > H ? k : 0;
  }
  if (threadIdx.x == 0) plan[B] = make_int2(count, all_slots);
}

__device__ __forceinline__ bool find_planned(const G4PagedDecodeArgs& a, const int2* plan, int lane, Piece& out) {
  const int H = a.cache.kv_heads, B = a.batch;
  int want;
  if (!my_piece(plan[B].x, want)) return false;
  int b = 0, n = B;  // the row is one of b .. b + n - 1
  while (n > 1) {
    const int step = (n + 63) / 64, at = lane * step;
    const int before = at < n ? plan[b + at].x : 0x7fffffff;
    const int skip = (__builtin_popcountll(__ballot(before <= want)) - 1) * step;
    b += skip;
    n = n - skip < step ? n - skip : step;
  }
  const int2 first = plan[b];
  const int kk = __builtin_amdgcn_readfirstlane((plan[b + 1].x - first.x) / H), local = want - first.x;
  out.b = b;
  out.h = __builtin_amdgcn_readfirstlane(local / kk);
  out.index = local - out.h * kk;
  out.count = kk;
  out.slot = first.y + local;
  out.keys = row_keys(a, a.lengths[b]);
  return true;
}

template <int D, bool F8, int WAVES, bool SPLIT>
__global__ __launch_bounds__((Groups<D, WAVES>::THREADS)) __attribute__((amdgpu_waves_per_eu(Groups<D, WAVES>::SIMD_WAVES)))
void paged_decode_kernel(G4PagedDecodeArgs a, Workspace ws, int room, int large) {
  using G = Groups<D, WAVES>;
  constexpr int kThreads = G::THREADS, kKeys = G::KEYS, DW = D / G::PARTS;
  using Sh = Shape<DW, F8>;
  constexpr int kChunkBytes = 32 * D * Sh::BYTES;
  // [kKeys][R][o_stride(D)] o, in its place before that the score exchange | [R][q_stride(D)] q | [kKeys][16] m, l
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int R = a.group, H = a.cache.kv_heads, ps = a.cache.page_size;
  uint16_t* q_lds = reinterpret_cast<uint16_t*>(lds + o_floats<D, WAVES>(R));
  float* m_lds = reinterpret_cast<float*>(q_lds + R * q_stride(D));
  float* l_lds = m_lds + kKeys * 16;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int key_wave = w / G::PARTS, half = G::PARTS == 2 ? w & 1 : 0;
  const int page_shift = __builtin_ctz(ps) - 5;  // chunks per page, log2

  Piece piece{0, 0, 0, 1, 0, RowKeys{0, 0}};
  if constexpr (SPLIT) {
    if (!(ws.plan ? find_planned(a, ws.plan, lane, piece) : find_piece(a, room, kKeys, lane, piece))) return;
  } else {
    const int pairs = a.batch * H, share = (pairs + kXcds - 1) / kXcds;
    const int y = blockIdx.x / kXcds, pair = (int)(blockIdx.x % kXcds) * share + y;
    if (y >= share || pair >= pairs) return;
    piece.b = pair / H;
    piece.h = pair - piece.b * H;
    piece.keys = row_keys(a, a.lengths[piece.b]);
  }
  const int b = piece.b, h = piece.h, pair = b * H + h;
  const RowKeys keys = piece.keys;
  const int n = keys.chunks();
  // piece i of k: chunks [i n / k, (i + 1) n / k)
  const int c_first = keys.first() + (SPLIT ? (int)((int64_t)n * piece.index / piece.count) : 0);
  const int last = keys.first() + (SPLIT ? (int)((int64_t)n * (piece.index + 1) / piece.count) : n);

  // the q rows on their way to LDS, asked for before the keys: loads return in order
  constexpr int kQLoads = 16 * D / 8 / kThreads > 0 ? 16 * D / 8 / kThreads : 1;
  u32x4 qv[kQLoads];
#pragma unroll
  for (int j = 0; j < kQLoads; ++j)
    if (tid + j * kThreads < R * D / 8)
      qv[j] = load16(reinterpret_cast<const uint16_t*>(a.q) + (int64_t)pair * R * D + (tid + j * kThreads) * 8);

  float m = kNegInf, l = 0.f;
  floatx4 o[DW / 16];
#pragma unroll
  for (int t = 0; t < DW / 16; ++t) o[t] = floatx4{0.f, 0.f, 0.f, 0.f};

  // One chunk ahead: the loads of a wave's next chunk are issued as the registers of this one's keys, then of
  // its values, become free. A chunk without a page has a resource of no bytes: its loads give zeros.
  u32x4 kv[2][Sh::KRUNS], vv[Sh::VLOADS];
  uint2 kscale = make_uint2(0, 0), vscale = make_uint2(0, 0);
  const int32_t* table = a.page_table + b * a.table_stride;
  struct Place {
    int64_t slot;  // slots before the chunk in the pool, of this head
    bool there;
  };
  auto place_of = [&](int page, int c) -> Place {
    const bool there = (uint32_t)page < (uint32_t)a.cache.num_pages;
    return Place{((int64_t)(there ? page : 0) * H + h) * ps + (c * 32 & (ps - 1)), there};
  };
  // the pages of this wave's next 64 chunks, one per lane
  int pages = -1;
  auto load_pages = [&](int c) {
    const int mine = c + lane * kKeys;
    pages = mine < last ? table[mine >> page_shift] : -1;
  };
  auto wait_pages = [&]() { __asm__ volatile("" : "+v"(pages)); };  // here, not at every use behind a branch
  int c = c_first + key_wave, turn = 0;  // the wave's chunk and its number among the wave's
  // the first page by the scalar cache, the sooner
  const int entry = (c < last ? c : (last > 0 ? last - 1 : 0)) >> page_shift;
  const int page = __builtin_amdgcn_readfirstlane(table[entry]);
  // Keys and values that this call reads once pass the caches by (non-temporal loads), unless a row beside this one
  // has the same page where this piece begins, or the call is so small that its latency counts (kStreamBytes). One
  // answer for the workgroup, whose waves meet at barriers in what follows.
  const int32_t* mine = table + (c_first >> page_shift);
  const int own = mine[0], above = mine[b > 0 ? -a.table_stride : 0], below = mine[b + 1 < a.batch ? a.table_stride : 0];
  const bool stream = large && !(b > 0 && above == own) && !(b + 1 < a.batch && below == own);
  auto load_keys = [&](const Place& at, auto nt) {
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc(reinterpret_cast<const uint8_t*>(a.cache.key) + at.slot * (D * Sh::BYTES), at.there ? kChunkBytes : 0);
    const int lane_at = col * 64 + grp * 16;
#pragma unroll
    for (int i = 0; i < 2 * Sh::KRUNS; ++i) kv[i % 2][i / 2] = load_piece(nt, r, lane_at, (2 * half * Sh::KRUNS + i) * 1024);
    if constexpr (F8) {
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.cache.key_scale + at.slot, at.there ? 32 : 0);
      kscale = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * grp, 0, 0));
    }
  };
  auto load_values = [&](const Place& at, auto nt) {
    const __amdgpu_buffer_rsrc_t r =
        make_rsrc(reinterpret_cast<const uint8_t*>(a.cache.value) + at.slot * (D * Sh::BYTES), at.there ? kChunkBytes : 0);
    const int lane_at = (grp * (D * Sh::BYTES / 2) + col) * 16;
#pragma unroll
    for (int t = 0; t < Sh::VLOADS; ++t) vv[t] = load_piece(nt, r, lane_at, (half * Sh::VLOADS + t) * 256);
    if constexpr (F8) {
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.cache.value_scale + at.slot, at.there ? 32 : 0);
      vscale = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * grp, 0, 0));
    }
  };

  load_pages(c);
  auto attend = [&](auto nt) {
    // every load below is issued by every wave, so that the waits for them can count: no branch but zero bytes
    Place at = place_of(c < last ? page : -1, c);
    load_keys(at, nt);
    wait_pages();
#pragma unroll
    for (int j = 0; j < kQLoads; ++j)
      if (tid + j * kThreads < R * D / 8)
        *reinterpret_cast<u32x4*>(q_lds + (tid + j * kThreads) / (D / 8) * q_stride(D) + tid % (D / 8) * 8) = qv[j];
    __syncthreads();
    load_values(at, nt);  // behind the barrier: a CU issues the loads of its waves one after the other, the keys' first
    // the columns beyond the R rows compute on the last row and are dropped
    const uint16_t* qrow = q_lds + (col < R ? col : R - 1) * q_stride(D) + half * DW + (F8 ? 16 : 8) * grp;
    // operand s: e4m3 keys come 16 consecutive dims a load, two operands
    auto qop = [&](int s) -> bf16x8 { return as_bf16x8(load16(qrow + (F8 ? 64 * (s / 2) + 8 * (s % 2) : 32 * s))); };
    // two parts meet at a barrier in every turn, so all waves take the turns of the first
    const int turns = (last - (G::PARTS == 2 ? c_first : c) + kKeys - 1) / kKeys;
    while (turn < turns) {
      const bool more = c + kKeys < last;
      ++turn;
      if ((turn & 63) == 0) {
        load_pages(c + kKeys);
        wait_pages();
      }
      const Place next = place_of(more ? __builtin_amdgcn_readlane(pages, turn & 63) : -1, c + kKeys);
      const int lo = at.there ? keys.lo : keys.hi, hi = keys.hi;  // this chunk's keys are those in [lo, hi)
      floatx4 sc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int s = 0; s < Sh::KRUNS; ++s)
#pragma unroll
        for (int bb = 0; bb < 2; ++bb) {
          if constexpr (F8) {
            sc[bb] = mfma16x16x32(e4m3_operand(kv[bb][s][0], kv[bb][s][1]), qop(2 * s), sc[bb]);
            sc[bb] = mfma16x16x32(e4m3_operand(kv[bb][s][2], kv[bb][s][3]), qop(2 * s + 1), sc[bb]);
          } else {
            sc[bb] = mfma16x16x32(as_bf16x8(kv[bb][s]), qop(s), sc[bb]);
          }
        }
      if constexpr (G::PARTS == 2) {  // the sum of both halves' scores, the same in both waves
        float* mine = lds + (((turn & 1) * G::WAVES + w) * 64 + lane) * 8;
        const float* other = lds + (((turn & 1) * G::WAVES + (w ^ 1)) * 64 + lane) * 8;
        *reinterpret_cast<floatx4*>(mine) = sc[0];
        *reinterpret_cast<floatx4*>(mine + 4) = sc[1];
        wg_barrier();
        sc[0] += *reinterpret_cast<const floatx4*>(other);
        sc[1] += *reinterpret_cast<const floatx4*>(other + 4);
      }
      if constexpr (F8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[j / 4][j % 4] *= exp2_byte((j < 4 ? kscale.x : kscale.y) >> (8 * (j % 4)) & 0xff);
      }
      __builtin_amdgcn_sched_barrier(0);
      load_keys(next, nt);
      __builtin_amdgcn_sched_barrier(0);

      // keys 8 grp + j of the chunk
      const bool inner = c * 32 >= lo && c * 32 + 32 <= hi;  // every slot is an attended key
      float p[8], mx = m;
      bool on[8];
      const int j_lo = lo - (c * 32 + 8 * grp), j_hi = hi - (c * 32 + 8 * grp);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        on[j] = (j >= j_lo) & (j < j_hi);
        p[j] = on[j] ? sc[j / 4][j % 4] : kNegInf;
        mx = fmaxf(mx, p[j]);
      }
      mx = column_max(mx);
      const float base = mx == kNegInf ? 0.f : mx;
      if (__any(mx > m)) {
        const float alpha = __builtin_amdgcn_exp2f((m - base) * kLog2e);
        m = mx;
        l *= alpha;
#pragma unroll
        for (int t = 0; t < DW / 16; ++t) o[t] *= alpha;
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = __builtin_amdgcn_exp2f((p[j] - base) * kLog2e);
        l += p[j];
        if constexpr (F8) {
          const float v = p[j] * exp2_byte((j < 4 ? vscale.x : vscale.y) >> (8 * (j % 4)) & 0xff);
          p[j] = on[j] ? v : 0.f;
        }
      }
      const bf16x8 pop = as_bf16x8(u32x4{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]),
                                         pack_bf16x2(p[6], p[7])});
      if (!inner) {  // the slots of no attended key may hold anything: 0 x NaN is no 0
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          // e4m3: dword i is keys 4 (i % 2) .. + 3; bf16: keys 2 i, 2 i + 1
          constexpr int KEYS = F8 ? 4 : 2;
          uint32_t mask = 0;
#pragma unroll
          for (int j = 0; j < KEYS; ++j) mask |= on[KEYS * (i % (8 / KEYS)) + j] ? (F8 ? 0xffu : 0xffffu) << (32 / KEYS * j) : 0u;
#pragma unroll
          for (int t = 0; t < Sh::VLOADS; ++t) vv[t][i] &= mask;
        }
      }
#pragma unroll
      for (int t = 0; t < Sh::VLOADS; ++t) {
        if constexpr (F8) {
          o[2 * t] = mfma16x16x32(e4m3_operand(vv[t][0], vv[t][1]), pop, o[2 * t]);
          o[2 * t + 1] = mfma16x16x32(e4m3_operand(vv[t][2], vv[t][3]), pop, o[2 * t + 1]);
        } else {
          o[t] = mfma16x16x32(as_bf16x8(vv[t]), pop, o[t]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      load_values(next, nt);
      __builtin_amdgcn_sched_barrier(0);
      at = next;
      c += kKeys;
    }
  };
  if (stream)
    attend(std::true_type{});
  else
    attend(std::false_type{});

  // the waves' parts joined: o = sum_w exp(m_w - m) o_w, l likewise
  l = column_sum(l);
  if constexpr (G::PARTS == 2) __syncthreads();  // o takes the place of the last turn's exchange
  if (grp == 0 && half == 0) m_lds[key_wave * 16 + col] = m, l_lds[key_wave * 16 + col] = l;
  if (col < R) {
    float* dst = lds + (key_wave * R + col) * o_stride(D) + half * DW;
    // row 4 grp + i of tile t is dim 16 t + 4 grp + i (bf16), or 32 (t / 2) + 2 (4 grp + i) + t % 2 (e4m3)
    if constexpr (F8) {
#pragma unroll
      for (int t = 0; t < DW / 32; ++t) {
        const floatx4 x = o[2 * t], y = o[2 * t + 1];
        *reinterpret_cast<floatx4*>(dst + 32 * t + 8 * grp) = floatx4{x[0], y[0], x[1], y[1]};
        *reinterpret_cast<floatx4*>(dst + 32 * t + 8 * grp + 4) = floatx4{x[2], y[2], x[3], y[3]};
      }
    } else {
#pragma unroll
      for (int t = 0; t < DW / 16; ++t) *reinterpret_cast<floatx4*>(dst + 16 * t + 4 * grp) = o[t];
    }
  }
  __syncthreads();
  const bool whole = !SPLIT || piece.count == 1;
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)pair * R * D;
  for (int i = 4 * tid; i < R * D; i += 4 * kThreads) {
    const int r = i / D;
    float mm = kNegInf;
#pragma unroll
    for (int v = 0; v < kKeys; ++v) mm = fmaxf(mm, m_lds[v * 16 + r]);
    const float base = mm == kNegInf ? 0.f : mm;
    floatx4 num = {0.f, 0.f, 0.f, 0.f};
    float den = 0.f;
#pragma unroll
    for (int v = 0; v < kKeys; ++v) {
      const float x = __builtin_amdgcn_exp2f((m_lds[v * 16 + r] - base) * kLog2e);
      num += x * *reinterpret_cast<const floatx4*>(lds + (v * R + r) * o_stride(D) + i % D);
      den += x * l_lds[v * 16 + r];
    }
    if (whole) {
      const float inv = 1.f / den;
      num = den == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : num * inv;
      *reinterpret_cast<uint2*>(out + i) = make_uint2(pack_bf16x2(num[0], num[1]), pack_bf16x2(num[2], num[3]));
    } else {
      *reinterpret_cast<floatx4*>(ws.o + (int64_t)piece.slot * R * D + i) = num;
      if (i % D == 0) *reinterpret_cast<float2*>(ws.ml + ((int64_t)piece.slot * R + r) * 2) = make_float2(mm, den);
    }
  }
  if (SPLIT && piece.index == 0 && tid == 0) ws.ranges[pair] = whole ? make_int2(0, 0) : make_int2(piece.slot, piece.count);
}

constexpr int kJoinDims = 64;  // elements of o per workgroup: 16 lanes of 4, 16 parts at a time
constexpr int kJoinThreads = 256;
constexpr int kJoinGroups = 2048;  // workgroups of a join, about
constexpr int kJoinParts = kJoinThreads / (kJoinDims / 4);

// The pieces of a (row, head), joined in their order; blockIdx.y of gridDim.y takes every so many stretches of
// kJoinDims elements.
__global__ __launch_bounds__(kJoinThreads) void paged_join_kernel(G4PagedDecodeArgs a, Workspace ws) {
  __shared__ float m_s[kJoinParts], l_s[kJoinParts];
  __shared__ __attribute__((aligned(16))) floatx4 o_s[kJoinParts][kJoinDims / 4];
  const int R = a.group, D = a.cache.head_dim;
  const int pair = blockIdx.x;
  const int2 range = ws.ranges[pair];
  if (range.y == 0) return;
  const int x = threadIdx.x % (kJoinDims / 4), y = threadIdx.x / (kJoinDims / 4);
  for (int i0 = blockIdx.y * kJoinDims; i0 < R * D; i0 += gridDim.y * kJoinDims) {
    const int r = i0 / D;
    // this lane's pieces y, y + 16, ..., each step's loads independent of the sums
    float m = kNegInf, l = 0.f;
    floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int j = y; j < range.y; j += kJoinParts) {
      const int64_t at = (int64_t)(range.x + j) * R;
      const float2 ml = *reinterpret_cast<const float2*>(ws.ml + (at + r) * 2);
      const floatx4 part = *reinterpret_cast<const floatx4*>(ws.o + at * D + i0 + 4 * x);
      const float mx = fmaxf(m, ml.x), base = mx == kNegInf ? 0.f : mx;
      const float f = __builtin_amdgcn_exp2f((m - base) * kLog2e), g = __builtin_amdgcn_exp2f((ml.x - base) * kLog2e);
      m = mx;
      l = f * l + g * ml.y;
      o = f * o + g * part;
    }
    if (x == 0) m_s[y] = m, l_s[y] = l;
    o_s[y][x] = o;
    __syncthreads();
    if (y == 0) {
      float mx = kNegInf;
#pragma unroll
      for (int j = 0; j < kJoinParts; ++j) mx = fmaxf(mx, m_s[j]);
      const float base = mx == kNegInf ? 0.f : mx;
      l = 0.f;
      o = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kJoinParts; ++j) {
        const float f = __builtin_amdgcn_exp2f((m_s[j] - base) * kLog2e);
        l += f * l_s[j];
        o += f * o_s[j][x];
      }
      const float inv = 1.f / l;
      if (l == 0.f) o = floatx4{0.f, 0.f, 0.f, 0.f};
      else o *= inv;
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + (int64_t)pair * R * D + i0 + 4 * x) =
          make_uint2(pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3]));
    }
    __syncthreads();
  }
}

template <int D, int WAVES>
size_t lds_bytes(int R) {
  return ((size_t)o_floats<D, WAVES>(R) + (size_t)R * q_stride(D) / 2 + 2 * Groups<D, WAVES>::KEYS * 16) * sizeof(float);
}

// Whether the rows are cut into pieces: where a row can have more chunks than one workgroup is as fast with. Finding
// the pieces and joining them takes about 4 us up to 512 rows, the plan of 1024 4 us more, of 4096 8. us per call at 256
// dims from twelve caches in turn, whole / split, bf16 and e4m3:
//     pairs   512 keys               1024 keys               2048 keys
//       2     9.7/9.2   7.8/8.9      15.2/9.4   11.4/8.9     26.2/10.7  17.8/9.5
//      16     12.8/10.6 8.7/10.1     21.9/11.2  14.1/9.6     39.9/13.6  23.3/11.1
//      64     14.5/13.4 10.2/11.1    23.6/19.5  15.4/14.7    45.0/29.5  26.1/19.5
//     128     16.2/20.0 11.3/14.8    28.0/29.5  17.6/19.6    51.4/49.7  29.6/29.5
//     512     43.7/47.3 24.7/28.1    84.0/87.5  45.0/48.0    164/168    85.6/88.8
// Up to 64 pairs the border is set at 20 chunks, beyond at 32, although equal rows stay faster whole: a long row among
// short ones would hold its one CU alone. One border for all head dims and formats, although a row's work goes with its
// bytes. Just behind it, at windows of 640 (up to 64 pairs) and 1024, whole / cut:
//                       2 pairs    16         80         128        256        512
//     64 dims, e4m3     6.1/8.0    6.2/8.1    7.3/10.5   7.4/12.3   9.7/14.3   13.5/19.4
//     128 dims, bf16    7.2/8.3    7.4/8.5    12.8/14.8  16.0/19.7  23.3/30.8  45/56
//     256 dims, e4m3    9.4/9.3    9.5/9.6    14.1/14.6  17.1/18.5  23.3/30.4  45/48
//     256 dims, bf16    11.2/9.6   11.4/9.8   25.7/20.8  28.6/29.2  44.0/51.3  86/89
// and at 512 dims in e4m3 (1, 8, 32, 40, 64, 128, 256 pairs) 17.4/11.8, 17.8/12.2, 18.3/14.2, 18.9/19.1, 24.1/24.0,
// 34.7/37.0, 48/52. A window may begin inside a chunk, so it counts 31 positions more.
constexpr int kSplitPairs = 64, kWholeChunksFew = 20, kWholeChunks = 32;
bool split(const G4PagedDecodeArgs& a) {
  const int64_t cap = (int64_t)a.max_pages * a.cache.page_size;
  const int64_t keys = a.window > 0 && a.window < cap ? a.window + 31 : cap;
  const bool few = (int64_t)a.batch * a.cache.kv_heads <= kSplitPairs;
  return (keys + 31) / 32 > (few ? kWholeChunksFew : kWholeChunks);
}

// Whether the call's keys and values are many enough to pass the caches by. From caches in turn that together pass
// the last-level cache (us per call, plain / non-temporal): 512 pairs of 200 - 767 keys in bf16, 256 MB, 54.4 / 48.2, 16 x 2
// rows of up to 32768 keys 102 / 90 (e4m3 58.4 / 51.3), 128 pairs of 512 keys in e4m3 13.2 / 12.1, but 2 pairs of 512 keys
// 10.6 / 12.1. Rows that share pages read them from their XCD's cache: 64 rows, 8 of each with the same 4096 positions,
// 28.2 / 35.5.
constexpr int64_t kStreamBytes = 8 << 20;
bool large(const G4PagedDecodeArgs& a) {
  const int64_t cap = (int64_t)a.max_pages * a.cache.page_size;
  const int64_t keys = a.window > 0 && a.window < cap ? a.window : cap;
  return keys * a.batch * a.cache.kv_heads * a.cache.head_dim * (a.cache.format == G4_PAGES_E4M3 ? 2 : 4) >= kStreamBytes;
}

// A split (row, head) of n > per chunks has at most 2 n / per pieces, and per >= total / room but for the f32
// division's rounding, for which there is room for a few more.
constexpr int kSpare = 8;
size_t slots(const G4PagedDecodeArgs& a) { return 2 * (size_t)resident(a.cache.head_dim) + kSpare; }

size_t workspace_bytes(const G4PagedDecodeArgs& a) {
  if (!split(a)) return 0;
  const size_t plan = a.batch > kRows ? (size_t)a.batch + 1 : 0;
  return slots(a) * a.group * ((size_t)a.cache.head_dim + 2) * 4 + ((size_t)a.batch * a.cache.kv_heads + plan) * 8;
}

template <int D, bool F8, int WAVES, bool SPLIT>
int launch_kernel(const G4PagedDecodeArgs& a, const Workspace& ws, int64_t groups, hipStream_t st) {
  const size_t lds = lds_bytes<D, WAVES>(a.group);
  const void* fn = (const void*)paged_decode_kernel<D, F8, WAVES, SPLIT>;
  if (lds > 64 * 1024) {
    int dev = 0;
    const int rc = device_setup(&dev);
    if (rc != G4_OK) return rc;
    if (!lds_limit_raised(dev, fn))
      return fail(G4_ERR_LAUNCH, "g4_paged_decode_attention: the kernel's LDS limit could not be raised");
  }
  const dim3 grid((unsigned)((groups + kXcds - 1) / kXcds * kXcds));
  hipLaunchKernelGGL((paged_decode_kernel<D, F8, WAVES, SPLIT>), grid, dim3(Groups<D, WAVES>::THREADS), lds, st, a, ws,
                     resident(D), (int)large(a));
  return check_launch("g4_paged_decode_attention");
}

// Waves of a whole row's workgroup. A CU's vector cache gives 64 bytes a clock, which four waves of bf16 loads take
// up, so more of them only add to the join at the end (512 keys of 256 dims, us per call, 8 / 4 waves: 2 pairs 9.6 /
// 8.7, 64 pairs 11.5 / 10.5, 512 pairs 50.1 / 48.6). e4m3 halves the bytes and adds the conversions, which eight waves
// share better while CUs are to spare (2 pairs 7.9 / 8.7, 64 pairs 9.2 / 9.9, 256 pairs 14.2 / 13.6, 512 pairs 30.4 /
// 27.3).
constexpr int kFewPairs = 256;

template <int D, bool F8>
int launch(const G4PagedDecodeArgs& a, hipStream_t st) {
  const int64_t pairs = (int64_t)a.batch * a.cache.kv_heads;
  Workspace ws{};
  if (!split(a)) {
    if constexpr (D == 512) {
      return launch_kernel<D, F8, 8, false>(a, ws, pairs, st);
    } else {
      if constexpr (F8)
        if (pairs < kFewPairs) return launch_kernel<D, F8, 8, false>(a, ws, pairs, st);
      return launch_kernel<D, F8, 4, false>(a, ws, pairs, st);
    }
  }
  ws.o = reinterpret_cast<float*>(a.workspace);
  ws.ml = ws.o + slots(a) * a.group * D;
  ws.ranges = reinterpret_cast<int2*>(ws.ml + slots(a) * a.group * 2);
  if (a.batch > kRows) {
    ws.plan = ws.ranges + pairs;
    hipLaunchKernelGGL(paged_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, a, ws.plan, resident(D),
                       (int)Groups<D, split_waves(D)>::KEYS);
    const int rc = check_launch("g4_paged_decode_attention");
    if (rc != G4_OK) return rc;
  }
  const int rc = launch_kernel<D, F8, split_waves(D), true>(a, ws, resident(D) + pairs + kSpare, st);
  if (rc != G4_OK) return rc;
  const int stretches = a.group * D / kJoinDims;
  const dim3 grid((unsigned)pairs, (unsigned)(pairs * stretches <= kJoinGroups ? stretches : (pairs < kJoinGroups ? kJoinGroups / pairs : 1)));
  hipLaunchKernelGGL(paged_join_kernel, grid, dim3(kJoinThreads), 0, st, a, ws);
  return check_launch("g4_paged_decode_attention");
}

template <int D, bool F8, int WAVES, bool SPLIT>
void setup(int device) {
  const size_t most = lds_bytes<D, WAVES>(16);
  if (most > 64 * 1024) raise_lds_limit(device, (const void*)paged_decode_kernel<D, F8, WAVES, SPLIT>, (int)most);
}
template <int D, bool F8>
void setup(int device) {
  if constexpr (F8 || D == 512) setup<D, F8, 8, false>(device);
  if constexpr (D < 512) setup<D, F8, 4, false>(device);
  setup<D, F8, split_waves(D), true>(device);
}
template <int D>
void setup(int device) {
  setup<D, false>(device), setup<D, true>(device);
}

}  // namespace

int setup_paged_kernels(int device) {
  setup<64>(device), setup<128>(device), setup<256>(device), setup<512>(device);
  return G4_OK;
}

namespace {

// A grid of as many workgroups of up to 512 threads, the pieces' and XCDs' spare ones included, has its threads counted
// in 32 bits.
constexpr int64_t kMaxPairs = kMaxThreads / 512 - resident(64) - kSpare - kXcds;

int check_decode(const G4PagedDecodeArgs& a, const char* who) {
  int rc = check_paged_cache(a.cache, who);
  if (rc == G4_OK) rc = check_page_table(a.page_table, a.max_pages, a.table_stride, a.cache.page_size, who);
  if (rc != G4_OK) return rc;
  if (a.batch <= 0 || a.group <= 0 || a.group > 16 || a.window < 0)
    return fail(G4_ERR_INVALID, "%s: batch %d group %d (1..16) window %d", who, a.batch, a.group, a.window);
  if ((int64_t)a.batch * a.cache.kv_heads > kMaxPairs)
    return fail(G4_ERR_UNSUPPORTED, "%s: batch %d x %d kv heads", who, a.batch, a.cache.kv_heads);
  if ((int64_t)a.max_pages * a.cache.page_size > 1 << 27)
    return fail(G4_ERR_UNSUPPORTED, "%s: %d pages of %d positions pass 2^27 positions", who, a.max_pages, a.cache.page_size);
  if ((int64_t)a.batch * a.cache.kv_heads * ((int64_t)a.max_pages * a.cache.page_size / 32) > 0x3fffffffLL)
    return fail(G4_ERR_UNSUPPORTED, "%s: batch %d x %d kv heads x %d pages pass 2^35 positions", who, a.batch,
                a.cache.kv_heads, a.max_pages);
  if (!a.lengths || !a.q || !a.out) return fail(G4_ERR_INVALID, "%s: lengths / q / out is NULL", who);
  if (reinterpret_cast<uintptr_t>(a.q) % 16 || reinterpret_cast<uintptr_t>(a.out) % 16)
    return fail(G4_ERR_INVALID, "%s: q / out must be 16-byte aligned", who);
  return G4_OK;
}

}  // namespace
}  // namespace g4

extern "C" size_t g4_paged_decode_workspace_size(const G4PagedDecodeArgs* args) {
  if (!args || g4::check_decode(*args, "g4_paged_decode_workspace_size") != G4_OK) return 0;
  return g4::workspace_bytes(*args);
}

extern "C" int g4_paged_decode_attention(const G4PagedDecodeArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_decode_attention";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedDecodeArgs& a = *args;
  const int rc = check_decode(a, who);
  if (rc != G4_OK) return rc;
  const size_t need = workspace_bytes(a);
  if (need && (!a.workspace || a.workspace_bytes < need || reinterpret_cast<uintptr_t>(a.workspace) % 16))
    return fail(G4_ERR_WORKSPACE, "%s needs %zu bytes of 16-byte aligned workspace", who, need);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool f8 = a.cache.format == G4_PAGES_E4M3;
  switch (a.cache.head_dim) {
    case 64: return f8 ? launch<64, true>(a, st) : launch<64, false>(a, st);
    case 128: return f8 ? launch<128, true>(a, st) : launch<128, false>(a, st);
    case 256: return f8 ? launch<256, true>(a, st) : launch<256, false>(a, st);
    default: return f8 ? launch<512, true>(a, st) : launch<512, false>(a, st);
  }
}
