// Causal attention of packed prompts (g4_packed_prefill_attention): sequences of any lengths one behind the other,
// without pads, each token over its own sequence's tokens up to itself, optionally the last `window` of them. The
// scores and the softmax of model.py:320-335, 496-499 per sequence.
//
// The query rows of one kv head are the (token, r) pairs in order, T R of them; a workgroup takes the next
// 128 or 64, whatever sequences they belong to, and walks the 32-key chunks from the first key that one of them
// sees to its last token. A row's keys are one interval [lo, hi], so that a mask is two comparisons: no list of
// tiles, and short sequences share a workgroup. Per chunk S^T = K q^T and O^T += V^T P^T by MFMA 16x16x32, the
// layouts' operand order making the scores' registers the value product's operand.
//
// One pass: p = exp(s - m) with a row maximum m that follows the scores' maximum lazily. m stays while no score of the wave passes it
// by more than kSlack: p then grows to e^kSlack at most, which neither f32 sums nor bf16's relative rounding feel,
// and the four lanes that share a row need not exchange their maxima, nor the accumulators be rescaled, in most chunks. Scores,
// probabilities and sums are f32; p is rounded to bf16 as the MFMA's operand, the result once.
//
// NaN and infinities in keys that a row does not see must not reach it: a masked score is replaced, not multiplied, but a
// masked p = 0 times a NaN value is NaN. A wave whose accumulators are not all finite forms them again from
// memory, key by key where a chunk holds such values (`careful_values`), which costs other calls one look at the accumulators.
#include <algorithm>

#include "g4_attn_tiles.h"
#include "g4_common.h"
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.0f;

// A workgroup's work: NB blocks of 16 query rows by each of NW waves, 128 rows (BIG) or 64. Head dims up to 256: four waves of two
// blocks (at 256 250 registers) or one, two workgroups on a CU, each of which fills the other's barriers, softmax and loads; K and
// V^T take two chunks of LDS each, 64 KiB at 256. (8 x 4096 tokens of 2 x 4 heads of 256, before the blocks were sorted: 506 us; one
// workgroup of eight waves with four chunks of each 586, of one block per wave 589.) Head dim 512: eight waves of one block alone on
// the CU, two chunks of each in 128 KiB, or four, two workgroups, one chunk of each (ONE).
template <int D, bool BIG>
struct Shape {
  static constexpr int NB = BIG && D != 512 ? 2 : 1, NW = BIG && D == 512 ? 8 : 4;
  static constexpr bool ONE = D == 512 && !BIG;
  static constexpr int KS = D / 32;
  static constexpr int T = D / 16;                  // 1 KiB operand tiles of a chunk's K and of its V^T
  static constexpr int CHUNK = T * 1024;
  static constexpr int TW = T / NW;                 // tiles that a wave fetches of each
  static constexpr int ROWS = NW * NB * 16;         // query rows of a workgroup
  static_assert(T % NW == 0, "the waves share the tiles evenly");
  static constexpr int SLOTS = ONE ? 2 : 4;
  static_assert(ROWS * D * 2 <= SLOTS * CHUNK, "the result goes out through the rings");
};

// Over the 16 columns of an MFMA tile, whose values every row of 16 lanes holds.
template <typename F>
__device__ __forceinline__ int columns_reduce(int v, F op) {
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0x128, 0xf, 0xf, true));  // row_ror:8
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0x124, 0xf, 0xf, true));  // row_ror:4
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0x4e, 0xf, 0xf, true));   // quad_perm:[2,3,0,1]
  v = op(v, __builtin_amdgcn_update_dpp(v, v, 0xb1, 0xf, 0xf, true));   // quad_perm:[1,0,3,2]
  return __builtin_amdgcn_readfirstlane(v);
}

// row / R of rows below 2^31: floor(row m / 2^s) with m = ceil(2^s / R), s = 31 + ceil(log2 R) (exact, since row (m R - 2^s) < 2^s).
struct Group {
  uint32_t m;
  int s;
  explicit Group(int R) : s(31) {
    while (1 << (s - 31) < R) ++s;
    m = (uint32_t)(((1ull << s) + R - 1) / R);
  }
  __device__ __forceinline__ int token(int row) const { return (int)((uint64_t)(uint32_t)row * m >> s); }
};

// The wave's rows. This lane's row of column block cb (lane % 16) sees the keys [keys[cb].x, keys[cb].y].
struct Rows {
  int2 keys[2];
  int first, last;            // the keys that some row sees lie in [first, last]
  int all_from[2], all_to[2];  // every row of the column block that sees any sees [all_from, all_to]
  __device__ __forceinline__ bool any(int c) const { return (c << 5) + 31 >= first && (c << 5) <= last; }
  __device__ __forceinline__ bool full(int cb, int c) const { return (c << 5) >= all_from[cb] && (c << 5) + 31 <= all_to[cb]; }
  // bit e <-> key k + e
  __device__ static __forceinline__ uint32_t bits(int2 seen, int k) {
    const int from = min(max(seen.x - k, 0), 8), to = min(max(seen.y - k + 1, 0), 8);  // elements [from, to)
    return (0xffu << from) & ((1u << to) - 1u);
  }
};

// Softmax of one chunk's scores: `p` as the value product's operand, the row statistics brought forward.
// p = exp2(s log2(e) - m log2(e)) takes one fma per score, but the rounding of m log2(e) is another for each maximum, and for one of 2^31
// it is larger than any exponent. Rows whose maximum passes kFar, where it is 2^-14, therefore take their scores less an origin, a
// maximum of theirs, exactly where it counts. That goes with the mask, which such a wave's blocks then have in every chunk: other waves
// pay for it in masked chunks only (packed prompts of up to 8191 tokens 373 -> 376 us; 379 with a branch of its own behind the maximum).
constexpr float kFar = 1024.0f;
template <int NB, int VT>
struct Softmax {
  float m[NB], l[NB];  // row maximum in use, less the origin; this lane's share of the sum
  float origin[NB];

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) m[cb] = kNegInf, l[cb] = origin[cb] = 0.f;
  }
  __device__ static __forceinline__ bool is_far(float x) { return fabsf(x) > kFar && fabsf(x) < -kNegInf; }
  // what an exponent subtracts (before the first key, with scores of -inf alone, nothing)
  __device__ __forceinline__ float base(int cb) const { return m[cb] == kNegInf ? 0.f : m[cb] * kLog2e; }

  __device__ __forceinline__ void chunk(Rows& rows, int c, int lane, floatx4 (&acc)[NB][2], bf16x8 (&pop)[NB],
                                        floatx4 (&oacc)[NB][VT]) {
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) {  // (a wave across a sequence's end masks one of them in every chunk)
      if (rows.full(cb, c)) continue;
      int k = c << 5;
      __asm__ volatile("" : "+s"(k));  // hidden: else its place relative to every row advances in registers
      const uint32_t bits = Rows::bits(rows.keys[cb], k + 8 * (lane >> 4));
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t seen = (uint32_t)__builtin_amdgcn_sbfe((int)bits, e, 1);  // all bits or none
        acc[cb][e >> 2][e & 3] = __uint_as_float((seen & __float_as_uint(acc[cb][e >> 2][e & 3])) | (~seen & 0xff800000u)) - origin[cb];
      }
    }
    float top[NB];
    bool rise = false;
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) {
      top[cb] = acc[cb][0][0];
#pragma unroll
      for (int e = 1; e < 8; ++e) top[cb] = fmaxf(top[cb], acc[cb][e >> 2][e & 3]);
      rise |= top[cb] > m[cb] + kSlack;
    }
    if (__any(rise)) {  // (uniform)
      const bool fresh = c << 5 <= rows.first;  // the wave's first chunk: the accumulators are 0
#pragma unroll
      for (int cb = 0; cb < NB; ++cb) {
        const float next = fmaxf(m[cb], column_max(top[cb]));
        // (before the first key m = -inf: nothing to scale yet)
        const float scale = next > m[cb] ? __builtin_amdgcn_exp2f((m[cb] - next) * kLog2e) : 1.f;
        m[cb] = next;
        l[cb] *= scale;
        if (!fresh) {
#pragma unroll
          for (int i = 0; i < VT; ++i) oacc[cb][i] *= scale;
        }
      }
      bool beyond = false;
#pragma unroll
      for (int cb = 0; cb < NB; ++cb) beyond |= is_far(m[cb]);
      if (__builtin_expect(__any(beyond), 0)) {  // (what a row has summed up stays: sums of another origin's weigh e^-kFar)
#pragma unroll
        for (int cb = 0; cb < NB; ++cb) {
          const float by = is_far(m[cb]) ? m[cb] : 0.f;
          origin[cb] += by;
          m[cb] -= by;
          acc[cb][0] -= by;
          acc[cb][1] -= by;
          rows.all_from[cb] = 0x7fffffff;  // no chunk is full
        }
      }
    }
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) {
      const float ml = base(cb);
      float p[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(acc[cb][e >> 2][e & 3], kLog2e, -ml));
        sum += p[e];
      }
      l[cb] += sum;
      pop[cb] = as_bf16x8(pack8(p));
    }
  }
};

// 16 dims of one column block's values again, chunk by chunk from memory, with the final row maximum: a chunk whose
// values are not all finite key by key, so that a row takes only those that it sees. For waves that met such values: few
// registers and little code matter here, speed does not (the scores are formed anew for every 16 dims).
template <int D>
__device__ __forceinline__ floatx4 careful_values(const Rows& rows, int cb, float origin, float ml, const uint16_t* q,
                                                  __amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv, int i) {
  constexpr int KS = D / 32;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const uint32_t k_lane = (uint32_t)(col * 64 + grp * 16), v_lane = vt_operand_bytes(grp, col, D);
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int c = rows.first >> 5; c << 5 <= rows.last; ++c) {
    floatx4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll 1
    for (int s = 0; s < KS; ++s) {
      const bf16x8 qs = as_bf16x8(q ? load16(q + 32 * s + 8 * grp) : u32x4{0u, 0u, 0u, 0u});
#pragma unroll
      for (int bb = 0; bb < 2; ++bb)
        acc[bb] = mfma16x16x32(as_bf16x8(buffer_load16(rk, k_lane, (uint32_t)c * (uint32_t)(64 * D) + (uint32_t)(2 * s + bb) * 1024u)),
                               qs, acc[bb]);
    }
    uint32_t seen = 0;  // bit k <-> key 32 c + k
#pragma unroll
    for (int g = 0; g < 4; ++g) seen |= Rows::bits(rows.keys[cb], (c << 5) + 8 * g) << (8 * g);
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      p[e] = seen >> (8 * grp + e) & 1u ? __builtin_amdgcn_exp2f(fmaf(acc[e >> 2][e & 3] - origin, kLog2e, -ml)) : 0.f;
    const u32x4 pop = pack8(p);
    const u32x4 v = buffer_load16(rv, v_lane, (uint32_t)c * (uint32_t)(64 * D) + 256u * i);
    bool odd = false;
#pragma unroll
    for (int q = 0; q < 4; ++q) odd |= (v[q] & 0x7f80u) == 0x7f80u || (v[q] & 0x7f800000u) == 0x7f800000u;
    if (!__any(odd)) {
      o = mfma16x16x32(as_bf16x8(v), as_bf16x8(pop), o);
      continue;
    }
#pragma unroll 1
    for (int k = 0; k < 32; ++k) {  // this key alone
      u32x4 keep;
#pragma unroll
      for (int q = 0; q < 4; ++q) keep[q] = k >> 3 == grp && (k & 7) >> 1 == q ? (k & 1 ? 0xffff0000u : 0xffffu) : 0u;
      const floatx4 sum = mfma16x16x32(as_bf16x8(v & keep), as_bf16x8(pop & keep), o);
      if (seen >> k & 1u) o = sum;
    }
  }
  return o;
}

// Which block of rows and head workgroup i takes. Workgroups are dealt to the 8 XCDs round robin: runs of consecutive blocks of a
// head, which read the same keys, go to one XCD and its L2. Runs of kRun in `order`, or of kLongRun, the latest tokens' first (256
// prompts of 32 .. 480 tokens, window 512: single blocks 181 us, runs of 4 178, 8 174, 16 174; of 256 each 177, 171, 149, 151).
constexpr int kXcds = 8, kRun = 4, kLongRun = 8;
__device__ __forceinline__ void place_block(int i, int n_blk, int H, const int32_t* order, int& blk, int& h) {
  const int each = order ? kRun : kLongRun;
  const int even = n_blk * H / (kXcds * each) * (kXcds * each);  // as many as fill whole turns of runs
  int u = i;
  if (i < even) {
    const int x = i % kXcds, j = i / kXcds;
    u = ((j / each) * kXcds + x) * each + j % each;
  }
  // u in the order (run of blocks, head, block of the run); the last run may be short
  const int run = u / (each * H), rest = u - run * each * H, len = min(each, n_blk - run * each);
  h = rest / len;
  blk = n_blk - 1 - ((order && len == each ? order[run] : run) * each + rest - h * len);
}

// Where few blocks would leave CUs idle for long, a block's chunks are taken in pieces, a workgroup each, whose sums a second
// launch joins; a block that has chunks for one piece only writes its result itself.
constexpr int kMostPieces = 16;
struct Piece {
  float m, l;    // row maximum in use, less the origin; sum
  int pieces;    // of the row's block (in piece 0's; 1: nothing to join)
  float origin;
};
struct Pieces {
  float* o;      // [most][H][padded rows][D], not divided by the sums
  Piece* stats;  // [most][H][padded rows]
  int most, chunks;  // pieces of a block at most; chunks of each, the last's maybe more
  int32_t* order;    // [blocks / kRun] the runs of blocks in the order that they are taken; NULL: the latest first
};

// The runs of blocks by the chunks of their longest block, most first: the last workgroups to start are short ones (CUs at work for 71 %
// of the time on 3 prompts of up to 8191 tokens without it, 81 % with; 398 -> 368 us). By bins of 2^shift chunks, within one in any
// order, which no result depends on. One workgroup, 4 us with its launch. (By single blocks, whose neighbours then lie on other XCDs:
// 420 us.)
constexpr int kBins = 1024;
__global__ __launch_bounds__(kBins) void packed_order_kernel(G4PackedPrefillArgs a, Group group, int n_blk, int rows, int shift,
                                                             int32_t* order) {
  __shared__ int bins[kBins], sums[kBins / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, T = a.tokens, runs = n_blk / kRun;
  const auto bin = [&](int run) {  // a block's chunks: from its first token's first key to its last token
    int most = 0;
#pragma unroll
    for (int i = 0; i < kRun; ++i) {
      const int b = n_blk - 1 - run * kRun - i, t0 = group.token(b * rows), t1 = min(group.token(b * rows + rows - 1), T - 1);
      const int start = a.starts[t0], lo = max(start, a.window > 0 ? t0 - a.window + 1 : 0);
      most = max(most, start < 0 ? 0 : (t1 - lo) >> 5);
    }
    return kBins - 1 - min(most >> shift, kBins - 1);
  };
  bins[tid] = 0;
  __syncthreads();
  for (int run = tid; run < runs; run += kBins) atomicAdd(&bins[bin(run)], 1);
  __syncthreads();
  const int mine = bins[tid];
  int x = mine;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int y = __shfl_up(x, d, 64);
    x += lane >= d ? y : 0;
  }
  if (lane == 63) sums[wave] = x;
  __syncthreads();
  for (int i = 0; i < wave; ++i) x += sums[i];
  bins[tid] = x - mine;
  __syncthreads();
  for (int run = tid; run < runs; run += kBins) order[atomicAdd(&bins[bin(run)], 1)] = run;
}

// A step per chunk c: behind its barrier, which every wave's share of K(c) and V(c - 1) has landed before, K(c + 1) and V(c) are
// asked for; then the values of chunk c - 1, the scores of chunk c and their softmax. Of a workgroup that has the CU alone (head
// dim 512) the waves of the second half, which share the SIMDs with those of the first, take the softmax of chunk c - 1
// first: one runs MFMAs while the other runs vector work (8 x 4096 tokens of 8 heads 1098 us, 1112 without). ONE asks for K(c + 1)
// behind the scores of chunk c and for V(c) behind the values of chunk c - 1. Chunks of which a wave sees nothing it skips.
template <int D, bool BIG, bool CUT>
__global__ __launch_bounds__((BIG && D == 512 ? 512 : 256), 2) void packed_prefill_kernel(G4PackedPrefillArgs a, Group group,
                                                                                         Pieces pieces) {
  using S = Shape<D, BIG>;
  constexpr int NB = S::NB, NW = S::NW, KS = S::KS, VT = S::T;
  // K in slots 0 and 1, V^T in 2 and 3, chunk c in slot (c - c_begin) % 2 of its ring (ONE: K in 0, V^T in 1); read with
  // inline-assembly LDS reads only: the compiler adds no waits of its own for the DMAs in flight
  __shared__ __attribute__((aligned(1024))) unsigned char ring[S::SLOTS][S::CHUNK];
  __shared__ int2 spans[NW];

  const int R = a.group, H = a.kv_heads, T = a.tokens;
  const int n_blk = (int)(gridDim.x / (unsigned)(CUT ? H * pieces.most : H));
  const int piece = CUT ? (int)(blockIdx.x / (unsigned)(n_blk * H)) : 0;
  int blk, h;
  place_block((int)blockIdx.x - piece * n_blk * H, n_blk, H, CUT ? nullptr : pieces.order, blk, h);
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row0 = blk * S::ROWS + w * (NB * 16);

  Rows rows{{}, 0x7fffffff, -1, {0, 0}, {0x7fffffff, 0x7fffffff}};
  bf16x8 qop[NB][KS];
  int token[NB], start[NB];
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    token[cb] = group.token(row0 + cb * 16 + col);
    start[cb] = a.starts[min(token[cb], T - 1)];
  }
  __builtin_amdgcn_sched_barrier(0);  // the starts are asked for, and so arrive, before q
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    // rows behind the last token read the last row and are not stored; flat over (t, r) of a head
    const int64_t at = (int64_t)min(row0 + cb * 16 + col, T * R - 1);
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (at + ((int64_t)min(token[cb], T - 1) * (H - 1) + h) * R) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) qop[cb][s] = as_bf16x8(load16(q + 32 * s + 8 * grp));
  }
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    const int t = token[cb];
    const bool has_keys = t < T && start[cb] >= 0 && start[cb] <= t;
    const int lo = has_keys ? max(start[cb], a.window > 0 ? t - a.window + 1 : 0) : 0, hi = has_keys ? t : -1;
    rows.keys[cb] = make_int2(lo, hi);
    if (has_keys) {
      rows.first = min(rows.first, lo);
      rows.last = max(rows.last, hi);
      rows.all_from[cb] = lo;
      rows.all_to[cb] = hi;
    }
  }
  const auto least = [](int x, int y) { return min(x, y); };
  const auto most = [](int x, int y) { return max(x, y); };
  rows.first = columns_reduce(rows.first, least);
  rows.last = columns_reduce(rows.last, most);
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    rows.all_from[cb] = columns_reduce(rows.all_from[cb], most);
    rows.all_to[cb] = columns_reduce(rows.all_to[cb], least);
  }
  if (lane == 0) spans[w] = make_int2(rows.first, rows.last);
  wg_barrier();  // (q is still on its way)
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < NW; ++i) first = min(first, spans[i].x), last = max(last, spans[i].y);
  // chunks c_begin .. c_end (none: c_begin > c_end); keys < T <= k_stride
  int c_begin = __builtin_amdgcn_readfirstlane(first) >> 5, c_end = __builtin_amdgcn_readfirstlane(last) >> 5;
  int n_pieces = 1;
  if constexpr (CUT) {
    n_pieces = c_begin > c_end ? 1 : min((c_end - c_begin) / pieces.chunks + 1, pieces.most);
    if (piece >= n_pieces) return;  // (the whole workgroup)
    c_begin += piece * pieces.chunks;
    if (piece < n_pieces - 1) c_end = c_begin + pieces.chunks - 1;  // (the last takes what is left)
    rows.first = max(rows.first, c_begin << 5);
    rows.last = min(rows.last, (c_end << 5) + 31);
  }

  const int64_t plane = (int64_t)h * a.k_stride * D;
  const __amdgpu_buffer_rsrc_t rk = make_rsrc(reinterpret_cast<const uint16_t*>(a.k) + plane, (uint32_t)a.k_stride * D * 2u);
  const __amdgpu_buffer_rsrc_t rv = make_rsrc(reinterpret_cast<const uint16_t*>(a.vt) + plane, (uint32_t)a.k_stride * D * 2u);
  const uint32_t k_lane = (uint32_t)(col * 64 + grp * 16), v_lane = vt_operand_bytes(grp, col, D);
  auto issue_k = [&](int c, int slot) {
#pragma unroll
    for (int i = 0; i < S::TW; ++i) {
      const int t = w * S::TW + i, bb = t / KS, s = t - bb * KS;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void*)&ring[slot][1024 * t], 16, k_lane,
                                               (uint32_t)c * (uint32_t)(64 * D) + (uint32_t)(2 * s + bb) * 1024u, 0, 0);
    }
  };
  auto issue_v = [&](int c, int slot) {
#pragma unroll
    for (int i = 0; i < S::TW; ++i) {
      const int t = w * S::TW + i;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void*)&ring[slot][1024 * t], 16, v_lane,
                                               (uint32_t)c * (uint32_t)(64 * D) + 256u * t, 0, 0);
    }
  };
  const uint32_t ring0 = lds_addr(&ring[0][0]) + 16u * (uint32_t)lane;  // this lane's piece of a tile

  floatx4 oacc[NB][VT];
  Softmax<NB, VT> soft;
  soft.init();
#pragma unroll
  for (int cb = 0; cb < NB; ++cb)
#pragma unroll
    for (int i = 0; i < VT; ++i) oacc[cb][i] = floatx4{0.f, 0.f, 0.f, 0.f};

  if (c_begin <= c_end) {  // (uniform over the workgroup)
    const bool late = NW == 8 && w >= NW / 2;
    floatx4 acc[NB][2];
    bf16x8 pop[NB];
    issue_k(c_begin, 0);
    // the q operands have landed here, not inside the loop, where their wait would drain the DMAs in flight
#pragma unroll
    for (int cb = 0; cb < NB; ++cb)
#pragma unroll
      for (int s = 0; s < KS; ++s) {
        u32x4 v = __builtin_bit_cast(u32x4, qop[cb][s]);
        __asm__ volatile("" : "+v"(v));
        qop[cb][s] = as_bf16x8(v);
      }
    if constexpr (S::ONE) {
#pragma unroll 1
      for (int c = c_begin; c <= c_end; ++c) {
        const bool now = rows.any(c), more = c < c_end;
        wait_vmcnt<0>();
        wg_barrier();  // K(c) is there, V(c - 1) done with
        issue_v(c, 1);
        if (now) pf_qk<VT, KS, NB, 4>(ring0, qop, acc);
        if (more) {
          wg_barrier();  // K(c) is done with
          issue_k(c + 1, 0);
        }
        if (now) soft.chunk(rows, c, lane, acc, pop, oacc);
        if (more) wait_vmcnt<S::TW>();
        else wait_vmcnt<0>();
        wg_barrier();  // V(c) is there
        if (now) pf_pv<VT, NB, 4>(ring0 + (uint32_t)S::CHUNK, pop, oacc);
      }
    } else {
#pragma unroll 1
      for (int c = c_begin, i = 0; c <= c_end; ++c, ++i) {
        wait_vmcnt<0>();
        wg_barrier();
        if (c + 1 <= c_end) issue_k(c + 1, (i + 1) & 1);
        issue_v(c, 2 + (i & 1));
        const bool before = c > c_begin && rows.any(c - 1), now = rows.any(c);
        if (late && before) soft.chunk(rows, c - 1, lane, acc, pop, oacc);
        if (before) pf_pv<VT, NB, 4>(ring0 + (uint32_t)((2 + ((i - 1) & 1)) * S::CHUNK), pop, oacc);
        if (now) pf_qk<VT, KS, NB, 4>(ring0 + (uint32_t)((i & 1) * S::CHUNK), qop, acc);
        if (!late && now) soft.chunk(rows, c, lane, acc, pop, oacc);
      }
      wait_vmcnt<0>();
      wg_barrier();
      if (rows.any(c_end)) {
        if (late) soft.chunk(rows, c_end, lane, acc, pop, oacc);
        pf_pv<VT, NB, 4>(ring0 + (uint32_t)((2 + ((c_end - c_begin) & 1)) * S::CHUNK), pop, oacc);
      }
    }
  }

  if (CUT && n_pieces > 1) {  // what this piece's keys give, for the join
    const int64_t base = ((int64_t)piece * H + h) * ((int64_t)n_blk * S::ROWS) + row0;
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) {
      float l = column_sum(soft.l[cb]);
      if (rows.keys[cb].y < 0) l = 0.f;  // (chunks that all other rows see whole were not masked)
      const int64_t row = base + cb * 16 + col;
      if (grp == 0) pieces.stats[row] = Piece{soft.m[cb], l, n_pieces, soft.origin[cb]};
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < VT; ++i) {
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = fmaf(oacc[cb][i][e], 0.f, sum);
        *reinterpret_cast<floatx4*>(pieces.o + row * D + 16 * i + 4 * grp) = oacc[cb][i];
      }
      if (__any(!(sum == 0.f))) {
        const int g = min(row0 + cb * 16 + col, T * R - 1), t = group.token(g);
        const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (((int64_t)t * H + h) * R + (g - t * R)) * D;
#pragma unroll 1
        for (int i = 0; i < VT; ++i)
          *reinterpret_cast<floatx4*>(pieces.o + row * D + 16 * i + 4 * grp) = careful_values<D>(rows, cb, soft.origin[cb], soft.base(cb), q, rk, rv, i);
      }
    }
    return;
  }
  // The result through LDS (the rings are done with), where the lanes' 4-dim pieces become whole rows: 16 bytes a lane,
  // a row's 16-byte units turned by its number so that neither side meets a bank twice. The rows' places are computed afresh (the
  // lane is hidden from the compiler), not kept in registers since the q loads.
  constexpr int UNITS = D / 8, RPI = 64 / UNITS;  // 16-byte units of a row, rows per store instruction
  wg_barrier();
  unsigned char* mine = &ring[0][0] + w * (NB * 16 * D * 2);
  int lane_o = lane;
  __asm__ volatile("" : "+v"(lane_o));
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    const float l = column_sum(soft.l[cb]);
    const int row = row0 + cb * 16 + (lane_o & 15), t = group.token(row);
    if (CUT && lane_o < 16) pieces.stats[(int64_t)h * ((int64_t)n_blk * S::ROWS) + row] = Piece{0.f, 0.f, 1, 0.f};  // nothing to join
    const bool none = rows.keys[cb].y < 0 || l == 0.f;
    const float inv = none ? 0.f : 1.0f / l;
    const auto pack = [&](floatx4 x) {
      x = none ? floatx4{0.f, 0.f, 0.f, 0.f} : x * inv;
      return make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    };
    const auto store = [&](int i, uint2 x) {
      const int r = lane_o & 15, unit = (2 * i + (lane_o >> 5)) ^ (r & (UNITS - 1));
      *reinterpret_cast<uint2*>(mine + (cb * 16 + r) * (D * 2) + unit * 16 + (lane_o >> 4 & 1) * 8) = x;
    };
    float sum = 0.f;  // not 0 where an element is not finite: 0 x is 0 or NaN
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      const uint2 x = pack(oacc[cb][i]);
      const bf16x2_t zero = {0, 0};
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x.x), zero, sum, false);
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, x.y), zero, sum, false);
      store(i, x);
    }
    if (__any(!(sum == 0.f))) {
      const uint16_t* q = t < T ? reinterpret_cast<const uint16_t*>(a.q) + (((int64_t)t * H + h) * R + (row - t * R)) * D : nullptr;
#pragma unroll 1
      for (int i = 0; i < VT; ++i) store(i, pack(careful_values<D>(rows, cb, soft.origin[cb], soft.base(cb), q, rk, rv, i)));
    }
    __builtin_amdgcn_wave_barrier();  // (a wave's rows are its own: its LDS operations keep their order)
#pragma unroll
    for (int i = 0; i < 16 / RPI; ++i) {
      const int r = i * RPI + lane_o / UNITS, unit = lane_o % UNITS;
      const int to = __shfl(t, r, 64), g = row0 + cb * 16 + r;
      const u32x4 x = *reinterpret_cast<const u32x4*>(mine + (cb * 16 + r) * (D * 2) + (unit ^ (r & (UNITS - 1))) * 16);
      if (to < T)
        __builtin_nontemporal_store(x, reinterpret_cast<u32x4*>(reinterpret_cast<uint16_t*>(a.out) +
                                                                 (((int64_t)to * H + h) * R + (g - to * R)) * D + unit * 8));
    }
  }
}

// A row's result from its pieces', one wave per row: each piece's sums weigh exp(its maximum - the largest).
template <int D>
__global__ __launch_bounds__(256) void packed_join_kernel(G4PackedPrefillArgs a, Group group, Pieces pieces, int64_t padded) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63, H = a.kv_heads, R = a.group;
  const int64_t i = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6), rows = (int64_t)a.tokens * R;
  if (i >= rows * H) return;
  const int h = (int)(i / rows), row = (int)(i - h * rows);
  const int n = __builtin_amdgcn_readfirstlane(pieces.stats[h * padded + row].pieces);  // (one row per wave)
  if (n <= 1) return;
  Piece p{kNegInf, 0.f, 0, 0.f};
  if (lane < n) p = pieces.stats[((int64_t)lane * H + h) * padded + row];
  const bool none = p.l == 0.f;  // (a row of no sequence, no key of the row here, or scores of -inf alone)
  const float m = p.origin - wave_max(none ? kNegInf : p.origin) + p.m;  // (origins are maxima: one with weight is next to the largest)
  const float top = wave_max(none ? kNegInf : m);
  const float weight = none ? 0.f : __builtin_amdgcn_exp2f((m - top) * kLog2e);
  const float l = wave_sum(none ? 0.f : weight * p.l);
  const bool some = __any(!none);
  float o[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = 0.f;
#pragma unroll 1
  for (int s = 0; s < n; s += 4) {  // four loads in flight
    float x[4][PER];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      __builtin_memcpy(x[j], __builtin_assume_aligned(pieces.o + (((int64_t)min(s + j, n - 1) * H + h) * padded + row) * D + lane * PER,
                                                      PER * 4 < 16 ? PER * 4 : 16), PER * 4);  // (the workspace: 16 bytes)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (s + j >= n) break;
      const float w = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, weight), s + j));
#pragma unroll
      for (int e = 0; e < PER; ++e) o[e] = fmaf(w, x[j][e], o[e]);
    }
  }
  const float inv = some ? 1.0f / l : 0.f;
  const int t = group.token(row);
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (((int64_t)t * H + h) * R + (row - t * R)) * D + lane * PER;
#pragma unroll
  for (int e = 0; e < PER; ++e) o[e] = some ? o[e] * inv : 0.f;
  if constexpr (PER == 1) {
    *out = (uint16_t)f32_to_bf16_bits(o[0]);
  } else {
    uint32_t x[PER / 2];
#pragma unroll
    for (int e = 0; e < PER / 2; ++e) x[e] = pack_bf16x2(o[2 * e], o[2 * e + 1]);
    __builtin_memcpy(__builtin_assume_aligned(out, PER * 2), x, PER * 2);
  }
}

// How a call is laid out. Blocks of 64 rows where those of 128 would leave CUs without a workgroup: more, smaller workgroups then end
// sooner (one prompt of 500 tokens, 2 x 4 heads of 256: 16 us, 23 of 128). Between one and two of 128 per CU these are all
// at work at once, which is faster where their keys are about as many (8000 tokens with window 1024: 76 us, 94 in twice as many of
// 64; 8 prompts of 1000 52 and 58) and slower where a few have most (one of 8000 300 and 267). Head dim 512, whose blocks of 64 share
// a CU and those of 128 do not: of 64 up to two of 128 per CU (8 heads: 500 tokens 26 and 32 us, 2 prompts of 1200 and 2000 83 and
// 94), beyond that the keys' second way through the L2 costs more (8000 tokens of 2 x 8 heads 963 and 924).
// Pieces: only where whole blocks leave CUs free and the longest sequence has 768 tokens (one of 600, 4 x 4 heads of 128: 15.6
// us in pieces, 13.4 whole; of 1000, 2 x 4 of 256, 23 and 28) that a window does not cut (4000 with window 512: 53 and 26).
// As many as the CUs take at once, of 8 chunks or more: each piece's sums cost a pass through memory (one prompt of 2000, 2
// x 4 heads of 256: whole 50, in 2 pieces 41, in 4 46 us; 1 head: whole 48, 8 pieces 20). Where the pieces stay long, of 32
// chunks or more, twice that, as the blocks with the most keys come first and the rest fill up behind them (one of 8000, 1
// x 2 heads of 128: whole 128, 2 pieces 81, 4 66; one of 4000, 8 heads of 512: whole 198, 2 pieces 163, in blocks of 128).
// Sorting: more blocks than are at work at once, whose keys may differ (no window that makes them alike), the longest of them long beside
// the rounds that all take (8 prompts of 4096, 2 x 4 heads of 256: 504 -> 450 us; 30 of 100 .. 900 72 -> 60; 64 of 32 .. 1000 136 -> 129).
// Else the end weighs little, and the launch and the keys that neighbours no longer share cost more (256 of 32 .. 480 188 -> 190, 512
// of them 337 -> 358, before runs of 8 blocks went to an XCD: unsorted 173 and 328 since). Where the longest is not known up to four
// rounds are sorted. "At work at once" is two workgroups per CU, of 128 rows at head dim 512 one, as 256 and 512 hold them, at which nearly
// all of this was measured. At 64 and 128 more fit (at 128 three of 128 rows, four of 64), which the rules do not count: grids of these
// are sorted, or left whole, that the CUs would take at once.
struct Plan {
  bool big;                // Shape's
  int most, chunks;        // pieces of a block at most (1: whole blocks), chunks of one
  int64_t blocks, padded;  // workgroups without pieces; rows per head, the last block's filled up
  bool sort;               // the runs of blocks by their chunks
};
Plan plan_of(const G4PackedPrefillArgs& a) {
  const int64_t rows = (int64_t)a.tokens * a.group;
  const auto per_head = [&](bool big) { return (rows + (big ? 127 : 63)) / (big ? 128 : 64); };
  Plan p{};
  const int64_t longest = a.longest > 0 && a.longest < a.tokens ? a.longest : a.tokens, chunks = (longest + 31) / 32;
  const bool cut = a.window > 0 && a.window < longest, alike = cut || longest * 4 < a.tokens;
  p.big = per_head(true) * a.kv_heads > (a.head_dim != 512 && alike ? 256 : 512);
  const int64_t resident = a.head_dim == 512 && p.big ? 256 : 512;
  p.blocks = per_head(p.big) * a.kv_heads;
  p.padded = per_head(p.big) * (p.big ? 128 : 64);
  p.most = 1;
  if (!p.big && p.blocks < resident && chunks >= 24 && !cut) {
    const int64_t most = std::min<int64_t>(kMostPieces, std::max(std::min(resident / p.blocks, chunks / 8),
                                                                std::min(2 * resident / p.blocks, chunks / 32)));
    if (most > 1) {
      p.chunks = (int)((chunks + most - 1) / most);
      p.most = (int)((chunks + p.chunks - 1) / p.chunks);
    }
  }
  p.sort = p.most == 1 && p.blocks > resident && p.blocks >= 2 * kRun * (int64_t)a.kv_heads && chunks >= 8 && !cut &&
           (a.longest > 0 ? chunks : std::min<int64_t>(chunks, 24)) * resident >= 6 * p.blocks;
  return p;
}

size_t carve(Pieces& p, void* base, const G4PackedPrefillArgs& a, const Plan& plan) {
  const int64_t rows = (int64_t)plan.most * a.kv_heads * plan.padded;
  p.most = plan.most;
  p.chunks = plan.chunks;
  p.o = static_cast<float*>(base);
  p.stats = reinterpret_cast<Piece*>(p.o + rows * a.head_dim);
  p.order = plan.sort ? static_cast<int32_t*>(base) : nullptr;
  if (plan.sort) return (size_t)(plan.blocks / a.kv_heads / kRun) * 4;
  return plan.most > 1 ? (size_t)rows * (a.head_dim * 4 + sizeof(Piece)) : 0;
}

template <int D, bool BIG>
int launch_packed(const G4PackedPrefillArgs& a, const Plan& plan, const Pieces& pieces, hipStream_t st) {
  static const char who[] = "g4_packed_prefill_attention";
  using S = Shape<D, BIG>;
  const int64_t blocks = plan.blocks * plan.most;
  const Group group(a.group);
  if (plan.most == 1) {
    if (plan.sort) {
      int shift = 0;
      while (a.tokens >> 5 >> shift >= kBins) ++shift;
      hipLaunchKernelGGL(packed_order_kernel, dim3(1), dim3(kBins), 0, st, a, group, (int)(blocks / a.kv_heads), S::ROWS, shift,
                         pieces.order);
      const int rc = check_launch(who);
      if (rc != G4_OK) return rc;
    }
    hipLaunchKernelGGL((packed_prefill_kernel<D, BIG, false>), dim3((unsigned)blocks), dim3(S::NW * 64), 0, st, a, group, pieces);
    return check_launch(who);
  }
  if constexpr (!BIG) {
    hipLaunchKernelGGL((packed_prefill_kernel<D, false, true>), dim3((unsigned)blocks), dim3(S::NW * 64), 0, st, a, group, pieces);
    const int rc = check_launch(who);
    if (rc != G4_OK) return rc;
    const int64_t rows = (int64_t)a.tokens * a.group * a.kv_heads;
    hipLaunchKernelGGL(packed_join_kernel<D>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, a, group, pieces, plan.padded);
  }
  return check_launch(who);
}
template <int D>
int launch_packed(const G4PackedPrefillArgs& a, const Plan& plan, const Pieces& pieces, hipStream_t st) {
  return plan.big ? launch_packed<D, true>(a, plan, pieces, st) : launch_packed<D, false>(a, plan, pieces, st);
}

// starts[t]: the first token of t's sequence, -1 behind the last sequence. One thread per token, a binary search.
__global__ __launch_bounds__(256) void packed_starts_kernel(const int32_t* cu, int n, int tokens, int32_t* starts) {
  const int t = (int)(blockIdx.x * 256u + threadIdx.x);
  if (t >= tokens) return;
  int lo = 0, hi = n + 1;  // the first of cu[0 .. n] beyond t
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] > t) hi = mid;
    else lo = mid + 1;
  }
  starts[t] = lo == 0 || lo == n + 1 ? -1 : cu[lo - 1];
}

}  // namespace
}  // namespace g4

extern "C" int g4_packed_starts(int32_t sequences, const int32_t* cu_seqlens, int32_t tokens, int32_t* starts, void* stream) {
  using namespace g4;
  if (sequences <= 0 || sequences == 0x7fffffff || tokens <= 0 || tokens > 0x7fffffff - 256 || !cu_seqlens || !starts)
    return fail(G4_ERR_INVALID, "g4_packed_starts: %d sequences, %d tokens%s", sequences, tokens,
                cu_seqlens && starts ? "" : ", NULL pointer");
  hipLaunchKernelGGL(packed_starts_kernel, dim3((unsigned)((tokens + 255) / 256)), dim3(256), 0,
                     reinterpret_cast<hipStream_t>(stream), cu_seqlens, sequences, tokens, starts);
  return check_launch("g4_packed_starts");
}

extern "C" int g4_packed_prefill_attention(const G4PackedPrefillArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_packed_prefill_attention";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PackedPrefillArgs& a = *args;
  if (a.tokens <= 0 || a.kv_heads <= 0 || a.group <= 0 || a.window < 0 || a.longest < 0)
    return fail(G4_ERR_INVALID, "%s: tokens %d, kv_heads %d, group %d must be positive, window %d, longest %d not negative", who,
                a.tokens, a.kv_heads, a.group, a.window, a.longest);
  if (a.head_dim != 64 && a.head_dim != 128 && a.head_dim != 256 && a.head_dim != 512)
    return fail(G4_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128, 256 or 512)", who, a.head_dim);
  if (a.group > 64) return fail(G4_ERR_UNSUPPORTED, "%s: group %d (at most 64)", who, a.group);
  if (a.k_stride < a.tokens || a.k_stride % 64)
    return fail(G4_ERR_INVALID, "%s: k_stride %d (need >= tokens, multiple of 64)", who, a.k_stride);
  if (!a.starts || !a.q || !a.k || !a.vt || !a.out) return fail(G4_ERR_INVALID, "%s: NULL pointer", who);
  if (((uintptr_t)a.q | (uintptr_t)a.k | (uintptr_t)a.vt | (uintptr_t)a.out) % 16)
    return fail(G4_ERR_INVALID, "%s: q / k / vt / out must be 16-byte aligned", who);
  // a head's keys are addressed by 32-bit byte offsets, rows by 32-bit indexes
  if ((int64_t)a.k_stride * a.head_dim * 2 > 0xffffffffLL || (int64_t)a.tokens * a.group > 0x7fffffffLL - 1024)
    return fail(G4_ERR_UNSUPPORTED, "%s: too many tokens (%d of %d x %d rows of %d)", who, a.tokens, a.kv_heads, a.group, a.head_dim);
  const Plan plan = plan_of(a);
  if (plan.blocks * plan.most * (a.head_dim == 512 && plan.big ? 512 : 256) > 0xffffffffLL)
    return fail(G4_ERR_UNSUPPORTED, "%s: too many tokens (%d of %d heads)", who, a.tokens, a.kv_heads);
  Pieces pieces;
  const size_t need = carve(pieces, a.workspace, a, plan);
  if (need && (!a.workspace || a.workspace_bytes < need))
    return fail(G4_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a.workspace ? a.workspace_bytes : 0, need);
  if (need && (uintptr_t)a.workspace % 16) return fail(G4_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a.head_dim) {
    case 64: return launch_packed<64>(a, plan, pieces, st);
    case 128: return launch_packed<128>(a, plan, pieces, st);
    case 256: return launch_packed<256>(a, plan, pieces, st);
    default: return launch_packed<512>(a, plan, pieces, st);
  }
}

extern "C" size_t g4_packed_prefill_workspace_size(const G4PackedPrefillArgs* args) {
  using namespace g4;
  if (!args || args->tokens <= 0 || args->kv_heads <= 0 || args->group <= 0 || args->group > 64 || args->head_dim <= 0) return 0;
  Pieces pieces;
  return carve(pieces, nullptr, *args, plan_of(*args));
}
