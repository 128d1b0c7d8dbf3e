// Causal attention of packed prompts (g4_packed_prefill_attention): sequences of any lengths one behind the other,
// without pads, each token over its own sequence's tokens up to itself, optionally the last `window` of them. The
// scores and the softmax of model.py:320-335, 496-499 per sequence.
//
// The query rows of one kv head are the (token, r) pairs in order, T R of them; a workgroup takes the next
// NW * NB * 16, whatever sequences they belong to, and walks the 32-key chunks from the first key that one of them
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
#include "g4_attn_tiles.h"
#include "g4_common.h"
#include "g4_internal.h"

namespace g4 {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();
constexpr float kSlack = 8.0f;

template <int D, int NB_, int NW_>
struct Shape {
  static constexpr int NB = NB_, NW = NW_;
  static constexpr int KS = D / 32;
  static constexpr int T = D / 16;                  // 1 KiB operand tiles of a chunk's K and of its V^T
  static constexpr int SLOTS = D == 512 ? 2 : 4;    // chunks of each in LDS
  static constexpr int CHUNK = T * 1024;
  static constexpr int TW = T / NW;                 // tiles that a wave fetches of each
  static constexpr int ROWS = NW * NB * 16;         // query rows of a workgroup
  static_assert(T % NW == 0, "the waves share the tiles evenly");
};

__device__ __forceinline__ int wave_min(int v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = min(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int m = 32; m; m >>= 1) v = max(v, __shfl_xor(v, m, 64));
  return v;
}
__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The keys [lo, hi] of the wave's rows: this lane's, and over all rows of the wave that have any.
template <int NB>
struct Rows {
  int lo[NB], hi[NB];
  int first, last;            // the keys that some row sees lie in [first, last]
  int all_from, all_to;       // every row sees [all_from, all_to]
  __device__ __forceinline__ bool any(int c) const { return (c << 5) + 31 >= first && (c << 5) <= last; }
  __device__ __forceinline__ bool full(int c) const { return (c << 5) >= all_from && (c << 5) + 31 <= all_to; }
  // bit e <-> key 32 c + 8 grp + e
  __device__ __forceinline__ uint32_t bits(int c, int grp, int cb) const {
    const int k = (c << 5) + 8 * grp;
    const int from = min(max(lo[cb] - k, 0), 8), to = min(max(hi[cb] - k + 1, 0), 8);  // elements [from, to)
    return (0xffu << from) & ((1u << to) - 1u);
  }
};

// Softmax of one chunk's scores: `p` as the value product's operand, the row statistics brought forward.
template <int NB, int VT>
struct Softmax {
  float m[NB], ml[NB], l[NB];  // row maximum in use, the same times log2(e), this lane's share of the sum

  __device__ __forceinline__ void init() {
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) m[cb] = kNegInf, ml[cb] = 0.f, l[cb] = 0.f;
  }

  __device__ __forceinline__ void chunk(const Rows<NB>& rows, int c, int grp, floatx4 (&acc)[NB][2], bf16x8 (&pop)[NB],
                                        floatx4 (&oacc)[NB][VT]) {
    if (!rows.full(c)) {
#pragma unroll
      for (int cb = 0; cb < NB; ++cb) {
        const uint32_t bits = rows.bits(c, grp, cb);
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[cb][e >> 2][e & 3] = bits >> e & 1u ? acc[cb][e >> 2][e & 3] : kNegInf;
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
#pragma unroll
      for (int cb = 0; cb < NB; ++cb) {
        const float next = fmaxf(m[cb], column_max(top[cb]));
        // (before the first key m = -inf: nothing to scale yet)
        const float scale = next > m[cb] ? __builtin_amdgcn_exp2f((m[cb] - next) * kLog2e) : 1.f;
        m[cb] = next;
        ml[cb] = next == kNegInf ? 0.f : next * kLog2e;
        l[cb] *= scale;
#pragma unroll
        for (int i = 0; i < VT; ++i) oacc[cb][i] *= scale;
      }
    }
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) {
      float p[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        p[e] = __builtin_amdgcn_exp2f(fmaf(acc[cb][e >> 2][e & 3], kLog2e, -ml[cb]));
        sum += p[e];
      }
      l[cb] += sum;
      pop[cb] = as_bf16x8(pack8(p));
    }
  }
};

// The values of one column block again, chunk by chunk from memory, with the final row maximum: a chunk whose values
// are not all finite key by key, so that a row takes only those that it sees. For waves that met such values; speed
// does not matter.
template <int D, int NB>
__device__ __forceinline__ void careful_values(const Rows<NB>& rows, int cb, float ml, const bf16x8 (&qop)[D / 32],
                                               __amdgpu_buffer_rsrc_t rk, __amdgpu_buffer_rsrc_t rv,
                                               floatx4 (&oacc)[D / 16]) {
  constexpr int KS = D / 32, VT = D / 16;
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const uint32_t k_lane = (uint32_t)(col * 64 + grp * 16), v_lane = vt_operand_bytes(grp, col, D);
#pragma unroll
  for (int i = 0; i < VT; ++i) oacc[i] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
  for (int c = rows.first >> 5; c << 5 <= rows.last; ++c) {
    floatx4 acc[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int t = 0; t < 2 * KS; ++t) {
      const u32x4 k = buffer_load16(rk, k_lane, (uint32_t)c * (uint32_t)(64 * D) + (uint32_t)(2 * (t % KS) + t / KS) * 1024u);
      acc[t / KS] = mfma16x16x32(as_bf16x8(k), qop[t % KS], acc[t / KS]);
    }
    uint32_t seen = 0;  // bit k <-> key 32 c + k
#pragma unroll
    for (int g = 0; g < 4; ++g) seen |= rows.bits(c, g, cb) << (8 * g);
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e)
      p[e] = seen >> (8 * grp + e) & 1u ? __builtin_amdgcn_exp2f(fmaf(acc[e >> 2][e & 3], kLog2e, -ml)) : 0.f;
    const u32x4 pop = pack8(p);
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      const u32x4 v = buffer_load16(rv, v_lane, (uint32_t)c * (uint32_t)(64 * D) + 256u * i);
      bool odd = false;
#pragma unroll
      for (int q = 0; q < 4; ++q) odd |= (v[q] & 0x7f80u) == 0x7f80u || (v[q] & 0x7f800000u) == 0x7f800000u;
      if (!__any(odd)) {
        oacc[i] = mfma16x16x32(as_bf16x8(v), as_bf16x8(pop), oacc[i]);
        continue;
      }
#pragma unroll 1
      for (int k = 0; k < 32; ++k) {  // this key alone
        u32x4 keep;
#pragma unroll
        for (int q = 0; q < 4; ++q) keep[q] = k >> 3 == grp && (k & 7) >> 1 == q ? (k & 1 ? 0xffff0000u : 0xffffu) : 0u;
        const floatx4 sum = mfma16x16x32(as_bf16x8(v & keep), as_bf16x8(pop & keep), oacc[i]);
        if (seen >> k & 1u) oacc[i] = sum;
      }
    }
  }
}

// Waves of the two halves of a workgroup (those that share a SIMD) are half a step apart, as in
// prefill_bf16_lds_kernel: one runs the MFMAs (the values of chunk c - 1, then the scores of chunk c), at raised
// priority, while the other runs the softmax of a chunk. Chunks of which a wave sees nothing it skips.
template <int D, int NB, int NW>
__global__ __launch_bounds__(NW * 64) void packed_prefill_kernel(G4PackedPrefillArgs a) {
  using S = Shape<D, NB, NW>;
  constexpr int KS = S::KS, VT = S::T, SLOTS = S::SLOTS;
  // read with inline-assembly LDS reads only: the compiler adds no waits of its own for the DMAs in flight
  __shared__ __attribute__((aligned(1024))) unsigned char ring[2 * SLOTS][S::CHUNK];
  __shared__ int2 spans[NW];

  const int R = a.group, H = a.kv_heads, T = a.tokens;
  const int n_blk = (int)(gridDim.x / (unsigned)H);
  // the latest tokens first, whose keys are the most
  const int blk = n_blk - 1 - (int)(blockIdx.x / (unsigned)H), h = (int)(blockIdx.x % (unsigned)H);
  const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int row0 = blk * S::ROWS + w * (NB * 16);

  Rows<NB> rows;
  bool row_ok[NB], has_keys[NB];
  bf16x8 qop[NB][KS];
  rows.first = 0x7fffffff, rows.last = -1, rows.all_from = 0, rows.all_to = 0x7fffffff;
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    const int row = row0 + cb * 16 + col, t = row / R;
    row_ok[cb] = t < T;
    const int start = row_ok[cb] ? a.starts[t] : -1;
    has_keys[cb] = start >= 0 && start <= t;
    rows.lo[cb] = has_keys[cb] ? max(start, a.window > 0 ? t - a.window + 1 : 0) : 0;
    rows.hi[cb] = has_keys[cb] ? t : -1;
    if (has_keys[cb]) {
      rows.first = min(rows.first, rows.lo[cb]);
      rows.last = max(rows.last, rows.hi[cb]);
      rows.all_from = max(rows.all_from, rows.lo[cb]);
      rows.all_to = min(rows.all_to, rows.hi[cb]);
    }
    const uint16_t* q = reinterpret_cast<const uint16_t*>(a.q) + (((int64_t)t * H + h) * R + (row - t * R)) * D;
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 v = {0u, 0u, 0u, 0u};
      if (has_keys[cb]) v = load16(q + 32 * s + 8 * grp);
      qop[cb][s] = as_bf16x8(v);
    }
  }
  rows.first = __builtin_amdgcn_readfirstlane(wave_min(rows.first));
  rows.last = __builtin_amdgcn_readfirstlane(wave_max(rows.last));
  rows.all_from = __builtin_amdgcn_readfirstlane(wave_max(rows.all_from));
  rows.all_to = __builtin_amdgcn_readfirstlane(wave_min(rows.all_to));
  // the q operands have landed here, not inside the loop, where their wait would drain the DMAs in flight
#pragma unroll
  for (int cb = 0; cb < NB; ++cb)
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      u32x4 v = __builtin_bit_cast(u32x4, qop[cb][s]);
      __asm__ volatile("" : "+v"(v));
      qop[cb][s] = as_bf16x8(v);
    }
  if (lane == 0) spans[w] = make_int2(rows.first, rows.last);
  __syncthreads();
  int first = 0x7fffffff, last = -1;
#pragma unroll
  for (int i = 0; i < NW; ++i) first = min(first, spans[i].x), last = max(last, spans[i].y);
  // chunks c_begin .. c_end (none: c_begin > c_end); keys < T <= k_stride
  const int c_begin = __builtin_amdgcn_readfirstlane(first) >> 5, c_end = __builtin_amdgcn_readfirstlane(last) >> 5;

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
    const bool lead = w < NW / 2;
    // chunk j sits in slot (j - c_begin) % SLOTS of both rings (V^T behind K); K(c) and V(c - 1) are read in step c
    // only, whose barrier queues K(c + SLOTS - 1) and V(c + SLOTS - 2) into the slots that step c - 1 finished reading
    auto wait_step = [&](int c) {
      constexpr int n = S::TW;
      if (SLOTS == 2) wait_vmcnt<0>();
      else if (c + 2 <= c_end) wait_vmcnt<4 * n>();
      else if (c + 1 <= c_end) wait_vmcnt<3 * n>();
      else wait_vmcnt<n>();
      wg_barrier();
    };
    floatx4 acc[NB][2];
    bf16x8 pop[NB];
    issue_k(c_begin, 0);
    if constexpr (SLOTS == 4) {
      if (c_begin + 1 <= c_end) issue_k(c_begin + 1, 1);
      issue_v(c_begin, SLOTS);
      if (c_begin + 2 <= c_end) issue_k(c_begin + 2, 2);
      if (c_begin + 1 <= c_end) issue_v(c_begin + 1, SLOTS + 1);
    }
#pragma unroll 1
    for (int c = c_begin, i = 0; c <= c_end; ++c, ++i) {
      wait_step(c);
      if (c + SLOTS - 1 <= c_end) issue_k(c + SLOTS - 1, (i + SLOTS - 1) & (SLOTS - 1));
      if (c + SLOTS - 2 <= c_end) issue_v(c + SLOTS - 2, SLOTS + ((i + SLOTS - 2) & (SLOTS - 1)));
      const bool before = c > c_begin && rows.any(c - 1), now = rows.any(c);
      if (!lead && before) soft.chunk(rows, c - 1, grp, acc, pop, oacc);
      __builtin_amdgcn_s_setprio(1);
      if (before) pf_pv<VT, NB, 4>(ring0 + (uint32_t)((SLOTS + ((i - 1) & (SLOTS - 1))) * S::CHUNK), pop, oacc);
      if (now) pf_qk<VT, KS, NB, 4>(ring0 + (uint32_t)((i & (SLOTS - 1)) * S::CHUNK), qop, acc);
      __builtin_amdgcn_s_setprio(0);
      if (lead && now) soft.chunk(rows, c, grp, acc, pop, oacc);
    }
    wait_vmcnt<0>();
    wg_barrier();
    if (rows.any(c_end)) {
      if (!lead) soft.chunk(rows, c_end, grp, acc, pop, oacc);
      pf_pv<VT, NB, 4>(ring0 + (uint32_t)((SLOTS + ((c_end - c_begin) & (SLOTS - 1))) * S::CHUNK), pop, oacc);
    }
  }

  const auto store = [&](int cb, const floatx4 (&o)[VT]) {
    const float l = column_sum(soft.l[cb]);
    const float inv = has_keys[cb] && l != 0.f ? 1.0f / l : 0.f;
    if (!row_ok[cb]) return;
    const int row = row0 + cb * 16 + col, t = row / R;
    uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (((int64_t)t * H + h) * R + (row - t * R)) * D;
#pragma unroll
    for (int i = 0; i < VT; ++i) {
      const floatx4 x = inv == 0.f ? floatx4{0.f, 0.f, 0.f, 0.f} : o[i] * inv;
      *reinterpret_cast<uint2*>(out + 16 * i + 4 * grp) = make_uint2(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]));
    }
  };
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) {
    float sum = 0.f;  // not finite where an accumulator is not: 0 x is 0 or NaN
#pragma unroll
    for (int i = 0; i < VT; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = fmaf(oacc[cb][i][e], 0.f, sum);
    if (__any(!(sum == 0.f))) careful_values<D, NB>(rows, cb, soft.ml[cb], qop[cb], rk, rv, oacc[cb]);
    store(cb, oacc[cb]);
  }
}

template <int D>
int launch_packed(const G4PackedPrefillArgs& a, hipStream_t st) {
  using S = Shape<D, D == 512 ? 1 : 2, D == 64 ? 4 : 8>;
  const int64_t blocks = ((int64_t)a.tokens * a.group + S::ROWS - 1) / S::ROWS * a.kv_heads;
  if (blocks * S::NW * 64 > 0xffffffffLL) return fail(G4_ERR_UNSUPPORTED, "g4_packed_prefill_attention: too many tokens");
  hipLaunchKernelGGL((packed_prefill_kernel<D, S::NB, S::NW>), dim3((unsigned)blocks), dim3(S::NW * 64), 0, st, a);
  return check_launch("g4_packed_prefill_attention");
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
  if (a.tokens <= 0 || a.kv_heads <= 0 || a.group <= 0 || a.window < 0)
    return fail(G4_ERR_INVALID, "%s: tokens %d, kv_heads %d, group %d must be positive, window %d not negative", who, a.tokens,
                a.kv_heads, a.group, a.window);
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
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a.head_dim) {
    case 64: return launch_packed<64>(a, st);
    case 128: return launch_packed<128>(a, st);
    case 256: return launch_packed<256>(a, st);
    default: return launch_packed<512>(a, st);
  }
}
