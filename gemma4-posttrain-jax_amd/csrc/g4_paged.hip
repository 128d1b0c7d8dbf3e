// The paged KV cache's writes and reads: g4_paged_append and g4_paged_read (g4_paged_decode.hip has the
// attention). No reference counterpart beyond the arithmetic of model.py:463-482, 368-390.
#include <initializer_list>

#include "g4_paged.h"

namespace g4 {

int check_paged_cache(const G4PagedCache& c, const char* who) {
  if (c.format != G4_PAGES_BF16 && c.format != G4_PAGES_E4M3) return fail(G4_ERR_INVALID, "%s: page format %d", who, c.format);
  if (c.num_pages <= 0 || c.kv_heads <= 0)
    return fail(G4_ERR_INVALID, "%s: num_pages %d / kv_heads %d must be positive", who, c.num_pages, c.kv_heads);
  if (c.head_dim != 64 && c.head_dim != 128 && c.head_dim != 256 && c.head_dim != 512)
    return fail(G4_ERR_UNSUPPORTED, "%s: head_dim %d (64, 128, 256 or 512)", who, c.head_dim);
  if (c.page_size < 32 || c.page_size > 1024 || (c.page_size & (c.page_size - 1)))
    return fail(G4_ERR_INVALID, "%s: page_size %d (a power of two, 32 .. 1024)", who, c.page_size);
  if (!c.key || !c.value) return fail(G4_ERR_INVALID, "%s: key / value pages are NULL", who);
  if (reinterpret_cast<uintptr_t>(c.key) % 16 || reinterpret_cast<uintptr_t>(c.value) % 16)
    return fail(G4_ERR_INVALID, "%s: key / value pages must be 16-byte aligned", who);
  if (c.format == G4_PAGES_E4M3) {
    if (!c.key_scale || !c.value_scale) return fail(G4_ERR_INVALID, "%s: e4m3 pages need key_scale / value_scale", who);
    if (reinterpret_cast<uintptr_t>(c.key_scale) % 8 || reinterpret_cast<uintptr_t>(c.value_scale) % 8)
      return fail(G4_ERR_INVALID, "%s: key_scale / value_scale must be 8-byte aligned", who);
  }
  return G4_OK;
}

int check_page_table(const int32_t* table, int32_t max_pages, int64_t table_stride, int32_t page_size, const char* who) {
  if (max_pages <= 0 || table_stride < max_pages || !table)
    return fail(G4_ERR_INVALID, "%s: page table (max_pages %d, table_stride %lld%s)", who, max_pages,
                (long long)table_stride, table ? "" : ", NULL");
  if ((int64_t)max_pages * page_size > 0x7fffffffLL - 1024)
    return fail(G4_ERR_UNSUPPORTED, "%s: %d pages of %d positions pass 2^31 positions", who, max_pages, page_size);
  return G4_OK;
}

namespace {

// --- append ------------------------------------------------------------------------------------------------
//
// A head vector is held by LANES = min(64, D / 4) lanes, so a wave has 64 / LANES of them at once; lane l of its
// group holds elements [l PER, (l + 1) PER), and a rotation's partner (d +- D / 2) is the same element of lane
// l ^ LANES / 2. f32 throughout, rounded once where it is stored: with i = (mean(x^2) + eps)^-1/2, c and s the
// rotary row and w the norm's weights,
//   y_d = i (x_d (w_d c_d) + x_(d +- D/2) (-+ w_(d +- D/2) s_d)),
// whose factors w c and w s are formed once per token for all its heads.

template <int D>
struct Lanes {
  static constexpr int LANES = D >= 256 ? 64 : D / 4;
  static constexpr int PER = D / LANES;     // 4, 8 at D = 512
  static constexpr int VECS = 64 / LANES;  // head vectors of a wave at once
  int in, sub;  // lane in its vector, vector of the wave
  __device__ __forceinline__ explicit Lanes(int lane) : in(lane % LANES), sub(lane / LANES) {}

  // Over the lanes of one vector, the result in each (every lane of the wave active).
  template <typename F>
  __device__ static __forceinline__ float reduce(float v, F op) {
    if constexpr (LANES >= 64) v = across32(v, op);
    if constexpr (LANES >= 32) v = across16(v, op);
    v = op(v, dpp<0x128>(v));    // row_ror:8
    v = op(v, dpp<0x124>(v));    // row_ror:4
    v = op(v, dpp<0x4e>(v));     // quad_perm:[2,3,0,1]
    return op(v, dpp<0xb1>(v));  // quad_perm:[1,0,3,2]
  }

  // The value of the partner lane in the vector's other half.
  __device__ __forceinline__ float partner(float x) const {
    const uint32_t u = __float_as_uint(x);
    if constexpr (LANES == 64) {
      const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
      return __uint_as_float(low() ? r[1] : r[0]);
    } else if constexpr (LANES == 32) {
      const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
      return __uint_as_float(low() ? r[1] : r[0]);
    } else {
      return dpp<0x128>(x);  // row_ror:8
    }
  }
  __device__ __forceinline__ bool low() const { return in < LANES / 2; }
};

// PER bf16 elements of a row, and the way back.
template <int PER>
__device__ __forceinline__ void load_row(const uint16_t* p, bool vec, float (&x)[PER]) {
  uint32_t w[PER / 2];
  if (vec) {
    __builtin_memcpy(w, __builtin_assume_aligned(p, PER * 2), PER * 2);
  } else {
#pragma unroll
    for (int i = 0; i < PER / 2; ++i) w[i] = p[2 * i] | (uint32_t)p[2 * i + 1] << 16;
  }
#pragma unroll
  for (int i = 0; i < PER / 2; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
template <int PER>
__device__ __forceinline__ void store_row(uint16_t* p, const float (&x)[PER]) {
  uint32_t w[PER / 2];
#pragma unroll
  for (int i = 0; i < PER / 2; ++i) w[i] = pack_bf16x2(x[2 * i], x[2 * i + 1]);
  __builtin_memcpy(__builtin_assume_aligned(p, PER * 2), w, PER * 2);
}

// What a token's q or k heads have in common.
template <int D>
struct Prepare {
  static constexpr int PER = Lanes<D>::PER;
  float own[PER], other[PER];  // factors of x_d and of its partner; other unused without rotation
  bool norm, rope;
  float eps;

  // weight: [D] or NULL; c, s: this lane's elements of the token's rotary row
  __device__ __forceinline__ void load(const uint16_t* weight, bool vec, const float (&c)[PER], const float (&s)[PER],
                                       const Lanes<D>& ln) {
#pragma unroll
    for (int e = 0; e < PER; ++e) own[e] = 1.f;
    if (weight) load_row<PER>(weight + ln.in * PER, vec, own);
    if (!rope) return;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const float partner = ln.partner(own[e]);
      other[e] = (ln.low() ? -partner : partner) * s[e];
      own[e] *= c[e];
    }
  }

  __device__ __forceinline__ void apply(float (&x)[PER], const Lanes<D>& ln) const {
    const float inv = norm ? inverse_rms(x, eps) : 1.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      float y = x[e] * own[e];
      if (rope) y += ln.partner(x[e]) * other[e];
      x[e] = norm ? y * inv : y;
    }
  }

  __device__ static __forceinline__ float inverse_rms(const float (&x)[PER], float eps) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) ss += x[e] * x[e];
    return __builtin_amdgcn_rsqf(Lanes<D>::reduce(ss, SumOp()) * (1.0f / D) + eps);
  }
};

// A vector's scale byte and its e4m3 bytes (this lane's in `w`).
template <int D>
__device__ __forceinline__ int quantise(const float (&x)[Lanes<D>::PER], uint32_t (&w)[Lanes<D>::PER / 4]) {
  constexpr int PER = Lanes<D>::PER;
  float a = 0.f;
  bool odd_one = false;
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    a = fmaxf(a, fabsf(x[e]));  // of the numbers
    odd_one |= !finite_f32(x[e]);
  }
  const bool odd_ones = __any(odd_one);
  if (odd_ones) {  // the largest of the finite elements
    a = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) a = fmaxf(a, finite_f32(x[e]) ? fabsf(x[e]) : 0.f);
  }
  const int byte = scale_byte(Lanes<D>::reduce(a, MaxOp()));
  const float inv = __uint_as_float((uint32_t)(2 * kScaleBias - byte) << 23);
#pragma unroll
  for (int i = 0; i < PER / 4; ++i) {
    uint32_t v = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i] * inv, x[4 * i + 1] * inv, 0, false);
    v = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2] * inv, x[4 * i + 3] * inv, (int)v, true);
    if (odd_ones) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (!finite_f32(x[4 * i + e])) v |= 0x7fu << (8 * e);  // NaN (either sign)
    }
    w[i] = v;
  }
  return byte;
}

template <int PER>
__device__ __forceinline__ void store_bytes(uint8_t* p, const uint32_t (&w)[PER / 4]) {
  __builtin_memcpy(__builtin_assume_aligned(p, PER), w, PER);
}

// The rotary rows and factors of one token.
template <int D>
struct Token {
  static constexpr int PER = Lanes<D>::PER;
  Prepare<D> q, k;
  bool norm_v;

  __device__ __forceinline__ void load(const G4PagedAppendArgs& a, int64_t token, bool vec, bool with_k, const Lanes<D>& ln) {
    float c[PER], s[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) c[e] = s[e] = 0.f;
    if (a.flags & (G4_APPEND_ROPE_Q | G4_APPEND_ROPE_K)) {
      __builtin_memcpy(c, a.rope_cos + token * D + ln.in * PER, PER * 4);
      __builtin_memcpy(s, a.rope_sin + token * D + ln.in * PER, PER * 4);
    }
    q.norm = a.flags & G4_APPEND_NORM_Q, q.rope = a.flags & G4_APPEND_ROPE_Q, q.eps = a.eps;
    k.norm = a.flags & G4_APPEND_NORM_K, k.rope = a.flags & G4_APPEND_ROPE_K, k.eps = a.eps;
    norm_v = a.flags & G4_APPEND_NORM_V;
    if (a.q) q.load(q.norm ? reinterpret_cast<const uint16_t*>(a.q_norm_weight) : nullptr, vec, c, s, ln);
    if (with_k) k.load(k.norm ? reinterpret_cast<const uint16_t*>(a.k_norm_weight) : nullptr, vec, c, s, ln);
  }

  __device__ __forceinline__ void prepare_v(float (&x)[PER], float eps) const {
    if (!norm_v) return;
    const float inv = Prepare<D>::inverse_rms(x, eps);
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] *= inv;
  }
};

// A prepared key or value vector into its slot (where `on`): keys in the page's runs, values one element per
// 8-slot group.
template <int D, bool F8, bool KEY>
__device__ __forceinline__ void store_vector(const G4PagedCache& c, int64_t block, int slot, const float (&x)[Lanes<D>::PER],
                                             bool on, const Lanes<D>& ln) {
  constexpr int PER = Lanes<D>::PER;
  uint8_t* pages = reinterpret_cast<uint8_t*>(KEY ? c.key : c.value) + block * D * (F8 ? 1 : 2);
  if constexpr (F8) {
    uint32_t w[PER / 4];
    const int byte = quantise<D>(x, w);
    if (!on) return;
    if (ln.in == 0) (KEY ? c.key_scale : c.value_scale)[block + slot] = (uint8_t)byte;
    if constexpr (KEY) {
      store_bytes<PER>(pages + paged_key_index<true>(slot, ln.in * PER, D), w);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) pages[vt_index(slot, ln.in * PER + e, D)] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
    }
  } else {
    if (!on) return;
    uint16_t* p = reinterpret_cast<uint16_t*>(pages);
    if constexpr (KEY) {
      store_row<PER>(p + paged_key_index<false>(slot, ln.in * PER, D), x);
    } else {
#pragma unroll
      for (int e = 0; e < PER; ++e) p[vt_index(slot, ln.in * PER + e, D)] = (uint16_t)f32_to_bf16_bits(x[e]);
    }
  }
}

// The page of position `pos` of row b if token s is stored there, else -1.
__device__ __forceinline__ int page_of(const G4PagedAppendArgs& a, int b, int64_t pos, int s) {
  const int shift = __builtin_ctz(a.cache.page_size);
  if (pos < 0 || (pos >> shift) >= a.max_pages || (a.keep > 0 && s < a.seq - a.keep)) return -1;
  const int page = a.page_table[b * a.table_stride + (pos >> shift)];
  return (uint32_t)page < (uint32_t)a.cache.num_pages ? page : -1;
}

// A step's tokens (and chunks of fewer than 8): one workgroup per token, one wave per 64 / LANES head vectors of a
// kind (looping over more than 16). A wave's vectors are a chain of loads, so nothing is staged: 256 tokens of
// 2 x (4 + 2) heads of 256 in 4.4 us, of which an empty launch takes 1.7.
template <int D, bool F8>
__global__ __launch_bounds__(1024) void paged_append_kernel(G4PagedAppendArgs a, int vec) {
  constexpr int PER = Lanes<D>::PER, VECS = Lanes<D>::VECS;
  const Lanes<D> ln(threadIdx.x & 63);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nwaves = blockDim.x >> 6;
  const int S = a.seq, H = a.cache.kv_heads;
  const int token = blockIdx.x, b = token / S, s = token - b * S;
  const int nq = a.q ? H * a.group : 0, q_waves = (nq + VECS - 1) / VECS, kv_waves = (H + VECS - 1) / VECS;
  const int64_t in_base = (int64_t)token * a.in_row_stride + ln.in * PER;
  const int64_t pos = (int64_t)a.write_pos[b] + s;
  const int page = page_of(a, b, pos, s);
  const int slot = (int)(pos & (a.cache.page_size - 1));
  Token<D> t;
  t.load(a, token, vec, true, ln);
  for (int u = wave; u < q_waves + 2 * kv_waves; u += nwaves) {
    float x[PER];
    if (u < q_waves) {
      const int v = u * VECS + ln.sub, at = v < nq ? v : nq - 1;
      load_row<PER>(reinterpret_cast<const uint16_t*>(a.q) + in_base + (int64_t)at * D, vec, x);
      t.q.apply(x, ln);
      if (v < nq) store_row<PER>(reinterpret_cast<uint16_t*>(a.q_out) + ((int64_t)token * nq + v) * D + ln.in * PER, x);
      continue;
    }
    if (page < 0) continue;
    const bool key = u < q_waves + kv_waves;
    const int v = (u - q_waves - (key ? 0 : kv_waves)) * VECS + ln.sub, head = v < H ? v : H - 1;
    const int64_t block = ((int64_t)page * H + head) * a.cache.page_size;
    load_row<PER>(reinterpret_cast<const uint16_t*>(key ? a.k : a.v) + in_base + (int64_t)head * D, vec, x);
    if (key) {
      t.k.apply(x, ln);
      store_vector<D, F8, true>(a.cache, block, slot, x, v < H, ln);
    } else {
      t.prepare_v(x, a.eps);
      store_vector<D, F8, false>(a.cache, block, slot, x, v < H, ln);
    }
  }
}

// Chunks of 8 tokens and more: one workgroup per 8 positions p, p % 8 == 0, of a row, one token per wave, whose
// head vectors are loaded kTileVecs at a time. The page holds 8 positions' values of a dim side by side, so the
// value rows of a full group pass through LDS and are stored as whole 16-byte pieces; a group that the chunk, the
// pads or `keep` cut stores its values one by one. Bound by HBM: 256 x 256 tokens of 2 x (4 + 2) heads of 256 into e4m3
// pages, 797 MB, in 159 us (5.0 TB/s; a plain copy of that size reaches 5.7, or 6.4 non-temporally); with one workgroup
// per token and every value byte stored alone 524 us.
constexpr int kTileTok = 8;
constexpr int kTileThreads = 64 * kTileTok;
constexpr int kTileVecs = 4;
constexpr int kTileValueBytes = 32 * 1024;  // LDS for value rows; more heads than fit go in turns

template <int D, bool F8>
__global__ __launch_bounds__(kTileThreads) __attribute__((amdgpu_waves_per_eu(D >= 512 ? 4 : 8))) void
paged_append_tile_kernel(G4PagedAppendArgs a, int vec, int groups) {
  constexpr int PER = Lanes<D>::PER, VECS = Lanes<D>::VECS, BYTES = F8 ? 1 : 2;
  constexpr int kHeads = kTileValueBytes / (kTileTok * D * BYTES);
  extern __shared__ __attribute__((aligned(16))) uint8_t v_lds[];  // [min(H, kHeads)][8 tokens][D]
  const Lanes<D> ln(threadIdx.x & 63);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int S = a.seq, H = a.cache.kv_heads;
  const int b = (int)blockIdx.x / groups;
  const int64_t start = a.write_pos[b];
  const int64_t p0 = (start & ~(int64_t)(kTileTok - 1)) + ((int)blockIdx.x - b * groups) * kTileTok;
  const int64_t s0 = p0 - start;  // token of p0: -7 ..
  if (s0 >= S) return;
  const bool full = s0 >= 0 && s0 + kTileTok <= S && page_of(a, b, p0, (int)s0) >= 0;  // one page, the first token the earliest
  const int64_t s64 = s0 + wave;
  const bool on = s64 >= 0 && s64 < S;
  const int s = on ? (int)s64 : 0;
  const int page = on ? page_of(a, b, p0 + wave, s) : -1;
  const int slot = (int)((p0 + wave) & (a.cache.page_size - 1));
  const int64_t token = (int64_t)b * S + s, in_base = token * a.in_row_stride + ln.in * PER;
  Token<D> t;
  if (on) t.load(a, token, vec, page >= 0, ln);
  if (on && a.q) {
    const int nq = H * a.group;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(a.q) + in_base;
    uint16_t* dst = reinterpret_cast<uint16_t*>(a.q_out) + token * nq * D + ln.in * PER;
    for (int v0 = 0; v0 < nq; v0 += kTileVecs * VECS) {
      float x[kTileVecs][PER];
#pragma unroll
      for (int i = 0; i < kTileVecs; ++i) {
        const int v = v0 + i * VECS + ln.sub;
        if (v0 + i * VECS < nq) load_row<PER>(src + (v < nq ? v : nq - 1) * D, vec, x[i]);
      }
#pragma unroll
      for (int i = 0; i < kTileVecs; ++i)
        if (v0 + i * VECS < nq) {
          const int v = v0 + i * VECS + ln.sub;
          t.q.apply(x[i], ln);
          if (v < nq) store_row<PER>(dst + v * D, x[i]);
        }
    }
  }
  const int64_t page_block = (int64_t)page * H;
  for (int h0 = 0; h0 < H; h0 += kHeads) {
    const int h1 = h0 + kHeads < H ? h0 + kHeads : H;
    if (page >= 0) {
      const uint16_t* ksrc = reinterpret_cast<const uint16_t*>(a.k) + in_base;
      const uint16_t* vsrc = reinterpret_cast<const uint16_t*>(a.v) + in_base;
      for (int h = h0; h < h1; h += kTileVecs / 2 * VECS) {
        float x[kTileVecs][PER];
#pragma unroll
        for (int i = 0; i < kTileVecs / 2; ++i) {
          const int v = h + i * VECS + ln.sub, head = v < h1 ? v : h1 - 1;
          if (h + i * VECS < h1) {
            load_row<PER>(ksrc + (int64_t)head * D, vec, x[2 * i]);
            load_row<PER>(vsrc + (int64_t)head * D, vec, x[2 * i + 1]);
          }
        }
#pragma unroll
        for (int i = 0; i < kTileVecs / 2; ++i) {
          if (h + i * VECS >= h1) break;
          const int v = h + i * VECS + ln.sub, head = v < h1 ? v : h1 - 1;
          const int64_t block = (page_block + head) * a.cache.page_size;
          t.k.apply(x[2 * i], ln);
          store_vector<D, F8, true>(a.cache, block, slot, x[2 * i], v < h1, ln);
          t.prepare_v(x[2 * i + 1], a.eps);
          if (!full) {
            store_vector<D, F8, false>(a.cache, block, slot, x[2 * i + 1], v < h1, ln);
            continue;
          }
          uint8_t* row = v_lds + ((head - h0) * kTileTok + wave) * D * BYTES;
          if constexpr (F8) {
            uint32_t w[PER / 4];
            const int byte = quantise<D>(x[2 * i + 1], w);
            if (v >= h1) continue;
            if (ln.in == 0) a.cache.value_scale[block + slot] = (uint8_t)byte;
            store_bytes<PER>(row + ln.in * PER, w);
          } else {
            if (v < h1) store_row<PER>(reinterpret_cast<uint16_t*>(row) + ln.in * PER, x[2 * i + 1]);
          }
        }
      }
    }
    if (!full) continue;  // uniform over the workgroup
    __syncthreads();
    // 32 bytes per thread: 8 slots of 4 (e4m3) or 2 (bf16) dims, of which LDS holds a dword per slot
    const int slot0 = (int)(p0 & (a.cache.page_size - 1));
    constexpr int DWORDS = D * BYTES / 4;  // per row
    for (int i = threadIdx.x; i < (h1 - h0) * DWORDS; i += kTileThreads) {
      const int head = i / DWORDS, dw = i - head * DWORDS;
      const uint32_t* col = reinterpret_cast<const uint32_t*>(v_lds) + head * kTileTok * DWORDS + dw;
      uint32_t r[kTileTok];
#pragma unroll
      for (int j = 0; j < kTileTok; ++j) r[j] = col[j * DWORDS];
      uint32_t out[8];
      if constexpr (F8) {
        // bytes of slots 4 g .. 4 g + 3: dim k's are byte k of each
#pragma unroll
        for (int g = 0; g < 2; ++g) {
          const uint32_t lo01 = __builtin_amdgcn_perm(r[4 * g + 1], r[4 * g], 0x05010400);  // d0: s0 s1, d1: s0 s1
          const uint32_t hi01 = __builtin_amdgcn_perm(r[4 * g + 1], r[4 * g], 0x07030602);  // d2: s0 s1, d3: s0 s1
          const uint32_t lo23 = __builtin_amdgcn_perm(r[4 * g + 3], r[4 * g + 2], 0x05010400);
          const uint32_t hi23 = __builtin_amdgcn_perm(r[4 * g + 3], r[4 * g + 2], 0x07030602);
          out[0 + g] = __builtin_amdgcn_perm(lo23, lo01, 0x05040100);
          out[2 + g] = __builtin_amdgcn_perm(lo23, lo01, 0x07060302);
          out[4 + g] = __builtin_amdgcn_perm(hi23, hi01, 0x05040100);
          out[6 + g] = __builtin_amdgcn_perm(hi23, hi01, 0x07060302);
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          out[j] = __builtin_amdgcn_perm(r[2 * j + 1], r[2 * j], 0x05040100);
          out[4 + j] = __builtin_amdgcn_perm(r[2 * j + 1], r[2 * j], 0x07060302);
        }
      }
      const int64_t block = (page_block + h0 + head) * a.cache.page_size;  // full: every wave has the group's page
      u32x4* dst = reinterpret_cast<u32x4*>(reinterpret_cast<uint8_t*>(a.cache.value) + (block + slot0) * D * BYTES + dw * 32);
      dst[0] = u32x4{out[0], out[1], out[2], out[3]};
      dst[1] = u32x4{out[4], out[5], out[6], out[7]};
    }
    if (h1 < H) __syncthreads();
  }
}

template <int D, bool F8>
int launch_append(const G4PagedAppendArgs& a, bool vec, hipStream_t st) {
  const int H = a.cache.kv_heads;
  if (a.seq >= kTileTok) {
    // 8 consecutive positions from any start on lie in ceil((seq + 7) / 8) groups at most
    const int64_t groups = ((int64_t)a.seq + 2 * kTileTok - 2) / kTileTok;
    if (a.batch * groups * kTileThreads > kMaxThreads)
      return fail(G4_ERR_UNSUPPORTED, "g4_paged_append: too many tokens (%d rows of %d)", a.batch, a.seq);
    constexpr int kHeads = kTileValueBytes / (kTileTok * D * (F8 ? 1 : 2));
    const size_t lds = (size_t)(H < kHeads ? H : kHeads) * kTileTok * D * (F8 ? 1 : 2);
    hipLaunchKernelGGL((paged_append_tile_kernel<D, F8>), dim3((unsigned)(a.batch * groups)), dim3(kTileThreads), lds, st, a,
                       (int)vec, (int)groups);
  } else {
    constexpr int VECS = Lanes<D>::VECS;
    const int nvec = ((a.q ? H * a.group : 0) + VECS - 1) / VECS + 2 * ((H + VECS - 1) / VECS);
    const int64_t tokens = (int64_t)a.batch * a.seq, threads = 64 * (nvec > 16 ? 16 : nvec);
    if (tokens * threads > kMaxThreads)
      return fail(G4_ERR_UNSUPPORTED, "g4_paged_append: too many tokens (%d rows of %d)", a.batch, a.seq);
    hipLaunchKernelGGL((paged_append_kernel<D, F8>), dim3((unsigned)tokens), dim3((unsigned)threads), 0, st, a, (int)vec);
  }
  return check_launch("g4_paged_append");
}
template <int D>
int launch_append(const G4PagedAppendArgs& a, bool vec, hipStream_t st) {
  return a.cache.format == G4_PAGES_E4M3 ? launch_append<D, true>(a, vec, st) : launch_append<D, false>(a, vec, st);
}

// --- read back ---------------------------------------------------------------------------------------------

constexpr int kReadThreads = 256;

// One workgroup per (row, head, 32-slot chunk) and array: the chunk's 16-byte pieces are asked for at once, in the
// page's order, and turned into token-major rows in LDS. Bound by HBM: 16 rows of up to 8191 positions of 2 heads of 256
// out of e4m3 pages, 353 MB, in 70 us (5.0 TB/s; a plain copy 5.7); 500 positions of 512 dims in 4.1 us, 6.3 with both
// arrays in one workgroup.
template <int D, bool F8>
__global__ __launch_bounds__(kReadThreads) void paged_read_kernel(G4PagedReadArgs a, int first_chunk, int n_chunks) {
  constexpr int RS = D + 8;                            // LDS row stride, elements
  constexpr int PIECES = 32 * D * (F8 ? 1 : 2) / 16;   // 16-byte pieces of a chunk
  constexpr int LOADS = (PIECES + kReadThreads - 1) / kReadThreads;
  __shared__ __attribute__((aligned(16))) uint16_t rows[32 * RS];
  const bool values = blockIdx.y;
  const int H = a.cache.kv_heads, ps = a.cache.page_size, tid = threadIdx.x;
  const int c = first_chunk + (int)(blockIdx.x % n_chunks);
  const int bh = blockIdx.x / n_chunks, b = bh / H, h = bh - b * H;
  const int p0 = c * 32;  // < 2^31: the host bounds start + count
  int len = a.lengths[b];
  if (len > a.max_pages * ps) len = a.max_pages * ps;
  int page = -1;
  if (p0 < len) page = a.page_table[b * a.table_stride + (p0 >> __builtin_ctz(ps))];
  const bool there = (uint32_t)page < (uint32_t)a.cache.num_pages;
  if (there) {
    const int64_t block = ((int64_t)page * H + h) * ps + (p0 & (ps - 1));  // slots before the chunk
    const uint8_t* src = reinterpret_cast<const uint8_t*>(values ? a.cache.value : a.cache.key) + block * D * (F8 ? 1 : 2);
    const uint8_t* scale = F8 ? (values ? a.cache.value_scale : a.cache.key_scale) + block : nullptr;
    u32x4 w[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j)
      if (PIECES % kReadThreads == 0 || tid + j * kReadThreads < PIECES)
        w[j] = *reinterpret_cast<const u32x4*>(src + (tid + j * kReadThreads) * 16);
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
      const int i = tid + j * kReadThreads;
      if (PIECES % kReadThreads != 0 && i >= PIECES) break;
      if (!values) {
        // a key piece: 16 (e4m3) or 8 (bf16) dims of one slot
        const int col = i / 4 % 16, half = i / 64 % 2, run = i / 128;
        const int slot = 8 * (col >> 2) + 4 * half + (col & 3);
        if constexpr (F8) {
          const float sc = exp2_byte(scale[slot]);
          uint32_t o[8];
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            o[2 * q] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j][q], sc, false));
            o[2 * q + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j][q], sc, true));
          }
          u32x4* dst = reinterpret_cast<u32x4*>(rows + slot * RS + run * 64 + i % 4 * 16);
          dst[0] = u32x4{o[0], o[1], o[2], o[3]};
          dst[1] = u32x4{o[4], o[5], o[6], o[7]};
        } else {
          *reinterpret_cast<u32x4*>(rows + slot * RS + run * 32 + i % 4 * 8) = w[j];
        }
      } else {
        // a value piece: 8 slots of two dims (e4m3) or one dim (bf16)
        const int d = F8 ? i * 2 % D : i % D, g = F8 ? i * 2 / D : i / D;
        if constexpr (F8) {
          const uint2 sc = *reinterpret_cast<const uint2*>(scale + 8 * g);
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const uint32_t two = (w[j][q / 4] >> (8 * (q % 4)) & 0xffu) | ((w[j][2 + q / 4] >> (8 * (q % 4)) & 0xffu) << 8);
            *reinterpret_cast<uint32_t*>(rows + (8 * g + q) * RS + d) = __builtin_bit_cast(
                uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(
                              two, exp2_byte((q < 4 ? sc.x : sc.y) >> (8 * (q % 4)) & 0xff), false));
          }
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) rows[(8 * g + q) * RS + d] = (uint16_t)(w[j][q / 2] >> (16 * (q % 2)));
        }
      }
    }
    __syncthreads();
  }
  uint16_t* out = reinterpret_cast<uint16_t*>(values ? a.v_out : a.k_out);
#pragma unroll 4
  for (int i = tid; i < 32 * D / 8; i += kReadThreads) {
    const int slot = i / (D / 8), d = i % (D / 8) * 8;
    const int p = p0 + slot;
    if (p < a.start || p >= a.start + a.count) continue;
    u32x4 w = {0u, 0u, 0u, 0u};
    if (there && p < len) w = *reinterpret_cast<const u32x4*>(rows + slot * RS + d);
    *reinterpret_cast<u32x4*>(out + (((int64_t)b * a.count + (p - a.start)) * H + h) * D + d) = w;
  }
}

template <int D>
void launch_read(const G4PagedReadArgs& a, int first, int n, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.cache.kv_heads * n), 2);
  if (a.cache.format == G4_PAGES_E4M3)
    hipLaunchKernelGGL((paged_read_kernel<D, true>), grid, dim3(kReadThreads), 0, st, a, first, n);
  else
    hipLaunchKernelGGL((paged_read_kernel<D, false>), grid, dim3(kReadThreads), 0, st, a, first, n);
}

}  // namespace
}  // namespace g4

extern "C" int g4_paged_append(const G4PagedAppendArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_append";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedAppendArgs& a = *args;
  int rc = check_paged_cache(a.cache, who);
  if (rc == G4_OK) rc = check_page_table(a.page_table, a.max_pages, a.table_stride, a.cache.page_size, who);
  if (rc != G4_OK) return rc;
  if (a.batch <= 0 || a.seq <= 0 || a.keep < 0)
    return fail(G4_ERR_INVALID, "%s: batch %d / seq %d must be positive, keep %d not negative", who, a.batch, a.seq, a.keep);
  if ((int64_t)a.batch * a.seq > 0x7fffffffLL) return fail(G4_ERR_UNSUPPORTED, "%s: too many tokens", who);
  if (!a.k || !a.v || !a.write_pos) return fail(G4_ERR_INVALID, "%s: k / v / write_pos is NULL", who);
  if (a.q && (a.group <= 0 || !a.q_out)) return fail(G4_ERR_INVALID, "%s: q needs group > 0 and q_out", who);
  const int64_t heads = (int64_t)a.cache.kv_heads * (a.q ? a.group : 1);
  if (heads > 0xffff) return fail(G4_ERR_UNSUPPORTED, "%s: %lld heads", who, (long long)heads);
  if ((int64_t)a.batch * a.seq > 1 && a.in_row_stride < heads * a.cache.head_dim)
    return fail(G4_ERR_INVALID, "%s: in_row_stride %lld too small", who, (long long)a.in_row_stride);
  if ((a.flags & (G4_APPEND_ROPE_K | G4_APPEND_ROPE_Q)) && (!a.rope_cos || !a.rope_sin))
    return fail(G4_ERR_INVALID, "%s: RoPE flags need rope_cos / rope_sin", who);
  if ((a.flags & G4_APPEND_NORM_K) && !a.k_norm_weight) return fail(G4_ERR_INVALID, "%s: NORM_K needs k_norm_weight", who);
  if ((a.flags & G4_APPEND_NORM_Q) && a.q && !a.q_norm_weight)
    return fail(G4_ERR_INVALID, "%s: NORM_Q needs q_norm_weight", who);
  // each lane's 4 or 8 elements move in one access where every row is aligned to them
  const uintptr_t al = a.cache.head_dim == 512 ? 16 : 8;
  bool vec = (a.in_row_stride * 2) % (int64_t)al == 0;
  for (const void* p : std::initializer_list<const void*>{a.k, a.v, a.q, a.k_norm_weight, a.q_norm_weight})
    vec = vec && reinterpret_cast<uintptr_t>(p) % al == 0;
  if (reinterpret_cast<uintptr_t>(a.q_out) % al) return fail(G4_ERR_INVALID, "%s: q_out must be %d-byte aligned", who, (int)al);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a.cache.head_dim) {
    case 64: return launch_append<64>(a, vec, st);
    case 128: return launch_append<128>(a, vec, st);
    case 256: return launch_append<256>(a, vec, st);
    default: return launch_append<512>(a, vec, st);
  }
}

extern "C" int g4_paged_read(const G4PagedReadArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_read";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedReadArgs& a = *args;
  int rc = check_paged_cache(a.cache, who);
  if (rc == G4_OK) rc = check_page_table(a.page_table, a.max_pages, a.table_stride, a.cache.page_size, who);
  if (rc != G4_OK) return rc;
  if (a.batch <= 0 || a.start < 0 || a.count <= 0 || (int64_t)a.start + a.count > 0x7fffffffLL - 1024)
    return fail(G4_ERR_INVALID, "%s: batch %d, start %d, count %d", who, a.batch, a.start, a.count);
  if (!a.lengths || !a.k_out || !a.v_out) return fail(G4_ERR_INVALID, "%s: lengths / k_out / v_out is NULL", who);
  if (reinterpret_cast<uintptr_t>(a.k_out) % 16 || reinterpret_cast<uintptr_t>(a.v_out) % 16)
    return fail(G4_ERR_INVALID, "%s: k_out / v_out must be 16-byte aligned", who);
  const int first = a.start / 32, n = (a.start + a.count - 1) / 32 - first + 1;
  if ((int64_t)a.batch * a.cache.kv_heads * n > kMaxThreads / kReadThreads) return fail(G4_ERR_UNSUPPORTED, "%s: too many positions", who);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a.cache.head_dim) {
    case 64: launch_read<64>(a, first, n, st); break;
    case 128: launch_read<128>(a, first, n, st); break;
    case 256: launch_read<256>(a, first, n, st); break;
    default: launch_read<512>(a, first, n, st); break;
  }
  return check_launch(who);
}
