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

// One head vector of a token per wave: lane l holds elements [l * PER, (l + 1) * PER), PER = D / 64, so a
// rotation's partner (d +- D / 2) is lane l ^ 32. f32 throughout: y = x * (mean(x^2) + eps)^-1/2 * w, then
// y cos + rotate_half(y) sin.
template <int D>
struct HeadVec {
  static constexpr int PER = D / 64;
  float x[PER];

  __device__ __forceinline__ void load(const uint16_t* p, int lane, bool vec) {
    if (PER == 1 || !vec) {
#pragma unroll
      for (int e = 0; e < PER; ++e) x[e] = bf16_bits_to_f32(p[lane * PER + e]);
    } else {
      uint32_t w[PER / 2 > 0 ? PER / 2 : 1];
      __builtin_memcpy(w, __builtin_assume_aligned(p + lane * PER, PER * 2), PER * 2);
#pragma unroll
      for (int i = 0; i < PER / 2; ++i) x[2 * i] = __uint_as_float(w[i] << 16), x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  }

  __device__ __forceinline__ void norm(const HeadVec* w, float eps) {
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) ss += x[e] * x[e];
    ss = wave_sum(ss);
    const float inv = 1.0f / __fsqrt_rn(ss * (1.0f / D) + eps);
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] = w ? x[e] * inv * w->x[e] : x[e] * inv;
  }

  __device__ __forceinline__ void rotate(const float* c, const float* s, int lane) {
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const uint32_t u = __float_as_uint(x[e]);
      const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);  // the low / high half's value
      const float partner = lane < 32 ? -__uint_as_float(r[1]) : __uint_as_float(r[0]);
      x[e] = x[e] * c[e] + partner * s[e];
    }
  }

  // The scale byte of the whole vector, and this lane's elements divided by it.
  __device__ __forceinline__ int quantise() {
    float a = 0.f;
#pragma unroll
    for (int e = 0; e < PER; ++e) a = fmaxf(a, finite_f32(x[e]) ? fabsf(x[e]) : 0.f);
    const int byte = scale_byte(wave_max(a));
    const float inv = __uint_as_float((uint32_t)(2 * kScaleBias - byte) << 23);
#pragma unroll
    for (int e = 0; e < PER; ++e) x[e] *= inv;
    return byte;
  }
};

enum VecKind { kQ = 0, kK = 1, kV = 2 };

// One workgroup per token, one wave per head vector (looping over more than 16).
template <int D, bool F8>
__global__ __launch_bounds__(1024) void paged_append_kernel(G4PagedAppendArgs a, int vec) {
  constexpr int PER = D / 64;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), nwaves = blockDim.x >> 6;
  const int S = a.seq, H = a.cache.kv_heads, R = a.group, ps = a.cache.page_size;
  const int token = blockIdx.x, b = token / S, s = token - b * S;
  const int nq = a.q ? H * R : 0, nvec = nq + 2 * H;

  const int64_t pos = (int64_t)a.write_pos[b] + s;
  int page = -1;
  if (pos >= 0 && pos < (int64_t)a.max_pages * ps && (a.keep == 0 || s >= S - a.keep))
    page = a.page_table[b * a.table_stride + pos / ps];
  const bool stored = (uint32_t)page < (uint32_t)a.cache.num_pages;
  const int slot = (int)(pos & (ps - 1));

  const int64_t in_base = (int64_t)token * a.in_row_stride, rope_base = (int64_t)token * D + lane * PER;
  for (int v = wave; v < nvec; v += nwaves) {
    const int kind = v < nq ? kQ : (v < nq + H ? kK : kV);
    const int head = kind == kQ ? v : (kind == kK ? v - nq : v - nq - H);  // q: its place among H * R
    if (kind != kQ && !stored) continue;
    const uint16_t* src = reinterpret_cast<const uint16_t*>(kind == kQ ? a.q : (kind == kK ? a.k : a.v));
    HeadVec<D> x;
    x.load(src + in_base + (int64_t)head * D, lane, vec);
    const bool norm = a.flags & (kind == kQ ? G4_APPEND_NORM_Q : (kind == kK ? G4_APPEND_NORM_K : G4_APPEND_NORM_V));
    if (norm) {
      HeadVec<D> w;
      if (kind != kV) w.load(reinterpret_cast<const uint16_t*>(kind == kQ ? a.q_norm_weight : a.k_norm_weight), lane, vec);
      x.norm(kind != kV ? &w : nullptr, a.eps);
    }
    if (kind != kV && (a.flags & (kind == kQ ? G4_APPEND_ROPE_Q : G4_APPEND_ROPE_K))) {
      float c[PER], sn[PER];
#pragma unroll
      for (int e = 0; e < PER; ++e) c[e] = a.rope_cos[rope_base + e], sn[e] = a.rope_sin[rope_base + e];
      x.rotate(c, sn, lane);
    }
    if (kind == kQ) {
      uint16_t* dst = reinterpret_cast<uint16_t*>(a.q_out) + ((int64_t)token * nq + head) * D + lane * PER;
#pragma unroll
      for (int e = 0; e < PER; ++e) dst[e] = (uint16_t)f32_to_bf16_bits(x.x[e]);
      continue;
    }
    const int64_t block = ((int64_t)page * H + head) * ps;
    if constexpr (F8) {
      const int byte = x.quantise();
      if (lane == 0) (kind == kK ? a.cache.key_scale : a.cache.value_scale)[block + slot] = (uint8_t)byte;
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const int d = lane * PER + e;
      const int64_t at = block * D + (kind == kK ? paged_key_index<F8>(slot, d, D) : (int)vt_index(slot, d, D));
      void* dst = kind == kK ? a.cache.key : a.cache.value;
      if constexpr (F8)
        reinterpret_cast<uint8_t*>(dst)[at] = (uint8_t)pack_e4m3x2(x.x[e], 0.f);
      else
        reinterpret_cast<uint16_t*>(dst)[at] = (uint16_t)f32_to_bf16_bits(x.x[e]);
    }
  }
}

template <int D>
void launch_append(const G4PagedAppendArgs& a, bool vec, hipStream_t st) {
  const int nvec = (a.q ? a.cache.kv_heads * a.group : 0) + 2 * a.cache.kv_heads;
  const dim3 grid((unsigned)((int64_t)a.batch * a.seq)), block((unsigned)(64 * (nvec > 16 ? 16 : nvec)));
  if (a.cache.format == G4_PAGES_E4M3)
    hipLaunchKernelGGL((paged_append_kernel<D, true>), grid, block, 0, st, a, (int)vec);
  else
    hipLaunchKernelGGL((paged_append_kernel<D, false>), grid, block, 0, st, a, (int)vec);
}

// --- read back ---------------------------------------------------------------------------------------------

constexpr int kReadThreads = 256;

// One workgroup per (row, head, 32-slot chunk): a chunk's keys, then its values, are read in 16-byte
// pieces in the page's order and turned into token-major rows in LDS.
template <int D, bool F8>
__global__ __launch_bounds__(kReadThreads) void paged_read_kernel(G4PagedReadArgs a, int first_chunk, int n_chunks) {
  constexpr int RS = D + 8;                        // LDS row stride, elements
  constexpr int PIECES = 32 * D * (F8 ? 1 : 2) / 16;  // 16-byte pieces of a chunk
  __shared__ __attribute__((aligned(16))) uint16_t rows[32 * RS];
  const int H = a.cache.kv_heads, ps = a.cache.page_size;
  const int c = first_chunk + (int)(blockIdx.x % n_chunks);
  const int bh = blockIdx.x / n_chunks, b = bh / H, h = bh - b * H;
  const int p0 = c * 32;  // < 2^31: the host bounds start + count
  int len = a.lengths[b];
  if (len > a.max_pages * ps) len = a.max_pages * ps;
  int page = -1;
  if (p0 < len) page = a.page_table[b * a.table_stride + p0 / ps];
  const bool there = (uint32_t)page < (uint32_t)a.cache.num_pages;
  const int64_t block = ((int64_t)page * H + h) * ps;
  const int chunk = (p0 & (ps - 1)) >> 5;
  for (int part = 0; part < 2; ++part) {
    if (there) {
      const uint8_t* src = reinterpret_cast<const uint8_t*>(part ? a.cache.value : a.cache.key) +
                           (block * D + (int64_t)chunk * 32 * D) * (F8 ? 1 : 2);
      const uint8_t* scale = F8 ? (part ? a.cache.value_scale : a.cache.key_scale) + block + chunk * 32 : nullptr;
      for (int i = threadIdx.x; i < PIECES; i += kReadThreads) {
        const u32x4 w = *reinterpret_cast<const u32x4*>(src + i * 16);
        if (part == 0) {
          // a key piece: 16 (e4m3) or 8 (bf16) dims of one slot
          const int col = i / 4 % 16, half = i / 64 % 2, run = i / 128;
          const int slot = 8 * (col >> 2) + 4 * half + (col & 3);
          if constexpr (F8) {
            const float sc = exp2_byte(scale[slot]);
            uint32_t o[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              o[2 * j] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j], sc, false));
              o[2 * j + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w[j], sc, true));
            }
            u32x4* dst = reinterpret_cast<u32x4*>(rows + slot * RS + run * 64 + i % 4 * 16);
            dst[0] = u32x4{o[0], o[1], o[2], o[3]};
            dst[1] = u32x4{o[4], o[5], o[6], o[7]};
          } else {
            *reinterpret_cast<u32x4*>(rows + slot * RS + run * 32 + i % 4 * 8) = w;
          }
        } else {
          // a value piece: 8 slots of two dims (e4m3) or one dim (bf16)
          const int d = F8 ? i * 2 % D : i % D, g = F8 ? i * 2 / D : i / D;
          if constexpr (F8) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const int slot = 8 * g + j;
              const uint32_t two = (w[j / 4] >> (8 * (j % 4)) & 0xffu) | ((w[2 + j / 4] >> (8 * (j % 4)) & 0xffu) << 8);
              *reinterpret_cast<uint32_t*>(rows + slot * RS + d) = __builtin_bit_cast(
                  uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(two, exp2_byte(scale[slot]), false));
            }
          } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) rows[(8 * g + j) * RS + d] = (uint16_t)(w[j / 2] >> (16 * (j % 2)));
          }
        }
      }
    }
    __syncthreads();
    uint16_t* out = reinterpret_cast<uint16_t*>(part ? a.v_out : a.k_out);
    for (int i = threadIdx.x; i < 32 * D / 8; i += kReadThreads) {
      const int slot = i / (D / 8), d = i % (D / 8) * 8;
      const int p = p0 + slot;
      if (p < a.start || p >= a.start + a.count) continue;
      u32x4 w = {0u, 0u, 0u, 0u};
      if (there && p < len) w = *reinterpret_cast<const u32x4*>(rows + slot * RS + d);
      *reinterpret_cast<u32x4*>(out + (((int64_t)b * a.count + (p - a.start)) * H + h) * D + d) = w;
    }
    __syncthreads();
  }
}

template <int D>
void launch_read(const G4PagedReadArgs& a, int first, int n, hipStream_t st) {
  const dim3 grid((unsigned)((int64_t)a.batch * a.cache.kv_heads * n));
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
  if (a.in_row_stride < (int64_t)a.cache.kv_heads * a.cache.head_dim)
    return fail(G4_ERR_INVALID, "%s: in_row_stride %lld too small", who, (long long)a.in_row_stride);
  if ((a.flags & (G4_APPEND_ROPE_K | G4_APPEND_ROPE_Q)) && (!a.rope_cos || !a.rope_sin))
    return fail(G4_ERR_INVALID, "%s: RoPE flags need rope_cos / rope_sin", who);
  if ((a.flags & G4_APPEND_NORM_K) && !a.k_norm_weight) return fail(G4_ERR_INVALID, "%s: NORM_K needs k_norm_weight", who);
  if ((a.flags & G4_APPEND_NORM_Q) && a.q && !a.q_norm_weight)
    return fail(G4_ERR_INVALID, "%s: NORM_Q needs q_norm_weight", who);
  // each lane's D / 64 elements move in one access where every row is aligned to them
  const uintptr_t al = (uintptr_t)(a.cache.head_dim / 64) * 2;
  bool vec = (a.in_row_stride * 2) % (int64_t)al == 0;
  for (const void* p : std::initializer_list<const void*>{a.k, a.v, a.q, a.k_norm_weight, a.q_norm_weight})
    vec = vec && reinterpret_cast<uintptr_t>(p) % al == 0;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a.cache.head_dim) {
    case 64: launch_append<64>(a, vec, st); break;
    case 128: launch_append<128>(a, vec, st); break;
    case 256: launch_append<256>(a, vec, st); break;
    default: launch_append<512>(a, vec, st); break;
  }
  return check_launch(who);
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
  if ((int64_t)a.batch * a.cache.kv_heads * n > 0x7fffffffLL) return fail(G4_ERR_UNSUPPORTED, "%s: too many positions", who);
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  switch (a.cache.head_dim) {
    case 64: launch_read<64>(a, first, n, st); break;
    case 128: launch_read<128>(a, first, n, st); break;
    case 256: launch_read<256>(a, first, n, st); break;
    default: launch_read<512>(a, first, n, st); break;
  }
  return check_launch(who);
}
