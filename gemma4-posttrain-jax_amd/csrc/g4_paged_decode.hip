// One-token attention over a paged cache (g4_paged_decode_attention).
//
// Per (row, kv head): scores s = q . k on MFMA with the keys as the A operand, so that a lane holds the
// scores of keys 8 g .. 8 g + 7 (g = lane / 16) of its query column lane % 16 -- which is the B operand of
// the value product, V^T as A. Neither scores nor probabilities leave the registers. One pass over
// the keys: per wave a running maximum m and sum l in f32, o rescaled where m grows.
#include "g4_paged.h"

namespace g4 {
namespace {

constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

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

template <int D, bool F8>
struct Shape {
  static constexpr int KRUNS = F8 ? D / 64 : D / 32;  // 16-byte key loads per lane, chunk and half
  static constexpr int VLOADS = F8 ? D / 32 : D / 16;  // 16-byte value loads per lane and chunk
  static constexpr int BYTES = F8 ? 1 : 2;
  static constexpr int CHUNK = 32 * D * BYTES;  // bytes of a chunk's keys, and of its values
};

template <int D, bool F8>
__global__ __launch_bounds__(kWaves * 64) void paged_decode_kernel(G4PagedDecodeArgs a) {
  using Sh = Shape<D, F8>;
  extern __shared__ __attribute__((aligned(16))) float lds[];  // [kWaves][R][D] o | [kWaves][16] m | [kWaves][16] l
  const int R = a.group, H = a.cache.kv_heads, ps = a.cache.page_size;
  float* m_lds = lds + kWaves * R * D;
  float* l_lds = m_lds + kWaves * 16;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int pair = blockIdx.x, b = pair / H, h = pair - b * H;

  int hi = a.lengths[b];
  if (hi > a.max_pages * ps) hi = a.max_pages * ps;
  const int lo = a.window > 0 && hi > a.window ? hi - a.window : 0;

  const uint16_t* qrow = reinterpret_cast<const uint16_t*>(a.q) + ((int64_t)pair * R + col) * D;
  bf16x8 qop[D / 32];
#pragma unroll
  for (int s = 0; s < D / 32; ++s) {
    // e4m3: a 16-byte key load is 16 consecutive dims, two operands
    const int d = F8 ? 64 * (s / 2) + 16 * grp + 8 * (s % 2) : 32 * s + 8 * grp;
    u32x4 v = {0u, 0u, 0u, 0u};
    if (col < R) v = load16(qrow + d);
    qop[s] = as_bf16x8(v);
  }

  float m = kNegInf, l = 0.f;
  floatx4 o[D / 16];
#pragma unroll
  for (int t = 0; t < D / 16; ++t) o[t] = floatx4{0.f, 0.f, 0.f, 0.f};

  for (int c = lo / 32 + w; c * 32 < hi; c += kWaves) {
    const int page = __builtin_amdgcn_readfirstlane(a.page_table[b * a.table_stride + c * 32 / ps]);
    if ((uint32_t)page >= (uint32_t)a.cache.num_pages) continue;
    const int64_t block = ((int64_t)page * H + h) * ps + (c * 32 & (ps - 1));  // slots before this chunk
    const uint8_t* kp = reinterpret_cast<const uint8_t*>(a.cache.key) + block * D * Sh::BYTES + col * 64 + grp * 16;
    const uint8_t* vp = reinterpret_cast<const uint8_t*>(a.cache.value) + block * D * Sh::BYTES +
                        (grp * (Sh::VLOADS * 16) + col) * 16;
    u32x4 kv[2][Sh::KRUNS], vv[Sh::VLOADS];
#pragma unroll
    for (int s = 0; s < Sh::KRUNS; ++s)
#pragma unroll
      for (int bb = 0; bb < 2; ++bb) kv[bb][s] = *reinterpret_cast<const u32x4*>(kp + (s * 2 + bb) * 1024);
#pragma unroll
    for (int t = 0; t < Sh::VLOADS; ++t) vv[t] = *reinterpret_cast<const u32x4*>(vp + t * 256);
    uint2 kscale = make_uint2(0, 0), vscale = make_uint2(0, 0);
    if constexpr (F8) {
      kscale = *reinterpret_cast<const uint2*>(a.cache.key_scale + block + 8 * grp);
      vscale = *reinterpret_cast<const uint2*>(a.cache.value_scale + block + 8 * grp);
    }

    floatx4 sc[2] = {floatx4{0.f, 0.f, 0.f, 0.f}, floatx4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
    for (int s = 0; s < Sh::KRUNS; ++s)
#pragma unroll
      for (int bb = 0; bb < 2; ++bb) {
        if constexpr (F8) {
          sc[bb] = mfma16x16x32(e4m3_operand(kv[bb][s][0], kv[bb][s][1]), qop[2 * s], sc[bb]);
          sc[bb] = mfma16x16x32(e4m3_operand(kv[bb][s][2], kv[bb][s][3]), qop[2 * s + 1], sc[bb]);
        } else {
          sc[bb] = mfma16x16x32(as_bf16x8(kv[bb][s]), qop[s], sc[bb]);
        }
      }

    // keys 8 grp + j of the chunk
    float p[8], mx = m;
    const int first = c * 32 + 8 * grp;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float s = sc[j / 4][j % 4];
      if constexpr (F8) s *= exp2_byte((j < 4 ? kscale.x : kscale.y) >> (8 * (j % 4)) & 0xff);
      p[j] = first + j >= lo && first + j < hi ? s : kNegInf;
      mx = fmaxf(mx, p[j]);
    }
    mx = column_max(mx);
    const float base = mx == kNegInf ? 0.f : mx;
    const float alpha = __builtin_amdgcn_exp2f((m - base) * kLog2e);
    m = mx;
    l *= alpha;
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[t] *= alpha;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const bool on = first + j >= lo && first + j < hi;
      p[j] = __builtin_amdgcn_exp2f((p[j] - base) * kLog2e);
      l += p[j];
      if constexpr (F8) p[j] = on ? p[j] * exp2_byte((j < 4 ? vscale.x : vscale.y) >> (8 * (j % 4)) & 0xff) : 0.f;
    }
    const bf16x8 pop = as_bf16x8(u32x4{pack_bf16x2(p[0], p[1]), pack_bf16x2(p[2], p[3]), pack_bf16x2(p[4], p[5]),
                                       pack_bf16x2(p[6], p[7])});
    if (c * 32 < lo || c * 32 + 32 > hi) {  // the slots of no attended key may hold anything: 0 x NaN is no 0
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (F8) {
          uint32_t mask = 0;  // dword i % 2: keys 4 (i % 2) .. + 3
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (first + 4 * (i % 2) + j >= lo && first + 4 * (i % 2) + j < hi) mask |= 0xffu << (8 * j);
#pragma unroll
          for (int t = 0; t < Sh::VLOADS; ++t) vv[t][i] &= mask;
        } else {
          uint32_t mask = 0;  // dword i: keys 2 i, 2 i + 1
#pragma unroll
          for (int j = 0; j < 2; ++j)
            if (first + 2 * i + j >= lo && first + 2 * i + j < hi) mask |= 0xffffu << (16 * j);
#pragma unroll
          for (int t = 0; t < Sh::VLOADS; ++t) vv[t][i] &= mask;
        }
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
  }

  // the waves' parts joined: o = sum_w exp(m_w - m) o_w, l likewise
  l = column_sum(l);
  if (grp == 0) m_lds[w * 16 + col] = m, l_lds[w * 16 + col] = l;
  if (col < R) {
    float* dst = lds + (w * R + col) * D;
#pragma unroll
    for (int t = 0; t < D / 16; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        // row 4 grp + i of tile t is dim 16 t + 4 grp + i (bf16), or 32 (t / 2) + 2 (4 grp + i) + t % 2 (e4m3)
        const int d = F8 ? 32 * (t / 2) + 2 * (4 * grp + i) + t % 2 : 16 * t + 4 * grp + i;
        dst[d] = o[t][i];
      }
  }
  __syncthreads();
  uint16_t* out = reinterpret_cast<uint16_t*>(a.out) + (int64_t)pair * R * D;
  for (int i = tid; i < R * D; i += kWaves * 64) {
    const int r = i / D;
    float mm = kNegInf;
    for (int v = 0; v < kWaves; ++v) mm = fmaxf(mm, m_lds[v * 16 + r]);
    const float base = mm == kNegInf ? 0.f : mm;
    float num = 0.f, den = 0.f;
    for (int v = 0; v < kWaves; ++v) {
      const float f = __builtin_amdgcn_exp2f((m_lds[v * 16 + r] - base) * kLog2e);
      num += f * lds[v * R * D + i];
      den += f * l_lds[v * 16 + r];
    }
    out[i] = (uint16_t)f32_to_bf16_bits(den == 0.f ? 0.f : num / den);
  }
}

size_t lds_bytes(int R, int D) { return ((size_t)kWaves * R * D + 2 * kWaves * 16) * sizeof(float); }

template <int D, bool F8>
int launch(const G4PagedDecodeArgs& a, hipStream_t st) {
  const size_t lds = lds_bytes(a.group, D);
  if (lds > 64 * 1024) {
    int dev = 0;
    const int rc = device_setup(&dev);
    if (rc != G4_OK) return rc;
    if (!lds_limit_raised(dev, (const void*)paged_decode_kernel<D, F8>))
      return fail(G4_ERR_LAUNCH, "g4_paged_decode_attention: the kernel's LDS limit could not be raised");
  }
  hipLaunchKernelGGL((paged_decode_kernel<D, F8>), dim3((unsigned)(a.batch * a.cache.kv_heads)), dim3(kWaves * 64), lds, st, a);
  return check_launch("g4_paged_decode_attention");
}

}  // namespace

int setup_paged_kernels(int device) {
  raise_lds_limit(device, (const void*)paged_decode_kernel<512, false>, (int)lds_bytes(16, 512));
  raise_lds_limit(device, (const void*)paged_decode_kernel<512, true>, (int)lds_bytes(16, 512));
  raise_lds_limit(device, (const void*)paged_decode_kernel<256, false>, (int)lds_bytes(16, 256));
  raise_lds_limit(device, (const void*)paged_decode_kernel<256, true>, (int)lds_bytes(16, 256));
  return G4_OK;
}

namespace {

int check_decode(const G4PagedDecodeArgs& a, const char* who) {
  int rc = check_paged_cache(a.cache, who);
  if (rc == G4_OK) rc = check_page_table(a.page_table, a.max_pages, a.table_stride, a.cache.page_size, who);
  if (rc != G4_OK) return rc;
  if (a.batch <= 0 || a.group <= 0 || a.group > 16 || a.window < 0)
    return fail(G4_ERR_INVALID, "%s: batch %d group %d (1..16) window %d", who, a.batch, a.group, a.window);
  if ((int64_t)a.batch * a.cache.kv_heads > 0x7fffffLL)
    return fail(G4_ERR_UNSUPPORTED, "%s: batch %d x %d kv heads", who, a.batch, a.cache.kv_heads);
  if (!a.lengths || !a.q || !a.out) return fail(G4_ERR_INVALID, "%s: lengths / q / out is NULL", who);
  if (reinterpret_cast<uintptr_t>(a.q) % 16 || reinterpret_cast<uintptr_t>(a.out) % 16)
    return fail(G4_ERR_INVALID, "%s: q / out must be 16-byte aligned", who);
  return G4_OK;
}

}  // namespace
}  // namespace g4

extern "C" size_t g4_paged_decode_workspace_size(const G4PagedDecodeArgs* args) {
  if (!args) return 0;
  return 0;
}

extern "C" int g4_paged_decode_attention(const G4PagedDecodeArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_paged_decode_attention";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4PagedDecodeArgs& a = *args;
  const int rc = check_decode(a, who);
  if (rc != G4_OK) return rc;
  hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  const bool f8 = a.cache.format == G4_PAGES_E4M3;
  switch (a.cache.head_dim) {
    case 64: return f8 ? launch<64, true>(a, st) : launch<64, false>(a, st);
    case 128: return f8 ? launch<128, true>(a, st) : launch<128, false>(a, st);
    case 256: return f8 ? launch<256, true>(a, st) : launch<256, false>(a, st);
    default: return f8 ? launch<512, true>(a, st) : launch<512, false>(a, st);
  }
}
