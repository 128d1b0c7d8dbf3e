// What the paged-cache kernels share: element places in a page, the e4m3 format with power-of-two
// scales, the page lookup, and the host-side checks of a G4PagedCache.
#pragma once

#include "g4_common.h"
#include "g4_internal.h"

namespace g4 {

constexpr int kScaleBias = 127;
constexpr int kScaleMinExp = -100;  // probability x scale stays a normal bf16 down to probabilities of 2^-26
constexpr int kScaleMaxExp = 120;   // the scale of the largest finite f32 vector

// Place of (slot, dim) in a page and head's block (the dense layouts; e4m3 keys in runs of 64 dims).
template <bool F8>
__host__ __device__ __forceinline__ int paged_key_index(int slot, int d, int D) {
  constexpr int KR = F8 ? 64 : 32;
  const int r = slot & 31;
  const int col = ((r >> 3) << 2) | (r & 3);
  return ((((slot >> 5) * (D / KR) + d / KR) * 2 + ((r >> 2) & 1)) * 16 + col) * KR + d % KR;
}

// The scale byte of a vector whose largest finite magnitude is `amax` (>= 0): the least e with
// amax <= 448 * 2^e. amax = m * 2^k with 1 <= m < 2 and 448 = 1.75 * 2^8, so e = k - 8, one more for m > 1.75.
__device__ __forceinline__ int scale_byte(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int e = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
  return (e < kScaleMinExp ? kScaleMinExp : (e > kScaleMaxExp ? kScaleMaxExp : e)) + kScaleBias;
}

__device__ __forceinline__ float exp2_byte(int byte) { return __uint_as_float((uint32_t)byte << 23); }

__device__ __forceinline__ bool finite_f32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// 4 packed e4m3 bytes -> 4 bf16 (exact).
__device__ __forceinline__ void unpack_e4m3(uint32_t w, uint32_t& lo, uint32_t& hi) {
  lo = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
  hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
}

// Host-side checks of one layer's pages and table; G4_OK or the error (text under `who`).
constexpr int64_t kMaxThreads = 0xffffffff;  // of a grid's dimension
int check_paged_cache(const G4PagedCache& c, const char* who);
int check_page_table(const int32_t* table, int32_t max_pages, int64_t table_stride, int32_t page_size, const char* who);

}  // namespace g4
