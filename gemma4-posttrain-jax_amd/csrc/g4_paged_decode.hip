// One-token attention over a paged cache (g4_paged_decode_attention).
//
// Per (row, kv head): scores s = q . k on MFMA with the keys as the A operand, so that a lane holds the
// scores of keys 8 g .. 8 g + 7 (g = lane / 16) of its query column lane % 16 -- which is the B operand of
// the value product, V^T as A. Neither scores nor probabilities leave the registers. One pass over
// the keys: per wave a running maximum m and sum l in f32, o rescaled where m grows.
//
// The work is the rows' 32-slot chunks, row by row and head by head in one sequence, of which every
// workgroup takes an equal range: ragged rows, few long rows and many short ones fill the chip alike. The
// lengths stand on the device, so each workgroup sums up the chunks of the rows itself. A (row, head) that lies
// in one range is finished there; the others leave (m, l, o) per range, which a second launch joins in the
// ranges' order.
#include "g4_paged.h"

namespace g4 {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * 64;
constexpr int kMaxRows = 2048;  // rows of one launch: their chunk sums stand in LDS beside the largest o
constexpr int kMinChunks = kWaves;  // chunks per workgroup at least: one per wave
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNegInf = -__builtin_inff();

constexpr int kCus = 256;
// workgroups that a CU holds at once (by registers)
constexpr int groups_per_cu(int D) { return D == 512 ? 1 : (D == 256 ? 2 : (D == 128 ? 3 : 4)); }
constexpr int q_stride(int D) { return D + 8; }  // elements between q rows in LDS: 16 lanes' reads fall on different banks

struct Workspace {
  float* o;      // [2 groups][R][D] o of a range's first and last (row, head) where those pass its ends
  float* ml;     // [2 groups][R][2] their m and l
  int2* ranges;  // [pairs] first range and number of ranges with a part of the (row, head), {0, 0}: none to join
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

template <int D, bool F8>
struct Shape {
  static constexpr int KRUNS = F8 ? D / 64 : D / 32;  // 16-byte key loads per lane, chunk and half
  static constexpr int VLOADS = F8 ? D / 32 : D / 16;  // 16-byte value loads per lane and chunk
  static constexpr int BYTES = F8 ? 1 : 2;
  static constexpr int CHUNK = 32 * D * BYTES;  // bytes of a chunk's keys, and of its values
};

struct RowKeys {
  int lo, hi;  // attended positions [lo, hi)
  __device__ __forceinline__ int first() const { return lo >> 5; }
  __device__ __forceinline__ int chunks() const { return hi > lo ? ((hi + 31) >> 5) - (lo >> 5) : 0; }
};

__device__ __forceinline__ RowKeys row_keys(const G4PagedDecodeArgs& a, int b) {
  const int cap = a.max_pages * a.cache.page_size;
  int hi = a.lengths[b];
  hi = hi < 0 ? 0 : (hi > cap ? cap : hi);
  return RowKeys{a.window > 0 && hi > a.window ? hi - a.window : 0, hi};
}

// sums[b] = chunks of the rows before b, b = 0 .. batch (every thread of the workgroup calls it).
__device__ __forceinline__ void sum_chunks(const G4PagedDecodeArgs& a, int* sums, int* wave_sums) {
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6;
  const int per = (a.batch + kThreads - 1) / kThreads;
  const int b0 = tid * per, b1 = b0 + per < a.batch ? b0 + per : a.batch;
  int own = 0;
  for (int b = b0; b < b1; ++b) own += row_keys(a, b).chunks();
  int incl = own;
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const int below = __shfl_up(incl, d, 64);
    if (lane >= d) incl += below;
  }
  if (lane == 63) wave_sums[w] = incl;
  __syncthreads();
  int base = incl - own;
  for (int i = 0; i < w; ++i) base += wave_sums[i];
  if (tid == 0) sums[0] = 0;
  for (int b = b0; b < b1; ++b) {
    base += row_keys(a, b).chunks();
    sums[b + 1] = base;
  }
  __syncthreads();
}

template <int D, bool F8>
__global__ __launch_bounds__(kThreads, groups_per_cu(D)) void paged_decode_kernel(G4PagedDecodeArgs a, Workspace ws) {
  using Sh = Shape<D, F8>;
  // [kWaves][R][D] o | [R][q_stride(D)] q | [kWaves][16] m, l | chunk sums
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int R = a.group, H = a.cache.kv_heads, ps = a.cache.page_size;
  uint16_t* q_lds = reinterpret_cast<uint16_t*>(lds + kWaves * R * D);
  float* m_lds = reinterpret_cast<float*>(q_lds + R * q_stride(D));
  float* l_lds = m_lds + kWaves * 16;
  int* wave_sums = reinterpret_cast<int*>(l_lds + kWaves * 16);
  int* sums = wave_sums + kWaves;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, grp = lane >> 4;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int page_shift = __builtin_ctz(ps) - 5;  // chunks per page, log2

  sum_chunks(a, sums, wave_sums);
  const int64_t total = (int64_t)sums[a.batch] * H;
  int64_t per = (total + gridDim.x - 1) / gridDim.x;
  if (per < kMinChunks) per = kMinChunks;
  int64_t f = blockIdx.x * per;
  const int64_t f_end = f + per < total ? f + per : total;

  // rows without a key
  uint16_t* out_all = reinterpret_cast<uint16_t*>(a.out);
  for (int b = blockIdx.x; b < a.batch; b += gridDim.x) {
    if (sums[b + 1] != sums[b]) continue;
    for (int i = tid; i < H * R * D; i += kThreads) out_all[(int64_t)b * H * R * D + i] = 0;
    for (int h = tid; h < H; h += kThreads) ws.ranges[b * H + h] = make_int2(0, 0);
  }
  if (f >= f_end) return;

  int b = 0;  // the row of chunk f: the last with sums[b] * H <= f
  for (int lo = 0, hi = a.batch; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if ((int64_t)sums[mid] * H <= f) lo = mid; else hi = mid;
    b = lo;
  }

  while (f < f_end) {
    while (sums[b + 1] == sums[b] || (int64_t)sums[b + 1] * H <= f) ++b;
    b = __builtin_amdgcn_readfirstlane(b);
    const RowKeys keys = row_keys(a, b);
    const int n = keys.chunks();
    const int64_t row_f = f - (int64_t)sums[b] * H;
    const int h = __builtin_amdgcn_readfirstlane((int)(row_f / n));
    const int pair = b * H + h;
    const int64_t pair_f = (int64_t)sums[b] * H + (int64_t)h * n;  // the pair's first chunk
    const int c0 = __builtin_amdgcn_readfirstlane((int)(f - pair_f));
    const int64_t f_next = pair_f + n < f_end ? pair_f + n : f_end;
    const int c1 = __builtin_amdgcn_readfirstlane((int)(f_next - pair_f));

    float m = kNegInf, l = 0.f;
    floatx4 o[D / 16];
#pragma unroll
    for (int t = 0; t < D / 16; ++t) o[t] = floatx4{0.f, 0.f, 0.f, 0.f};

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
    auto page_of = [&](int c) -> int { return __builtin_amdgcn_readfirstlane(table[c >> page_shift]); };
    auto load_keys = [&](const Place& at) {
      const __amdgpu_buffer_rsrc_t r =
          make_rsrc(reinterpret_cast<const uint8_t*>(a.cache.key) + at.slot * (D * Sh::BYTES), at.there ? Sh::CHUNK : 0);
#pragma unroll
      for (int s = 0; s < Sh::KRUNS; ++s)
#pragma unroll
        for (int bb = 0; bb < 2; ++bb) kv[bb][s] = buffer_load16(r, col * 64 + grp * 16, (s * 2 + bb) * 1024);
      if constexpr (F8) {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.cache.key_scale + at.slot, at.there ? 32 : 0);
        kscale = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * grp, 0, 0));
      }
    };
    auto load_values = [&](const Place& at) {
      const __amdgpu_buffer_rsrc_t r =
          make_rsrc(reinterpret_cast<const uint8_t*>(a.cache.value) + at.slot * (D * Sh::BYTES), at.there ? Sh::CHUNK : 0);
#pragma unroll
      for (int t = 0; t < Sh::VLOADS; ++t) vv[t] = buffer_load16(r, (grp * (Sh::VLOADS * 16) + col) * 16, t * 256);
      if constexpr (F8) {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(a.cache.value_scale + at.slot, at.there ? 32 : 0);
        vscale = __builtin_bit_cast(uint2, __builtin_amdgcn_raw_buffer_load_b64(rs, 8 * grp, 0, 0));
      }
    };

    const int last = keys.first() + c1;
    int c = keys.first() + c0 + w;
    Place at{0, false};
    int page_next = 0;
    if (c < last) {
      at = place_of(page_of(c), c);
      load_keys(at);
      load_values(at);
      if (c + kWaves < last) page_next = page_of(c + kWaves);
    }
    // q rows in LDS; the columns beyond them compute on the last row and are dropped
    for (int i = tid; i < R * D / 8; i += kThreads)
      *reinterpret_cast<u32x4*>(q_lds + i / (D / 8) * q_stride(D) + i % (D / 8) * 8) =
          load16(reinterpret_cast<const uint16_t*>(a.q) + (int64_t)pair * R * D + i * 8);
    __syncthreads();
    const uint16_t* qrow = q_lds + (col < R ? col : R - 1) * q_stride(D) + (F8 ? 16 : 8) * grp;
    // operand s: e4m3 keys come 16 consecutive dims a load, two operands
    auto qop = [&](int s) -> bf16x8 { return as_bf16x8(load16(qrow + (F8 ? 64 * (s / 2) + 8 * (s % 2) : 32 * s))); };
    for (; c < last; c += kWaves) {
      const bool more = c + kWaves < last;
      const Place next = place_of(more ? page_next : -1, c + kWaves);
      if (c + 2 * kWaves < last) page_next = page_of(c + 2 * kWaves);
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
      if constexpr (F8) {
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[j / 4][j % 4] *= exp2_byte((j < 4 ? kscale.x : kscale.y) >> (8 * (j % 4)) & 0xff);
      }
      __builtin_amdgcn_sched_barrier(0);
      if (more) load_keys(next);
      __builtin_amdgcn_sched_barrier(0);

      // keys 8 grp + j of the chunk
      const bool inner = c * 32 >= lo && c * 32 + 32 <= hi;  // every slot is an attended key
      float p[8], mx = m;
      const int first = c * 32 + 8 * grp;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        p[j] = inner || (first + j >= lo && first + j < hi) ? sc[j / 4][j % 4] : kNegInf;
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
        p[j] = __builtin_amdgcn_exp2f((p[j] - base) * kLog2e);
        l += p[j];
        if constexpr (F8) {
          const float v = p[j] * exp2_byte((j < 4 ? vscale.x : vscale.y) >> (8 * (j % 4)) & 0xff);
          p[j] = inner || (first + j >= lo && first + j < hi) ? v : 0.f;
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
          for (int j = 0; j < KEYS; ++j) {
            const int key = first + KEYS * (i % (8 / KEYS)) + j;
            if (key >= lo && key < hi) mask |= (F8 ? 0xffu : 0xffffu) << (32 / KEYS * j);
          }
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
      if (more) load_values(next);
      __builtin_amdgcn_sched_barrier(0);
      at = next;
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
    const bool whole = c0 == 0 && c1 == n;
    const int64_t part = 2 * (int64_t)blockIdx.x + (c0 == 0 ? 1 : 0);  // begun here: the range's last, else its first
    uint16_t* out = out_all + (int64_t)pair * R * D;
    for (int i = tid; i < R * D; i += kThreads) {
      const int r = i / D;
      float mm = kNegInf;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) mm = fmaxf(mm, m_lds[v * 16 + r]);
      const float base = mm == kNegInf ? 0.f : mm;
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int v = 0; v < kWaves; ++v) {
        const float x = __builtin_amdgcn_exp2f((m_lds[v * 16 + r] - base) * kLog2e);
        num += x * lds[v * R * D + i];
        den += x * l_lds[v * 16 + r];
      }
      if (whole) {
        out[i] = (uint16_t)f32_to_bf16_bits(den == 0.f ? 0.f : num / den);
      } else {
        ws.o[part * R * D + i] = num;
        if (i % D == 0) ws.ml[(part * R + r) * 2] = mm, ws.ml[(part * R + r) * 2 + 1] = den;
      }
    }
    if (c0 == 0 && tid == 0) {
      const int first_range = (int)(pair_f / per), last_range = (int)((pair_f + n - 1) / per);
      ws.ranges[pair] = whole ? make_int2(0, 0) : make_int2(first_range, last_range - first_range + 1);
    }
    f = f_next;
    if (f < f_end) __syncthreads();
  }
}

constexpr int kJoinDims = 64;  // elements of o per workgroup: 16 lanes of 4, 16 parts at a time
constexpr int kJoinParts = kThreads / (kJoinDims / 4);

// The ranges' parts of a (row, head), joined in their order.
__global__ __launch_bounds__(kThreads) void paged_join_kernel(G4PagedDecodeArgs a, Workspace ws) {
  __shared__ float m_s[kJoinParts], l_s[kJoinParts];
  __shared__ __attribute__((aligned(16))) floatx4 o_s[kJoinParts][kJoinDims / 4];
  const int R = a.group, D = a.cache.head_dim;
  const int pair = blockIdx.x, i0 = blockIdx.y * kJoinDims, r = i0 / D;
  const int2 range = ws.ranges[pair];
  if (range.y == 0) return;
  const int x = threadIdx.x % (kJoinDims / 4), y = threadIdx.x / (kJoinDims / 4);
  // part j of the pair: the last of its first range, the first of the others
  auto part = [&](int j) -> int64_t { return 2 * (int64_t)(range.x + j) + (j == 0 ? 1 : 0); };
  float m = kNegInf;
  for (int j = y; j < range.y; j += kJoinParts) m = fmaxf(m, ws.ml[(part(j) * R + r) * 2]);
  if (x == 0) m_s[y] = m;
  __syncthreads();
  m = kNegInf;
#pragma unroll
  for (int j = 0; j < kJoinParts; ++j) m = fmaxf(m, m_s[j]);
  const float base = m == kNegInf ? 0.f : m;
  float l = 0.f;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int j = y; j < range.y; j += kJoinParts) {
    const int64_t at = part(j) * R + r;
    const float f = __builtin_amdgcn_exp2f((ws.ml[at * 2] - base) * kLog2e);
    l += f * ws.ml[at * 2 + 1];
    o += f * *reinterpret_cast<const floatx4*>(ws.o + part(j) * R * D + i0 + 4 * x);
  }
  if (x == 0) l_s[y] = l;
  o_s[y][x] = o;
  __syncthreads();
  if (y > 0) return;
  for (int j = 1; j < kJoinParts; ++j) o += o_s[j][x], l += l_s[j];
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (l == 0.f) o = floatx4{0.f, 0.f, 0.f, 0.f};
  uint2 w = make_uint2(pack_bf16x2(o[0] * inv, o[1] * inv), pack_bf16x2(o[2] * inv, o[3] * inv));
  *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.out) + (int64_t)pair * R * D + i0 + 4 * x) = w;
}

size_t lds_bytes(int R, int D, int batch) {
  return ((size_t)kWaves * R * D + (size_t)R * q_stride(D) / 2 + 2 * kWaves * 16 + kWaves + batch + 1) * sizeof(float);
}

int groups(const G4PagedDecodeArgs& a) { return kCus * groups_per_cu(a.cache.head_dim); }

// Rows of a launch: at most kMaxRows, and their chunks' sum fits 31 bits.
int rows_per_launch(const G4PagedDecodeArgs& a) {
  const int64_t chunks = (int64_t)a.max_pages * a.cache.page_size / 32;  // >= 1, < 2^26
  const int64_t rows = 0x7fffffffLL / chunks;
  return (int)(rows < kMaxRows ? (rows < a.batch ? rows : a.batch) : (kMaxRows < a.batch ? kMaxRows : a.batch));
}

size_t workspace_bytes(const G4PagedDecodeArgs& a) {
  const size_t parts = 2 * (size_t)groups(a) * a.group;
  return parts * a.cache.head_dim * 4 + parts * 8 + (size_t)rows_per_launch(a) * a.cache.kv_heads * 8;
}

template <int D, bool F8>
int launch(const G4PagedDecodeArgs& a, hipStream_t st) {
  const size_t lds = lds_bytes(a.group, D, rows_per_launch(a));
  if (lds > 64 * 1024) {
    int dev = 0;
    const int rc = device_setup(&dev);
    if (rc != G4_OK) return rc;
    if (!lds_limit_raised(dev, (const void*)paged_decode_kernel<D, F8>))
      return fail(G4_ERR_LAUNCH, "g4_paged_decode_attention: the kernel's LDS limit could not be raised");
  }
  const int g = groups(a);
  Workspace ws;
  ws.o = reinterpret_cast<float*>(a.workspace);
  ws.ml = ws.o + 2 * (size_t)g * a.group * D;
  ws.ranges = reinterpret_cast<int2*>(ws.ml + 2 * (size_t)g * a.group * 2);
  G4PagedDecodeArgs part = a;
  for (int b = 0; b < a.batch; b += part.batch) {
    part.batch = a.batch - b < rows_per_launch(a) ? a.batch - b : rows_per_launch(a);
    const int64_t at = (int64_t)b * a.cache.kv_heads * a.group * D;
    part.page_table = a.page_table + b * a.table_stride;
    part.lengths = a.lengths + b;
    part.q = reinterpret_cast<const uint16_t*>(a.q) + at;
    part.out = reinterpret_cast<uint16_t*>(a.out) + at;
    hipLaunchKernelGGL((paged_decode_kernel<D, F8>), dim3((unsigned)g), dim3(kThreads), lds, st, part, ws);
    hipLaunchKernelGGL(paged_join_kernel, dim3((unsigned)(part.batch * a.cache.kv_heads), (unsigned)(a.group * D / kJoinDims)),
                       dim3(kThreads), 0, st, part, ws);
  }
  return check_launch("g4_paged_decode_attention");
}

}  // namespace

int setup_paged_kernels(int device) {
  const struct {
    const void* fn;
    int dim;
  } kernels[] = {
      {(const void*)paged_decode_kernel<64, false>, 64},   {(const void*)paged_decode_kernel<64, true>, 64},
      {(const void*)paged_decode_kernel<128, false>, 128}, {(const void*)paged_decode_kernel<128, true>, 128},
      {(const void*)paged_decode_kernel<256, false>, 256}, {(const void*)paged_decode_kernel<256, true>, 256},
      {(const void*)paged_decode_kernel<512, false>, 512}, {(const void*)paged_decode_kernel<512, true>, 512},
  };
  for (const auto& k : kernels) {
    const size_t most = lds_bytes(16, k.dim, kMaxRows);
    if (most > 64 * 1024) raise_lds_limit(device, k.fn, (int)most);
  }
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
  if (!a.workspace || a.workspace_bytes < need || reinterpret_cast<uintptr_t>(a.workspace) % 16)
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
