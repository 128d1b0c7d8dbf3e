// Verification of drafted tokens (g4_verify_draft): how many of a row's K drafts the target's probabilities accept, and
// the token that follows them, from given random numbers. Speculative sampling (Leviathan, Kalman, Matias, "Fast
// inference from transformers via speculative decoding", ICML 2023): draft s is accepted while u_s q_s(x_s) < p_s(x_s); at the
// first rejection the token is drawn from max(p - q, 0), after all drafts from p. The draw is the race of exponentials,
// argmax_v w_v / -log(noise_v), which needs no normalisation and no running sum, so that f32 decides it as well as 64 bits
// but for near ties.
//
// Bound by reading the logits: K + 1 target and K draft rows of the vocabulary once, for their maxima and sums of
// exponentials (statistics per chunk of a row), then of two rows per b and the noise for the race. Which rows these are
// every workgroup of the second launch finds from the statistics by itself.
#include "g4_common.h"
#include "g4_internal.h"

namespace g4 {
namespace {

#include "g4_sample_common.h"

constexpr int kThreads = 256, kWaves = kThreads / 64;
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxDrafts = 63;  // decided by one wave
constexpr int kNoColumn = 0x7fffffff;
enum Mode { kGreedy, kUnit, kHeat };  // temperature <= 0, 1, other

struct Stats {  // of a chunk of a row, or of a row
  float m;     // largest logit
  float heat;  // sum exp((x - m) / temperature)
  float unit;  // sum exp(x - m)
  int idx;     // kGreedy: the first column of the largest
};
struct Decision {
  int count;        // accepted drafts
  float m, unit;    // of the row that the last token is drawn from
  int token;        // kGreedy: the token
};
struct VerifyWorkspace {
  Stats* stats;      // [batch][rows][splits], the K + 1 target rows first
  uint64_t* race;    // [batch][splits][2] the best of the residual weights and of p
  Decision* made;    // [batch]
};

int chunk_of(const G4VerifyArgs& a) {
  const int64_t rows = (int64_t)a.batch * (a.drafts + 1 + (a.draft_logits ? a.drafts : 0));
  return rows * a.vocab >= 2048LL * 16384 ? 16384 : 4096;
}
int splits_of(const G4VerifyArgs& a) { return (int)(((int64_t)a.vocab + chunk_of(a) - 1) / chunk_of(a)); }

size_t carve(VerifyWorkspace& w, void* base, const G4VerifyArgs& a) {
  const int64_t splits = splits_of(a);
  size_t at = 0;
  const auto take = [&](int64_t bytes) {
    void* p = base ? static_cast<char*>(base) + at : nullptr;
    at += ((size_t)bytes + 15) / 16 * 16;
    return p;
  };
  w.stats = static_cast<Stats*>(take(a.batch * (2LL * a.drafts + 1) * splits * (int64_t)sizeof(Stats)));
  w.race = static_cast<uint64_t*>(take(a.batch * splits * 16));
  w.made = static_cast<Decision*>(take(a.batch * (int64_t)sizeof(Decision)));
  return at;
}

// --- logits ----------------------------------------------------------------------------------------------------

template <typename T>
struct Unaligned {
  T v;
} __attribute__((packed, aligned(2)));

// 8 logits from p on, of which `n` are there (others -inf). Rows stand at any element: such loads need no alignment.
template <bool BF16>
__device__ __forceinline__ void load8(const void* row, int64_t i, int n, float (&x)[8]) {
  if (n >= 8) {
    if constexpr (BF16) {
      unpack8(reinterpret_cast<const Unaligned<u32x4>*>(static_cast<const uint16_t*>(row) + i)->v, x);
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const u32x4 v = reinterpret_cast<const Unaligned<u32x4>*>(static_cast<const float*>(row) + i + 4 * j)->v;
#pragma unroll
        for (int q = 0; q < 4; ++q) x[4 * j + q] = __uint_as_float(v[q]);
      }
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = e < n ? Elem<BF16>::load(static_cast<const typename Elem<BF16>::T*>(row), i + e) : -__builtin_inff();
}

template <bool BF16>
__device__ __forceinline__ float logit(const void* row, int64_t i) {
  return Elem<BF16>::load(static_cast<const typename Elem<BF16>::T*>(row), i);
}

template <bool BF16>
__device__ __forceinline__ const void* row_at(const void* base, int64_t batch_stride, int64_t row_stride, int b, int r) {
  return static_cast<const char*>(base) + (b * batch_stride + r * row_stride) * (BF16 ? 2 : 4);
}

__device__ __forceinline__ int drafts_of(const G4VerifyArgs& a, int b) {
  return a.draft_lengths ? min(max(a.draft_lengths[b], 0), a.drafts) : a.drafts;
}

// exp(t c) for t <= 0 with c = 1 / temperature, c log2(e) held in two parts: the rounding of a large t c log2(e) would
// be the result's largest error.
struct Heat {
  float hi, lo;  // log2(e) / temperature
  __device__ __forceinline__ float exp(float t) const {
    const float y = t * hi;
    const float e = __builtin_amdgcn_exp2f(y);
    const float rest = fmaf(t, hi, -y) + t * lo;  // (NaN where t is -inf: e is 0 there)
    return e == 0.f ? e : fmaf(e, rest * 0.6931471805599453f, e);
  }
};

template <int MODE>
__device__ __forceinline__ void join(Stats& s, const Stats& o, float c) {
  if (MODE == kGreedy && (o.m > s.m || (o.m == s.m && o.idx < s.idx))) s.idx = o.idx;
  const float top = fmaxf(s.m, o.m), m = fmaxf(top, kF32Min);  // (m finite where there is no logit but -inf)
  const float a = s.m - m, b = o.m - m;
  if (MODE != kGreedy) s.heat = s.heat * __builtin_amdgcn_exp2f(a * c) + o.heat * __builtin_amdgcn_exp2f(b * c);
  if (MODE != kUnit) s.unit = s.unit * __builtin_amdgcn_exp2f(a * kLog2e) + o.unit * __builtin_amdgcn_exp2f(b * kLog2e);
  s.m = top;
}

template <int MODE>
__device__ __forceinline__ Stats wave_join(Stats s, float c) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    Stats o;
    o.m = __shfl_xor(s.m, d, 64);
    o.heat = MODE != kGreedy ? __shfl_xor(s.heat, d, 64) : 0.f;
    o.unit = MODE != kUnit ? __shfl_xor(s.unit, d, 64) : 0.f;
    o.idx = MODE == kGreedy ? __shfl_xor(s.idx, d, 64) : 0;
    join<MODE>(s, o, c);
  }
  if (MODE == kUnit) s.unit = s.heat;
  return s;
}

// --- first launch: a chunk's statistics ------------------------------------------------------------------------------

template <bool BF16, int MODE, int VECS>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(G4VerifyArgs a, VerifyWorkspace w, int rows, int splits) {
  __shared__ Stats part[kWaves];
  const int split = blockIdx.x % splits, br = blockIdx.x / splits, b = br / rows, r = br - b * rows;
  const bool draft = r > a.drafts;
  const int n = drafts_of(a, b);
  if (draft ? r - a.drafts - 1 >= n : r > n) return;  // (uniform) no draft reaches this row
  const void* row = draft ? row_at<BF16>(a.draft_logits, a.draft_batch_stride, a.draft_row_stride, b, r - a.drafts - 1)
                          : row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, r);
  const float c = kLog2e / a.temperature;
  const int64_t i0 = (int64_t)split * (VECS * kThreads * 8) + threadIdx.x * 8;
  float x[VECS][8];
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int64_t i = i0 + v * (kThreads * 8);
    load8<BF16>(row, i, (int)min((int64_t)8, a.vocab - i), x[v]);
  }
  Stats s{-__builtin_inff(), 0.f, 0.f, kNoColumn};
#pragma unroll
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (MODE == kGreedy && x[v][e] > s.m) s.idx = (int)(i0 + v * (kThreads * 8)) + e;
      s.m = fmaxf(s.m, x[v][e]);
    }
  const float m = fmaxf(s.m, kF32Min);
#pragma unroll
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float t = x[v][e] - m;
      if (MODE != kGreedy) s.heat += __builtin_amdgcn_exp2f(t * c);
      if (MODE != kUnit) s.unit += __builtin_amdgcn_exp2f(t * kLog2e);
    }
  s = wave_join<MODE>(s, c);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kWaves; ++i) join<MODE>(s, part[i], c);
    if (MODE == kUnit) s.unit = s.heat;
    w.stats[((int64_t)b * rows + r) * splits + split] = s;
  }
}

// --- which drafts are accepted ------------------------------------------------------------------------------------------

// The rows' statistics from their chunks' (by all waves, rows in turns; a wave's lanes take the chunks).
template <int MODE>
__device__ __forceinline__ void join_rows(const G4VerifyArgs& a, const VerifyWorkspace& w, int b, int rows, int splits, int n,
                                          Stats* out) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / a.temperature;
  for (int r = threadIdx.x >> 6; r < rows; r += kWaves) {
    if (r > a.drafts ? r - a.drafts - 1 >= n : r > n) continue;
    Stats s{-__builtin_inff(), 0.f, 0.f, kNoColumn};
    for (int i = lane; i < splits; i += 64) {
      const Stats o = w.stats[((int64_t)b * rows + r) * splits + i];
      join<MODE>(s, o, c);
    }
    s = wave_join<MODE>(s, c);
    if (lane == 0) out[r] = s;
  }
  __syncthreads();
}

// The log-probability of column i of a row under the unscaled logits.
__device__ __forceinline__ float log_prob(float x, const Stats& s) { return (x - s.m) - logf(s.unit); }

// How many drafts are accepted (by the first wave; lane s decides draft s).
template <bool BF16, int MODE>
__device__ __forceinline__ int accepted(const G4VerifyArgs& a, int b, int n, const Stats* st) {
  const int s = threadIdx.x & 63;
  bool good = false;
  if (s < n) {
    const int d = a.draft_tokens[(int64_t)b * a.drafts + s];
    if constexpr (MODE == kGreedy) {
      good = d == st[s].idx;
    } else if ((uint32_t)d < (uint32_t)a.vocab) {
      const double c = 1.0 / (double)a.temperature;
      const float x = logit<BF16>(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, s), d);
      const double p = exp(((double)x - st[s].m) * c) / (double)st[s].heat;
      double q = 1.0;
      if (a.draft_logits) {
        const Stats& t = st[a.drafts + 1 + s];
        const float y = logit<BF16>(row_at<BF16>(a.draft_logits, a.draft_batch_stride, a.draft_row_stride, b, s), d);
        q = exp(((double)y - t.m) * c) / (double)t.heat;
      }
      good = (double)a.uniforms[(int64_t)b * a.drafts + s] * q < p;
    }
  }
  const uint64_t all = __ballot(good);
  return all == ~0ull ? 64 : __builtin_ctzll(~all);
}

// The accepted tokens with their log-probabilities, and what stands behind the last token (by the first wave).
template <bool BF16>
__device__ __forceinline__ void write_accepted(const G4VerifyArgs& a, int b, int count, const Stats* st) {
  const int s = threadIdx.x & 63;
  if (s == 0) a.count_out[b] = count;
  if (s > a.drafts || s == count) return;
  const int64_t at = (int64_t)b * (a.drafts + 1) + s;
  if (s > count) {
    a.token_out[at] = -1;
    a.logp_out[at] = 0.f;
    return;
  }
  const int d = a.draft_tokens[(int64_t)b * a.drafts + s];
  a.token_out[at] = d;
  a.logp_out[at] = log_prob(logit<BF16>(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, s), d), st[s]);
}

// --- second launch: the race, a chunk per workgroup ----------------------------------------------------------------------

// 1 / -log(u), the factor of a weight in the race: 0 for u = 0, and finite for u = 1.
__device__ __forceinline__ float pace(float u) {
  return u >= kF32Tiny ? __builtin_amdgcn_rcpf(fmaxf(-log_pos_normal(u), 0x1p-25f)) : 0.f;
}

// A score and its column in one word that grows with the score and falls with the column; 0 for no score above 0.
__device__ __forceinline__ uint64_t entry(float score, int64_t column) {
  return score > 0.f ? (uint64_t)__float_as_uint(score) << 32 | (0xffffffffu - (uint32_t)column) : 0;
}

__device__ __forceinline__ uint64_t wave_top(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) {
    const uint64_t o = (uint64_t)__shfl_xor((long long)v, d, 64);
    v = o > v ? o : v;
  }
  return v;
}

template <bool BF16, int MODE, int VECS>
__global__ __launch_bounds__(kThreads) void verify_race_kernel(G4VerifyArgs a, VerifyWorkspace w, int rows, int splits) {
  __shared__ Stats st[2 * kMaxDrafts + 1];
  __shared__ int decided;
  __shared__ uint64_t best[kWaves][2];
  const int split = blockIdx.x % splits, b = blockIdx.x / splits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)split * (VECS * kThreads * 8) + threadIdx.x * 8;
  // the noise is asked for before the decision
  float u[VECS][8];
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int64_t i = i0 + v * (kThreads * 8);
    load8<false>(a.noise + b * a.noise_stride, i, (int)min((int64_t)8, a.vocab - i), u[v]);
  }
  const int n = drafts_of(a, b);
  join_rows<MODE>(a, w, b, rows, splits, n, st);
  if (wave == 0) {
    const int count = accepted<BF16, MODE>(a, b, n, st);
    if (lane == 0) decided = count;
    if (split == 0) {
      write_accepted<BF16>(a, b, count, st);
      if (lane == 0) w.made[b] = Decision{count, st[count].m, st[count].unit, 0};
    }
  }
  __syncthreads();
  const int count = decided;
  const bool rejected = count < n;
  const void* prow = row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, count);
  const void* qrow = rejected && a.draft_logits
                         ? row_at<BF16>(a.draft_logits, a.draft_batch_stride, a.draft_row_stride, b, count) : nullptr;
  const int64_t away = rejected && !qrow ? a.draft_tokens[(int64_t)b * a.drafts + count] : -1;
  const Stats ps = st[count], qs = st[qrow ? a.drafts + 1 + count : count];
  const float pz = 1.0f / ps.heat, qz = 1.0f / qs.heat;
  const double c = 1.4426950408889634074 / (double)a.temperature;
  const Heat heat{(float)c, (float)(c - (double)(float)c)};
  uint64_t top = 0, top_p = 0;
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    const int64_t i = i0 + v * (kThreads * 8);
    const int there = (int)min((int64_t)8, a.vocab - i);
    float x[8], y[8];
    load8<BF16>(prow, i, there, x);
    if (qrow) load8<BF16>(qrow, i, there, y);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e >= there) continue;
      const float p = heat.exp(x[e] - ps.m) * pz, g = pace(u[v][e]);
      float r = p;
      if (qrow) r = fmaxf(p - heat.exp(y[e] - qs.m) * qz, 0.f);
      else if (i + e == away) r = 0.f;
      const uint64_t k = entry(r * g, i + e), kp = entry(p * g, i + e);
      top = k > top ? k : top;
      top_p = kp > top_p ? kp : top_p;
    }
  }
  top = wave_top(top);
  top_p = wave_top(top_p);
  if (lane == 0) best[wave][0] = top, best[wave][1] = top_p;
  __syncthreads();
  if (threadIdx.x < 2) {
    uint64_t k = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) k = best[i][threadIdx.x] > k ? best[i][threadIdx.x] : k;
    w.race[((int64_t)b * splits + split) * 2 + threadIdx.x] = k;
  }
}

// --- last launch: the token ------------------------------------------------------------------------------------------------

template <bool BF16, int MODE>
__global__ __launch_bounds__(MODE == kGreedy ? kThreads : 64) void verify_token_kernel(G4VerifyArgs a, VerifyWorkspace w, int rows,
                                                                                      int splits) {
  __shared__ Stats st[MODE == kGreedy ? kMaxDrafts + 1 : 1];
  const int b = blockIdx.x, lane = threadIdx.x & 63;
  Decision d;
  if constexpr (MODE == kGreedy) {
    const int n = drafts_of(a, b);
    join_rows<MODE>(a, w, b, rows, splits, n, st);
    if (threadIdx.x >= 64) return;
    d.count = accepted<BF16, MODE>(a, b, n, st);
    write_accepted<BF16>(a, b, d.count, st);
    d.m = st[d.count].m, d.unit = st[d.count].unit;
    d.token = st[d.count].idx != kNoColumn ? st[d.count].idx : 0;  // (a row of nothing but -inf and NaN)
  } else {
    d = w.made[b];
    uint64_t k = 0, kp = 0;
    for (int i = lane; i < splits; i += 64) {
      const uint64_t o = w.race[((int64_t)b * splits + i) * 2], op = w.race[((int64_t)b * splits + i) * 2 + 1];
      k = o > k ? o : k;
      kp = op > kp ? op : kp;
    }
    k = wave_top(k);
    kp = wave_top(kp);
    if (!k) k = kp;  // no weight is left: p = q but for rounding
    d.token = k ? (int)(0xffffffffu - (uint32_t)k) : 0;
  }
  if (lane != 0) return;
  const int64_t at = (int64_t)b * (a.drafts + 1) + d.count;
  const float x = logit<BF16>(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, d.count), d.token);
  a.token_out[at] = d.token;
  a.logp_out[at] = log_prob(x, Stats{d.m, 0.f, d.unit, 0});
}

template <bool BF16, int MODE, int VECS>
int launch_verify(const G4VerifyArgs& a, const VerifyWorkspace& w, hipStream_t st) {
  static const char who[] = "g4_verify_draft";
  const int splits = splits_of(a), rows = a.drafts + 1 + (MODE != kGreedy && a.draft_logits ? a.drafts : 0);
  const int64_t blocks = (int64_t)a.batch * rows * splits;
  if (blocks * kThreads > 0xffffffffLL) return fail(G4_ERR_UNSUPPORTED, "%s: too many logits", who);
  hipLaunchKernelGGL((verify_stats_kernel<BF16, MODE, VECS>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a, w, rows, splits);
  int rc = check_launch(who);
  if (rc != G4_OK) return rc;
  if constexpr (MODE != kGreedy) {
    hipLaunchKernelGGL((verify_race_kernel<BF16, MODE, VECS>), dim3((unsigned)((int64_t)a.batch * splits)), dim3(kThreads), 0, st, a, w,
                       rows, splits);
    if ((rc = check_launch(who)) != G4_OK) return rc;
  }
  hipLaunchKernelGGL((verify_token_kernel<BF16, MODE>), dim3((unsigned)a.batch), dim3(MODE == kGreedy ? kThreads : 64), 0, st, a, w,
                     rows, splits);
  return check_launch(who);
}

template <bool BF16, int MODE>
int launch_verify(const G4VerifyArgs& a, const VerifyWorkspace& w, hipStream_t st) {
  return chunk_of(a) == 16384 ? launch_verify<BF16, MODE, 8>(a, w, st) : launch_verify<BF16, MODE, 2>(a, w, st);
}
template <bool BF16>
int launch_verify(const G4VerifyArgs& a, const VerifyWorkspace& w, hipStream_t st) {
  if (a.temperature <= 0.f) return launch_verify<BF16, kGreedy>(a, w, st);
  return a.temperature == 1.f ? launch_verify<BF16, kUnit>(a, w, st) : launch_verify<BF16, kHeat>(a, w, st);
}

}  // namespace
}  // namespace g4

extern "C" size_t g4_verify_draft_workspace_size(const G4VerifyArgs* a) {
  g4::VerifyWorkspace w;
  return !a || a->batch <= 0 || a->drafts <= 0 || a->vocab <= 0 ? 0 : g4::carve(w, nullptr, *a);
}

extern "C" int g4_verify_draft(const G4VerifyArgs* args, void* stream) {
  using namespace g4;
  static const char who[] = "g4_verify_draft";
  if (!args) return fail(G4_ERR_INVALID, "%s: args is NULL", who);
  const G4VerifyArgs& a = *args;
  if (a.dtype != G4_DTYPE_F32 && a.dtype != G4_DTYPE_BF16) return fail(G4_ERR_INVALID, "%s: dtype %d", who, a.dtype);
  if (a.batch <= 0 || a.drafts <= 0 || a.vocab <= 0)
    return fail(G4_ERR_INVALID, "%s: batch %d, drafts %d and vocab %d must be positive", who, a.batch, a.drafts, a.vocab);
  if (a.drafts > kMaxDrafts) return fail(G4_ERR_UNSUPPORTED, "%s: %d drafts (at most %d)", who, a.drafts, kMaxDrafts);
  if (a.vocab > 0x7fffffff - 65536) return fail(G4_ERR_UNSUPPORTED, "%s: vocab %d", who, a.vocab);
  if (!(a.temperature < __builtin_inff()) || (a.temperature > 0.f && a.temperature < 1e-6f))
    return fail(G4_ERR_INVALID, "%s: temperature %g (0 or less, or 1e-6 and more, finite)", who, (double)a.temperature);
  if (!a.logits || !a.draft_tokens || !a.token_out || !a.count_out || !a.logp_out) return fail(G4_ERR_INVALID, "%s: NULL pointer", who);
  if (a.temperature > 0.f && (!a.uniforms || !a.noise)) return fail(G4_ERR_INVALID, "%s: a draw needs uniforms and noise", who);
  const uintptr_t el = a.dtype == G4_DTYPE_BF16 ? 2 : 4;
  if ((uintptr_t)a.logits % el || (uintptr_t)a.draft_logits % el || (uintptr_t)a.noise % 4)
    return fail(G4_ERR_INVALID, "%s: logits and noise must be aligned to their elements", who);
  if (a.row_stride < a.vocab || (a.batch > 1 && a.batch_stride < a.vocab) ||
      (a.draft_logits && ((a.drafts > 1 && a.draft_row_stride < a.vocab) || (a.batch > 1 && a.draft_batch_stride < a.vocab))) ||
      (a.temperature > 0.f && a.batch > 1 && a.noise_stride < a.vocab))
    return fail(G4_ERR_INVALID, "%s: strides below a row of %d", who, a.vocab);
  const size_t need = g4_verify_draft_workspace_size(args);
  if (!a.workspace || a.workspace_bytes < need)
    return fail(G4_ERR_WORKSPACE, "%s: workspace of %zu bytes, %zu needed", who, a.workspace ? a.workspace_bytes : 0, need);
  if ((uintptr_t)a.workspace % 16) return fail(G4_ERR_INVALID, "%s: workspace must be 16-byte aligned", who);
  VerifyWorkspace w;
  carve(w, a.workspace, a);
  const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
  return a.dtype == G4_DTYPE_BF16 ? launch_verify<true>(a, w, st) : launch_verify<false>(a, w, st);
}
