// Verification of drafted tokens (g4_verify_draft): how many of a row's K drafts the target's probabilities accept, and
// the token that follows them, from given random numbers. Speculative sampling (Leviathan, Kalman, Matias, "Fast
// inference from transformers via speculative decoding", ICML 2023): draft s is accepted while u_s q_s(x_s) < p_s(x_s); at the
// first rejection the token is drawn from max(p - q, 0), after all drafts from p. The draw is the race of exponentials,
// argmax_v w_v / -log(noise_v), which needs no normalisation and no running sum, so that f32 decides it as well as 64 bits
// but for near ties (p - q, too, is that of f32 probabilities: where all of it is below 1e-6 of p, its rounding decides).
//
// Bound by reading the logits (64 rows of 9 x 262144 in bf16, 369 MB with the noise, 75 us: 4.9 TB/s) and, while it does, by
// vector instructions: K + 1 target and K draft rows of the vocabulary once, for their largest logits and sums of
// exponentials (a first launch, statistics per chunk of a row, which also clears the counters by which the last of a b's
// workgroups in the race, which writes the token, is found), then of two rows per b and the noise for the race (a
// third). Which rows these are a launch between finds from the statistics, or the race itself.
#include <algorithm>

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
  float m;     // largest logit, or one at most kSlack below it (kGreedy: the largest)
  float heat;  // sum exp((x - m) / temperature)
  float unit;  // sum exp(x - m)
  int idx;     // kGreedy: the first column of the largest
};
struct Decision {  // of one b
  int count;           // accepted drafts
  int32_t away;        // rejected without a drafter's logits: the draft's id, which has no weight; else -1
  int32_t residual;    // whether the drafter's row counts
  float unit;          // of the target's row: sum exp(x - m)
  float pm, pz, qm, qz;  // m and sum exp((x - m) / temperature) of both rows
};
struct VerifyWorkspace {
  Stats* stats;       // [batch][rows][splits], the K + 1 target rows first
  Decision* made;     // [batch]
  uint64_t* best;     // [batch][splits of the race] the workgroups' best
  uint32_t* arrived;  // [batch * kApart] workgroups that have brought theirs, a cache line each
};
constexpr int kApart = 32;  // (counters that share lines: the race of 64 rows 51 us instead of 27)

// Logits per workgroup: in the first launch 2^14 where that makes 2048 workgroups or more, else 2^12 (one row of 9 x 262144
// is 576 of them); in the race 2^12. A thread takes the 2^14 in two steps, all loads ahead of both. us per call, 64 rows of 9 x
// 262144: first launch one step of 4 vectors of 8 per thread 81, two of 4 77, four of 4 79, two of 2 80; the race with 2
// vectors 74.8, 1 77.7, 4 75.8. One row 13.3 (first launch 2 vectors, race 1), 12.8 (2 and 2), 15.0 (1 and 1).
constexpr int kStep = 4, kSteps = 2, kLong = kStep * kSteps, kShort = 2;  // vectors of 8 per thread
constexpr int kRace = 2;                                                  // in the race
int vecs_of(const G4VerifyArgs& a) {
  const int64_t rows = (int64_t)a.batch * (a.drafts + 1 + (a.draft_logits ? a.drafts : 0));
  return rows * a.vocab >= 2048LL * kLong * 8 * kThreads ? kLong : kShort;
}
int splits_of(const G4VerifyArgs& a, int vecs) { return (int)(((int64_t)a.vocab + vecs * 8 * kThreads - 1) / (vecs * 8 * kThreads)); }

size_t carve(VerifyWorkspace& w, void* base, const G4VerifyArgs& a) {
  const int64_t splits = splits_of(a, vecs_of(a));
  size_t at = 0;
  const auto take = [&](int64_t bytes) {
    void* p = base ? static_cast<char*>(base) + at : nullptr;
    at += ((size_t)bytes + 15) / 16 * 16;
    return p;
  };
  w.stats = static_cast<Stats*>(take(a.batch * (2LL * a.drafts + 1) * splits * (int64_t)sizeof(Stats)));
  w.made = static_cast<Decision*>(take(a.batch * (int64_t)sizeof(Decision)));
  w.best = static_cast<uint64_t*>(take(a.batch * (int64_t)splits_of(a, kRace) * 8));
  w.arrived = static_cast<uint32_t*>(take(a.batch * 4LL * kApart));
  return at;
}

// --- logits ----------------------------------------------------------------------------------------------------

typedef u32x4 u32x4_anywhere __attribute__((aligned(2)));

// 8 logits as they stand in memory. Rows stand at any element: such loads need no alignment.
// NT: past the caches (the first launch where it is long: 98 -> 94 us; short ones lose up to 1 us by it).
template <bool BF16>
struct Eight {
  u32x4 raw[BF16 ? 1 : 2];
  template <bool NT = false>
  __device__ __forceinline__ void load(const void* row, int64_t i) {
    const u32x4_anywhere* p = reinterpret_cast<const u32x4_anywhere*>(static_cast<const char*>(row) + i * (BF16 ? 2 : 4));
#pragma unroll
    for (int j = 0; j < (BF16 ? 1 : 2); ++j) raw[j] = NT ? __builtin_nontemporal_load(p + j) : p[j];
  }
  __device__ __forceinline__ void values(float (&x)[8]) const {
    if constexpr (BF16) {
      unpack8(raw[0], x);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(raw[e >> 2][e & 3]);
    }
  }
};

// The logits from i on, of which `n` are there (others -inf).
template <bool BF16>
__device__ __forceinline__ void load8(const void* row, int64_t i, int n, float (&x)[8]) {
  if (n >= 8) {
    Eight<BF16> v;
    v.load(row, i);
    v.values(x);
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

// exp(t c) for t c <= kSlack with c = 1 / temperature, c log2(e) held in two parts: the rounding of a large t c log2(e) would
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

// exp2(x c - m c) with one fma per x, where |m c| is below 2^27 (`tame`): the rounding of m c, alike for every x of a sum, is made up
// for once, by `rest`. It is at most 4 there, so that both factors are within 2^4 of what they would be without it; of a larger m c
// it may pass 127, one factor be 0 and the other infinite.
struct Below {
  float c, mc, rest;
  __device__ __forceinline__ Below(float m, float c_) : c(c_), mc(m * c_), rest(__builtin_amdgcn_exp2f(-fmaf(m, c_, -mc))) {}
  __device__ __forceinline__ bool tame() const { return fabsf(mc) < 0x1p27f; }
  __device__ __forceinline__ float exp(float x) const { return __builtin_amdgcn_exp2f(fmaf(x, c, -mc)); }
};

// A wave's statistics from its lanes', in every lane. (m is finite in the differences where there is no logit but -inf.)
template <int MODE>
__device__ __forceinline__ Stats wave_join(Stats s, float c) {
  const float top = wave_max(s.m), d = s.m - fmaxf(top, kF32Min);
  if (MODE == kGreedy) {
    int idx = s.m == top ? s.idx : kNoColumn;
#pragma unroll
    for (int i = 32; i; i >>= 1) idx = min(idx, __shfl_xor(idx, i, 64));
    s.idx = idx;
  }
  if (MODE != kGreedy) s.heat = wave_sum(s.heat * __builtin_amdgcn_exp2f(d * c));
  if (MODE != kUnit) s.unit = wave_sum(s.unit * __builtin_amdgcn_exp2f(d * kLog2e));
  s.m = top;
  return s;
}

// --- first launch: a chunk's statistics ------------------------------------------------------------------------------

template <int VECS>
__device__ __forceinline__ float sum_exp(const float (&x)[VECS][8], float m, float c) {
  float sum = 0.f;
  const Below below(m, c);
  if (below.tame()) {
#pragma unroll
    for (int v = 0; v < VECS; ++v)
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += below.exp(x[v][e]);
    return sum * below.rest;
  }
#pragma unroll
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += __builtin_amdgcn_exp2f((x[v][e] - m) * c);
  return sum;
}

// Of three floats that are no signalling NaN (fmaxf makes sure of that by an instruction each).
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  __asm__("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
  return d;
}

// A thread's statistics, VECS vectors at a time. The vector work is as long as the loads: instructions count (77 us; 94 with fmaxf,
// a bounds check around each load and the reduction over the workgroup after every 4 vectors). The largest logit that exponents
// refer to follows lazily: it stays while no logit passes it by more than `slack` (exponents of at most kSlack), but for
// kGreedy, which asks for the largest itself.
constexpr float kSlack = 8.f;
template <int MODE, int VECS>
struct Running {
  Stats s{-__builtin_inff(), 0.f, 0.f, kNoColumn};
  float m = kF32Min;  // s.m, finite where there is no logit but -inf
  float c, slack;     // log2(e) / temperature
  __device__ __forceinline__ Running(float temperature)
      : c(kLog2e / temperature), slack(MODE == kGreedy ? 0.f : MODE == kHeat ? kSlack * fminf(temperature, 1.f) : kSlack) {}

  __device__ __forceinline__ void take(const float (&x)[VECS][8], int64_t i, bool draft) {
    float top = s.m;
#pragma unroll
    for (int v = 0; v < VECS; ++v)
#pragma unroll
      for (int e = 0; e < 8; e += 2) {
        if (MODE == kGreedy) {
#pragma unroll
          for (int f = e; f < e + 2; ++f) {
            if (x[v][f] > top) s.idx = (int)i + v * (kThreads * 8) + f;
            top = fmaxf(top, x[v][f]);
          }
        } else {
          top = max3(top, x[v][e], x[v][e + 1]);
        }
      }
    if (top > s.m + slack) {
      const float next = fmaxf(top, kF32Min);
      if (MODE != kGreedy) s.heat *= __builtin_amdgcn_exp2f((m - next) * c);
      if (MODE != kUnit) s.unit *= __builtin_amdgcn_exp2f((m - next) * kLog2e);
      s.m = top;
      m = next;
    }
    if (MODE != kGreedy) s.heat += sum_exp<VECS>(x, m, c);
    if (MODE != kUnit && !draft) s.unit += sum_exp<VECS>(x, m, kLog2e);  // (the log-probabilities are the target's)
  }
};

template <bool BF16, int MODE, int VECS, int TIMES>
__global__ __launch_bounds__(kThreads) void verify_stats_kernel(G4VerifyArgs a, VerifyWorkspace w, int rows, int splits) {
  __shared__ Stats part[kWaves];
  const int split = blockIdx.x % splits, br = blockIdx.x / splits, b = br / rows, r = br - b * rows;
  const bool draft = r > a.drafts;
  const int n = drafts_of(a, b);
  if (draft ? r - a.drafts - 1 >= n : r > n) return;  // (uniform) no draft reaches this row
  if (MODE != kGreedy && r == 0 && split == 0 && threadIdx.x == 0) w.arrived[(int64_t)b * kApart] = 0;
  const void* row = draft ? row_at<BF16>(a.draft_logits, a.draft_batch_stride, a.draft_row_stride, b, r - a.drafts - 1)
                          : row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, r);
  constexpr int STEP = kThreads * 8;
  const int64_t from = (int64_t)split * (TIMES * VECS * STEP), i0 = from + threadIdx.x * 8;
  Running<MODE, VECS> run(a.temperature);
  float x[VECS][8];
  if (from + TIMES * VECS * STEP <= a.vocab) {  // (uniform) all there: all loads ahead of the work
    Eight<BF16> raw[TIMES][VECS];
#pragma unroll
    for (int t = 0; t < TIMES; ++t)
#pragma unroll
      for (int v = 0; v < VECS; ++v) raw[t][v].template load<(TIMES > 1)>(row, i0 + (t * VECS + v) * STEP);
#pragma unroll
    for (int t = 0; t < TIMES; ++t) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) raw[t][v].values(x[v]);
      run.take(x, i0 + t * VECS * STEP, draft);
    }
  } else {
#pragma unroll 1
    for (int t = 0; t < TIMES; ++t) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        const int64_t i = i0 + (t * VECS + v) * STEP;
        load8<BF16>(row, i, (int)min((int64_t)8, a.vocab - i), x[v]);
      }
      run.take(x, i0 + t * VECS * STEP, draft);
    }
  }
  Stats s = wave_join<MODE>(run.s, run.c);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x < 64) {
    static_assert(kWaves == 4, "lanes 0 .. 3 hold the waves'");
    s = wave_join<MODE>(threadIdx.x < kWaves ? part[threadIdx.x] : Stats{-__builtin_inff(), 0.f, 0.f, kNoColumn}, run.c);
    if (MODE == kUnit) s.unit = s.heat;
    if (threadIdx.x == 0) w.stats[((int64_t)b * rows + r) * splits + split] = s;
  }
}

// --- which drafts are accepted ------------------------------------------------------------------------------------------

// The first column of -inf in a row of nothing but -inf and NaN, by one wave (kNoColumn: none).
template <bool BF16>
__device__ __forceinline__ int first_lowest(const void* row, int vocab) {
  const int lane = threadIdx.x & 63;
#pragma unroll 1
  for (int i = 0; i < vocab; i += 64) {
    const uint64_t low = __ballot(i + lane < vocab && logit<BF16>(row, i + lane) == -__builtin_inff());
    if (low) return i + __builtin_ctzll(low);
  }
  return kNoColumn;
}

// The rows' statistics from their chunks' (the waves take rows in turns, a wave's lanes the chunks).
template <bool BF16, int MODE>
__device__ __forceinline__ void join_rows(const G4VerifyArgs& a, const VerifyWorkspace& w, int b, int rows, int splits, int n,
                                          Stats* out) {
  const int lane = threadIdx.x & 63;
  const float c = kLog2e / a.temperature;
  const Stats none{-__builtin_inff(), 0.f, 0.f, kNoColumn};
  const auto reached = [&](int r) { return r < rows && (r > a.drafts ? r - a.drafts - 1 < n : r <= n); };
  const auto load = [&](int r, int i) { return reached(r) && i < splits ? w.stats[((int64_t)b * rows + r) * splits + i] : none; };
  int r = threadIdx.x >> 6;
  Stats s = load(r, lane);
  for (; r < rows; r += kWaves) {
    const Stats next = load(r + kWaves, lane);
    Stats all = wave_join<MODE>(s, c);
    for (int i = 64; i < splits; i += 64) {  // (joined pairwise: lane 0 the ones before)
      const Stats more = wave_join<MODE>(load(r, i + lane), c);
      all = wave_join<MODE>(lane == 0 ? all : lane == 1 ? more : none, c);
    }
    if (MODE == kUnit) all.unit = all.heat;
    if (MODE == kGreedy && all.idx == kNoColumn && reached(r))  // (uniform) no logit above -inf
      all.idx = first_lowest<BF16>(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, r), a.vocab);
    if (lane == 0 && reached(r)) out[r] = all;
    s = next;
  }
  __syncthreads();
}

// The log-probability of column i of a row under the unscaled logits.
__device__ __forceinline__ float log_prob(float x, const Stats& s) { return (x - s.m) - logf(s.unit); }

// What deciding a draft takes from memory but the statistics (lane s: draft s), asked for before they are joined.
struct Draft {
  int id;
  float x, y, u;  // target's and drafter's logit, the random number
  bool there;     // an id of the vocabulary
};
template <bool BF16, int MODE>
__device__ __forceinline__ Draft load_draft(const G4VerifyArgs& a, int b, int n) {
  const int s = threadIdx.x & 63;
  Draft d{0, 0.f, 0.f, 0.f, false};
  if (s >= n) return d;
  d.id = a.draft_tokens[(int64_t)b * a.drafts + s];
  if constexpr (MODE != kGreedy) d.u = a.uniforms[(int64_t)b * a.drafts + s];
  d.there = (uint32_t)d.id < (uint32_t)a.vocab;
  if (!d.there) return d;
  d.x = logit<BF16>(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, s), d.id);
  if (MODE != kGreedy && a.draft_logits)
    d.y = logit<BF16>(row_at<BF16>(a.draft_logits, a.draft_batch_stride, a.draft_row_stride, b, s), d.id);
  return d;
}

// How many drafts are accepted (by the first wave; lane s decides draft s).
template <bool BF16, int MODE>
__device__ __forceinline__ int accepted(const G4VerifyArgs& a, int n, const Draft& d, const Stats* st) {
  const int s = threadIdx.x & 63;
  bool good = false;
  if (s < n) {
    if constexpr (MODE == kGreedy) {
      good = d.there && d.id == st[s].idx;
    } else if (d.there) {
      // u q < p, both sides times both sums, in 64 bits: neither over- nor underflows where the draft is unlikely
      const double c = 1.0 / (double)a.temperature, p = exp(((double)d.x - st[s].m) * c);
      if (a.draft_logits) {
        const Stats& t = st[a.drafts + 1 + s];
        good = d.u * exp(((double)d.y - t.m) * c) * st[s].heat < p * t.heat;
      } else {
        good = (double)d.u * st[s].heat < p;
      }
    }
  }
  const uint64_t all = __ballot(good);
  return all == ~0ull ? 64 : __builtin_ctzll(~all);
}

// The accepted tokens with their log-probabilities, and what stands behind the last token (by the first wave).
__device__ __forceinline__ void write_accepted(const G4VerifyArgs& a, int b, int count, const Draft& d, const Stats* st) {
  const int s = threadIdx.x & 63;
  if (s == 0) a.count_out[b] = count;
  if (s > a.drafts || s == count) return;
  const int64_t at = (int64_t)b * (a.drafts + 1) + s;
  a.token_out[at] = s < count ? d.id : -1;
  a.logp_out[at] = s < count ? log_prob(d.x, st[s]) : 0.f;
}
template <bool BF16>
__device__ __forceinline__ void write_token(const G4VerifyArgs& a, int b, int count, int token, float m, float unit) {
  const int64_t at = (int64_t)b * (a.drafts + 1) + count;
  a.token_out[at] = token;
  a.logp_out[at] = log_prob(logit<BF16>(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, count), token), Stats{m, 0.f, unit, 0});
}

// The decision on row b by a workgroup, in its LDS; `write`: with the accepted tokens, or greedily all of them, to memory.
struct Decided {
  Stats st[2 * kMaxDrafts + 1];
  Decision made;
};
template <bool BF16, int MODE>
__device__ __forceinline__ void decide(const G4VerifyArgs& a, const VerifyWorkspace& w, int b, int rows, int splits, bool write,
                                       Decided& out) {
  const int n = drafts_of(a, b);
  const Draft draft = load_draft<BF16, MODE>(a, b, threadIdx.x < 64 ? n : 0);
  const Stats* st = out.st;
  join_rows<BF16, MODE>(a, w, b, rows, splits, n, out.st);
  if (threadIdx.x >= 64) return;
  const int count = accepted<BF16, MODE>(a, n, draft, st);
  if (write) write_accepted(a, b, count, draft, st);
  const int id = __shfl(draft.id, count < 63 ? count : 63, 64);
  if (threadIdx.x != 0) return;
  if constexpr (MODE == kGreedy) {
    // (a row of nothing but NaN has no largest)
    write_token<BF16>(a, b, count, st[count].idx != kNoColumn ? st[count].idx : 0, st[count].m, st[count].unit);
  } else {
    const bool rejected = count < n, residual = rejected && a.draft_logits;
    const Stats &p = st[count], &q = st[residual ? a.drafts + 1 + count : count];
    out.made = Decision{count, rejected && !residual ? id : -1, residual, p.unit, p.m, p.heat, q.m, q.heat};
  }
}

// --- second launch: the decision, one workgroup per b -----------------------------------------------------------------------

// Where the race has few workgroups each decides for itself, and this launch is saved: 1 row of 4 drafts over 262144 logits (64
// workgroups) 13.0 -> 11.4 us, 16 rows (1024) 31.0 -> 29.6; 32 rows 46.2 -> 47.6, 64 rows 76.8 -> 80.5.
constexpr int kOwn = 1024;
template <bool BF16, int MODE>
__global__ __launch_bounds__(kThreads) void verify_decide_kernel(G4VerifyArgs a, VerifyWorkspace w, int rows, int splits) {
  __shared__ Decided decided;
  decide<BF16, MODE>(a, w, blockIdx.x, rows, splits, true, decided);
  if (MODE != kGreedy && threadIdx.x == 0) w.made[blockIdx.x] = decided.made;
}

// --- third launch: the race, a chunk per workgroup ----------------------------------------------------------------------

// 1 / -log(u), the factor of a weight in the race; 0 for u = 0 and outside [0, 1).
__device__ __forceinline__ float pace(float u) {
  return u >= kF32Tiny && u < 1.f ? __builtin_amdgcn_rcpf(-log_pos_normal(u)) : 0.f;
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

// A row's probabilities, roughly and well: the rough ones are within 1e-5 of the others.
struct Row {
  const void* at;
  float m, inv;
  Below rough;
  __device__ __forceinline__ Row(const void* p, float m_, float z, float c) : at(p), m(m_), inv(1.0f / z), rough(m_, c) {
    rough.rest *= inv;
  }
  __device__ __forceinline__ float well(const Heat& heat, float x) const { return heat.exp(x - m) * inv; }
};

// The race is decided by scores within a few f32 ulps, which take some 50 instructions each. Rough ones take 15 and give
// each score's bounds; an element whose upper bound is below the workgroup's largest lower one is out: one per
// workgroup remains, or a few. (64 rows of 262144: 55 -> 29 us.)
template <bool BF16, int MODE, int VECS, bool OWN>
__global__ __launch_bounds__(kThreads) void verify_race_kernel(G4VerifyArgs a, VerifyWorkspace w, Heat heat, int splits, int rows,
                                                               int stats_splits) {
  __shared__ uint64_t best_of[kWaves];
  __shared__ float bars[kWaves];
  __shared__ bool last;
  const int split = blockIdx.x % splits, b = blockIdx.x / splits, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t i0 = (int64_t)split * (VECS * kThreads * 8) + threadIdx.x * 8;
  constexpr int STEP = kThreads * 8;
  const float* noise = a.noise + b * a.noise_stride;
  const bool whole = (int64_t)(split + 1) * (VECS * STEP) <= a.vocab;  // (uniform) else a chunk that ends inside: load8
  Eight<false> us[VECS];
  if (whole) {
#pragma unroll
    for (int v = 0; v < VECS; ++v) us[v].load(noise, i0 + v * STEP);
  }
  Decision d;
  if constexpr (OWN) {
    __shared__ Decided decided;
    decide<BF16, MODE>(a, w, b, rows, stats_splits, split == 0, decided);
    __syncthreads();
    d = decided.made;
  } else {
    d = w.made[b];
  }
  const bool residual = d.residual;
  const int64_t away = d.away;
  const Row p(row_at<BF16>(a.logits, a.batch_stride, a.row_stride, b, d.count), d.pm, d.pz, heat.hi);
  const Row q(residual ? row_at<BF16>(a.draft_logits, a.draft_batch_stride, a.draft_row_stride, b, d.count) : nullptr, d.qm, d.qz,
              heat.hi);
  float u[VECS][8], x[VECS][8], y[VECS][8];
  if (whole) {
    Eight<BF16> xs[VECS], ys[VECS];
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      xs[v].load(p.at, i0 + v * STEP);
      if (residual) ys[v].load(q.at, i0 + v * STEP);
    }
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      us[v].values(u[v]);
      xs[v].values(x[v]);
      if (residual) ys[v].values(y[v]);
    }
  } else {
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int64_t i = i0 + v * STEP;
      const int n = (int)min((int64_t)8, a.vocab - i);
      load8<false>(noise, i, n, u[v]);
      load8<BF16>(p.at, i, n, x[v]);
      if (residual) load8<BF16>(q.at, i, n, y[v]);
    }
  }
  // ln 2 times the scores' bounds (the pace by log2): the rough probabilities are within 1e-5, and q <= p where r >= 0
  const bool tame = p.rough.tame() && q.rough.tame();  // else there are none, and every element may win
  float high[VECS][8], bar = 0.f;
#pragma unroll
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float pr = p.rough.exp(x[v][e]) * p.rough.rest;
      float r = pr;
      if (residual) r = fmaf(-q.rough.exp(y[v][e]), q.rough.rest, pr);
      else if (i0 + v * STEP + e == away) r = 0.f;
      const float g = u[v][e] < 1.f ? -__builtin_amdgcn_rcpf(__builtin_amdgcn_logf(u[v][e])) : 0.f;
      high[v][e] = fmaf(pr, 4e-5f, r) * g;
      bar = fmaxf(bar, fmaf(pr, -4e-5f, r) * g);
    }
  bar = wave_max(bar);
  if (lane == 0) bars[wave] = bar;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kWaves; ++i) bar = fmaxf(bar, bars[i]);
  bar *= 0.9999f;
  uint32_t mask = 0;  // this lane's elements that may win
#pragma unroll
  for (int v = 0; v < VECS; ++v)
#pragma unroll
    for (int e = 0; e < 8; ++e) mask |= high[v][e] >= bar || !tame ? 1u << (v * 8 + e) : 0u;
  uint64_t top = 0;
  while (mask) {
    const int j = __builtin_ctz(mask);
    mask &= mask - 1;
    const int64_t i = i0 + (j >> 3) * STEP + (j & 7);
    if (i >= a.vocab) continue;
    const float pw = p.well(heat, logit<BF16>(p.at, i));
    float r = pw;
    if (residual) r = fmaxf(pw - q.well(heat, logit<BF16>(q.at, i)), 0.f);
    else if (i == away) r = 0.f;
    const uint64_t k = entry(r * pace(noise[i]), i);
    top = k > top ? k : top;
  }
  top = wave_top(top);
  if (lane == 0) best_of[wave] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int i = 1; i < kWaves; ++i) top = best_of[i] > top ? best_of[i] : top;
    // The best is in memory, where every XCD sees it, once the store has returned; only then is the arrival counted. (With
    // fences instead, each workgroup writes its L2 back: 85 us in all.)
    __hip_atomic_store(w.best + blockIdx.x, top, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __asm__ volatile("s_waitcnt vmcnt(0)" ::: "memory");
    last = __hip_atomic_fetch_add(w.arrived + (int64_t)b * kApart, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (uint32_t)splits - 1;
  }
  __syncthreads();
  if (!last) return;
  top = 0;
  for (int i = lane; i < splits; i += 64) {  // (every wave all of them)
    const uint64_t k = __hip_atomic_load(w.best + (int64_t)b * splits + i, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    top = k > top ? k : top;
  }
  top = wave_top(top);
  if (top == 0) {  // (uniform) no weight is left, p = q but for rounding: from p, by this workgroup alone
    for (int64_t i = threadIdx.x; i < a.vocab; i += kThreads) {
      const uint64_t k = entry(p.well(heat, logit<BF16>(p.at, i)) * pace(noise[i]), i);
      top = k > top ? k : top;
    }
    top = wave_top(top);
    __syncthreads();
    if (lane == 0) best_of[wave] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kWaves; ++i) top = best_of[i] > top ? best_of[i] : top;
  }
  if (threadIdx.x == 0) write_token<BF16>(a, b, d.count, top ? (int)(0xffffffffu - (uint32_t)top) : 0, d.pm, d.unit);
}

template <bool BF16, int MODE, int VECS, int TIMES>
int launch_verify(const G4VerifyArgs& a, const VerifyWorkspace& w, hipStream_t st) {
  static const char who[] = "g4_verify_draft";
  const int splits = splits_of(a, VECS * TIMES), rows = a.drafts + 1 + (MODE != kGreedy && a.draft_logits ? a.drafts : 0);
  const int race = splits_of(a, kRace);
  const int64_t blocks = (int64_t)a.batch * rows * splits, racers = (int64_t)a.batch * race;  // (either may be the larger grid)
  if (std::max(blocks, MODE == kGreedy ? 0 : racers) * kThreads > 0xffffffffLL) return fail(G4_ERR_UNSUPPORTED, "%s: too many logits", who);
  hipLaunchKernelGGL((verify_stats_kernel<BF16, MODE, VECS, TIMES>), dim3((unsigned)blocks), dim3(kThreads), 0, st, a, w, rows, splits);
  int rc = check_launch(who);
  if (rc != G4_OK) return rc;
  const double c = 1.4426950408889634074 / (double)a.temperature;
  const Heat heat{(float)c, (float)(c - (double)(float)c)};
  if (MODE == kGreedy || racers > kOwn) {
    hipLaunchKernelGGL((verify_decide_kernel<BF16, MODE>), dim3((unsigned)a.batch), dim3(kThreads), 0, st, a, w, rows, splits);
    if ((rc = check_launch(who)) != G4_OK) return rc;
  }
  if constexpr (MODE != kGreedy) {
    const auto kernel = racers > kOwn ? verify_race_kernel<BF16, MODE, kRace, false> : verify_race_kernel<BF16, MODE, kRace, true>;
    hipLaunchKernelGGL(kernel, dim3((unsigned)racers), dim3(kThreads), 0, st, a, w, heat, race, rows, splits);
    rc = check_launch(who);
  }
  return rc;
}

template <bool BF16, int MODE>
int launch_verify(const G4VerifyArgs& a, const VerifyWorkspace& w, hipStream_t st) {
  return vecs_of(a) == kLong ? launch_verify<BF16, MODE, kStep, kSteps>(a, w, st) : launch_verify<BF16, MODE, kShort, 1>(a, w, st);
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
