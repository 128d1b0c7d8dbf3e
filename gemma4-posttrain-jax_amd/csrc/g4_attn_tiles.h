// Products of the LDS-staged attention kernels over whole prompts (g4_prefill_lds.h, g4_packed.hip): MFMA
// 16x16x32 operand tiles of 1 KiB read from LDS through a rolling window, requested right after the MFMAs that free
// their registers, so that the LDS latency hides behind the MFMAs in flight.
#pragma once

#include "g4_common.h"

namespace g4 {

template <int N>
__device__ __forceinline__ void wait_vmcnt() {
  __asm__ volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}

// S^T of one chunk for the wave's NB column blocks: K operand tiles (KT = 2 halves x KS d-slices,
// 1 KiB each, this lane's pieces from LDS address kbase) against the q operands in registers, a rolling window of WIN
// tiles in flight (each read waited for right before its MFMAs; the chunk's DMA is covered by the
// caller's vmcnt wait + barrier).
template <int KT, int KS, int NB, int WIN>
__device__ __forceinline__ void pf_qk(uint32_t kbase, const bf16x8 (&qop)[NB][KS], floatx4 (&acc)[NB][2]) {
  static_assert(WIN >= 1 && WIN <= 8 && WIN <= KT, "window of LDS reads (lgkm_wait counts up to 7)");
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int cb = 0; cb < NB; ++cb) acc[cb][0] = acc[cb][1] = floatx4{0.f, 0.f, 0.f, 0.f};
  u32x4 kv[WIN];
#pragma unroll
  for (int j = 0; j < WIN; ++j) kv[j] = lds_read16_at(kbase, 1024 * j);
#pragma unroll
  for (int t = 0; t < KT; ++t) {
    const int bb = t / KS, s = t - bb * KS;
    const int later = KT - 1 - t < WIN - 1 ? KT - 1 - t : WIN - 1;  // reads issued after tile t's
    lgkm_wait(later, kv[t % WIN]);
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) acc[cb][bb] = mfma16x16x32(as_bf16x8(kv[t % WIN]), qop[cb][s], acc[cb][bb]);
    if (t + WIN < KT) kv[t % WIN] = lds_read16_at(kbase, 1024 * (t + WIN));
  }
  __builtin_amdgcn_sched_barrier(0);
}

// O^T += V^T P^T over one chunk: VT value operand tiles (one per 16-dim block, 1 KiB each, this
// lane's pieces from LDS address vbase) against the wave's probabilities, a rolling window of WIN tiles in flight.
template <int VT, int NB, int WIN>
__device__ __forceinline__ void pf_pv(uint32_t vbase, const bf16x8 (&pop)[NB], floatx4 (&oacc)[NB][VT]) {
  static_assert(WIN >= 1 && WIN <= 8 && WIN <= VT, "window of LDS reads (lgkm_wait counts up to 7)");
  __builtin_amdgcn_sched_barrier(0);
  u32x4 vv[WIN];
#pragma unroll
  for (int i = 0; i < WIN; ++i) vv[i] = lds_read16_at(vbase, 1024 * i);
#pragma unroll
  for (int i = 0; i < VT; ++i) {
    const int later = VT - 1 - i < WIN - 1 ? VT - 1 - i : WIN - 1;
    lgkm_wait(later, vv[i % WIN]);
#pragma unroll
    for (int cb = 0; cb < NB; ++cb) oacc[cb][i] = mfma16x16x32(as_bf16x8(vv[i % WIN]), pop[cb], oacc[cb][i]);
    if (i + WIN < VT) vv[i % WIN] = lds_read16_at(vbase, 1024 * (i + WIN));
  }
  __builtin_amdgcn_sched_barrier(0);
}

}  // namespace g4
