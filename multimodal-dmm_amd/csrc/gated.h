// Device helpers of the gated recurrence and the block norms (gated_scan.hip, block_norm.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/mdmm_hip.h"

namespace mdmm {

__device__ __forceinline__ float load1(const float* p) { return *p; }
__device__ __forceinline__ float load1(const __bf16* p) { return (float)*p; }
__device__ __forceinline__ void store1(float* p, float v) { *p = v; }
__device__ __forceinline__ void store1(__bf16* p, float v) { *p = (__bf16)v; }     // (to nearest, ties to even)

// a = sigmoid(f) and k = 1 - a, both to fp32 accuracy: e = exp(-|f|) never overflows, and the smaller of the two is formed
// as e / (1 + e), not as a difference from 1 (at f = 10 the difference keeps 9 bits of k)
struct Gate {
  float a, k;
  __device__ __forceinline__ explicit Gate(float f) {
    // exp(-x) = 2^(y + d), y = -x log2(e) rounded and d what the rounding dropped (without d the relative error of e
    // grows with x: 1e-6 at x = 15); beyond 200 e is 0 in fp32, and the bound keeps an infinite f out of y's difference
    const float m = fabsf(f), x = m > 200.0f ? 200.0f : m;
    const float y = x * -1.44269504088896341f;
    const float d = fmaf(x, -1.44269504088896341f, -y) + x * -1.92596299e-8f;
    const float e0 = __builtin_amdgcn_exp2f(y);
    const float e = fmaf(e0, d * 0.69314718055994531f, e0);
    const float r = __builtin_amdgcn_rcpf(1.0f + e), s = e * r;
    a = f >= 0.0f ? r : s;
    k = f >= 0.0f ? s : r;
  }
};

// exp(-x) as 2^y (1 + d ln(2)) with Gate's y and d, of any size (infinite from x = -89 on); an infinite x, which has no d, as 200
__device__ __forceinline__ float exp_neg(float x) {
  x = __builtin_amdgcn_fmed3f(x, -200.0f, 200.0f);
  const float y = x * -1.44269504088896341f;
  const float d = fmaf(x, -1.44269504088896341f, -y);
  return __builtin_amdgcn_exp2f(y) * fmaf(x, -1.92596299e-8f * 0.69314718055994531f, fmaf(d, 0.69314718055994531f, 1.0f));
}

// sigmoid alone, accurate wherever x lies (1 / (1 + 2^(-x log2(e))) is off by 6e-8 (1 + |x|) of itself)
__device__ __forceinline__ float sigmoid_(float x) { return __builtin_amdgcn_rcpf(1.0f + exp_neg(x)); }

// Host side.  The bytes that `rows` rows of n elements of `size` bytes take, `step` elements apart; whether two regions meet
struct Region { const char* at; int64_t bytes; };
inline Region region(const void* p, int64_t rows, int64_t step, int64_t n, int64_t size) {
  return {(const char*)p, p ? ((rows - 1) * step + n) * size : 0};
}
inline bool meet(const Region& a, const Region& b) { return a.at && b.at && a.at < b.at + b.bytes && b.at < a.at + a.bytes; }

// h_last, written while other workgroups still read, shares memory with an input (one that is h0 itself, a time step in place,
// does not: a thread writes what it alone has read)
inline bool last_state_on_input(const mdmm_gated_scan_t* a) {
  if (!a->h_last) return false;
  const Region last = region(a->h_last, a->B, a->H, a->H, 4);
  const bool in_place = a->T == 1 && a->h_last == a->h0 && a->h0_sb == a->H;
  if (!in_place && meet(last, region(a->h0, a->B, a->h0_sb, a->H, 4))) return true;
  const int64_t es = a->gates_bf16 ? 2 : 4, past = (a->T - 1) * a->gates_st, mpast = (a->T - 1) * a->mask_st;
  Region gates = region(a->gates, a->B, a->gates_sb, 2 * (int64_t)a->H, es), mask = region(a->mask, a->B, a->mask_sb, 1, 1);
  gates.at += (past < 0 ? past : 0) * es;
  gates.bytes += (past < 0 ? -past : past) * es;
  mask.at += mask.at && mpast < 0 ? mpast : 0;
  mask.bytes += mpast < 0 ? -mpast : mpast;
  return meet(last, gates) || meet(last, mask);
}

}  // namespace mdmm
