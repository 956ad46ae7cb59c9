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

// sigmoid alone, to the same accuracy wherever x lies (1 / (1 + 2^(-x log2(e))) is off by 6e-8 (1 + |x|) of itself)
__device__ __forceinline__ float sigmoid_(float x) { return Gate(x).a; }

}  // namespace mdmm
