// Gated linear recurrence over time: h_t = a_t h_{t-1} + k_t c_t with a_t = sigmoid(f_t), k_t = 1 - a_t, per channel; a step
// whose mask byte is 0 leaves h as it is (a = 1, k = 0).  Backward: G_t = g_t + a_{t+1} G_{t+1} (g = the gradient of h_t),
// dc = G k, df = G (h_{t-1} - c) a k, dh0 = a_0 G_0.
//
// Bound by HBM: forward reads f, c and writes h, backward reads f, c, g and writes df, dc; neither keeps h (the backward
// pass forms it again from one state per tile of time).  A step h -> a h + b composes, (a2, b2)(a1, b1) = (a2 a1, a2 b1 + b2), so time is
// taken in tiles: a workgroup of up to 8 waves holds 64 VEC channels and a tile of 8 waves x 8 steps in registers, each wave
// composes its 8 steps, the pieces meet in LDS, and every wave then runs its steps from the state in front of them.  Every
// load of a tile is in flight at once, each tensor passes once, and the next tile's loads are issued before the present
// tile's are used up.  Where the channels alone do not fill the chip, time is also split over workgroups: a first launch
// composes each split (reading f, c once more; backward f, g), the second starts each split from the splits in front of it.
// Nothing waits for another workgroup, and no sum is formed by atomics: results do not depend on the schedule.
#include "gated.h"

namespace mdmm {
namespace {

constexpr int S = 8, WMAX = 8, TILE = S * WMAX;      // steps of a wave, waves, steps of a tile

template <typename IO, int VEC> struct Raw;          // VEC elements as loaded
template <> struct Raw<float, 1> { float x; };
template <> struct Raw<float, 2> { float2 x; };
template <> struct Raw<float, 4> { float4 x; };
template <> struct Raw<__bf16, 1> { unsigned short x; };
template <> struct Raw<__bf16, 2> { unsigned x; };
template <> struct Raw<__bf16, 4> { uint2 x; };

__device__ __forceinline__ void widen(const Raw<float, 1>& r, float* v) { v[0] = r.x; }
__device__ __forceinline__ void widen(const Raw<float, 2>& r, float* v) { v[0] = r.x.x; v[1] = r.x.y; }
__device__ __forceinline__ void widen(const Raw<float, 4>& r, float* v) { v[0] = r.x.x; v[1] = r.x.y; v[2] = r.x.z; v[3] = r.x.w; }
__device__ __forceinline__ void widen(const Raw<__bf16, 1>& r, float* v) { v[0] = __uint_as_float((unsigned)r.x << 16); }
__device__ __forceinline__ void widen2(unsigned x, float* v) { v[0] = __uint_as_float(x << 16); v[1] = __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ void widen(const Raw<__bf16, 2>& r, float* v) { widen2(r.x, v); }
__device__ __forceinline__ void widen(const Raw<__bf16, 4>& r, float* v) { widen2(r.x.x, v); widen2(r.x.y, v + 2); }

template <int VEC> __device__ __forceinline__ void put(float* p, const float* v) {
  Raw<float, VEC> r;
  __builtin_memcpy(&r, v, sizeof r);
  *(Raw<float, VEC>*)p = r;
}
template <int VEC> __device__ __forceinline__ void put(__bf16* p, const float* v) {
  __bf16 t[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) t[e] = (__bf16)v[e];
  Raw<__bf16, VEC> r;
  __builtin_memcpy(&r, t, sizeof r);
  *(Raw<__bf16, VEC>*)p = r;
}

struct Plan {
  int vec, waves, splits;
  int64_t chunks;              // VEC-wide pieces of a row of H channels
  int64_t wgs;                 // workgroups over the channels
  int64_t tiles, per;          // tiles of time, tiles of a split
};

// A thread's channels: VEC neighbours of one sequence
struct Lane {
  int64_t b, j, q;             // sequence, first channel, flat index b H + j
  bool live;
  template <int VEC> __device__ __forceinline__ void at(const mdmm_gated_scan_t& p, int64_t chunks, int lane) {
    int64_t i = (int64_t)blockIdx.x * 64 + lane;
    live = i < chunks * p.B;
    if (!live) i = 0;          // (loads stay in bounds; nothing is stored)
    b = i / chunks;
    j = (i - b * chunks) * VEC;
    q = b * p.H + j;
  }
};

__device__ __forceinline__ int64_t time_of(const mdmm_gated_scan_t& p, int64_t i) { return p.reverse ? p.T - 1 - i : i; }

// raw f, c of a wave's 8 steps from step i0 on (steps past the end: the last one's, not used), mask bits in `on`
template <typename IO, int VEC, bool C>
__device__ __forceinline__ unsigned fetch(const mdmm_gated_scan_t& p, const Lane& l, int64_t i0, Raw<IO, VEC>* f, Raw<IO, VEC>* c) {
  unsigned on = 0;
#pragma unroll
  for (int s = 0; s < S; ++s) {
    const int64_t i = i0 + s < p.T ? i0 + s : p.T - 1, t = time_of(p, i);
    const IO* row = (const IO*)p.gates + t * p.gates_st + l.b * p.gates_sb + l.j;
    f[s] = *(const Raw<IO, VEC>*)row;
    if (C) c[s] = *(const Raw<IO, VEC>*)(row + p.H);
    if (i0 + s < p.T && (!p.mask || p.mask[t * p.mask_st + l.b * p.mask_sb])) on |= 1u << s;
  }
  return on;
}

// a state (prefix) in front of split `z`: the composition of the splits before it applied to the start
template <int VEC>
__device__ __forceinline__ void lead_in(const float* ws, int64_t stride, int z, bool from_end, int splits, int64_t q, float* h) {
  const int n = from_end ? splits - 1 - z : z;
#pragma unroll 4
  for (int i = 0; i < n; ++i) {
    const float* a = ws + 2 * stride * (from_end ? splits - 1 - i : i) + q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] = fmaf(a[e], h[e], a[stride + e]);
  }
}

// Composition of each split: BWD of D -> a (g + D) from its last step to its first, else of h -> a h + k c
template <typename IO, typename HO, int VEC, bool BWD>
__global__ __launch_bounds__(64 * WMAX) void scan_split_kernel(mdmm_gated_scan_t p, Plan pl) {
  __shared__ float sa[WMAX][64 * VEC], sb[WMAX][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = pl.waves;
  Lane l;
  l.at<VEC>(p, pl.chunks, lane);
  const int64_t t0 = blockIdx.y * pl.per, t1 = t0 + pl.per < pl.tiles ? t0 + pl.per : pl.tiles;
  // a wave composes every step of its own, tile by tile (they interleave with the other waves'), so the order over the split
  // is kept by giving each wave one run of consecutive tiles
  const int64_t run = (t1 - t0 + W - 1) / W;
  const int64_t u0 = t0 + wave * run < t1 ? t0 + wave * run : t1, u1 = u0 + run < t1 ? u0 + run : t1;
  float A[VEC], B[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; }
  const int64_t first = u0 * TILE, last = u1 * TILE < p.T ? u1 * TILE : p.T;
  for (int64_t i = first; i < last; i += S) {
    const int64_t i0 = BWD ? first + (last - 1 - i) / S * S : i;       // (first + a multiple of S, walked downwards)
    Raw<IO, VEC> f[S], c[S];
    Raw<HO, VEC> g[S];
    const unsigned on = fetch<IO, VEC, !BWD>(p, l, i0, f, c);
    if (BWD && p.g_h) {
#pragma unroll
      for (int s = 0; s < S; ++s) {
        const int64_t t = time_of(p, i0 + s < p.T ? i0 + s : p.T - 1);
        g[s] = *(const Raw<HO, VEC>*)((const HO*)p.g_h + t * p.B * p.H + l.q);
      }
    }
#pragma unroll
    for (int s_ = 0; s_ < S; ++s_) {
      const int s = BWD ? S - 1 - s_ : s_;
      float fv[VEC], cv[VEC], gv[VEC];
      widen(f[s], fv);
      if (!BWD) widen(c[s], cv);
      if (BWD && p.g_h) widen(g[s], gv);
      const bool in = on >> s & 1, some = i0 + s < last;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Gate x(fv[e]);
        const float a = in ? x.a : 1.0f;
        if (BWD) {
          if (some) B[e] = a * ((p.g_h ? gv[e] : 0.0f) + B[e]);
        } else B[e] = in ? fmaf(x.a, B[e], x.k * cv[e]) : B[e];
        A[e] *= a;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) { sa[wave][e * 64 + lane] = A[e]; sb[wave][e * 64 + lane] = B[e]; }
  __syncthreads();
  if (wave == 0 && l.live) {
    const int64_t stride = (int64_t)p.B * p.H;
    float* out = p.ws + 2 * stride * blockIdx.y + l.q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      float a = 1.0f, b = 0.0f;
      for (int w_ = 0; w_ < W; ++w_) {
        const int w = BWD ? W - 1 - w_ : w_;
        b = fmaf(sa[w][e * 64 + lane], b, sb[w][e * 64 + lane]);
        a *= sa[w][e * 64 + lane];
      }
      out[e] = a;
      out[stride + e] = b;
    }
  }
}

template <typename IO, typename HO, int VEC>
__global__ __launch_bounds__(64 * WMAX) void scan_fwd_kernel(mdmm_gated_scan_t p, Plan pl) {
  __shared__ float sa[2][WMAX][64 * VEC], sb[2][WMAX][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = pl.waves;
  Lane l;
  l.at<VEC>(p, pl.chunks, lane);
  const int64_t stride = (int64_t)p.B * p.H;
  const int64_t t0 = blockIdx.y * pl.per, t1 = t0 + pl.per < pl.tiles ? t0 + pl.per : pl.tiles;
  float h0[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) h0[e] = p.h0 ? p.h0[l.b * p.h0_sb + l.j + e] : 0.0f;
  lead_in<VEC>(p.ws, stride, blockIdx.y, false, pl.splits, l.q, h0);
  Raw<IO, VEC> f[S], c[S];
  unsigned on = fetch<IO, VEC, true>(p, l, t0 * TILE + wave * S, f, c);
  for (int64_t tile = t0; tile < t1; ++tile) {
    const int64_t i0 = tile * TILE + wave * S;
    float a[S][VEC], b[S][VEC], A[VEC], B[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float fv[VEC], cv[VEC];
      widen(f[s], fv);
      widen(c[s], cv);
      const bool in = on >> s & 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Gate x(fv[e]);
        a[s][e] = in ? x.a : 1.0f;
        b[s][e] = in ? x.k * cv[e] : 0.0f;
        B[e] = fmaf(a[s][e], B[e], b[s][e]);
        A[e] *= a[s][e];
      }
    }
    if (tile + 1 < t1) on = fetch<IO, VEC, true>(p, l, i0 + TILE, f, c);
    const int z = tile & 1;
    if (W > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) { sa[z][wave][e * 64 + lane] = A[e]; sb[z][wave][e * 64 + lane] = B[e]; }
      __syncthreads();         // (two sets of pieces: a wave a tile ahead writes the other one)
    }
    if (p.states && wave == 0 && l.live) put<VEC>(p.states + tile * stride + l.q, h0);
    float h[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] = h0[e];
    if (W > 1) {
      for (int w = 0; w < W; ++w) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          h0[e] = fmaf(sa[z][w][e * 64 + lane], h0[e], sb[z][w][e * 64 + lane]);
          if (w + 1 == wave) h[e] = h0[e];
        }
      }
    }
#pragma unroll
    for (int s = 0; s < S; ++s) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[e] = fmaf(a[s][e], h[e], b[s][e]);
      if (i0 + s < p.T && l.live) put<VEC>((HO*)p.h + time_of(p, i0 + s) * stride + l.q, h);
    }
    if (W == 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) h0[e] = h[e];
    }
  }
  if (p.h_last && t1 == pl.tiles && wave == 0 && l.live) put<VEC>(p.h_last + l.q, h0);
}

template <typename IO, typename HO, int VEC>
__global__ __launch_bounds__(64 * WMAX) void scan_bwd_kernel(mdmm_gated_scan_t p, Plan pl) {
  __shared__ float sa[2][WMAX][64 * VEC], sb[2][WMAX][64 * VEC], sg[2][WMAX][64 * VEC];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, W = pl.waves;
  Lane l;
  l.at<VEC>(p, pl.chunks, lane);
  const int64_t stride = (int64_t)p.B * p.H;
  const int64_t t0 = blockIdx.y * pl.per, t1 = t0 + pl.per < pl.tiles ? t0 + pl.per : pl.tiles;
  float d0[VEC];               // a G of the step behind the present tile
#pragma unroll
  for (int e = 0; e < VEC; ++e) d0[e] = p.g_last ? p.g_last[l.q + e] : 0.0f;
  lead_in<VEC>(p.ws, stride, blockIdx.y, true, pl.splits, l.q, d0);
  for (int64_t tile = t1 - 1; tile >= t0; --tile) {
    const int64_t i0 = tile * TILE + wave * S;
    Raw<IO, VEC> f[S], c[S];
    Raw<HO, VEC> g[S];
    const unsigned on = fetch<IO, VEC, true>(p, l, i0, f, c);
#pragma unroll
    for (int s = 0; s < S; ++s) {
      g[s] = Raw<HO, VEC>{};
      if (p.g_h && i0 + s < p.T) g[s] = *(const Raw<HO, VEC>*)((const HO*)p.g_h + time_of(p, i0 + s) * stride + l.q);
    }
    float hs[VEC];             // the state in front of the tile
#pragma unroll
    for (int e = 0; e < VEC; ++e)
      hs[e] = p.states ? p.states[tile * stride + l.q + e] : p.h0 ? p.h0[l.b * p.h0_sb + l.j + e] : 0.0f;
    float a[S][VEC], k[S][VEC], A[VEC], B[VEC], D[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; D[e] = 0.0f; }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float fv[VEC], cv[VEC];
      widen(f[s], fv);
      widen(c[s], cv);
      const bool in = on >> s & 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Gate x(fv[e]);
        a[s][e] = in ? x.a : 1.0f;
        k[s][e] = in ? x.k : 0.0f;
        B[e] = fmaf(a[s][e], B[e], in ? k[s][e] * cv[e] : 0.0f);
        A[e] *= a[s][e];
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      float gv[VEC];
      widen(g[s], gv);
#pragma unroll
      for (int e = 0; e < VEC; ++e) D[e] = a[s][e] * (gv[e] + D[e]);
    }
    float h[VEC], d[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { h[e] = hs[e]; d[e] = d0[e]; }
    const int z = tile & 1;
    if (W > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        sa[z][wave][e * 64 + lane] = A[e];
        sb[z][wave][e * 64 + lane] = B[e];
        sg[z][wave][e * 64 + lane] = D[e];
      }
      __syncthreads();
      for (int w = 0; w < W; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (w < wave) h[e] = fmaf(sa[z][w][e * 64 + lane], h[e], sb[z][w][e * 64 + lane]);
      for (int w = W - 1; w >= 0; --w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          d0[e] = fmaf(sa[z][w][e * 64 + lane], d0[e], sg[z][w][e * 64 + lane]);
          if (w - 1 == wave) d[e] = d0[e];
        }
    } else {
#pragma unroll
      for (int e = 0; e < VEC; ++e) d0[e] = fmaf(A[e], d0[e], D[e]);
    }
    float before[S][VEC];      // h_{t-1} - c_t
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float cv[VEC];
      widen(c[s], cv);
      const bool in = on >> s & 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        before[s][e] = in ? h[e] - cv[e] : 0.0f;
        h[e] = in ? fmaf(a[s][e], h[e], k[s][e] * cv[e]) : h[e];
      }
    }
#pragma unroll
    for (int s = S - 1; s >= 0; --s) {
      float gv[VEC], df[VEC], dc[VEC];
      widen(g[s], gv);
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float G = gv[e] + d[e];
        dc[e] = G * k[s][e];
        df[e] = dc[e] * a[s][e] * before[s][e];
        d[e] = a[s][e] * G;
      }
      if (i0 + s < p.T && l.live) {
        IO* out = (IO*)p.g_gates + time_of(p, i0 + s) * p.g_gates_st + l.b * p.g_gates_sb + l.j;
        put<VEC>(out, df);
        put<VEC>(out + p.H, dc);
      }
    }
  }
  if (p.g_h0 && t0 == 0 && wave == 0 && l.live) put<VEC>(p.g_h0 + l.q, d0);
}

int check(const mdmm_gated_scan_t* a) {
  if (!a || a->T < 0 || a->B < 0 || a->H < 0) return MDMM_E_ARG;
  if (!a->gates_bf16 && a->h_bf16) return MDMM_E_ARG;
  if (a->T > 0 && a->B > 0 && a->H > 0 && !a->gates) return MDMM_E_ARG;
  return 0;
}

bool none(const mdmm_gated_scan_t* a) { return a->T == 0 || a->B == 0 || a->H == 0; }

Plan plan(const mdmm_gated_scan_t* a, bool bwd) {
  Plan p;
  const uintptr_t es = a->gates_bf16 ? 2 : 4, hs = a->h_bf16 ? 2 : 4;
  auto fits = [&](int v) {
    const uintptr_t m = (uintptr_t)v * es - 1, mh = (uintptr_t)v * hs - 1, m4 = (uintptr_t)v * 4 - 1;
    return a->H % v == 0 && ((uintptr_t)a->gates & m) == 0 && a->gates_st % v == 0 && a->gates_sb % v == 0 &&
           ((uintptr_t)a->h & mh) == 0 && ((uintptr_t)a->g_h & mh) == 0 && ((uintptr_t)a->g_gates & m) == 0 &&
           a->g_gates_st % v == 0 && a->g_gates_sb % v == 0 && ((uintptr_t)a->states & m4) == 0 &&
           ((uintptr_t)a->h_last & m4) == 0 && ((uintptr_t)a->g_h0 & m4) == 0;
  };
  p.vec = fits(2) ? 2 : 1;
  if (!bwd && fits(4) && (int64_t)a->B * a->H >= 64 * 4 * 512) p.vec = 4;
  p.chunks = a->H / p.vec;
  p.wgs = (p.chunks * a->B + 63) / 64;
  const int64_t waves = (a->T + S - 1) / S;
  p.waves = (int)(waves < WMAX ? waves : WMAX);
  p.tiles = ((int64_t)a->T + TILE - 1) / TILE;
  int64_t splits = 1;
  if (p.wgs < 512 && p.tiles > 1) {
    splits = (1024 + p.wgs - 1) / p.wgs;
    if (splits > p.tiles) splits = p.tiles;
    if (splits > 64) splits = 64;
  }
  p.per = (p.tiles + splits - 1) / splits;
  p.splits = (int)((p.tiles + p.per - 1) / p.per);
  return p;
}

template <typename IO, typename HO>
int launch(const mdmm_gated_scan_t* a, const Plan& pl, bool bwd, hipStream_t s) {
  const dim3 grid((unsigned)pl.wgs, (unsigned)pl.splits), block(64 * pl.waves);
#define RUN(K) hipLaunchKernelGGL(K, grid, block, 0, s, *a, pl)
  if (bwd) {
    if (pl.splits > 1) {
      if (pl.vec == 1) RUN((scan_split_kernel<IO, HO, 1, true>)); else RUN((scan_split_kernel<IO, HO, 2, true>));
    }
    if (pl.vec == 1) RUN((scan_bwd_kernel<IO, HO, 1>)); else RUN((scan_bwd_kernel<IO, HO, 2>));
  } else {
    if (pl.splits > 1) {
      if (pl.vec == 1) RUN((scan_split_kernel<IO, HO, 1, false>)); else RUN((scan_split_kernel<IO, HO, 2, false>));
    }
    if (pl.vec == 1) RUN((scan_fwd_kernel<IO, HO, 1>));
    else if (pl.vec == 2) RUN((scan_fwd_kernel<IO, HO, 2>));
    else RUN((scan_fwd_kernel<IO, HO, 4>));
  }
#undef RUN
  return (int)hipGetLastError();
}

int run(const mdmm_gated_scan_t* a, bool bwd, hipStream_t s) {
  const Plan pl = plan(a, bwd);
  if (pl.wgs > 0x7fffffff) return MDMM_E_LIMIT;
  if (pl.splits > 1 && !a->ws) return MDMM_E_ARG;
  if (!a->gates_bf16) return launch<float, float>(a, pl, bwd, s);
  return a->h_bf16 ? launch<__bf16, __bf16>(a, pl, bwd, s) : launch<__bf16, float>(a, pl, bwd, s);
}

}  // namespace
}  // namespace mdmm

using namespace mdmm;

extern "C" int64_t mdmm_gated_scan_states(const mdmm_gated_scan_t* a) {
  if (check(a)) return -1;
  const int64_t tiles = ((int64_t)a->T + TILE - 1) / TILE;
  return tiles > 1 ? tiles * a->B * a->H : 0;         // (a single tile starts at h0)
}

extern "C" int64_t mdmm_gated_scan_ws(const mdmm_gated_scan_t* a, int bwd) {
  if (check(a)) return -1;
  if (none(a)) return 0;
  const Plan pl = plan(a, bwd);
  return pl.splits > 1 ? 2 * (int64_t)pl.splits * a->B * a->H : 0;
}

extern "C" int mdmm_gated_scan_fwd(const mdmm_gated_scan_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (none(a)) return 0;
  if (!a->h) return MDMM_E_ARG;
  return run(a, false, (hipStream_t)stream);
}

extern "C" int mdmm_gated_scan_bwd(const mdmm_gated_scan_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (none(a)) return 0;
  if (!a->g_gates || (a->T > TILE && !a->states)) return MDMM_E_ARG;
  return run(a, true, (hipStream_t)stream);
}
