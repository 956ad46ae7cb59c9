// Gated linear recurrence over time: h_t = a_t h_{t-1} + k_t c_t with a_t = sigmoid(f_t), k_t = 1 - a_t, per channel; a step
// whose mask byte is 0 leaves h as it is (a = 1, k = 0).  Backward: G_t = g_t + a_{t+1} G_{t+1} (g = the gradient of h_t),
// dc = G k, df = G (h_{t-1} - c) a k, dh0 = a_0 G_0.
//
// Bound by HBM: forward reads f, c and writes h, backward reads f, c, g and writes df, dc; neither keeps h (the backward
// pass forms it again from one state per tile of time).  A step h -> a h + b composes, (a2, b2)(a1, b1) = (a2 a1, a2 b1 + b2), so time is
// taken in tiles: a workgroup of up to 8 waves holds 64 VEC channels and a tile of 8 steps a wave in registers, each wave
// composes its 8 steps, the pieces meet in LDS, and every wave then runs its steps from the state in front of them.  Every
// load of a tile is in flight at once, each tensor passes once, and the next tile's loads are issued before the present
// tile's are used up.  Where the channels alone do not fill the chip, time is also split over workgroups: a first launch
// composes each split (reading f, c once more; backward f, g), the second starts each split from the splits in front of it.
// Nothing waits for another workgroup, and no sum is formed by atomics: results do not depend on the schedule.
// 512 x 256 x 512 in bf16: forward 97 us (403 MB, 4.2 TB/s), backward 155 (672 MB, 4.3 TB/s).  20011 x 3 x 200 in fp32, split:
// 22 + 32 forward, 22 + 51 backward.  One step of 16 x 256: 4.7 us in fp32, 5.0 in bf16.
#include "gated.h"

namespace mdmm {
namespace {

// steps of a wave; most waves; up to ONE steps are one tile; beyond, steps of a tile, whose first state is kept for the
// backward pass
constexpr int S = 8, WMAX = 8, ONE = S * WMAX, KEEP = 32;

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

template <typename T, int VEC> struct Raw;           // VEC elements as loaded
template <> struct Raw<float, 1> { unsigned x; };
template <> struct Raw<float, 2> { u32x2 x; };
template <> struct Raw<__bf16, 1> { unsigned short x; };
template <> struct Raw<__bf16, 2> { unsigned x; };

template <int VEC> __device__ __forceinline__ void widen(const Raw<float, VEC>& r, float* v) { __builtin_memcpy(v, &r, sizeof r); }
__device__ __forceinline__ void widen(const Raw<__bf16, 1>& r, float* v) { v[0] = __uint_as_float((unsigned)r.x << 16); }
__device__ __forceinline__ void widen(const Raw<__bf16, 2>& r, float* v) {
  v[0] = __uint_as_float(r.x << 16);
  v[1] = __uint_as_float(r.x & 0xffff0000u);
}

template <typename T, int VEC> __device__ __forceinline__ Raw<T, VEC> narrow(const float* v) {
  T t[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) t[e] = (T)v[e];      // (bf16: to nearest, ties to even)
  Raw<T, VEC> r;
  __builtin_memcpy(&r, t, sizeof r);
  return r;
}

// One time step of a tensor.  BUF: a buffer from its first element on, addressed by 32-bit byte offsets; `live` false makes
// it empty, an empty step's reads give 0 and its writes are dropped, as are those of a thread without channels (its offset is
// past every end), so no access needs a branch and the compiler can count what is in flight.  Else (a step's elements 2 GiB
// apart, as in a long batch-first tensor): pointers, 64-bit offsets, branches.
template <typename T, int VEC, bool BUF> struct Step;
template <typename T, int VEC> struct Step<T, VEC, true> {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Step(const void* base, int64_t at, bool live)
      : r(__builtin_amdgcn_make_buffer_rsrc((void*)((T*)base + at), 0, live && base ? 0x7fffffff : 0, 0x00020000)) {}
  __device__ __forceinline__ Raw<T, VEC> get(unsigned o) const {
    Raw<T, VEC> v;
    if constexpr (sizeof(v) == 8) v.x = __builtin_amdgcn_raw_buffer_load_b64(r, o, 0, 0);
    else if constexpr (sizeof(v) == 4) v.x = __builtin_amdgcn_raw_buffer_load_b32(r, o, 0, 0);
    else v.x = __builtin_amdgcn_raw_buffer_load_b16(r, o, 0, 0);
    return v;
  }
  __device__ __forceinline__ void put(unsigned o, const float* f) const {
    const Raw<T, VEC> v = narrow<T, VEC>(f);
    if constexpr (sizeof(v) == 8) __builtin_amdgcn_raw_buffer_store_b64(v.x, r, o, 0, 0);
    else if constexpr (sizeof(v) == 4) __builtin_amdgcn_raw_buffer_store_b32(v.x, r, o, 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(v.x, r, o, 0, 0);
  }
};
template <typename T, int VEC> struct Step<T, VEC, false> {
  char* p;
  __device__ __forceinline__ Step(const void* base, int64_t at, bool live) : p(live && base ? (char*)((T*)base + at) : nullptr) {}
  __device__ __forceinline__ Raw<T, VEC> get(int64_t o) const { return p && o >= 0 ? *(const Raw<T, VEC>*)(p + o) : Raw<T, VEC>{}; }
  __device__ __forceinline__ void put(int64_t o, const float* f) const {
    if (p && o >= 0) *(Raw<T, VEC>*)(p + o) = narrow<T, VEC>(f);
  }
};
template <bool BUF> struct Off { typedef unsigned type; };
template <> struct Off<false> { typedef int64_t type; };

struct Plan {
  int vec, waves, splits;
  bool buf;                    // a time step of every tensor within 2 GiB
  int64_t chunks;              // VEC-wide pieces of a row of H channels
  int64_t wgs;                 // workgroups over the channels
  int64_t tile, tiles, per;    // steps of a tile, tiles of time, tiles of a split
};

// A thread's channels: VEC neighbours of one sequence, as byte offsets into a time step of each tensor (-1, which as an
// unsigned one is past every buffer's end: no channels)
template <typename IO, typename HO, bool BUF> struct Lane {
  typedef typename Off<BUF>::type off;
  int64_t b, j, q;             // sequence, first channel, flat index b H + j (0 for a thread without channels)
  off gates, h, f32, g_gates, mask;
  bool live;
  __device__ __forceinline__ Lane(const mdmm_gated_scan_t& p, int64_t chunks, int vec) {
    int64_t i = (int64_t)blockIdx.x * 64 + (threadIdx.x & 63);
    live = i < chunks * p.B;
    if (!live) i = 0;
    b = i / chunks;
    j = (i - b * chunks) * vec;
    q = b * p.H + j;
    gates = live ? (off)((b * p.gates_sb + j) * (int64_t)sizeof(IO)) : (off)-1;
    g_gates = live ? (off)((b * p.g_gates_sb + j) * (int64_t)sizeof(IO)) : (off)-1;
    h = live ? (off)(q * (int64_t)sizeof(HO)) : (off)-1;
    f32 = live ? (off)(q * 4) : (off)-1;
    mask = live ? (off)(b * p.mask_sb) : (off)-1;
  }
};

__device__ __forceinline__ int64_t time_of(const mdmm_gated_scan_t& p, int64_t i) { return p.reverse ? p.T - 1 - i : i; }
__device__ __forceinline__ int64_t onward(const mdmm_gated_scan_t& p) { return p.reverse ? -1 : 1; }

// f, c and the mask of a wave's S steps from step i0 on as loaded (a step past the end: zeros)
template <typename IO, typename HO, int VEC, bool BUF> struct Steps {
  Raw<IO, VEC> f[S], c[S];
  unsigned char m[S];
  template <bool C> __device__ __forceinline__ void fetch(const mdmm_gated_scan_t& p, const Lane<IO, HO, BUF>& l, int64_t i0, bool any) {
    const int64_t step = onward(p) * p.gates_st, mstep = onward(p) * p.mask_st;
    int64_t at = time_of(p, i0) * p.gates_st, mat = time_of(p, i0) * p.mask_st;
#pragma unroll
    for (int s = 0; s < S; ++s, at += step, mat += mstep) {
      const bool in = any && i0 + s < p.T;
      f[s] = Step<IO, VEC, BUF>(p.gates, at, in).get(l.gates);
      if (C) c[s] = Step<IO, VEC, BUF>(p.gates, at + p.H, in).get(l.gates);
      if constexpr (BUF) {
        __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void*)(p.mask + mat), 0, in && p.mask ? 0x7fffffff : 0, 0x00020000);
        m[s] = __builtin_amdgcn_raw_buffer_load_b8(r, l.mask, 0, 0);
      } else m[s] = in && p.mask && l.live ? p.mask[mat + l.mask] : 0;
    }
  }
  // bit s: step s is there and its mask lets it through
  __device__ __forceinline__ unsigned on(const mdmm_gated_scan_t& p, int64_t i0) const {
    const int64_t left = p.T - i0;
    unsigned all = left >= S ? (1u << S) - 1 : left > 0 ? (1u << left) - 1 : 0, some = 0;
    if (!p.mask) return all;
#pragma unroll
    for (int s = 0; s < S; ++s) some |= m[s] ? 1u << s : 0u;
    return all & some;
  }
};

// h (from_end: the adjoint) of the start taken through the splits in front of split z: every wave composes its share of
// them, the shares meet in LDS
template <int VEC>
__device__ __forceinline__ void lead_in(const float* ws, int64_t stride, int z, bool from_end, const Plan& pl, int64_t q, float* h,
                                        float (*sa)[64 * VEC], float (*sb)[64 * VEC]) {
  if (pl.splits == 1) return;
  const int n = from_end ? pl.splits - 1 - z : z, W = pl.waves;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  float A[VEC], B[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; }
#pragma unroll 8
  for (int i = n * wave / W; i < n * (wave + 1) / W; ++i) {
    const float* a = ws + 2 * stride * (from_end ? pl.splits - 1 - i : i) + q;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      B[e] = fmaf(a[e], B[e], a[stride + e]);
      A[e] *= a[e];
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) { sa[wave][e * 64 + lane] = A[e]; sb[wave][e * 64 + lane] = B[e]; }
  __syncthreads();
  for (int w = 0; w < W; ++w)
#pragma unroll
    for (int e = 0; e < VEC; ++e) h[e] = fmaf(sa[w][e * 64 + lane], h[e], sb[w][e * 64 + lane]);
  __syncthreads();
}

// Composition of each split: BWD of D -> a (g + D) from its last step to its first, else of h -> a h + k c.  Each wave takes
// one run of the split's tiles, the runs are joined in LDS
template <typename IO, typename HO, int VEC, bool BUF, bool BWD>
__global__ __launch_bounds__(64 * WMAX) void scan_split_kernel(mdmm_gated_scan_t p, Plan pl) {
  __shared__ float sa[WMAX][64 * VEC], sb[WMAX][64 * VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = pl.waves;
  const Lane<IO, HO, BUF> l(p, pl.chunks, VEC);
  const int64_t stride = (int64_t)p.B * p.H;
  const int64_t t0 = blockIdx.y * pl.per, t1 = t0 + pl.per < pl.tiles ? t0 + pl.per : pl.tiles;
  const int64_t first_all = t0 * pl.tile, last_all = t1 * pl.tile < p.T ? t1 * pl.tile : p.T;
  const int64_t run = ((last_all - first_all + W - 1) / W + S - 1) / S * S;
  const int64_t first = first_all + wave * run < last_all ? first_all + wave * run : last_all;
  const int64_t last = first + run < last_all ? first + run : last_all;
  float A[VEC], B[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; }
  Steps<IO, HO, VEC, BUF> x;
  Raw<HO, VEC> g[S];
  const int64_t n = (last - first + S - 1) / S;
  auto fetch = [&](int64_t i) {
    const int64_t i0 = first + (BWD ? n - 1 - i : i) * S;
    x.template fetch<!BWD>(p, l, i0, i < n);
    if (BWD) {
      int64_t at = time_of(p, i0) * stride;
#pragma unroll
      for (int s = 0; s < S; ++s, at += onward(p) * stride)
        g[s] = Step<HO, VEC, BUF>(p.g_h, at, i < n && i0 + s < p.T).get(l.h);
    }
  };
  fetch(0);
  for (int64_t i = 0; i < n; ++i) {
    const unsigned on = x.on(p, first + (BWD ? n - 1 - i : i) * S);
    float fv[S][VEC], cv[S][VEC];
#pragma unroll
    for (int s = 0; s < S; ++s) {
      widen(x.f[s], fv[s]);
      if (BWD) widen(g[s], cv[s]); else widen(x.c[s], cv[s]);
    }
    fetch(i + 1);
#pragma unroll
    for (int s_ = 0; s_ < S; ++s_) {
      const int s = BWD ? S - 1 - s_ : s_;
      const bool in = on >> s & 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Gate y(fv[s][e]);
        const float a = in ? y.a : 1.0f;
        if (BWD) B[e] = a * (cv[s][e] + B[e]);            // (a step past the end: its g is 0)
        else B[e] = in ? fmaf(y.a, B[e], y.k * cv[s][e]) : B[e];
        A[e] *= a;
      }
    }
  }
#pragma unroll
  for (int e = 0; e < VEC; ++e) { sa[wave][e * 64 + lane] = A[e]; sb[wave][e * 64 + lane] = B[e]; }
  __syncthreads();
  if (wave == 0 && l.live) {
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

template <typename IO, typename HO, int VEC, bool BUF>
__global__ __launch_bounds__(64 * WMAX, 4) void scan_fwd_kernel(mdmm_gated_scan_t p, Plan pl) {
  __shared__ float sa[2][WMAX][64 * VEC], sb[2][WMAX][64 * VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = pl.waves;
  const Lane<IO, HO, BUF> l(p, pl.chunks, VEC);
  const int64_t stride = (int64_t)p.B * p.H;
  const int64_t t0 = blockIdx.y * pl.per, t1 = t0 + pl.per < pl.tiles ? t0 + pl.per : pl.tiles;
  Steps<IO, HO, VEC, BUF> x;
  x.template fetch<true>(p, l, t0 * pl.tile + wave * S, true);
  float h0[VEC];
#pragma unroll
  for (int e = 0; e < VEC; ++e) h0[e] = p.h0 ? p.h0[l.b * p.h0_sb + l.j + e] : 0.0f;
  lead_in<VEC>(p.ws, stride, blockIdx.y, false, pl, l.q, h0, sa[0], sb[0]);
  for (int64_t tile = t0; tile < t1; ++tile) {
    const int64_t i0 = tile * pl.tile + wave * S;
    const unsigned on = x.on(p, i0);
    float a[S][VEC], b[S][VEC], A[VEC], B[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float fv[VEC], cv[VEC];
      widen(x.f[s], fv);
      widen(x.c[s], cv);
      const bool in = on >> s & 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Gate y(fv[e]);
        a[s][e] = in ? y.a : 1.0f;
        b[s][e] = in ? y.k * cv[e] : 0.0f;
        B[e] = fmaf(a[s][e], B[e], b[s][e]);
        A[e] *= a[s][e];
      }
    }
    x.template fetch<true>(p, l, i0 + pl.tile, tile + 1 < t1);      // in flight behind the rest of this tile
    const int z = tile & 1;
    if (W > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) { sa[z][wave][e * 64 + lane] = A[e]; sb[z][wave][e * 64 + lane] = B[e]; }
      __syncthreads();         // (two sets of pieces: a wave a tile ahead writes the other one)
    }
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
    if (wave == 0) Step<float, VEC, BUF>(p.states, tile * stride, true).put(l.f32, h);
    int64_t at = time_of(p, i0) * stride;
#pragma unroll
    for (int s = 0; s < S; ++s, at += onward(p) * stride) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) h[e] = fmaf(a[s][e], h[e], b[s][e]);
      Step<HO, VEC, BUF>(p.h, at, i0 + s < p.T).put(l.h, h);
    }
    if (W == 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) h0[e] = h[e];
    }
  }
  if (t1 == pl.tiles && wave == 0) Step<float, VEC, BUF>(p.h_last, 0, true).put(l.f32, h0);
}

template <typename IO, typename HO, int VEC, bool BUF>
__global__ __launch_bounds__(64 * WMAX) void scan_bwd_kernel(mdmm_gated_scan_t p, Plan pl) {
  __shared__ float sa[2][WMAX][64 * VEC], sb[2][WMAX][64 * VEC], sg[2][WMAX][64 * VEC];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), W = pl.waves;
  const Lane<IO, HO, BUF> l(p, pl.chunks, VEC);
  const int64_t stride = (int64_t)p.B * p.H;
  const int64_t t0 = blockIdx.y * pl.per, t1 = t0 + pl.per < pl.tiles ? t0 + pl.per : pl.tiles;
  Steps<IO, HO, VEC, BUF> x;
  Raw<HO, VEC> g[S];
  Raw<float, VEC> start;       // the state in front of the tile
  auto fetch = [&](int64_t tile) {
    const bool any = tile >= t0;
    const int64_t i0 = tile * pl.tile + wave * S;
    x.template fetch<true>(p, l, i0, any);
    int64_t at = time_of(p, i0) * stride;
#pragma unroll
    for (int s = 0; s < S; ++s, at += onward(p) * stride) g[s] = Step<HO, VEC, BUF>(p.g_h, at, any && i0 + s < p.T).get(l.h);
    start = Step<float, VEC, BUF>(p.states, tile * stride, any).get(l.f32);
  };
  fetch(t1 - 1);
  float d0[VEC], h00[VEC];     // a G of the step behind the present tile; the state in front of a single tile
#pragma unroll
  for (int e = 0; e < VEC; ++e) {
    d0[e] = p.g_last ? p.g_last[l.q + e] : 0.0f;
    h00[e] = !p.states && p.h0 ? p.h0[l.b * p.h0_sb + l.j + e] : 0.0f;
  }
  lead_in<VEC>(p.ws, stride, blockIdx.y, true, pl, l.q, d0, sa[0], sb[0]);
  for (int64_t tile = t1 - 1; tile >= t0; --tile) {
    const int64_t i0 = tile * pl.tile + wave * S;
    const unsigned on = x.on(p, i0);
    float a[S][VEC], k[S][VEC], cv[S][VEC], gv[S][VEC], A[VEC], B[VEC], D[VEC], h[VEC], d[VEC];
    widen(start, h);
#pragma unroll
    for (int e = 0; e < VEC; ++e) { A[e] = 1.0f; B[e] = 0.0f; D[e] = 0.0f; if (!p.states) h[e] = h00[e]; }
#pragma unroll
    for (int s = 0; s < S; ++s) {
      float fv[VEC];
      widen(x.f[s], fv);
      widen(x.c[s], cv[s]);
      widen(g[s], gv[s]);
      const bool in = on >> s & 1;
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const Gate y(fv[e]);
        a[s][e] = in ? y.a : 1.0f;
        k[s][e] = in ? y.k : 0.0f;
        cv[s][e] = in ? cv[s][e] : 0.0f;
        B[e] = fmaf(a[s][e], B[e], k[s][e] * cv[s][e]);
        A[e] *= a[s][e];
      }
    }
    fetch(tile - 1);           // in flight behind the rest of this tile
#pragma unroll
    for (int s = S - 1; s >= 0; --s)
#pragma unroll
      for (int e = 0; e < VEC; ++e) D[e] = a[s][e] * (gv[s][e] + D[e]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) d[e] = d0[e];
    const int z = tile & 1;
    if (W > 1) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        sa[z][wave][e * 64 + lane] = A[e];
        sb[z][wave][e * 64 + lane] = B[e];
        sg[z][wave][e * 64 + lane] = D[e];
      }
      __syncthreads();
      for (int w = 0; w < wave; ++w)
#pragma unroll
        for (int e = 0; e < VEC; ++e) h[e] = fmaf(sa[z][w][e * 64 + lane], h[e], sb[z][w][e * 64 + lane]);
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
#pragma unroll
    for (int s = 0; s < S; ++s)          // cv becomes h_{t-1} - c_t (0 where the mask is: k is 0 there too)
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float before = h[e];
        h[e] = fmaf(a[s][e], h[e], k[s][e] * cv[s][e]);
        cv[s][e] = (on >> s & 1) ? before - cv[s][e] : 0.0f;
      }
    int64_t at = time_of(p, i0 + S - 1) * p.g_gates_st;
#pragma unroll
    for (int s = S - 1; s >= 0; --s, at -= onward(p) * p.g_gates_st) {
      float df[VEC], dc[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const float G = gv[s][e] + d[e];
        dc[e] = on >> s & 1 ? G * k[s][e] : 0.0f;          // (whatever G is)
        df[e] = dc[e] * a[s][e] * cv[s][e];
        d[e] = a[s][e] * G;
      }
      Step<IO, VEC, BUF>(p.g_gates, at, i0 + s < p.T).put(l.g_gates, df);
      Step<IO, VEC, BUF>(p.g_gates, at + p.H, i0 + s < p.T).put(l.g_gates, dc);
    }
  }
  if (t0 == 0 && wave == 0) Step<float, VEC, BUF>(p.g_h0, 0, true).put(l.f32, d0);
}

// sum over the sequences of g_h0: 16 columns and 64 threads down each a workgroup, joined in a fixed order
__global__ __launch_bounds__(1024) void scan_rows_kernel(const float* __restrict__ g, int64_t rows, int H, float* out) {
  __shared__ float part[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
  float s = 0.0f;
  if (c < H) {
#pragma unroll 8
    for (int64_t i = r; i < rows; i += 64) s += g[i * H + c];
  }
  part[r][threadIdx.x & 15] = s;
  __syncthreads();
  if (r == 0 && c < H) {
    s = 0.0f;
#pragma unroll 16
    for (int i = 0; i < 64; ++i) s += part[i][threadIdx.x & 15];
    out[c] = s;
  }
}

int check(const mdmm_gated_scan_t* a) {
  if (!a || a->T < 0 || a->B < 0 || a->H < 0) return MDMM_E_ARG;
  if (!a->gates_bf16 && a->h_bf16) return MDMM_E_ARG;
  if (a->gates_sb < 0 || a->g_gates_sb < 0 || a->mask_sb < 0) return MDMM_E_ARG;         // (a negative offset: no channels)
  if (a->T > 0 && a->B > 0 && a->H > 0 && !a->gates) return MDMM_E_ARG;
  return 0;
}

bool none(const mdmm_gated_scan_t* a) { return a->T == 0 || a->B == 0 || a->H == 0; }

Plan plan(const mdmm_gated_scan_t* a) {
  Plan p;
  const uintptr_t es = a->gates_bf16 ? 2 : 4, hs = a->h_bf16 ? 2 : 4;
  auto fits = [&](int v) {
    const uintptr_t m = (uintptr_t)v * es - 1, mh = (uintptr_t)v * hs - 1, m4 = (uintptr_t)v * 4 - 1;
    return a->H % v == 0 && ((uintptr_t)a->gates & m) == 0 && a->gates_st % v == 0 && a->gates_sb % v == 0 &&
           ((uintptr_t)a->h & mh) == 0 && ((uintptr_t)a->g_h & mh) == 0 && ((uintptr_t)a->g_gates & m) == 0 &&
           a->g_gates_st % v == 0 && a->g_gates_sb % v == 0 && ((uintptr_t)a->states & m4) == 0 &&
           ((uintptr_t)a->h_last & m4) == 0 && ((uintptr_t)a->g_h0 & m4) == 0;
  };
  // (four channels a thread spill in the forward pass: 123 us at 512 x 256 x 512 in bf16, with two 97)
  p.vec = fits(2) ? 2 : 1;
  auto reach = [&](int64_t sb) { return (sb < 0 ? 0x80000000ll : (a->B - 1) * sb + 2 * (int64_t)a->H) * 4 < 0x7fffffffll; };
  p.buf = reach(a->gates_sb) && reach(a->g_gates_sb) && reach(a->H) && reach(a->mask_sb);
  p.chunks = a->H / p.vec;
  p.wgs = (p.chunks * a->B + 63) / 64;
  // up to ONE steps one tile; beyond, tiles of 4 waves (at 512 x 256 x 512 in bf16 94 us forward and 155 backward, of 8
  // waves 98 and 179, before the masked steps' zeros cost the backward pass 2: three workgroups of 4 waves fit a CU's registers
  // there, but one of 8)
  const int64_t waves = (a->T + S - 1) / S;
  p.waves = (int)(a->T <= ONE ? waves : KEEP / S);
  p.tile = p.waves * S;
  p.tiles = (a->T + p.tile - 1) / p.tile;
  // Few workgroups over a long time: time over workgroups too, two a CU (20011 x 3 x 200 in fp32: 130 us for the four launches
  // of a training pass, with four a CU 140 -- every split reads through all those before it).  The launch that composes the
  // splits costs 4 to 5 us and reads two of the tensors again, so it pays where a split leaves out most of the tiles and the
  // workgroups are far from filling the chip.  Training passes in us, one workgroup over all of time and split:
  //   up to 64 workgroups from 4 tiles on   (1 x 4: 3 tiles 20 and 21, 4 tiles 25 and 22; 64 workgroups, 4 tiles 27 and 24)
  //   up to 128 from 8 tiles on             (80 workgroups, 4 tiles 28 and 29; 128: 6 tiles 39 and 43, 8 tiles 50 and 48)
  //   beyond, from 12 on and with narrow types, up to 170 workgroups (bf16, fp32 states) or 192 (bf16): 160 workgroups, 32 tiles
  //   163 and 122 in bf16, 265 and 262 with its norm in fp32, 187 and 197 all in fp32; 192, 63 tiles 311 and 289, 585 and 642,
  //   374 and 550; 256 workgroups, 63 tiles 313 and 347 in bf16
  int64_t splits = 1;
  const int64_t from = p.wgs <= 64 ? 4 : p.wgs <= 128 ? 8 : 12, most = a->h_bf16 ? 192 : a->gates_bf16 ? 170 : 128;
  if (p.wgs <= most && p.tiles >= from) {
    splits = (512 + p.wgs - 1) / p.wgs;
    if (splits > p.tiles) splits = p.tiles;
    if (splits > 512) splits = 512;
  }
  p.per = (p.tiles + splits - 1) / splits;
  p.splits = (int)((p.tiles + p.per - 1) / p.per);
  return p;
}

template <typename IO, typename HO, int VEC, bool BUF>
int launch(const mdmm_gated_scan_t* a, const Plan& pl, bool bwd, hipStream_t s) {
  const dim3 grid((unsigned)pl.wgs, (unsigned)pl.splits), block(64 * pl.waves);
#define RUN(K) hipLaunchKernelGGL(K, grid, block, 0, s, *a, pl)
  if (pl.splits > 1) {
    if (bwd) RUN((scan_split_kernel<IO, HO, VEC, BUF, true>));
    else RUN((scan_split_kernel<IO, HO, VEC, BUF, false>));
  }
  if (bwd) RUN((scan_bwd_kernel<IO, HO, VEC, BUF>));
  else RUN((scan_fwd_kernel<IO, HO, VEC, BUF>));
#undef RUN
  return (int)hipGetLastError();
}

template <typename IO, typename HO>
int launch(const mdmm_gated_scan_t* a, const Plan& pl, bool bwd, hipStream_t s) {
  if (!pl.buf) return pl.vec == 1 ? launch<IO, HO, 1, false>(a, pl, bwd, s) : launch<IO, HO, 2, false>(a, pl, bwd, s);
  return pl.vec == 1 ? launch<IO, HO, 1, true>(a, pl, bwd, s) : launch<IO, HO, 2, true>(a, pl, bwd, s);
}

int run(const mdmm_gated_scan_t* args, bool bwd, hipStream_t s) {
  mdmm_gated_scan_t keep = *args, *a = &keep;
  if (a->T <= ONE) a->states = nullptr;                // (room for none of them: mdmm_gated_scan_states)
  const Plan pl = plan(a);
  if (pl.wgs > (1 << 22)) return MDMM_E_LIMIT;         // (a grid's threads fit 32 bits)
  if (pl.splits > 1 && !a->ws) return MDMM_E_ARG;
  if (!a->gates_bf16) return launch<float, float>(a, pl, bwd, s);
  return a->h_bf16 ? launch<__bf16, __bf16>(a, pl, bwd, s) : launch<__bf16, float>(a, pl, bwd, s);
}

}  // namespace
}  // namespace mdmm

using namespace mdmm;

extern "C" int64_t mdmm_gated_scan_states(const mdmm_gated_scan_t* a) {
  if (check(a)) return -1;
  return a->T > ONE ? ((int64_t)a->T + KEEP - 1) / KEEP * a->B * a->H : 0;         // (a single tile starts at h0)
}

extern "C" int64_t mdmm_gated_scan_ws(const mdmm_gated_scan_t* a, int) {
  if (check(a)) return -1;
  if (none(a)) return 0;
  const Plan pl = plan(a);
  return pl.splits > 1 ? 2 * (int64_t)pl.splits * a->B * a->H : 0;
}

extern "C" int mdmm_gated_scan_fwd(const mdmm_gated_scan_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (none(a)) return 0;
  if (!a->h) return MDMM_E_ARG;
  if (last_state_on_input(a)) return MDMM_E_ALIAS;
  return run(a, false, (hipStream_t)stream);
}

extern "C" int mdmm_gated_scan_bwd(const mdmm_gated_scan_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (none(a)) return 0;
  if (!a->g_gates || (a->T > ONE && !a->states)) return MDMM_E_ARG;
  if (a->g_h0_sum && !a->g_h0) return MDMM_E_ARG;
  const int e = run(a, true, (hipStream_t)stream);
  if (e || !a->g_h0_sum) return e;
  hipLaunchKernelGGL(scan_rows_kernel, dim3((a->H + 15) / 16), dim3(1024), 0, (hipStream_t)stream, a->g_h0, (int64_t)a->B, a->H,
                     a->g_h0_sum);
  return (int)hipGetLastError();
}
