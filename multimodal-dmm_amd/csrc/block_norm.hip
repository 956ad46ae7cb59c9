// Norms before and after a residual block fused with the block's gate and residual scale (mdmm_block_norm_t):
//   u = y r w, r = rsqrt(mean(y^2) + eps);  out = res + s silu(g) u;  n = out r' w'
// Backward, with d = g_out + r' (q - out r'^2 mean(q out)), q = g_n w' :  d_res = d, d_s = sum d silu(g) u,
// d_g = d s u silu'(g), p = d s silu(g):  d_w = sum p y r,  d_y = r (p w - y r mean(p w y r)),  d_w' = sum g_n out r'.
// Bound by HBM: a row is held in registers from its loads to its stores, so every tensor passes once, and the next row's
// loads are in flight behind the present row's sums.  Up to 256 columns a row is one wave's (4 a workgroup, no barrier in a
// sum); a longer one a workgroup's, 4 columns a thread (8 from 2049 on), whose waves meet in LDS once a sum.  Rows that are
// not aligned to 4 elements take columns one by one.  The three column sums of the backward pass stay in a thread over all
// of its rows and leave as one slab a workgroup; norm_fold_kernel adds the slabs up in a fixed order, without atomics.
// 65536 x 1280 in bf16: forward 167 us (840 MB, 5.0 TB/s; a copy's 5.35 but for the gate's exponential), backward 300 (1.34 GB,
// 4.5 TB/s: three sums a row between its loads and its last store), fold 8; in fp32 forward 331, both 877.  Eight rows: 2.6 us,
// a launch (1.8 for one that fills a word).
#include <type_traits>
#include "gated.h"

namespace mdmm {
namespace {

typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// VEC columns as loaded
template <typename T, int VEC> struct Raw;
template <> struct Raw<float, 4> { u32x4 x; };
template <> struct Raw<float, 1> { unsigned x; };
template <> struct Raw<__bf16, 4> { u32x2 x; };
template <> struct Raw<__bf16, 1> { unsigned short x; };

template <int VEC> __device__ __forceinline__ void widen(const Raw<float, VEC>& r, float* v) { __builtin_memcpy(v, &r, sizeof r); }
__device__ __forceinline__ void widen(const Raw<__bf16, 4>& r, float* v) {
  v[0] = __uint_as_float(r.x[0] << 16); v[1] = __uint_as_float(r.x[0] & 0xffff0000u);
  v[2] = __uint_as_float(r.x[1] << 16); v[3] = __uint_as_float(r.x[1] & 0xffff0000u);
}
__device__ __forceinline__ void widen(const Raw<__bf16, 1>& r, float* v) { v[0] = __uint_as_float((unsigned)r.x << 16); }

// One row of a tensor as a buffer of its H columns (none: H = 0): a read past the end gives 0 and a write there is dropped by
// the address check, so no piece needs a branch -- with branches around the stores the compiler waits for ALL memory
// operations before it uses the row fetched ahead, the present row's stores among them
template <typename T, int VEC> struct Row {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ Row(const void* base, int64_t at, int H)
      : r(__builtin_amdgcn_make_buffer_rsrc((void*)((T*)base + at), 0, base ? H * (int)sizeof(T) : 0, 0x00020000)) {}
  __device__ __forceinline__ void get(Raw<T, VEC>& v, int c) const {
    if constexpr (sizeof(v) == 16) v.x = __builtin_amdgcn_raw_buffer_load_b128(r, c * (int)sizeof(T), 0, 0);
    else if constexpr (sizeof(v) == 8) v.x = __builtin_amdgcn_raw_buffer_load_b64(r, c * (int)sizeof(T), 0, 0);
    else if constexpr (sizeof(v) == 4) v.x = __builtin_amdgcn_raw_buffer_load_b32(r, c * (int)sizeof(T), 0, 0);
    else v.x = __builtin_amdgcn_raw_buffer_load_b16(r, c * (int)sizeof(T), 0, 0);
  }
  template <typename F> __device__ __forceinline__ void put(const F* f, int c) const {
    Raw<T, VEC> v;
    T t[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) t[e] = (T)(float)f[e];          // (bf16: to nearest, ties to even)
    __builtin_memcpy(&v, t, sizeof v);
    if constexpr (sizeof(v) == 16) __builtin_amdgcn_raw_buffer_store_b128(v.x, r, c * (int)sizeof(T), 0, 0);
    else if constexpr (sizeof(v) == 8) __builtin_amdgcn_raw_buffer_store_b64(v.x, r, c * (int)sizeof(T), 0, 0);
    else if constexpr (sizeof(v) == 4) __builtin_amdgcn_raw_buffer_store_b32(v.x, r, c * (int)sizeof(T), 0, 0);
    else __builtin_amdgcn_raw_buffer_store_b16(v.x, r, c * (int)sizeof(T), 0, 0);
  }
};

// A thread's pieces of a vector over the columns, kept in registers over all rows (read again for each row, the three vectors
// in fp32 are more bytes than a bf16 row); `none` where it is not there
template <int VEC, int NV>
__device__ __forceinline__ void keep(float (&v)[NV][VEC], const float* base, float none, const int (&c)[NV], int H) {
  const Row<float, VEC> row(base, 0, H);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    Raw<float, VEC> x;
    row.get(x, c[k]);
    widen(x, v[k]);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[k][e] = base ? v[k][e] : none;
  }
}

template <typename T, int VEC, int NV>
__device__ __forceinline__ void fetch(Raw<T, VEC> (&r)[NV], const void* base, int64_t at, const int (&c)[NV], int H) {
  const Row<T, VEC> row(base, at, H);
#pragma unroll
  for (int k = 0; k < NV; ++k) row.get(r[k], c[k]);
}

// sum over rows of 16 lanes by DPP moves (no LDS round trip), in each of them
template <int CTRL, int ROWS> __device__ __forceinline__ float dpp_add(float v) {
  return v + __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, ROWS, 0xf, false));
}
__device__ __forceinline__ float row16_total(float v) {
  v = dpp_add<0xb1, 0xf>(v);        // neighbours
  v = dpp_add<0x4e, 0xf>(v);        // pairs
  v = dpp_add<0x141, 0xf>(v);       // half rows mirrored
  return dpp_add<0x140, 0xf>(v);    // rows mirrored
}
__device__ __forceinline__ float wave_total(float v) {
  v = row16_total(v);
  v = dpp_add<0x142, 0xa>(v);       // row 0 into row 1, row 2 into row 3
  v = dpp_add<0x143, 0xc>(v);       // rows 0 and 1 into rows 2 and 3: lane 63 holds the sum
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}

__device__ __forceinline__ double wave_total(double v) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  return v;
}
__device__ __forceinline__ float rsqrt_(float v) { return rsqrtf(v); }
__device__ __forceinline__ double rsqrt_(double v) { return 1.0 / sqrt(v); }
// act = silu(g) = g a and slope = silu'(g) = a (1 + g k), a = sigmoid(g), k = 1 - a formed apart: as a difference from 1 it
// would leave the slope of large gates, which is 1, off by 6e-8 |g|
__device__ __forceinline__ void gate_(float g, float& act, float& slope) {
  const float e = exp_neg(g), a = __builtin_amdgcn_rcpf(1.0f + e);
  act = g * a;
  slope = fmaf(act, fminf(e * a, 1.0f), a);            // (e infinite, a 0: k is 1)
}
__device__ __forceinline__ void gate_(double g, double& act, double& slope) {
  const double a = 1.0 / (1.0 + exp(-g));
  act = g * a;
  slope = fma(act, 1.0 / (1.0 + exp(g)), a);
}
__device__ __forceinline__ float fma_(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fma_(double a, double b, double c) { return fma(a, b, c); }

// N sums over a row's threads (a wave, or WIDE the workgroup of up to 16 waves), in every one of them.  lds: 2 sets of
// 2 x 16 words, the words past the last wave zero (a wave that runs ahead writes the other set)
template <bool WIDE, int N, typename A> __device__ __forceinline__ void row_sums(A (&v)[N], float* lds, int& slot) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = wave_total(v[i]);
  if constexpr (WIDE) {
    float* s = lds + (slot ^= 1) * 32;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) s[i * 16 + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = row16_total(s[i * 16 + (threadIdx.x & 15)]);
  }
}
template <bool WIDE, typename A> __device__ __forceinline__ A row_sum(A v, float* lds, int& slot) {
  A a[1] = {v};
  row_sums<WIDE, 1>(a, lds, slot);
  return a[0];
}
template <bool WIDE> __device__ __forceinline__ void clear_sums(float* lds) {
  if constexpr (WIDE) {
    if (threadIdx.x < 64) lds[threadIdx.x] = 0.0f;
    __syncthreads();
  }
}

template <typename Y, typename Br, typename R, int VEC, int NV, int MAXT, bool ALL>
__global__ __launch_bounds__(MAXT) void norm_fwd_kernel(mdmm_block_norm_t p) {
  constexpr bool WIDE = MAXT > 256;
  __shared__ float lds[64];
  clear_sums<WIDE>(lds);
  int slot = 0, c[NV];
  const int lane = WIDE ? (int)threadIdx.x : (int)(threadIdx.x & 63), tpr = WIDE ? (int)blockDim.x : 64;
#pragma unroll
  for (int k = 0; k < NV; ++k) c[k] = (k * tpr + lane) * VEC;
  const float inv = 1.0f / (float)p.H;
  const int wave = WIDE ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t step = (int64_t)gridDim.x * (WIDE ? 1 : 4);
  int64_t row = (int64_t)blockIdx.x * (WIDE ? 1 : 4) + wave;
  float w[NV][VEC], s[NV][VEC], wn[NV][VEC];
  keep<VEC, NV>(w, p.w, 0.0f, c, p.H);
  keep<VEC, NV>(s, p.scale, 1.0f, c, p.H);
  keep<VEC, NV>(wn, p.w_next, 0.0f, c, p.H);
  Raw<R, VEC> res[NV];
  Raw<Y, VEC> ry[NV];
  Raw<Br, VEC> rg[NV];
  auto fetch_row = [&](int64_t at) {         // (past the last row: empty rows)
    const int H = at < p.rows ? p.H : 0;
    if (ALL || p.y) fetch<Y, VEC, NV>(ry, p.y, at * p.y_st, c, H);
    if (ALL || p.gate) fetch<Br, VEC, NV>(rg, p.gate, at * p.gate_st, c, H);
    fetch<R, VEC, NV>(res, p.res, at * p.res_st, c, H);
  };
  fetch_row(row);
  for (; row < p.rows; row += step) {
    float o[NV][VEC], y[NV][VEC], g[NV][VEC];
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      widen(res[k], o[k]);
      if (ALL || p.y) widen(ry[k], y[k]);
      if (ALL || p.gate) widen(rg[k], g[k]);
      if (ALL || p.y)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += y[k][e] * y[k][e];
    }
    fetch_row(row + step);                   // in flight behind this row's arithmetic
    if (ALL || p.y) {
      const float r = rsqrtf(row_sum<WIDE>(ss, lds, slot) * inv + p.eps);
      const Row<R, VEC> out(p.out, row * p.out_st, p.H);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          float u = y[k][e] * r * w[k][e];
          if (ALL || p.gate) u *= g[k][e] * sigmoid_(g[k][e]);
          o[k][e] = fmaf(s[k][e], u, o[k][e]);
        }
        out.put(o[k], c[k]);
      }
    }
    if (ALL || p.w_next) {
      ss = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += o[k][e] * o[k][e];
      const float r = rsqrtf(row_sum<WIDE>(ss, lds, slot) * inv + p.eps);
      const Row<Br, VEC> n(p.n, row * p.n_st, p.H);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) o[k][e] *= r * wn[k][e];
        n.put(o[k], c[k]);
      }
    }
  }
}

template <typename Y, typename Br, typename R, int VEC, int NV, int MAXT, bool ALL>
__global__ __launch_bounds__(MAXT, MAXT == 512 && NV * VEC == 4 ? (sizeof(Y) + sizeof(R) == 4 ? 5 : 4) : 1)
void norm_bwd_kernel(mdmm_block_norm_t p) {
  constexpr bool WIDE = MAXT > 256;
  // Rows of up to four columns in 64 bits: a norm's gradient is what q w' keeps beside the direction of out, eps alone for one
  // column and little for two (300 x 1, the residual's gradient: 3e-8 off, in fp32 7e-6 and by fp32 tensor operations the same)
  typedef typename std::conditional<VEC == 1 && NV == 1, double, float>::type A;
  __shared__ float lds[64];
  __shared__ float fold[WIDE ? 1 : 256 * VEC];
  clear_sums<WIDE>(lds);
  int slot = 0, c[NV];
  const int lane = WIDE ? (int)threadIdx.x : (int)(threadIdx.x & 63), tpr = WIDE ? (int)blockDim.x : 64;
#pragma unroll
  for (int k = 0; k < NV; ++k) c[k] = (k * tpr + lane) * VEC;
  const A inv = (A)1.0 / (A)p.H;
  const int wave = WIDE ? 0 : __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t step = (int64_t)gridDim.x * (WIDE ? 1 : 4);
  int64_t row = (int64_t)blockIdx.x * (WIDE ? 1 : 4) + wave;
  A aw[NV][VEC] = {}, as[NV][VEC] = {}, an[NV][VEC] = {};
  float w[NV][VEC], s[NV][VEC], wn[NV][VEC];
  keep<VEC, NV>(w, p.w, 0.0f, c, p.H);
  keep<VEC, NV>(s, p.scale, 1.0f, c, p.H);
  keep<VEC, NV>(wn, p.w_next, 0.0f, c, p.H);
  Raw<R, VEC> res[NV], rd[NV];
  Raw<Y, VEC> ry[NV];
  Raw<Br, VEC> rg[NV], rq[NV];
  auto fetch_row = [&](int64_t at) {         // (past the last row: empty rows)
    const int H = at < p.rows ? p.H : 0;
    if (ALL || p.y) fetch<Y, VEC, NV>(ry, p.y, at * p.y_st, c, H);
    if (ALL || p.gate) fetch<Br, VEC, NV>(rg, p.gate, at * p.gate_st, c, H);
    if (ALL || p.g_n) fetch<R, VEC, NV>(res, p.res, at * p.res_st, c, H);      // (read for the next norm alone)
    if (ALL || p.g_n) fetch<Br, VEC, NV>(rq, p.g_n, at * p.g_n_st, c, H);
    fetch<R, VEC, NV>(rd, p.g_out, at * p.g_out_st, c, H);
  };
  fetch_row(row);
  for (; row < p.rows; row += step) {
    A x[NV][VEC], g[NV][VEC], slope[NV][VEC], o[NV][VEC], q[NV][VEC], d[NV][VEC];        // (g: silu(gate) once taken)
    A ss = 0.0f;
    auto taken = [](const auto& raw, A* v) {
      float f[VEC];
      widen(raw, f);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[e] = f[e];
    };
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      if (ALL || p.y) taken(ry[k], x[k]);
      if (ALL || p.gate) taken(rg[k], g[k]);
      if (ALL || p.g_n) taken(res[k], o[k]);
      if (ALL || p.g_n) taken(rq[k], q[k]);
      taken(rd[k], d[k]);
      if (ALL || p.y)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += x[k][e] * x[k][e];
    }
    fetch_row(row + step);                   // in flight behind this row's arithmetic
    A r = 0.0f;
    if (ALL || p.y) {
      r = rsqrt_(row_sum<WIDE>(ss, lds, slot) * inv + p.eps);
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          x[k][e] *= r;
          if (ALL || p.gate) gate_(g[k][e], g[k][e], slope[k][e]);
          else g[k][e] = (A)1.0, slope[k][e] = (A)0.0;
        }
    }
    if (ALL || p.g_n) {
      A sums[2] = {0.0f, 0.0f};
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          if (ALL || p.y) {
            const A u = x[k][e] * w[k][e] * g[k][e];
            o[k][e] = fma_((A)s[k][e], u, o[k][e]);
          }
          sums[0] += o[k][e] * o[k][e];
          sums[1] += q[k][e] * wn[k][e] * o[k][e];
        }
      row_sums<WIDE, 2>(sums, lds, slot);
      const A r2 = rsqrt_(sums[0] * inv + p.eps), m = sums[1] * inv * r2 * r2;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          an[k][e] += q[k][e] * o[k][e] * r2;
          d[k][e] += r2 * (q[k][e] * wn[k][e] - o[k][e] * m);
        }
    }
    if (ALL || p.d_res) {
      const Row<R, VEC> out(p.d_res, row * p.d_res_st, p.H);
#pragma unroll
      for (int k = 0; k < NV; ++k) out.put(d[k], c[k]);
    }
    if (ALL || p.y) {
      A sm = 0.0f;
      const Row<Br, VEC> out(p.d_gate, row * p.d_gate_st, p.H);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        A dg[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const A u = x[k][e] * w[k][e], ds = d[k][e] * s[k][e];
          as[k][e] += d[k][e] * g[k][e] * u;
          dg[e] = ds * u * slope[k][e];
          const A t = ds * g[k][e];
          aw[k][e] += t * x[k][e];
          d[k][e] = t * w[k][e];
          sm += d[k][e] * x[k][e];
        }
        if (ALL || p.d_gate) out.put(dg, c[k]);
      }
      sm = row_sum<WIDE>(sm, lds, slot) * inv;
      if (ALL || p.d_y) {
        const Row<Y, VEC> dst(p.d_y, row * p.d_y_st, p.H);
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          A dy[VEC];
#pragma unroll
          for (int e = 0; e < VEC; ++e) dy[e] = r * (d[k][e] - x[k][e] * sm);
          dst.put(dy, c[k]);
        }
      }
    }
  }
  // this workgroup's slab: d_w | d_scale | d_w_next
  float* slab = p.ws + (int64_t)blockIdx.x * 3 * p.H;
#pragma unroll
  for (int which = 0; which < 3; ++which)
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      auto& acc = which == 0 ? aw[k] : which == 1 ? as[k] : an[k];
      if constexpr (!WIDE) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) fold[threadIdx.x * VEC + e] = (float)acc[e];
        __syncthreads();
        if (threadIdx.x < 64 * VEC) {
          const int i = threadIdx.x, col = k * 64 * VEC + i;
          if (col < p.H) slab[which * p.H + col] = fold[i] + fold[64 * VEC + i] + fold[128 * VEC + i] + fold[192 * VEC + i];
        }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e)
          if (c[k] + e < p.H) slab[which * p.H + c[k] + e] = (float)acc[e];
      }
    }
}

// One time step of the recurrence with its block norm: a row b of the state, TPR threads
template <typename Br, typename R, int NV, int TPR>
__global__ __launch_bounds__(TPR) void step_kernel(mdmm_gated_scan_t q, mdmm_block_norm_t p) {
  constexpr bool WIDE = TPR > 64;
  __shared__ float lds[64];
  clear_sums<WIDE>(lds);
  int slot = 0;
  const int64_t b = blockIdx.x;
  const float inv = 1.0f / (float)p.H;
  const bool live = !q.mask || q.mask[b * q.mask_sb];
  const Br* row = (const Br*)q.gates + b * q.gates_sb;
  float h[NV], o[NV];
  float ss = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = k * TPR + threadIdx.x;
    h[k] = o[k] = 0.0f;
    if (c < p.H) {
      h[k] = q.h0 ? q.h0[b * q.h0_sb + c] : 0.0f;
      if (live) {
        const Gate g(load1(row + c));
        h[k] = g.a * h[k] + g.k * load1(row + p.H + c);
      }
      q.h_last[b * p.H + c] = h[k];
      o[k] = load1((const R*)p.res + b * p.res_st + c);
    }
    ss += h[k] * h[k];
  }
  float r = rsqrtf(row_sum<WIDE>(ss, lds, slot) * inv + p.eps);
  ss = 0.0f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = k * TPR + threadIdx.x;
    if (c < p.H) {
      float u = h[k] * r * p.w[c];
      if (p.gate) {
        const float g = load1((const Br*)p.gate + b * p.gate_st + c);
        u *= g * sigmoid_(g);
      }
      o[k] = p.scale ? fmaf(p.scale[c], u, o[k]) : o[k] + u;
      store1((R*)p.out + b * p.out_st + c, o[k]);
    }
    ss += o[k] * o[k];
  }
  if (!p.w_next) return;
  r = rsqrtf(row_sum<WIDE>(ss, lds, slot) * inv + p.eps);
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = k * TPR + threadIdx.x;
    if (c < p.H) store1((Br*)p.n + b * p.n_st + c, o[k] * r * p.w_next[c]);
  }
}

template <typename Br, typename R>
int launch_step(const mdmm_gated_scan_t* q, const mdmm_block_norm_t* p, hipStream_t s) {
  const dim3 g((unsigned)p->rows);
  if (p->H <= 256) hipLaunchKernelGGL((step_kernel<Br, R, 4, 64>), g, dim3(64), 0, s, *q, *p);
  else if (p->H <= 1024) hipLaunchKernelGGL((step_kernel<Br, R, 4, 256>), g, dim3(256), 0, s, *q, *p);
  else hipLaunchKernelGGL((step_kernel<Br, R, 8, 1024>), g, dim3(1024), 0, s, *q, *p);
  return (int)hipGetLastError();
}

// column sums of the slabs: 16 columns (64 bytes of a slab) and 64 threads down each a workgroup, joined in a fixed order;
// at 1024 slabs a thread has 16 loads, all in flight (with 16 threads down a column the launch took 20 us at H = 256)
__global__ __launch_bounds__(1024) void norm_fold_kernel(const float* __restrict__ ws, int slabs, int H, float* d_w, float* d_s,
                                                         float* d_n) {
  __shared__ float part[64][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
  float s = 0.0f;
  if (c < 3 * H) {
#pragma unroll 16
    for (int i = r; i < slabs; i += 64) s += ws[(int64_t)i * 3 * H + c];
  }
  part[r][threadIdx.x & 15] = s;
  __syncthreads();
  if (threadIdx.x < 256) {
    const int q = threadIdx.x >> 4, k = threadIdx.x & 15;
    part[q][k] = (part[q][k] + part[q + 16][k]) + (part[q + 32][k] + part[q + 48][k]);
  }
  __syncthreads();
  if (r == 0 && c < 3 * H) {
    s = 0.0f;
    for (int i = 0; i < 16; ++i) s += part[i][threadIdx.x & 15];
    float* dst = c < H ? d_w : c < 2 * H ? d_s : d_n;
    if (dst) dst[c % H] = s;
  }
}

struct Plan { int vec, nv, maxt, threads; };

bool aligned(const void* p, int64_t st, int bf16) {
  return !p || (((uintptr_t)p & (bf16 ? 7 : 15)) == 0 && (st & 3) == 0);
}

Plan plan(const mdmm_block_norm_t* a) {
  const bool v4 = (a->H & 3) == 0 && aligned(a->y, a->y_st, a->y_bf16) && aligned(a->gate, a->gate_st, a->branch_bf16) &&
                  aligned(a->res, a->res_st, a->res_bf16) && aligned(a->out, a->out_st, a->res_bf16) &&
                  aligned(a->n, a->n_st, a->branch_bf16) && aligned(a->g_out, a->g_out_st, a->res_bf16) &&
                  aligned(a->g_n, a->g_n_st, a->branch_bf16) && aligned(a->d_y, a->d_y_st, a->y_bf16) &&
                  aligned(a->d_gate, a->d_gate_st, a->branch_bf16) && aligned(a->d_res, a->d_res_st, a->res_bf16) &&
                  aligned(a->w, 0, 0) && aligned(a->scale, 0, 0) && aligned(a->w_next, 0, 0);
  if (a->H <= 4) return {1, 1, 256, 256};          // (64-bit arithmetic: norm_bwd_kernel)
  const int h = a->H, w4 = (h + 255) / 256 * 64, w8 = (h + 511) / 512 * 64;
  if (v4) {
    if (h <= 256) return {4, 1, 256, 256};
    if (h <= 2048) return {4, 1, 512, w4};
    if (h <= 4096) return {4, 2, 512, w8};
    return {4, 2, 1024, w8};
  }
  const int u4 = (h + 255) / 256 * 64, u8 = (h + 511) / 512 * 64;
  if (h <= 256) return {1, 4, 256, 256};
  if (h <= 2048) return {1, 4, 512, u4};
  if (h <= 4096) return {1, 4, 1024, u4};
  return {1, 8, 1024, u8};
}

// Workgroups: as many as the registers let the chip hold at once (16 or, bf16 backward, 20 waves a CU), each walking over
// rows -- a few more than that would run as a second, nearly empty round (1024 workgroups where 768 fit: 480 us instead of
// 383 at 65536 x 1280) -- and no more than one for eight rows beyond 1024 of them (each leaves a slab of 3 H sums)
int64_t grid_of(const mdmm_block_norm_t* a, const Plan& q, bool bwd) {
  const int rpw = q.maxt == 256 ? 4 : 1, waves = q.threads / 64;
  const int64_t need = (a->rows + rpw - 1) / rpw;
  const int per_cu = ((bwd ? a->y_bf16 && a->res_bf16 && q.maxt == 512 && q.nv * q.vec == 4 : false) ? 20 : 16) / waves;
  int64_t top = 256 * (int64_t)(per_cu > 0 ? per_cu : 1);
  if (top > 1024 && top > need / 8) top = need / 8 > 1024 ? need / 8 : 1024;
  if (top > 2048) top = 2048;
  return need < top ? need : top;
}

int check(const mdmm_block_norm_t* a) {
  if (!a || a->rows < 0 || a->H < 1 || !(a->eps >= 0.0f)) return MDMM_E_ARG;
  if (a->H > MDMM_NORM_MAX_H) return MDMM_E_LIMIT;
  if (a->rows > 0 && !a->res) return MDMM_E_ARG;
  if (a->y && !a->w) return MDMM_E_ARG;
  if (!a->y && (a->gate || a->scale || !a->w_next)) return MDMM_E_ARG;
  const int t = (a->y_bf16 ? 4 : 0) | (a->branch_bf16 ? 2 : 0) | (a->res_bf16 ? 1 : 0);
  if (a->y && t != 0 && t != 7 && t != 6 && t != 2 && t != 3) return MDMM_E_ARG;
  if (!a->y && !a->branch_bf16 && a->res_bf16) return MDMM_E_ARG;
  return 0;
}

// every operand of a whole block there: a variant without the tests for what is missing
bool whole(const mdmm_block_norm_t* a, bool bwd) {
  return a->y && a->gate && a->w_next && (!bwd || (a->g_out && a->g_n && a->d_y && a->d_gate && a->d_res));
}

template <typename Y, typename Br, typename R, int VEC, int NV, int MAXT>
int launch(const mdmm_block_norm_t* a, int64_t grid, int threads, bool bwd, hipStream_t s) {
  const dim3 g((unsigned)grid), t(threads);
  const bool all = whole(a, bwd);
  if (bwd && all) hipLaunchKernelGGL((norm_bwd_kernel<Y, Br, R, VEC, NV, MAXT, true>), g, t, 0, s, *a);
  else if (bwd) hipLaunchKernelGGL((norm_bwd_kernel<Y, Br, R, VEC, NV, MAXT, false>), g, t, 0, s, *a);
  else if (all) hipLaunchKernelGGL((norm_fwd_kernel<Y, Br, R, VEC, NV, MAXT, true>), g, t, 0, s, *a);
  else hipLaunchKernelGGL((norm_fwd_kernel<Y, Br, R, VEC, NV, MAXT, false>), g, t, 0, s, *a);
  return (int)hipGetLastError();
}

template <typename Y, typename Br, typename R>
int dispatch(const mdmm_block_norm_t* a, bool bwd, hipStream_t s) {
  const Plan q = plan(a);
  const int64_t g = grid_of(a, q, bwd);
#define CASE(v, n, t) if (q.vec == v && q.nv == n && q.maxt == t) return launch<Y, Br, R, v, n, t>(a, g, q.threads, bwd, s)
  CASE(4, 1, 256); CASE(4, 1, 512); CASE(4, 2, 512); CASE(4, 2, 1024);
  CASE(1, 1, 256); CASE(1, 4, 256); CASE(1, 4, 512); CASE(1, 4, 1024); CASE(1, 8, 1024);
#undef CASE
  return MDMM_E_ARG;
}

int run(const mdmm_block_norm_t* a, bool bwd, hipStream_t s) {
  if (a->y ? a->y_bf16 : a->res_bf16)
    return a->res_bf16 ? dispatch<__bf16, __bf16, __bf16>(a, bwd, s) : dispatch<__bf16, __bf16, float>(a, bwd, s);
  if (!a->branch_bf16) return dispatch<float, float, float>(a, bwd, s);
  return a->res_bf16 ? dispatch<float, __bf16, __bf16>(a, bwd, s) : dispatch<float, __bf16, float>(a, bwd, s);
}

}  // namespace
}  // namespace mdmm

using namespace mdmm;

extern "C" int64_t mdmm_block_norm_ws(const mdmm_block_norm_t* a) {
  if (check(a)) return -1;
  return (a->rows < 2048 ? a->rows : 2048) * 3 * a->H;       // (the most workgroups any plan takes)
}

extern "C" int mdmm_block_norm_fwd(const mdmm_block_norm_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (a->rows == 0) return 0;
  if ((a->y && !a->out) || (a->w_next && !a->n)) return MDMM_E_ARG;
  return run(a, false, (hipStream_t)stream);
}

extern "C" int mdmm_block_norm_bwd(const mdmm_block_norm_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (a->rows == 0) return 0;
  if (!a->ws || (!a->g_out && !a->g_n) || (a->g_n && !a->w_next)) return MDMM_E_ARG;
  const int e = run(a, true, (hipStream_t)stream);
  if (e) return e;
  if (!a->d_w && !a->d_scale && !a->d_w_next) return 0;
  hipLaunchKernelGGL(norm_fold_kernel, dim3((3 * a->H + 15) / 16), dim3(1024), 0, (hipStream_t)stream, a->ws,
                     (int)grid_of(a, plan(a), true), a->H, a->d_w, a->d_scale, a->d_w_next);
  return (int)hipGetLastError();
}

extern "C" int mdmm_gated_block_step(const mdmm_gated_scan_t* q, const mdmm_block_norm_t* p, void* stream) {
  if (!q || !p || q->B < 0 || q->H < 1 || p->rows != q->B || p->H != q->H || !(p->eps >= 0.0f)) return MDMM_E_ARG;
  if (q->H > MDMM_NORM_MAX_H) return MDMM_E_LIMIT;
  if (q->B == 0) return 0;
  if (q->T != 1 || !q->gates || !q->h_last || !p->res || !p->out || !p->w || (p->w_next && !p->n)) return MDMM_E_ARG;
  if (!!q->gates_bf16 != !!p->branch_bf16 || (!p->branch_bf16 && p->res_bf16)) return MDMM_E_ARG;
  const Region last = region(q->h_last, q->B, q->H, q->H, 4);
  if (last_state_on_input(q) || meet(last, region(p->res, q->B, p->res_st, q->H, p->res_bf16 ? 2 : 4)) ||
      meet(last, region(p->gate, q->B, p->gate_st, q->H, p->branch_bf16 ? 2 : 4)) || meet(last, region(p->w, 1, 0, q->H, 4)) ||
      meet(last, region(p->scale, 1, 0, q->H, 4)) || meet(last, region(p->w_next, 1, 0, q->H, 4)))
    return MDMM_E_ALIAS;
  hipStream_t s = (hipStream_t)stream;
  if (!p->branch_bf16) return launch_step<float, float>(q, p, s);
  return p->res_bf16 ? launch_step<__bf16, __bf16>(q, p, s) : launch_step<__bf16, float>(q, p, s);
}

extern "C" int mdmm_gated_block_fwd(const mdmm_gated_scan_t* q, const mdmm_block_norm_t* p, void* stream) {
  if (!q || !p || p->y != q->h || p->H != q->H || p->rows != (int64_t)q->T * q->B) return MDMM_E_ARG;
  const int rc = mdmm_gated_scan_fwd(q, stream);
  return rc ? rc : mdmm_block_norm_fwd(p, stream);
}

extern "C" int mdmm_gated_block_bwd(const mdmm_gated_scan_t* q, const mdmm_block_norm_t* p, void* stream) {
  if (!q || !p || p->H != q->H || p->rows != (int64_t)q->T * q->B) return MDMM_E_ARG;
  if (p->g_out || p->g_n) {
    if (p->d_y != q->g_h) return MDMM_E_ARG;
    const int rc = mdmm_block_norm_bwd(p, stream);
    if (rc) return rc;
  }
  return mdmm_gated_scan_bwd(q, stream);
}
