// Norms before and after a residual block fused with the block's gate and residual scale (mdmm_block_norm_t):
//   u = y r w, r = rsqrt(mean(y^2) + eps);  out = res + s silu(g) u;  n = out r' w'
// Backward, with d = g_out + r' (q - out r'^2 mean(q out)), q = g_n w' :  d_res = d, d_s = sum d silu(g) u,
// d_g = d s u silu'(g), p = d s silu(g):  d_w = sum p y r,  d_y = r (p w - y r mean(p w y r)),  d_w' = sum g_n out r'.
// A row is held in registers by TPR threads (NV pieces of VEC columns each) from its loads to its stores, so every tensor
// passes once; the three column sums are kept per thread over all rows of a workgroup and leave as one slab a workgroup,
// which fold_kernel adds up in a fixed order.
#include "gated.h"

namespace mdmm {
namespace {

template <int VEC> __device__ __forceinline__ void load_v(const float* p, float* v) {
  if constexpr (VEC == 4) {
    const float4 x = *(const float4*)p;
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else v[0] = *p;
}
template <int VEC> __device__ __forceinline__ void load_v(const __bf16* p, float* v) {
  if constexpr (VEC == 4) {
    const uint2 x = *(const uint2*)p;
    v[0] = __uint_as_float(x.x << 16); v[1] = __uint_as_float(x.x & 0xffff0000u);
    v[2] = __uint_as_float(x.y << 16); v[3] = __uint_as_float(x.y & 0xffff0000u);
  } else v[0] = (float)*p;
}
template <int VEC> __device__ __forceinline__ void store_v(float* p, const float* v) {
  if constexpr (VEC == 4) *(float4*)p = make_float4(v[0], v[1], v[2], v[3]);
  else *p = v[0];
}
template <int VEC> __device__ __forceinline__ void store_v(__bf16* p, const float* v) {
  if constexpr (VEC == 4) {
    typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
    bf16x4 x;
    x[0] = (__bf16)v[0]; x[1] = (__bf16)v[1]; x[2] = (__bf16)v[2]; x[3] = (__bf16)v[3];
    *(bf16x4*)p = x;
  } else *p = (__bf16)v[0];
}

// sum over the TPR threads of a row, in every one of them
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* lds, int& slot) {
  for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
  if constexpr (TPR > 64) {
    constexpr int W = TPR / 64;
    float* s = lds + (slot ^= 1) * W;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
    for (int w = 0; w < W; ++w) v += s[w];
  }
  return v;
}

template <typename Y, typename Br, typename R, int VEC, int NV, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_fwd_kernel(mdmm_block_norm_t p) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPW = NT / TPR;
  __shared__ float lds[2 * (TPR / 64)];
  int slot = 0;
  const int lane = threadIdx.x % TPR;
  const float inv = 1.0f / (float)p.H;
  for (int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR; row < p.rows; row += (int64_t)gridDim.x * RPW) {
    float o[NV][VEC], y[NV][VEC], g[NV][VEC];
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[k][e] = y[k][e] = g[k][e] = 0.0f;
      if (c < p.H) {
        load_v<VEC>((const R*)p.res + row * p.res_st + c, o[k]);
        if (p.y) load_v<VEC>((const Y*)p.y + row * p.y_st + c, y[k]);
        if (p.gate) load_v<VEC>((const Br*)p.gate + row * p.gate_st + c, g[k]);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += y[k][e] * y[k][e];
    }
    if (p.y) {
      const float r = rsqrtf(row_sum<TPR>(ss, lds, slot) * inv + p.eps);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H) {
          float w[VEC], s[VEC];
          load_v<VEC>(p.w + c, w);
          if (p.scale) load_v<VEC>(p.scale + c, s);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float u = y[k][e] * r * w[e];
            if (p.gate) u *= g[k][e] * sigmoid_(g[k][e]);
            o[k][e] = p.scale ? fmaf(s[e], u, o[k][e]) : o[k][e] + u;
          }
          store_v<VEC>((R*)p.out + row * p.out_st + c, o[k]);
        }
      }
    }
    if (p.w_next) {
      ss = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) ss += o[k][e] * o[k][e];
      const float r = rsqrtf(row_sum<TPR>(ss, lds, slot) * inv + p.eps);
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H) {
          float w[VEC];
          load_v<VEC>(p.w_next + c, w);
#pragma unroll
          for (int e = 0; e < VEC; ++e) o[k][e] *= r * w[e];
          store_v<VEC>((Br*)p.n + row * p.n_st + c, o[k]);
        }
      }
    }
  }
}

template <typename Y, typename Br, typename R, int VEC, int NV, int TPR>
__global__ __launch_bounds__(TPR > 256 ? TPR : 256) void norm_bwd_kernel(mdmm_block_norm_t p) {
  constexpr int NT = TPR > 256 ? TPR : 256, RPW = NT / TPR;
  __shared__ float lds[2 * (TPR / 64)];
  __shared__ float fold[RPW > 1 ? RPW * TPR * VEC : 1];
  int slot = 0;
  const int lane = threadIdx.x % TPR;
  const float inv = 1.0f / (float)p.H;
  float aw[NV][VEC] = {}, as[NV][VEC] = {}, an[NV][VEC] = {};
  for (int64_t row = (int64_t)blockIdx.x * RPW + threadIdx.x / TPR; row < p.rows; row += (int64_t)gridDim.x * RPW) {
    float o[NV][VEC], y[NV][VEC], g[NV][VEC], d[NV][VEC], q[NV][VEC];
    float ss = 0.0f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + lane) * VEC;
#pragma unroll
      for (int e = 0; e < VEC; ++e) o[k][e] = y[k][e] = g[k][e] = d[k][e] = q[k][e] = 0.0f;
      if (c < p.H) {
        load_v<VEC>((const R*)p.res + row * p.res_st + c, o[k]);
        if (p.y) load_v<VEC>((const Y*)p.y + row * p.y_st + c, y[k]);
        if (p.gate) load_v<VEC>((const Br*)p.gate + row * p.gate_st + c, g[k]);
        if (p.g_out) load_v<VEC>((const R*)p.g_out + row * p.g_out_st + c, d[k]);
        if (p.g_n) load_v<VEC>((const Br*)p.g_n + row * p.g_n_st + c, q[k]);
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) ss += y[k][e] * y[k][e];
    }
    float r = 0.0f;
    if (p.y) r = rsqrtf(row_sum<TPR>(ss, lds, slot) * inv + p.eps);
    if (p.g_n) {
      float s2 = 0.0f, sq = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H) {
          float w[VEC], s[VEC], wn[VEC];
          if (p.y) load_v<VEC>(p.w + c, w);
          if (p.scale) load_v<VEC>(p.scale + c, s);
          load_v<VEC>(p.w_next + c, wn);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            if (p.y) {
              float u = y[k][e] * r * w[e];
              if (p.gate) u *= g[k][e] * sigmoid_(g[k][e]);
              o[k][e] = p.scale ? fmaf(s[e], u, o[k][e]) : o[k][e] + u;
            }
            s2 += o[k][e] * o[k][e];
            sq += q[k][e] * wn[e] * o[k][e];
          }
        }
      }
      const float r2 = rsqrtf(row_sum<TPR>(s2, lds, slot) * inv + p.eps);
      const float m = row_sum<TPR>(sq, lds, slot) * inv * r2 * r2;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H) {
          float wn[VEC];
          load_v<VEC>(p.w_next + c, wn);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            an[k][e] += q[k][e] * o[k][e] * r2;
            d[k][e] += r2 * (q[k][e] * wn[e] - o[k][e] * m);
          }
        }
      }
    }
    if (p.d_res) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H) store_v<VEC>((R*)p.d_res + row * p.d_res_st + c, d[k]);
      }
    }
    if (p.y) {
      float sm = 0.0f;
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H) {
          float w[VEC], s[VEC], dg[VEC];
          load_v<VEC>(p.w + c, w);
          if (p.scale) load_v<VEC>(p.scale + c, s);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            const float x = y[k][e] * r, u = x * w[e], sc = p.scale ? s[e] : 1.0f;
            float act = 1.0f, slope = 0.0f;
            if (p.gate) {
              const Gate sg(g[k][e]);
              act = g[k][e] * sg.a;
              slope = sg.a * fmaf(g[k][e], sg.k, 1.0f);
            }
            as[k][e] += d[k][e] * act * u;
            dg[e] = d[k][e] * sc * u * slope;
            const float t = d[k][e] * sc * act;
            aw[k][e] += t * x;
            y[k][e] = x;
            d[k][e] = t * w[e];
            sm += d[k][e] * x;
          }
          if (p.d_gate) store_v<VEC>((Br*)p.d_gate + row * p.d_gate_st + c, dg);
        }
      }
      sm = row_sum<TPR>(sm, lds, slot) * inv;
      if (p.d_y) {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
          const int c = (k * TPR + lane) * VEC;
          if (c < p.H) {
            float dy[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) dy[e] = r * (d[k][e] - y[k][e] * sm);
            store_v<VEC>((Y*)p.d_y + row * p.d_y_st + c, dy);
          }
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
      float (&acc)[VEC] = which == 0 ? aw[k] : which == 1 ? as[k] : an[k];
      if constexpr (RPW > 1) {
        __syncthreads();
#pragma unroll
        for (int e = 0; e < VEC; ++e) fold[(threadIdx.x / TPR * TPR + lane) * VEC + e] = acc[e];
        __syncthreads();
        for (int i = threadIdx.x; i < TPR * VEC; i += NT) {
          const int c = k * TPR * VEC + i;
          if (c < p.H) {
            float s = 0.0f;
            for (int w = 0; w < RPW; ++w) s += fold[w * TPR * VEC + i];
            slab[which * p.H + c] = s;
          }
        }
      } else {
        const int c = (k * TPR + lane) * VEC;
        if (c < p.H)
          for (int e = 0; e < VEC; ++e) slab[which * p.H + c + e] = acc[e];
      }
    }
}

// One time step of the recurrence with its block norm: a row b of the state, TPR threads
template <typename Br, typename R, int NV, int TPR>
__global__ __launch_bounds__(TPR) void step_kernel(mdmm_gated_scan_t q, mdmm_block_norm_t p) {
  __shared__ float lds[2 * (TPR / 64)];
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
  float r = rsqrtf(row_sum<TPR>(ss, lds, slot) * inv + p.eps);
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
  r = rsqrtf(row_sum<TPR>(ss, lds, slot) * inv + p.eps);
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

// column sums of the slabs: 16 columns a workgroup, 16 threads down each column, joined in a fixed order
__global__ __launch_bounds__(256) void norm_fold_kernel(const float* __restrict__ ws, int slabs, int H, float* d_w, float* d_s,
                                                        float* d_n) {
  __shared__ float part[16][17];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15), r = threadIdx.x >> 4;
  float s = 0.0f;
  if (c < 3 * H)
    for (int i = r; i < slabs; i += 16) s += ws[(int64_t)i * 3 * H + c];
  part[r][threadIdx.x & 15] = s;
  __syncthreads();
  if (r == 0 && c < 3 * H) {
    s = 0.0f;
    for (int i = 0; i < 16; ++i) s += part[i][threadIdx.x & 15];
    float* dst = c < H ? d_w : c < 2 * H ? d_s : d_n;
    if (dst) dst[c % H] = s;
  }
}

struct Plan { int vec, nv, tpr; };

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
  if (v4) {
    if (a->H <= 256) return {4, 1, 64};
    if (a->H <= 512) return {4, 2, 64};
    if (a->H <= 1024) return {4, 4, 64};
    if (a->H <= 2048) return {4, 2, 256};
    if (a->H <= 4096) return {4, 4, 256};
    return {4, 2, 1024};
  }
  if (a->H <= 256) return {1, 4, 64};
  if (a->H <= 1024) return {1, 4, 256};
  if (a->H <= 4096) return {1, 4, 1024};
  return {1, 8, 1024};
}

int64_t grid_of(const mdmm_block_norm_t* a, const Plan& q) {
  const int rpw = q.tpr >= 256 ? 1 : 256 / q.tpr;
  const int64_t g = (a->rows + rpw - 1) / rpw;
  const int64_t top = q.tpr > 256 ? 512 : 1024;
  return g < top ? g : top;
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

template <typename Y, typename Br, typename R, int VEC, int NV, int TPR>
int launch(const mdmm_block_norm_t* a, int64_t grid, bool bwd, hipStream_t s) {
  constexpr int NT = TPR > 256 ? TPR : 256;
  if (bwd) hipLaunchKernelGGL((norm_bwd_kernel<Y, Br, R, VEC, NV, TPR>), dim3((unsigned)grid), dim3(NT), 0, s, *a);
  else hipLaunchKernelGGL((norm_fwd_kernel<Y, Br, R, VEC, NV, TPR>), dim3((unsigned)grid), dim3(NT), 0, s, *a);
  return (int)hipGetLastError();
}

template <typename Y, typename Br, typename R>
int dispatch(const mdmm_block_norm_t* a, bool bwd, hipStream_t s) {
  const Plan q = plan(a);
  const int64_t g = grid_of(a, q);
#define CASE(v, n, t) if (q.vec == v && q.nv == n && q.tpr == t) return launch<Y, Br, R, v, n, t>(a, g, bwd, s)
  CASE(4, 1, 64); CASE(4, 2, 64); CASE(4, 4, 64); CASE(4, 2, 256); CASE(4, 4, 256); CASE(4, 2, 1024);
  CASE(1, 4, 64); CASE(1, 4, 256); CASE(1, 4, 1024); CASE(1, 8, 1024);
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
  return (a->rows < 1024 ? a->rows : 1024) * 3 * a->H;       // (the most workgroups any plan takes)
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
  hipLaunchKernelGGL(norm_fold_kernel, dim3((3 * a->H + 15) / 16), dim3(256), 0, (hipStream_t)stream, a->ws,
                     (int)grid_of(a, plan(a)), a->H, a->d_w, a->d_scale, a->d_w_next);
  return (int)hipGetLastError();
}

extern "C" int mdmm_gated_block_step(const mdmm_gated_scan_t* q, const mdmm_block_norm_t* p, void* stream) {
  if (!q || !p || q->B < 0 || q->H < 1 || p->rows != q->B || p->H != q->H || !(p->eps >= 0.0f)) return MDMM_E_ARG;
  if (q->H > MDMM_NORM_MAX_H) return MDMM_E_LIMIT;
  if (q->B == 0) return 0;
  if (q->T != 1 || !q->gates || !q->h_last || !p->res || !p->out || !p->w || (p->w_next && !p->n)) return MDMM_E_ARG;
  if (!!q->gates_bf16 != !!p->branch_bf16 || (!p->branch_bf16 && p->res_bf16)) return MDMM_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  if (!p->branch_bf16) return launch_step<float, float>(q, p, s);
  return p->res_bf16 ? launch_step<__bf16, __bf16>(q, p, s) : launch_step<__bf16, float>(q, p, s);
}
