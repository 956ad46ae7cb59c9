// Orthogonalised matrix updates by Newton-Schulz products (mdmm_ortho_t): X = M / (|M|_F + eps), then
// X <- ca X + (cb A + cc A A) X with A = X X^T.  X lies down (n rows <= m columns), so both Gram-side products are n x n.
// The iteration multiplies a small singular value by up to ca per step (ca^5 = 485 over five), and a rounding of X with it:
// everything stays in fp32, on the fp32 matrix instruction.
// Workspace per matrix, n and m rounded up to whole tiles with zeros (which every product keeps): two X buffers, A and the
// polynomial P = ca I + cb A + cc A A.  All matrices of a call share each launch.
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/mdmm_hip.h"

namespace mdmm {
namespace {

constexpr int NT = 256, TILE = 64, KB = 16, SUMS = 64;
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct Item {               // one matrix's padded sizes and workspace
  float *x0, *x1, *gram, *poly, *sums;
  int32_t n, m, tall, reserved;
};
struct Items {
  Item it[MDMM_ORTHO_MAX];
  int32_t first[MDMM_ORTHO_MAX + 1];       // first tile of each matrix in this launch
  int32_t n;
};

__device__ __forceinline__ int find(const int32_t* first, int n, int tile) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (first[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float src_at(const mdmm_ortho_t& p, const mdmm_ortho_item_t& t, int64_t r, int64_t c) {
  const int64_t i = r * t.src_ld + c;
  return p.src_bf16 ? (float)((const __bf16*)t.src)[i] : ((const float*)t.src)[i];
}

// element (r, c) of the result: stored, or taken as one optimizer step
__device__ __forceinline__ void put(const mdmm_ortho_t& p, const mdmm_ortho_item_t& t, int64_t r, int64_t c, float v) {
  const int64_t o = r * t.dst_ld + c;
  if (p.update) {
    float* d = (float*)t.dst + o;
    const float lr = p.lr_dev ? *p.lr_dev : p.lr;
    *d = fmaf(-lr * t.gain, v, (1.0f - lr * p.decay) * *d);
  } else if (p.dst_bf16) ((__bf16*)t.dst)[o] = (__bf16)v;
  else ((float*)t.dst)[o] = v;
}

// momentum, and the sum of squares in SUMS pieces
__global__ __launch_bounds__(NT) void ortho_sums_kernel(mdmm_ortho_t p, Items q) {
  const int k = blockIdx.y;
  const mdmm_ortho_item_t& t = p.item[k];
  const int64_t total = (int64_t)t.rows * t.cols;
  float s = 0.0f;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < total; i += (int64_t)SUMS * NT) {
    float v = src_at(p, t, i / t.cols, i % t.cols);
    if (t.mom) {
      const float mv = fmaf(p.momentum, t.mom[i], v);
      t.mom[i] = mv;
      v = p.nesterov ? fmaf(p.momentum, mv, v) : mv;
    }
    s = fmaf(v, v, s);
  }
  __shared__ float part[NT / 64];
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) q.it[k].sums[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

__global__ __launch_bounds__(NT) void ortho_pack_kernel(mdmm_ortho_t p, Items q) {
  const int k = blockIdx.y;
  const mdmm_ortho_item_t& t = p.item[k];
  const Item& w = q.it[k];
  float s = 0.0f;
  for (int i = 0; i < SUMS; ++i) s += w.sums[i];
  const float inv = 1.0f / (sqrtf(s) + p.eps);
  const int64_t total = (int64_t)w.n * w.m;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < total; i += (int64_t)gridDim.x * NT) {
    const int64_t a = i / w.m, b = i % w.m, r = w.tall ? b : a, c = w.tall ? a : b;
    float v = 0.0f;
    if (r < t.rows && c < t.cols) {
      v = src_at(p, t, r, c);
      if (t.mom) {
        const float mv = t.mom[r * t.cols + c];
        v = p.nesterov ? fmaf(p.momentum, mv, v) : mv;
      }
      v *= inv;
    }
    w.x0[i] = v;
  }
}

enum { GRAM, POLY, APPLY };

// One 64 x 64 tile of a product, four waves of 32 x 32: GRAM A = X X^T, POLY P = ca I + cb A + cc A A (A symmetric: its
// columns are read as rows), APPLY X' = P X (the last one into dst)
template <int MODE>
__global__ __launch_bounds__(NT) void ortho_product_kernel(mdmm_ortho_t p, Items q, int flip, int last) {
  __shared__ float As[KB][TILE + 4], Bs[KB][TILE + 4];
  const int k = find(q.first, q.n, blockIdx.x);
  const Item& w = q.it[k];
  const float* x = flip ? w.x1 : w.x0;
  float* xn = flip ? w.x0 : w.x1;
  const int K = MODE == GRAM ? w.m : w.n, J = MODE == APPLY ? w.m : w.n;
  const int tile = blockIdx.x - q.first[k], tj = J / TILE;
  const int i0 = tile / tj * TILE, j0 = tile % tj * TILE;
  const float* a = MODE == GRAM ? x : MODE == POLY ? w.gram : w.poly;       // (n, K), rows
  const float* b = MODE == POLY ? w.gram : x;                               // NT: (J, K) rows; APPLY: (K, J) rows
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wi = (wave >> 1) * 32, wj = (wave & 1) * 32;
  f32x16 acc = {};
  for (int k0 = 0; k0 < K; k0 += KB) {
    const int r = tid >> 2, c = (tid & 3) * 4;
    const float4 va = *(const float4*)(a + (int64_t)(i0 + r) * K + k0 + c);
    float4 vb;
    const int br = tid >> 4, bc = (tid & 15) * 4;
    if (MODE == APPLY) vb = *(const float4*)(b + (int64_t)(k0 + br) * J + j0 + bc);
    else vb = *(const float4*)(b + (int64_t)(j0 + r) * K + k0 + c);
    __syncthreads();
    As[c][r] = va.x; As[c + 1][r] = va.y; As[c + 2][r] = va.z; As[c + 3][r] = va.w;
    if (MODE == APPLY) *(float4*)&Bs[br][bc] = vb;
    else { Bs[c][r] = vb.x; Bs[c + 1][r] = vb.y; Bs[c + 2][r] = vb.z; Bs[c + 3][r] = vb.w; }
    __syncthreads();
#pragma unroll
    for (int kk = 0; kk < KB; kk += 2) {
      const float fa = As[kk + (lane >> 5)][wi + (lane & 31)], fb = Bs[kk + (lane >> 5)][wj + (lane & 31)];
      acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa, fb, acc, 0, 0, 0);
    }
  }
  const mdmm_ortho_item_t& t = p.item[k];
#pragma unroll
  for (int e = 0; e < 16; ++e) {
    const int64_t i = i0 + wi + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3), j = j0 + wj + (lane & 31);
    float v = acc[e];
    if (MODE == GRAM) w.gram[i * J + j] = v;
    if (MODE == POLY) w.poly[i * J + j] = fmaf(p.cc, v, fmaf(p.cb, w.gram[i * J + j], i == j ? p.ca : 0.0f));
    if (MODE == APPLY && !last) xn[i * J + j] = v;
    if (MODE == APPLY && last) {
      const int64_t r = w.tall ? j : i, c = w.tall ? i : j;
      if (r < t.rows && c < t.cols) {
        put(p, t, r, c, v);
      }
    }
  }
}

__global__ __launch_bounds__(NT) void ortho_copy_kernel(mdmm_ortho_t p, Items q) {       // steps = 0: X itself
  const mdmm_ortho_item_t& t = p.item[blockIdx.y];
  const Item& w = q.it[blockIdx.y];
  const int64_t total = (int64_t)t.rows * t.cols;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < total; i += (int64_t)gridDim.x * NT) {
    const int64_t r = i / t.cols, c = i % t.cols;
    const float v = w.tall ? w.x0[c * w.m + r] : w.x0[r * w.m + c];
    put(p, t, r, c, v);
  }
}

int check(const mdmm_ortho_t* a) {
  if (!a || a->n < 0 || a->steps < 0 || !(a->eps >= 0.0f)) return MDMM_E_ARG;
  if (a->n > MDMM_ORTHO_MAX) return MDMM_E_LIMIT;
  if (a->update && a->dst_bf16) return MDMM_E_ARG;
  for (int i = 0; i < a->n; ++i) {
    const mdmm_ortho_item_t& t = a->item[i];
    if (t.rows < 1 || t.cols < 1 || t.src_ld < t.cols || t.dst_ld < t.cols) return MDMM_E_ARG;
    if (t.rows > 65536 || t.cols > 65536) return MDMM_E_LIMIT;
  }
  return 0;
}

int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }

// fills the workspace pointers (base may be NULL: sizes only) and returns the bytes used
int64_t lay_out(const mdmm_ortho_t* a, Items* q) {
  char* base = (char*)a->ws;
  int64_t off = 0;
  q->n = a->n;
  for (int i = 0; i < a->n; ++i) {
    const mdmm_ortho_item_t& t = a->item[i];
    Item& w = q->it[i];
    w.tall = t.rows > t.cols;
    w.n = (int32_t)up(w.tall ? t.cols : t.rows, TILE);
    w.m = (int32_t)up(w.tall ? t.rows : t.cols, TILE);
    const int64_t x = (int64_t)w.n * w.m, g = (int64_t)w.n * w.n;
    w.x0 = (float*)(base + off); off += 4 * x;
    w.x1 = (float*)(base + off); off += 4 * x;
    w.gram = (float*)(base + off); off += 4 * g;
    w.poly = (float*)(base + off); off += 4 * g;
    w.sums = (float*)(base + off); off += 4 * SUMS;
  }
  return off;
}

int tiles(Items* q, bool wide) {
  int64_t total = 0;
  for (int i = 0; i < q->n; ++i) {
    q->first[i] = (int32_t)total;
    total += (int64_t)(q->it[i].n / TILE) * ((wide ? q->it[i].m : q->it[i].n) / TILE);
  }
  q->first[q->n] = (int32_t)total;
  return (int)total;
}

}  // namespace
}  // namespace mdmm

using namespace mdmm;

extern "C" int64_t mdmm_ortho_ws(const mdmm_ortho_t* a) {
  if (check(a)) return -1;
  Items q;
  return lay_out(a, &q);
}

extern "C" int mdmm_ortho(const mdmm_ortho_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (a->n == 0) return 0;
  if (!a->ws || ((uintptr_t)a->ws & 255)) return a->ws ? MDMM_E_ALIGN : MDMM_E_ARG;
  for (int i = 0; i < a->n; ++i)
    if (!a->item[i].src || !a->item[i].dst) return MDMM_E_ARG;
  hipStream_t s = (hipStream_t)stream;
  Items q;
  lay_out(a, &q);
  hipLaunchKernelGGL(ortho_sums_kernel, dim3(SUMS, a->n), dim3(NT), 0, s, *a, q);
  hipLaunchKernelGGL(ortho_pack_kernel, dim3(256, a->n), dim3(NT), 0, s, *a, q);
  if (a->steps == 0) hipLaunchKernelGGL(ortho_copy_kernel, dim3(256, a->n), dim3(NT), 0, s, *a, q);
  const int square = tiles(&q, false);
  Items qw = q;
  const int wide = tiles(&qw, true);
  for (int k = 0; k < a->steps; ++k) {
    hipLaunchKernelGGL(ortho_product_kernel<GRAM>, dim3(square), dim3(NT), 0, s, *a, q, k & 1, 0);
    hipLaunchKernelGGL(ortho_product_kernel<POLY>, dim3(square), dim3(NT), 0, s, *a, q, k & 1, 0);
    hipLaunchKernelGGL(ortho_product_kernel<APPLY>, dim3(wide), dim3(NT), 0, s, *a, qw, k & 1, k + 1 == a->steps);
  }
  return (int)hipGetLastError();
}
