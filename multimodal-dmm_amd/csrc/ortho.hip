// Orthogonalised matrix updates by Newton-Schulz products (mdmm_ortho_t): X = M / (|M|_F + eps), then
// X <- ca X + P X with P = cb A + cc A A, A = X X^T.  X lies down (n rows <= m columns).
//
// The iteration multiplies a small singular value by up to ca a step (ca^5 = 485 over five), and a rounding of X with it, so
// bf16 operands are out; fp32 ones would run on the fp32 matrix instruction, a sixteenth of the fp16 one's rate.  Matrices
// with more than 128 rows are kept as two fp16 planes instead, s x = h + l with h = fp16(s x), l = fp16(s x - h): 22 to 23
// bits.  s is as large as the entries allow (X and A stay below 2: 2^14; P below 16: 2^12), so that l is a normal number down
// to entries of 1e-5 and below those wrong by 2e-12.  A product is h h' + h l' + l h': three fp16 matrix instructions, the
// dropped l l' 2^-23 of a term: the result is nearer to 64 bits than fp32 products by the library (6e-7 against 2.9e-6 at
// 2048 x 2048).  ca X is added in fp32.  (Up to 128 rows: fp32, see WHOLE.)
//
// A fixed s would lose X where eps makes it small (|M|_F of 1e-12 at eps 1e-7: 3e-5 off, in fp32 6e-8).  So what is kept is
// 2^k X with k from a bound t of X's singular values, |M|_F / (|M|_F + eps) at first and the polynomial's largest value on
// [0, t] after a step (Range); k = 0 from t = 1/2 on.  Then A is kept as 4^k A, P as 4^k P 2^-q.
//
// X is stored both ways (n x m for A, m x n for P X) so that every product runs over two operands' rows.  A row keeps 32
// columns of h, then the same 32 of l: one cache line for a step of 32 (with the planes apart, each step took half lines and
// two 2048 x 2048 products 142 us); fp32 rows take the same bytes.  Tiles come straight into LDS, a step or more ahead, chunks
// of 16 bytes swapped within a row so that the matrix instruction's reads meet all banks; neighbouring tiles go to one XCD,
// whose L2 then holds their rows.  A and P are symmetric: tiles at and above the diagonal only, stored twice.  Sizes are rounded up to whole tiles with
// zeros, which every product keeps.  All matrices of a size class share each launch: with large and small tiles in one call
// there are two chains of launches, one behind the other.
//
// Large matrices are bound by feeding the matrix instruction: P X of two 2048 x 2048 takes 118 us (880 TFLOP/s of fp16, the
// library's own fp16 product of that size 640), without its loads 78, without its matrix instructions 76.  Small ones are
// bound by the seventeen launches of five steps, 7 to 11 us each.
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>
#include <type_traits>
#include "../../include/mdmm_hip.h"

namespace mdmm {
namespace {

constexpr int NT = 256, SUMS = 256;
constexpr int FLUSH = 128;                        // columns of one sum inside the matrix instruction
constexpr float SX = 16384.0f, SP = 4096.0f;      // scales of X and A, and of P
typedef _Float16 half_t;
typedef half_t half4 __attribute__((ext_vector_type(4)));
typedef half_t half8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

// BM x BN tile of a product by WI x WJ waves, BK deep, ST buffers, OCC waves a SIMD wanted
template <int BM_, int BN_, int BK_, int ST_, int WI_, int WJ_, int OCC_> struct Cfg {
  static constexpr int BM = BM_, BN = BN_, BK = BK_, ST = ST_, WI = WI_, WJ = WJ_, OCC = OCC_;
  static constexpr int T = 64 * WI * WJ;                        // threads
  static constexpr int TI = BM / 32 / WI, TJ = BN / 32 / WJ;    // 32 x 32 pieces of a wave
  static constexpr int CPR = BK / 4;                            // chunks of a row: 8 halves each, h and l
  static constexpr int HALVES = (BM + BN) * BK * 2;             // of a buffer: A's rows, then B's
  static constexpr int LOADS = HALVES / 8 / T;                  // chunks a thread loads for a buffer
  static_assert(BM * CPR % T == 0 && BN * CPR % T == 0, "a load instruction of the workgroup stays in one operand");
};
// A matrix whose shorter side fits two small tiles is kept in fp32 and multiplied by the fp32 matrix instruction.  The fp16 one
// aligns the products of eight columns to the largest of them and drops what falls below its last bit: no matter beside the
// rounding of fp32 sums over hundreds of rows, but over a few of them the larger error (7 x 146: 2.1e-6 off against 0.7e-6
// in fp32 by the library, 65 x 1500: 1.6e-6 against 1.1e-6; here 0.9e-6 and 0.8e-6).  A wave's step takes 1024 cycles instead of
// 192, which such a matrix's few steps have room for.
constexpr int WHOLE = 128;
// (two workgroups a CU, four buffers each.  P X of two 256 x 4096: 13.6 us, with one of 128 KB 17)
typedef Cfg<64, 64, 32, 4, 2, 2, 2> Small;
static_assert(Small::TI * Small::TJ == 1, "fp32 rows: one piece a wave");
// (two workgroups a CU, two buffers each.  Measured on P X of two 2048 x 2048: 115 us; one workgroup with four buffers 127, one
// of 256 x 128 and 8 waves with three 126, 8 waves 125, tiles of 128 x 64 139, steps of 64 columns 126)
typedef Cfg<128, 128, 32, 2, 2, 2, 2> Large;

struct Item {               // one matrix's padded sizes and workspace
  half_t *xn, *xt[2], *gram, *poly;
  float* part;              // split sums of A
  double* sums;
  int32_t n, m, tall, splits;
};
enum { PACKS, GRAMS, POLYS, APPLIES, LISTS };
struct Items {
  Item it[MDMM_ORTHO_MAX];
  int32_t first[LISTS][MDMM_ORTHO_MAX + 1];       // first tile of each matrix in a launch (past the last one: INT32_MAX)
  int32_t n, reserved;
};
// |x (ca + cb x^2 + cc x^4)| at its extrema, value[i] at x^2 = at[i] (none: infinity), and q, with which |cb| + |cc| / 4 stays
// below P's 15.5: what a step needs to bound its result and to scale P
struct Range {
  float at[2], value[2];
  int32_t q;
};
// What the launches of one size class share (p.item: that class's matrices alone, in q.it's order).  The first launch takes it
// as its argument and leaves it in the workspace; the others read it there: arguments live in host memory, where each of the
// dependent loads that find a tile's matrix would wait for the bus
struct Call {
  mdmm_ortho_t p;
  Items q;
  Range r;
};
static_assert(sizeof(Call) <= 3968, "a launch's arguments");

// A launch finds a tile's matrix in one round trip to memory: each lane loads one matrix's entries, at the same time as the
// table of first tiles that tells which lane's are wanted (one after the other, 3 us more over the seventeen launches of eleven
// small matrices)
static_assert(MDMM_ORTHO_MAX <= 64, "a wave's lanes");
template <class T> struct Entries {
  unsigned v[sizeof(T) / 4];
  __device__ __forceinline__ Entries(const T* table) {
    const int lane = threadIdx.x & 63;
    __builtin_memcpy(v, table + (lane < MDMM_ORTHO_MAX ? lane : 0), sizeof(T));
  }
  __device__ __forceinline__ T of(int k) const {
    unsigned u[sizeof(T) / 4];
#pragma unroll
    for (int i = 0; i < (int)(sizeof(T) / 4); ++i) u[i] = __builtin_amdgcn_readlane(v[i], k);
    T t;
    __builtin_memcpy(&t, u, sizeof(T));
    return t;
  }
};
struct Found { int k, first; };          // the matrix that tile belongs to, its first tile
__device__ __forceinline__ Found find(const int32_t* first, int tile) {
  const int lane = threadIdx.x & 63, l = lane < MDMM_ORTHO_MAX ? lane : 0;
  const int begin = first[l], end = first[l + 1];
  const int k = (int)__popcll(__ballot(lane < MDMM_ORTHO_MAX && end <= tile));
  return {k, __builtin_amdgcn_readlane(begin, k)};
}

// the bound of every matrix's X, of even and odd steps: behind the call in the workspace
struct Bounds { float t[2][MDMM_ORTHO_MAX]; };
__device__ __forceinline__ Bounds* bounds(const Call* call) { return (Bounds*)(call + 1); }
// k of a bound t: 2^k t in [1/2, 1) below 1/2, up to 2^120 (X below 2^-120: as fp32 runs out)
__device__ __forceinline__ int shift_of(float t) {
  if (!(t > 0.0f && t < 0.5f)) return 0;
  const int k = -__builtin_amdgcn_frexp_expf(t);
  return k < 120 ? k : 120;
}
__device__ __forceinline__ float next_bound(const mdmm_ortho_t& p, const Range& r, float t) {
  const float u = t * t;
  float v = fabsf(t * (p.ca + u * (p.cb + u * p.cc)));
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (u > r.at[i] && r.value[i] > v) v = r.value[i];
  return v;
}

__device__ __forceinline__ void split(float x, half_t& h, half_t& l) {       // x: already scaled
  h = (half_t)x;
  l = (half_t)(x - (float)h);
}

// column c of a row of `cols` columns as pairs: h there, l 32 further
__device__ __forceinline__ int64_t at(int64_t row, int64_t cols, int64_t c) { return row * cols * 2 + (c >> 5) * 64 + (c & 31); }

// Elements of a matrix in either format: pairs, or (whole) fp32 in the same bytes of a row.  A row is 2 cols halves in both
__device__ __forceinline__ half_t* place(half_t* m, int64_t row, int64_t cols, int64_t c, bool whole) {
  return whole ? m + (row * cols + c) * 2 : m + at(row, cols, c);
}
__device__ __forceinline__ void put(half_t* d, float v, bool whole) {
  if (whole) {
    *(float*)d = v;
    return;
  }
  half_t h, l;
  split(v, h, l);
  d[0] = h;
  d[32] = l;
}
// four neighbours of a row (c a multiple of four)
__device__ __forceinline__ void put4(half_t* m, int64_t row, int64_t cols, int64_t c, const float* v, bool whole) {
  if (whole) {
    *(float4*)place(m, row, cols, c, true) = make_float4(v[0], v[1], v[2], v[3]);
    return;
  }
  half4 h4, l4;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    half_t h, l;
    split(v[e], h, l);
    h4[e] = h;
    l4[e] = l;
  }
  half_t* d = place(m, row, cols, c, false);
  *(half4*)d = h4;
  *(half4*)(d + 32) = l4;
}
struct Four { u32x2 a, b; };         // as loaded: two fp32 each, or four h and four l
__device__ __forceinline__ Four get4(const half_t* m, int64_t row, int64_t cols, int64_t c, bool whole) {
  const half_t* d = place((half_t*)m, row, cols, c, whole);
  return {*(const u32x2*)d, *(const u32x2*)(d + (whole ? 4 : 32))};
}
__device__ __forceinline__ float of4(const Four& f, int e, bool whole) {
  const half4 h = __builtin_bit_cast(half4, f.a), l = __builtin_bit_cast(half4, f.b);
  const unsigned x = e == 0 ? f.a[0] : e == 1 ? f.a[1] : e == 2 ? f.b[0] : f.b[1];
  return whole ? __builtin_bit_cast(float, x) : (float)h[e] + (float)l[e];
}

__device__ __forceinline__ float src_at(const mdmm_ortho_t& p, const mdmm_ortho_item_t& t, int64_t r, int64_t c) {
  const int64_t i = r * t.src_ld + c;
  return p.src_bf16 ? (float)((const __bf16*)t.src)[i] : ((const float*)t.src)[i];
}

// momentum, and the sum of squares in SUMS pieces (in 64 bits: an error of the norm is a scale of X and grows like one).
// LONG: eight loads of a thread on their way at once, where most elements lie in rows that have them (one 2048 x 2048 20 -> 9 us,
// 1000 x 4096 21 -> 9; four 1000 x 1000 8 -> 14, eleven small matrices 6.4 -> 10)
template <bool LONG> __global__ __launch_bounds__(NT) void ortho_sums_kernel(Call call, Call* keep) {
  const mdmm_ortho_t& p = call.p;
  const int k = blockIdx.y;
  const mdmm_ortho_item_t& t = p.item[k];
  if (blockIdx.x == 0 && k == 0) {
    const __attribute__((address_space(4))) unsigned* args = (const __attribute__((address_space(4))) unsigned*)__builtin_amdgcn_kernarg_segment_ptr();
    for (int i = threadIdx.x; i < (int)(sizeof(Call) / 4); i += NT) ((unsigned*)keep)[i] = args[i];
  }
  double s = 0.0;
  // a workgroup's rows, its threads over the columns (rows shorter than a workgroup: several of them at once)
  const int wide = t.cols < NT ? (t.cols < 16 ? 16 : t.cols < 64 ? 64 : NT) : NT, high = NT / wide;
  for (int64_t r = (int64_t)blockIdx.x * high + threadIdx.x / wide; r < t.rows; r += (int64_t)SUMS * high) {
    int64_t c = threadIdx.x % wide;
    auto take = [&](float v, float before, int64_t at) {
      if (t.mom) {
        const float mv = fmaf(p.momentum, before, v);
        t.mom[at] = mv;
        v = p.nesterov ? fmaf(p.momentum, mv, v) : mv;
      }
      s += (double)v * v;
    };
    if constexpr (LONG)
      for (; c + 7 * wide < t.cols; c += 8 * wide) {
        float v[8], before[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          v[e] = src_at(p, t, r, c + e * wide);
          before[e] = t.mom ? t.mom[r * t.cols + c + e * wide] : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) take(v[e], before[e], r * t.cols + c + e * wide);
      }
    for (; c < t.cols; c += wide) take(src_at(p, t, r, c), t.mom ? t.mom[r * t.cols + c] : 0.0f, r * t.cols + c);
  }
  __shared__ double part[NT / 64];
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) call.q.it[k].sums[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// X both ways, 64 x 64 elements a workgroup
__global__ __launch_bounds__(NT) void ortho_pack_kernel(const Call* __restrict__ call) {
  __shared__ float tile[64][65];
  const mdmm_ortho_t& p = call->p;
  const Items& q = call->q;
  const Entries<mdmm_ortho_item_t> ts(p.item);
  const Entries<Item> ws(q.it);
  const Found f = find(q.first[PACKS], blockIdx.x);
  const mdmm_ortho_item_t t = ts.of(f.k);
  const Item w = ws.of(f.k);
  const int me = blockIdx.x - f.first, across = (w.tall ? w.n : w.m) / 64;       // tiles of the source's rows
  const int64_t r0 = me / across * 64, c0 = me % across * 64;
  // the source's orientation: lying or standing plane pair
  half_t* same = w.tall ? w.xt[0] : w.xn;
  half_t* other = w.tall ? w.xn : w.xt[0];
  const int64_t ld_same = w.tall ? w.n : w.m, ld_other = w.tall ? w.m : w.n;
  float x[4096 / NT];                  // every load on its way before the first is used
#pragma unroll
  for (int u = 0; u < 4096 / NT; ++u) {
    const int i = threadIdx.x + u * NT;
    const int64_t r = r0 + i / 64, c = c0 + i % 64;
    x[u] = 0.0f;
    if (r < t.rows && c < t.cols) {
      x[u] = src_at(p, t, r, c);
      if (t.mom) {
        const float mv = t.mom[r * t.cols + c];
        x[u] = p.nesterov ? fmaf(p.momentum, mv, x[u]) : mv;
      }
    }
  }
  __shared__ double part[NT / 64];
  double s = w.sums[threadIdx.x];
  for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
  __syncthreads();
  s = (part[0] + part[1]) + (part[2] + part[3]);
  const double norm = sqrt(s), bound = norm / (norm + (double)p.eps);
  // 2^k SX / (|M| + eps) as inv 2^e: with eps 0 it need not fit fp32
  const double scale = (double)SX / (norm + (double)p.eps);
  const int e = __builtin_amdgcn_frexp_exp(scale);
  const float inv = (float)__builtin_amdgcn_frexp_mant(scale);
  const int exponent = e + shift_of((float)bound);
  if (me == 0 && threadIdx.x == 0) bounds(call)->t[0][f.k] = (float)bound;
  auto store = [&](auto as) {
    constexpr bool whole = decltype(as)::value;
#pragma unroll
    for (int u = 0; u < 4096 / NT; ++u) {
      const int i = threadIdx.x + u * NT;
      const float v = ldexpf(x[u], exponent) * inv;
      tile[i / 64][i % 64] = v;
      put(place(same, r0 + i / 64, ld_same, c0 + i % 64, whole), v, whole);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 4096; i += NT) put(place(other, c0 + i / 64, ld_other, r0 + i % 64, whole), tile[i % 64][i / 64], whole);
  };
  if (w.n <= WHOLE) store(std::true_type{});
  else store(std::false_type{});
}

enum { GRAM, POLY, APPLY, LAST };          // (LAST: an APPLY whose result goes to dst)

// four consecutive rows i of one column j of a symmetric matrix of n x n, both ways.  On the diagonal's tiles (i, j) and
// (j, i) are both computed, and may round differently: there the upper one is stored in both places, the lower one nowhere
__device__ __forceinline__ void put_sym(half_t* dst, int64_t n, int64_t i, int64_t j, const float* v, bool diagonal, bool whole) {
  half_t* down = place(dst, i, n, j, whole);
  if (!diagonal) put4(dst, j, n, i, v, whole);
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (!diagonal || i + e <= j) {
      put(down + 2 * e * n, v[e], whole);
      if (diagonal) put(place(dst, j, n, i + e, whole), v[e], whole);
    }
}

// tile t of those that reach the diagonal or lie above it, row by row; a row of tiles starts R tiles further right than the
// one above (R = BM / BN)
template <int R> __device__ __forceinline__ void triangle(int t, int across, int& ti, int& tj) {
  // rows before r hold f(r) = r across - R r (r - 1) / 2 tiles
  const float b = across + 0.5f * R;
  int r = (int)((b - sqrtf(fmaxf(b * b - 2.0f * R * t, 0.0f))) / R);
  const int rows = across / R;
  r = r < 0 ? 0 : r >= rows ? rows - 1 : r;
  while (r > 0 && r * across - R * r * (r - 1) / 2 > t) --r;
  while ((r + 1) * across - R * (r + 1) * r / 2 <= t) ++r;
  ti = r;
  tj = R * r + t - (r * across - R * r * (r - 1) / 2);
}

// all but the last N loads have landed, and this wave's reads of LDS are done
template <int N> __device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

template <class C> __host__ __device__ int tri(int n) {          // tiles at and above the diagonal
  constexpr int R = C::BM / C::BN;
  const int rows = n / C::BM;
  return rows * (n / C::BN) - R * rows * (rows - 1) / 2;
}

// tile `tile` of one matrix's product, in one of the formats
template <int MODE, class C, bool whole>
__device__ __forceinline__ void product(half_t (&lds)[C::ST * C::HALVES], const Call* __restrict__ call, const Item& w,
                                        const mdmm_ortho_item_t& t, int tile, int flip, float bound, float next) {
  constexpr bool PX = MODE == APPLY || MODE == LAST;
  const mdmm_ortho_t& p = call->p;
  const float ca = p.ca, cb = p.cb, cc = p.cc, decay = p.decay;
  const bool update = p.update, low = p.dst_bf16;
  const float lr = MODE == LAST && update ? (p.lr_dev ? *p.lr_dev : p.lr) : 0.0f;
  const int n = w.n, J = PX ? w.m : n;
  int ti, tj, slice = 0;
  if (PX) {
    ti = tile / (J / C::BN);
    tj = tile % (J / C::BN);
  } else {
    const int all = tri<C>(n);
    if (MODE == GRAM) { slice = tile / all; tile %= all; }
    triangle<C::BM / C::BN>(tile, n / C::BN, ti, tj);
  }
  const int i0 = ti * C::BM, j0 = tj * C::BN;
  const half_t* xt = flip ? w.xt[1] : w.xt[0];
  const half_t* a = MODE == GRAM ? w.xn : MODE == POLY ? w.gram : w.poly;
  const half_t* b = MODE == GRAM ? w.xn : MODE == POLY ? w.gram : xt;
  const int64_t K = MODE == GRAM ? w.m : n;               // columns of both
  const int steps_all = (int)(K / C::BK);
  const int per = MODE == GRAM ? (steps_all + w.splits - 1) / w.splits : steps_all;
  const int s0 = slice * per, nk = s0 + per < steps_all ? per : steps_all - s0;
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // this thread's chunks of a buffer: where they come from
  const half_t* from[C::LOADS];
#pragma unroll
  for (int c = 0; c < C::LOADS; ++c) {
    const bool in_b = c * C::T >= C::BM * C::CPR;
    const int ck = c * C::T - (in_b ? C::BM * C::CPR : 0) + tid;
    const int row = ck / C::CPR, ch = (ck % C::CPR) ^ (row / (16 / C::CPR) % C::CPR);
    from[c] = (in_b ? b + (j0 + row) * K * 2 : a + (i0 + row) * K * 2) + (int64_t)s0 * C::BK * 2 + ch * 8;
  }
  auto load = [&](int buf) {
#pragma unroll
    for (int c = 0; c < C::LOADS; ++c) {
      half_t* to = lds + buf * C::HALVES + (c * C::T + wave * 64) * 8;
      __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)from[c],
                                       (__attribute__((address_space(3))) void*)to, 16, 0, 0);
    }
  };
  auto advance = [&] {
#pragma unroll
    for (int c = 0; c < C::LOADS; ++c) from[c] += 2 * C::BK;
  };
  // what the result is joined with, on its way while the product runs (the small tile has the registers)
  constexpr bool EARLY = MODE != GRAM && C::TI * C::TJ == 1;
  const int wi = wave / C::WJ * 32 * C::TI, wj = wave % C::WJ * 32 * C::TJ;
  const half_t* beside = MODE == POLY ? w.gram : xt;
  Four early[EARLY ? 4 : 1];
  if constexpr (EARLY) {
#pragma unroll
    for (int g = 0; g < 4; ++g) early[g] = get4(beside, j0 + wj + (lane & 31), n, i0 + wi + 8 * g + 4 * (lane >> 5), whole);
  }
  f32x16 sum[C::TI][C::TJ] = {};
  // a piece's operands in registers: chunk of h, l's is 4 further (columns kk 16 + (lane / 32) 8 on, of each 32 columns' pair
  // of half lines)
  struct Part { half8 ah[C::TI], al[C::TI], bh[C::TJ], bl[C::TJ]; };
  auto read = [&](Part& f, int buf, int kk) {
    const half_t* A = lds + buf * C::HALVES;
    const half_t* B = A + 2 * C::BM * C::BK;
    const int c = kk / 2 * 8 + kk % 2 * 2 + (lane >> 5);
#pragma unroll
    for (int t = 0; t < C::TI; ++t) {
      const int row = wi + t * 32 + (lane & 31), z = row / (16 / C::CPR) % C::CPR;
      f.ah[t] = *(const half8*)(A + row * C::BK * 2 + (c ^ z) * 8);
      f.al[t] = *(const half8*)(A + row * C::BK * 2 + ((c + 4) ^ z) * 8);
    }
#pragma unroll
    for (int t = 0; t < C::TJ; ++t) {
      const int row = wj + t * 32 + (lane & 31), z = row / (16 / C::CPR) % C::CPR;
      f.bh[t] = *(const half8*)(B + row * C::BK * 2 + (c ^ z) * 8);
      f.bl[t] = *(const half8*)(B + row * C::BK * 2 + ((c + 4) ^ z) * 8);
    }
  };
  f32x16 acc[C::TI][C::TJ];
  auto multiply = [&](const Part& f) {
    if constexpr (whole) {
      // the reads hold columns 4 c .. 4 c + 3 of both operands; an instruction takes one from each half of the wave
      const f32x4 a0 = __builtin_bit_cast(f32x4, f.ah[0]), a1 = __builtin_bit_cast(f32x4, f.al[0]);
      const f32x4 b0 = __builtin_bit_cast(f32x4, f.bh[0]), b1 = __builtin_bit_cast(f32x4, f.bl[0]);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a0[e], b0[e], acc[0][0], 0, 0, 0);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x2f32(a1[e], b1[e], acc[0][0], 0, 0, 0);
      return;
    }
    // (the three products of a piece apart: none waits for the one before)
#pragma unroll
    for (int x = 0; x < C::TI; ++x)
#pragma unroll
      for (int y = 0; y < C::TJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[x], f.bl[y], acc[x][y], 0, 0, 0);
#pragma unroll
    for (int x = 0; x < C::TI; ++x)
#pragma unroll
      for (int y = 0; y < C::TJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.al[x], f.bh[y], acc[x][y], 0, 0, 0);
#pragma unroll
    for (int x = 0; x < C::TI; ++x)
#pragma unroll
      for (int y = 0; y < C::TJ; ++y) acc[x][y] = __builtin_amdgcn_mfma_f32_32x32x16_f16(f.ah[x], f.bh[y], acc[x][y], 0, 0, 0);
  };
  // FLUSH columns at a time, the pieces added by the vector unit: the matrix instruction does not round its sum to nearest,
  // and over a diagonal of A (1662 positive terms) that came to 4e-6 (6e-7 with pieces)
  constexpr int RUN = FLUSH / C::BK;
  if constexpr (C::TI * C::TJ == 1) {
    // a wave alone on its SIMD, so a step's operands are read from LDS under the products of the step before.  At the barrier
    // of step s every wave holds step s in registers: its buffer takes step s + ST
    static_assert(C::BK == 32 && RUN % 2 == 0, "two pieces a step, two steps' registers in turn");
    Part r[2][2];
#pragma unroll
    for (int s = 0; s < C::ST; ++s)
      if (s < nk) load(s), advance();
    if (C::ST <= nk) wait_loads<(C::ST - 1) * C::LOADS>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    read(r[0][0], 0, 0);
    read(r[0][1], 0, 1);
    for (int from_s = 0; from_s < nk; from_s += RUN) {
      acc[0][0] = f32x16{};
#pragma unroll
      for (int u = 0; u < RUN; ++u) {
        const int s = from_s + u;
        if (s >= nk) break;
        if (s + 1 < nk) {
          // buffer s + 1 has landed when no more than the loads of the buffers behind it are in flight
          if (s + C::ST - 1 < nk) wait_loads<(C::ST - 2) * C::LOADS>();
          else wait_loads<0>();
          __builtin_amdgcn_s_barrier();
          asm volatile("" ::: "memory");
          if (s + C::ST < nk) load(s % C::ST);
          advance();
          read(r[(u + 1) & 1][0], (s + 1) % C::ST, 0);
          read(r[(u + 1) & 1][1], (s + 1) % C::ST, 1);
        }
        multiply(r[u & 1][0]);
        multiply(r[u & 1][1]);
        if (whole && u + 1 < RUN) {              // (a sum of 32 columns)
          sum[0][0] += acc[0][0];
          acc[0][0] = f32x16{};
        }
      }
      sum[0][0] += acc[0][0];
    }
  } else {
#pragma unroll
    for (int s = 0; s < C::ST - 1; ++s)
      if (s < nk) load(s), advance();
    for (int from_s = 0; from_s < nk; from_s += RUN) {
      const int to_s = from_s + RUN < nk ? from_s + RUN : nk;
#pragma unroll
      for (int x = 0; x < C::TI; ++x)
#pragma unroll
        for (int y = 0; y < C::TJ; ++y) acc[x][y] = f32x16{};
      for (int s = from_s; s < to_s; ++s) {
        // buffer s has landed when no more than the loads of the buffers behind it are in flight
        if (s + C::ST - 2 < nk) wait_loads<(C::ST - 2) * C::LOADS>();
        else wait_loads<0>();
        __builtin_amdgcn_s_barrier();             // (every wave's share; and all are done with the buffer that is filled next)
        asm volatile("" ::: "memory");
        if (s + C::ST - 1 < nk) load((s + C::ST - 1) % C::ST);
        advance();
#pragma unroll
        for (int kk = 0; kk < C::BK / 16; ++kk) {
          Part f;
          read(f, s % C::ST, kk);
          multiply(f);
        }
      }
#pragma unroll
      for (int x = 0; x < C::TI; ++x)
#pragma unroll
        for (int y = 0; y < C::TJ; ++y) sum[x][y] += acc[x][y];
    }
  }
  // v: the result in its planes' scale
  const int64_t nn = (int64_t)n * n, m = w.m;
  const int k = shift_of(bound), up = MODE == APPLY ? shift_of(next) - k : 0, q = k ? call->r.q : 0;
  const float pa = ldexpf(cc * (SP / SX / SX), -2 * k - q), pb = ldexpf(cb * (SP / SX), -q);          // of POLY
  const float xa = ldexpf(ca, up), xb = ldexpf(1.0f / SP, up - 2 * k + q), out = ldexpf(1.0f / SX, -k);      // of P X
#pragma unroll
  for (int x = 0; x < C::TI; ++x)
#pragma unroll
    for (int y = 0; y < C::TJ; ++y)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        // four consecutive rows of one column
        const int64_t i = i0 + wi + x * 32 + 8 * g + 4 * (lane >> 5), j = j0 + wj + y * 32 + (lane & 31);
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = sum[x][y][4 * g + e];
        Four with;
        if constexpr (EARLY) with = early[g];
        else if constexpr (MODE != GRAM) with = get4(beside, j, n, i, whole);
        if (MODE == GRAM) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= 1.0f / SX;
          if (w.splits == 1) put_sym(w.gram, n, i, j, v, j0 < i0 + C::BM, whole);
          else *(float4*)(w.part + slice * nn + j * n + i) = make_float4(v[0], v[1], v[2], v[3]);
        }
        if (MODE == POLY) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(pa, v[e], pb * of4(with, e, whole));
          put_sym(w.poly, n, i, j, v, j0 < i0 + C::BM, whole);
        }
        if (PX) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = fmaf(xa, of4(with, e, whole), v[e] * xb);
        }
        if (MODE == APPLY) {
          half_t* down = place(w.xn, i, m, j, whole);
#pragma unroll
          for (int e = 0; e < 4; ++e) put(down + 2 * e * m, v[e], whole);
          put4(flip ? w.xt[0] : w.xt[1], j, n, i, v, whole);
        }
        if (MODE == LAST) {
          const int64_t r = w.tall ? j : i, c = w.tall ? i : j, step = w.tall ? 1 : t.dst_ld;
          const int64_t end = w.tall ? (r < t.rows ? t.cols - c : 0) : (c < t.cols ? t.rows - r : 0);      // of the four
          const int64_t o = r * t.dst_ld + c;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float u = v[e] * out;
            if (e >= end) continue;
            if (update) {
              float* d = (float*)t.dst + o + e * step;
              *d = fmaf(-lr * t.gain, u, (1.0f - lr * decay) * *d);
            } else if (low) ((__bf16*)t.dst)[o + e * step] = (__bf16)u;
            else ((float*)t.dst)[o + e * step] = u;
          }
        }
      }
}

template <int MODE, class C>
__global__ __launch_bounds__(C::T, C::OCC) void ortho_product_kernel(const Call* __restrict__ call, int flip) {
  __shared__ __align__(16) half_t lds[C::ST * C::HALVES];
  constexpr int LIST = MODE == GRAM ? GRAMS : MODE == POLY ? POLYS : APPLIES;
  const Items& q = call->q;
  // consecutive workgroups go round the 8 XCDs: each XCD takes a run of consecutive tiles instead
  const int total = gridDim.x, xcd = blockIdx.x & 7, each = total >> 3, more = total & 7;
  const int me = xcd * each + (xcd < more ? xcd : more) + (blockIdx.x >> 3);
  const Entries<mdmm_ortho_item_t> ts(call->p.item);
  const Entries<Item> ws(q.it);
  const int lane = threadIdx.x & 63, l = lane < MDMM_ORTHO_MAX ? lane : 0;
  const Bounds* t_of = bounds(call);
  const float t_now = MODE == GRAM ? 0.0f : t_of->t[flip][l], t_next = MODE == APPLY ? t_of->t[flip ^ 1][l] : 0.0f;
  const Found f = find(q.first[LIST], me);
  const Item w = ws.of(f.k);
  auto of_k = [&](float v) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), f.k)); };
  const float bound = of_k(t_now), next = of_k(t_next);
  if (MODE == POLY && me == f.first && threadIdx.x == 0) bounds(call)->t[flip ^ 1][f.k] = next_bound(call->p, call->r, bound);
  mdmm_ortho_item_t t = {};
  if (MODE == LAST) t = ts.of(f.k);
  if constexpr (C::TI * C::TJ == 1)
    if (w.n <= WHOLE) {
      product<MODE, C, true>(lds, call, w, t, me - f.first, flip, bound, next);
      return;
    }
  product<MODE, C, false>(lds, call, w, t, me - f.first, flip, bound, next);
}

// the slices of A added up (each keeps the tiles at and above the diagonal, column by column)
template <int BM, int BN> __global__ __launch_bounds__(NT) void ortho_fold_kernel(const Call* __restrict__ call) {
  const Item w = call->q.it[blockIdx.y];
  if (w.splits == 1) return;
  const int64_t n = w.n, nn = n * n;
  auto join = [&](auto as) {
    constexpr bool whole = decltype(as)::value;
    for (int64_t e = ((int64_t)blockIdx.x * NT + threadIdx.x) * 4; e < nn; e += (int64_t)gridDim.x * NT * 4) {
      const int64_t j = e / n, i = e % n;
      const int64_t i0 = i / BM * BM, j0 = j / BN * BN;
      if (j0 < i0) continue;
      float4 v = *(const float4*)(w.part + e);
      for (int s = 1; s < w.splits; ++s) {
        const float4 x = *(const float4*)(w.part + s * nn + e);
        v.x += x.x; v.y += x.y; v.z += x.z; v.w += x.w;
      }
      const float f[4] = {v.x, v.y, v.z, v.w};
      put_sym(w.gram, n, i, j, f, j0 < i0 + BM, whole);
    }
  };
  if (n <= WHOLE) join(std::true_type{});
  else join(std::false_type{});
}

__global__ __launch_bounds__(NT) void ortho_copy_kernel(const Call* __restrict__ call) {       // steps = 0: X itself
  const mdmm_ortho_t& p = call->p;
  const Items& q = call->q;
  const mdmm_ortho_item_t& t = p.item[blockIdx.y];
  const Item& w = q.it[blockIdx.y];
  const int64_t total = (int64_t)t.rows * t.cols;
  for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < total; i += (int64_t)gridDim.x * NT) {
    const int64_t r = i / t.cols, c = i % t.cols;
    const bool whole = w.n <= WHOLE;
    const half_t* x = place(w.xn, w.tall ? c : r, w.m, w.tall ? r : c, whole);
    const float v = (whole ? *(const float*)x : (float)x[0] + (float)x[32]) * ldexpf(1.0f / SX, -shift_of(bounds(call)->t[0][blockIdx.y]));
    const int64_t to = r * t.dst_ld + c;
    if (p.update) {
      float* d = (float*)t.dst + to;
      const float lr = p.lr_dev ? *p.lr_dev : p.lr;
      *d = fmaf(-lr * t.gain, v, (1.0f - lr * p.decay) * *d);
    } else if (p.dst_bf16) ((__bf16*)t.dst)[to] = (__bf16)v;
    else ((float*)t.dst)[to] = v;
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

constexpr int64_t up(int64_t v, int64_t to) { return (v + to - 1) / to * to; }
constexpr int64_t KEPT = up(sizeof(Call) + sizeof(Bounds), 256);         // of a size class in the workspace

// A call's larger matrices (more than 384 rows) can take 128 x 128 tiles in P X: they halve what a product loads, but both
// sides are then padded to 128 for all three products, and a CU's two places have to be filled.  Five steps with them and with
// small tiles:
//   full rounds of the 256 CUs: one 2048 x 2048 (256 tiles) 902 us and 957, two (512) 1462 and 1687, 1000 x 4096 (256) 479 and
//   514, sixteen 1024 x 1024 (1024) 1667 and 1806; half a round more: two 768 x 4096 (384) 528 and 552, eleven 768 x 768 (396)
//   620 and 637, ten 1024 x 1024 (640) 1146 and 1130; less of it: eleven 640 x 640 (275) 495 and 463, two 1500 x 1500 (288) 831
//   and 798, nine 1024 x 1024 (576) 1064 and 1022
//   padding: four 640 x 2060 (1.03 of the small tiles' work) 483 and 492, two 900 x 2001 (1.15) 472 and 434, four 520 x 2060
//   (1.28) 469 and 413, eleven 520 x 520 (1.37) 485 and 333, sixteen 390 x 390 (1.49) 368 and 290
// So they are taken by matrices that they pad by no more than a twentieth, where those have a round of tiles and the last
// round is at least half full.  A and P take small ones always (two of 2048 x 2048 on large ones 1553, one 971).
int64_t large_tiles(const mdmm_ortho_item_t& t) {
  const int64_t n = t.rows < t.cols ? t.rows : t.cols, m = t.rows < t.cols ? t.cols : t.rows;
  if (n <= 384) return 0;
  auto work = [&](int64_t pad) { return up(n, pad) * up(n, pad) * (3 * up(m, pad) + up(n, pad)); };
  if (20 * work(Large::BM) > 21 * work(Small::BM)) return 0;
  return up(n, Large::BM) / Large::BM * (up(m, Large::BN) / Large::BN);
}
bool fills(int64_t tiles) { return tiles >= 256 && (tiles - 1) % 256 >= 127; }

// the workspace: fills both size classes' lists (base NULL: sizes only), returns the bytes used
int64_t lay_out(const mdmm_ortho_t* a, Items (&q)[2], mdmm_ortho_item_t (*items)[MDMM_ORTHO_MAX] = nullptr) {
  char* base = (char*)a->ws;
  int64_t off = up(2 * KEPT, 4096);         // (two 256 x 4096: 185 us, at 2 KEPT 188)
  auto take = [&](int64_t bytes) { char* p = base + off; off += up(bytes, 256); return p; };
  q[0].n = q[1].n = 0;
  int64_t total = 0;
  for (int i = 0; i < a->n; ++i) total += large_tiles(a->item[i]);
  for (int i = 0; i < a->n; ++i) {
    const mdmm_ortho_item_t& t = a->item[i];
    const bool big = fills(total) && large_tiles(t) > 0;
    Items& l = q[big];
    if (items) items[big][l.n] = t;
    Item& w = l.it[l.n++];
    const int pad = big ? Large::BM : Small::BM;
    w.tall = t.rows > t.cols;
    w.n = (int32_t)up(w.tall ? t.cols : t.rows, pad);
    w.m = (int32_t)up(w.tall ? t.rows : t.cols, pad);
    // slices of A: from 2048 columns on, while the tiles leave CUs idle, of 512 columns at least (joining them is a launch
    // more, 4 us with its gap, which is what 768 columns take in one piece)
    const int64_t tiles = tri<Small>(w.n);
    int64_t splits = w.m >= 2048 ? (128 / tiles < w.m / 512 ? 128 / tiles : w.m / 512) : 1;
    if (splits < 1) splits = 1;
    const int64_t steps = w.m / Small::BK, per = (steps + splits - 1) / splits;
    w.splits = (int32_t)((steps + per - 1) / per);
    const int64_t x = (int64_t)w.n * w.m, g = (int64_t)w.n * w.n;
    w.xn = (half_t*)take(4 * x);
    w.xt[0] = (half_t*)take(4 * x);
    w.xt[1] = (half_t*)take(4 * x);
    w.gram = (half_t*)take(4 * g);
    w.poly = (half_t*)take(4 * g);
    w.part = (float*)take(w.splits > 1 ? 4 * g * w.splits : 0);
    w.sums = (double*)take(8 * SUMS);
  }
  return off;
}

template <class F> int tiles(Items& q, int list, F count) {
  int64_t total = 0;
  for (int i = 0; i < q.n; ++i) {
    q.first[list][i] = (int32_t)total;
    total += count(q.it[i]);
  }
  for (int i = q.n; i <= MDMM_ORTHO_MAX; ++i) q.first[list][i] = i == q.n ? (int32_t)total : INT32_MAX;
  return (int)total;
}

Range range_of(const mdmm_ortho_t* a) {
  Range r = {{INFINITY, INFINITY}, {0.0f, 0.0f}, 0};
  const double ca = a->ca, cb = a->cb, cc = a->cc;
  double at[2] = {INFINITY, INFINITY};
  if (cc != 0.0) {
    const double root = 9.0 * cb * cb - 20.0 * ca * cc;
    if (root >= 0.0)
      for (int i = 0; i < 2; ++i) at[i] = (-3.0 * cb + (i ? 1.0 : -1.0) * sqrt(root)) / (10.0 * cc);
  } else if (cb != 0.0) at[0] = -ca / (3.0 * cb);
  for (int i = 0; i < 2; ++i)
    if (at[i] > 0.0 && at[i] < 16.0) {
      r.at[i] = (float)at[i];
      r.value[i] = (float)(sqrt(at[i]) * fabs(ca + at[i] * (cb + at[i] * cc)));
    }
  const double top = (fabs(cb) + fabs(cc) / 4.0) / 15.5;
  if (top > 1.0 && top < 1e30) r.q = ilogb(top) + 1;
  return r;
}

// C: the tile of A and P, D: that of P X
template <class C, class D> void launch(const mdmm_ortho_t* a, const Items& items, const mdmm_ortho_item_t* mats, Call* keep, hipStream_t s) {
  if (!items.n) return;
  Call c;
  c.p = *a;
  for (int i = 0; i < MDMM_ORTHO_MAX; ++i) c.p.item[i] = mats[i];
  c.q = items;
  c.r = range_of(a);
  Items& q = c.q;
  const int packs = tiles(q, PACKS, [](const Item& w) { return (int64_t)(w.n / 64) * (w.m / 64); });
  const int gram = tiles(q, GRAMS, [](const Item& w) { return (int64_t)tri<C>(w.n) * w.splits; });
  const int poly = tiles(q, POLYS, [](const Item& w) { return (int64_t)tri<C>(w.n); });
  const int apply = tiles(q, APPLIES, [](const Item& w) { return (int64_t)(w.n / D::BM) * (w.m / D::BN); });
  int64_t fold = 0;
  for (int i = 0; i < q.n; ++i)
    if (q.it[i].splits > 1 && (int64_t)q.it[i].n * q.it[i].n > fold) fold = (int64_t)q.it[i].n * q.it[i].n;
  int64_t all = 0, wide = 0;               // elements, those in rows of eight workgroups' widths
  for (int i = 0; i < q.n; ++i) {
    const int64_t size = (int64_t)mats[i].rows * mats[i].cols;
    all += size;
    if (mats[i].cols >= 8 * NT) wide += size;
  }
  if (2 * wide > all) hipLaunchKernelGGL(ortho_sums_kernel<true>, dim3(SUMS, q.n), dim3(NT), 0, s, c, keep);
  else hipLaunchKernelGGL(ortho_sums_kernel<false>, dim3(SUMS, q.n), dim3(NT), 0, s, c, keep);
  hipLaunchKernelGGL(ortho_pack_kernel, dim3(packs), dim3(NT), 0, s, keep);
  if (a->steps == 0) hipLaunchKernelGGL(ortho_copy_kernel, dim3(256, q.n), dim3(NT), 0, s, keep);
  for (int k = 0; k < a->steps; ++k) {
    hipLaunchKernelGGL((ortho_product_kernel<GRAM, C>), dim3(gram), dim3(C::T), 0, s, keep, k & 1);
    if (fold) hipLaunchKernelGGL((ortho_fold_kernel<C::BM, C::BN>), dim3((unsigned)(fold / (4 * NT)), q.n), dim3(NT), 0, s, keep);
    hipLaunchKernelGGL((ortho_product_kernel<POLY, C>), dim3(poly), dim3(C::T), 0, s, keep, k & 1);
    if (k + 1 < a->steps) hipLaunchKernelGGL((ortho_product_kernel<APPLY, D>), dim3(apply), dim3(D::T), 0, s, keep, k & 1);
    else hipLaunchKernelGGL((ortho_product_kernel<LAST, D>), dim3(apply), dim3(D::T), 0, s, keep, k & 1);
  }
}

}  // namespace
}  // namespace mdmm

using namespace mdmm;

extern "C" int64_t mdmm_ortho_ws(const mdmm_ortho_t* a) {
  if (const int rc = check(a)) return rc;
  Items q[2];
  return lay_out(a, q);
}

extern "C" int mdmm_ortho(const mdmm_ortho_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (a->n == 0) return 0;
  if (!a->ws || ((uintptr_t)a->ws & 255)) return a->ws ? MDMM_E_ALIGN : MDMM_E_ARG;
  for (int i = 0; i < a->n; ++i)
    if (!a->item[i].src || !a->item[i].dst) return MDMM_E_ARG;
  Items q[2] = {};
  mdmm_ortho_item_t mats[2][MDMM_ORTHO_MAX] = {};
  lay_out(a, q, mats);
  launch<Small, Small>(a, q[0], mats[0], (Call*)a->ws, (hipStream_t)stream);
  launch<Small, Large>(a, q[1], mats[1], (Call*)((char*)a->ws + KEPT), (hipStream_t)stream);
  return (int)hipGetLastError();
}
