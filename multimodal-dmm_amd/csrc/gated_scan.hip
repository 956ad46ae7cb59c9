// Gated linear recurrence over time: h_t = a_t h_{t-1} + (1 - a_t) c_t with a_t = sigmoid(f_t), per channel; a step whose
// mask byte is 0 leaves h as it is (a = 1, nothing added).  Backward: G_t = g_t + a_{t+1} G_{t+1} (g = the gradient of h_t),
// dc = G (1 - a), df = G (h_{t-1} - c) a (1 - a), dh0 = a_0 G_0.
#include "gated.h"

namespace mdmm {
namespace {

constexpr int NT = 256;

// one thread per channel, one step after the other
template <typename IO, typename HO>
__global__ __launch_bounds__(NT) void scan_fwd_kernel(mdmm_gated_scan_t p) {
  const int64_t q = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (q >= (int64_t)p.B * p.H) return;
  const int64_t b = q / p.H, j = q % p.H;
  float h = p.h0 ? p.h0[b * p.h0_sb + j] : 0.0f;
  for (int i = 0; i < p.T; ++i) {
    const int64_t t = p.reverse ? p.T - 1 - i : i;
    if (p.states) p.states[t * p.B * p.H + q] = h;
    const IO* row = (const IO*)p.gates + t * p.gates_st + b * p.gates_sb + j;
    if (!p.mask || p.mask[t * p.mask_st + b * p.mask_sb]) {
      const Gate g(load1(row));
      h = g.a * h + g.k * load1(row + p.H);
    }
    if (p.h) store1((HO*)p.h + t * p.B * p.H + q, h);
  }
  if (p.h_last) p.h_last[q] = h;
}

template <typename IO, typename HO>
__global__ __launch_bounds__(NT) void scan_bwd_kernel(mdmm_gated_scan_t p) {
  const int64_t q = (int64_t)blockIdx.x * NT + threadIdx.x;
  if (q >= (int64_t)p.B * p.H) return;
  const int64_t b = q / p.H, j = q % p.H;
  float d = p.g_last ? p.g_last[q] : 0.0f;       // a_{t+1} G_{t+1}
  for (int i = p.T - 1; i >= 0; --i) {
    const int64_t t = p.reverse ? p.T - 1 - i : i;
    const IO* row = (const IO*)p.gates + t * p.gates_st + b * p.gates_sb + j;
    IO* out = (IO*)p.g_gates + t * p.g_gates_st + b * p.g_gates_sb + j;
    float df = 0.0f, dc = 0.0f;
    if (p.g_h) d += load1((const HO*)p.g_h + t * p.B * p.H + q);
    if (!p.mask || p.mask[t * p.mask_st + b * p.mask_sb]) {
      const Gate g(load1(row));
      dc = d * g.k;
      df = dc * g.a * (p.states[t * p.B * p.H + q] - load1(row + p.H));
      d *= g.a;
    }
    store1(out, df);
    store1(out + p.H, dc);
  }
  if (p.g_h0) p.g_h0[q] = d;
}

int check(const mdmm_gated_scan_t* a) {
  if (!a || a->T < 0 || a->B < 0 || a->H < 0) return MDMM_E_ARG;
  if (a->T > 0 && a->B > 0 && a->H > 0 && !a->gates) return MDMM_E_ARG;
  return 0;
}

}  // namespace
}  // namespace mdmm

using namespace mdmm;

extern "C" int64_t mdmm_gated_scan_states(const mdmm_gated_scan_t* a) {
  return check(a) ? -1 : (int64_t)a->T * a->B * a->H;
}

extern "C" int64_t mdmm_gated_scan_ws(const mdmm_gated_scan_t* a, int) { return check(a) ? -1 : 0; }

#define SCAN_LAUNCH(kern)                                                                                   \
  do {                                                                                                      \
    const int64_t wgs = ((int64_t)a->B * a->H + NT - 1) / NT;                                               \
    if (!a->gates_bf16) hipLaunchKernelGGL((kern<float, float>), dim3((unsigned)wgs), dim3(NT), 0, (hipStream_t)stream, *a); \
    else if (a->h_bf16) hipLaunchKernelGGL((kern<__bf16, __bf16>), dim3((unsigned)wgs), dim3(NT), 0, (hipStream_t)stream, *a); \
    else hipLaunchKernelGGL((kern<__bf16, float>), dim3((unsigned)wgs), dim3(NT), 0, (hipStream_t)stream, *a); \
    return (int)hipGetLastError();                                                                          \
  } while (0)

extern "C" int mdmm_gated_scan_fwd(const mdmm_gated_scan_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (!a->gates_bf16 && a->h_bf16) return MDMM_E_ARG;
  if (a->T == 0 || a->B == 0 || a->H == 0) return 0;
  SCAN_LAUNCH(scan_fwd_kernel);
}

extern "C" int mdmm_gated_scan_bwd(const mdmm_gated_scan_t* a, void* stream) {
  const int rc = check(a);
  if (rc) return rc;
  if (!a->gates_bf16 && a->h_bf16) return MDMM_E_ARG;
  if (a->T == 0 || a->B == 0 || a->H == 0) return 0;
  if (!a->g_gates || !a->states) return MDMM_E_ARG;
  SCAN_LAUNCH(scan_bwd_kernel);
}
