// The gated feed-forward product and its gradients.
//
//   g = x Wg^T + bg,  u = x Wu^T + bu,  h = a(g) u            x [M, K], W [F, K], h [M, F]
//   dg = dh u a'(g),  du = dh a(g),
//   dx = dg Wg + du Wu,  dWg = dg^T x,  dWu = du^T x,  dbg, dbu = column sums of dg, du
//
// The forward that a gradient follows keeps g and u in float32 (they are what
// the accumulators hold): rounded to the 16-bit type, they would put two more
// roundings into every gradient, which nearly doubles its error (1.8 instead
// of 1.4 times one rounding). dg and du are rounded to the inputs' type once,
// because the tensor cores multiply 16-bit operands.
#include <type_traits>

#include "common.cuh"
#include "gated.cuh"
#include "kernels.h"

namespace gfx {
namespace gated {

// ---------------------------------------------------------------------------
// dg, du (one row of dgu [M, 2F]: dg then du) and, per block of rows, their column sums
// ---------------------------------------------------------------------------
// Memory-bound: float32 g and u and 16-bit dh read, dg and du written, 14 bytes an element; 128 us for 4608 x 12288
// (792 MB), 6.2 TB/s.
constexpr int kRowsPerBlock = 64;

template <typename T, int kAct>
__global__ void __launch_bounds__(256) gate_grad_kernel(const T* dh, long long ldh, const float* save, T* dgu,
                                                        float* partial, int* counters, int M, int F) {
  pdl_trigger();
  pdl_wait();
  // the products that follow want their counters at zero
  if (blockIdx.x == 0 && blockIdx.y == 0)
    for (int i = threadIdx.x; i < (int)(kGatedCounterBytes / sizeof(int)); i += 256) counters[i] = 0;
  // a warp: 128 columns (4 a lane) of every eighth row
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int f = blockIdx.y * 128 + lane * 4;
  const long long r0 = (long long)blockIdx.x * kRowsPerBlock;
  float sum[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) sum[j] = 0.0f;
  if (f < F) {
    for (long long r = r0 + warp; r < r0 + kRowsPerBlock && r < M; r += 8) {
      const float4 g = *reinterpret_cast<const float4*>(save + r * F + f);
      const float4 u = *reinterpret_cast<const float4*>(save + (M + r) * F + f);
      const uint2 w = *reinterpret_cast<const uint2*>(dh + r * ldh + f);
      const T* d = reinterpret_cast<const T*>(&w);
      const float gv[4] = {g.x, g.y, g.z, g.w}, uv[4] = {u.x, u.y, u.z, u.w};
      uint2 og, ou;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float a, da;
        activation_grad<kAct>(gv[j], a, da);
        const float dv = to_f32<T>(d[j]), dg = dv * uv[j] * da, du = dv * a;
        sum[j] += dg;
        sum[4 + j] += du;
        reinterpret_cast<T*>(&og)[j] = from_f32<T>(dg);
        reinterpret_cast<T*>(&ou)[j] = from_f32<T>(du);
      }
      *reinterpret_cast<uint2*>(dgu + r * 2 * F + f) = og;
      *reinterpret_cast<uint2*>(dgu + r * 2 * F + F + f) = ou;
    }
  }
  if (partial == nullptr) return;
  __shared__ float s[8][8][32];
#pragma unroll
  for (int j = 0; j < 8; ++j) s[warp][j][lane] = sum[j];
  __syncthreads();
  // thread (j, l): column j & 3 of lane l's four, of dg (j < 4) or du
  const int j = threadIdx.x >> 5, c = blockIdx.y * 128 + lane * 4 + (j & 3);
  if (c >= F) return;
  float v = 0.0f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += s[k][j][lane];
  partial[((long long)blockIdx.x * 2 + (j >> 2)) * F + c] = v;
}

// db = the sums over blocks of rows, in order
template <typename T>
__global__ void __launch_bounds__(256) bias_grad_kernel(const float* partial, int blocks, int F, T* dbg, T* dbu) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  pdl_trigger();
  pdl_wait();
  if (c >= 2 * F) return;
  T* out = c < F ? dbg : dbu;
  if (out == nullptr) return;
  float v = 0.0f;
#pragma unroll 8
  for (int b = 0; b < blocks; ++b) v += partial[(long long)b * 2 * F + c];
  out[c < F ? c : c - F] = from_f32<T>(v);
}

}  // namespace gated

static int row_blocks(int M) { return (M + gated::kRowsPerBlock - 1) / gated::kRowsPerBlock; }

size_t gated_forward_workspace(int M, int K, int F, int sms) {
  return M <= kGatedFewTokens ? 0 : gated_forward_tc_workspace(M, K, F, sms);
}

int launch_gated_forward(const GatedArgs& a, int dtype, int act, void* h, float* save, void* workspace,
                         cudaStream_t st, int sms) {
  // Up to 128 tokens (the few-token form's TMEM holds no more) that form is the faster one everywhere measured: 128
  // tokens at 3072 x 12288 take 43 us there and 45 in 256-row tiles, at 2048 x 5632 20 and 21, one token 29 and 54.
  if (a.M <= kGatedFewTokens) return launch_gated_forward_few(a, dtype, act, h, save, st, sms);
  return launch_gated_forward_tc(a, dtype, act, h, save, workspace, st, sms);
}

// The backward's workspace: counters and sums of the products, dg and du, the column sums.
static size_t dgu_offset(const GatedArgs& a, int sms) {
  return align_up(gated_backward_tc_workspace(a.M, a.K, a.F, sms), 256);
}
static size_t sums_offset(const GatedArgs& a, int sms) {
  return dgu_offset(a, sms) + align_up((size_t)a.M * 2 * a.F * 2, 256);
}

size_t gated_backward_workspace(int M, int K, int F, int sms) {
  GatedArgs a{};
  a.M = M, a.K = K, a.F = F;
  return sums_offset(a, sms) + (size_t)row_blocks(M) * 2 * F * sizeof(float);
}

template <typename T>
static int gated_backward_t(const GatedArgs& a, int act, const void* dh, long long ldh, const float* save,
                            const GatedGrads& d, void* workspace, cudaStream_t st, int sms) {
  char* ws = static_cast<char*>(workspace);
  T* dgu = reinterpret_cast<T*>(ws + dgu_offset(a, sms));
  float* partial = reinterpret_cast<float*>(ws + sums_offset(a, sms));
  const int blocks = row_blocks(a.M);
  const bool bias = d.b_gate || d.b_up;
  const dim3 grid(blocks, (a.F + 127) / 128);
  auto go = [&](auto kern) {
    launch_overlapped(kern, grid, 256, st, (const T*)dh, ldh, save, dgu, bias ? partial : nullptr,
                      static_cast<int*>(workspace), a.M, a.F);
  };
  if (act == gated::kSilu)
    go(gated::gate_grad_kernel<T, gated::kSilu>);
  else if (act == gated::kGelu)
    go(gated::gate_grad_kernel<T, gated::kGelu>);
  else
    go(gated::gate_grad_kernel<T, gated::kGeluTanh>);
  int rc = check_launch("gate_grad_kernel");
  if (rc) return rc;
  if (bias) {
    launch_overlapped(gated::bias_grad_kernel<T>, dim3((2 * a.F + 255) / 256), 256, st, partial, blocks, a.F,
                      (T*)d.b_gate, (T*)d.b_up);
    if ((rc = check_launch("bias_grad_kernel"))) return rc;
  }
  constexpr int kDtype = std::is_same<T, __half>::value ? GFX_DTYPE_F16 : GFX_DTYPE_BF16;
  if (d.x && (rc = launch_gated_input_grad(a, kDtype, dgu, d.x, workspace, st, sms))) return rc;
  if (d.w_gate || d.w_up) return launch_gated_weight_grad(a, kDtype, dgu, d.w_gate, d.w_up, workspace, st, sms);
  return GFX_OK;
}

int launch_gated_backward(const GatedArgs& a, int dtype, int act, const void* dh, long long ldh, const float* save,
                          const GatedGrads& d, void* workspace, cudaStream_t st, int sms) {
  return dtype == GFX_DTYPE_F16 ? gated_backward_t<__half>(a, act, dh, ldh, save, d, workspace, st, sms)
                                : gated_backward_t<__nv_bfloat16>(a, act, dh, ldh, save, d, workspace, st, sms);
}

}  // namespace gfx
