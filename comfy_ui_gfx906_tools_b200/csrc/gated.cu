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
#include "common.cuh"
#include "gated.cuh"
#include "kernels.h"

namespace gfx {
namespace gated {

// ---------------------------------------------------------------------------
// C[i, j] = sum over segments s and k of A_s[i, k] B_s[j, k], any strides: 64 x 64 tiles, 4 x 4 a thread
// ---------------------------------------------------------------------------
template <typename T>
struct Operand {
  const T* p;
  long long row, k;  // strides
};

constexpr int kTile = 64, kDeep = 16;

template <typename T>
__device__ __forceinline__ void load_tile(float (*s)[kTile + 1], const Operand<T>& o, int i0, int rows, int k0, int K) {
  for (int e = threadIdx.x; e < kTile * kDeep; e += 256) {
    const int i = e / kDeep, k = e % kDeep;
    s[k][i] = i0 + i < rows && k0 + k < K ? to_f32<T>(o.p[(i0 + i) * o.row + (k0 + k) * o.k]) : 0.0f;
  }
}

// acc += A B^T over k < K
template <typename T>
__device__ __forceinline__ void tile_product(float (&acc)[4][4], float (*sa)[kTile + 1], float (*sb)[kTile + 1],
                                             const Operand<T>& a, const Operand<T>& b, int i0, int I, int j0, int J,
                                             int K) {
  const int ti = threadIdx.x / 16 * 4, tj = threadIdx.x % 16 * 4;
  for (int k0 = 0; k0 < K; k0 += kDeep) {
    __syncthreads();
    load_tile<T>(sa, a, i0, I, k0, K);
    load_tile<T>(sb, b, j0, J, k0, K);
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDeep; ++k)
#pragma unroll
      for (int y = 0; y < 4; ++y)
#pragma unroll
        for (int x = 0; x < 4; ++x) acc[y][x] += sa[k][ti + y] * sb[k][tj + x];
  }
}

template <typename T, int kAct>
__global__ void __launch_bounds__(256) forward_kernel(Operand<T> x, Operand<T> wg, Operand<T> wu, const T* bg,
                                                      const T* bu, T* h, float* save, int M, int K, int F) {
  __shared__ float sa[kDeep][kTile + 1], sb[kDeep][kTile + 1];
  const int i0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
  float g[4][4] = {}, u[4][4] = {};
  tile_product<T>(g, sa, sb, x, wg, i0, M, j0, F, K);
  tile_product<T>(u, sa, sb, x, wu, i0, M, j0, F, K);
  const int ti = i0 + threadIdx.x / 16 * 4, tj = j0 + threadIdx.x % 16 * 4;
  for (int y = 0; y < 4; ++y)
    for (int c = 0; c < 4; ++c) {
      const long long i = ti + y;
      const int j = tj + c;
      if (i >= M || j >= F) continue;
      const float gv = g[y][c] + (bg ? to_f32<T>(bg[j]) : 0.0f), uv = u[y][c] + (bu ? to_f32<T>(bu[j]) : 0.0f);
      h[i * F + j] = from_f32<T>(activation<kAct>(gv) * uv);
      if (save) save[i * F + j] = gv, save[(long long)M * F + i * F + j] = uv;
    }
}

template <typename T>
__global__ void __launch_bounds__(256) product_kernel(Operand<T> a0, Operand<T> b0, Operand<T> a1, Operand<T> b1,
                                                      int segments, T* c, int I, int J, int K) {
  __shared__ float sa[kDeep][kTile + 1], sb[kDeep][kTile + 1];
  const int i0 = blockIdx.y * kTile, j0 = blockIdx.x * kTile;
  float acc[4][4] = {};
  tile_product<T>(acc, sa, sb, a0, b0, i0, I, j0, J, K);
  if (segments == 2) tile_product<T>(acc, sa, sb, a1, b1, i0, I, j0, J, K);
  const int ti = i0 + threadIdx.x / 16 * 4, tj = j0 + threadIdx.x % 16 * 4;
  for (int y = 0; y < 4; ++y)
    for (int x = 0; x < 4; ++x)
      if (ti + y < I && tj + x < J) c[(long long)(ti + y) * J + tj + x] = from_f32<T>(acc[y][x]);
}

// ---------------------------------------------------------------------------
// dg, du (one row of dgu [M, 2F]: dg then du) and, per block of rows, their column sums
// ---------------------------------------------------------------------------
constexpr int kRowsPerBlock = 64;

template <typename T, int kAct>
__global__ void __launch_bounds__(256) gate_grad_kernel(const T* dh, long long ldh, const float* save, T* dgu,
                                                        float* partial, int M, int F) {
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
  if (c >= 2 * F) return;
  T* out = c < F ? dbg : dbu;
  if (out == nullptr) return;
  float v = 0.0f;
  for (int b = 0; b < blocks; ++b) v += partial[(long long)b * 2 * F + c];
  out[c < F ? c : c - F] = from_f32<T>(v);
}

}  // namespace gated

static int row_blocks(int M) { return (M + gated::kRowsPerBlock - 1) / gated::kRowsPerBlock; }

size_t gated_backward_workspace(int M, int F) {
  return align_up((size_t)M * 2 * F * 2, 256) + (size_t)row_blocks(M) * 2 * F * sizeof(float);
}

template <typename T>
static int gated_forward_t(const GatedArgs& a, int act, void* h, float* save, cudaStream_t st) {
  using O = gated::Operand<T>;
  const O x{(const T*)a.x, a.ldx, 1}, wg{(const T*)a.w_gate, a.ldg, 1}, wu{(const T*)a.w_up, a.ldu, 1};
  const dim3 grid((a.F + gated::kTile - 1) / gated::kTile, (a.M + gated::kTile - 1) / gated::kTile);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, st>>>(x, wg, wu, (const T*)a.b_gate, (const T*)a.b_up, (T*)h, save, a.M, a.K, a.F);
  };
  if (act == gated::kSilu)
    go(gated::forward_kernel<T, gated::kSilu>);
  else if (act == gated::kGelu)
    go(gated::forward_kernel<T, gated::kGelu>);
  else
    go(gated::forward_kernel<T, gated::kGeluTanh>);
  return check_launch("gated forward_kernel");
}

int launch_gated_forward(const GatedArgs& a, int dtype, int act, void* h, float* save, cudaStream_t st, int sms) {
  (void)sms;
  return dtype == GFX_DTYPE_F16 ? gated_forward_t<__half>(a, act, h, save, st)
                                : gated_forward_t<__nv_bfloat16>(a, act, h, save, st);
}

template <typename T>
static int gated_backward_t(const GatedArgs& a, int act, const void* dh, long long ldh, const float* save,
                            const GatedGrads& d, void* workspace, cudaStream_t st) {
  T* dgu = static_cast<T*>(workspace);
  float* partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + align_up((size_t)a.M * 2 * a.F * 2, 256));
  const int blocks = row_blocks(a.M);
  const bool bias = d.b_gate || d.b_up;
  const dim3 grid(blocks, (a.F + 127) / 128);
  auto go = [&](auto kern) {
    kern<<<grid, 256, 0, st>>>((const T*)dh, ldh, save, dgu, bias ? partial : nullptr, a.M, a.F);
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
    gated::bias_grad_kernel<T><<<(2 * a.F + 255) / 256, 256, 0, st>>>(partial, blocks, a.F, (T*)d.b_gate, (T*)d.b_up);
    if ((rc = check_launch("bias_grad_kernel"))) return rc;
  }
  using O = gated::Operand<T>;
  const int t = gated::kTile;
  const long long F = a.F;
  if (d.x) {  // dx = dg Wg + du Wu
    gated::product_kernel<T><<<dim3((a.K + t - 1) / t, (a.M + t - 1) / t), 256, 0, st>>>(
        O{dgu, 2 * F, 1}, O{(const T*)a.w_gate, 1, a.ldg}, O{dgu + F, 2 * F, 1}, O{(const T*)a.w_up, 1, a.ldu}, 2,
        (T*)d.x, a.M, a.K, a.F);
    if ((rc = check_launch("gated product_kernel"))) return rc;
  }
  for (int w = 0; w < 2; ++w) {  // dW = d^T x
    T* out = (T*)(w ? d.w_up : d.w_gate);
    if (!out) continue;
    const O A{dgu + w * F, 1, 2 * F}, B{(const T*)a.x, 1, a.ldx};
    gated::product_kernel<T><<<dim3((a.K + t - 1) / t, (a.F + t - 1) / t), 256, 0, st>>>(A, B, A, B, 1, out, a.F, a.K,
                                                                                         a.M);
    if ((rc = check_launch("gated product_kernel"))) return rc;
  }
  return GFX_OK;
}

int launch_gated_backward(const GatedArgs& a, int dtype, int act, const void* dh, long long ldh, const float* save,
                          const GatedGrads& d, void* workspace, cudaStream_t st, int sms) {
  (void)sms;
  return dtype == GFX_DTYPE_F16 ? gated_backward_t<__half>(a, act, dh, ldh, save, d, workspace, st)
                                : gated_backward_t<__nv_bfloat16>(a, act, dh, ldh, save, d, workspace, st);
}

}  // namespace gfx
