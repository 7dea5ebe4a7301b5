// q/k RMS normalisation with multi-axis rotary positions, forward and backward.
//
// A head row x of D elements (per batch, head and token):
//   xh = x r,  r = 1 / sqrt(mean(x^2) + eps)         (where the tensor has a scale w)
//   z  = w xh
//   y  = R z:  pair p of axis a turns by  t = position[a] theta^(-2 j / d_a),
//        (y0, y1) = (z0 cos t - z1 sin t, z0 sin t + z1 cos t);
//        elements past the rotated ones pass through.
// Backward, from dy:
//   dz = R^T dy,  dw = sum over rows of dz xh,
//   dx = r (w dz - xh mean(w dz xh)).
// Pairs are neighbours (2p, 2p + 1), or split halves (p, p + R/2) of the R
// rotated elements; axis a owns d_a / 2 consecutive pairs.
//
// Angles: position * frequency is formed in float64 in units of a turn, and
// only the fraction of a turn goes to float32, so the angle's error does not
// grow with the position (in float32 it is 1e-4 rad at position 2000, far
// above a float32 result's rounding). Statistics and sums are float32.
//
// Memory-bound. A warp owns one token of a part of its heads, so a lane
// computes the sines of its own four pairs once and reuses them for every head;
// G = 8, 16 or 32 lanes hold a row, eight elements each (two runs of four where
// the pairs are split halves), and a warp's rows are 32 / G heads at a time.
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "kernels.h"

namespace gfx {
namespace rotary {

constexpr int kWarps = 8;

// The eight elements of a lane: elements e0 .. e0 + 3 and e1 .. e1 + 3.
template <typename T>
__device__ __forceinline__ void load8(const T* row, int e0, int e1, bool vec, float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      const float4 a = *reinterpret_cast<const float4*>(row + e0), b = *reinterpret_cast<const float4*>(row + e1);
      f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
      return;
    }
  } else {
    if (vec) {
      uint2 w[2];
      if (e1 == e0 + 4) {
        const uint4 q = *reinterpret_cast<const uint4*>(row + e0);
        w[0] = make_uint2(q.x, q.y), w[1] = make_uint2(q.z, q.w);
      } else {
        w[0] = *reinterpret_cast<const uint2*>(row + e0);
        w[1] = *reinterpret_cast<const uint2*>(row + e1);
      }
      const T* h = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = to_f32<T>(h[j]);
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) f[j] = to_f32<T>(row[e0 + j]), f[4 + j] = to_f32<T>(row[e1 + j]);
}

template <typename T>
__device__ __forceinline__ void store8(T* row, int e0, int e1, bool vec, const float (&f)[8]) {
  if constexpr (sizeof(T) == 4) {
    if (vec) {
      *reinterpret_cast<float4*>(row + e0) = make_float4(f[0], f[1], f[2], f[3]);
      *reinterpret_cast<float4*>(row + e1) = make_float4(f[4], f[5], f[6], f[7]);
      return;
    }
  } else {
    if (vec) {
      uint2 w[2];
      T* h = reinterpret_cast<T*>(w);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = from_f32<T>(f[j]);
      if (e1 == e0 + 4) {
        *reinterpret_cast<uint4*>(row + e0) = make_uint4(w[0].x, w[0].y, w[1].x, w[1].y);
      } else {
        *reinterpret_cast<uint2*>(row + e0) = w[0];
        *reinterpret_cast<uint2*>(row + e1) = w[1];
      }
      return;
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) row[e0 + j] = from_f32<T>(f[j]), row[e1 + j] = from_f32<T>(f[4 + j]);
}

__device__ __forceinline__ double position_at(const void* pos, int dtype, long long i) {
  if (dtype == kPositionF32) return (double)static_cast<const float*>(pos)[i];
  if (dtype == kPositionI32) return (double)static_cast<const int*>(pos)[i];
  return (double)static_cast<const long long*>(pos)[i];
}

// A scale vector's value in any of the three float types.
__device__ __forceinline__ float scale_at(const void* w, int dtype, int i) {
  if (dtype == GFX_DTYPE_F32) return static_cast<const float*>(w)[i];
  if (dtype == GFX_DTYPE_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// Pairs (j, j + 1) of f for neighbours, (j, j + 4) for split halves, turned by (c, s).
template <bool kPairs>
__device__ __forceinline__ void turn(float (&f)[8], const float (&c)[4], const float (&s)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float& a = f[kPairs ? 2 * j : j];
    float& b = f[kPairs ? 2 * j + 1 : j + 4];
    const float x = a, y = b;
    a = x * c[j] - y * s[j];
    b = x * s[j] + y * c[j];
  }
}

template <int G>
__device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = G / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  return v;
}

// kBackward: y is dy, x the forward's input (read where the tensor has a
// scale), out is dx, and each block leaves its sums of dz xh in partial
// [block][2][D] (q, then k).
template <typename T, int G, bool kPairs, bool kBackward>
__global__ void __launch_bounds__(kWarps * 32) rope_kernel(const __grid_constant__ RopeArgs a) {
  __shared__ float sums[kBackward ? kWarps : 1][2][kBackward ? 8 * G : 1];
  constexpr int kRows = 32 / G;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % G, grp = lane / G;
  const int D = a.D, half = a.pairs;
  // elements of this lane and its pairs
  int e0 = 8 * sub, e1 = e0 + 4, p0 = 4 * sub;
  if (!kPairs && 8 * sub < 2 * half) e0 = 4 * sub, e1 = half + 4 * sub;
  const bool live = 8 * sub < D;
  double freq[4];
  int axis[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool turned = live && p0 + j < half;
    freq[j] = turned ? a.freq[p0 + j] : 0.0;
    axis[j] = turned ? (int)a.axis[p0 + j] : 0;
  }
  float dw[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) dw[0][j] = dw[1][j] = 0.0f;

  const long long units = (long long)a.B * a.L * a.parts;
  for (long long u = (long long)blockIdx.x * kWarps + warp; u < units; u += (long long)gridDim.x * kWarps) {
    const long long token = u / a.parts;
    const int part = (int)(u - token * a.parts);
    const long long b = token / a.L, l = token - b * a.L;
    float c[4], s[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      double t = 0.0;
      if (freq[j] != 0.0)
        t = position_at(a.pos, a.pos_dtype, b * a.pos_stride[0] + l * a.pos_stride[1] + axis[j] * a.pos_stride[2]) *
            freq[j];
      t -= rint(t);
      sincospif(2.0f * (float)t, &s[j], &c[j]);
      if (kBackward) s[j] = -s[j];
    }
    // steps of 32 / G heads: q's, then k's
    const int s0 = part * a.steps_per_part;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const RopeTensor& x = a.t[w];
      const int first = w ? (a.heads[0] + kRows - 1) / kRows : 0;
      const int last = min(first + (a.heads[w] + kRows - 1) / kRows, s0 + a.steps_per_part);
      const bool norm = x.scale != nullptr;
      float scale[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        scale[j] = norm && live ? scale_at(x.scale, a.scale_dtype, (j < 4 ? e0 : e1 - 4) + j) : 0.0f;
      for (int step = max(first, s0); step < last; ++step) {
        const long long h = (step - first) * kRows + grp;
        const bool row = h < a.heads[w] && live;
        float f[8], xv[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = 0.0f, xv[j] = 0.0f;
        if (row) {
          const T* src = static_cast<const T*>(x.in) + b * x.in_stride[0] + h * x.in_stride[1] + l * x.in_stride[2];
          load8<T>(src, e0, e1, a.vec, f);
          if (kBackward && norm) {
            const T* xs = static_cast<const T*>(x.x) + b * x.x_stride[0] + h * x.x_stride[1] + l * x.x_stride[2];
            load8<T>(xs, e0, e1, a.vec, xv);
          }
        }
        if constexpr (!kBackward) {
          if (norm) {
            float ss = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
            const float r = rsqrtf(row_sum<G>(ss) / (float)D + a.eps);
#pragma unroll
            for (int j = 0; j < 8; ++j) f[j] = f[j] * r * scale[j];
          }
          turn<kPairs>(f, c, s);
        } else {
          turn<kPairs>(f, c, s);  // dz
          if (norm) {
            float ss = 0.0f, dot = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              ss += xv[j] * xv[j];
              dot += f[j] * scale[j] * xv[j];
            }
            const float r = rsqrtf(row_sum<G>(ss) / (float)D + a.eps);
            const float mean = row_sum<G>(dot) * r / (float)D;  // mean(w dz xh)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              const float xh = xv[j] * r;
              dw[w][j] += f[j] * xh;
              f[j] = r * (f[j] * scale[j] - xh * mean);
            }
          }
        }
        if (row) {
          T* dst = static_cast<T*>(x.out) + b * x.out_stride[0] + h * x.out_stride[1] + l * x.out_stride[2];
          store8<T>(dst, e0, e1, a.vec, f);
        }
      }
    }
  }
  if constexpr (kBackward) {
    if (a.partial == nullptr) return;
    // rows of a warp, then the block's warps, always in the same order
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = dw[w][j];
#pragma unroll
        for (int o = G; o < 32; o <<= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
        if (grp == 0 && live) sums[warp][w][(j < 4 ? e0 : e1 - 4) + j] = v;
      }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v += sums[k][i / D][i % D];
      a.partial[(long long)blockIdx.x * 2 * D + i] = v;
    }
  }
}

// dw[t][e] = sum over blocks of partial[block][t][e]: one block per 32 elements, 32 rows of threads.
__global__ void __launch_bounds__(1024) scale_grad_kernel(const float* partial, int blocks, int D, void* dq, void* dk,
                                                          int dtype) {
  __shared__ float s[32][33];
  const int e = blockIdx.x * 32 + threadIdx.x, t = blockIdx.y;
  float v = 0.0f;
  if (e < D)
    for (int b = threadIdx.y; b < blocks; b += 32) v += partial[((long long)b * 2 + t) * D + e];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  if (threadIdx.y == 0 && e < D) {
    float sum = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) sum += s[k][threadIdx.x];
    void* out = t ? dk : dq;
    if (out == nullptr) return;
    if (dtype == GFX_DTYPE_F32)
      static_cast<float*>(out)[e] = sum;
    else if (dtype == GFX_DTYPE_F16)
      static_cast<__half*>(out)[e] = __float2half_rn(sum);
    else
      static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(sum);
  }
}

}  // namespace rotary

// Turns per unit of position of every pair, and the axis that moves it.
void rope_frequencies(RopeArgs* a, const int* axes_dims, int n_axes, double theta) {
  int p = 0;
  for (int i = 0; i < n_axes; ++i)
    for (int j = 0; j < axes_dims[i] / 2; ++j, ++p) {
      a->freq[p] = pow(theta, -2.0 * j / axes_dims[i]) / 6.283185307179586476925286766559;
      a->axis[p] = (unsigned char)i;
    }
  a->pairs = p;
}

// Blocks of the launch, and how many parts a token's heads are cut into: a
// whole token per warp amortises the sines best, but a short sequence is cut
// until the GPU has two warps for every scheduler or a part is one step.
static int plan(RopeArgs* a, int rows, int sms) {
  const long long tokens = (long long)a->B * a->L;
  const int steps = (a->heads[0] + rows - 1) / rows + (a->heads[1] + rows - 1) / rows;
  long long parts = 1;
  while (parts < steps && tokens * parts < (long long)sms * 8) ++parts;
  a->steps_per_part = (int)((steps + parts - 1) / parts);
  a->parts = (steps + a->steps_per_part - 1) / a->steps_per_part;
  const long long warps = tokens * a->parts, blocks = (warps + rotary::kWarps - 1) / rotary::kWarps;
  return (int)(blocks < kRopeMaxBlocks ? blocks : kRopeMaxBlocks);
}

static int lanes_per_row(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }

template <typename T, int G, bool kPairs>
static int launch_t(const RopeArgs& a, bool backward, int blocks, cudaStream_t st) {
  if (backward)
    rotary::rope_kernel<T, G, kPairs, true><<<blocks, rotary::kWarps * 32, 0, st>>>(a);
  else
    rotary::rope_kernel<T, G, kPairs, false><<<blocks, rotary::kWarps * 32, 0, st>>>(a);
  return check_launch("rope_kernel");
}

template <typename T, int G>
static int launch_p(const RopeArgs& a, bool pairs, bool backward, int blocks, cudaStream_t st) {
  return pairs ? launch_t<T, G, true>(a, backward, blocks, st) : launch_t<T, G, false>(a, backward, blocks, st);
}

template <typename T>
static int launch_g(const RopeArgs& a, bool pairs, bool backward, int blocks, cudaStream_t st) {
  const int g = lanes_per_row(a.D);
  if (g == 8) return launch_p<T, 8>(a, pairs, backward, blocks, st);
  if (g == 16) return launch_p<T, 16>(a, pairs, backward, blocks, st);
  return launch_p<T, 32>(a, pairs, backward, blocks, st);
}

int launch_rope(RopeArgs& a, int dtype, bool pairs, bool backward, void* dq_scale, void* dk_scale, cudaStream_t st,
                int sms) {
  const int blocks = plan(&a, 32 / lanes_per_row(a.D), sms);
  int rc;
  if (dtype == GFX_DTYPE_F32)
    rc = launch_g<float>(a, pairs, backward, blocks, st);
  else if (dtype == GFX_DTYPE_F16)
    rc = launch_g<__half>(a, pairs, backward, blocks, st);
  else
    rc = launch_g<__nv_bfloat16>(a, pairs, backward, blocks, st);
  if (rc || !backward || a.partial == nullptr) return rc;
  rotary::scale_grad_kernel<<<dim3((a.D + 31) / 32, 2), dim3(32, 32), 0, st>>>(a.partial, blocks, a.D, dq_scale,
                                                                               dk_scale, a.scale_dtype);
  return check_launch("scale_grad_kernel");
}

}  // namespace gfx
