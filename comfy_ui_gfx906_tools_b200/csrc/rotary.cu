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
// Memory-bound, but the sines cost more than the rows they turn if every warp
// computes its own: a block of four warps first fills a table for its 4 tokens
// (fewer where the sequence is short), each angle once, and a warp then walks
// the heads of one token. G = 8, 16 or 32 lanes hold a row, eight elements each
// (two runs of four where the pairs are split halves), a warp 32 / G heads a
// step. The rows of three steps (two in the backward, which reads two arrays)
// are loaded before the first is used, without a branch between the loads.
// Arithmetic is on pairs of floats, one instruction for two. Measured on B200:
// forward of 4608 tokens x 48 heads x 128 in bfloat16 (113 MB) 21 us, 5.4 TB/s;
// 19982 tokens x 40 heads x 64, forward 48 us (205 MB), backward 89 us (307 MB).
// The forward runs at 32 warps an SM and issues 64% of the cycles, in 16-bit
// conversions and reductions between the loads. The backward waits on loads: its
// registers (109 to 123) leave 16 warps an SM, 47% of the cycles issue, and
// nothing is in flight while a warp works on the rows that it has.
#include <math.h>
#include <string.h>

#include "common.cuh"
#include "kernels.h"

namespace gfx {
namespace rotary {

constexpr int kWarps = 4;

// The eight elements of a lane as they lie in memory: four at p and four at p + gap.
template <typename T>
struct Raw {
  uint32_t w[2 * sizeof(T)];
};

// kOnce: a forward's input, which is not wanted in the cache again.
template <typename T, bool kVec, bool kOnce>
__device__ __forceinline__ Raw<T> load8(const T* p, int gap) {
  Raw<T> r;
  if constexpr (kVec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(r.w) = *reinterpret_cast<const uint4*>(p);
      *reinterpret_cast<uint4*>(r.w + 4) = *reinterpret_cast<const uint4*>(p + gap);
    } else if (gap == 4) {  // one run of eight
      *reinterpret_cast<uint4*>(r.w) = kOnce ? __ldcs(reinterpret_cast<const uint4*>(p)) : *reinterpret_cast<const uint4*>(p);
    } else {
      *reinterpret_cast<uint2*>(r.w) = *reinterpret_cast<const uint2*>(p);
      *reinterpret_cast<uint2*>(r.w + 2) = *reinterpret_cast<const uint2*>(p + gap);
    }
  } else {
    T* h = reinterpret_cast<T*>(r.w);
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = p[j], h[4 + j] = p[gap + j];
  }
  return r;
}

// r, or zeros
template <typename T>
__device__ __forceinline__ Raw<T> masked(Raw<T> r, bool keep) {
#pragma unroll
  for (int i = 0; i < (int)(2 * sizeof(T)); ++i) r.w[i] = keep ? r.w[i] : 0u;
  return r;
}

template <typename T, bool kVec>
__device__ __forceinline__ void store8(T* p, int gap, const Raw<T>& r) {
  if constexpr (kVec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.w);
      *reinterpret_cast<uint4*>(p + gap) = *reinterpret_cast<const uint4*>(r.w + 4);
    } else if (gap == 4) {
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.w);
    } else {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(r.w);
      *reinterpret_cast<uint2*>(p + gap) = *reinterpret_cast<const uint2*>(r.w + 2);
    }
  } else {
    const T* h = reinterpret_cast<const T*>(r.w);
#pragma unroll
    for (int j = 0; j < 4; ++j) p[j] = h[j], p[gap + j] = h[4 + j];
  }
}

__device__ __forceinline__ float sum(F2 a, F2 b) {
  float p, q, r, s;
  split(a, p, q), split(b, r, s);
  return (p + q) + (r + s);
}

// Position in memory (0 .. 7) of value i: values 0 .. 3 are the pairs' first elements, 4 .. 7 their second ones.
template <bool kPairs>
__device__ __forceinline__ constexpr int place(int i) {
  return kPairs ? (i < 4 ? 2 * i : 2 * (i - 4) + 1) : i;
}

__device__ __forceinline__ void halves(uint32_t w, float& lo, float& hi, __half) {
  const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
  lo = v.x, hi = v.y;
}
__device__ __forceinline__ void halves(uint32_t w, float& lo, float& hi, __nv_bfloat16) {
  lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xFFFF0000u);
}
__device__ __forceinline__ uint32_t join(float lo, float hi, __half) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t join(float lo, float hi, __nv_bfloat16) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}

template <typename T, bool kPairs>
__device__ __forceinline__ void unpack(const Raw<T>& r, F2 (&f)[4]) {
  float m[8];  // in memory's order
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4)
      m[2 * i] = __uint_as_float(r.w[2 * i]), m[2 * i + 1] = __uint_as_float(r.w[2 * i + 1]);
    else
      halves(r.w[i], m[2 * i], m[2 * i + 1], T());
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = f2(m[place<kPairs>(2 * i)], m[place<kPairs>(2 * i + 1)]);
}

template <typename T, bool kPairs>
__device__ __forceinline__ Raw<T> pack(const F2 (&f)[4]) {
  float m[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) split(f[i], m[place<kPairs>(2 * i)], m[place<kPairs>(2 * i + 1)]);
  Raw<T> r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4)
      r.w[2 * i] = __float_as_uint(m[2 * i]), r.w[2 * i + 1] = __float_as_uint(m[2 * i + 1]);
    else
      r.w[i] = join(m[2 * i], m[2 * i + 1], T());
  }
  return r;
}

__device__ __forceinline__ double position_at(const void* pos, int dtype, long long i) {
  if (dtype == kPositionI64) return (double)static_cast<const long long*>(pos)[i];
  if (dtype == kPositionI32) return (double)static_cast<const int*>(pos)[i];
  return (double)static_cast<const float*>(pos)[i];
}

// A scale vector's value in any of the three float types.
__device__ __forceinline__ float scale_at(const void* w, int dtype, int i) {
  if (dtype == GFX_DTYPE_F32) return static_cast<const float*>(w)[i];
  if (dtype == GFX_DTYPE_F16) return __half2float(static_cast<const __half*>(w)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
}

// Pairs (f[0..1], f[2..3]) turned by angles of cosine c and sine s; ns = -s. Unless kWhole, only the first n of the four
// are turned: a pair that passes through keeps its values, which a turn by the angle 0 would not do (an infinity times
// the sine 0 is a NaN in the pair's other value).
template <bool kWhole>
__device__ __forceinline__ void turn(F2 (&f)[4], const F2 (&c)[2], const F2 (&s)[2], const F2 (&ns)[2], int n) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const F2 x = f[i], y = f[2 + i];
    f[i] = fma2(x, c[i], y * ns[i]);
    f[2 + i] = fma2(x, s[i], y * c[i]);
    if constexpr (!kWhole) {
      float x0, x1, y0, y1, a, b;
      split(x, x0, x1), split(y, y0, y1);
      split(f[i], a, b);
      f[i] = f2(n > 2 * i ? a : x0, n > 2 * i + 1 ? b : x1);
      split(f[2 + i], a, b);
      f[2 + i] = f2(n > 2 * i ? a : y0, n > 2 * i + 1 ? b : y1);
    }
  }
}

// kBackward: in is dy, x the forward's input (read where the tensor has a
// scale), out is dx, and each block leaves its sums of dz xh in partial
// [block][2][D] (q, then k).
// kVec: every row starts at a multiple of 16 bytes. kWhole: no pair passes through.
// Eight blocks an SM hold the forward to 64 registers: 16-bit rows fit, float32 ones spill 4 to 36 bytes a thread.
template <typename T, int G, bool kPairs, bool kVec, bool kBackward, bool kWhole>
__global__ void __launch_bounds__(kWarps * 32, kBackward ? 4 : 8) rope_kernel(const __grid_constant__ RopeArgs a) {
  constexpr int kRows = 32 / G, kLanePairs = 4 * G;
  constexpr int kAhead = kBackward ? 2 : 3;  // steps whose rows are in flight at once
  __shared__ __align__(16) float scales[2][8 * G];
  __shared__ __align__(16) float cosines[kWarps][kLanePairs], sines[kWarps][kLanePairs];  // of the block's tokens
  __shared__ float sums[kBackward ? kWarps : 1][2][kBackward ? 8 * G : 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane % G, grp = lane / G;
  const int D = a.D, half = a.pairs;
  // this lane's elements are e0 .. e0 + 3 and e0 + gap .. e0 + gap + 3; its pairs 4 sub .. 4 sub + 3
  const bool apart = !kPairs && 8 * sub < 2 * half;
  const int e0 = apart ? 4 * sub : 8 * sub, gap = kPairs ? 4 : (apart ? half : 4);
  const bool live = 8 * sub < D;
  const int turned = half - 4 * sub;  // how many of this lane's pairs turn: all from 4 on, none from 0 down
  pdl_trigger();
  pdl_wait();
  for (int i = threadIdx.x; i < 16 * G; i += kWarps * 32) {
    const int w = i / (8 * G), e = i % (8 * G);
    scales[w][e] = a.t[w].scale != nullptr && e < D ? scale_at(a.t[w].scale, a.scale_dtype, e) : 0.0f;
  }
  // value i's place in a row that was cut as this lane's elements are
  auto element = [&](int i) {
    const int m = place<kPairs>(i);
    return m < 4 ? e0 + m : e0 + gap + m - 4;
  };
  F2 dw[2][4];
#pragma unroll
  for (int i = 0; i < 4; ++i) dw[0][i] = dw[1][i] = f2(0.0f, 0.0f);

  // this thread's pair of the table; its tokens are threadIdx.x / kLanePairs and so on
  const int pair = threadIdx.x % kLanePairs;
  const double freq = pair < half ? a.freq[pair] : 0.0;
  const long long axis_at = pair < half ? a.axis[pair] * a.pos_stride[2] : 0;
  const uint32_t tokens = a.tokens, group = a.group;  // tokens a block holds at once: 1, 2 or 4
  const int slot = warp % group;                      // this warp's token of them
  const int part = warp / group + (int)blockIdx.y * (kWarps / group);

  for (uint32_t t0 = blockIdx.x * group; t0 < tokens; t0 += gridDim.x * group) {
    if (kBackward) __syncthreads();  // the last tokens' table is no longer read
    for (uint32_t i = threadIdx.x / kLanePairs; i < group; i += kWarps * 32 / kLanePairs) {
      const uint32_t token = min(t0 + i, tokens - 1), b = token / (uint32_t)a.L, l = token - b * (uint32_t)a.L;
      double t = 0.0;
      if (pair < half) t = position_at(a.pos, a.pos_dtype, b * a.pos_stride[0] + l * a.pos_stride[1] + axis_at) * freq;
      t -= rint(t);
      float sn, cs;
      sincospif(2.0f * (float)t, &sn, &cs);
      cosines[i][pair] = cs;
      sines[i][pair] = kBackward ? -sn : sn;
    }
    __syncthreads();
    const uint32_t token = t0 + slot;
    if (token >= tokens) continue;
    const uint32_t bi = token / (uint32_t)a.L;
    const long long b = bi, l = token - bi * (uint32_t)a.L;
    F2 c[2], s[2], ns[2];
    {
      const float4 cv = *reinterpret_cast<const float4*>(&cosines[slot][4 * sub]);
      const float4 sv = *reinterpret_cast<const float4*>(&sines[slot][4 * sub]);
      c[0] = f2(cv.x, cv.y), c[1] = f2(cv.z, cv.w), s[0] = f2(sv.x, sv.y), s[1] = f2(sv.z, sv.w);
      ns[0] = f2(-sv.x, -sv.y), ns[1] = f2(-sv.z, -sv.w);
    }
    // steps of 32 / G heads: q's, then k's
    const int s0 = part * a.steps_per_part;
#pragma unroll
    for (int w = 0; w < 2; ++w) {
      const RopeTensor& x = a.t[w];
      const int first = w ? (a.heads[0] + kRows - 1) / kRows : 0;
      const int start = max(first, s0);
      const int last = min(first + (a.heads[w] + kRows - 1) / kRows, s0 + a.steps_per_part);
      if (start >= last) continue;
      const bool norm = x.scale != nullptr;
      F2 scale[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) scale[i] = f2(scales[w][element(2 * i)], scales[w][element(2 * i + 1)]);
      // this lane's head of the first step, how many of the steps it has a row in, and where that row lies
      const int h0 = (start - first) * kRows + grp;
      const int count = live ? min(last - start, (a.heads[w] - h0 + kRows - 1) / kRows) : 0;
      const T* in0 = static_cast<const T*>(x.in) + b * x.in_stride[0] + l * x.in_stride[2];
      const T* org0 = static_cast<const T*>(x.x) + b * x.x_stride[0] + l * x.x_stride[2];
      const T* src = in0 + h0 * x.in_stride[1] + e0;
      const T* org = org0 + h0 * x.x_stride[1] + e0;
      T* dst = static_cast<T*>(x.out) + b * x.out_stride[0] + h0 * x.out_stride[1] + l * x.out_stride[2] + e0;
      const long long src_step = kRows * x.in_stride[1], org_step = kRows * x.x_stride[1];
      const long long dst_step = kRows * x.out_stride[1];
      for (int i0 = 0; i0 < last - start; i0 += kAhead) {
        Raw<T> in[kAhead], xs[kBackward ? kAhead : 1];
        // a lane without a row reads the token's first head instead, so that no load waits behind a branch
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          const bool row = i0 + q < count;
          in[q] = load8<T, kVec, !kBackward>(row ? src : in0, row ? gap : 4);
          if (kBackward && norm) xs[q] = load8<T, kVec, !kBackward>(row ? org : org0, row ? gap : 4);
          src += src_step;
          if (kBackward) org += org_step;
        }
        // the rows' sums go through the lanes side by side, so that their shuffles overlap
        float ss[kAhead], dot[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          in[q] = masked<T>(in[q], i0 + q < count);
          ss[q] = dot[q] = 0.0f;
          if (norm) {
            F2 xv[4];
            if constexpr (kBackward) {
              xs[q] = masked<T>(xs[q], i0 + q < count);
              F2 t[4];
              unpack<T, kPairs>(in[q], t);
              turn<kWhole>(t, c, s, ns, turned);
              unpack<T, kPairs>(xs[q], xv);
#pragma unroll
              for (int i = 0; i < 4; ++i) t[i] = t[i] * scale[i];
              dot[q] = sum(fma2(t[1], xv[1], t[0] * xv[0]), fma2(t[3], xv[3], t[2] * xv[2]));
            } else {
              unpack<T, kPairs>(in[q], xv);
            }
            ss[q] = sum(fma2(xv[1], xv[1], xv[0] * xv[0]), fma2(xv[3], xv[3], xv[2] * xv[2]));
          }
        }
        if (norm) {
#pragma unroll
          for (int o = G / 2; o > 0; o >>= 1)
#pragma unroll
            for (int q = 0; q < kAhead; ++q) {
              ss[q] += __shfl_xor_sync(0xFFFFFFFFu, ss[q], o);
              if (kBackward) dot[q] += __shfl_xor_sync(0xFFFFFFFFu, dot[q], o);
            }
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
          F2 f[4];
          unpack<T, kPairs>(in[q], f);
          if (norm) {
            float r = rsqrtf(ss[q] * a.inv_dim + a.eps);
            // a lane without a row has ss = 0: with eps = 0 its r would be infinite, and 0 * r in dw a NaN
            if (kBackward && i0 + q >= count) r = 0.0f;
            const F2 rr = f2(r, r);
            if constexpr (!kBackward) {
#pragma unroll
              for (int i = 0; i < 4; ++i) f[i] = f[i] * rr * scale[i];
              turn<kWhole>(f, c, s, ns, turned);
            } else {
              turn<kWhole>(f, c, s, ns, turned);  // dz
              const float mean = dot[q] * r * a.inv_dim;  // mean(w dz xh)
              const F2 less = f2(-mean, -mean);
              F2 xv[4];
              unpack<T, kPairs>(xs[q], xv);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const F2 xh = xv[i] * rr;
                dw[w][i] = fma2(f[i], xh, dw[w][i]);
                f[i] = fma2(xh, less, f[i] * scale[i]) * rr;
              }
            }
          } else {
            turn<kWhole>(f, c, s, ns, turned);
          }
          if (i0 + q < count) store8<T, kVec>(dst, gap, pack<T, kPairs>(f));
          dst += dst_step;
        }
      }
    }
    if (!kBackward) break;  // one set of tokens a block
  }
  if constexpr (kBackward) {
    if (a.partial == nullptr) return;
    // rows of a warp, then the block's warps, always in the same order
#pragma unroll
    for (int w = 0; w < 2; ++w)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float v[2];
        split(dw[w][i], v[0], v[1]);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int o = G; o < 32; o <<= 1) v[j] += __shfl_xor_sync(0xFFFFFFFFu, v[j], o);
          if (grp == 0 && live) sums[warp][w][element(2 * i + j)] = v[j];
        }
      }
    __syncthreads();
    float* out = a.partial + (long long)(blockIdx.y * gridDim.x + blockIdx.x) * 2 * D;
    for (int i = threadIdx.x; i < 2 * D; i += kWarps * 32) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) v += sums[k][i / D][i % D];
      out[i] = v;
    }
  }
}

// dw[t][e] = sum over blocks of partial[block][t][e], eight columns a block of 8 x 128 threads, in a fixed order.
__global__ void __launch_bounds__(1024) scale_grad_kernel(const float* partial, int blocks, int D, void* dq, void* dk,
                                                          int dtype) {
  __shared__ float s[128][9];
  const int x = threadIdx.x & 7, y = threadIdx.x >> 3, e = blockIdx.x * 8 + x, t = blockIdx.y;
  const float* from = partial + (long long)t * D + e;
  pdl_trigger();
  pdl_wait();
  float v = 0.0f;
#pragma unroll 8
  for (int b = y; b < blocks; b += 128) v += from[(long long)b * 2 * D];
  s[y][x] = v;
  __syncthreads();
  for (int n = 64; n > 0; n >>= 1) {
    if (y < n) s[y][x] += s[y + n][x];
    __syncthreads();
  }
  void* out = t ? dk : dq;
  if (y != 0 || out == nullptr) return;
  if (dtype == GFX_DTYPE_F32)
    static_cast<float*>(out)[e] = s[0][x];
  else if (dtype == GFX_DTYPE_F16)
    static_cast<__half*>(out)[e] = __float2half_rn(s[0][x]);
  else
    static_cast<__nv_bfloat16*>(out)[e] = __float2bfloat16_rn(s[0][x]);
}

}  // namespace rotary

// Turns per unit of position of every pair, and the axis that moves it. Computed again only when the axes or theta
// are others than the thread's last call had (64 powers take longer than the launch).
void rope_frequencies(RopeArgs* a, const int* axes_dims, int n_axes, double theta) {
  struct Table {
    int n = 0, dims[kRopeMaxAxes], pairs;
    double theta, freq[kRopeMaxDim / 2];
    unsigned char axis[kRopeMaxDim / 2];
  };
  static thread_local Table t;
  if (t.n != n_axes || t.theta != theta || memcmp(t.dims, axes_dims, sizeof(int) * n_axes) != 0) {
    int p = 0;
    for (int i = 0; i < n_axes; ++i)
      for (int j = 0; j < axes_dims[i] / 2; ++j, ++p) {
        t.freq[p] = pow(theta, -2.0 * j / axes_dims[i]) / 6.283185307179586476925286766559;
        t.axis[p] = (unsigned char)i;
      }
    t.n = n_axes, t.theta = theta, t.pairs = p;
    memcpy(t.dims, axes_dims, sizeof(int) * n_axes);
  }
  memcpy(a->freq, t.freq, sizeof(double) * t.pairs);
  memcpy(a->axis, t.axis, t.pairs);
  a->pairs = t.pairs;
  a->axes = n_axes;
}

// A block's four warps hold 4 tokens, or fewer with several warps a token where that leaves less than six blocks an SM:
// more tokens a block share the table's cost, more blocks fill the SMs. Forward, us with three / six / twelve blocks:
//   48 heads x 128   1900 tokens 18.8 / 12.0 / 13.2   3300 19.4 / 17.7 / 19.4   4608 20.6 / 20.6 / 22.3   6000 32.8 / 32.8 / 30.9
//   16 heads x 64    1900 tokens 7.9 / 6.2 / 8.9      3300 8.3 / 8.7 / 13.3     4608 8.4 / 8.4 / 10.5     6000 11.0 / 11.0 / 12.9
// A lone token's heads are spread over blocks too, down to one step a warp. A backward that sums scale gradients keeps to
// a fixed number of blocks, which walk the tokens.
static dim3 plan(RopeArgs* a, int rows, int sms) {
  const long long tokens = (long long)a->B * a->L;
  const int steps = (a->heads[0] + rows - 1) / rows + (a->heads[1] + rows - 1) / rows;
  int group = rotary::kWarps;
  while (group > 1 && tokens / group < 6ll * sms) group /= 2;
  const int warps = rotary::kWarps / group;  // of a token, in one block
  int spread = 1;
  while (group == 1 && spread * warps < steps && tokens * spread < sms) ++spread;
  a->tokens = (unsigned)tokens;
  a->group = group;
  a->steps_per_part = (steps + spread * warps - 1) / (spread * warps);
  const long long blocks = (tokens + group - 1) / group, most = a->partial != nullptr ? kRopeMaxBlocks / spread : blocks;
  return dim3((unsigned)(blocks < most ? blocks : most), (unsigned)spread);
}

static int lanes_per_row(int D) { return D <= 64 ? 8 : (D <= 128 ? 16 : 32); }

template <typename T, int G, bool kPairs, bool kVec>
static int launch_t(const RopeArgs& a, bool backward, dim3 blocks, cudaStream_t st) {
  auto go = [&](auto kern) { launch_overlapped(kern, blocks, rotary::kWarps * 32, st, a); };
  // forms of their own where the whole row is turned: with one form that tests for it, the backward of 19982 tokens x 40
  // heads x 64 took 94 us instead of 89, the forward 49.5 instead of 48.6
  const bool whole = 2 * a.pairs == a.D;
  if (backward)
    whole ? go(rotary::rope_kernel<T, G, kPairs, kVec, true, true>) : go(rotary::rope_kernel<T, G, kPairs, kVec, true, false>);
  else
    whole ? go(rotary::rope_kernel<T, G, kPairs, kVec, false, true>) : go(rotary::rope_kernel<T, G, kPairs, kVec, false, false>);
  return check_launch("rope_kernel");
}

template <typename T, int G>
static int launch_p(const RopeArgs& a, bool pairs, bool backward, dim3 blocks, cudaStream_t st) {
  if (a.vec)
    return pairs ? launch_t<T, G, true, true>(a, backward, blocks, st) : launch_t<T, G, false, true>(a, backward, blocks, st);
  return pairs ? launch_t<T, G, true, false>(a, backward, blocks, st) : launch_t<T, G, false, false>(a, backward, blocks, st);
}

template <typename T>
static int launch_g(const RopeArgs& a, bool pairs, bool backward, dim3 blocks, cudaStream_t st) {
  const int g = lanes_per_row(a.D);
  if (g == 8) return launch_p<T, 8>(a, pairs, backward, blocks, st);
  if (g == 16) return launch_p<T, 16>(a, pairs, backward, blocks, st);
  return launch_p<T, 32>(a, pairs, backward, blocks, st);
}

int launch_rope(RopeArgs& a, int dtype, bool pairs, bool backward, void* dq_scale, void* dk_scale, cudaStream_t st,
                int sms) {
  const dim3 blocks = plan(&a, 32 / lanes_per_row(a.D), sms);
  int rc;
  if (dtype == GFX_DTYPE_F32)
    rc = launch_g<float>(a, pairs, backward, blocks, st);
  else if (dtype == GFX_DTYPE_F16)
    rc = launch_g<__half>(a, pairs, backward, blocks, st);
  else
    rc = launch_g<__nv_bfloat16>(a, pairs, backward, blocks, st);
  if (rc || !backward || a.partial == nullptr) return rc;
  launch_overlapped(rotary::scale_grad_kernel, dim3(a.D / 8, 2), 1024, st, a.partial, (int)(blocks.x * blocks.y), a.D,
                    dq_scale, dk_scale, a.scale_dtype);
  return check_launch("scale_grad_kernel");
}

}  // namespace gfx
