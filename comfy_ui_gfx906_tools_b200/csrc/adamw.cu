// One AdamW step over many tensors in one launch, first and second moments in
// float32 or in 8 bits with one float32 scale per 256 elements.
//
//   m <- b1 m + (1 - b1) g          v <- b2 v + (1 - b2) g^2
//   p <- p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// 8-bit moments are companded: a code c stands for the value c |c| s, so the
// steps between neighbouring codes shrink towards zero. The first moment holds
// c in [-127, 127]; the second moment holds its square root, c in [0, 255],
// and a positive one keeps at least the code 1: rounded to 0 it would leave
// the next update of that element nothing but eps to divide by. s is the
// block's largest magnitude over 127^2 (255^2). Every step of the coding is a
// correctly rounded float32 operation, so its result is the same wherever it
// is computed.
//
// Memory-bound: p is read and written, g read, each moment read and written.
// A warp owns 256 consecutive elements at a time, which is one block of the
// 8-bit form: its largest magnitude is one warp-wide integer maximum
// (magnitudes order as their bit patterns do, and a NaN lies above every
// number, so it is not lost). A lane holds elements 4 l .. 4 l + 3 of each
// 128-element half, so every access of the warp is one contiguous run.
//
// Measured on B200, 151 M bfloat16 elements: 32-bit moments 492 us, 6.7 TB/s,
// the memory's rate. With 8-bit moments (1.52 GB, 232 us of memory) the
// arithmetic takes longer than the memory: 441 us, bound by the issue of 74
// instructions an element. With every root correctly rounded it was 100
// instructions and 758 us, so the full blocks' path takes the hardware's
// approximate roots, off by 2^-23, and decides a code by them unless the root
// lies so near the middle between two codes that this error could matter; a
// lane that sees such an element (one in five thousand), or a vanishing root,
// does its eight elements again exactly. The parameters' move, which no code
// depends on, takes them too: it is off by some 2^-22 of itself there, and exact
// to the division's rounding in a tensor's ragged end and in the 32-bit form, so
// a parameter's last bit may depend on its place in the tensor. Codes are turned into floats and back
// by adding 2^23 and 1.5 * 2^23, not by the quarter-rate conversions. Packed
// pairs of floats are not used here: the compiler fuses a packed product and
// sum, and the moments' definition rounds both.
#include "common.cuh"
#include "kernels.h"

namespace gfx {
namespace adamw {

constexpr int kWarps = 8;
constexpr int kBlock = 256;  // elements per warp step = elements per 8-bit scale

struct Args {
  AdamwTensor t[kAdamwMaxTensors];
  int count;
  int blocks_per_cta;  // 256-element blocks one CTA takes
  const float* grad_scale;
  float beta1, one_minus_beta1, beta2, one_minus_beta2, decay, step_size, root_scale, eps;
};

template <typename T>
struct Quad;
template <>
struct Quad<float> {
  using V = float4;
  static __device__ __forceinline__ void unpack(const V& v, float (&f)[4]) {
    f[0] = v.x, f[1] = v.y, f[2] = v.z, f[3] = v.w;
  }
  static __device__ __forceinline__ V pack(const float (&f)[4]) { return make_float4(f[0], f[1], f[2], f[3]); }
};
template <typename T, typename T2>
struct Quad16 {
  using V = uint2;
  static __device__ __forceinline__ void unpack(const V& v, float (&f)[4]) {
    const T2 a = *reinterpret_cast<const T2*>(&v.x), b = *reinterpret_cast<const T2*>(&v.y);
    f[0] = to_f32<T>(a.x), f[1] = to_f32<T>(a.y), f[2] = to_f32<T>(b.x), f[3] = to_f32<T>(b.y);
  }
  static __device__ __forceinline__ V pack(const float (&f)[4]) {
    T2 a, b;
    a.x = from_f32<T>(f[0]), a.y = from_f32<T>(f[1]), b.x = from_f32<T>(f[2]), b.y = from_f32<T>(f[3]);
    return make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
  }
};
template <>
struct Quad<__half> : Quad16<__half, __half2> {};
template <>
struct Quad<__nv_bfloat16> : Quad16<__nv_bfloat16, __nv_bfloat162> {};

// Elements e .. e + 3 of a tensor of n; vec: the tensor's arrays are 16-byte aligned.
template <typename T>
__device__ __forceinline__ void load4(const void* base, long long e, long long n, bool vec, float (&f)[4]) {
  const T* p = static_cast<const T*>(base) + e;
  if (vec && e + 4 <= n) {
    Quad<T>::unpack(*reinterpret_cast<const typename Quad<T>::V*>(p), f);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = e + j < n ? to_f32<T>(p[j]) : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void store4(void* base, long long e, long long n, bool vec, const float (&f)[4]) {
  T* p = static_cast<T*>(base) + e;
  if (vec && e + 4 <= n) {
    *reinterpret_cast<typename Quad<T>::V*>(p) = Quad<T>::pack(f);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e + j < n) p[j] = from_f32<T>(f[j]);
  }
}

__device__ __forceinline__ uint32_t load_codes(const void* base, long long e, long long n, bool vec) {
  const uint8_t* p = static_cast<const uint8_t*>(base) + e;
  if (vec && e + 4 <= n) return *reinterpret_cast<const uint32_t*>(p);
  uint32_t w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (e + j < n) w |= (uint32_t)p[j] << (8 * j);
  return w;
}

__device__ __forceinline__ void store_codes(void* base, long long e, long long n, bool vec, uint32_t w) {
  uint8_t* p = static_cast<uint8_t*>(base) + e;
  if (vec && e + 4 <= n) {
    *reinterpret_cast<uint32_t*>(p) = w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (e + j < n) p[j] = (uint8_t)(w >> (8 * j));
  }
}

// The value that code c stands for under scale s: first moment, or root of the second.
__device__ __forceinline__ float first_value(uint32_t w, int j, float s) {
  const int c = (int)(int8_t)(w >> (8 * j));
  return __fmul_rn((float)(c * abs(c)), s);
}
__device__ __forceinline__ float root_value(uint32_t w, int j, float s) {
  const int c = (int)((w >> (8 * j)) & 0xFFu);
  return __fmul_rn((float)(c * c), s);
}

// Scale of a block whose largest magnitude has these bits, and its reciprocal. A largest magnitude too small
// for a normal scale codes the block as zeros; an infinite or NaN one gives a NaN scale, which decodes as NaN.
__device__ __forceinline__ float block_scale(uint32_t amax_bits, float over, float& inv) {
  const float s = __fmul_rn(__uint_as_float(amax_bits), over);
  inv = 0.0f;
  if (amax_bits >= 0x7F800000u) return __uint_as_float(0x7FC00000u);
  if (s < 1.17549435e-38f) return 0.0f;
  inv = __frcp_rn(s);
  return s;
}

__device__ __forceinline__ uint32_t code_of(float magnitude, float inv, int top) {
  return (uint32_t)min(__float2int_rn(__fsqrt_rn(__fmul_rn(magnitude, inv))), top);
}

// Four int8 codes (as offset binary) or uint8 codes as floats: the bytes become the low end of 2^23 + u.
__device__ __forceinline__ float code_float(uint32_t w, int j, float offset) {
  return __uint_as_float(prmt(w, 0x4B000000u, 0x7650u & ~0xFu | (uint32_t)j)) - offset;
}

__device__ __forceinline__ float root_approx(float x) {
  float r;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ float reciprocal_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

__device__ __forceinline__ uint32_t low_bytes(float a, float b, float c, float d) {
  const uint32_t lo = prmt(__float_as_uint(a), __float_as_uint(b), 0x0040u);
  const uint32_t hi = prmt(__float_as_uint(c), __float_as_uint(d), 0x0040u);
  return prmt(lo, hi, 0x5410u);
}

constexpr float kRound = 12582912.0f;  // 1.5 * 2^23: adding it rounds to a whole number, whose low byte is the code
// How near the middle between two codes a root may come before it is taken exactly. An approximate root is off by 2^-23
// of itself: a first moment's (up to 127) differs from the exact one by at most 1.5 * 2^-23, a second's (up to 255),
// which is a root of a scaled root, by 2.5 * 2^-23, so by 2.3e-5 and 7.6e-5.
constexpr float kNearFirst = 0.5f - 3e-5f, kNearSecond = 0.5f - 9e-5f;

// m and v of one element after the step
__device__ __forceinline__ void moments(const Args& a, float g, float& m, float& v) {
  m = __fadd_rn(__fmul_rn(m, a.beta1), __fmul_rn(g, a.one_minus_beta1));
  v = __fadd_rn(__fmul_rn(v, a.beta2), __fmul_rn(__fmul_rn(g, g), a.one_minus_beta2));
}

__device__ __forceinline__ float moved(const Args& a, float p, float m, float root) {
  return p * a.decay - a.step_size * (m / (root * a.root_scale + a.eps));
}

// The exact codes of four elements (first moments as int8, roots as uint8).
__device__ __forceinline__ void exact_codes(const float (&m)[4], const float (&root)[4], float mi, float vi,
                                            uint32_t& mw, uint32_t& vw) {
  mw = vw = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = (int)code_of(fabsf(m[j]), mi, 127);
    mw |= ((uint32_t)(m[j] < 0.0f ? -c : c) & 0xFFu) << (8 * j);
    uint32_t d = code_of(root[j], vi, 255);
    if (vi > 0.0f && root[j] > 0.0f && d == 0) d = 1;
    vw |= d << (8 * j);
  }
}

// One lane's eight elements (e .. e + 3 and e + 128 .. e + 131) of a full block, every root correctly rounded: read again
// from memory, which the lane has not written yet, so that the usual path holds less.
template <typename P, typename G>
__device__ __noinline__ void exact_lane(const Args& a, const AdamwTensor& t, long long e, float ms, float vs, float mi,
                                        float vi, float gs) {
#pragma unroll 1
  for (int h = 0; h < 2; ++h, e += 128) {
    float p[4], g[4], m[4], v[4];
    load4<P>(t.p, e, t.n, true, p);
    load4<G>(t.g, e, t.n, true, g);
    uint32_t mw = load_codes(t.m, e, t.n, true), vw = load_codes(t.v, e, t.n, true);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      m[j] = first_value(mw, j, ms);
      const float r = root_value(vw, j, vs);
      v[j] = __fmul_rn(r, r);
      moments(a, __fmul_rn(g[j], gs), m[j], v[j]);
      v[j] = __fsqrt_rn(v[j]);
      p[j] = moved(a, p[j], m[j], v[j]);
    }
    exact_codes(m, v, mi, vi, mw, vw);
    store4<P>(t.p, e, t.n, true, p);
    store_codes(t.m, e, t.n, true, mw);
    store_codes(t.v, e, t.n, true, vw);
  }
}

// A block of 256 whose elements all exist and whose arrays are aligned, 8-bit moments.
template <typename P, typename G>
__device__ __forceinline__ void full_block8(const Args& a, const AdamwTensor& t, long long b, int lane, float gs) {
  const long long e = b * kBlock + lane * 4;
  typename Quad<P>::V pv[2];
  typename Quad<G>::V gv[2];
  uint32_t mc[2], vc[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pv[h] = *reinterpret_cast<const typename Quad<P>::V*>(static_cast<const P*>(t.p) + e + 128 * h);
    gv[h] = *reinterpret_cast<const typename Quad<G>::V*>(static_cast<const G*>(t.g) + e + 128 * h);
    mc[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(t.m) + e + 128 * h);
    vc[h] = *reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(t.v) + e + 128 * h);
  }
  const float ms = t.m_scale[b], vs = t.v_scale[b];
  float m[2][4], root[2][4];
  uint32_t mb = 0, vb = 0;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float g[4];
    Quad<G>::unpack(gv[h], g);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float c = code_float(mc[h] ^ 0x80808080u, j, 8388736.0f), d = code_float(vc[h], j, 8388608.0f);
      const float r = __fmul_rn(d * d, vs);
      float v = __fmul_rn(r, r);
      m[h][j] = __fmul_rn(c * fabsf(c), ms);
      moments(a, __fmul_rn(g[j], gs), m[h][j], v);
      mb = max(mb, __float_as_uint(m[h][j]) & 0x7FFFFFFFu);
      vb = max(vb, __float_as_uint(v));
      root[h][j] = root_approx(v);
    }
  }
  mb = __reduce_max_sync(0xFFFFFFFFu, mb);
  vb = __reduce_max_sync(0xFFFFFFFFu, vb);  // of the values: the root of the largest is the largest root
  float mi, vi;
  const float ms1 = block_scale(mb, 1.0f / 16129.0f, mi);
  const float vs1 = block_scale(__float_as_uint(__fsqrt_rn(__uint_as_float(vb))), 1.0f / 65025.0f, vi);
  float least = kRound + 1.0f;  // the smallest second-moment code: 0 (a vanishing root) goes the exact way
  float far_m = 0.0f, far_v = 0.0f;  // the largest distances of the roots from their codes
  uint32_t mw[2], vw[2];
  typename Quad<P>::V out[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float r[4], q[4], p[4];
    Quad<P>::unpack(pv[h], p);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = copysignf(root_approx(fabsf(m[h][j]) * mi), m[h][j]), y = root_approx(root[h][j] * vi);
      r[j] = x + kRound, q[j] = y + kRound;
      far_m = fmaxf(far_m, fabsf(x - (r[j] - kRound)));
      far_v = fmaxf(far_v, fabsf(y - (q[j] - kRound)));
      least = fminf(least, q[j]);
      p[j] = p[j] * a.decay - a.step_size * (m[h][j] * reciprocal_approx(root[h][j] * a.root_scale + a.eps));
    }
    mw[h] = low_bytes(r[0], r[1], r[2], r[3]);
    vw[h] = low_bytes(q[0], q[1], q[2], q[3]);
    out[h] = Quad<P>::pack(p);
  }
  const bool exactly =
      !(far_m < kNearFirst) || !(far_v < kNearSecond) || !(least > kRound) || mi == 0.0f || vi == 0.0f;
  if (!exactly) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      *reinterpret_cast<typename Quad<P>::V*>(static_cast<P*>(t.p) + e + 128 * h) = out[h];
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(t.m) + e + 128 * h) = mw[h];
      *reinterpret_cast<uint32_t*>(static_cast<uint8_t*>(t.v) + e + 128 * h) = vw[h];
    }
  }
  if (lane == 0) {
    t.m_scale[b] = ms1;
    t.v_scale[b] = vs1;
  }
  if (exactly) exact_lane<P, G>(a, t, e, ms, vs, mi, vi, gs);
}

// The same with 32-bit moments.
template <typename P, typename G>
__device__ __forceinline__ void full_block32(const Args& a, const AdamwTensor& t, long long b, int lane, float gs) {
  const long long e = b * kBlock + lane * 4;
  typename Quad<P>::V pv[2];
  typename Quad<G>::V gv[2];
  float4 mv[2], vv[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    pv[h] = *reinterpret_cast<const typename Quad<P>::V*>(static_cast<const P*>(t.p) + e + 128 * h);
    gv[h] = *reinterpret_cast<const typename Quad<G>::V*>(static_cast<const G*>(t.g) + e + 128 * h);
    mv[h] = *reinterpret_cast<const float4*>(static_cast<const float*>(t.m) + e + 128 * h);
    vv[h] = *reinterpret_cast<const float4*>(static_cast<const float*>(t.v) + e + 128 * h);
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float p[4], g[4], m[4], v[4];
    Quad<P>::unpack(pv[h], p);
    Quad<G>::unpack(gv[h], g);
    Quad<float>::unpack(mv[h], m);
    Quad<float>::unpack(vv[h], v);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      moments(a, __fmul_rn(g[j], gs), m[j], v[j]);
      p[j] = moved(a, p[j], m[j], __fsqrt_rn(v[j]));
    }
    *reinterpret_cast<float4*>(static_cast<float*>(t.m) + e + 128 * h) = Quad<float>::pack(m);
    *reinterpret_cast<float4*>(static_cast<float*>(t.v) + e + 128 * h) = Quad<float>::pack(v);
    *reinterpret_cast<typename Quad<P>::V*>(static_cast<P*>(t.p) + e + 128 * h) = Quad<P>::pack(p);
  }
}

// A block that ends a tensor, or whose arrays are not aligned.
template <typename P, typename G, bool k8>
__device__ __noinline__ void ragged_block(const Args& a, const AdamwTensor& t, long long b, int lane, float gs) {
  const long long n = t.n;
  const bool vec = t.aligned != 0;
  float m[2][4], v[2][4];
  const float ms = k8 ? t.m_scale[b] : 0.0f, vs = k8 ? t.v_scale[b] : 0.0f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const long long e = b * kBlock + h * 128 + lane * 4;
    float p[4], g[4];
    load4<P>(t.p, e, n, vec, p);
    load4<G>(t.g, e, n, vec, g);
    if constexpr (k8) {
      const uint32_t mw = load_codes(t.m, e, n, vec), vw = load_codes(t.v, e, n, vec);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        m[h][j] = first_value(mw, j, ms);
        const float r = root_value(vw, j, vs);
        v[h][j] = __fmul_rn(r, r);
      }
    } else {
      load4<float>(t.m, e, n, vec, m[h]);
      load4<float>(t.v, e, n, vec, v[h]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) moments(a, __fmul_rn(g[j], gs), m[h][j], v[h][j]);
    if constexpr (!k8) {
      store4<float>(t.m, e, n, vec, m[h]);
      store4<float>(t.v, e, n, vec, v[h]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      v[h][j] = __fsqrt_rn(v[h][j]);
      p[j] = moved(a, p[j], m[h][j], v[h][j]);
    }
    store4<P>(t.p, e, n, vec, p);
  }
  if constexpr (k8) {
    uint32_t mb = 0, vb = 0;
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        mb = max(mb, __float_as_uint(m[h][j]) & 0x7FFFFFFFu);
        vb = max(vb, __float_as_uint(v[h][j]) & 0x7FFFFFFFu);
      }
    mb = __reduce_max_sync(0xFFFFFFFFu, mb);
    vb = __reduce_max_sync(0xFFFFFFFFu, vb);
    float mi, vi;
    const float ms1 = block_scale(mb, 1.0f / 16129.0f, mi), vs1 = block_scale(vb, 1.0f / 65025.0f, vi);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const long long e = b * kBlock + h * 128 + lane * 4;
      uint32_t mw, vw;
      exact_codes(m[h], v[h], mi, vi, mw, vw);
      store_codes(t.m, e, n, vec, mw);
      store_codes(t.v, e, n, vec, vw);
    }
    if (lane == 0) {
      t.m_scale[b] = ms1;
      t.v_scale[b] = vs1;
    }
  }
}

// Blocks an SM, 8-bit moments: six with 16-bit parameters and gradients (151 M elements 441 us; five 494, four 534),
// five where they are float32 (9 M elements 47 us; six spill and take 50).
template <typename P, typename G, bool k8>
__global__ void __launch_bounds__(kWarps * 32, k8 ? (sizeof(P) + sizeof(G) == 4 ? 6 : 5) : 4) adamw_kernel(const __grid_constant__ Args a) {
  // the tensor of this CTA: the last whose first CTA is not past it
  int lo = 0, hi = a.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.t[mid].first_cta <= (int)blockIdx.x) lo = mid; else hi = mid - 1;
  }
  const AdamwTensor& t = a.t[lo];
  const long long n = t.n, blocks = (n + kBlock - 1) / kBlock;
  const long long b0 = (long long)((int)blockIdx.x - t.first_cta) * a.blocks_per_cta;
  const long long b1 = b0 + a.blocks_per_cta < blocks ? b0 + a.blocks_per_cta : blocks;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  pdl_trigger();
  pdl_wait();
  const float gs = a.grad_scale != nullptr ? *a.grad_scale : 1.0f;
  for (long long b = b0 + warp; b < b1; b += kWarps) {
    if (t.aligned != 0 && (b + 1) * kBlock <= n) {
      if constexpr (k8) full_block8<P, G>(a, t, b, lane, gs);
      else full_block32<P, G>(a, t, b, lane, gs);
    } else {
      ragged_block<P, G, k8>(a, t, b, lane, gs);
    }
  }
}

// The values that 8-bit moments stand for (second: codes are roots, the value is squared).
template <bool kSecond>
__global__ void __launch_bounds__(kWarps * 32) moment_values_kernel(const void* codes, const float* scale, float* out,
                                                                    long long n, int vec) {
  const int lane = threadIdx.x & 31;
  const long long blocks = (n + kBlock - 1) / kBlock;
  constexpr int kAhead = 4;  // blocks whose codes are in flight at once
  pdl_trigger();
  pdl_wait();
  const long long stride = (long long)gridDim.x * kWarps;
  for (long long b = (long long)blockIdx.x * kWarps + (threadIdx.x >> 5); b < blocks; b += kAhead * stride) {
    uint32_t w[kAhead][2];
    float s[kAhead];
#pragma unroll
    for (int q = 0; q < kAhead; ++q) {
      const long long bq = b + q * stride;
      s[q] = bq < blocks ? scale[bq] : 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) w[q][h] = load_codes(codes, bq * kBlock + h * 128 + lane * 4, n, vec != 0);
    }
#pragma unroll
    for (int q = 0; q < kAhead; ++q)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float f[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          f[j] = kSecond ? root_value(w[q][h], j, s[q]) : first_value(w[q][h], j, s[q]);
          if (kSecond) f[j] = __fmul_rn(f[j], f[j]);
        }
        store4<float>(out, (b + q * stride) * kBlock + h * 128 + lane * 4, n, vec != 0, f);
      }
  }
}

}  // namespace adamw

template <typename P, typename G>
static int launch_adamw_t(const adamw::Args& a, bool bits8, int ctas, cudaStream_t st) {
  if (bits8)
    launch_overlapped(adamw::adamw_kernel<P, G, true>, dim3(ctas), adamw::kWarps * 32, st, a);
  else
    launch_overlapped(adamw::adamw_kernel<P, G, false>, dim3(ctas), adamw::kWarps * 32, st, a);
  return check_launch("adamw_kernel");
}

template <typename P>
static int launch_adamw_g(int g_dtype, const adamw::Args& a, bool bits8, int ctas, cudaStream_t st) {
  if (g_dtype == GFX_DTYPE_F32) return launch_adamw_t<P, float>(a, bits8, ctas, st);
  if (g_dtype == GFX_DTYPE_F16) return launch_adamw_t<P, __half>(a, bits8, ctas, st);
  return launch_adamw_t<P, __nv_bfloat16>(a, bits8, ctas, st);
}

int launch_adamw(const AdamwTensor* tensors, int count, int p_dtype, int g_dtype, bool bits8, const AdamwScalars& c,
                 cudaStream_t st, int sms) {
  adamw::Args a;
  a.grad_scale = c.grad_scale;
  a.beta1 = c.beta1, a.one_minus_beta1 = c.one_minus_beta1, a.beta2 = c.beta2, a.one_minus_beta2 = c.one_minus_beta2;
  a.decay = c.decay, a.step_size = c.step_size, a.root_scale = c.root_scale, a.eps = c.eps;
  // one 256-element block a warp where that is needed to fill the GPU, up to four, which amortise a CTA's start (with
  // one, 151 M elements took 584 us with 32-bit moments instead of 492, some of it for branches that are gone since)
  long long all = 0;
  for (int i = 0; i < count; ++i) all += (tensors[i].n + adamw::kBlock - 1) / adamw::kBlock;
  const long long per_warp = all / ((long long)sms * 48);
  a.blocks_per_cta = adamw::kWarps * (int)(per_warp < 1 ? 1 : (per_warp > 4 ? 4 : per_warp));
  for (int i = 0; i < count;) {
    // as many tensors as one launch's arguments hold; empty ones take no CTA
    a.count = 0;
    long long ctas = 0;
    for (; i < count && a.count < kAdamwMaxTensors; ++i) {
      const long long blocks = (tensors[i].n + adamw::kBlock - 1) / adamw::kBlock;
      if (blocks == 0) continue;
      const long long need = (blocks + a.blocks_per_cta - 1) / a.blocks_per_cta;
      if (ctas + need > 0x7FFFFFFFll) break;  // the grid's limit: the rest goes into the next launch
      a.t[a.count] = tensors[i];
      a.t[a.count].first_cta = (int)ctas;
      ++a.count;
      ctas += need;
    }
    if (a.count == 0) continue;
    int rc;
    if (p_dtype == GFX_DTYPE_F32)
      rc = launch_adamw_g<float>(g_dtype, a, bits8, (int)ctas, st);
    else if (p_dtype == GFX_DTYPE_F16)
      rc = launch_adamw_g<__half>(g_dtype, a, bits8, (int)ctas, st);
    else
      rc = launch_adamw_g<__nv_bfloat16>(g_dtype, a, bits8, (int)ctas, st);
    if (rc) return rc;
  }
  return GFX_OK;
}

int launch_moment_values(const void* codes, const float* scale, float* out, long long n, int second, int vec,
                         cudaStream_t st, int sms) {
  const long long need = ((n + adamw::kBlock - 1) / adamw::kBlock + adamw::kWarps - 1) / adamw::kWarps;
  const int ctas = (int)(need < (long long)sms * 8 ? need : (long long)sms * 8);
  if (second)
    launch_overlapped(adamw::moment_values_kernel<true>, dim3(ctas), adamw::kWarps * 32, st, codes, scale, out, n, vec);
  else
    launch_overlapped(adamw::moment_values_kernel<false>, dim3(ctas), adamw::kWarps * 32, st, codes, scale, out, n, vec);
  return check_launch("moment_values_kernel");
}

}  // namespace gfx
