// Device helpers of the dense operators: element types, the three-plane form of fp32, activations.
#pragma once
#include "dense.h"

namespace scl {

__host__ __device__ constexpr int64_t round_up8(int64_t x) { return (x + 7) & ~(int64_t)7; }

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
struct __attribute__((packed, aligned(2))) u16x8_any { unsigned short v[8]; };  // 16 bytes at any element address
struct __attribute__((packed, aligned(4))) f32x8_any { float v[8]; };

__device__ __forceinline__ float bf16_to_f32(unsigned short h) { return __uint_as_float((unsigned)h << 16); }
__device__ __forceinline__ unsigned short f32_to_bf16(float v) {  // round to nearest, ties to even; NaN stays NaN
  return __builtin_bit_cast(unsigned short, (__bf16)v);
}
__device__ __forceinline__ float f16_to_f32(unsigned short h) { return (float)__builtin_bit_cast(_Float16, h); }
__device__ __forceinline__ unsigned short f32_to_f16(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }

// v = p0 + p1 + p2 exactly, each piece a bf16: p0 is v rounded to 8 bits, the remainder (exact in fp32, at most 2^-8 |v|) gives p1,
// the next one (at most 8 bits left) is p2. Infinities and NaN sit in p0 alone. A v that would round up to infinity is cut instead. Below 2^-110
// (1e-33) the last bits fall under bf16's smallest step, 2^-133: fp32 products of such values lose them where they run in planes (relative
// error 4e-5 at 2^-120).
__device__ __forceinline__ void split3(float v, unsigned short& p0, unsigned short& p1, unsigned short& p2) {
  const unsigned u = __float_as_uint(v);
  if ((u & 0x7f800000u) == 0x7f800000u) {
    p0 = f32_to_bf16(v);
    p1 = p2 = 0;
    return;
  }
  p0 = f32_to_bf16(v);
  if ((p0 & 0x7f80u) == 0x7f80u) p0 = (unsigned short)(u >> 16);
  const float r1 = v - bf16_to_f32(p0);
  p1 = f32_to_bf16(r1);
  p2 = f32_to_bf16(r1 - bf16_to_f32(p1));
}

template <int T> struct Elem;  // 16-bit and fp32 elements
template <> struct Elem<D_F32> {
  typedef float type;
  static __device__ __forceinline__ float ld(const float* p) { return *p; }
  static __device__ __forceinline__ void st(float* p, float v) { *p = v; }
};
template <> struct Elem<D_BF16> {
  typedef unsigned short type;
  static __device__ __forceinline__ float ld(const unsigned short* p) { return bf16_to_f32(*p); }
  static __device__ __forceinline__ void st(unsigned short* p, float v) { *p = f32_to_bf16(v); }
};
template <> struct Elem<D_F16> {
  typedef unsigned short type;
  static __device__ __forceinline__ float ld(const unsigned short* p) { return f16_to_f32(*p); }
  static __device__ __forceinline__ void st(unsigned short* p, float v) { *p = f32_to_f16(v); }
};

// eight consecutive elements at off (elements from m.p); `n` of them are inside the matrix (the rest read as 0 / are not written,
// or, for an image of the library (m.pad), are written as zeros by the caller passing n = 8)
template <int T>
__device__ __forceinline__ void load8(const Mat& m, int64_t off, int n, float v[8]) {
  if constexpr (T == D_PL3) {
    const unsigned short* p = static_cast<const unsigned short*>(m.p) + off;
    const u16x8 a = *reinterpret_cast<const u16x8*>(p), b = *reinterpret_cast<const u16x8*>(p + m.plane),
                c = *reinterpret_cast<const u16x8*>(p + 2 * m.plane);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (bf16_to_f32(a[e]) + bf16_to_f32(b[e])) + bf16_to_f32(c[e]);
  } else {
    typedef typename Elem<T>::type E;
    const E* p = static_cast<const E*>(m.p) + off;
    if (n >= 8 && m.vec) {
      if constexpr (T == D_F32) {
        const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
      } else {
        const u16x8 a = *reinterpret_cast<const u16x8*>(p);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const unsigned short h = a[e];
          v[e] = Elem<T>::ld(&h);
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = e < n ? Elem<T>::ld(p + e) : 0.f;
    }
  }
}
// the same in two halves: the loads now, the values later
template <int T>
struct Raw8 {
  static constexpr int NV = T == D_PL3 ? 3 : (T == D_F32 ? 2 : 1);
  u16x8 r[NV];
  __device__ __forceinline__ void load(const Mat& m, int64_t off, int n) {
    if constexpr (T == D_PL3) {
      const unsigned short* p = static_cast<const unsigned short*>(m.p) + off;
#pragma unroll
      for (int i = 0; i < 3; ++i) r[i] = *reinterpret_cast<const u16x8*>(p + i * m.plane);
    } else {
      typedef typename Elem<T>::type E;
      const E* p = static_cast<const E*>(m.p) + off;
      if (n >= 8 && m.vec) {
#pragma unroll
        for (int i = 0; i < NV; ++i) r[i] = reinterpret_cast<const u16x8*>(p)[i];
      } else {
        E v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : (E)0;
        __builtin_memcpy(r, v, sizeof(v));
      }
    }
  }
  __device__ __forceinline__ void get(float v[8]) const {
    if constexpr (T == D_PL3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = (bf16_to_f32(r[0][e]) + bf16_to_f32(r[1][e])) + bf16_to_f32(r[2][e]);
    } else if constexpr (T == D_F32) {
      __builtin_memcpy(v, r, 32);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const unsigned short h = r[0][e];
        v[e] = Elem<T>::ld(&h);
      }
    }
  }
};
template <int T>
__device__ __forceinline__ void store8(const Mat& m, int64_t off, int n, const float v[8]) {
  if constexpr (T == D_PL3) {
    unsigned short* p = static_cast<unsigned short*>(m.p) + off;
    u16x8 a, b, c;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      unsigned short x, y, z;
      split3(v[e], x, y, z);
      a[e] = x; b[e] = y; c[e] = z;
    }
    *reinterpret_cast<u16x8*>(p) = a;
    *reinterpret_cast<u16x8*>(p + m.plane) = b;
    *reinterpret_cast<u16x8*>(p + 2 * m.plane) = c;
  } else {
    typedef typename Elem<T>::type E;
    E* p = static_cast<E*>(m.p) + off;
    if (n >= 8 && m.vec) {
      if constexpr (T == D_F32) {
        f32x4 a = {v[0], v[1], v[2], v[3]}, b = {v[4], v[5], v[6], v[7]};
        *reinterpret_cast<f32x4*>(p) = a;
        *reinterpret_cast<f32x4*>(p + 4) = b;
      } else {
        u16x8 a;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          unsigned short h;
          Elem<T>::st(&h, v[e]);
          a[e] = h;
        }
        *reinterpret_cast<u16x8*>(p) = a;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) Elem<T>::st(p + e, v[e]);
    }
  }
}

// Activations and their derivatives in fp32 (the value is rounded once, when it is stored). 1 / (1 + e^-v) and the normal tail are
// written out on the hardware's exp2 and reciprocal (one unit each): with erff and a division the epilogue of a 256 x 256 tile cost as
// much as eight of its stages.
__device__ __forceinline__ float sigmoid(float v) { return __builtin_amdgcn_rcpf(1.f + __expf(-v)); }
// erfc(x) / 2 for x = |z| / sqrt(2): e^(-x^2) t P(t), t = 1 / (1 + 0.3 x). P is the polynomial of degree 8 of least largest relative
// error on 0 <= x <= 10 (3e-8 with these coefficients); *e gets e^(-z^2 / 2). In fp32 the relative error is 5e-7 for |z| up to 2 and grows with the
// exponent, whose rounding it is: 2e-6 at 6, 7e-6 at 13, where the tail itself is 1e-9 and 1e-38.
__device__ __forceinline__ float normal_tail(float az, float* e) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3f * 0.70710678f, az, 1.f));
  *e = __expf(-0.5f * az * az);
  float p = -0.12952275f;
  p = fmaf(p, t, 0.48556247f);
  p = fmaf(p, t, -0.51227657f);
  p = fmaf(p, t, 0.54771831f);
  p = fmaf(p, t, -0.09464955f);
  p = fmaf(p, t, 0.21492557f);
  p = fmaf(p, t, 0.14833929f);
  p = fmaf(p, t, 0.17071521f);
  p = fmaf(p, t, 0.16918801f);
  return 0.5f * *e * t * p;
}
// At infinities the limits: z times a sigmoid that is zero, and z times 1 - sigmoid, are zero there and not NaN. (A saved fp16 argument of 65 520 is
// infinite already.) Nothing is clamped that is finite, and NaN stays NaN through the other factor.
constexpr float LARGEST = 3.40282347e38f;
// beyond 14 the tail is below 1e-43: the clamp keeps infinity times zero away
__device__ __forceinline__ float tail_arg(float z) { return fminf(fabsf(z), 14.f); }
template <int ACT>
__device__ __forceinline__ float act_apply(float z) {
  if constexpr (ACT == ACT_RELU) return z < 0.f ? 0.f : z;  // (NaN stays)
  if constexpr (ACT == ACT_SILU) return fmaxf(z, -LARGEST) * sigmoid(z);
  if constexpr (ACT == ACT_GELU) {
    float e;
    const float az = tail_arg(z), q = normal_tail(az, &e);
    return (z < 0.f ? 0.f : z) - az * q;
  }
  if constexpr (ACT == ACT_GELU_TANH) return fmaxf(z, -LARGEST) * sigmoid(1.5957691f * (z + 0.044715f * z * z * z));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_grad(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f ? 1.f : (z != z ? z : 0.f);
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid(z);
    return s * (1.f + __builtin_amdgcn_fmed3f(z, -LARGEST, LARGEST) * (1.f - s));
  }
  if constexpr (ACT == ACT_GELU) {
    float e;
    const float az = tail_arg(z), q = normal_tail(az, &e), zc = z != z ? z : fminf(fmaxf(z, -14.f), 14.f);
    return (z > 0.f ? 1.f - q : q) + zc * 0.39894228f * e;
  }
  if constexpr (ACT == ACT_GELU_TANH) {
    // from |z| = 12 the sigmoid is 0 or 1 to the last bit; z z, which overflows at 1.8e19, would meet 1 - s = 0
    z = z != z ? z : fminf(fmaxf(z, -12.f), 12.f);
    const float s = sigmoid(1.5957691f * (z + 0.044715f * z * z * z));
    return s + z * s * (1.f - s) * 1.5957691f * (1.f + 0.134145f * z * z);
  }
  return 1.f;
}
// eight at a time, the kind decided once
template <bool GRAD, int ACT>
__device__ __forceinline__ void act8_of(float v[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = GRAD ? act_grad<ACT>(v[e]) : act_apply<ACT>(v[e]);
}
template <bool GRAD>
__device__ __forceinline__ void act8(float v[8], int act) {
  switch (act) {
    case ACT_RELU: act8_of<GRAD, ACT_RELU>(v); break;
    case ACT_SILU: act8_of<GRAD, ACT_SILU>(v); break;
    case ACT_GELU: act8_of<GRAD, ACT_GELU>(v); break;
    case ACT_GELU_TANH: act8_of<GRAD, ACT_GELU_TANH>(v); break;
    default: act8_of<GRAD, ACT_NONE>(v);
  }
}

template <bool GRAD>
__device__ __forceinline__ float act_any(float z, int act) {
  switch (act) {
    case ACT_RELU: return GRAD ? act_grad<ACT_RELU>(z) : act_apply<ACT_RELU>(z);
    case ACT_SILU: return GRAD ? act_grad<ACT_SILU>(z) : act_apply<ACT_SILU>(z);
    case ACT_GELU: return GRAD ? act_grad<ACT_GELU>(z) : act_apply<ACT_GELU>(z);
    case ACT_GELU_TANH: return GRAD ? act_grad<ACT_GELU_TANH>(z) : act_apply<ACT_GELU_TANH>(z);
    default: return GRAD ? 1.f : z;
  }
}

}  // namespace scl
