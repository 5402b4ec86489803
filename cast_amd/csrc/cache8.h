// A paged cache in 8 bits: codes c of a block of tokens and head with a scale s stand for
// c * s.
//
// Codes are int8 in [-127, 127] or e4m3 (1 sign, 4 exponent and 3 mantissa bits, up to 448).
// A block's tokens follow each other in one page; page j / page of a request's table holds
// key j in row j % page, and that row's block is row / block.
#pragma once
#include "rcsa_common.h"

namespace rcsa {

// The smallest scale: blocks of zeros, and values that fp32 scales could not hold.
constexpr float kLeastScale = 0x1p-100f;
constexpr int64_t kMostSlots = 1ll << 30;  // of a request's table

template <bool E4M3>
struct Code8;

template <>
struct Code8<false> {
  // The scale of a block whose largest value is `most`: most / 127, rounded to fp32.
  static __device__ __forceinline__ float scale_for(float most) { return most / 127.0f; }
  // The codes nearest x / s, ties to even.  x * inv is off by 2^-23 of it, so that the whole
  // number next to it is the quotient's or one beside; the remainder x - q s is exact (fp32
  // values on a grid no finer than half of s's last place, below 2^24 steps of it), so that
  // comparing it with s / 2 decides as the real quotient would.  Infinities saturate, NaN
  // becomes 0.
  struct To {
    float s, inv, half;
    __device__ __forceinline__ To(float scale) : s(scale), inv(1.0f / scale), half(0.5f * scale) {}
    __device__ __forceinline__ int one(float x) const {
      float q = __builtin_rintf(x * inv);
      q = fminf(fmaxf(q, -127.0f), 127.0f);
      const float r = fmaf(-q, s, x), far = fabsf(r);
      const int c = static_cast<int>(q);
      const bool move = far > half || (far == half && (c & 1));
      int d = c + (move ? (r < 0.0f ? -1 : 1) : 0);
      d = d > 127 ? 127 : (d < -127 ? -127 : d);
      return x == x ? d : 0;
    }
    __device__ __forceinline__ uint32_t four(const float* x) const {
      return (one(x[0]) & 255) | (one(x[1]) & 255) << 8 | (one(x[2]) & 255) << 16 |
             static_cast<uint32_t>(one(x[3])) << 24;
    }
  };
  static __device__ __forceinline__ void values(uint32_t w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24);
  }
  // Codes c as the codes nearest c s0 / s, ties to even, for s0 <= s.  (fp64: c s0 is exact
  // there, and a quotient that is not halfway between two codes is 2^-32 of it away.)
  static __device__ __forceinline__ uint32_t again(uint32_t w, float s0, float s) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int c = static_cast<int>(w << (24 - 8 * i)) >> 24;
      const double y = __builtin_rint(static_cast<double>(c) * s0 / s);
      out |= (static_cast<uint32_t>(static_cast<int>(y)) & 255u) << (8 * i);
    }
    return out;
  }
};

template <>
struct Code8<true> {
  // The smallest power of two p with most <= 448 p (448 = 1.75 * 2^8).
  static __device__ __forceinline__ float scale_for(float most) {
    const uint32_t u = __float_as_uint(most);
    const int e = static_cast<int>(u >> 23) - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    return e < 1 ? 0.0f : __uint_as_float(static_cast<uint32_t>(e) << 23);
  }
  // x / s rounded to the type's values, ties to even; infinities saturate, NaN becomes 0.
  // Scales that are powers of two (scale_for's) are divided by exactly with their
  // reciprocal, others by a division, rounded once before the type.
  struct To {
    float s, inv;
    bool power;
    __device__ __forceinline__ To(float scale)
        : s(scale), inv(1.0f / scale), power((__float_as_uint(scale) & 0x7fffffu) == 0) {}
    __device__ __forceinline__ float one(float x) const {
      const float y = power ? x * inv : x / s;
      const float z = fminf(fmaxf(y, -448.0f), 448.0f);
      return x == x ? z : 0.0f;
    }
    __device__ __forceinline__ uint32_t four(const float* x) const {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(one(x[0]), one(x[1]), 0, false);
      return static_cast<uint32_t>(
          __builtin_amdgcn_cvt_pk_fp8_f32(one(x[2]), one(x[3]), lo, true));
    }
  };
  static __device__ __forceinline__ void values(uint32_t w, float* x) {
    const int v = static_cast<int>(w);
    x[0] = __builtin_amdgcn_cvt_f32_fp8(v, 0);
    x[1] = __builtin_amdgcn_cvt_f32_fp8(v, 1);
    x[2] = __builtin_amdgcn_cvt_f32_fp8(v, 2);
    x[3] = __builtin_amdgcn_cvt_f32_fp8(v, 3);
  }
  static __device__ __forceinline__ uint32_t again(uint32_t w, float s0, float s) {
    float x[4];
    values(w, x);
    const double f = static_cast<double>(s0) / s;  // (a power of two, of scale_for's)
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(x[i] * f);
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], lo, true));
  }
};

// Eight consecutive values of a tensor of type T as fp32, and back (rounded once).
template <typename T>
struct Run8 {
  typedef T V __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ void floats(const V& v, float* x) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = static_cast<float>(v[i]);
  }
  static __device__ __forceinline__ V of(const float* x) {
    V v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = static_cast<T>(x[i]);
    return v;
  }
};

}  // namespace rcsa
