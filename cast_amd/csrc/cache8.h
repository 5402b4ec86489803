// A paged cache in 8 bits: codes c of a block of tokens and head with a scale s stand for
// c * s.
//
// Codes are int8 in [-127, 127] or e4m3 (1 sign, 4 exponent and 3 mantissa bits, up to 448).
// A block's tokens follow each other in one page; page j / page of a request's table holds
// key j in row j % page, and that row's block is row / block.
#pragma once
#include <type_traits>

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
  // The codes nearest x / s, ties to even.  t = x * inv is off by 2^-23 of it, below 1.6e-5, so
  // that the whole number next to t is the quotient's unless t is that near the border of two
  // codes.  Where a lane has such a t (one value in 25000), the remainder x - q s decides: it
  // is exact (fp32 values on a grid no finer than half of s's last place, below 2^24 steps of
  // it).  t + 1.5 2^23 is t rounded, its code in the lowest byte.  Infinities saturate, NaN
  // becomes 0.
  struct To {
    float s, inv;
    __device__ __forceinline__ explicit To(float scale) : s(scale), inv(1.0f / scale) {}
    __device__ __forceinline__ int exactly(float x) const {
      const float half = 0.5f * s;
      const float q = fminf(fmaxf(__builtin_rintf(x * inv), -127.0f), 127.0f);
      const float r = fmaf(-q, s, x), far = fabsf(r);
      const int c = static_cast<int>(q);
      const bool move = far > half || (far == half && (c & 1));
      int d = c + (move ? (r < 0.0f ? -1 : 1) : 0);
      d = d > 127 ? 127 : (d < -127 ? -127 : d);
      return x == x ? d : 0;
    }
    // `plain`: no infinity or NaN among the values of the wavefront
    template <typename R>
    __device__ __forceinline__ uint2 eight(const typename R::V& v, bool plain) const {
      constexpr float kMagic = 12582912.0f;  // 1.5 * 2^23
      uint2 w = make_uint2(0u, 0u);
      if (!plain) {
#pragma unroll 1
        for (int i = 0; i < 4; ++i) {
          w.x |= static_cast<uint32_t>(exactly(static_cast<float>(v[i])) & 255) << (8 * i);
          w.y |= static_cast<uint32_t>(exactly(static_cast<float>(v[4 + i])) & 255) << (8 * i);
        }
        return w;
      }
      // (finite values only: |x / s| is 127 at most, but for roundings)
      uint32_t pair[4];
      auto pack = [](float u0, float u1) __attribute__((always_inline)) -> uint32_t {
        return __builtin_amdgcn_perm(__float_as_uint(u1), __float_as_uint(u0), 0x0c0c0400u);
      };
      float off = 0.0f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float t0 = static_cast<float>(v[2 * i]) * inv;
        const float t1 = static_cast<float>(v[2 * i + 1]) * inv;
        const float u0 = t0 + kMagic, u1 = t1 + kMagic;
        off = fmaxf(fmaxf(off, fabsf(t0 - (u0 - kMagic))), fabsf(t1 - (u1 - kMagic)));
        pair[i] = pack(u0, u1);
      }
      if (__ballot(off > 0.49998f) != 0) {
        auto near = [&](float x) __attribute__((always_inline)) -> float {
          const float u = fmaf(x, inv, kMagic);
          const float r = fmaf(kMagic - u, s, x), far = fabsf(r), half = 0.5f * s;
          const bool move = far > half || (far == half && (__float_as_uint(u) & 1u));
          return move ? u + (r < 0.0f ? -1.0f : 1.0f) : u;
        };
#pragma unroll
        for (int i = 0; i < 4; ++i)
          pair[i] = pack(near(static_cast<float>(v[2 * i])), near(static_cast<float>(v[2 * i + 1])));
      }
      w = make_uint2(__builtin_amdgcn_perm(pair[1], pair[0], 0x05040100u),
                     __builtin_amdgcn_perm(pair[3], pair[2], 0x05040100u));
      return w;
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
    __device__ __forceinline__ explicit To(float scale)
        : s(scale), inv(1.0f / scale), power((__float_as_uint(scale) & 0x7fffffu) == 0) {}
    static __device__ __forceinline__ uint32_t four(const float* y) {
      const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
      return static_cast<uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true));
    }
    template <typename R>
    __device__ __forceinline__ uint2 eight(const typename R::V& v, bool plain) const {
      float x[8];
      R::floats(v, x);
      float y[8];
      if (plain && power) {
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = x[i] * inv;  // (at most 448)
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float z = power ? x[i] * inv : x[i] / s;
          y[i] = x[i] == x[i] ? fminf(fmaxf(z, -448.0f), 448.0f) : 0.0f;
        }
      }
      return make_uint2(four(y), four(y + 4));
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
    return To::four(x);
  }
};

// Eight consecutive values of a tensor of type T as fp32, and back (rounded once); their
// largest size, which infinities and NaN exceed every number with, as bits of the type (fp32's
// its own).
template <typename T>
struct Run8 {
  typedef T V __attribute__((ext_vector_type(8), aligned(16)));
  static constexpr uint32_t kInfinity =
      std::is_same<T, __bf16>::value ? 0x7f80u : std::is_same<T, _Float16>::value ? 0x7c00u
                                                                                  : 0x7f800000u;
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
  // Of 16-bit types two running maxima in a word.
  static __device__ __forceinline__ void most(const V& v, uint32_t& m) {
    if constexpr (sizeof(T) == 2) {
      typedef unsigned short v2us __attribute__((ext_vector_type(2)));
      struct Words {
        uint32_t w[4];
      };
      const Words w = __builtin_bit_cast(Words, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const v2us a = __builtin_bit_cast(v2us, w.w[i] & 0x7fff7fffu);
        m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(a, __builtin_bit_cast(v2us, m)));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const uint32_t a = __float_as_uint(static_cast<float>(v[i])) & 0x7fffffffu;
        m = a > m ? a : m;
      }
    }
  }
  static __device__ __forceinline__ uint32_t larger(uint32_t a, uint32_t b) {
    return a > b ? a : b;
  }
  // The larger of a word's two (fp32: itself).
  static __device__ __forceinline__ uint32_t one_of(uint32_t m) {
    return sizeof(T) == 2 ? larger(m & 0xffffu, m >> 16) : m;
  }
  static __device__ __forceinline__ float value(uint32_t bits) {
    if constexpr (std::is_same<T, __bf16>::value) return __uint_as_float(bits << 16);
    else if constexpr (std::is_same<T, _Float16>::value)
      return static_cast<float>(__builtin_bit_cast(_Float16, static_cast<unsigned short>(bits)));
    else return __uint_as_float(bits);
  }
};

}  // namespace rcsa
