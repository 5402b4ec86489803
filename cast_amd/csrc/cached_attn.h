// Attention over pages of 8-bit codes: what the kernels of few rows (cached_units.hip) and
// of 128-row blocks (cached_tile.hip) share.
//
// Keys and values are codes c with a scale s for each block of tokens and head.  The matrix
// products take the codes as fp16 (exact: 8 bits or less), so that a logit is
//   (q . c_k) * s_k sm_scale,   out = sum_j w_j s_vj c_vj / sum_j w_j.
// Queries become fp16 with a power of two a row that brings its largest value to [2^14,
// 2^15): bf16 rows lose nothing down to 2^-29 of it, and 2^-39 of it at most below.
// A weight takes the scale of its value's block, relative to a power of two 2^e no smaller than
// any scale of the row's keys so far, before it is rounded to fp16; e grows with the tiles (the
// accumulators move by the difference), and the sums of weights know nothing of it.  A weight
// below 2^-32 of the largest, in a block whose scale is as large, is lost: values that
// differ by more than that between blocks give the smaller ones no more than fp32 sums would
// have left of them.
#pragma once
#include "window_attn.h"

namespace rcsa {

typedef _Float16 v2hf __attribute__((ext_vector_type(2)));

template <bool E4M3>
struct Widen;

template <>
struct Widen<false> {  // int8
  static constexpr int kShift = 9;  // columns() gives c 2^-9
  static __device__ __forceinline__ uint32_t tame(uint32_t w) { return w ^ 0x80808080u; }
  // c + 128 beneath the exponent of 1024, less 1152: exact
  static __device__ __forceinline__ v2hf pair(uint32_t tamed, bool hi) {
    const uint32_t p = hi ? __builtin_amdgcn_perm(0x64646464u, tamed, 0x04030402u)
                          : __builtin_amdgcn_perm(0x64646464u, tamed, 0x04010400u);
    return __builtin_bit_cast(v2hf, p) - static_cast<_Float16>(1152.0f);
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t w) { return w; }
};
template <>
struct Widen<true> {  // e4m3
  static constexpr int kShift = 0;
  static __device__ __forceinline__ uint32_t tame(uint32_t w) { return w; }
  static __device__ __forceinline__ v2hf pair(uint32_t w, bool hi) {
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, true)
              : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, false);
  }
  // Codes that hold no number (0x7f, 0xff) as 0: a weight of 0 would not hide them.
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    const uint32_t none = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~((none >> 7) * 255u);
  }
};

// Sixteen codes as two operands of eight.
template <bool E4M3>
__device__ __forceinline__ void widen16(v4i w, v8hf& lo, v8hf& hi) {
  using W = Widen<E4M3>;
  v2hf p[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t t = W::tame(static_cast<uint32_t>(w[i]));
    p[2 * i] = W::pair(t, false);
    p[2 * i + 1] = W::pair(t, true);
  }
  struct Two {
    v2hf p[8];
  };
  struct Ops {
    v8hf lo, hi;
  };
  Two two;
#pragma unroll
  for (int i = 0; i < 8; ++i) two.p[i] = p[i];
  const Ops o = __builtin_bit_cast(Ops, two);
  lo = o.lo;
  hi = o.hi;
}

// Column x of four words, byte by byte, as one word of four: column(x, w0 .. w3).
__device__ __forceinline__ uint32_t byte_column(int x, uint32_t w0, uint32_t w1, uint32_t w2,
                                                uint32_t w3) {
  const uint32_t s = 0x0c0c0400u + 0x0101u * static_cast<uint32_t>(x);
  const uint32_t lo = __builtin_amdgcn_perm(w1, w0, s);
  const uint32_t hi = __builtin_amdgcn_perm(w3, w2, s);
  return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// Byte x of eight (tamed) words as an operand of eight, times 2^-kShift.
template <bool E4M3>
__device__ __forceinline__ v8hf column8(int x, const uint32_t* w) {
  struct Four {
    v2hf p[4];
  };
  Four f;
  if constexpr (E4M3) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const uint32_t c = byte_column(x, w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
      f.p[2 * i] = Widen<true>::pair(c, false);
      f.p[2 * i + 1] = Widen<true>::pair(c, true);
    }
  } else {
    // a byte c + 128 alone is the subnormal (c + 128) 2^-24
    const uint32_t s = 0x0c040c00u + 0x00010001u * static_cast<uint32_t>(x);
    const v2hf up = {static_cast<_Float16>(32768.0f), static_cast<_Float16>(32768.0f)};
    const v2hf less = {static_cast<_Float16>(-0.25f), static_cast<_Float16>(-0.25f)};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f.p[i] = __builtin_elementwise_fma(
          __builtin_bit_cast(v2hf, __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], s)), up, less);
  }
  return __builtin_bit_cast(v8hf, f);
}

// 2^e of a normal number's exponent e.
__device__ __forceinline__ float power_of(int e) {
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

// Eight values of a query row as fp16 times `up`.
template <typename T>
__device__ __forceinline__ v8hf scaled8(typename Half<T>::op8 v, float up) {
  v8hf o;
#pragma unroll
  for (int i = 0; i < 8; ++i) o[i] = static_cast<_Float16>(static_cast<float>(v[i]) * up);
  return o;
}
// k with 2^14 <= most 2^k < 2^15, at most 100 (rows of zeros, and of no numbers: 0).
__device__ __forceinline__ int row_shift(float most) {
  if (!(most > 0.0f && most < INFINITY)) return 0;
  const int k = 14 - (static_cast<int>(__float_as_uint(most) >> 23) - 127);
  return k > 100 ? 100 : k;
}

// A step: its first key, and the pages of its two halves of 16 keys.
struct CodeStep {
  int key, page0, page1;
};
// The first row of a half in its page.
template <typename A>
__device__ __forceinline__ int slot_of(A& a, int key, int half) {
  const int k = (key < 0 ? 0 : key);
  const int slot = k - divide(k >> 4, a.by_half_page) * a.page;
  return half == 0 ? slot : (slot + 16 < a.page ? slot + 16 : 0);
}
template <typename A>
__device__ __forceinline__ CodeStep code_step(A& a, const Place& p, const int32_t* table, int s) {
  CodeStep r;
  r.key = key_of(p, s);
  const int key = r.key < 0 ? 0 : r.key;
  const int col = divide(key >> 4, a.by_half_page);
  r.page0 = ld_const(table + col);
  r.page1 = r.page0;
  if (!a.whole_tiles && key - col * a.page + 16 >= a.page)
    r.page1 = ld_const(table + (col + 1 < a.max_pages ? col + 1 : a.max_pages - 1));
  return r;
}
template <typename A>
__device__ __forceinline__ int halves_there(A& a, const CodeStep& s) {
  return (page_ok(a, s.page0) ? 1 : 0) + (page_ok(a, s.page1) ? 2 : 0);
}
// Where the first rows of a half of a step are (page 0's where it is not there: its codes are
// not seen, but read).  (32 x 32-bit products: a page spans less than 4 GiB.)
struct HalfAt {
  uint64_t k, v;
};
template <typename A>
__device__ __forceinline__ HalfAt half_at(A& a, const CodeStep& s, int half, uint32_t krb,
                                          uint32_t vrb) {
  const int pg = half ? s.page1 : s.page0;
  const uint32_t slot = static_cast<uint32_t>(slot_of(a, s.key, half));
  const uint32_t at = s.key >= 0 && page_ok(a, pg) ? static_cast<uint32_t>(pg) : 0u;
  return {static_cast<uint64_t>(at) * static_cast<uint32_t>(a.sk[0]) +
              static_cast<uint64_t>(slot) * krb,
          static_cast<uint64_t>(at) * static_cast<uint32_t>(a.sv[0]) +
              static_cast<uint64_t>(slot) * vrb};
}
// The scales of a step's two halves: of a page that is there, as the cache holds them if they are
// positive numbers below 2^126, else 0.  ks, vs: of the key head.
struct Scales {
  float k[2], v[2];
};
template <typename A>
__device__ __forceinline__ Scales scales_of(A& a, const CodeStep& s, const float* ks,
                                            const float* vs) {
  Scales r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int pg = h ? s.page1 : s.page0;
    const bool there = s.key >= 0 && page_ok(a, pg);
    const int mark = divide(slot_of(a, s.key, h) >> 4, a.by_half_mark);
    const int at = there ? pg : 0;
    const float k = ld_const(ks + (at * a.sks[0] + mark * a.sks[1]));
    const float v = ld_const(vs + (at * a.svs[0] + mark * a.svs[1]));
    r.k[h] = there && k > 0.0f && k < 0x1p126f ? k : 0.0f;
    r.v[h] = there && v > 0.0f && v < 0x1p126f ? v : 0.0f;
  }
  return r;
}

// The 32 keys of the tile at `key` that row `row` sees, as bits.
template <typename A>
__device__ __forceinline__ uint32_t seen_keys(A& a, const Place& p, int row, int key, int there) {
  const KeyRange kr = key_range(a, row_of(a, p, row).qi + p.shift, p.k_len);
  const int sink = a.sinks < kr.hi ? a.sinks : kr.hi;
  auto below = [&](int x) __attribute__((always_inline)) -> uint32_t {  // bits of keys < x
    const int n = x - key;
    return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u);
  };
  const uint32_t bits = below(kr.hi) & (~below(kr.lo) | below(sink));
  return bits & ((there & 1 ? 0xffffu : 0u) | (there & 2 ? 0xffff0000u : 0u));
}

// Few rows in units and their join, or one workgroup a key head (a.units 0); blocks of 128
// rows; type 0: bf16, 1: fp16.
int launch_cached_units(WindowArgs& a, int type, bool e4m3, int64_t D, int64_t units,
                        hipStream_t s);
void launch_cached_tile(WindowArgs& a, int type, bool e4m3, int64_t D, dim3 grid, hipStream_t s);

}  // namespace rcsa
