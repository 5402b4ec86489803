// Attention over pages of 8-bit codes: what the kernels of few rows (cached_units.hip) and
// of 128-row blocks (cached_tile.hip) share.
//
// Keys and values are codes c with a scale s for each block of tokens and head.  The matrix
// products take the codes as fp16 (exact: 8 bits or less), so that a logit is
//   (q . c_k) * s_k sm_scale,   out = sum_j w_j s_vj c_vj / sum_j w_j.
// Queries become fp16 with a power of two a row that brings its largest value to [2^14,
// 2^15): bf16 rows lose nothing down to 2^-29 of it, and 2^-39 of it at most below.
// A weight takes the scale of its value's block, relative to a power of two 2^e above any scale of
// the keys that the row has seen so far, before it is rounded to fp16; e grows with the tiles (the
// accumulators move by the difference), and the sums of weights know nothing of it.  A block may
// have any scale for the rows that do not see it: it counts as 0 there.  A weight below 2^-31 of
// the row's largest, in a block whose scale is the largest that the row has met, is lost (it may
// be 2^6 where the largest is 2^7, and fp16 drops what is below 2^-25); in a block of a scale
// 2^-n of that, one below 2^(n - 31).  That is relative to the largest scale met, not to the
// result: a seen block of a far larger scale takes bits from the others' weights even where its
// own are next to nothing.
#pragma once
#include "window_attn.h"

namespace rcsa {

typedef _Float16 v2hf __attribute__((ext_vector_type(2)));

template <bool E4M3>
struct Widen;

template <>
struct Widen<false> {  // int8
  static __device__ __forceinline__ uint32_t tame(uint32_t w) { return w ^ 0x80808080u; }
  // (c + kMore) / kUnit: a byte c + 128 alone is the subnormal number (c + 128) 2^-24.  For
  // products whose other side's sum is known.
  static constexpr float kUnit = 0x1p24f, kMore = 128.0f;
  static __device__ __forceinline__ v2hf biased(uint32_t tamed, bool hi) {
    return __builtin_bit_cast(v2hf, hi ? __builtin_amdgcn_perm(0u, tamed, 0x0c030c02u)
                                       : __builtin_amdgcn_perm(0u, tamed, 0x0c010c00u));
  }
  // c 2^-kShift from (c + 128) 2^-24, exactly
  static constexpr int kShift = 9;
  static __device__ __forceinline__ v2hf centred(v2hf b) {
    const v2hf up = {static_cast<_Float16>(32768.0f), static_cast<_Float16>(32768.0f)};
    const v2hf less = {static_cast<_Float16>(-0.25f), static_cast<_Float16>(-0.25f)};
    return __builtin_elementwise_fma(b, up, less);
  }
  static __device__ __forceinline__ uint32_t finite(uint32_t w) { return w; }
  static __device__ __forceinline__ bool odd(uint32_t, uint32_t) { return false; }
};
template <>
struct Widen<true> {  // e4m3
  static __device__ __forceinline__ uint32_t tame(uint32_t w) { return w; }
  static constexpr float kUnit = 1.0f, kMore = 0.0f;
  static __device__ __forceinline__ v2hf biased(uint32_t w, bool hi) {
    return hi ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, true)
              : __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(static_cast<int>(w), 1.0f, false);
  }
  static constexpr int kShift = 0;
  static __device__ __forceinline__ v2hf centred(v2hf b) { return b; }
  // Codes that hold no number (0x7f, 0xff) as 0: a weight of 0 would not hide them.
  static __device__ __forceinline__ uint32_t finite(uint32_t w) {
    const uint32_t none = ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
    return w & ~((none >> 7) * 255u);
  }
  // Whether a lane of the wavefront has one.
  static __device__ __forceinline__ bool odd(uint32_t w0, uint32_t w1) {
    const uint32_t a = (w0 & 0x7f7f7f7fu) + 0x01010101u, b = (w1 & 0x7f7f7f7fu) + 0x01010101u;
    return __ballot(((a | b) & 0x80808080u) != 0) != 0;
  }
};

// Eight codes as an operand, (c + kMore) / kUnit or, centred, c 2^-kShift.
template <bool E4M3, bool CENTRED>
__device__ __forceinline__ v8hf widen8(uint32_t w0, uint32_t w1) {
  using W = Widen<E4M3>;
  struct Four {
    v2hf p[4];
  };
  Four f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f.p[i] = W::biased(W::tame(i < 2 ? w0 : w1), i & 1);
    if constexpr (CENTRED) f.p[i] = W::centred(f.p[i]);
  }
  return __builtin_bit_cast(v8hf, f);
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
      f.p[2 * i] = Widen<true>::biased(c, false);
      f.p[2 * i + 1] = Widen<true>::biased(c, true);
    }
  } else {
    const uint32_t s = 0x0c040c00u + 0x00010001u * static_cast<uint32_t>(x);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      f.p[i] = Widen<false>::centred(
          __builtin_bit_cast(v2hf, __builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], s)));
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
// The sum of a lane's share of a row.
template <int N>
__device__ __forceinline__ float sum_of(const v8hf (&q)[N]) {
  float sum = 0.0f;
#pragma unroll
  for (int st = 0; st < N; ++st)
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += static_cast<float>(q[st][i]);
  return sum;
}
// k with 2^14 <= most 2^k < 2^15, at most 100 (rows of zeros, and of no numbers: 0).
__device__ __forceinline__ int row_shift(float most) {
  if (!(most > 0.0f && most < INFINITY)) return 0;
  const int k = 14 - (static_cast<int>(__float_as_uint(most) >> 23) - 127);
  return k > 100 ? 100 : k;
}

// A share's tiles one after the other: where the codes of the present one are, and which scales
// are its.  All of it is scalar work, which takes its turn with the vector work of a wavefront:
// pages of whole tiles (WHOLE) are stepped along by additions, the table is looked into where one
// ends, a page ahead; otherwise the two halves of 16 keys are looked up each on their own.
// FORM kWhole: blocks of whole tiles, one scale a tile; kHalves: blocks of 16 keys, two; kAny:
// pages or blocks of neither, the entries of a tile asked for a tile ahead.  Arguments that only
// some steps need are read again there: scalar registers are short.  Past the share's last tile,
// and on pages that are not there, the codes stand where some page's are: they are read, and not
// seen.
enum CodeForm { kWhole, kHalves, kAny };
inline CodeForm code_form(const WindowArgs& a) {
  if (!a.whole_tiles) return kAny;
  return a.mark % kTileKeys == 0 ? kWhole : a.mark == kTileKeys / 2 ? kHalves : kAny;
}
template <CodeForm FORM>
struct Scales {
  static constexpr int N = FORM == kWhole ? 1 : 2;
  float k[N], v[N];
};
template <CodeForm FORM>
struct TileRef {
  static constexpr int N = FORM == kWhole ? 1 : 2;
  int key, there;  // the first key, -1: no tile; which halves are there (bits)
  int k[N], v[N];  // where their scales are
};
template <CodeForm FORM, typename A>
struct CodeStream {
  static constexpr bool WHOLE = FORM != kAny;
  A& a;
  const int32_t* table;
  int hk, page, mark;
  uint32_t krb, vrb;
  int left, sinks, window;  // tiles left, those of the first keys, the window's first key
  int slot, in_mark;
  int col, ahead;            // WHOLE: the column of the page, the entry behind it
  int key1, ahead1;          // kAny: the next tile's first key, its pages `ahead` and `ahead1`
  const char *kp, *vp;
  int page1, slot1;
  TileRef<FORM> ref;

  __device__ __forceinline__ CodeStream(A& args, const Place& p)
      : a(args),
        table(args.table + p.b * args.table_stride),
        hk(p.hk),
        page(args.page),
        mark(args.mark),
        krb(static_cast<uint32_t>(args.sk[1])),
        vrb(static_cast<uint32_t>(args.sv[1])) {
    left = p.steps;
    sinks = p.tiles.sink_n - p.begin;
    window = p.tiles.win_t0 * kTileKeys;
    slot1 = page1 = in_mark = col = key1 = ahead1 = 0;
    const int first = left <= 0 ? -1 : sinks > 0 ? p.begin * kTileKeys
                                                 : window - sinks * kTileKeys;
    if constexpr (WHOLE) {
      jump(args, first);
    } else {
      look(args, first);
      pass(args);
      look(args, after(first));
    }
  }
  // kAny: the first key of the tile behind the present one.
  __device__ __forceinline__ int after(int key) const {
    return left <= 1 ? -1 : sinks == 1 ? window : key + kTileKeys;
  }
  template <typename X>
  __device__ __forceinline__ void look(X& x, int key) {
    key1 = key;
    const int half = (key < 0 ? 0 : key) >> 4;
    ahead = entry(x, divide(half, x.by_half_page));
    ahead1 = entry(x, divide(half + 1, x.by_half_page));
  }
  template <typename X>
  __device__ __forceinline__ void pass(X& x) {
    ref.key = key1;
    const int k = key1 < 0 ? 0 : key1;
    slot = k - divide(k >> 4, x.by_half_page) * page;
    slot1 = slot + 16 < page ? slot + 16 : 0;
    page1 = ahead1;
    on_page(x, 0, ahead, slot);
    on_page(x, 1, page1, slot1);
  }
  template <typename X>
  __device__ __forceinline__ int entry(X& x, int c) const {
    return ld_const(table + (c < x.max_pages ? c : x.max_pages - 1));
  }
  // Row `at_slot` of a page (page 0's where it is not there).  (32 x 32-bit products: a page
  // spans less than 4 GiB.)
  struct At {
    const char *k, *v;
  };
  template <typename X>
  __device__ __forceinline__ At row_at(X& x, bool there, int pg, int at_slot) const {
    const uint32_t at = there ? static_cast<uint32_t>(pg) : 0u;
    const uint32_t row = static_cast<uint32_t>(at_slot);
    return {static_cast<const char*>(x.k) + hk * x.sk[2] +
                static_cast<uint64_t>(at) * static_cast<uint32_t>(x.sk[0]) +
                static_cast<uint64_t>(row) * krb,
            static_cast<const char*>(x.v) + hk * x.sv[2] +
                static_cast<uint64_t>(at) * static_cast<uint32_t>(x.sv[0]) +
                static_cast<uint64_t>(row) * vrb};
  }
  template <typename X>
  __device__ __forceinline__ void on_page(X& x, int h, int pg, int at_slot) {
    const bool there = ref.key >= 0 && page_ok(x, pg);
    if (h == 0) {
      const At at = row_at(x, there, pg, at_slot);
      kp = at.k;
      vp = at.v;
    }
    const int nth = divide(at_slot >> 4, x.by_half_mark), at = there ? pg : 0;
    ref.k[h] = at * x.sks[0] + nth * x.sks[1];
    ref.v[h] = at * x.svs[0] + nth * x.svs[1];
    if constexpr (WHOLE) {
      ref.there = there ? 3 : 0;
      in_mark = at_slot - nth * mark;
      if constexpr (FORM == kHalves) {
        ref.k[1] = ref.k[0] + x.sks[1];
        ref.v[1] = ref.v[0] + x.svs[1];
      }
    } else {
      ref.there = h == 0 ? (there ? 1 : 0) : ref.there + (there ? 2 : 0);
    }
  }
  template <typename X>
  __device__ __forceinline__ void jump(X& x, int key) {
    ref.key = key;
    const int k = key < 0 ? 0 : key;
    col = divide(k >> 4, x.by_half_page);
    slot = k - col * page;
    on_page(x, 0, entry(x, col), slot);
    ahead = entry(x, col + 1);
  }
  __device__ __forceinline__ void next() {
    --left;
    --sinks;
    if constexpr (WHOLE) {
      if (left <= 0) {
        ref.key = -1;
        return;
      }
      if (sinks == 0) {
        jump(late_args(), window);
        return;
      }
      ref.key += kTileKeys;
      slot += kTileKeys;
      if (slot >= page) {
        LateArgs& x = late_args();
        ++col;
        slot = 0;
        on_page(x, 0, ahead, 0);
        ahead = entry(x, col + 1);
        return;
      }
      kp += kTileKeys * krb;
      vp += kTileKeys * vrb;
      if constexpr (FORM == kHalves) {
        const int dk = 2 * (ref.k[1] - ref.k[0]), dv = 2 * (ref.v[1] - ref.v[0]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          ref.k[h] += dk;
          ref.v[h] += dv;
        }
        return;
      }
      in_mark += kTileKeys;
      if (in_mark >= mark) {
        LateArgs& x = late_args();
        in_mark = 0;
        ref.k[0] += x.sks[1];
        ref.v[0] += x.svs[1];
      }
    } else {
      LateArgs& x = late_args();
      pass(x);
      look(x, after(ref.key));
    }
  }
  // The first rows of a half.
  __device__ __forceinline__ At half(int h) const {
    if constexpr (WHOLE) {
      return {kp + h * 16 * krb, vp + h * 16 * vrb};
    } else {
      return h == 0 ? At{kp, vp} : row_at(late_args(), ref.there & 2, page1, slot1);
    }
  }
};
// A positive number below 2^126, or 0.
__device__ __forceinline__ float scale_or_0(float s) {
  const uint32_t u = __float_as_uint(s);
  return u - 1u < 0x7e800000u - 1u ? s : 0.0f;
}
// The scales of a tile (ks, vs: of the key head), 0 for a half that is not there.
template <CodeForm FORM>
__device__ __forceinline__ Scales<FORM> scales_of(const TileRef<FORM>& t, const float* ks,
                                                   const float* vs) {
  Scales<FORM> r;
#pragma unroll
  for (int h = 0; h < TileRef<FORM>::N; ++h) {
    r.k[h] = scale_or_0(ld_const(ks + t.k[h]));
    r.v[h] = (t.there >> h) & 1 ? scale_or_0(ld_const(vs + t.v[h])) : 0.0f;
  }
  return r;
}
// `s` in the lanes of a mask, 0 in the others.
__device__ __forceinline__ float in_lanes(uint64_t mask, float s) {
  return __builtin_amdgcn_inverse_ballot_w64(mask) ? s : 0.0f;
}
// The unit 2^e of a row's accumulators, as its bits: above the scales of all values that it has
// seen so far.
constexpr uint32_t kLeastUnit = 1u << 23;
__device__ __forceinline__ float per_unit(uint32_t unit) {  // 2^-e
  return __uint_as_float((254u << 23) - unit);
}
// The unit raised above a scale s, where it is not, and the factor to it.
__device__ __forceinline__ float raise_unit(uint32_t& unit, float s) {
  const uint32_t e = (__float_as_uint(s) >> 23) + 1u;  // (at most 253)
  if (__float_as_uint(s) < unit) return 1.0f;
  const uint32_t down = e - (unit >> 23);
  unit = e << 23;
  return down >= 127u ? 0.0f : __uint_as_float((127u - down) << 23);
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
