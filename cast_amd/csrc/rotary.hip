// Rotary positions, and the norms of queries and keys with the rotation in the
// same pass (and, with a paged cache, the append of keys and values).
//
// Pair i of a head's first R channels, (a, b) = channels (i, i + R/2) or
// (2i, 2i + 1), turns by t = position[axis(i)] * frequency(i):
//   a' = s (a cos t - b sin t),  b' = s (a sin t + b cos t);
// the other channels pass through.  With norms x is first
//   x * rsqrt(mean(x^2) + eps) * w, the mean over a head or over all heads.
//
// HBM-bound: each element is read once, written once, and rounded once (fp32
// between).  A position times a frequency needs more than 24 bits once the
// positions are far (at position 10^6 an fp32 angle is off by 0.06), so the
// angle is a product in turns in 64 bits, reduced to [-1/2, 1/2] turns there,
// and only then fp32: exact to an fp32 rounding at any position, with no table
// to read.  The sines are taken once per token and pair into LDS and shared by
// all heads of the token.
#include "rotary.h"

namespace rcsa {

// 8 consecutive elements as fp32, and back with one rounding.
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&f)[8]);
template <>
__device__ __forceinline__ void load8<__bf16>(const __bf16* p, float (&f)[8]) {
  Vec8<u16>::load(reinterpret_cast<const u16*>(p), f);
}
template <>
__device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
  Vec8<float>::load(p, f);
}
template <>
__device__ __forceinline__ void load8<_Float16>(const _Float16* p, float (&f)[8]) {
  const v8h r = *reinterpret_cast<const v8h*>(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = static_cast<float>(r[i]);
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  typedef T vec __attribute__((ext_vector_type(8)));
  vec r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = static_cast<T>(f[i]);
  *reinterpret_cast<vec*>(p) = r;
}

__device__ __forceinline__ float weight_at(const void* w, int dtype, int64_t i) {
  if (dtype == RCSA_F32) return static_cast<const float*>(w)[i];
  if (dtype == RCSA_F16) return static_cast<float>(static_cast<const _Float16*>(w)[i]);
  return bf16_to_f32(static_cast<const u16*>(w)[i]);
}
__device__ __forceinline__ void weight8(const void* w, int dtype, int64_t i, float (&f)[8]) {
  if (dtype == RCSA_F32) load8(static_cast<const float*>(w) + i, f);
  else if (dtype == RCSA_F16) load8(static_cast<const _Float16*>(w) + i, f);
  else load8(static_cast<const __bf16*>(w) + i, f);
}

// cos and sin (times the scale) of pair i of the token at (b, t).
__device__ __forceinline__ float2 turn_of(const RotaryArgs& a, int64_t b, int64_t t, int i) {
  int ax = a.axis == nullptr ? 0 : a.axis[i];
  ax = ax < 0 || ax >= a.n_axes ? 0 : ax;
  const int64_t at = b * a.pos_b + t * a.pos_l + ax * a.pos_a;
  const double p = a.pos_i64 ? static_cast<double>(static_cast<const int64_t*>(a.pos)[at])
                             : static_cast<double>(static_cast<const int32_t*>(a.pos)[at]);
  double turns = p * a.turns[i];
  turns -= __builtin_rint(turns);
  float s, c;
  sincospif(2.0f * static_cast<float>(turns), &s, &c);
  return make_float2(c * a.scale, s * a.scale);
}

// What a token's rows are: live or not, and where its keys and values go
// (element offsets of the row, -1: dropped).
struct TokenRows {
  int64_t b, t, q, k, v;
  bool live;
};
__device__ __forceinline__ TokenRows token_rows(const RotaryArgs& a, int64_t token) {
  TokenRows r;
  r.b = token / a.L;
  r.t = token - r.b * a.L;
  r.live = a.lengths == nullptr || r.t < a.lengths[r.b];
  r.q = r.b * a.qo[0] + r.t * a.qo[1];
  r.k = r.b * a.ko[0] + r.t * a.ko[1];
  r.v = -1;
  if (a.table != nullptr) {
    r.k = -1;
    const int64_t at = (a.starts == nullptr ? 0 : static_cast<int64_t>(a.starts[r.b])) + r.t;
    if (r.live && at >= 0 && at < a.max_pages * a.page_size) {
      const int64_t col = at / a.page_size;
      const int64_t page = a.table[r.b * a.table_stride + col];
      if (page >= 0 && page < a.n_pages) {
        const int64_t slot = at - col * a.page_size;
        r.k = page * a.ko[0] + slot * a.ko[1];
        r.v = page * a.vo[0] + slot * a.vo[1];
      }
    }
  }
  return r;
}

// The vector form: a lane holds 16 channels of a head, the 8 first and the 8
// second channels of 8 pairs (16 channels in a row where nothing turns or the
// pairs are interleaved), `lanes` = a power of two >= D / 16 lanes a head.  A
// workgroup takes `tokens` tokens; its threads run over their (token, head)
// list, queries, then keys, then values, so that no lane idles where a tensor
// has few heads.
template <typename T, bool INTER, int NORM>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int np = a.n_pairs, nt = a.tokens, nh = a.Hq + a.Hk + a.Hv;
  float* const s_cos = reinterpret_cast<float*>(smem);       // [nt][np]
  float* const s_sin = s_cos + nt * np;                      // [nt][np]
  float* const s_w = s_sin + nt * np;                        // [2][D] shared weights
  float* const s_sum = s_w + (NORM ? 2 * a.D : 0);           // [nt][Hq + Hk]
  // element offsets of every token's source and destination rows by tensor
  __shared__ int64_t s_src[3][kMaxTokens], s_dst[3][kMaxTokens];
  const int tid = threadIdx.x;
  const int64_t token0 = static_cast<int64_t>(blockIdx.x) * nt;
  const int64_t total = a.B * a.L;
  for (int i = tid; i < nt * np; i += 256) {
    const int64_t token = token0 + i / np;
    if (token < total) {
      const int64_t b = token / a.L;
      const float2 cs = turn_of(a, b, token - b * a.L, i % np);
      s_cos[i] = cs.x;
      s_sin[i] = cs.y;
    }
  }
  if (NORM)  // weights shared by the heads; others are read where they are used
    for (int i = tid; i < 2 * a.D; i += 256) {
      const void* w = i < a.D ? a.qw : a.kw;
      s_w[i] = w == nullptr ? 1.0f : weight_at(w, a.w_dtype, i < a.D ? i : i - a.D);
    }
  if (tid < nt) {
    const int64_t token = token0 + tid;
    TokenRows r{0, 0, -1, -1, -1, false};
    if (token < total) r = token_rows(a, token);
    s_src[0][tid] = r.b * a.qs[0] + r.t * a.qs[1];
    s_src[1][tid] = r.b * a.ks[0] + r.t * a.ks[1];
    s_src[2][tid] = r.b * a.vs[0] + r.t * a.vs[1];
    s_dst[0][tid] = r.live ? r.q : -1;
    s_dst[1][tid] = r.live ? r.k : -1;
    s_dst[2][tid] = r.live ? r.v : -1;
  }
  __syncthreads();

  const int lanes = 1 << a.lanes_log2;
  const int u = tid & (lanes - 1);
  const bool in_head = u * 16 < a.D;
  const bool turns = in_head && u * 16 < 2 * np;
  const int c0 = turns && !INTER ? 8 * u : 16 * u;       // the lane's two runs of 8 channels
  const int c1 = turns && !INTER ? np + 8 * u : 16 * u + 8;
  const int rows = nt * nh, step = 256 >> a.lanes_log2;

  // (token, head) of list entry i; the source row and which tensor it is
  auto entry = [&](int i, int& tl, int& h, int& part) __attribute__((always_inline)) {
    tl = i / nh;
    h = i - tl * nh;
    part = h < a.Hq ? 0 : h < a.Hq + a.Hk ? 1 : 2;
    h -= part == 0 ? 0 : part == 1 ? a.Hq : a.Hq + a.Hk;
  };
  auto load = [&](int tl, int h, int part, float (&x)[8], float (&y)[8])
      __attribute__((always_inline)) {
    const T* const p = static_cast<const T*>(part == 0 ? a.q : part == 1 ? a.k : a.v) +
                       s_src[part][tl] +
                       h * (part == 0 ? a.qs[2] : part == 1 ? a.ks[2] : a.vs[2]);
    load8(p + c0, x);
    load8(p + c1, y);
  };
  auto square_sum = [&](const float (&x)[8], const float (&y)[8])
      __attribute__((always_inline)) -> float {
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(x[j], x[j], fmaf(y[j], y[j], s));
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
    return s;
  };

  if (NORM == 2) {  // the sums of every (token, head), then of every token in a fixed order
    for (int i = tid >> a.lanes_log2; i < rows; i += step) {
      int tl, h, part;
      entry(i, tl, h, part);
      float x[8] = {}, y[8] = {};
      const int64_t dst = part < 2 ? s_dst[part][tl] : -1;
      if (in_head && dst >= 0) load(tl, h, part, x, y);
      const float s = square_sum(x, y);
      if (u == 0 && part < 2) s_sum[tl * (a.Hq + a.Hk) + (part == 0 ? h : a.Hq + h)] = s;
    }
    __syncthreads();
    float s = 0.0f;
    if (tid < 2 * nt) {
      const float* const p = s_sum + (tid >> 1) * (a.Hq + a.Hk) + (tid & 1 ? a.Hq : 0);
      const int n = tid & 1 ? a.Hk : a.Hq;
      for (int h = 0; h < n; ++h) s += p[h];
    }
    __syncthreads();
    if (tid < 2 * nt) s_sum[tid] = s;
    __syncthreads();
  }

  for (int i = tid >> a.lanes_log2; i < rows; i += step) {
    int tl, h, part;
    entry(i, tl, h, part);
    const int64_t dst = s_dst[part][tl];
    const bool ok = in_head && dst >= 0;
    float x[8] = {}, y[8] = {};
    if (ok) load(tl, h, part, x, y);
    if (NORM && part < 2) {  // (a row's lanes agree on part)
      float s, n = static_cast<float>(a.D);
      if (NORM == 2) {
        s = s_sum[2 * tl + part];
        n *= static_cast<float>(part == 0 ? a.Hq : a.Hk);
      } else {
        s = square_sum(x, y);
      }
      const float r = 1.0f / sqrtf(s / n + a.eps);
      if (in_head) {
        float w0[8], w1[8];
        const int64_t ws = part == 0 ? a.qw_h : a.kw_h;
        if (ws == 0) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            w0[j] = s_w[part * a.D + c0 + j];
            w1[j] = s_w[part * a.D + c1 + j];
          }
        } else {
          const void* const w = part == 0 ? a.qw : a.kw;
          weight8(w, a.w_dtype, h * ws + c0, w0);
          weight8(w, a.w_dtype, h * ws + c1, w1);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          x[j] *= r * w0[j];
          y[j] *= r * w1[j];
        }
      }
    }
    if (!ok) continue;
    if (turns && part < 2) {
      const float* const cs = s_cos + tl * np + 8 * u;
      const float* const sn = s_sin + tl * np + 8 * u;
      float c[8], s[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        c[j] = cs[j];
        s[j] = sn[j];
      }
      if (INTER) {  // pairs (0, 1), (2, 3) ... of the 16 channels
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float p = x[2 * j], q = x[2 * j + 1], m = y[2 * j], n = y[2 * j + 1];
          x[2 * j] = p * c[j] - q * s[j];
          x[2 * j + 1] = p * s[j] + q * c[j];
          y[2 * j] = m * c[4 + j] - n * s[4 + j];
          y[2 * j + 1] = m * s[4 + j] + n * c[4 + j];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const float p = x[j], q = y[j];
          x[j] = p * c[j] - q * s[j];
          y[j] = p * s[j] + q * c[j];
        }
      }
    }
    T* const o = static_cast<T*>(part == 0 ? a.qout : part == 1 ? a.kout : a.vout) + dst +
                 h * (part == 0 ? a.qo[2] : part == 1 ? a.ko[2] : a.vo[2]);
    store8(o + c0, x);
    store8(o + c1, y);
  }
}

// Any head size, pair count, stride and alignment: a wavefront takes one
// token's heads of one tensor, a lane the channels or pairs lane, lane + 64, ...
template <typename T, bool INTER, int NORM>
__global__ void __launch_bounds__(64) rotary_any_kernel(RotaryArgs a) {
  __shared__ float2 s_cs[kMaxDim / 2];
  const int lane = threadIdx.x;
  const int64_t token = blockIdx.x;
  const int part = blockIdx.y, np = a.n_pairs;
  const TokenRows r = token_rows(a, token);
  const int64_t dst = part == 0 ? r.q : part == 1 ? r.k : r.v;
  if (!r.live || dst < 0) return;  // (the whole wavefront)
  if (part < 2)
    for (int i = lane; i < np; i += kWave) s_cs[i] = turn_of(a, r.b, r.t, i);
  __syncthreads();
  const int64_t* const in = part == 0 ? a.qs : part == 1 ? a.ks : a.vs;
  const int64_t* const on = part == 0 ? a.qo : part == 1 ? a.ko : a.vo;
  const T* const src = static_cast<const T*>(part == 0 ? a.q : part == 1 ? a.k : a.v) +
                       r.b * in[0] + r.t * in[1];
  T* const out = static_cast<T*>(part == 0 ? a.qout : part == 1 ? a.kout : a.vout) + dst;
  const int H = part == 0 ? a.Hq : part == 1 ? a.Hk : a.Hv;
  const void* const w = part == 0 ? a.qw : a.kw;
  const int64_t ws = part == 0 ? a.qw_h : a.kw_h;
  const bool normed = NORM && part < 2;
  float rs = 1.0f;
  if (NORM == 2 && normed) {
    float s = 0.0f;
    for (int h = 0; h < H; ++h)
      for (int c = lane; c < a.D; c += kWave) {
        const float x = static_cast<float>(src[h * in[2] + c]);
        s = fmaf(x, x, s);
      }
    rs = 1.0f / sqrtf(wave_sum(s) / (static_cast<float>(a.D) * H) + a.eps);
  }
  for (int h = 0; h < H; ++h) {
    const T* const p = src + h * in[2];
    T* const o = out + h * on[2];
    if (NORM == 1 && normed) {
      float s = 0.0f;
      for (int c = lane; c < a.D; c += kWave) {
        const float x = static_cast<float>(p[c]);
        s = fmaf(x, x, s);
      }
      rs = 1.0f / sqrtf(wave_sum(s) / static_cast<float>(a.D) + a.eps);
    }
    auto at = [&](int c) __attribute__((always_inline)) -> float {
      float x = static_cast<float>(p[c]);
      if (normed) x *= rs * (w == nullptr ? 1.0f : weight_at(w, a.w_dtype, h * ws + c));
      return x;
    };
    const int turned = part < 2 ? np : 0;
    for (int i = lane; i < turned; i += kWave) {
      const int ca = INTER ? 2 * i : i, cb = INTER ? 2 * i + 1 : i + np;
      const float x = at(ca), y = at(cb);
      const float2 cs = s_cs[i];
      o[ca] = static_cast<T>(x * cs.x - y * cs.y);
      o[cb] = static_cast<T>(x * cs.y + y * cs.x);
    }
    for (int c = 2 * turned + lane; c < a.D; c += kWave) o[c] = static_cast<T>(at(c));
  }
}

template <typename T, bool INTER, int NORM>
static int launch(RotaryArgs& a, hipStream_t s) {
  const int64_t total = a.B * a.L;
  const int nh = a.Hq + a.Hk + a.Hv;
  const int64_t vec = 16 / static_cast<int64_t>(sizeof(T));
  bool wide = a.D % 16 == 0 && a.D <= 256 && a.n_pairs % 8 == 0;
  for (int i = 0; i < 3; ++i)
    wide = wide && a.qs[i] % vec == 0 && a.ks[i] % vec == 0 && a.vs[i] % vec == 0 &&
           a.qo[i] % vec == 0 && a.ko[i] % vec == 0 && a.vo[i] % vec == 0;
  for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.qout),
                        static_cast<const void*>(a.kout), static_cast<const void*>(a.vout)})
    wide = wide && aligned16(p);
  if (NORM) wide = wide && aligned16(a.qw) && aligned16(a.kw);
  if (!wide) {
    if (total >= (1ll << 31)) return RCSA_ERR_SHAPE;
    rotary_any_kernel<T, INTER, NORM>
        <<<dim3(static_cast<unsigned>(total), a.Hv ? 3 : a.Hk ? 2 : 1), dim3(kWave), 0, s>>>(a);
    return launch_status();
  }
  a.lanes_log2 = a.D <= 16 ? 0 : a.D <= 32 ? 1 : a.D <= 64 ? 2 : a.D <= 128 ? 3 : 4;
  // Tokens of a workgroup: about 8 rounds of its 256 lanes, fewer where that would
  // leave compute units without a workgroup.
  const int64_t lanes = static_cast<int64_t>(nh) << a.lanes_log2;
  int64_t nt = (2048 + lanes - 1) / lanes;
  nt = nt > kMaxTokens ? kMaxTokens : nt;
  while (nt > 1 && total / nt < 1024) nt /= 2;
  auto bytes = [&]() -> int64_t {
    return 4 * (2 * nt * a.n_pairs + (NORM ? 2 * a.D + nt * (a.Hq + a.Hk) + 2 : 0));
  };
  while (nt > 1 && bytes() > (32 << 10)) nt /= 2;
  if (bytes() > (60 << 10)) return RCSA_ERR_SHAPE;
  a.tokens = static_cast<int>(nt);
  const int64_t grid = (total + nt - 1) / nt;
  if (grid >= (1ll << 31) || nt * nh >= (1 << 30)) return RCSA_ERR_SHAPE;
  rotary_kernel<T, INTER, NORM><<<dim3(static_cast<unsigned>(grid)), dim3(256),
                                  static_cast<unsigned>(bytes()), s>>>(a);
  return launch_status();
}

template <typename T>
static int launch_type(RotaryArgs& a, bool inter, int norm, hipStream_t s) {
  if (norm == 0) return inter ? launch<T, true, 0>(a, s) : launch<T, false, 0>(a, s);
  if (norm == 1) return inter ? launch<T, true, 1>(a, s) : launch<T, false, 1>(a, s);
  return inter ? launch<T, true, 2>(a, s) : launch<T, false, 2>(a, s);
}

static int run(RotaryArgs& a, int dtype, bool inter, int norm, hipStream_t s) {
  if (a.B <= 0 || a.L <= 0 || a.Hq <= 0 || a.D <= 0 || a.D > kMaxDim || a.n_pairs < 0 ||
      2 * a.n_pairs > a.D || a.n_axes < 1 || a.B > (1ll << 31) / a.L)
    return RCSA_ERR_SHAPE;
  if (dtype == RCSA_BF16) return launch_type<__bf16>(a, inter, norm, s);
  if (dtype == RCSA_F16) return launch_type<_Float16>(a, inter, norm, s);
  return launch_type<float>(a, inter, norm, s);
}

static bool float_code(int dtype) {
  return dtype == RCSA_BF16 || dtype == RCSA_F16 || dtype == RCSA_F32;
}

static void positions(RotaryArgs& a, const void* pos, int pos_i64, const int64_t* ps,
                      int64_t n_axes, const double* turns, const int32_t* axis, int64_t n_pairs,
                      float scale) {
  a.pos = pos;
  a.pos_i64 = pos_i64;
  a.pos_b = ps[0];
  a.pos_l = ps[1];
  a.pos_a = ps[2];
  a.n_axes = static_cast<int>(n_axes);
  a.turns = turns;
  a.axis = axis;
  a.n_pairs = static_cast<int>(n_pairs);
  a.scale = scale;
}

}  // namespace rcsa

using namespace rcsa;

extern "C" int rcsa_rope(const void* x, void* out, int dtype, int64_t B, int64_t L, int64_t H,
                         int64_t D, const int64_t* strides, const void* pos, int pos_i64,
                         const int64_t* pos_strides, int64_t n_axes, const double* turns,
                         const int32_t* axis, int64_t n_pairs, int interleaved, float scale,
                         hipStream_t stream) {
  if (!x || !out || !strides || !pos || !pos_strides || (n_pairs > 0 && !turns))
    return RCSA_ERR_NULL;
  if (!float_code(dtype)) return RCSA_ERR_DTYPE;
  if (H <= 0 || H > kMaxHeads || D > kMaxDim || n_pairs > kMaxDim || n_axes > kMaxDim)
    return RCSA_ERR_SHAPE;
  RotaryArgs a{};
  a.q = x;
  a.qout = out;
  a.B = B;
  a.L = L;
  a.Hq = static_cast<int>(H);
  a.D = static_cast<int>(D);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.qo[i] = strides[3 + i];
  }
  positions(a, pos, pos_i64, pos_strides, n_axes, turns, axis, n_pairs, scale);
  return run(a, dtype, interleaved != 0, 0, stream);
}

extern "C" int rcsa_norm_rope(const void* q, const void* k, const void* v, void* q_out,
                              void* k_out, void* v_out, int dtype, const int64_t* dims,
                              const int64_t* strides, const void* q_weight, const void* k_weight,
                              int weight_dtype, int64_t q_weight_stride, int64_t k_weight_stride,
                              float eps, int across_heads, const void* pos, int pos_i64,
                              const int64_t* pos_strides, int64_t n_axes, const double* turns,
                              const int32_t* axis, int64_t n_pairs, int interleaved, float scale,
                              const int32_t* block_table, int64_t table_stride,
                              int64_t max_pages, int64_t n_pages, int64_t page_size,
                              const int32_t* starts, const int32_t* lengths,
                              hipStream_t stream) {
  if (!q || !k || !q_out || !k_out || !dims || !strides || !pos || !pos_strides ||
      (n_pairs > 0 && !turns))
    return RCSA_ERR_NULL;
  if ((v == nullptr) != (v_out == nullptr) || (v == nullptr) != (block_table == nullptr))
    return RCSA_ERR_NULL;
  if (!float_code(dtype) || !float_code(weight_dtype)) return RCSA_ERR_DTYPE;
  if (dims[2] <= 0 || dims[3] <= 0 || dims[2] > kMaxHeads || dims[3] > kMaxHeads ||
      dims[4] > kMaxDim || n_pairs > kMaxDim || n_axes > kMaxDim)
    return RCSA_ERR_SHAPE;
  if (block_table && (max_pages <= 0 || n_pages <= 0 || page_size <= 0 ||
                      max_pages > (1ll << 40) / page_size))
    return RCSA_ERR_SHAPE;
  RotaryArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.qout = q_out;
  a.kout = k_out;
  a.vout = v_out;
  a.B = dims[0];
  a.L = dims[1];
  a.Hq = static_cast<int>(dims[2]);
  a.Hk = static_cast<int>(dims[3]);
  a.Hv = v ? a.Hk : 0;
  a.D = static_cast<int>(dims[4]);
  for (int i = 0; i < 3; ++i) {
    a.qs[i] = strides[i];
    a.ks[i] = strides[3 + i];
    a.qo[i] = strides[9 + i];
    a.ko[i] = strides[12 + i];
    if (v) {
      a.vs[i] = strides[6 + i];
      a.vo[i] = strides[15 + i];
    }
  }
  a.qw = q_weight;
  a.kw = k_weight;
  a.w_dtype = weight_dtype;
  a.qw_h = q_weight ? q_weight_stride : 0;
  a.kw_h = k_weight ? k_weight_stride : 0;
  a.eps = eps;
  a.table = block_table;
  a.table_stride = table_stride;
  a.max_pages = max_pages;
  a.n_pages = n_pages;
  a.page_size = page_size;
  a.starts = starts;
  a.lengths = lengths;
  positions(a, pos, pos_i64, pos_strides, n_axes, turns, axis, n_pairs, scale);
  return run(a, dtype, interleaved != 0, across_heads ? 2 : 1, stream);
}
