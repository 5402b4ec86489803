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
// between).  44 frames x 24 heads of 128 80 us, 5.9 TB/s; with joint norms and the append to
// pages 3520 x 72 heads 34 us, 3.8 TB/s (a token's sums stand between its loads and its
// stores, and 130 MB are few beside a launch's start and end); with norms of heads 16391 x 48
// heads of 128 71 us, 5.7 TB/s, 32782 x 20 heads of 64 40 us, 4.2 TB/s; one token of 8
// requests 3.6 us, with norms and pages of 64 requests 5.7 us: a launch and its loads.
// A position times a frequency needs more than 24 bits once the positions are far (at
// position 10^6 an fp32 angle is off by 0.06), so the angle is a product in turns in 64
// bits, reduced to [-1/2, 1/2] turns there, and only then fp32: exact to an fp32 rounding at
// any position, with no table to read.  The sines are taken once per token and pair into LDS
// and shared by all heads of the token.
#include "rotary.h"

namespace rcsa {

__device__ __forceinline__ float weight_at(const void* w, int dtype, int64_t i) {
  if (dtype == RCSA_F32) return static_cast<const float*>(w)[i];
  if (dtype == RCSA_F16) return static_cast<float>(static_cast<const _Float16*>(w)[i]);
  return bf16_to_f32(static_cast<const u16*>(w)[i]);
}
template <typename W, int V>
__device__ __forceinline__ void widen(const void* w, int64_t i, float (&f)[V]) {
  typedef W vec __attribute__((ext_vector_type(V)));
  const vec r = *reinterpret_cast<const vec*>(static_cast<const W*>(w) + i);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = static_cast<float>(r[j]);
}
template <int V>
__device__ __forceinline__ void weight_run(const void* w, int dtype, int64_t i, float (&f)[V]) {
  if (dtype == RCSA_F32) widen<float, V>(w, i, f);
  else if (dtype == RCSA_F16) widen<_Float16, V>(w, i, f);
  else widen<__bf16, V>(w, i, f);
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
// (element offsets of the row, -1: dropped).  In three steps, each of which waits for the one
// before: its request's lengths, its page, its rows.
struct TokenAt {
  int b, t, length, start;
};
__device__ __forceinline__ TokenAt token_at(const RotaryArgs& a, int token) {
  TokenAt r;
  r.b = divide(token, a.by_L);
  r.t = token - r.b * static_cast<int>(a.L);
  r.length = a.lengths == nullptr ? static_cast<int>(a.L) : a.lengths[r.b];
  r.start = a.starts == nullptr ? 0 : a.starts[r.b];
  return r;
}
// Index of the token's keys in its request's pages (-1: none, or dropped) and their page.
struct TokenPage {
  int at, page;
};
__device__ __forceinline__ TokenPage token_page(const RotaryArgs& a, const TokenAt& r) {
  if (a.table == nullptr) return {-1, -1};
  const int64_t at = static_cast<int64_t>(r.start) + r.t;
  if (r.t >= r.length || at < 0 || at >= a.max_pages * a.page_size) return {-1, -1};
  const int i = static_cast<int>(at);
  return {i, a.table[r.b * a.table_stride + divide(i, a.by_page)]};
}
struct TokenRows {
  int64_t q, k, v;
  bool live;
};
__device__ __forceinline__ TokenRows token_rows(const RotaryArgs& a, const TokenAt& p,
                                                const TokenPage& g) {
  TokenRows r;
  r.live = p.t < p.length;
  r.q = p.b * a.qo[0] + p.t * a.qo[1];
  r.k = p.b * a.ko[0] + p.t * a.ko[1];
  r.v = -1;
  if (a.table != nullptr) {
    r.k = -1;
    if (g.page >= 0 && g.page < a.n_pages) {
      const int64_t slot = g.at - divide(g.at, a.by_page) * static_cast<int>(a.page_size);
      r.k = g.page * a.ko[0] + slot * a.ko[1];
      r.v = g.page * a.vo[0] + slot * a.vo[1];
    }
  }
  return r;
}

// A launch's workgroups lie in even rows of at most 2^16 (a dimension holds less than 2^32
// threads); the few that even rows add have nothing to do.
static dim3 grid_of(int64_t workgroups, int parts = 1) {
  const int64_t rows = (workgroups + 65535) / 65536;
  return dim3(static_cast<unsigned>((workgroups + rows - 1) / rows), static_cast<unsigned>(rows),
              static_cast<unsigned>(parts));
}
__device__ __forceinline__ int workgroup_index() {
  return static_cast<int>(blockIdx.y * gridDim.x + blockIdx.x);
}

// The vector form.  A lane holds two runs of V channels of a head: V pairs of the half
// layout, or 2 V / 2 interleaved ones; `lanes` = a power of two >= D / 2V lanes a head.  A
// workgroup takes `tokens` tokens; its threads run over their (token, head) list, queries,
// keys, then values, so that no lane idles where a tensor has few heads, U entries at a time:
// the loads of all U are issued first, those of the first U ahead of the sines (rows
// that are in flight, not the work on them, set the pace).  Joint norms need a token's
// sum before its first store: a list of U entries stays in registers in between, a
// longer one is read again.  Rows go past the caches both ways (non-temporal; us without,
// inputs out of the caches: 44 frames x 24 heads 79 and 91, 3520 x 72 heads with joint
// norms 34 and 40, 16391 x 48 heads 80 and 86).  A memory-bound reader of the outputs right
// behind loses what that gains or, at 84 MB of them, 7% of the pair; the reader here is
// the attention.
template <typename T>
constexpr int kWide = 16 / static_cast<int>(sizeof(T));
// Entries of a thread.  Wide runs: two for the rotation alone (44 frames x 24 heads 80 us, one
// 89), one with norms of heads (16391 tokens x 48 heads 71 us, two 75, three 79), three with
// joint norms, which the list of a token should fit (3520 x 72 heads 34 us, two 42, four 38, five
// 34; 9000 x 40 heads 51, 50, 51, 50; 3520 x 48 heads fp32 36, 41, 40, 43); narrow
// runs six (3 x 14097 x 9 heads of 80 56 us, four 61): 4 bytes a lane move at 2.2 TB/s, half of
// what the wide runs reach.
template <int V, int NORM>
constexpr int kEntries = V == 2 ? 6 : (NORM == 0 ? 2 : (NORM == 1 ? 1 : 3));
template <typename T, int V>
struct Run {
  typedef T vec __attribute__((ext_vector_type(V)));
};
template <typename T, int V, bool INTER, int NORM>
__global__ void __launch_bounds__(256) rotary_kernel(RotaryArgs a) {
  typedef typename Run<T, V>::vec vec;
  constexpr int U = kEntries<V, NORM>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int np = a.n_pairs, nt = a.tokens, nn = a.Hq + a.Hk, nh = nn + a.Hv;
  float* const s_cos = reinterpret_cast<float*>(smem);       // [nt][np]
  float* const s_sin = s_cos + nt * np;                      // [nt][np]
  float* const s_w = s_sin + nt * np;                        // [2][D] shared weights
  float* const s_sum = s_w + (NORM ? 2 * a.D : 0);           // [nt][Hq + Hk]
  float* const s_all = s_sum + nt * nn;                      // [nt][2] sums of a token
  // element offsets of every token's destination rows by tensor, -1: none
  __shared__ int64_t s_dst[3][kMaxTokens];
  const int tid = threadIdx.x, threads = blockDim.x;
  const int total = static_cast<int>(a.B * a.L);
  const int token0 = workgroup_index() * nt;
  if (token0 >= total) return;
  const int left = total - token0 < nt ? total - token0 : nt;  // tokens of this workgroup

  const int lanes = 1 << a.lanes_log2;
  const int u = tid & (lanes - 1), group = tid >> a.lanes_log2, step = threads >> a.lanes_log2;
  const bool in_head = u * 2 * V < a.D;
  // the lane's two runs, and whether they turn
  int c0 = V * u, c1 = a.D / 2 + V * u;
  bool turn0, turn1;
  if (INTER) {
    turn0 = c0 < 2 * np;
    turn1 = c1 < 2 * np;
  } else {
    const int nu = np / V;
    turn0 = turn1 = u < nu;
    if (turn0) c1 = np + V * u;
    else c0 = 2 * np + V * (u - nu), c1 = np + a.D / 2 + V * (u - nu);
  }
  const int rows = left * nh;

  // entry i of the list: token, tensor (0 queries, 1 keys, 2 values), head
  struct Entry {
    int tl, part, h;
  };
  auto entry = [&](int i) __attribute__((always_inline)) -> Entry {
    const int tl = divide(i, a.by_heads), h = i - tl * nh;
    return {tl, h < a.Hq ? 0 : (h < nn ? 1 : 2), h - (h < a.Hq ? 0 : (h < nn ? a.Hq : nn))};
  };
  auto source = [&](const Entry& e) __attribute__((always_inline)) -> const T* {
    const int token = token0 + e.tl, b = divide(token, a.by_L);
    const int64_t* const s = e.part == 0 ? a.qs : (e.part == 1 ? a.ks : a.vs);
    return static_cast<const T*>(e.part == 0 ? a.q : (e.part == 1 ? a.k : a.v)) + b * s[0] +
           (token - b * static_cast<int>(a.L)) * s[1] + e.h * s[2];
  };
  vec x[U], y[U];
  auto load = [&](int i0) __attribute__((always_inline)) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + group + k * step;
      if (in_head && i < rows) {
        const T* const p = source(entry(i));
        x[k] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(p + c0));
        y[k] = __builtin_nontemporal_load(reinterpret_cast<const vec*>(p + c1));
      }
    }
  };
  // The first wavefronts take the sines, the second (of one: the only) the weights, the last the
  // places of the tokens' rows, whose lengths are asked for ahead of the rows: the loads of
  // a small call are its time.
  const int wave = uniform_int(tid >> 6), last = (threads >> 6) - 1;
  TokenAt at{};
  if (wave == last) at = token_at(a, token0 + ((tid & 63) < left ? tid & 63 : 0));
  load(0);
  TokenPage page{};
  if (wave == last) page = token_page(a, at);
  if (NORM && (last == 0 || wave == 1))  // (weights of a head's own: where they are used)
    for (int i = tid & 63; i < 2 * a.D / V; i += kWave) {
      const bool key = i * V >= a.D;
      const void* const w = key ? a.kw : a.qw;
      float f[V];
#pragma unroll
      for (int j = 0; j < V; ++j) f[j] = 1.0f;
      if (w != nullptr && (key ? a.kw_h : a.qw_h) == 0)
        weight_run<V>(w, a.w_dtype, i * V - (key ? a.D : 0), f);
#pragma unroll
      for (int j = 0; j < V; ++j) s_w[i * V + j] = f[j];
    }
  for (int i = tid; i < left * np; i += threads) {
    const int tl = divide(i, a.by_pairs), token = token0 + tl, b = divide(token, a.by_L);
    const float2 cs = turn_of(a, b, token - b * static_cast<int>(a.L), i - tl * np);
    s_cos[i] = cs.x;
    s_sin[i] = cs.y;
  }
  if (wave == last && (tid & 63) < left) {
    const TokenRows r = token_rows(a, at, page);
    s_dst[0][tid & 63] = r.live ? r.q : -1;
    s_dst[1][tid & 63] = r.live ? r.k : -1;
    s_dst[2][tid & 63] = r.live ? r.v : -1;
  }
  __syncthreads();

  auto square_sum = [&](const vec& p, const vec& q, bool ok) __attribute__((always_inline)) -> float {
    float s = 0.0f;
    if (ok) {
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float f = static_cast<float>(p[j]), g = static_cast<float>(q[j]);
        s = fmaf(f, f, fmaf(g, g, s));
      }
    }
    for (int o = lanes >> 1; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
    return s;
  };
  const bool held = rows <= U * step;  // the whole list is in registers
  if (NORM == 2) {  // the sums of every (token, head), then of every token in a fixed order
    for (int i0 = 0; i0 < rows; i0 += U * step) {
      if (i0 != 0) load(i0);
#pragma unroll
      for (int k = 0; k < U; ++k) {
        const int i = i0 + group + k * step;
        const float s = square_sum(x[k], y[k], in_head && i < rows);
        const Entry e = entry(i);
        if (u == 0 && i < rows && e.part < 2) s_sum[e.tl * nn + (e.part ? a.Hq : 0) + e.h] = s;
      }
    }
    __syncthreads();
    for (int j = tid >> 4; j < 2 * left; j += threads >> 4) {  // 16 lanes a token and tensor
      const float* const p = s_sum + (j >> 1) * nn + (j & 1 ? a.Hq : 0);
      const int n = j & 1 ? a.Hk : a.Hq;
      float s = 0.0f;
      for (int h = tid & 15; h < n; h += 16) s += p[h];
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
      if ((tid & 15) == 0) s_all[j] = s;
    }
    __syncthreads();
  }

  for (int i0 = 0; i0 < rows; i0 += U * step) {
    if (i0 != 0 || (NORM == 2 && !held)) load(i0);
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + group + k * step;
      if (i >= rows) break;  // (a head's lanes agree)
      const Entry e = entry(i);
      const int64_t dst = s_dst[e.part][e.tl];
      T* const o = static_cast<T*>(e.part == 0 ? a.qout : (e.part == 1 ? a.kout : a.vout)) + dst +
                   e.h * (e.part == 0 ? a.qo[2] : (e.part == 1 ? a.ko[2] : a.vo[2]));
      if (e.part == 2) {  // values as they are
        if (in_head && dst >= 0) {
          __builtin_nontemporal_store(x[k], reinterpret_cast<vec*>(o + c0));
          __builtin_nontemporal_store(y[k], reinterpret_cast<vec*>(o + c1));
        }
        continue;
      }
      float p[V], q[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        p[j] = static_cast<float>(x[k][j]);
        q[j] = static_cast<float>(y[k][j]);
      }
      if (NORM) {
        float s, n = static_cast<float>(a.D);
        if (NORM == 2) {
          s = s_all[2 * e.tl + e.part];
          n *= static_cast<float>(e.part ? a.Hk : a.Hq);
        } else {
          s = square_sum(x[k], y[k], in_head);
        }
        const float r = 1.0f / sqrtf(s / n + a.eps);
        const int64_t ws = e.part ? a.kw_h : a.qw_h;
        if (in_head) {
          if (ws == 0) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
              p[j] *= r * s_w[e.part * a.D + c0 + j];
              q[j] *= r * s_w[e.part * a.D + c1 + j];
            }
          } else {
            const void* const w = e.part ? a.kw : a.qw;
            float w0[V], w1[V];
            weight_run<V>(w, a.w_dtype, e.h * ws + c0, w0);
            weight_run<V>(w, a.w_dtype, e.h * ws + c1, w1);
#pragma unroll
            for (int j = 0; j < V; ++j) {
              p[j] *= r * w0[j];
              q[j] *= r * w1[j];
            }
          }
        }
      }
      if (!in_head || dst < 0) continue;
      if (INTER) {  // pairs (0, 1), (2, 3) ... of either run
        auto turn = [&](float (&f)[V], int c) __attribute__((always_inline)) {
          const float* const cs = s_cos + e.tl * np + c / 2;
          const float* const sn = s_sin + e.tl * np + c / 2;
#pragma unroll
          for (int j = 0; j < V / 2; ++j) {
            const float f0 = f[2 * j], f1 = f[2 * j + 1];
            f[2 * j] = f0 * cs[j] - f1 * sn[j];
            f[2 * j + 1] = f0 * sn[j] + f1 * cs[j];
          }
        };
        if (turn0) turn(p, c0);
        if (turn1) turn(q, c1);
      } else if (turn0) {
        const float* const cs = s_cos + e.tl * np + V * u;
        const float* const sn = s_sin + e.tl * np + V * u;
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float f0 = p[j], f1 = q[j];
          p[j] = f0 * cs[j] - f1 * sn[j];
          q[j] = f0 * sn[j] + f1 * cs[j];
        }
      }
      vec o0, o1;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        o0[j] = static_cast<T>(p[j]);
        o1[j] = static_cast<T>(q[j]);
      }
      __builtin_nontemporal_store(o0, reinterpret_cast<vec*>(o + c0));
      __builtin_nontemporal_store(o1, reinterpret_cast<vec*>(o + c1));
    }
  }
}

// Any head size, pair count, stride and alignment: a wavefront takes one
// token's heads of one tensor, a lane the channels or pairs lane, lane + 64, ...
template <typename T, bool INTER, int NORM>
__global__ void __launch_bounds__(64) rotary_any_kernel(RotaryArgs a) {
  __shared__ float2 s_cs[kMaxDim / 2];
  const int lane = threadIdx.x;
  const int token = workgroup_index();
  if (token >= static_cast<int>(a.B * a.L)) return;
  const int part = blockIdx.z, np = a.n_pairs;
  const TokenAt tok = token_at(a, token);
  const TokenRows r = token_rows(a, tok, token_page(a, tok));
  const int64_t dst = part == 0 ? r.q : part == 1 ? r.k : r.v;
  if (!r.live || dst < 0) return;  // (the whole wavefront)
  if (part < 2)
    for (int i = lane; i < np; i += kWave) s_cs[i] = turn_of(a, tok.b, tok.t, i);
  __syncthreads();
  const int64_t* const in = part == 0 ? a.qs : part == 1 ? a.ks : a.vs;
  const int64_t* const on = part == 0 ? a.qo : part == 1 ? a.ko : a.vo;
  const T* const src = static_cast<const T*>(part == 0 ? a.q : part == 1 ? a.k : a.v) +
                       tok.b * in[0] + tok.t * in[1];
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

// Whether rows, strides and pointers suit runs of V channels.
template <typename T>
static bool runs_of(const RotaryArgs& a, int V, bool inter) {
  if (a.D % (2 * V) || a.D > 128 * V || (inter ? 2 * a.n_pairs : a.n_pairs) % V) return false;
  for (int i = 0; i < 3; ++i)
    for (const int64_t* s : {a.qs, a.ks, a.vs, a.qo, a.ko, a.vo})
      if (s[i] % V) return false;
  for (const void* p : {a.q, a.k, a.v, static_cast<const void*>(a.qout),
                        static_cast<const void*>(a.kout), static_cast<const void*>(a.vout)})
    if (reinterpret_cast<uintptr_t>(p) % (V * sizeof(T) < 16 ? V * sizeof(T) : 16)) return false;
  const size_t w = V * (a.w_dtype == RCSA_F32 ? 4 : 2);
  for (const void* p : {a.qw, a.kw})
    if (reinterpret_cast<uintptr_t>(p) % (w < 16 ? w : 16)) return false;
  return a.qw_h % V == 0 && a.kw_h % V == 0;
}

template <typename T, int V, bool INTER, int NORM>
static int launch_runs(RotaryArgs& a, hipStream_t s) {
  const int64_t total = a.B * a.L;
  const int nh = a.Hq + a.Hk + a.Hv;
  a.lanes_log2 = 0;
  while ((2 * V) << a.lanes_log2 < a.D) ++a.lanes_log2;
  // Tokens of a workgroup: as many as its lanes hold at once, fewer where that would
  // leave compute units without a workgroup; lanes: whole wavefronts that share the list
  // evenly.
  constexpr int U = kEntries<V, NORM>;
  const int64_t per = static_cast<int64_t>(nh) << a.lanes_log2;
  int64_t nt = U * 256 / per;
  nt = nt < 1 ? 1 : (nt > kMaxTokens ? kMaxTokens : nt);
  while (nt > 1 && total / nt < 512) nt /= 2;
  auto bytes = [&]() -> int64_t {
    return 4 * (2 * nt * a.n_pairs + (NORM ? 2 * a.D + nt * (a.Hq + a.Hk + 2) : 0));
  };
  while (nt > 1 && bytes() > (32 << 10)) nt /= 2;
  if (bytes() > (60 << 10)) return RCSA_ERR_SHAPE;
  a.tokens = static_cast<int>(nt);
  a.by_heads = divisor(static_cast<uint32_t>(nh));
  a.by_pairs = divisor(a.n_pairs > 0 ? static_cast<uint32_t>(a.n_pairs) : 1u);
  const int64_t grid = (total + nt - 1) / nt;
  const int64_t rounds = (nt * per + 255) / 256;
  const int64_t threads = ((nt * per + rounds - 1) / rounds + kWave - 1) / kWave * kWave;
  rotary_kernel<T, V, INTER, NORM><<<grid_of(grid), dim3(static_cast<unsigned>(threads)),
                                     static_cast<unsigned>(bytes()), s>>>(a);
  return launch_status();
}

// Runs of 16 bytes where sizes, strides and pointers allow, of 2 channels where they allow
// that, else element by element.
template <typename T, bool INTER, int NORM>
static int launch(RotaryArgs& a, hipStream_t s) {
  if (a.B * a.L >= (1ll << 30)) return RCSA_ERR_SHAPE;
  a.by_L = divisor(static_cast<uint32_t>(a.L));
  if (a.table) a.by_page = divisor(static_cast<uint32_t>(a.page_size));
  constexpr int W = kWide<T>;
  if (runs_of<T>(a, W, INTER)) return launch_runs<T, W, INTER, NORM>(a, s);
  if (runs_of<T>(a, 2, INTER)) return launch_runs<T, 2, INTER, NORM>(a, s);
  rotary_any_kernel<T, INTER, NORM>
      <<<grid_of(a.B * a.L, a.Hv ? 3 : a.Hk ? 2 : 1), dim3(kWave), 0, s>>>(a);
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
                      max_pages >= (1ll << 31) / page_size))
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
