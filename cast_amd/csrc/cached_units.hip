// Attention of few rows over pages of 8-bit codes (one new token of each request, or a few): at
// most 32 rows of a key head, dealt as in window_units.hip to workgroups of eight wavefronts
// or to units of one.
//
// The codes of values go from memory to the matrix operands through registers alone: a lane of
// O^T = V^T P^T holds D / 32 neighbouring channels of the 16 keys whose weights it has, one
// load a key (a load instruction covers two whole rows), turned byte by byte into operands.
// A lane of S = K Q^T holds a key's channels: loaded as they stand, every load would touch 32
// lines for a fourth of each (48 ragged requests, 248 us with two tiles in flight so, in more
// lines than the first cache has), so keys are loaded by whole rows and go through LDS.
//
// Bound by HBM where the cache is long: 48 requests of up to 32768 keys, 32 heads on 8 of D 128,
// 191 us for 1.02 GB (5.3 TB/s) and 7 for the join; in all 198, and while that was 213 keys by
// their lanes' rows took 228 us, by copies to LDS 222.  Short calls are latency: 1 request, 1024
// keys of 8 heads 8.2 us and 3 to 4 for the join.
#include "cached_attn.h"

namespace rcsa {

// Wavefronts to a SIMD: those of D 64 leave registers for two workgroups of eight on a compute
// unit (48 requests of 1599 keys, 7 queries of 12 heads 57.7 us, so 51.4; 12 heads of 64 x 2000
// keys 66.5 and 60.7), or for three units.  (Those workgroups have 128 registers, which int8 codes
// with two scales a tile fill.)
constexpr int cached_waves(int D, bool group) { return D == 64 ? (group ? 4 : 3) : 2; }

template <typename T, bool E4M3, int D, CodeForm FORM, bool GROUP>
__global__ void __launch_bounds__(GROUP ? 64 * kGroupWaves : 64)
__attribute__((amdgpu_waves_per_eu(cached_waves(D, GROUP), cached_waves(D, GROUP))))
cached_unit_kernel(WindowArgs a) {
  constexpr bool WHOLE = FORM != kAny;
  constexpr int NW = GROUP ? kGroupWaves : 1;
  constexpr int KL = D / 32, NDT = D / 32;  // loads of a key's half row; channels of a lane
  typedef typename Half<T>::op8 op8;
  // a wavefront's keys; of a workgroup, its partial rows
  constexpr int TILE = kTileKeys * D, SLOT = GROUP ? kFewRows * D * 4 : TILE;
  __shared__ __attribute__((aligned(1024))) char s_k[NW][SLOT];
  __shared__ float2 s_ml[NW][kFewRows];
  const int lane = threadIdx.x & 63, hf = lane >> 5, lr = lane & 31;
  const int wave = GROUP ? uniform_int(static_cast<int>(threadIdx.x) >> 6) : 0;

  const int w = divide(static_cast<int>(blockIdx.x), a.by_Hk);
  Unit u;
  if constexpr (GROUP) {
    const Request r = request_of<true>(a, w);
    u = {w, wave, kGroupWaves, 0, {uniform_int(r.k_len), uniform_int(r.q_len)}};
  } else {
    u = find_unit<false>(a, w, lane);
    if (u.b < 0) return;
  }
  Place p;
  p.b = u.b;
  p.hk = static_cast<int>(blockIdx.x) - w * a.Hk;
  p.row0 = 0;
  p.n_rows = u.r.q_len * a.G;
  if (p.n_rows == 0) return;
  p.k_len = u.r.k_len;
  p.shift = u.r.k_len - u.r.q_len;
  p.shares = u.shares;
  const KeyRange first = row_range(a, p, 0), last = row_range(a, p, p.n_rows - 1);
  p.tiles = tiles_of(a, first, last);
  share_of(p, u.share);

  // The lane's row of the queries: step st of the products takes the channels of 8 bytes st & 1
  // of load st / 2.
  v8hf q_op[2 * KL];
  float c_row, less;  // of the products q . (c + kMore) / kUnit: a factor, and what is added
  {
    const Row my = row_of(a, p, lr);
    const T* const row = static_cast<const T*>(a.q) + p.b * a.sq[0] +
                         static_cast<int64_t>(my.qi) * a.sq[1] + my.head * a.sq[2];
    op8 raw[2 * KL];
    float most = 0.0f;
#pragma unroll
    for (int st = 0; st < 2 * KL; ++st) {
      raw[st] = *reinterpret_cast<const op8*>(row + (st >> 1) * 32 + hf * 16 + (st & 1) * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(static_cast<float>(raw[st][i])));
    }
    const int k = row_shift(pair_max(most));
    const float up = power_of(k);
#pragma unroll
    for (int st = 0; st < 2 * KL; ++st) q_op[st] = scaled8<T>(raw[st], up);
    const float unit = a.scale_log2 * power_of(-k);
    c_row = unit * Widen<E4M3>::kUnit;
    less = E4M3 ? 0.0f : -Widen<E4M3>::kMore / Widen<E4M3>::kUnit * pair_sum(sum_of<2 * KL>(q_op));
  }

  // A tile's keys: load i takes rows i RPC + lane / CPR, chunks of 16 bytes, which lie in LDS
  // swizzled by row so that the reads of a chunk of 16 keys meet no bank twice.  The lane's key is
  // lr, its channels those of chunks 2 i + hf; its channels of the values of key 8 (r / 4) + 4 hf + r % 4 are
  // NDT lr and the next ones.
  constexpr int CPR = D / 16, RPC = 64 / CPR, LOADS = kTileKeys / RPC;
  auto swizzle = [](int row) __attribute__((always_inline)) -> int {
    return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3;
  };
  CodeStream<FORM, WindowArgs> codes(a, p);
  const uint32_t krb = codes.krb, vrb = codes.vrb;
  const int crow = lane / CPR;
  const int k_lo = crow * static_cast<int>(krb) + lane % CPR * 16;
  v4i kr[LOADS];
  auto load_k = [&]() __attribute__((always_inline)) {
    const char* from = codes.half(0).k;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      if (!WHOLE && i * RPC == 16) from = codes.half(1).k;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(from), 0, (WHOLE ? 32 : 16) * static_cast<int>(krb), kRsrcWord3);
      kr[i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
          rs, k_lo, (WHOLE ? i * RPC : i * RPC & 15) * static_cast<int>(krb), 0));
    }
  };
  char* const slot = s_k[wave];
  int k_to[LOADS];
#pragma unroll
  for (int i = 0; i < LOADS; ++i)
    k_to[i] = i * 1024 + crow * D + ((lane % CPR) ^ swizzle(i * RPC + crow)) * 16;
  constexpr int AT = GROUP && D == 64 ? 1 : KL;  // (registers that are short hold one of two)
  int k_at[AT];
#pragma unroll
  for (int i = 0; i < AT; ++i) k_at[i] = lr * D + (((2 * i + hf) ^ swizzle(lr)) * 16);
  // rows 4 hf + 0 .. 3; the others are 8, 16 and 24 further (registers that are short hold one)
  constexpr int VL = GROUP && D == 64 ? 1 : 4;
  int v_lo[VL];
#pragma unroll
  for (int j = 0; j < VL; ++j) v_lo[j] = static_cast<int>((4 * hf + j) * vrb + NDT * lr);
  auto load_v = [&](uint32_t (&v)[16]) __attribute__((always_inline)) {
    const char* from = codes.half(0).v;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (!WHOLE && h == 1) from = codes.half(1).v;
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(from), 0, (WHOLE ? 32 : 16) * static_cast<int>(vrb), kRsrcWord3);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int off = (8 * (j >> 2) + (VL == 1 ? j & 3 : 0) + (WHOLE ? 16 * h : 0)) *
                        static_cast<int>(vrb);
        if constexpr (NDT == 4)
          v[8 * h + j] = static_cast<uint32_t>(
              __builtin_amdgcn_raw_buffer_load_b32(rs, v_lo[j & (VL - 1)], off, 0));
        else
          v[8 * h + j] = static_cast<uint16_t>(
              __builtin_amdgcn_raw_buffer_load_b16(rs, v_lo[j & (VL - 1)], off, 0));
      }
    }
  };

  const float* const ks = a.ks + p.hk * a.sks[2];
  const float* const vs = a.vs + p.hk * a.svs[2];
  uint32_t v[16];
  TileRef<FORM> cur = codes.ref;
  load_k();
  load_v(v);
  codes.next();
  Scales<FORM> sc = scales_of(cur, ks, vs);
  v16f o_acc[NDT];
#pragma unroll
  for (int x = 0; x < NDT; ++x)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[x][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;
  uint32_t unit = kLeastUnit;  // of the row's accumulators
  constexpr int kShift = Half<_Float16>::kShift;

  // `codes` stands at the tile behind the present one: its keys are asked for as soon as the
  // present ones are in LDS, its values as soon as the present ones are in operands.
  for (int s = 0; s < p.steps; ++s) {
    const int key = cur.key, there = cur.there;
    const Scales<FORM> ns = sc;
#pragma unroll
    for (int i = 0; i < LOADS; ++i) *reinterpret_cast<v4i*>(slot + k_to[i]) = kr[i];
    const bool more = s + 1 < p.steps;
    cur = codes.ref;
    if (more) load_k();
    v4i kc[KL];
    int second = 32;
    asm volatile("" : "+s"(second));
#pragma unroll
    for (int i = 0; i < KL; ++i)
      kc[i] = *reinterpret_cast<const v4i*>(slot + (i < AT ? k_at[i] : k_at[0] ^ second));
    v16f s_acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) s_acc[r] = 0.0f;
#pragma unroll
    for (int i = 0; i < KL; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        s_acc = Half<_Float16>::mfma(
            widen8<E4M3, false>(static_cast<uint32_t>(kc[i][2 * j]),
                                static_cast<uint32_t>(kc[i][2 * j + 1])),
            q_op[2 * i + j], s_acc);
    sc = scales_of(cur, ks, vs);
    // logits in log2 units: r < 8 of the first half's keys, the others of the second's
    constexpr int N = Scales<FORM>::N;
    const float c0 = c_row * ns.k[0], c1 = c_row * ns.k[N - 1];
    float rv[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) rv[r] = (s_acc[r] + less) * (r < 8 ? c0 : c1);
    const bool inside = there == 3 && key + kTileKeys <= first.hi &&
                        (key >= last.lo || key + kTileKeys <= a.sinks);
    uint64_t sees0 = ~0ull, sees1 = ~0ull;  // lanes of rows that see a key of the halves
    if (!inside) {
      const int at = lane_again();
      const uint32_t all = seen_keys(late_args(), p, at & 31, key, there);
      const uint32_t seen = all >> (at >> 5) * 4;
#pragma unroll
      for (int r = 0; r < 16; ++r)
        rv[r] = (seen >> (8 * (r >> 2) + (r & 3))) & 1u ? rv[r] : -INFINITY;
      sees0 = __ballot((all & (N == 1 ? ~0u : 0xffffu)) != 0);
      sees1 = N == 1 ? sees0 : __ballot((all & 0xffff0000u) != 0);
    }
    // the scales of the values that the row sees, relative to the largest so far
    const float top = fmaxf(in_lanes(sees0, ns.v[0]), in_lanes(sees1, ns.v[N - 1]));
    if (__ballot(__float_as_uint(top) >= unit) != 0) {
      const float f = raise_unit(unit, top);
#pragma unroll
      for (int x = 0; x < NDT; ++x)
#pragma unroll
        for (int r = 0; r < 16; ++r) o_acc[x][r] *= f;
    }
    const float f0 = in_lanes(sees0, ns.v[0] * per_unit(unit));
    const float f1 = in_lanes(sees1, ns.v[N - 1] * per_unit(unit));
    v8hf p_op[2];
    auto exps = [&]() __attribute__((always_inline)) -> float {
      const float bias = m_run == -INFINITY ? 0.0f : -m_run;
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float e = __builtin_amdgcn_exp2f(rv[r] + bias);
        p_op[r >> 3][r & 7] = static_cast<_Float16>(e * (r < 8 ? f0 : f1));
        sum[r & 3] += e;
      }
      return (sum[0] + sum[1]) + (sum[2] + sum[3]);
    };
    float part = exps();
    if (__ballot(m_run == -INFINITY || !(part <= kTauPow * (1 << kShift))) != 0) {
      float rmax = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) rmax = fmaxf(rmax, rv[r]);
      rmax = pair_max(rmax);
      const float m_blk = rmax == -INFINITY ? -INFINITY : rmax - kShift;
      if (__ballot(m_blk > m_run + kTau) != 0) {
        const float m_new = fmaxf(m_run, m_blk);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int x = 0; x < NDT; ++x)
#pragma unroll
          for (int r = 0; r < 16; ++r) o_acc[x][r] *= alpha;
        m_run = m_new;
        part = exps();
      }
    }
    l_run += part;
    uint32_t tamed[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) tamed[r] = Widen<E4M3>::tame(Widen<E4M3>::finite(v[r]));
    if (more) {
      load_v(v);
      codes.next();
    }
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int x = 0; x < NDT; ++x)
        o_acc[x] = Half<_Float16>::mfma(column8<E4M3>(x, tamed + 8 * h), p_op[h], o_acc[x]);
  }

  // The end of the rows: lane (row, hf) holds channels 32 g' + ... : register r of product x is
  // channel NDT (8 (r / 4) + 4 hf + r % 4) + x.
  // (the thread's place is found anew: the loop leaves no registers to hold it)
  LateArgs& e = late_args();
  const int at_end = static_cast<int>(
      __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)));
  const int row_end = at_end & 31, hf_end = at_end >> 5;
  const Row my = row_of(e, p, row_end);
  const float l = pair_sum(l_run);
  const float inv = l > 0.0f ? __uint_as_float(unit) / l : l;  // (a NaN sum stays one)
  auto value = [&](int r, int x) __attribute__((always_inline)) -> float {
    return l == 0.0f ? 0.0f : o_acc[x][r] * (1 << Widen<E4M3>::kShift) * inv;
  };
  const bool live = row_end < p.n_rows;
  if (GROUP || p.shares > 1) {
    const int64_t ws_row = GROUP ? 0 : static_cast<int64_t>(blockIdx.x) * e.Lq * e.G;
    float* const part_o =
        GROUP ? reinterpret_cast<float*>(slot) : e.ws_o + ws_row * D;
    float2* const part_ml = GROUP ? s_ml[wave] : e.ws_ml + ws_row;
    if (live) {
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float* const at = part_o + row_end * D + NDT * (8 * (r >> 2) + 4 * hf_end + (r & 3));
#pragma unroll
        for (int x = 0; x < NDT; ++x) at[x] = value(r, x);
      }
      if (hf_end == 0)
        part_ml[row_end] = make_float2(l > 0.0f ? m_run : (l == 0.0f ? -INFINITY : l), l);
    }
  } else if (live) {
    T* const op = static_cast<T*>(e.out) + p.b * e.so[0] + static_cast<int64_t>(my.qi) * e.so[1] +
                  my.head * e.so[2];
#pragma unroll
    for (int r = 0; r < 16; r += 4 / NDT) {
      typename Half<T>::op4 w4;
#pragma unroll
      for (int x = 0; x < 4; ++x) w4[x] = static_cast<T>(value(r + x / NDT, x % NDT));
      *reinterpret_cast<typename Half<T>::op4*>(
          op + NDT * (8 * (r >> 2) + 4 * hf_end + (r & 3))) = w4;
    }
    if (hf_end == 0 && e.lse)
      e.lse[(static_cast<int64_t>(p.b) * e.Hq + my.head) * e.Lq + my.qi] =
          l == 0.0f ? -INFINITY : (m_run + __log2f(l)) * 0.69314718055994531f;
  }
  if constexpr (GROUP) {
    __syncthreads();
    for (int i = 64 * wave + at_end; i < p.n_rows * (D / 4); i += 64 * NW) {
      const int row = i / (D / 4), c = i % (D / 4) * 4;
      float mx = -INFINITY;
#pragma unroll
      for (int s = 0; s < NW; ++s) mx = fmaxf(mx, s_ml[s][row].x);
      v4f acc = {0.0f, 0.0f, 0.0f, 0.0f};
      float sum = 0.0f;
#pragma unroll
      for (int s = 0; s < NW; ++s) {
        const float2 ml = s_ml[s][row];
        if (ml.x == -INFINITY) continue;
        const float f = ml.y * __builtin_amdgcn_exp2f(ml.x - mx);
        sum += f;
        const v4f o = *reinterpret_cast<const v4f*>(s_k[s] + (row * D + c) * 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = join(f, o[i], acc[i]);
      }
      const Row r = row_of(e, p, row);
      typename Half<T>::op4 out;
#pragma unroll
      for (int i = 0; i < 4; ++i) out[i] = static_cast<T>(sum == 0.0f ? 0.0f : acc[i] / sum);
      *reinterpret_cast<typename Half<T>::op4*>(
          static_cast<T*>(e.out) + p.b * e.so[0] + static_cast<int64_t>(r.qi) * e.so[1] +
          r.head * e.so[2] + c) = out;
      if (e.lse && c == 0)
        e.lse[(static_cast<int64_t>(p.b) * e.Hq + r.head) * e.Lq + r.qi] =
            sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
    }
  }
}

template <typename T, bool E4M3, int D, CodeForm FORM>
static int launch(WindowArgs& a, int64_t units, hipStream_t s) {
  if (a.units == 0) {
    const dim3 grid(static_cast<unsigned>(a.B * a.Hk)), block(64 * kGroupWaves);
    cached_unit_kernel<T, E4M3, D, FORM, true><<<grid, block, 0, s>>>(a);
    return launch_status();
  }
  cached_unit_kernel<T, E4M3, D, FORM, false>
      <<<dim3(static_cast<unsigned>(units)), dim3(64), 0, s>>>(a);
  return launch_unit_merge(a, std::is_same<T, __bf16>::value ? 0 : 1, D, s);
}

template <typename T, bool E4M3, int D>
static int launch_form(WindowArgs& a, int64_t units, hipStream_t s) {
  switch (code_form(a)) {
    case kWhole: return launch<T, E4M3, D, kWhole>(a, units, s);
    case kHalves: return launch<T, E4M3, D, kHalves>(a, units, s);
    default: return launch<T, E4M3, D, kAny>(a, units, s);
  }
}
template <typename T>
static int launch_type(WindowArgs& a, bool e4m3, int64_t D, int64_t units, hipStream_t s) {
  if (e4m3)
    return D == 128 ? launch_form<T, true, 128>(a, units, s) : launch_form<T, true, 64>(a, units, s);
  return D == 128 ? launch_form<T, false, 128>(a, units, s) : launch_form<T, false, 64>(a, units, s);
}

int launch_cached_units(WindowArgs& a, int type, bool e4m3, int64_t D, int64_t units,
                        hipStream_t s) {
  return type == 0 ? launch_type<__bf16>(a, e4m3, D, units, s)
                   : launch_type<_Float16>(a, e4m3, D, units, s);
}

}  // namespace rcsa
