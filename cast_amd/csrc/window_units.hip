// Windowed attention of few rows (one new token of each request, or a few): at most 32
// rows of a key head.  Few keys: one workgroup of eight wavefronts a key head, which
// joins their shares in LDS.  Many: one wavefront a unit of the visible tiles of all
// requests, joined by a second launch.
//
// The keys and values are read once and bound the time, so what counts is bytes in
// flight (48 ragged requests of up to 32768 keys in pages of 16, 32 heads on 8: 326 us,
// 5.4 TB/s, and 10 us for the join; one token over 1024 of 2500 keys 7.5 and 4.1 us, the
// latency of two launches): a wavefront holds the next tile (16 KB at D 128) in registers
// while it works on the one in its own LDS, eight wavefronts to a compute unit, no
// barriers.  The loop is one tile long: a unit of a few tiles runs through little code that
// is not yet in the instruction cache.
#include "window_attn.h"

namespace rcsa {

template <typename T, int D, bool PAGED, bool GROUP>
__global__ void __launch_bounds__(GROUP ? 64 * kGroupWaves : 64)
__attribute__((amdgpu_waves_per_eu(D == 64 ? 3 : 2, D == 64 ? 3 : 2)))
window_unit_kernel(WindowArgs a) {
  using R = RowTile<T, D>;
  constexpr int NW = GROUP ? kGroupWaves : 1;
  constexpr int RPU = 1024 / R::KROW;          // rows of a 1 KiB load
  constexpr int UPH = 16 * R::KROW / 1024;     // loads of a half tile, K and V each
  __shared__ __attribute__((aligned(1024))) char tiles[NW][2 * R::TILE];
  __shared__ float2 s_ml[NW][kFewRows];
  const int lane = threadIdx.x & 63, hf = lane >> 5, lr = lane & 31;
  const int wave = GROUP ? uniform_int(static_cast<int>(threadIdx.x) >> 6) : 0;
  char* const tile = tiles[wave];

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

  const char* const kbase = static_cast<const char*>(a.k) +
                            ((PAGED ? 0 : p.b * a.sk[0]) + p.hk * a.sk[2]) * 2;
  const char* const vbase = static_cast<const char*>(a.v) +
                            ((PAGED ? 0 : p.b * a.sv[0]) + p.hk * a.sv[2]) * 2;
  const uint32_t krb = static_cast<uint32_t>(a.sk[1] * 2), vrb = static_cast<uint32_t>(a.sv[1] * 2);
  const int32_t* const table = PAGED ? a.table + p.b * a.table_stride : nullptr;

  // load i of a half: rows i RPU + lane / CPR, chunk lane % CPR; rows past the keys and
  // pages that are not there read zeros through ranges that end before them
  v4i kst[2 * UPH], vst[2 * UPH];
  const int lrow = lane / R::CPR, chunk = lane % R::CPR;
  const uint32_t k_lo = lrow * krb + chunk * 16, v_lo = lrow * vrb + chunk * 16;
  auto load = [&](const Step& s) __attribute__((always_inline)) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const HalfRows hr = half_rows<PAGED>(a, s, h, p.k_len, krb, vrb);
      const __amdgpu_buffer_rsrc_t kr = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(kbase) + hr.k, 0, hr.rows * static_cast<int>(krb), kRsrcWord3);
      const __amdgpu_buffer_rsrc_t vr = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<char*>(vbase) + hr.v, 0, hr.rows * static_cast<int>(vrb), kRsrcWord3);
#pragma unroll
      for (int i = 0; i < UPH; ++i) {
        kst[h * UPH + i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
            kr, static_cast<int>(k_lo + i * RPU * krb), 0, 0));
        vst[h * UPH + i] = __builtin_bit_cast(v4i, __builtin_amdgcn_raw_buffer_load_b128(
            vr, static_cast<int>(v_lo + i * RPU * vrb), 0, 0));
      }
    }
  };
  Step cur = step_of<PAGED>(a, p, table, 0);
  Step next = step_of<PAGED>(a, p, table, 1);
  R t;
  {
    const Row r = row_of(a, p, lr);
    t.load_q(static_cast<const T*>(a.q) + p.b * a.sq[0] + static_cast<int64_t>(r.qi) * a.sq[1] +
                 r.head * a.sq[2], hf);
  }
  load(cur);
  t.init(lane);
  // Q has landed before the loop (its waits there would drain the loads of the next tile)
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(4 * UPH));
  // LDS places of the loads: the swizzles are sums of a row's bits modulo 2, and load i adds
  // bits i RPU to the lane's (none that V's takes)
  const int k_at = lrow * R::KROW + ((chunk ^ (swz_k<R::KROW>(lrow) & (R::CPR - 1))) * 16);
  const int v_at = R::TILE + lrow * R::KROW + ((chunk ^ (swz_v(lrow) & (R::CPR - 1))) * 16);
  for (int s = 0; s < p.steps; ++s) {
#pragma unroll
    for (int i = 0; i < 2 * UPH; ++i) {
      const int kx = (swz_k<R::KROW>(i * RPU) & (R::CPR - 1)) * 16;
      *reinterpret_cast<v4i*>(tile + (k_at ^ kx) + i * 1024) = kst[i];
      *reinterpret_cast<v4i*>(tile + v_at + i * 1024) = vst[i];
    }
    const Step now = cur;
    cur = next;
    if (s + 1 < p.steps) load(cur);
    const int there = halves_there<PAGED>(a, now);
    const bool inside = there == 3 && now.key + kTileKeys <= first.hi &&
                        (now.key >= last.lo || now.key + kTileKeys <= a.sinks);
    t.template step<0>(tile, a.scale_log2, inside, [&]() __attribute__((always_inline)) {
      return seen_bits(a, p, lr, hf, now.key, there);
    }, [&]() __attribute__((always_inline)) { next = step_of<PAGED>(a, p, table, s + 2); },
       []() __attribute__((always_inline)) {});
  }
  if constexpr (!GROUP) {
    const int64_t ws_row = static_cast<int64_t>(blockIdx.x) * a.Lq * a.G;
    finish_rows<T, D, PAGED>(p, t, late_args().ws_o + ws_row * D,
                             late_args().ws_ml + ws_row, tile);
    return;
  }
  // the wavefronts' partial rows meet in LDS, each in its own tile's place
  static_assert(kFewRows * D * 4 <= 2 * R::TILE, "partial rows fit a wavefront's tiles");
  finish_rows<T, D, PAGED>(p, t, reinterpret_cast<float*>(tile), s_ml[wave], tile);
  __syncthreads();
  for (int i = threadIdx.x; i < p.n_rows * (D / 4); i += 64 * NW) {
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
      const v4f o = *reinterpret_cast<const v4f*>(tiles[s] + (row * D + c) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] = join(f, o[e], acc[e]);
    }
    const Row r = row_of(a, p, row);
    typename Half<T>::op4 out;
#pragma unroll
    for (int e = 0; e < 4; ++e)
      out[e] = static_cast<T>(sum == 0.0f ? 0.0f : acc[e] / sum);
    *reinterpret_cast<typename Half<T>::op4*>(
        static_cast<T*>(a.out) + p.b * a.so[0] + static_cast<int64_t>(r.qi) * a.so[1] +
        r.head * a.so[2] + c) = out;
    if (a.lse && c == 0)
      a.lse[(static_cast<int64_t>(p.b) * a.Hq + r.head) * a.Lq + r.qi] =
          sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
  }
}

// The units of every row joined: w_s = l_s 2^(m_s - M), out = sum w_s O_s / sum w_s.  A
// workgroup takes one row, its threads (share, 8 channels); the shares are added in a
// fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(256) window_unit_merge_kernel(WindowArgs a) {
  constexpr int CPR = D / 8, GROUPS = 256 / CPR;
  __shared__ float s_acc[GROUPS][D], s_sum[GROUPS], s_max[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int R = a.Lq * a.G;
  const int row = static_cast<int>(blockIdx.x) % R;
  const int bh = static_cast<int>(blockIdx.x) / R;
  const int b = divide(bh, a.by_Hk), hk = bh - b * a.Hk;
  const Unit u = find_unit<true>(a, b, lane);
  if (row >= u.r.q_len * a.G) return;
  const int shares = u.shares;
  if (shares <= 1) return;  // written by its only unit
  const int64_t first = static_cast<int64_t>(u.before) * a.Hk + hk;
  auto at = [&](int s) __attribute__((always_inline)) -> int64_t {
    return (first + static_cast<int64_t>(s) * a.Hk) * R + row;
  };
  const int c = tid % CPR, g = tid / CPR;
  // (the thread's first share is asked for ahead of the maximum: with scalar loads of a single
  // request's lengths one token over 1024 keys of 8 heads 11.0 us, so 10.6; over 4096 15.2, 14.8)
  float2 ml = make_float2(-INFINITY, 0.0f);
  float ov[8];
  if (g < shares) {
    ml = a.ws_ml[at(g)];
    Vec8<float>::load(a.ws_o + at(g) * D + c * 8, ov);
  }
  float mx = -INFINITY;
  for (int s = tid; s < shares; s += 256) mx = fmaxf(mx, a.ws_ml[at(s)].x);
  mx = wave_max(mx);
  if (lane == 0) s_max[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float sum = 0.0f;
  for (int s = g; s < shares; s += GROUPS) {
    if (s != g) {
      ml = a.ws_ml[at(s)];
      Vec8<float>::load(a.ws_o + at(s) * D + c * 8, ov);
    }
    if (ml.x == -INFINITY) continue;
    const float w = ml.y * __builtin_amdgcn_exp2f(ml.x - mx);
    sum += w;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = join(w, ov[j], acc[j]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) s_acc[g][c * 8 + j] = acc[j];
  if (c == 0) s_sum[g] = sum;
  __syncthreads();
  if (tid >= D) return;
  float total = 0.0f, o = 0.0f;
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    total += s_sum[i];
    o += s_acc[i][tid];
  }
  const int qi = divide(row, a.by_G), head = hk * a.G + row - qi * a.G;
  static_cast<T*>(a.out)[b * a.so[0] + qi * a.so[1] + head * a.so[2] + tid] =
      static_cast<T>(total == 0.0f ? 0.0f : o / total);
  if (a.lse && tid == 0)
    a.lse[(static_cast<int64_t>(b) * a.Hq + head) * a.Lq + qi] =
        total == 0.0f ? -INFINITY : (mx + __log2f(total)) * 0.69314718055994531f;
}

template <typename T, int D>
static int launch_units(WindowArgs& a, int64_t units, hipStream_t s) {
  const int64_t heads = static_cast<int64_t>(a.B) * a.Hk;
  if (a.units == 0) {
    const dim3 grid(static_cast<unsigned>(heads)), block(64 * kGroupWaves);
    if (a.table) window_unit_kernel<T, D, true, true><<<grid, block, 0, s>>>(a);
    else window_unit_kernel<T, D, false, true><<<grid, block, 0, s>>>(a);
    return launch_status();
  }
  const int64_t rows = heads * a.Lq * a.G;  // (at most 2^24, of 256 threads: units_fit)
  const dim3 grid(static_cast<unsigned>(units)), block(64);
  if (a.table) window_unit_kernel<T, D, true, false><<<grid, block, 0, s>>>(a);
  else window_unit_kernel<T, D, false, false><<<grid, block, 0, s>>>(a);
  window_unit_merge_kernel<T, D><<<dim3(static_cast<unsigned>(rows)), dim3(256), 0, s>>>(a);
  return launch_status();
}

int launch_window_units(WindowArgs& a, int type, int64_t D, int64_t units, hipStream_t s) {
  if (type == 0)
    return D == 128 ? launch_units<__bf16, 128>(a, units, s)
                    : launch_units<__bf16, 64>(a, units, s);
  return D == 128 ? launch_units<_Float16, 128>(a, units, s)
                  : launch_units<_Float16, 64>(a, units, s);
}

}  // namespace rcsa
