// Attention over pages of 8-bit codes, blocks of 128 rows: window_tile.h's work with a tile's
// codes copied to LDS as they are, three tiles ahead of the products, and made fp16 by the
// wavefront that copied them (once a workgroup, not once a wavefront) one tile ahead.
//
// Bound by the matrix and the vector pipe, whose times add within a wavefront: four frames of 880
// rows on the last twenty of 44 and the first, 24 heads of D 128 in int8 pages of 128 keys, 890 to
// 940 us by card, 850 to 900 TFLOP/s, the matrix pipe 46% and the vector pipe 50% busy at 2.0 GHz,
// no bank conflicts.  There, on a card that takes 888: codes through registers ahead of LDS 1359 us;
// through LDS, three workgroups on a compute unit 1038; places carried from tile to tile instead of
// found for each 931; keys as subnormal fp16 numbers (a byte permutation alone) 913.  Without the
// scales' loads, whose scalar returns every wait for LDS waits for, 862 (a wrong result).
#include "cached_attn.h"

namespace rcsa {

// RowTile's step with a scale for each half of a tile's keys (a lane half's 16).
template <int D>
struct CodeTile : RowTile<_Float16, D> {
  using R = RowTile<_Float16, D>;
  using O = Half<_Float16>;
  // The products are q . (c + 128) 2^-24 for int8 codes: a logit in log2 units is the product
  // times c_row times the key's scale, and c_less times it.
  float c_row, c_less;
  uint32_t unit;  // of the row's accumulators
  // what a tile's scales give: a product's factor, what is added to it (c_less times the key's
  // scale and log2 of the weights' factor f), 1 / f
  float c, more, inv_f;

  // A key's and a value's scale of the lane's half, 0 where the row sees none of it; `top`: the
  // larger value scale of the row's halves.
  __device__ __forceinline__ void take(float ks, float vs, float top) {
    if (__ballot(__float_as_uint(top) >= unit) != 0) {
      const float f = raise_unit(unit, top);
#pragma unroll
      for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) this->o_acc[dt][r] *= f;
    }
    c = fmaxf(c_row * ks, 0x1p-126f);  // (0 * -inf is NaN)
    const float f = fmaxf(vs * per_unit(unit), 0x1p-60f);
    more = fmaf(c_less, ks, __builtin_amdgcn_logf(f));
    inv_f = __builtin_amdgcn_rcpf(f);
  }

  template <CodeForm FORM, typename Take, typename Bits, typename Pre>
  __device__ __forceinline__ void step8(const char* tile, bool inside, Take&& scales, Bits&& bits,
                                        Pre&& prefetch) {
    // (the chunks' places are sums modulo 2 of the first one's and theirs: registers are short)
    v4i kraw[R::QSTEPS];
    constexpr int HELD = FORM == kWhole ? 7 : 4;
    int far = 64;
    asm volatile("" : "+s"(far));
#pragma unroll
    for (int st = 0; st < R::QSTEPS; ++st)
      kraw[st] = *reinterpret_cast<const v4i*>(
          tile + (st < HELD ? this->k_off[st] : this->k_off[st - 4] ^ far));
    v16f s_acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) s_acc[r] = 0.0f;
#pragma unroll
    for (int st = 0; st < R::QSTEPS; ++st)
      s_acc = O::mfma(__builtin_bit_cast(v8hf, kraw[st]), this->q_op[st], s_acc);
    __builtin_amdgcn_sched_group_barrier(0x100, R::QSTEPS, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, R::QSTEPS, 0);
    __builtin_amdgcn_sched_barrier(0);
    if (FORM == kWhole) prefetch();
    float rv[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) rv[r] = s_acc[r];
    // the lanes that see a key: a block that a row does not see may have any scale, which must
    // neither raise its unit nor, of keys, add c_less times it to masked logits
    uint64_t seeing = ~0ull, sees0 = ~0ull, sees1 = ~0ull;  // of the lane's half; of each half
    if (!inside) {
      const uint32_t seen = bits();
      seeing = __ballot(seen != 0);
      sees0 = (seeing & 0xffffffffull) | seeing << 32;
      sees1 = (seeing >> 32) | (seeing & ~0xffffffffull);
#pragma unroll
      for (int r = 0; r < 16; ++r) rv[r] = ((seen >> r) & 1u) ? rv[r] : -INFINITY;
    }
    scales(seeing, sees0, sees1);
    if (FORM != kWhole) prefetch();
    v8hf p_op[2];
    auto exps = [&]() __attribute__((always_inline)) -> float {
      const float bias = more + (this->m_run == -INFINITY ? 0.0f : -this->m_run);
      float lsum[4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
          const float e = __builtin_amdgcn_exp2f(fmaf(rv[8 * u + jj], c, bias));
          p_op[u][jj] = static_cast<_Float16>(e);
          if (u == 0 && jj < 4) lsum[jj] = e;
          else lsum[jj & 3] += e;
        }
      return (lsum[0] + lsum[1]) + (lsum[2] + lsum[3]);
    };
    float part = exps();
    if (__ballot(this->m_run == -INFINITY || !(part <= kTauPow * (1 << O::kShift))) != 0) {
      float rmax = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) rmax = fmaxf(rmax, rv[r]);
      rmax = pair_max(fmaf(rmax, c, more + __builtin_amdgcn_logf(inv_f)));
      const float m_blk = rmax == -INFINITY ? -INFINITY : rmax - O::kShift;
      if (__ballot(m_blk > this->m_run + kTau) != 0) {
        const float m_new = fmaxf(this->m_run, m_blk);
        const float alpha =
            m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(this->m_run - m_new);
        this->l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) this->o_acc[dt][r] *= alpha;
        this->m_run = m_new;
        part = exps();
      }
    }
    this->l_run = fmaf(part, inv_f, this->l_run);
    int v0 = this->v_off[0];
    asm volatile("" : "+v"(v0));
    auto v_group = [&](int u, v8hf (&op)[R::NDT]) __attribute__((always_inline)) {
#pragma unroll
      for (int dt = 0; dt < R::NDT; ++dt) {
        const char* const p0 = tile + (v0 ^ (dt * 64)) + 8 * u * R::KROW;
        const auto lo = O::read_tr(p0);
        const auto hi = O::read_tr(p0 + 4 * R::KROW);
        op[dt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    };
    v8hf vop[2][R::NDT];
    v_group(0, vop[0]);
    v_group(1, vop[1]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < R::NDT; ++dt)
        this->o_acc[dt] = O::mfma(vop[u][dt], p_op[u], this->o_acc[dt]);
  }
};

template <typename T, bool E4M3, int D, CodeForm FORM>
__global__ void __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 3, D == 64 ? 4 : 3)))
cached_tile_kernel(WindowArgs a) {
  using C = CodeTile<D>;
  using R = RowTile<_Float16, D>;
  typedef typename Half<T>::op8 op8;
  constexpr int BM = 128;
  __shared__ __attribute__((aligned(1024))) char s_0[2 * R::TILE];
  __shared__ __attribute__((aligned(1024))) char s_1[2 * R::TILE];
  __shared__ __attribute__((aligned(1024))) char r_0[8192];
  __shared__ __attribute__((aligned(1024))) char r_1[8192];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform_int(tid >> 6);
  const int hf = lane >> 5, lr = lane & 31;

  const int xcd = static_cast<int>(blockIdx.x % kNumXcd);
  const int slot = static_cast<int>(blockIdx.x / kNumXcd);
  const int tail = slot - a.xcd_whole;
  Place p;
  p.shares = tail < 0 ? 1 : a.n_split;
  const int in_xcd = tail < 0 ? slot : a.xcd_whole + tail / a.n_split;
  const int share = tail < 0 ? 0 : tail % a.n_split;
  const ItemAt it = item_at(a, xcd, in_xcd);
  if (it.bh < 0) return;
  p.b = divide(it.bh, a.by_Hk);
  p.hk = it.bh - p.b * a.Hk;
  const Request rq = request_of<true>(a, p.b);
  const int q_len = uniform_int(rq.q_len);
  p.k_len = uniform_int(rq.k_len);
  p.n_rows = q_len * a.G;
  const int item_row0 = it.rblock * BM;
  if (item_row0 >= p.n_rows) return;
  p.row0 = item_row0 + wave * 32;
  p.shift = p.k_len - q_len;
  const int64_t per_tail = a.xcd_items - a.xcd_whole;
  const int64_t ws_row =
      (share * per_tail * kNumXcd + xcd * per_tail + in_xcd - a.xcd_whole) * BM + wave * 32;
  const KeyRange w_first = row_range(a, p, p.row0), w_last = row_range(a, p, p.row0 + 31);
  p.tiles = tiles_of(a, row_range(a, p, item_row0), row_range(a, p, item_row0 + BM - 1));
  share_of(p, share);

  C t;
  t.init(lane);
  t.unit = kLeastUnit;
  {
    const Row r = row_of(a, p, p.row0 + lr);
    const T* const row = static_cast<const T*>(a.q) + p.b * a.sq[0] +
                         static_cast<int64_t>(r.qi) * a.sq[1] + r.head * a.sq[2];
    op8 raw[R::QSTEPS];
    float most = 0.0f;
#pragma unroll
    for (int st = 0; st < R::QSTEPS; ++st) {
      raw[st] = *reinterpret_cast<const op8*>(row + (hf * R::QSTEPS + st) * 8);
#pragma unroll
      for (int i = 0; i < 8; ++i) most = fmaxf(most, fabsf(static_cast<float>(raw[st][i])));
    }
    const int k = row_shift(pair_max(most));
    const float up = power_of(k);
#pragma unroll
    for (int st = 0; st < R::QSTEPS; ++st) t.q_op[st] = scaled8<T>(raw[st], up);
    const float unit = a.scale_log2 * power_of(-k);
    t.c_row = unit * Widen<E4M3>::kUnit;
    t.c_less = E4M3 ? 0.0f : -Widen<E4M3>::kMore * unit * pair_sum(sum_of<R::QSTEPS>(t.q_op));
  }

  CodeStream<FORM, WindowArgs> codes(a, p);
  const uint32_t krb = codes.krb, vrb = codes.vrb;

  // Copies: a wavefront moves rows 8 w .. 8 w + 7 of a tile, which lie in its half w / 2, as they
  // are into its part of a slot (D 64: the lanes past them zeros), 16 bytes a lane.
  constexpr int LPR = D / 16;  // lanes of a row
  const int in_half = (8 * wave + lane / LPR) & 15;
  const uint32_t none = lane < 8 * LPR ? 0u : 0x80000000u;
  const uint32_t k_lo = (in_half * krb + lane % LPR * 16) | none;
  const uint32_t v_lo = (in_half * vrb + lane % LPR * 16) | none;
  auto stage = [&](char* dst) __attribute__((always_inline)) {
    const auto h = codes.half(wave >> 1);
    buffer_copy16(const_cast<char*>(h.k), 16 * static_cast<int>(krb), k_lo, dst + wave * 2048);
    buffer_copy16(const_cast<char*>(h.v), 16 * static_cast<int>(vrb), v_lo,
                  dst + wave * 2048 + 1024);
  };
  // Its own copies, landed, become fp16 in the tile: lane l the 8 codes of chunk l % CPR of rows
  // 8 w + l / CPR and, D 128, the one 4 further (its swizzle: K's chunk ^ 4).  Whole rows at a
  // time, so that the writes of a row meet no bank twice.
  const int trow = 8 * wave + lane / R::CPR, chunk = lane % R::CPR;
  const int raw = wave * 2048 + lane * 8;
  const int k_at = trow * R::KROW + ((chunk ^ (swz_k<R::KROW>(trow) & (R::CPR - 1))) * 16);
  const int v_at = R::TILE + trow * R::KROW + ((chunk ^ (swz_v(trow) & (R::CPR - 1))) * 16);
  auto widen = [&](const char* src, char* dst) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < D / 64; ++i) {
      const v2u k = *reinterpret_cast<const v2u*>(src + raw + 512 * i);
      v2u v = *reinterpret_cast<const v2u*>(src + raw + 1024 + 512 * i);
      if (Widen<E4M3>::odd(v[0], v[1]))
#pragma unroll
        for (int j = 0; j < 2; ++j) v[j] = Widen<E4M3>::finite(v[j]);
      *reinterpret_cast<v8hf*>(dst + (i == 0 ? k_at : (k_at ^ 64) + 4 * R::KROW)) =
          widen8<E4M3, false>(k[0], k[1]);
      *reinterpret_cast<v8hf*>(dst + v_at + i * 4 * R::KROW) =
          widen8<E4M3, true>(v[0], v[1]);
    }
  };

  // Tile j is in slot j % 2 as fp16, written during step j - 1 (every wavefront has left step
  // j - 2 by then); its codes landed in raw slot j % 2, asked for during step j - 3.
  // One scale a tile is asked for by a scalar load, used where it differs from the last one's.
  // Scales of halves come by vector loads, ahead of a later tile's copies: scalar ones return out
  // of order, so that waits for LDS would wait for them too (2926 queries on 4737 keys in pages of
  // 48, 24 heads 285 us, so 271; 318 on 862 in pages of 16 30.4 and 29.3; with one scale a tile the
  // case above 912, and 935 that way).
  const float* const ks = a.ks + p.hk * a.sks[2];
  const float* const vs = a.vs + p.hk * a.svs[2];
  typedef TileRef<FORM> Ref;
  Ref e0 = codes.ref, e1, e2;
  stage(r_0);
  __builtin_amdgcn_sched_barrier(0);
  codes.next();
  e1 = codes.ref;
  stage(r_1);
  __builtin_amdgcn_sched_barrier(0);
  codes.next();
  e2 = codes.ref;
  float k_scale, v_scale;
  auto load_scales = [&](const Ref& e) __attribute__((always_inline)) {
    if constexpr (FORM == kWhole) {
      const Scales<FORM> sc = scales_of(e, ks, vs);
      k_scale = sc.k[0];
      v_scale = sc.v[0];
    } else {
      int ki = hf ? e.k[1] : e.k[0], vi = hf ? e.v[1] : e.v[0];
      k_scale = ks[ki];
      v_scale = vs[vi];
    }
  };
  load_scales(e0);
  // (the first tile's copies have landed; of scales by vector loads, all: what the barriers
  // below count begins with the next copies)
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(FORM == kWhole ? 2 : 0));
  widen(r_0, s_0);
  __builtin_amdgcn_sched_barrier(0);  // (its codes are in registers)
  stage(r_0);
  codes.next();
  uint32_t had_k = ~0u, had_v = ~0u;  // (the scales of the tile before: none)
  auto iteration = [&](auto slot_c) __attribute__((always_inline)) {
    constexpr int J = decltype(slot_c)::value;
    char* const tile = J == 0 ? s_0 : s_1;
    char* const fill = J == 0 ? s_1 : s_0;
    char* const raw_slot = J == 0 ? r_1 : r_0;
    // (behind the copies that have to have landed: a tile's, and its scales)
    if constexpr (FORM == kWhole)
      asm volatile("s_waitcnt vmcnt(2) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    else
      asm volatile("s_waitcnt vmcnt(4) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    const int key = e0.key, there = e0.there;
    const float kn = k_scale, vn = v_scale;
    e0 = e1;
    e1 = e2;
    e2 = codes.ref;
    const bool inside = key >= 0 && there == 3 && key + kTileKeys <= w_first.hi &&
                        (key >= w_last.lo || key + kTileKeys <= a.sinks);
    t.template step8<FORM>(
        tile, inside,
        [&](uint64_t seeing, uint64_t sees0, uint64_t sees1) __attribute__((always_inline)) {
          if constexpr (FORM == kWhole) {
            if (!inside || __float_as_uint(kn) != had_k || __float_as_uint(vn) != had_v) {
              const float v = in_lanes(sees0 | sees1, vn);
              t.take(in_lanes(sees0 | sees1, kn), v, v);
            }
            had_k = inside ? __float_as_uint(kn) : ~0u;
            had_v = __float_as_uint(vn);
          } else {
            const float of_half = scale_or_0(vn);
            auto of_lane = [&](int l) __attribute__((always_inline)) -> float {
              return __uint_as_float(static_cast<uint32_t>(
                  __builtin_amdgcn_readlane(static_cast<int>(__float_as_uint(of_half)), l)));
            };
            t.take(in_lanes(seeing, scale_or_0(kn)), in_lanes(seeing, of_half),
                   fmaxf(in_lanes(sees0, of_lane(0)), in_lanes(sees1, of_lane(32))));
          }
        },
        [&]() __attribute__((always_inline)) {
          return key < 0 ? 0u : seen_bits(late_args(), p, p.row0 + lr, hf, key, there);
        },
        [&]() __attribute__((always_inline)) {
          widen(raw_slot, fill);
          if constexpr (FORM != kWhole) load_scales(e0);
          __builtin_amdgcn_sched_barrier(0);
          stage(raw_slot);
          if constexpr (FORM == kWhole) load_scales(e0);
          codes.next();
        });
  };
  const int rounds = (p.steps + 1) / 2;
  for (int rd = 0; rd < rounds; ++rd) {
    iteration(std::integral_constant<int, 0>{});
    iteration(std::integral_constant<int, 1>{});
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // trailing copies land before the slots are freed

  // the end of the wavefront's rows
  LateArgs& e = late_args();
  const float l = pair_sum(t.l_run), m = t.m_run;
  const float inv = l > 0.0f ? __uint_as_float(t.unit) / l : l;  // (a NaN sum stays one)
#pragma unroll
  for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r)
      t.o_acc[dt][r] = l == 0.0f ? 0.0f : t.o_acc[dt][r] * (1 << Widen<E4M3>::kShift) * inv;
  const Row my = row_of(e, p, p.row0 + lr);
  if (!my.live) return;
  if (p.shares > 1) {
    float* const wp = e.ws_o + (ws_row + lr) * D + 4 * hf;
#pragma unroll
    for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g)
        *reinterpret_cast<v4f*>(wp + 32 * dt + 8 * g) =
            v4f{t.o_acc[dt][4 * g], t.o_acc[dt][4 * g + 1], t.o_acc[dt][4 * g + 2],
                t.o_acc[dt][4 * g + 3]};
    if (hf == 0)
      e.ws_ml[ws_row + lr] = make_float2(l > 0.0f ? m : (l == 0.0f ? -INFINITY : l), l);
    return;
  }
  T* const op = static_cast<T*>(e.out) + p.b * e.so[0] + static_cast<int64_t>(my.qi) * e.so[1] +
                my.head * e.so[2] + 4 * hf;
#pragma unroll
  for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      typename Half<T>::op4 w;
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = static_cast<T>(t.o_acc[dt][4 * g + i]);
      *reinterpret_cast<typename Half<T>::op4*>(op + 32 * dt + 8 * g) = w;
    }
  if (hf == 0 && e.lse)
    e.lse[(static_cast<int64_t>(p.b) * e.Hq + my.head) * e.Lq + my.qi] =
        l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
}

template <typename T, bool E4M3, int D>
static void launch(WindowArgs& a, dim3 grid, hipStream_t s) {
  const dim3 block(256);
  switch (code_form(a)) {
    case kWhole: cached_tile_kernel<T, E4M3, D, kWhole><<<grid, block, 0, s>>>(a); break;
    case kHalves: cached_tile_kernel<T, E4M3, D, kHalves><<<grid, block, 0, s>>>(a); break;
    case kAny: cached_tile_kernel<T, E4M3, D, kAny><<<grid, block, 0, s>>>(a); break;
  }
}
template <typename T>
static void launch_type(WindowArgs& a, bool e4m3, int64_t D, dim3 grid, hipStream_t s) {
  if (e4m3) D == 128 ? launch<T, true, 128>(a, grid, s) : launch<T, true, 64>(a, grid, s);
  else D == 128 ? launch<T, false, 128>(a, grid, s) : launch<T, false, 64>(a, grid, s);
}

void launch_cached_tile(WindowArgs& a, int type, bool e4m3, int64_t D, dim3 grid, hipStream_t s) {
  if (type == 0) launch_type<__bf16>(a, e4m3, D, grid, s);
  else launch_type<_Float16>(a, e4m3, D, grid, s);
}

}  // namespace rcsa
