// Windowed attention, tiles of 128 rows: one pass over the visible keys with the
// running maximum and sum of the softmax.
//
// Work: a workgroup takes 128 rows of one key head (32 a wavefront, 4
// wavefronts) and streams the 32-key tiles that any of them sees: the tiles of
// the first keys, then those of the window.  Three workgroups share a compute
// unit, so that one's exponentials run beside another's matrix products.
// A tile's K and V go global -> LDS without registers into a ring of three
// slots; rows past the keys, and pages that are not there, land as zeros.
// S^T = K Q^T puts one query row in a lane (its 16 + 16 keys in the two lane
// halves), so a row's maximum and sum need one lane swap, and P^T is the second
// operand of O^T = V^T P^T as it stands.  Only the tiles at the window's edges
// are masked; a wavefront none of whose rows sees a tile only copies it.
#include "window_attn.h"

namespace rcsa {

template <typename T, int D, int NW_>
struct WindowCfg {
  static constexpr int NW = NW_, BM = 32 * NW, STAGES = 3;
  static constexpr int KROW = D * 2, CPR = KROW / 16;   // bytes and 16-byte chunks of a row
  static constexpr int QSTEPS = D / 16, NDT = D / 32;
  static constexpr int TILE = kTileKeys * KROW;         // bytes of a K (or V) tile
  static constexpr int RPU = 1024 / KROW;               // rows of a 1 KiB copy
  static constexpr int UPW = TILE / 1024 / NW;          // copies of a wavefront, K and V each
  static constexpr int OPS = 2 * UPW;
};

template <typename T, int D, bool PAGED, int NW>
__global__ void __launch_bounds__(64 * NW)
__attribute__((amdgpu_waves_per_eu(NW == 1 ? 1 : (D == 64 ? 4 : 3), D == 64 ? 4 : 3)))
window_kernel(WindowArgs a) {
  using C = WindowCfg<T, D, NW>;
  using O = Half<T>;
  typedef typename O::op8 op8;
  __shared__ __attribute__((aligned(1024))) char s_0[2 * C::TILE];
  __shared__ __attribute__((aligned(1024))) char s_1[2 * C::TILE];
  __shared__ __attribute__((aligned(1024))) char s_2[2 * C::TILE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = NW == 1 ? 0 : __builtin_amdgcn_readfirstlane(tid >> 6);
  const int hf = lane >> 5, lr = lane & 31;

  // The work of this workgroup: rows row0 .. of key head hk of request b, share `share` of
  // the `ns` shares of their tiles; its rows of the workspace start at ws_row.
  int b, hk, row0, share;
  uint32_t ns;
  int64_t ws_row;
  Request rq;
  if constexpr (NW > 1) {
    // XCD x (workgroups go round-robin) runs a contiguous run of items, so that neighbours
    // share most of their window in its L2, or every 8th from the longest on.
    const int xcd = static_cast<int>(blockIdx.x % kNumXcd);
    const int slot = static_cast<int>(blockIdx.x / kNumXcd);
    const int tail = slot - a.xcd_whole;
    ns = tail < 0 ? 1u : static_cast<uint32_t>(a.n_split);
    const int in_xcd = tail < 0 ? slot : a.xcd_whole + tail / a.n_split;
    share = tail < 0 ? 0 : tail % a.n_split;
    if (in_xcd >= a.xcd_items) return;
    const int64_t item = a.descending ? static_cast<int64_t>(in_xcd) * kNumXcd + xcd
                                      : static_cast<int64_t>(xcd) * a.xcd_items + in_xcd;
    if (item >= a.n_items) return;
    const uint32_t it = static_cast<uint32_t>(item), nrb = static_cast<uint32_t>(a.n_rblocks);
    const uint32_t heads = static_cast<uint32_t>(a.B * a.Hk);
    const int bh = static_cast<int>(a.descending ? it % heads : it / nrb);
    row0 = static_cast<int>(a.descending ? nrb - 1 - it / heads : it % nrb) * C::BM;
    b = bh / a.Hk;
    hk = bh - b * a.Hk;
    const int64_t n_tail = static_cast<int64_t>(a.xcd_items - a.xcd_whole) * kNumXcd;
    ws_row = (share * n_tail + xcd * (a.xcd_items - a.xcd_whole) + in_xcd - a.xcd_whole) * C::BM;
    rq = request_of(a, b);
  } else {
    const int w = static_cast<int>(blockIdx.x) / a.Hk;
    const Unit u = find_unit<false>(a, w, lane);
    if (u.b < 0) return;
    b = u.b;
    share = u.share;
    ns = static_cast<uint32_t>(u.shares);
    hk = static_cast<int>(blockIdx.x) - w * a.Hk;
    row0 = 0;
    ws_row = static_cast<int64_t>(blockIdx.x) * a.Lq * a.G;
    rq = u.r;
  }
  const int k_len = uniform_int(rq.k_len), q_len = uniform_int(rq.q_len);
  const int n_rows = q_len * a.G;
  if (row0 >= n_rows) return;
  const int shift = k_len - q_len;  // position of query 0

  // This lane's row; rows past the last stand at the last one's place, unwritten.  (Its
  // place and keys are found again where they are needed: registers are short.)
  struct Row {
    int row, qi, head;
    bool live;
  };
  auto my_row = [&]() __attribute__((always_inline)) -> Row {
    int row = row0 + wave * 32 + lr;
    asm volatile("" : "+v"(row));
    Row r;
    r.row = row;
    r.live = row < n_rows;
    const int at = r.live ? row : n_rows - 1;
    r.qi = at / a.G;
    r.head = hk * a.G + at - r.qi * a.G;
    return r;
  };

  // uniform ranges: of the item, and of this wavefront's first and last rows
  auto range_of = [&](int r) __attribute__((always_inline)) -> KeyRange {
    r = r < n_rows ? r : n_rows - 1;
    return key_range(a, r / a.G + shift, k_len);
  };
  const KeyRange i_first = range_of(row0), i_last = range_of(row0 + C::BM - 1);
  const KeyRange w_first = range_of(row0 + wave * 32), w_last = range_of(row0 + wave * 32 + 31);
  const Tiles tl = tiles_of(a, i_first, i_last);
  const int sink_n = tl.sink_n, win_t0 = tl.win_t0, all = tl.all();
  const int s_begin = static_cast<int>(static_cast<int64_t>(all) * share / ns);
  const int steps = static_cast<int>(static_cast<int64_t>(all) * (share + 1) / ns) - s_begin;

  op8 q_op[C::QSTEPS];
  {
    const Row r = my_row();
    const T* const qp = static_cast<const T*>(a.q) + b * a.sq[0] +
                        static_cast<int64_t>(r.qi) * a.sq[1] + r.head * a.sq[2];
#pragma unroll
    for (int st = 0; st < C::QSTEPS; ++st)
      q_op[st] = *reinterpret_cast<const op8*>(qp + (hf * C::QSTEPS + st) * 8);
  }

  v16f o_acc[C::NDT];
#pragma unroll
  for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) o_acc[dt][r] = 0.0f;
  float m_run = -INFINITY, l_run = 0.0f;

  const char* const kbase = static_cast<const char*>(a.k) +
                            ((PAGED ? 0 : b * a.sk[0]) + hk * a.sk[2]) * 2;
  const char* const vbase = static_cast<const char*>(a.v) +
                            ((PAGED ? 0 : b * a.sv[0]) + hk * a.sv[2]) * 2;
  const uint32_t krb = static_cast<uint32_t>(a.sk[1] * 2), vrb = static_cast<uint32_t>(a.sv[1] * 2);
  const uint32_t kpage = static_cast<uint32_t>(a.sk[0] * 2);  // (paged)
  const uint32_t vpage = static_cast<uint32_t>(a.sv[0] * 2);
  const int32_t* const table = PAGED ? a.table + b * a.table_stride : nullptr;

  // Copies: of four wavefronts, w moves rows 8w .. 8w + 7 of the tile (of its half w / 2 of
  // 16 rows, which lies in one page), RPU rows a copy, chunks swizzled by row; a
  // single one moves both halves.
  uint32_t k_lo[C::UPW], v_lo[C::UPW];
#pragma unroll
  for (int i = 0; i < C::UPW; ++i) {
    const int r = (wave * C::UPW + i) * C::RPU + lane / C::CPR;  // row of the tile
    const uint32_t in_half = static_cast<uint32_t>(r & 15);
    k_lo[i] = in_half * krb + (((lane % C::CPR) ^ (swz_k<C::KROW>(r) & (C::CPR - 1))) * 16);
    v_lo[i] = in_half * vrb + (((lane % C::CPR) ^ (swz_v(r) & (C::CPR - 1))) * 16);
  }
  // A step: its first key (-1: past the list) and, paged, the pages of its two halves
  // until they are staged, then whether they are there (bits 0 and 1).
  struct Step {
    int key, page0, page1;
  };
  struct Staged {
    int key, there;
  };
  auto key_of = [&](int s) __attribute__((always_inline)) -> int {
    const int t = s_begin + s;
    return s >= steps ? -1 : (t < sink_n ? t : win_t0 + t - sink_n) * kTileKeys;
  };
  auto page_ok = [&](int p) __attribute__((always_inline)) -> bool {
    return static_cast<uint32_t>(p) < static_cast<uint32_t>(a.n_pages);
  };
  // column of half tile h = key / 16 (scalar arithmetic: the unsigned division by an
  // invariant, two shifts and a high product)
  const uint32_t page = PAGED ? static_cast<uint32_t>(a.page) : 16u;
  auto col_of = [&](uint32_t h) __attribute__((always_inline)) -> uint32_t {
    const uint32_t t = __umulhi(a.page_mul, h);
    return (t + ((h - t) >> a.page_sh1)) >> a.page_sh2;
  };
  auto step_of = [&](int s) __attribute__((always_inline)) -> Step {
    Step r{key_of(s), 0, 0};
    if constexpr (PAGED) {  // (a half lies in one page: pages hold whole halves)
      const uint32_t key = r.key < 0 ? 0u : static_cast<uint32_t>(r.key);
      const uint32_t last = static_cast<uint32_t>(a.max_pages) - 1u;
      const uint32_t col0 = col_of(key >> 4);
      uint32_t col1 = col_of((key >> 4) + 1u);
      col1 = col1 < last ? col1 : last;
      r.page0 = ld_const(table + col0);
      r.page1 = ld_const(table + col1);
    }
    return r;
  };
  // copies [i0, i0 + n) of a step, all in half `half` of its tile
  auto stage_half = [&](const Step& s, char* dst, int half, int i0, auto n_c)
      __attribute__((always_inline)) {
    const uint32_t key = static_cast<uint32_t>(s.key < 0 ? 0 : s.key) + 16u * half;
    uint64_t krow, vrow;
    bool there = s.key >= 0;
    if constexpr (PAGED) {
      const int pg = half ? s.page1 : s.page0;
      there = there && page_ok(pg);
      const uint32_t slot = key - col_of(key >> 4) * page;
      // (32 x 32-bit scalar products: a page spans less than 4 GiB)
      const uint32_t at = there ? static_cast<uint32_t>(pg) : 0u;
      krow = static_cast<uint64_t>(at) * kpage + static_cast<uint64_t>(slot) * krb;
      vrow = static_cast<uint64_t>(at) * vpage + static_cast<uint64_t>(slot) * vrb;
    } else {
      krow = static_cast<uint64_t>(key) * krb;
      vrow = static_cast<uint64_t>(key) * vrb;
    }
    const int left = k_len - static_cast<int>(key);
    const int rows = __builtin_amdgcn_readfirstlane(
        !there || left <= 0 ? 0 : (left < 16 ? left : 16));
    char* const ks = const_cast<char*>(kbase) + krow;
    char* const vs = const_cast<char*>(vbase) + vrow;
    // (row strides are at least a row: a lane of row r < rows stays below)
    const int kn = rows * static_cast<int>(krb), vn = rows * static_cast<int>(vrb);
#pragma unroll
    for (int i = 0; i < decltype(n_c)::value; ++i) {
      buffer_copy16(ks, kn, k_lo[i0 + i], dst + (wave * C::UPW + i0 + i) * 1024);
      buffer_copy16(vs, vn, v_lo[i0 + i], dst + C::TILE + (wave * C::UPW + i0 + i) * 1024);
    }
  };
  auto stage = [&](const Step& s, char* dst) __attribute__((always_inline)) -> Staged {
    if constexpr (NW == 1) {
      stage_half(s, dst, 0, 0, std::integral_constant<int, C::UPW / 2>{});
      stage_half(s, dst, 1, C::UPW / 2, std::integral_constant<int, C::UPW / 2>{});
    } else {
      stage_half(s, dst, wave >> 1, 0, std::integral_constant<int, C::UPW>{});
    }
    return {s.key, PAGED ? (page_ok(s.page0) ? 1 : 0) + (page_ok(s.page1) ? 2 : 0) : 3};
  };

  // LDS read offsets (tile and step offsets are immediates)
  int k_off[C::QSTEPS];
  {
    const int r = key_perm(lr);
    const int sw = swz_k<C::KROW>(r) & (C::CPR - 1);
#pragma unroll
    for (int st = 0; st < C::QSTEPS; ++st)
      k_off[st] = r * C::KROW + (((hf * C::QSTEPS + st) ^ sw) * 16);
  }
  int v_off[C::NDT];
  {
    const int grp = lane >> 4, gi = lane & 15;
    const int r = 16 * (grp >> 1) + (gi >> 2);
    const int sw = swz_v(r) & (C::CPR - 1);
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt) {
      const int d = 32 * dt + 16 * (grp & 1) + 4 * (gi & 3);
      v_off[dt] = C::TILE + r * C::KROW + (((d >> 3) ^ sw) * 16) + (d & 7) * 2;
    }
  }
  v16f zero;
#pragma unroll
  for (int r = 0; r < 16; ++r) zero[r] = 0.0f;

  auto below = [&](int x) __attribute__((always_inline)) -> uint32_t {  // bits of keys < x
    const int n = x < 0 ? 0 : (x > 16 ? 16 : x);
    return (1u << n) - 1u;
  };
  // The scalar loads of a later step go out behind the first products (they return out of
  // order, so a wait for LDS behind them would wait for them too).
  auto compute = [&](const char* tile, const Staged& s, auto&& prefetch)
      __attribute__((always_inline)) {
    const bool pages = !PAGED || s.there == 3;
    // every row of the wavefront sees the whole tile
    const bool inside = pages && s.key + kTileKeys <= w_first.hi &&
                        (s.key >= w_last.lo || s.key + kTileKeys <= a.sinks);
    v4i kraw[C::QSTEPS];
#pragma unroll
    for (int st = 0; st < C::QSTEPS; ++st)
      kraw[st] = *reinterpret_cast<const v4i*>(tile + k_off[st]);
    v16f s_acc = zero;
#pragma unroll
    for (int st = 0; st < C::QSTEPS; ++st)
      s_acc = O::mfma(__builtin_bit_cast(op8, kraw[st]), q_op[st], s_acc);
    __builtin_amdgcn_sched_group_barrier(0x100, C::QSTEPS, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, C::QSTEPS, 0);
    __builtin_amdgcn_sched_barrier(0);
    prefetch();
    float rv[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) rv[r] = s_acc[r];
    if (!inside) {
      const KeyRange kr = key_range(a, my_row().qi + shift, k_len);
      const int sink = a.sinks < kr.hi ? a.sinks : kr.hi;
      const int k0 = s.key + 16 * hf;
      uint32_t bits = below(kr.hi - k0) & (~below(kr.lo - k0) | below(sink - k0));
      if (PAGED && !((s.there >> hf) & 1)) bits = 0;
#pragma unroll
      for (int r = 0; r < 16; ++r) rv[r] = ((bits >> r) & 1u) ? rv[r] : -INFINITY;
    }
    const float c = a.scale_log2;
    op8 p_op[2];
    auto exps = [&]() __attribute__((always_inline)) -> float {
      const float bias = m_run == -INFINITY ? 0.0f : -m_run;
      float lsum[4];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int jj = 0; jj < 8; ++jj) {
          const float e = __builtin_amdgcn_exp2f(fmaf(rv[8 * u + jj], c, bias));
          p_op[u][jj] = static_cast<T>(e);
          if (u == 0 && jj < 4) lsum[jj] = e;
          else lsum[jj & 3] += e;
        }
      return (lsum[0] + lsum[1]) + (lsum[2] + lsum[3]);
    };
    // the running maximum moves only when a term passes 2^kTau (a lane's partial
    // sum bounds its terms)
    float part = exps();
    if (__ballot(m_run == -INFINITY || !(part <= kTauPow)) != 0) {
      float rmax = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) rmax = fmaxf(rmax, rv[r]);
      rmax = pair_max(rmax);
      const float m_blk = rmax == -INFINITY ? -INFINITY : rmax * c;
      if (__ballot(m_blk > m_run + kTau) != 0) {
        const float m_new = fmaxf(m_run, m_blk);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o_acc[dt][r] *= alpha;
        m_run = m_new;
        part = exps();
      }
    }
    l_run += part;
    // (the reads of the second half of the keys are in flight beside the first half's
    // products)
    auto v_group = [&](int u, op8 (&op)[C::NDT]) __attribute__((always_inline)) {
#pragma unroll
      for (int dt = 0; dt < C::NDT; ++dt) {
        const char* const p0 = tile + v_off[dt] + 8 * u * C::KROW;
        const auto lo = O::read_tr(p0);
        const auto hi = O::read_tr(p0 + 4 * C::KROW);
        op[dt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    };
    op8 vop[2][C::NDT];
    v_group(0, vop[0]);
    v_group(1, vop[1]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < C::NDT; ++dt) o_acc[dt] = O::mfma(vop[u][dt], p_op[u], o_acc[dt]);
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * C::NDT, 0);
#pragma unroll
    for (int i = 0; i < 2 * C::NDT; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i < C::NDT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
    }
  };

  // ring: step j in slot j % 3, two steps in flight; every step copies (past the
  // list through empty ranges), so every wait counts the same operations
  Staged st[C::STAGES];
  const Step first = step_of(0), second = step_of(1);
  st[0] = stage(first, s_0);
  __builtin_amdgcn_sched_barrier(0);
  st[1] = stage(second, s_1);
  __builtin_amdgcn_sched_barrier(0);
  Step next = step_of(2);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * C::OPS));  // Q has landed
  auto iteration = [&](auto slot_c, int j) __attribute__((always_inline)) {
    constexpr int J = decltype(slot_c)::value;
    constexpr int F = (J + C::STAGES - 1) % C::STAGES;
    char* const tile = J == 0 ? s_0 : J == 1 ? s_1 : s_2;
    char* const fill = F == 0 ? s_0 : F == 1 ? s_1 : s_2;
    wait_vm_barrier<C::OPS>();
    st[F] = stage(next, fill);
    __builtin_amdgcn_sched_barrier(0);
    const Staged s = st[J];
    const bool seen = s.key >= 0 && s.key < w_last.hi &&
                      (s.key + kTileKeys > w_first.lo || s.key < a.sinks);
    auto prefetch = [&]() __attribute__((always_inline)) { next = step_of(j + C::STAGES); };
    if (seen) compute(tile, s, prefetch);
    else prefetch();
  };
  const int rounds = (steps + C::STAGES - 1) / C::STAGES;
  for (int rd = 0; rd < rounds; ++rd) {
    const int j = rd * C::STAGES;
    iteration(std::integral_constant<int, 0>{}, j);
    iteration(std::integral_constant<int, 1>{}, j + 1);
    iteration(std::integral_constant<int, 2>{}, j + 2);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // trailing copies land before the slots are freed

  const float l = pair_sum(l_run), m = m_run;
  const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // (a NaN sum stays one)
  bool bad = false;  // a product that is no number in a row whose sum is one
#pragma unroll
  for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      o_acc[dt][r] *= inv;
      bad = bad || !(fabsf(o_acc[dt][r]) < INFINITY);
    }
  const Row my = my_row();
  const int64_t wrow = ws_row + my.row - row0;
  T* const op = static_cast<T*>(a.out) + b * a.so[0] + static_cast<int64_t>(my.qi) * a.so[1] +
                my.head * a.so[2];
  if (my.live) {
#pragma unroll
    for (int dt = 0; dt < C::NDT; ++dt)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int d0 = 32 * dt + 8 * g + 4 * hf;
        if (ns > 1) {
          *reinterpret_cast<v4f*>(a.ws_o + wrow * D + d0) =
              v4f{o_acc[dt][4 * g], o_acc[dt][4 * g + 1], o_acc[dt][4 * g + 2],
                  o_acc[dt][4 * g + 3]};
        } else {
          typename O::op4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(o_acc[dt][4 * g + e]);
          *reinterpret_cast<typename O::op4*>(op + d0) = w;
        }
      }
    if (hf == 0) {
      if (ns > 1)
        a.ws_ml[wrow] = make_float2(l > 0.0f ? m : (l == 0.0f ? -INFINITY : l), l);
      else if (a.lse)
        a.lse[(static_cast<int64_t>(b) * a.Hq + my.head) * a.Lq + my.qi] =
            l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
    }
  }
  // A row whose products met a value that it does not see (0 * inf or 0 * NaN of a
  // masked key): its sum is taken again over its own keys, one row at a time.
  uint64_t again = __ballot(bad && my.live && l > 0.0f && l < INFINITY);
  again |= again >> 32;
  if (static_cast<uint32_t>(again) == 0) return;
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // (the stores above come first)
  for (uint32_t rows = static_cast<uint32_t>(again); rows != 0; rows &= rows - 1) {
    constexpr int N = D / 64;
    const int i = __builtin_ctz(rows);
    const int r = row0 + wave * 32 + i;
    const int ri = r / a.G, rh = hk * a.G + r - ri * a.G;
    const KeyRange rk = key_range(a, ri + shift, k_len);
    const int rsink = a.sinks < rk.hi ? a.sinks : rk.hi;
    const T* const rq = static_cast<const T*>(a.q) + b * a.sq[0] +
                        static_cast<int64_t>(ri) * a.sq[1] + rh * a.sq[2];
    const float rm = __shfl(m, i, kWave), rinv = __shfl(inv, i, kWave);
    float acc[N], qv[N];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      acc[c] = 0.0f;
      qv[c] = static_cast<float>(rq[lane + 64 * c]);
    }
    for (int s = 0; s < steps; ++s)
      for (int j = key_of(s), end = j + kTileKeys; j < end; ++j) {
        if (!(j < rk.hi && (j >= rk.lo || j < rsink))) continue;
        int64_t ko = j * a.sk[1], vo = j * a.sv[1];
        if constexpr (PAGED) {
          const int pg = table[j / a.page];
          if (!page_ok(pg)) continue;
          const int64_t slot = j % a.page;
          ko = pg * a.sk[0] + slot * a.sk[1];
          vo = pg * a.sv[0] + slot * a.sv[1];
        }
        const T* const kp = reinterpret_cast<const T*>(kbase) + ko;
        const T* const vp = reinterpret_cast<const T*>(vbase) + vo;
        float x = 0.0f;
#pragma unroll
        for (int c = 0; c < N; ++c) x = fmaf(qv[c], static_cast<float>(kp[lane + 64 * c]), x);
        const float p = __builtin_amdgcn_exp2f(fmaf(wave_sum(x), a.scale_log2, -rm));
#pragma unroll
        for (int c = 0; c < N; ++c)
          acc[c] = fmaf(p, static_cast<float>(vp[lane + 64 * c]), acc[c]);
      }
    const int64_t wr = ws_row + r - row0;
    T* const dst = static_cast<T*>(a.out) + b * a.so[0] + static_cast<int64_t>(ri) * a.so[1] +
                   rh * a.so[2];
#pragma unroll
    for (int c = 0; c < N; ++c) {
      if (ns > 1) a.ws_o[wr * D + lane + 64 * c] = acc[c] * rinv;
      else dst[lane + 64 * c] = static_cast<T>(acc[c] * rinv);
    }
  }
}

// The shares of the split row blocks joined: w_s = l_s 2^(m_s - M),
// out = sum w_s O_s / sum w_s.  One thread per row and 8 channels; the shares are added in
// their order.
template <typename T, int D>
__global__ void __launch_bounds__(256) window_merge_kernel(WindowArgs a) {
  constexpr int CPR = D / 8, BM = 128;
  const int64_t v = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  const int per = a.xcd_items - a.xcd_whole;
  const int64_t all_rows = static_cast<int64_t>(per) * kNumXcd * BM;
  const int64_t wrow = v / CPR;
  if (wrow >= all_rows) return;
  const int c = static_cast<int>(v % CPR);
  const int t = static_cast<int>(wrow / BM);
  const int xcd = t / per, in_xcd = a.xcd_whole + t % per;
  const int64_t item = a.descending ? static_cast<int64_t>(in_xcd) * kNumXcd + xcd
                                    : static_cast<int64_t>(xcd) * a.xcd_items + in_xcd;
  if (item >= a.n_items) return;
  const uint32_t it = static_cast<uint32_t>(item), nrb = static_cast<uint32_t>(a.n_rblocks);
  const uint32_t heads = static_cast<uint32_t>(a.B * a.Hk);
  const int bh = static_cast<int>(a.descending ? it % heads : it / nrb);
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const int q_len = request_of(a, b).q_len;
  const int row = static_cast<int>(a.descending ? nrb - 1 - it / heads : it % nrb) * BM +
                  static_cast<int>(wrow % BM);
  if (row >= q_len * a.G) return;
  const int qi = row / a.G, head = hk * a.G + row - qi * a.G;
  float mx = -INFINITY;
  for (int s = 0; s < a.n_split; ++s) mx = fmaxf(mx, a.ws_ml[s * all_rows + wrow].x);
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float sum = 0.0f;
  for (int s = 0; s < a.n_split; ++s) {
    const float2 ml = a.ws_ml[s * all_rows + wrow];
    if (ml.x == -INFINITY) continue;
    const float w = ml.y * __builtin_amdgcn_exp2f(ml.x - mx);
    sum += w;
    float o[8];
    Vec8<float>::load(a.ws_o + (s * all_rows + wrow) * D + c * 8, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, o[j], acc[j]);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  typename Half<T>::op8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = static_cast<T>(acc[j] * inv);
  T* const op = static_cast<T*>(a.out) + b * a.so[0] + qi * a.so[1] + head * a.so[2] + c * 8;
  *reinterpret_cast<typename Half<T>::op8*>(op) = r;
  if (a.lse && c == 0)
    a.lse[(static_cast<int64_t>(b) * a.Hq + head) * a.Lq + qi] =
        sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

// The same for units of few rows: a workgroup takes one row, its threads (share,
// 8 channels); the shares are added in a fixed order.
template <typename T, int D>
__global__ void __launch_bounds__(256) window_unit_merge_kernel(WindowArgs a) {
  constexpr int CPR = D / 8, GROUPS = 256 / CPR;
  __shared__ float s_acc[GROUPS][D], s_sum[GROUPS], s_max[4];
  const int tid = threadIdx.x, lane = tid & 63;
  const int R = a.Lq * a.G;
  const int row = static_cast<int>(blockIdx.x) % R;
  const int bh = static_cast<int>(blockIdx.x) / R;
  const int b = bh / a.Hk, hk = bh - b * a.Hk;
  const Unit u = find_unit<true>(a, b, lane);
  if (row >= u.r.q_len * a.G) return;
  const int shares = u.shares;
  if (shares <= 1) return;  // written by its only unit
  const int64_t first = static_cast<int64_t>(u.before) * a.Hk + hk;
  auto at = [&](int s) __attribute__((always_inline)) -> int64_t {
    return (first + static_cast<int64_t>(s) * a.Hk) * R + row;
  };
  float mx = -INFINITY;
  for (int s = tid; s < shares; s += 256) mx = fmaxf(mx, a.ws_ml[at(s)].x);
  mx = wave_max(mx);
  if (lane == 0) s_max[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(s_max[0], s_max[1]), fmaxf(s_max[2], s_max[3]));
  const int c = tid % CPR, g = tid / CPR;
  float acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  float sum = 0.0f;
  for (int s = g; s < shares; s += GROUPS) {
    const float2 ml = a.ws_ml[at(s)];
    if (ml.x == -INFINITY) continue;
    const float w = ml.y * __builtin_amdgcn_exp2f(ml.x - mx);
    sum += w;
    float o[8];
    Vec8<float>::load(a.ws_o + at(s) * D + c * 8, o);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(w, o[j], acc[j]);
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
  const int qi = row / a.G, head = hk * a.G + row - qi * a.G;
  static_cast<T*>(a.out)[b * a.so[0] + qi * a.so[1] + head * a.so[2] + tid] =
      static_cast<T>(total == 0.0f ? 0.0f : o / total);
  if (a.lse && tid == 0)
    a.lse[(static_cast<int64_t>(b) * a.Hq + head) * a.Lq + qi] =
        total == 0.0f ? -INFINITY : (mx + __log2f(total)) * 0.69314718055994531f;
}

template <typename T, int D>
static int launch_window(WindowArgs& a, hipStream_t s) {
  if (a.n_split == 0) {
    const int64_t n = 4ll * a.units + static_cast<int64_t>(a.B) * a.Hk;
    const int64_t rows = static_cast<int64_t>(a.B) * a.Hk * a.Lq * a.G;
    if (n >= (1ll << 31) || rows >= (1ll << 31)) return RCSA_ERR_SHAPE;
    const dim3 grid(static_cast<unsigned>(n));
    if (a.table) window_kernel<T, D, true, 1><<<grid, dim3(64), 0, s>>>(a);
    else window_kernel<T, D, false, 1><<<grid, dim3(64), 0, s>>>(a);
    if (a.units)
      window_unit_merge_kernel<T, D><<<dim3(static_cast<unsigned>(rows)), dim3(256), 0, s>>>(a);
    return launch_status();
  }
  const int64_t tail = a.xcd_items - a.xcd_whole;
  const int64_t wgs = (a.xcd_whole + tail * a.n_split) * kNumXcd;
  if (wgs >= (1ll << 31)) return RCSA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(wgs));
  if (a.table) window_kernel<T, D, true, 4><<<grid, dim3(256), 0, s>>>(a);
  else window_kernel<T, D, false, 4><<<grid, dim3(256), 0, s>>>(a);
  if (a.n_split > 1 && tail > 0) {
    const int64_t n = (tail * kNumXcd * 128 * (D / 8) + 255) / 256;
    window_merge_kernel<T, D><<<dim3(static_cast<unsigned>(n)), dim3(256), 0, s>>>(a);
  }
  return launch_status();
}

// Blocks of rows of a key head.
static int64_t row_blocks(int64_t Lq, int64_t G) { return (Lq * G + 127) / 128; }

static bool few_rows(const int64_t* d) { return d[1] * (d[3] / d[4]) <= kFewRows; }
// Wavefronts of few rows that fit at once: their rings fill a compute unit's 160 KB of LDS
// three (D 64: six) times.  Every one reads all lengths to find its unit, so past kMaxPlanned
// requests each key head is one unit.
static int64_t units_of_round(const int64_t* d) {
  return d[0] > kMaxPlanned ? 0 : (d[5] == 128 ? 3 : 6) * 256;
}
static bool window_dims(const int64_t* d) {
  for (int i = 0; i < 6; ++i)
    if (d[i] <= 0 && !(i == 2 && d[i] == 0)) return false;
  return d[4] <= d[3] && d[3] % d[4] == 0 && d[0] < (1 << 20) && d[1] < (1 << 24) &&
         d[3] < (1 << 16) && d[1] * (d[3] / d[4]) < (1 << 30) && (d[5] == 64 || d[5] == 128) &&
         d[0] * d[4] * row_blocks(d[1], d[3] / d[4]) < (1ll << 26);
}

// Row blocks of an XCD, and of these the ones in whole rounds of its compute units.
static int64_t xcd_items_of(const int64_t* d) {
  return (d[0] * d[4] * row_blocks(d[1], d[3] / d[4]) + kNumXcd - 1) / kNumXcd;
}
static int64_t xcd_cus() {
  const int64_t n = cus_per_xcd();
  return n > 0 ? n : 32;
}
static int64_t xcd_whole_of(int64_t items, int64_t n_split) {
  return n_split == 1 ? items : whole_items(items, xcd_cus());
}

}  // namespace rcsa

using namespace rcsa;

// Few rows of a key head go to units of one wavefront (n_split 0), more to blocks of 128
// rows.  Of these the ones past an XCD's whole rounds (one block to a compute unit; three
// share it in time) leave compute units idle: their keys go to n_split workgroups, which
// makes that round ceil(tail n / U) (keys / n + kFixed) tiles long.
extern "C" int rcsa_window_attn_plan(const int64_t* dims, int64_t max_keys, int64_t* n_split) {
  if (!dims || !n_split) return RCSA_ERR_NULL;
  if (!window_dims(dims) || max_keys < 0) return RCSA_ERR_SHAPE;
  *n_split = 0;
  if (few_rows(dims)) return RCSA_OK;
  *n_split = 1;
  const int64_t cux = xcd_cus(), items = xcd_items_of(dims);
  const int64_t tail = items % cux;
  if (tail == 0) return RCSA_OK;
  constexpr int64_t kFixed = 16;
  const int64_t tiles = (max_keys + kTileKeys - 1) / kTileKeys;
  int64_t best = tiles + kFixed;
  for (int64_t n = 2; n <= 16 && n * 4 <= tiles; ++n) {
    const int64_t cost = (tail * n + cux - 1) / cux * ((tiles + n - 1) / n + kFixed) +
                         kFixed;  // (the join)
    if (cost < best - best / 16) {
      best = cost;
      *n_split = n;
    }
  }
  return RCSA_OK;
}

extern "C" int64_t rcsa_window_attn_workspace_bytes(const int64_t* dims, int64_t n_split) {
  if (!dims || !window_dims(dims) || n_split < 0 || n_split > 64) return -1;
  const int64_t G = dims[3] / dims[4], row = dims[5] * 4 + 8;
  if (n_split == 0) {
    if (!few_rows(dims)) return -1;
    const int64_t units = units_of_round(dims);
    return units == 0 ? 0 : (4 * units + dims[0] * dims[4]) * dims[1] * G * row;
  }
  const int64_t items = xcd_items_of(dims);
  return n_split == 1 ? 0 : n_split * (items - xcd_whole_of(items, n_split)) * kNumXcd * 128 * row;
}

extern "C" int rcsa_window_attn(const void* q, const void* k, const void* v, void* out, float* lse,
                                int dtype, const int64_t* dims, const int64_t* strides,
                                const int32_t* q_lengths, const int32_t* k_lengths,
                                const int32_t* block_table, int64_t table_stride,
                                int64_t max_pages, int64_t n_pages, int64_t page_size,
                                int64_t window, int64_t sinks, int64_t block, float sm_scale,
                                int64_t n_split, void* workspace, int64_t workspace_bytes,
                                hipStream_t stream) {
  if (!q || !k || !v || !out || !dims || !strides) return RCSA_ERR_NULL;
  if (dtype != RCSA_BF16 && dtype != RCSA_F16) return RCSA_ERR_DTYPE;
  if (!window_dims(dims)) return RCSA_ERR_SHAPE;
  const int64_t most = 1ll << 30;  // positions, windows and blocks stay far from 2^31
  if (dims[2] >= most || window < 0 || sinks < 0 || block < 0) return RCSA_ERR_SHAPE;
  if (block == 0 && (window != 0 || sinks != 0)) return RCSA_ERR_SHAPE;
  if (block_table && (max_pages <= 0 || n_pages <= 0 || page_size <= 0 || page_size % 16 ||
                      n_pages >= most || page_size >= most || max_pages >= most / page_size))
    return RCSA_ERR_SHAPE;
  if (n_split < 0 || n_split > 64 || (n_split == 0 && !few_rows(dims))) return RCSA_ERR_SHAPE;
  for (int i = 0; i < 12; ++i)
    if (strides[i] < 0 || strides[i] % (i < 9 ? 8 : 4)) return RCSA_ERR_STRIDE;
  if (block_table && (strides[3] >= (1ll << 31) || strides[6] >= (1ll << 31)))
    return RCSA_ERR_STRIDE;
  // (rows of keys do not overlap; the stride of a single one says nothing)
  const bool one = !block_table && dims[2] <= 1;
  for (int i = 4; i < 8; i += 3)
    if (strides[i] >= (1 << 25) || (!one && strides[i] < dims[5])) return RCSA_ERR_STRIDE;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(out) & 7u))
    return RCSA_ERR_ALIGN;
  const int64_t need = rcsa_window_attn_workspace_bytes(dims, n_split);
  if (need > 0 && (!workspace || workspace_bytes < need)) return RCSA_ERR_SHAPE;
  WindowArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.lse = lse;
  for (int i = 0; i < 3; ++i) {
    a.sq[i] = strides[i];
    a.sk[i] = strides[3 + i];
    a.sv[i] = strides[6 + i];
    a.so[i] = strides[9 + i];
  }
  if (one) a.sk[1] = a.sv[1] = dims[5];
  a.B = static_cast<int>(dims[0]);
  a.Lq = static_cast<int>(dims[1]);
  a.Lk = static_cast<int>(dims[2]);
  a.Hq = static_cast<int>(dims[3]);
  a.Hk = static_cast<int>(dims[4]);
  a.G = a.Hq / a.Hk;
  a.q_len = q_lengths;
  a.k_len = k_lengths;
  a.table = block_table;
  a.table_stride = table_stride;
  a.max_pages = static_cast<int>(max_pages);
  a.n_pages = static_cast<int>(n_pages);
  a.page = static_cast<int>(page_size);
  if (block_table) {
    const uint64_t d = static_cast<uint64_t>(page_size) / 16;
    int l = 0;
    while ((1ull << l) < d) ++l;
    a.page_mul = static_cast<uint32_t>((1ull << 32) * ((1ull << l) - d) / d + 1);
    a.page_sh1 = l < 1 ? l : 1;
    a.page_sh2 = l < 1 ? 0 : l - 1;
  }
  a.window = static_cast<int>(window < most ? window : 0);
  a.sinks = static_cast<int>(sinks < most ? sinks : most);
  a.block = static_cast<int>(block < most ? block : most);
  a.scale_log2 = sm_scale * 1.4426950408889634f;
  a.n_rblocks = static_cast<int>(row_blocks(a.Lq, a.G));
  a.n_items = static_cast<int64_t>(a.B) * a.Hk * a.n_rblocks;
  a.n_split = static_cast<int>(n_split);
  a.units = n_split == 0 ? static_cast<int>(units_of_round(dims)) : 0;
  const int64_t xcd_items = xcd_items_of(dims);
  if (xcd_items >= (1ll << 30)) return RCSA_ERR_SHAPE;
  a.xcd_items = static_cast<int>(xcd_items);
  a.xcd_whole = static_cast<int>(xcd_whole_of(xcd_items, n_split));
  // rows without a window see more keys the later they stand
  a.descending = a.window == 0 && a.block != 0;
  const int64_t ws_rows = need / (dims[5] * 4 + 8);
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = need ? reinterpret_cast<float2*>(a.ws_o + ws_rows * dims[5]) : nullptr;
  if (dtype == RCSA_BF16)
    return dims[5] == 128 ? launch_window<__bf16, 128>(a, stream)
                          : launch_window<__bf16, 64>(a, stream);
  return dims[5] == 128 ? launch_window<_Float16, 128>(a, stream)
                        : launch_window<_Float16, 64>(a, stream);
}
