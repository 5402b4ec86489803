// Windowed attention, blocks of 128 rows: one pass over the visible keys with the
// running maximum and sum of the softmax.
//
// Work: a workgroup takes 128 rows of one key head (32 a wavefront, 4
// wavefronts) and streams the 32-key tiles that any of them sees: the tiles of
// the first keys, then those of the window.  Three workgroups share a compute
// unit, so that one's exponentials run beside another's matrix products.
// A tile's K and V go global -> LDS without registers into a ring of three
// slots; rows past the keys, and pages that are not there, land as zeros.
// Bound by the matrix products at the card's power limit: 44 frames of 880 tokens, a window of
// 12 and an anchor, 24 heads 3.9-4.2 ms by card, 1110-1200 TFLOP/s (a 16384^3 product 1362), the
// matrix pipe 75% busy at 1.45-1.6 GHz; window 4096 over 32773 tokens, 32 heads on 8 1.8-1.9 ms,
// 1090-1160 TFLOP/s, 72%.  Four frames on 44 in pages, 992 workgroups on 768 places, 755-795 us,
// 1010-1060 TFLOP/s, 61%.  D 64 has half the products a key beside the same exponentials: 16384
// tokens x 16 heads, window 4096, 288 us, 835 TFLOP/s, 51%.
// Only the tiles at the window's edges are masked.  A wavefront also works on the few
// tiles that none of its rows sees: with a branch around the work the copies could not
// go out between the matrix products (four frames against 20 of 44 708 us so, 722 with
// it; window 4096 over 32773 x 32 heads 1770 and 1797; window 1024 over 16384 x 8 87 and 86).
#pragma once
#include "window_attn.h"

namespace rcsa {

template <typename T, int D, bool PAGED>
__global__ void __launch_bounds__(256)
__attribute__((amdgpu_waves_per_eu(D == 64 ? 4 : 3, D == 64 ? 4 : 3)))
window_kernel(WindowArgs a) {
  using R = RowTile<T, D>;
  constexpr int BM = 128, STAGES = 3;
  constexpr int RPU = 1024 / R::KROW;         // rows of a 1 KiB copy
  constexpr int UPW = R::TILE / 1024 / 4;     // copies of a wavefront, K and V each
  constexpr int OPS = 2 * UPW;
  // (separate arrays and a loop unrolled over them: reads of one slot do not wait for
  // copies in flight into the others)
  __shared__ __attribute__((aligned(1024))) char s_0[2 * R::TILE];
  __shared__ __attribute__((aligned(1024))) char s_1[2 * R::TILE];
  __shared__ __attribute__((aligned(1024))) char s_2[2 * R::TILE];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = uniform_int(tid >> 6);
  const int hf = lane >> 5, lr = lane & 31;

  // XCD x (workgroups go round-robin) runs a contiguous run of items, so that neighbours
  // share most of their window in its L2, or every 8th from the longest on.
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

  // uniform ranges: of the item, and of this wavefront's first and last rows
  const KeyRange w_first = row_range(a, p, p.row0), w_last = row_range(a, p, p.row0 + 31);
  p.tiles = tiles_of(a, row_range(a, p, item_row0), row_range(a, p, item_row0 + BM - 1));
  share_of(p, share);

  R t;
  t.init(lane);
  {
    const Row r = row_of(a, p, p.row0 + lr);
    t.load_q(static_cast<const T*>(a.q) + p.b * a.sq[0] + static_cast<int64_t>(r.qi) * a.sq[1] +
                 r.head * a.sq[2], hf);
  }

  const char* const kbase = static_cast<const char*>(a.k) +
                            ((PAGED ? 0 : p.b * a.sk[0]) + p.hk * a.sk[2]) * 2;
  const char* const vbase = static_cast<const char*>(a.v) +
                            ((PAGED ? 0 : p.b * a.sv[0]) + p.hk * a.sv[2]) * 2;
  const uint32_t krb = static_cast<uint32_t>(a.sk[1] * 2), vrb = static_cast<uint32_t>(a.sv[1] * 2);
  const int32_t* const table = PAGED ? a.table + p.b * a.table_stride : nullptr;

  // Copies: wavefront w moves rows 8w .. 8w + 7 of the tile, which lie in its half w / 2,
  // RPU rows a copy, chunks swizzled by row.
  uint32_t k_lo[UPW], v_lo[UPW];
#pragma unroll
  for (int i = 0; i < UPW; ++i) {
    const int r = (wave * UPW + i) * RPU + lane / R::CPR;  // row of the tile
    const uint32_t in_half = static_cast<uint32_t>(r & 15);
    k_lo[i] = in_half * krb + (((lane % R::CPR) ^ (swz_k<R::KROW>(r) & (R::CPR - 1))) * 16);
    v_lo[i] = in_half * vrb + (((lane % R::CPR) ^ (swz_v(r) & (R::CPR - 1))) * 16);
  }
  struct Staged {
    int key, there;
  };
  auto stage = [&](const Step& s, char* dst) __attribute__((always_inline)) {
    const HalfRows h = half_rows<PAGED>(a, s, wave >> 1, p.k_len, krb, vrb);
    char* const ks = const_cast<char*>(kbase) + h.k;
    char* const vs = const_cast<char*>(vbase) + h.v;
    // (row strides are at least a row: a lane of row r < rows stays below)
    const int kn = h.rows * static_cast<int>(krb), vn = h.rows * static_cast<int>(vrb);
#pragma unroll
    for (int i = 0; i < UPW; ++i) {
      buffer_copy16(ks, kn, k_lo[i], dst + (wave * UPW + i) * 1024);
      buffer_copy16(vs, vn, v_lo[i], dst + R::TILE + (wave * UPW + i) * 1024);
    }
  };

  // ring: step j in slot j % 3, two steps in flight; every step copies (past the
  // list through empty ranges), so every wait counts the same operations; whole rounds,
  // so that the compiler keeps track of which slot a copy in flight writes
  Staged st[STAGES];
  const Step first = step_of<PAGED>(a, p, table, 0), second = step_of<PAGED>(a, p, table, 1);
  st[0] = {first.key, halves_there<PAGED>(a, first)};
  st[1] = {second.key, halves_there<PAGED>(a, second)};
  stage(first, s_0);
  __builtin_amdgcn_sched_barrier(0);
  stage(second, s_1);
  __builtin_amdgcn_sched_barrier(0);
  Step next = step_of<PAGED>(a, p, table, 2);
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(2 * OPS));  // Q has landed
  auto iteration = [&](auto slot_c, int j) __attribute__((always_inline)) {
    constexpr int J = decltype(slot_c)::value;
    constexpr int F = (J + STAGES - 1) % STAGES;
    char* const tile = J == 0 ? s_0 : J == 1 ? s_1 : s_2;
    char* const fill = F == 0 ? s_0 : F == 1 ? s_1 : s_2;
    wait_vm_barrier<OPS>();
    const Staged s = st[J];
    const Step cur = next;
    st[F] = {cur.key, halves_there<PAGED>(a, cur)};
    auto prefetch = [&]() __attribute__((always_inline)) {
      next = step_of<PAGED>(a, p, table, j + STAGES);
    };
    // every row of the wavefront sees the whole tile
    const bool inside = s.key >= 0 && (!PAGED || s.there == 3) &&
                        s.key + kTileKeys <= w_first.hi &&
                        (s.key >= w_last.lo || s.key + kTileKeys <= a.sinks);
    t.template step<OPS>(
        tile, a.scale_log2, inside,
        [&]() __attribute__((always_inline)) {
          return s.key < 0 ? 0u : seen_bits(a, p, p.row0 + lr, hf, s.key, s.there);
        },
        prefetch, [&]() __attribute__((always_inline)) { stage(cur, fill); });
  };
  const int rounds = (p.steps + STAGES - 1) / STAGES;
  for (int rd = 0; rd < rounds; ++rd) {
    const int j = rd * STAGES;
    iteration(std::integral_constant<int, 0>{}, j);
    iteration(std::integral_constant<int, 1>{}, j + 1);
    iteration(std::integral_constant<int, 2>{}, j + 2);
  }
  __builtin_amdgcn_s_waitcnt(vmcnt_imm(0));  // trailing copies land before the slots are freed
  __builtin_amdgcn_s_barrier();  // (the ring is read: a wavefront may need a part of it)
  finish_rows<T, D, PAGED>(p, t, a.ws_o + ws_row * D, a.ws_ml + ws_row,
                           (wave < 2 ? s_0 : s_1) + (wave & 1) * R::TILE);
}

}  // namespace rcsa
