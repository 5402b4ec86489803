// Windowed attention over dense or paged keys: what the kernels of 128-row blocks
// (window_attn.hip) and of units of few rows (window_units.hip) share.
//
// Query i of a request with q_len queries and k_len keys is at position
// p = i + k_len - q_len; e(p) = (floor(p / block) + 1) * block is the end of its
// block of positions.  It sees key j when
//   j < min(e, k_len) and (j >= e - window or j < sinks)
// (window 0: every key below e; block 0: every key), and
//   out = softmax_j(sm_scale q . k_j) v,  lse = log sum_j exp(sm_scale q . k_j).
// The G = Hq / Hk query heads of a key head are rows of one problem: row r is
// query r / G of head hk * G + r % G, so every staged key serves all of them and
// a tile of rows spans few positions.  Packed requests stand behind each other in q and in k
// and v; the batch and key lengths of the dense form are their offsets.
#pragma once
#include "packed.h"
#include "sparse_attn_kernel.h"

namespace rcsa {

typedef _Float16 v8hf __attribute__((ext_vector_type(8)));
typedef _Float16 v4hf __attribute__((ext_vector_type(4)));

constexpr int kTileKeys = 32;
constexpr int kDense = 0, kPaged = 1, kPacked = 2;  // forms of keys and values

struct WindowArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;                       // [B][Hq][Lq], nullable
  int64_t sq[3], sk[3], sv[3], so[3];  // (batch, row, head); paged k, v: (page, slot, head)
  int B, Lq, Lk, Hq, Hk, G;
  Divisor by_G, by_Hk, by_block, by_rblocks, by_heads;  // by_heads: B * Hk
  Divisor by_half_page;             // half tiles of a page
  int whole_tiles;                  // a page holds a multiple of 32 keys
  const int32_t *q_len, *k_len;     // [B], nullable: Lq, Lk
  const int32_t* table;             // [B][max_pages], nullable: dense k, v
  int64_t table_stride;
  int max_pages, n_pages, page;     // page: keys of a page, a multiple of 16
  int window, sinks, block;         // block 0: no order among positions
  float scale_log2;                 // sm_scale * log2(e)
  int n_rblocks;                    // blocks of rows of a key head
  int64_t n_items;                  // B * Hk * n_rblocks
  int n_split;
  float* ws_o;                      // [share][row][D] normalised partial outputs
  float2* ws_ml;                    // [share][row] their (max, sum)
  // Row blocks in XCD runs of xcd_items, of which the first xcd_whole run whole and the
  // others in n_split shares; descending: the longest (last) row blocks first, dealt
  // round-robin.
  int xcd_items, xcd_whole;
  int descending;
  // pages of 8-bit codes: their scales [page][block][head], 16 keys of a block
  const float *ks, *vs;
  int sks[3], svs[3];  // (their last one is below 2^29)
  Divisor by_half_mark;
  int mark;
  int e4m3;        // the codes' type; -1: 16-bit keys and values
  // packed: rows of the requests in q and in k, v ([B + 1] each), a request's row blocks
  // numbered through n_ranks
  const int32_t *q_off, *k_off;
  int n_ranks;
  int units;       // few rows in units: wavefronts of one round
  float per_unit;  // 1 / units
  int unit_tiles;  // kUnitTiles, of codes kCodeUnitTiles
};

constexpr int kFewRows = 32;        // rows of a key head that one wavefront takes
constexpr int kMaxPlanned = 512;    // requests whose lengths every wavefront reads
constexpr int kGroupWaves = 8;      // wavefronts of a workgroup that takes a key head
constexpr int64_t kMaxThreads = 1ll << 32;  // a grid's dimension holds fewer

// The keys of a position: [0, sink) and [lo, hi).
struct KeyRange {
  int lo, hi;
};
template <typename A>
__device__ __forceinline__ KeyRange key_range(A& a, int p, int k_len) {
  if (a.block == 0) return {0, k_len};
  if (p < 0) return {0, 0};
  const int e = a.block == 1 ? p + 1 : divide(p, a.by_block) * a.block + a.block;
  const int hi = e < k_len ? e : k_len;
  const int lo = a.window == 0 || e <= a.window ? 0 : e - a.window;
  return {lo < hi ? lo : hi, hi};
}

// A request's lengths, clamped to the storage; UNIFORM: of one request for the wavefront, by
// scalar loads.
struct Request {
  int k_len, q_len;
};
template <bool UNIFORM = false>
__device__ __forceinline__ Request request_of(const WindowArgs& a, int b) {
  const int cap = a.table != nullptr ? a.max_pages * a.page : a.Lk;
  auto at = [&](const int32_t* p) __attribute__((always_inline)) -> int {
    return UNIFORM ? ld_const(p + b) : p[b];
  };
  int k = a.k_len == nullptr ? cap : at(a.k_len);
  int q = a.q_len == nullptr ? a.Lq : at(a.q_len);
  k = k < 0 ? 0 : (k > cap ? cap : k);
  q = q < 0 ? 0 : (q > a.Lq ? a.Lq : q);
  return {k, q};
}
// The tiles that rows of key ranges first .. last see: sink_n of the first keys, then win_n
// from tile win_t0 on.
struct Tiles {
  int sink_n, win_t0, win_n;
  __device__ __forceinline__ int all() const { return sink_n + win_n; }
};
__device__ __forceinline__ Tiles tiles_of(const WindowArgs& a, KeyRange first, KeyRange last) {
  const int sinks = a.sinks < last.hi ? a.sinks : last.hi;
  Tiles t;
  t.win_t0 = first.lo / kTileKeys;
  t.win_n = (last.hi + kTileKeys - 1) / kTileKeys - t.win_t0;
  t.win_n = t.win_n < 0 ? 0 : t.win_n;
  t.sink_n = (sinks + kTileKeys - 1) / kTileKeys;
  t.sink_n = t.sink_n < t.win_t0 ? t.sink_n : t.win_t0;
  return t;
}

// Which key head and block of rows is entry in_xcd of XCD xcd's run (bh -1: none): a
// contiguous run of items, or every 8th from the longest (last) row blocks on.
struct ItemAt {
  int bh, rblock;
};
__device__ __forceinline__ ItemAt item_at(const WindowArgs& a, int xcd, int in_xcd) {
  const int64_t item = a.descending ? static_cast<int64_t>(in_xcd) * kNumXcd + xcd
                                    : static_cast<int64_t>(xcd) * a.xcd_items + in_xcd;
  if (in_xcd >= a.xcd_items || item >= a.n_items) return {-1, 0};
  const int i = static_cast<int>(item);
  if (a.descending) {
    const int back = divide(i, a.by_heads);
    return {i - back * static_cast<int>(a.by_heads.d), a.n_rblocks - 1 - back};
  }
  const int bh = divide(i, a.by_rblocks);
  return {bh, i - bh * a.n_rblocks};
}

// Few rows, many keys: the visible tiles of all requests are dealt to units of one wavefront each,
// `chunk` tiles of one key head at most, however uneven the lengths.  A wavefront reads
// the lengths, one lane a request, and finds its unit among them; unit index = (units
// of the requests before) * Hk + share * Hk + hk.
__device__ __forceinline__ int request_tiles(const WindowArgs& a, Request r) {
  if (r.q_len == 0) return -1;
  const int p = r.k_len - r.q_len;
  return tiles_of(a, key_range(a, p, r.k_len), key_range(a, p + r.q_len - 1, r.k_len)).all();
}
__device__ __forceinline__ int units_of(int tiles, int chunk) {
  return tiles < 0 ? 0 : (tiles <= chunk ? 1 : (tiles + chunk - 1) / chunk);
}
// One round of the wavefronts that fit (a.units) where that leaves units of up to
// kUnitTiles tiles; beyond, units of that size, or more of them than four rounds.  A unit
// costs about 5 us before its first tile has landed (a tile streams in 0.4 to 1), and the
// units of a last, short round leave compute units idle.  Tiles of 8-bit codes are half the
// bytes: units of twice as many (48 ragged requests of up to 32768 keys: of 16 tiles 211 us, 32
// 198, 64 257).
// (Sums and products in fp32, at most 14 roundings of 2^-24, that the factor rounds up: a plan,
// the same for every wavefront.  The tiles of all requests pass 32 bits where tables share
// pages; a request has at most 2^25, so that a chunk of kMostTiles leaves it whole.)
constexpr int kLeastTiles = 2, kUnitTiles = 16, kCodeUnitTiles = 32, kMostTiles = 1 << 26;
__device__ __forceinline__ int chunk_of(const WindowArgs& a, float total) {
  const float t = total * static_cast<float>(a.Hk) * 1.000001f;
  auto chunk = [](float x) { return static_cast<int>(fminf(x, kMostTiles)) + 1; };
  const int one = chunk(t * a.per_unit);
  int c = chunk(t * (0.25f * a.per_unit));
  c = c < a.unit_tiles ? a.unit_tiles : c;
  c = c < one ? c : one;
  return c < kLeastTiles ? kLeastTiles : c;
}
struct Unit {
  int b, share, shares;  // b -1: no such unit
  int before;            // units (of one key head) of the requests before b
  Request r;
};
__device__ __forceinline__ float lane_sum(float x) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) x += __shfl_xor(x, o, kWave);
  return x;
}
__device__ __forceinline__ int lane_prefix(int x, int lane) {  // inclusive
#pragma unroll
  for (int o = 1; o < kWave; o <<= 1) {
    const int up = __shfl_up(x, o, kWave);
    x += lane >= o ? up : 0;
  }
  return x;
}
// Unit index `w` of a key head (of_request false), or the units of request w (true).  Every
// lane of the wavefront calls it; the result is uniform.
template <bool OF_REQUEST>
__device__ __forceinline__ Unit find_unit(const WindowArgs& a, int w, int lane) {
  if (a.B <= kWave) {  // one load of the lengths (a single request needs no lanes' sums)
    Request r{0, 0};
    if (a.B == 1) r = request_of<true>(a, 0);
    else if (lane < a.B) r = request_of(a, lane);
    const int tiles = lane < a.B ? request_tiles(a, r) : -1;
    const int mine = tiles > 0 ? tiles : 0;
    const float own = static_cast<float>(a.B == 1 ? uniform_int(mine) : mine);
    const int chunk = uniform_int(chunk_of(a, a.B == 1 ? own : lane_sum(own)));
    const int n = units_of(tiles, chunk);
    const int upto = a.B == 1 ? n : lane_prefix(n, lane);
    int l = w;
    if (!OF_REQUEST) {
      const uint64_t past = __ballot(lane < a.B && upto > w);
      if (past == 0) return {-1, 0, 0, 0, {0, 0}};
      l = __builtin_ctzll(past);
    }
    auto at = [&](int x) __attribute__((always_inline)) { return __builtin_amdgcn_readlane(x, l); };
    const int shares = at(n), before = at(upto) - shares;
    return {l, w - before, shares, before, {at(r.k_len), at(r.q_len)}};
  }
  float total = 0.0f;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int t = b0 + lane < a.B ? request_tiles(a, request_of(a, b0 + lane)) : 0;
    total += lane_sum(static_cast<float>(t > 0 ? t : 0));
  }
  const int chunk = uniform_int(chunk_of(a, total));
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    Request r{0, 0};
    if (b0 + lane < a.B) r = request_of(a, b0 + lane);
    const int n = b0 + lane < a.B ? units_of(request_tiles(a, r), chunk) : 0;
    const int upto = before + lane_prefix(n, lane);
    const uint64_t past =
        OF_REQUEST ? (w - b0 < kWave ? 1ull << (w - b0) : 0) : __ballot(upto > w);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      auto at = [&](int x) __attribute__((always_inline)) {
        return __builtin_amdgcn_readlane(x, l);
      };
      const int shares = at(n), bef = at(upto) - shares;
      return {b0 + l, w - bef, shares, bef, {at(r.k_len), at(r.q_len)}};
    }
    before = __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return {-1, 0, 0, 0, {0, 0}};
}

template <typename T>
struct Half;  // the 16-bit types' matrix products and LDS transpose reads
template <>
struct Half<__bf16> {
  typedef v8bf op8;
  typedef v4bf op4;
  static constexpr int kShift = 0;  // (fp32's range)
  static __device__ __forceinline__ v16f mfma(op8 x, op8 y, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ op4 read_tr(const char* p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4bf16(RCSA_LDS(op4, p));
  }
};
template <>
struct Half<_Float16> {
  typedef v8hf op8;
  typedef v4hf op4;
  static constexpr int kShift = 7;  // (a term: at most 2^(kTau + kShift) = 2^15)
  static __device__ __forceinline__ v16f mfma(op8 x, op8 y, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ op4 read_tr(const char* p) {
    return __builtin_bit_cast(op4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(RCSA_LDS(v4bf, p)));
  }
};

// Where a wavefront's 32 rows stand: rows row0 .. of key head hk of request b, of n_rows;
// position of query 0; the tiles [begin, begin + steps) of the rows' tiles are its
// share's, one of `shares`.
struct Place {
  int b, hk, row0, n_rows, shift, k_len;
  int q0, k0;  // packed: the request's first rows
  int shares, begin, steps;
  Tiles tiles;
};
// Where a request's queries and outputs (s: strides), and the keys or values of its key head,
// begin, in elements.
template <int FORM, typename S>
__device__ __forceinline__ int64_t rows_at(const Place& p, S& s) {
  return FORM == kPacked ? p.q0 * s[1] : p.b * s[0];
}
template <int FORM, typename S>
__device__ __forceinline__ int64_t keys_at(const Place& p, S& s) {
  return (FORM == kPaged ? 0 : FORM == kPacked ? p.k0 * s[1] : p.b * s[0]) + p.hk * s[2];
}
// Its place in lse ([B][Hq][Lq], packed [Hq][Lq]).
template <int FORM, typename A>
__device__ __forceinline__ int64_t lse_at(A& a, const Place& p, int head, int qi) {
  return FORM == kPacked ? static_cast<int64_t>(head) * a.Lq + p.q0 + qi
                         : (static_cast<int64_t>(p.b) * a.Hq + head) * a.Lq + qi;
}
// First key of step s, -1 past the last.
__device__ __forceinline__ int key_of(const Place& p, int s) {
  const int t = p.begin + s;
  return s >= p.steps ? -1
                      : (t < p.tiles.sink_n ? t : p.tiles.win_t0 + t - p.tiles.sink_n) * kTileKeys;
}
template <typename A>
__device__ __forceinline__ KeyRange row_range(A& a, const Place& p, int row) {
  row = row < p.n_rows ? row : p.n_rows - 1;
  return key_range(a, divide(row, a.by_G) + p.shift, p.k_len);
}
// The lane's row; rows past the last stand at the last one's place, unwritten.  (Found again
// where it is needed: registers are short.)
struct Row {
  int row, qi, head;
  bool live;
};
template <typename A>
__device__ __forceinline__ Row row_of(A& a, const Place& p, int row) {
  asm volatile("" : "+v"(row));
  const bool live = row < p.n_rows;
  const int at = live ? row : p.n_rows - 1, qi = divide(at, a.by_G);
  return {row, qi, p.hk * a.G + at - qi * a.G, live};
}

// A step: its first key and, paged, the pages of its two halves of 16 keys (a half lies in
// one page: pages hold whole halves).  Scalar arithmetic and loads throughout.
struct Step {
  int key, page0, page1;
};
template <typename A>
__device__ __forceinline__ bool page_ok(A& a, int p) {
  return static_cast<uint32_t>(p) < static_cast<uint32_t>(a.n_pages);
}
template <bool PAGED, typename A>
__device__ __forceinline__ Step step_of(A& a, const Place& p, const int32_t* table,
                                        int s) {
  Step r{key_of(p, s), 0, 0};
  if constexpr (PAGED) {
    const int half = (r.key < 0 ? 0 : r.key) >> 4;
    const int col0 = divide(half, a.by_half_page);
    r.page0 = ld_const(table + col0);
    if (a.whole_tiles) {  // pages of whole tiles: one entry for both halves
      r.page1 = r.page0;
    } else {
      const int col1 = divide(half + 1, a.by_half_page);
      r.page1 = ld_const(table + (col1 < a.max_pages ? col1 : a.max_pages - 1));
    }
  }
  return r;
}
// This share's part of all tiles (parts differ by at most one tile).
__device__ __forceinline__ void share_of(Place& p, int share) {
  const uint32_t n = static_cast<uint32_t>(p.tiles.all()), k = static_cast<uint32_t>(p.shares);
  const int q = uniform_int(static_cast<int>(k == 1 ? n : n / k));
  const int rem = static_cast<int>(n) - q * p.shares;
  p.begin = share * q + (share < rem ? share : rem);
  p.steps = q + (share < rem ? 1 : 0);
}
// Whether the step's halves are there: bits 0 and 1.
template <bool PAGED, typename A>
__device__ __forceinline__ int halves_there(A& a, const Step& s) {
  return PAGED ? (page_ok(a, s.page0) ? 1 : 0) + (page_ok(a, s.page1) ? 2 : 0) : 3;
}
// The 16 rows of a half of a step: offsets of its first row, rows that are there.  (32 x
// 32-bit products: a page spans less than 4 GiB.)
struct HalfRows {
  uint64_t k, v;
  int rows;
};
template <bool PAGED, typename A>
__device__ __forceinline__ HalfRows half_rows(A& a, const Step& s, int half,
                                              int k_len, uint32_t krb, uint32_t vrb) {
  const int key = (s.key < 0 ? 0 : s.key) + 16 * half;
  HalfRows r;
  bool there = s.key >= 0;
  if constexpr (PAGED) {
    const int pg = half ? s.page1 : s.page0;
    there = there && page_ok(a, pg);
    const uint32_t slot = static_cast<uint32_t>(key - divide(key >> 4, a.by_half_page) * a.page);
    const uint32_t at = there ? static_cast<uint32_t>(pg) : 0u;
    r.k = static_cast<uint64_t>(at) * static_cast<uint32_t>(a.sk[0] * 2) +
          static_cast<uint64_t>(slot) * krb;
    r.v = static_cast<uint64_t>(at) * static_cast<uint32_t>(a.sv[0] * 2) +
          static_cast<uint64_t>(slot) * vrb;
  } else {
    r.k = static_cast<uint64_t>(static_cast<uint32_t>(key)) * krb;
    r.v = static_cast<uint64_t>(static_cast<uint32_t>(key)) * vrb;
  }
  const int left = k_len - key;
  r.rows = uniform_int(!there || left <= 0 ? 0 : (left < 16 ? left : 16));
  return r;
}

// 32 rows against staged tiles of 32 keys: S^T = K Q^T puts a query row in a lane (its
// 16 + 16 keys in the two lane halves), so a row's maximum and sum need one lane swap,
// and P^T is the second operand of O^T = V^T P^T as it stands.  The running maximum moves
// only when a term passes 2^kTau.  P is rounded to the type for its product (half a step of
// a weight; fp32 products have a sixteenth of the rate), the sums keep fp32.
// m_run stands kShift below the running maximum, so that terms, sums and products carry a
// factor 2^kShift: fp16 keeps all bits of weights down to 2^-21 of the largest and some down
// to 2^-32 (without it 2^-14 and 2^-25: 2^18 keys at 2^-25.2 lost all of their 0.7%).
template <typename T, int D>
struct RowTile {
  using O = Half<T>;
  typedef typename O::op8 op8;
  static constexpr int KROW = D * 2, CPR = KROW / 16;  // bytes and 16-byte chunks of a row
  static constexpr int QSTEPS = D / 16, NDT = D / 32;
  static constexpr int TILE = kTileKeys * KROW;        // bytes of a K (or V) tile
  op8 q_op[QSTEPS];
  v16f o_acc[NDT];
  float m_run, l_run;
  int k_off[QSTEPS], v_off[NDT];  // LDS read offsets (V behind K)

  __device__ __forceinline__ void init(int lane) {
    const int hf = lane >> 5, lr = lane & 31;
    const int kr = key_perm(lr), ks = swz_k<KROW>(kr) & (CPR - 1);
#pragma unroll
    for (int st = 0; st < QSTEPS; ++st)
      k_off[st] = kr * KROW + (((hf * QSTEPS + st) ^ ks) * 16);
    const int grp = lane >> 4, gi = lane & 15;
    const int vr = 16 * (grp >> 1) + (gi >> 2), vs = swz_v(vr) & (CPR - 1);
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt) {
      const int d = 32 * dt + 16 * (grp & 1) + 4 * (gi & 3);
      v_off[dt] = TILE + vr * KROW + (((d >> 3) ^ vs) * 16) + (d & 7) * 2;
    }
#pragma unroll
    for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) o_acc[dt][r] = 0.0f;
    m_run = -INFINITY;
    l_run = 0.0f;
  }
  __device__ __forceinline__ void load_q(const T* row, int hf) {
#pragma unroll
    for (int st = 0; st < QSTEPS; ++st)
      q_op[st] = *reinterpret_cast<const op8*>(row + (hf * QSTEPS + st) * 8);
  }

  // One tile: `inside` when every row sees all of it, else bits() gives the lane's 16 keys.
  // prefetch() issues scalar loads for later steps: behind the first products (they return
  // out of order, so a wait for LDS behind them would wait for them too).  copies() issues
  // a later step's OPS copies, which go out between the second products.
  template <int OPS, typename Bits, typename Pre, typename Cp>
  __device__ __forceinline__ void step(const char* tile, float c, bool inside, Bits&& bits,
                                       Pre&& prefetch, Cp&& copies) {
    v4i kraw[QSTEPS];
#pragma unroll
    for (int st = 0; st < QSTEPS; ++st)
      kraw[st] = *reinterpret_cast<const v4i*>(tile + k_off[st]);
    v16f s_acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) s_acc[r] = 0.0f;
#pragma unroll
    for (int st = 0; st < QSTEPS; ++st)
      s_acc = O::mfma(__builtin_bit_cast(op8, kraw[st]), q_op[st], s_acc);
    __builtin_amdgcn_sched_group_barrier(0x100, QSTEPS, 0);
    __builtin_amdgcn_sched_group_barrier(0x008, QSTEPS, 0);
    __builtin_amdgcn_sched_barrier(0);
    prefetch();
    float rv[16];
#pragma unroll
    for (int r = 0; r < 16; ++r) rv[r] = s_acc[r];
    if (!inside) {
      const uint32_t seen = bits();
#pragma unroll
      for (int r = 0; r < 16; ++r) rv[r] = ((seen >> r) & 1u) ? rv[r] : -INFINITY;
    }
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
    // (a lane's partial sum bounds its terms)
    float part = exps();
    if (__ballot(m_run == -INFINITY || !(part <= kTauPow * (1 << O::kShift))) != 0) {
      float rmax = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) rmax = fmaxf(rmax, rv[r]);
      rmax = pair_max(rmax);
      const float m_blk = rmax == -INFINITY ? -INFINITY : rmax * c - O::kShift;
      if (__ballot(m_blk > m_run + kTau) != 0) {
        const float m_new = fmaxf(m_run, m_blk);
        const float alpha = m_new == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m_run - m_new);
        l_run *= alpha;
#pragma unroll
        for (int dt = 0; dt < NDT; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) o_acc[dt][r] *= alpha;
        m_run = m_new;
        part = exps();
      }
    }
    l_run += part;
    copies();
    // (the reads of the second half of the keys are in flight beside the first half's
    // products)
    auto v_group = [&](int u, op8 (&op)[NDT]) __attribute__((always_inline)) {
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) {
        const char* const p0 = tile + v_off[dt] + 8 * u * KROW;
        const auto lo = O::read_tr(p0);
        const auto hi = O::read_tr(p0 + 4 * KROW);
        op[dt] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
    };
    op8 vop[2][NDT];
    v_group(0, vop[0]);
    v_group(1, vop[1]);
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < NDT; ++dt) o_acc[dt] = O::mfma(vop[u][dt], p_op[u], o_acc[dt]);
    __builtin_amdgcn_sched_group_barrier(0x100, 2 * NDT, 0);
#pragma unroll
    for (int i = 0; i < 2 * NDT; ++i) {
      __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
      if (i < NDT) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
      if (i < OPS) __builtin_amdgcn_sched_group_barrier(0x010, 1, 0);
    }
  }
};

// The lane's 16 keys of the tile at `key` that row `row` sees, as bits.
template <typename A>
__device__ __forceinline__ uint32_t seen_bits(A& a, const Place& p, int row, int hf,
                                              int key, int there) {
  const KeyRange kr = key_range(a, row_of(a, p, row).qi + p.shift, p.k_len);
  const int k0 = key + 16 * hf, sink = a.sinks < kr.hi ? a.sinks : kr.hi;
  auto below = [](int x) -> uint32_t {  // bits of keys < x
    const int n = x < 0 ? 0 : (x > 16 ? 16 : x);
    return (1u << n) - 1u;
  };
  const uint32_t bits = below(kr.hi - k0) & (~below(kr.lo - k0) | below(sink - k0));
  return (there >> hf) & 1 ? bits : 0u;
}

// The launch's arguments (its first and only one) read again behind the loop: kept in scalar
// registers through it they would spill.
typedef const __attribute__((address_space(4))) WindowArgs LateArgs;
__device__ __forceinline__ LateArgs& late_args() {
  LateArgs* late = (LateArgs*)__builtin_amdgcn_kernarg_segment_ptr();
  asm volatile("" : "+s"(late));
  return *late;
}

// The lane, counted afresh (no register holds it through the loop).
__device__ __forceinline__ int lane_again() {
  uint32_t none = 0;
  asm volatile("" : "+v"(none));  // (else it is counted at the start)
  return static_cast<int>(__builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, none)));
}

// Rows whose products met a value that they do not see (0 * inf or 0 * NaN of a masked
// key): a wavefront's 32 rows taken again at their known maxima m, tile by tile through
// TILE bytes of LDS, values that are no numbers staged as 0 and added only where a row
// sees their key.  One load at a time, five to seven times the first pass (32K causal
// tokens x 32 heads, every head's first value infinite, so that all rows are taken again: on
// 8 key heads 43 ms in all, without it 7.4, on 32 57 and 7.3); batches of loads spill.
template <typename T, int D, int FORM>
__device__ __forceinline__ void rows_again(LateArgs& a, const Place& p, RowTile<T, D>& t,
                                           int lane, float m, char* lds) {
  using R = RowTile<T, D>;
  typedef typename R::op8 op8;
  constexpr bool PAGED = FORM == kPaged;
  constexpr int RPU = 1024 / R::KROW, LOADS = R::TILE / 1024;
  constexpr uint32_t kExp = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
  const int hf = lane >> 5, lr = lane & 31;
  const char* const kbase = static_cast<const char*>(a.k) + keys_at<FORM>(p, a.sk) * 2;
  const char* const vbase = static_cast<const char*>(a.v) + keys_at<FORM>(p, a.sv) * 2;
  const uint32_t krb = static_cast<uint32_t>(a.sk[1] * 2), vrb = static_cast<uint32_t>(a.sv[1] * 2);
  const int32_t* const table = PAGED ? a.table + p.b * a.table_stride : nullptr;
#pragma unroll
  for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) t.o_acc[dt][r] = 0.0f;
  const int lrow = lane / R::CPR, chunk = lane % R::CPR;
  // (one load at a time and fences between the products: few registers)
  // 16-byte chunk `chunk` of row i RPU + lrow of the tile
  auto load = [&](const char* base, uint64_t off0, uint64_t off1, int rows0, int rows1,
                  uint32_t rb, int i) __attribute__((always_inline)) -> v4i {
    const int row = i * RPU + lrow, in_half = row & 15;
    const bool second = i * RPU >= 16;
    v4i x = {0, 0, 0, 0};
    if (in_half < (second ? rows1 : rows0))
      x = *reinterpret_cast<const v4i*>(base + (second ? off1 : off0) +
                                        static_cast<uint64_t>(in_half) * rb + chunk * 16);
    return x;
  };
  for (int s = 0; s < p.steps; ++s) {
    const Step st = step_of<PAGED>(a, p, table, s);
    const HalfRows h0 = half_rows<PAGED>(a, st, 0, p.k_len, krb, vrb);
    const HalfRows h1 = half_rows<PAGED>(a, st, 1, p.k_len, krb, vrb);
#pragma unroll 1
    for (int i = 0; i < LOADS; ++i) {
      const int row = i * RPU + lrow;
      *reinterpret_cast<v4i*>(lds + row * R::KROW +
                              ((chunk ^ (swz_k<R::KROW>(row) & (R::CPR - 1))) * 16)) =
          load(kbase, h0.k, h1.k, h0.rows, h1.rows, krb, i);
    }
    v16f s_acc;
#pragma unroll
    for (int r = 0; r < 16; ++r) s_acc[r] = 0.0f;
#pragma unroll
    for (int q = 0; q < R::QSTEPS; ++q) {
      s_acc = Half<T>::mfma(
          __builtin_bit_cast(op8, *reinterpret_cast<const v4i*>(lds + t.k_off[q])), t.q_op[q],
          s_acc);
      __builtin_amdgcn_sched_barrier(0);
    }
    const uint32_t own = seen_bits(a, p, p.row0 + lr, hf, st.key, halves_there<PAGED>(a, st));
    const uint32_t other = __shfl_xor(own, 32, kWave);
    const uint32_t seen = hf ? other | (own << 16) : own | (other << 16);
    op8 p_op[2];
#pragma unroll
    for (int r = 0; r < 16; ++r)
      p_op[r >> 3][r & 7] = static_cast<T>(
          (own >> r) & 1u ? __builtin_amdgcn_exp2f(fmaf(s_acc[r], a.scale_log2, -m)) : 0.0f);
    uint32_t odd = 0;  // keys of the tile with values that are no numbers
#pragma unroll 1
    for (int i = 0; i < LOADS; ++i) {
      const int row = i * RPU + lrow;
      v4i x = load(vbase, h0.v, h1.v, h0.rows, h1.rows, vrb, i);
      bool bad = false;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const uint32_t v = static_cast<uint32_t>(x[w]);
        const bool lo = (v & kExp) == kExp, hi = (v & (kExp << 16)) == kExp << 16;
        x[w] = static_cast<int>((lo ? 0u : v & 0xffffu) | (hi ? 0u : v & 0xffff0000u));
        bad = bad || lo || hi;
      }
      const uint64_t lanes = __ballot(bad);
#pragma unroll
      for (int r = 0; r < RPU; ++r)  // (CPR lanes a row)
        if ((lanes >> (r * R::CPR)) & ((1ull << R::CPR) - 1)) odd |= 1u << (i * RPU + r);
      *reinterpret_cast<v4i*>(lds + row * R::KROW +
                              ((chunk ^ (swz_v(row) & (R::CPR - 1))) * 16)) = x;
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
#pragma unroll
      for (int dt = 0; dt < R::NDT; ++dt) {
        const char* const p0 = lds + t.v_off[dt] - R::TILE + 8 * u * R::KROW;
        const auto lo = Half<T>::read_tr(p0);
        const auto hi = Half<T>::read_tr(p0 + 4 * R::KROW);
        t.o_acc[dt] = Half<T>::mfma(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7),
                                    p_op[u], t.o_acc[dt]);
        __builtin_amdgcn_sched_barrier(0);
      }
    for (; odd != 0; odd &= odd - 1) {
      const int j = __builtin_ctz(odd);
      const char* const row = vbase + (j < 16 ? h0.v : h1.v) + static_cast<uint64_t>(j & 15) * vrb;
      const bool sees = (seen >> j) & 1u;
#pragma unroll
      for (int dt = 0; dt < R::NDT; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const typename Half<T>::op4 v = *reinterpret_cast<const typename Half<T>::op4*>(
              row + (32 * dt + 8 * g + 4 * hf) * 2);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float f = static_cast<float>(v[e]);
            if (sees && !(fabsf(f) < INFINITY)) t.o_acc[dt][4 * g + e] += f;
          }
          __builtin_amdgcn_sched_barrier(0);
        }
    }
  }
}

// The end of a wavefront's rows: normalise, write the rows and the LSE, or with more than one
// share the share's partial rows to part_o [32][D] and their (max, sum) to part_ml [32].
// lds: TILE bytes of the wavefront's own.
template <typename T, int D, int FORM>
__device__ __forceinline__ void finish_rows(const Place& p, RowTile<T, D>& t, float* part_o,
                                            float2* part_ml, char* lds) {
  LateArgs& a = late_args();
  const int lane = lane_again();
  typedef typename Half<T>::op4 op4;
  const int hf = lane >> 5, lr = lane & 31;
  const float l = pair_sum(t.l_run), m = t.m_run;
  const float inv = l > 0.0f ? 1.0f / l : l;  // (a NaN sum stays one)
  // a product that is no number, in a row whose sum is one
  bool bad = false;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) bad = bad || !(fabsf(t.o_acc[dt][r]) < INFINITY);
  if (__ballot(bad && l > 0.0f && l < INFINITY) != 0)
    rows_again<T, D, FORM>(a, p, t, lane, m == -INFINITY ? 0.0f : m, lds);
  // (a select: a row that sees no key may hold 0 * inf of its neighbours' tiles)
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int r = 0; r < 16; ++r) t.o_acc[dt][r] = l == 0.0f ? 0.0f : t.o_acc[dt][r] * inv;
  const Row my = row_of(a, p, p.row0 + lr);
  if (my.live) {
    if (p.shares > 1) {
      float* const wp = part_o + lr * D + 4 * hf;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *reinterpret_cast<v4f*>(wp + 32 * dt + 8 * g) =
              v4f{t.o_acc[dt][4 * g], t.o_acc[dt][4 * g + 1], t.o_acc[dt][4 * g + 2],
                  t.o_acc[dt][4 * g + 3]};
      if (hf == 0)
        part_ml[lr] = make_float2(l > 0.0f ? m : (l == 0.0f ? -INFINITY : l), l);
    } else {
      T* const op = static_cast<T*>(a.out) + rows_at<FORM>(p, a.so) +
                    static_cast<int64_t>(my.qi) * a.so[1] + my.head * a.so[2] + 4 * hf;
#pragma unroll
      for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          op4 w;
#pragma unroll
          for (int e = 0; e < 4; ++e) w[e] = static_cast<T>(t.o_acc[dt][4 * g + e]);
          *reinterpret_cast<op4*>(op + 32 * dt + 8 * g) = w;
        }
      if (hf == 0 && a.lse)
        a.lse[lse_at<FORM>(a, p, my.head, my.qi)] =
            l == 0.0f ? -INFINITY : (m + __log2f(l)) * 0.69314718055994531f;
    }
  }
}

// Packed requests.  A row block's number is its rank, in one of two orders.
//
// In their order (windows, whose blocks cost alike; no order among positions; more than
// kMaxRanked requests): request b has the ranks from floor(q_off[b] G / 128) + b on, one more at
// most than it has blocks.
// Longest first, where rows see every key before them and B <= kMaxRanked: the level of block i
// of a request is i and the blocks that its earlier keys would fill, and ranks go through the
// levels from the highest on, at one level through the requests.  The rank's level
// is searched by counting the blocks at or above one, a lane a request.
constexpr int kMaxRanked = 512;

// Over the lanes, of values that are not negative, in registers: a shuffle through LDS takes
// ten times as long.
template <typename F>
__device__ __forceinline__ int lanes_fold(int x, F&& f) {
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true));  // row_shr:1
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true));  // row_shr:2
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true));  // row_shr:4
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true));  // row_shr:8
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, true));  // row_bcast:15
  x = f(x, __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, true));  // row_bcast:31
  return __builtin_amdgcn_readlane(x, kWave - 1);
}
__device__ __forceinline__ int lanes_sum(int x) {
  return lanes_fold(x, [](int a, int b) __attribute__((always_inline)) { return a + b; });
}
__device__ __forceinline__ int lanes_max(int x) {
  return lanes_fold(x, [](int a, int b) __attribute__((always_inline)) { return a > b ? a : b; });
}
// Which block of ranks and key head workgroup `id` of a share takes (rank -1: none).  Longest
// first: the key heads of a rank side by side.  In their order: XCD x (workgroups go
// round-robin) a contiguous run of a key head's ranks, so that neighbours share most of their
// window in its L2 (clips of up to 20 frames, window 12 and the first, 24 heads 2572 us; key heads
// side by side 2710).
struct RankAt {
  int rank, hk;
};
__device__ __forceinline__ RankAt rank_at(const WindowArgs& a, int id) {
  if (a.descending) {
    const int rank = divide(id, a.by_Hk);
    return {rank, id - rank * a.Hk};
  }
  const int item = id % kNumXcd * a.xcd_items + id / kNumXcd;
  const int hk = divide(item, a.by_rblocks);
  return {hk < a.Hk ? item - hk * a.n_ranks : -1, hk};
}
struct Packed {
  int b, rblock;  // b -1: no such block
};
__device__ __forceinline__ Packed packed_at(const WindowArgs& a, int rank, int lane) {
  auto blocks_of = [&](int b, int* level) __attribute__((always_inline)) -> int {
    const RowsOf q = rows_of(a.q_off, b, a.Lq), k = rows_of(a.k_off, b, a.Lk);
    const int before = k.count - q.count;
    const int64_t full = (before > 0 ? static_cast<int64_t>(before) * a.G : 0) >> 7;
    *level = static_cast<int>(full < (1 << 29) ? full : 1 << 29);  // (an order alone)
    return (q.count * a.G + 127) >> 7;
  };
  if (!a.descending) {
    auto first = [&](int b) __attribute__((always_inline)) -> int64_t {
      int o = a.q_off[b];
      o = o < 0 ? 0 : (o > a.Lq ? a.Lq : o);
      return ((static_cast<int64_t>(o) * a.G) >> 7) + b;
    };
    const int b = request_at(a.B, rank, lane, first);
    if (b < 0) return {-1, 0};
    int level;
    const int rblock = static_cast<int>(rank - first(b));
    return {rblock < blocks_of(b, &level) ? b : -1, rblock};
  }
  constexpr int PER = kMaxRanked / kWave;
  int n[PER], at[PER], top = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    n[i] = at[i] = 0;
    if (i * kWave < a.B && i * kWave + lane < a.B) n[i] = blocks_of(i * kWave + lane, &at[i]);
    top = n[i] > 0 && at[i] + n[i] > top ? at[i] + n[i] : top;
  }
  auto from = [&](int level) __attribute__((always_inline)) -> int {  // blocks at it or above
    int c = 0;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      if (i * kWave >= a.B) break;
      const int x = at[i] + n[i] - level;
      c += x < 0 ? 0 : (x < n[i] ? x : n[i]);
    }
    return lanes_sum(c);
  };
  int lo = 0, hi = top;  // from(lo) > rank >= from(hi)
  if (from(0) <= rank) return {-1, 0};
  hi = lanes_max(hi);
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (from(mid) > rank) lo = mid;
    else hi = mid;
  }
  int skip = rank - from(lo + 1);  // requests with a block at level lo before the rank's
  for (int i = 0; i < PER; ++i) {
    int ni = 0, ai = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (j == i) {
        ni = n[j];
        ai = at[j];
      }
    const bool has = ai <= lo && lo < ai + ni;
    const uint64_t with = __ballot(has);
    const int c = __builtin_popcountll(with);
    if (skip < c) {
      const int mine = static_cast<int>(__builtin_amdgcn_mbcnt_hi(
          static_cast<uint32_t>(with >> 32),
          __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(with), 0)));
      const int l = __builtin_ctzll(__ballot(has && mine == skip));
      return {i * kWave + l, lo - __builtin_amdgcn_readlane(ai, l)};
    }
    skip -= c;
  }
  return {-1, 0};
}
// The rows of block `rblock` of packed request b: lengths and first rows (n_rows 0: none).
__device__ __forceinline__ int packed_place(const WindowArgs& a, Place& p) {
  const RowsOf q = rows_of(a.q_off, p.b, a.Lq), k = rows_of(a.k_off, p.b, a.Lk);
  p.q0 = uniform_int(q.first);
  p.k0 = uniform_int(k.first);
  p.k_len = uniform_int(k.count);
  return uniform_int(q.count);
}

// acc += w o in a join: the weight of a share far below the row's maximum underflows to 0,
// which must not turn an infinity that the row sees into 0 * inf.
__device__ __forceinline__ float join(float w, float o, float acc) {
  return fmaf(w == 0.0f && !(fabsf(o) < INFINITY) ? 1.0f : w, o, acc);
}

// Blocks of 128 rows over pages (window_paged.hip); type 0: bf16, 1: fp16.
void launch_window_paged(WindowArgs& a, int type, int64_t D, dim3 grid, hipStream_t s);
// Packed requests, whole or in shares and their join (window_packed.hip).
int launch_window_packed(WindowArgs& a, int type, int64_t D, hipStream_t s);
// Few rows (window_units.hip): in units and their join, or one workgroup a key head
// (a.units 0); `units` of them are launched.
int launch_window_units(WindowArgs& a, int type, int64_t D, int64_t units, hipStream_t s);
int launch_unit_merge(WindowArgs& a, int type, int64_t D, hipStream_t s);

}  // namespace rcsa
