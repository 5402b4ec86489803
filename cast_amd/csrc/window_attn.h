// Windowed attention over dense or paged keys: arguments and helpers shared by
// the tile kernel (window_attn.hip).
//
// Query i of a request with q_len queries and k_len keys is at position
// p = i + k_len - q_len; e(p) = (floor(p / block) + 1) * block is the end of its
// block of positions.  It sees key j when
//   j < min(e, k_len) and (j >= e - window or j < sinks)
// (window 0: every key below e; block 0: every key), and
//   out = softmax_j(sm_scale q . k_j) v,  lse = log sum_j exp(sm_scale q . k_j).
// The G = Hq / Hk query heads of a key head are rows of one problem: row r is
// query r / G of head hk * G + r % G, so every staged key serves all of them and
// a tile of rows spans few positions.
#pragma once
#include "sparse_attn_kernel.h"

namespace rcsa {

typedef _Float16 v8hf __attribute__((ext_vector_type(8)));
typedef _Float16 v4hf __attribute__((ext_vector_type(4)));

constexpr int kTileKeys = 32;

struct WindowArgs {
  const void *q, *k, *v;
  void* out;
  float* lse;                       // [B][Hq][Lq], nullable
  int64_t sq[3], sk[3], sv[3], so[3];  // (batch, row, head); paged k, v: (page, slot, head)
  int B, Lq, Lk, Hq, Hk, G;
  const int32_t *q_len, *k_len;     // [B], nullable: Lq, Lk
  const int32_t* table;             // [B][max_pages], nullable: dense k, v
  int64_t table_stride;
  int max_pages, n_pages, page;     // page: keys of a page, a multiple of 16
  uint32_t page_mul;                // division of half tiles by the halves of a page
  int page_sh1, page_sh2;
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
  int units;  // few rows: the wavefronts that fit in one round, 0: one unit a key head
};

constexpr int kFewRows = 32;        // rows of a key head that one wavefront takes
constexpr int kMaxPlanned = 512;    // requests whose lengths every wavefront reads

// The keys of a position: [0, sink) and [lo, hi).
struct KeyRange {
  int lo, hi;
};
__device__ __forceinline__ KeyRange key_range(const WindowArgs& a, int p, int k_len) {
  if (a.block == 0) return {0, k_len};
  if (p < 0) return {0, 0};
  const int e = (a.block == 1 ? p : p / a.block * a.block + a.block - 1) + 1;
  const int hi = e < k_len ? e : k_len;
  const int lo = a.window == 0 || e <= a.window ? 0 : e - a.window;
  return {lo < hi ? lo : hi, hi};
}

// A request's lengths, clamped to the storage.
struct Request {
  int k_len, q_len;
};
__device__ __forceinline__ Request request_of(const WindowArgs& a, int b) {
  const int cap = a.table != nullptr ? a.max_pages * a.page : a.Lk;
  int k = a.k_len == nullptr ? cap : a.k_len[b];
  int q = a.q_len == nullptr ? a.Lq : a.q_len[b];
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

// Few rows: the visible tiles of all requests are dealt to units of one wavefront each,
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
// units of a last, short round leave compute units idle.
constexpr int kLeastTiles = 2, kUnitTiles = 16;
__device__ __forceinline__ int chunk_of(const WindowArgs& a, int64_t total) {
  const int64_t t = total * a.Hk;
  const int64_t one = (t + a.units - 1) / a.units;
  int64_t c = (t + 4 * a.units - 1) / (4 * a.units);
  c = c < kUnitTiles ? kUnitTiles : c;
  c = c < one ? c : one;
  return static_cast<int>(c < kLeastTiles ? kLeastTiles : c);
}
struct Unit {
  int b, share, shares;  // b -1: no such unit
  int before;            // units (of one key head) of the requests before b
  Request r;
};
__device__ __forceinline__ int uniform_int(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ int lane_sum(int x) {
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
  if (a.units == 0) {  // a unit for every request
    if (w >= a.B) return {-1, 0, 0, 0, {0, 0}};
    const Request r = request_of(a, w);
    return {w, 0, 1, w, {uniform_int(r.k_len), uniform_int(r.q_len)}};
  }
  if (a.B <= kWave) {  // one load of the lengths (a single request needs no lanes' sums)
    Request r{0, 0};
    if (lane < a.B) r = request_of(a, lane);
    const int tiles = lane < a.B ? request_tiles(a, r) : -1;
    const int mine = tiles > 0 ? tiles : 0;
    const int chunk = chunk_of(a, a.B == 1 ? uniform_int(mine) : uniform_int(lane_sum(mine)));
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
  int64_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int t = b0 + lane < a.B ? request_tiles(a, request_of(a, b0 + lane)) : 0;
    total += lane_sum(t > 0 ? t : 0);
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
  static __device__ __forceinline__ v16f mfma(op8 x, op8 y, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x, y, c, 0, 0, 0);
  }
  static __device__ __forceinline__ op4 read_tr(const char* p) {
    return __builtin_bit_cast(op4, __builtin_amdgcn_ds_read_tr16_b64_v4bf16(RCSA_LDS(v4bf, p)));
  }
};

}  // namespace rcsa
