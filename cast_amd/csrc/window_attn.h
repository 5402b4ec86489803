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
  float* ws_o;                      // [n_split][n_items][rows][D] normalised partial outputs
  float2* ws_ml;                    // [n_split][n_items][rows] their (max, sum)
  // few rows (one wavefront a unit): units wanted in all, 0: one a key head
  int units;
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

// Few rows: the visible tiles of all requests are dealt to about a.units wavefronts in
// units of `chunk` tiles of one key head, however uneven the lengths.  A wavefront
// reads the lengths (one lane a request) and finds its unit; u = (units of the
// requests before) * Hk + share * Hk + hk.
constexpr int kLeastTiles = 2;
__device__ __forceinline__ int request_tiles(const WindowArgs& a, int b) {
  const Request r = request_of(a, b);
  if (r.q_len == 0) return -1;
  const int p = r.k_len - r.q_len;
  return tiles_of(a, key_range(a, p, r.k_len), key_range(a, p + r.q_len - 1, r.k_len)).all();
}
// Tiles of a unit: all lanes of the wavefront call it.
__device__ __forceinline__ int unit_chunk(const WindowArgs& a, int lane) {
  if (a.units == 0) return 1 << 30;
  int64_t total = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int n = b0 + lane < a.B ? request_tiles(a, b0 + lane) : 0;
    int s = n > 0 ? n : 0;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
    total += s;
  }
  const int64_t c = (total * a.Hk + a.units - 1) / a.units;
  return c < kLeastTiles ? kLeastTiles : static_cast<int>(c);
}
__device__ __forceinline__ int units_of(int tiles, int chunk) {
  return tiles < 0 ? 0 : (tiles <= chunk ? 1 : (tiles + chunk - 1) / chunk);
}
// Units of the requests before b (all lanes call it).
__device__ __forceinline__ int units_before(const WindowArgs& a, int b, int chunk, int lane) {
  if (a.units == 0) return b;
  int s = 0;
  for (int b0 = 0; b0 < b; b0 += kWave)
    if (b0 + lane < b) s += units_of(request_tiles(a, b0 + lane), chunk);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, kWave);
  return s;
}
// The request, share and number of shares of unit index w (of one key head), b -1 past
// the last (all lanes call it).
struct Unit {
  int b, share, shares;
};
__device__ __forceinline__ Unit unit_at(const WindowArgs& a, int w, int chunk, int lane) {
  if (a.units == 0) return {w < a.B ? w : -1, 0, 1};
  int before = 0;
  for (int b0 = 0; b0 < a.B; b0 += kWave) {
    const int n = b0 + lane < a.B ? units_of(request_tiles(a, b0 + lane), chunk) : 0;
    int sum = n;  // inclusive prefix over the lanes
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
      const int up = __shfl_up(sum, o, kWave);
      if (lane >= o) sum += up;
    }
    const uint64_t past = __ballot(before + sum > w);
    if (past != 0) {
      const int l = __builtin_ctzll(past);
      return {b0 + l, w - before - __shfl(sum - n, l, kWave), __shfl(n, l, kWave)};
    }
    before += __shfl(sum, kWave - 1, kWave);
  }
  return {-1, 0, 0};
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
