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
  int window, sinks, block;         // block 0: no order among positions
  float scale_log2;                 // sm_scale * log2(e)
  int n_rblocks;                    // blocks of rows of a key head
  int64_t n_items;                  // B * Hk * n_rblocks
  int n_split;
  float* ws_o;                      // [n_split][n_items][rows][D] normalised partial outputs
  float2* ws_ml;                    // [n_split][n_items][rows] their (max, sum)
};

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
