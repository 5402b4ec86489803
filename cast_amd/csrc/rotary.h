// Arguments of the rotary kernels (rotary.hip).
#pragma once
#include "rcsa_common.h"

namespace rcsa {

constexpr int kMaxTokens = 32;   // tokens of a workgroup
constexpr int kMaxDim = 512;     // channels of a head
constexpr int kMaxHeads = 4096;

struct RotaryArgs {
  const void *q, *k, *v;      // [B, L, H, D] by strides (batch, token, head)
  void *qout, *kout, *vout;   // the same, or with a table pages by (page, slot, head)
  int64_t qs[3], ks[3], vs[3], qo[3], ko[3], vo[3];
  int64_t B, L;
  int Hq, Hk, Hv, D;
  const void* pos;            // int32 or int64, by (batch, token, axis) strides
  int pos_i64, n_axes;
  int64_t pos_b, pos_l, pos_a;
  const double* turns;        // turns per position of every pair
  const int32_t* axis;        // its position axis (NULL: 0)
  int n_pairs;
  float scale;
  const void *qw, *kw;        // norm weights (NULL: 1), head strides 0 or D
  int w_dtype;
  int64_t qw_h, kw_h;
  float eps;
  const int32_t* table;       // [B][max_pages] pages of every request's cache
  int64_t table_stride, max_pages, n_pages, page_size;
  const int32_t *starts, *lengths;
  Divisor by_L, by_page;
  // the vector form's launch: tokens of a workgroup, lanes of a head (log2), divisors
  int tokens, lanes_log2;
  Divisor by_heads, by_pairs;  // by_heads: Hq + Hk + Hv
};

}  // namespace rcsa
