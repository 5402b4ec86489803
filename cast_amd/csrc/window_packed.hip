// Attention over packed requests: window_tile.h's blocks of 128 rows, found from the offsets on
// the device, so that a captured call follows them and the host reads nothing back.  Blocks with
// many keys go first where there is no window (see packed_at).
//
// Bound by the matrix pipe under the power limit: 9 prompts of up to 8192 tokens behind up to
// 1500 held ones, 32 heads on 8 of D 128, 1475 us, 1150 TFLOP/s (pipe 69% busy at 1.66 GHz); clips
// of up to 20 frames of 880 under a window of 12 and the first, 24 heads, 2540 us, 1140 TFLOP/s
// (72%).
// 40 prompts of up to 301 tokens take 11.8 us: a launch, the search and one short row block.
#include "window_tile.h"

namespace rcsa {

// The shares of the row blocks joined (window_merge_kernel's sums): a thread a row and 8 channels,
// a workgroup inside one row block.
template <typename T, int D>
__global__ void __launch_bounds__(256) packed_merge_kernel(WindowArgs a) {
  constexpr int CPR = D / 8, BM = 128, WGS = BM * CPR / 256;  // workgroups of a row block
  const int id = static_cast<int>(blockIdx.x) / WGS;
  const RankAt at = rank_at(a, id);
  if (at.rank < 0) return;
  const Packed it = packed_at(a, at.rank, threadIdx.x & 63);
  if (it.b < 0) return;
  Place p;
  p.b = it.b;
  const int n_rows = packed_place(a, p) * a.G;
  const int v = static_cast<int>(blockIdx.x) % WGS * 256 + threadIdx.x;
  const int in_block = v / CPR, c = v % CPR, row = it.rblock * BM + in_block;
  if (row >= n_rows) return;
  const int qi = divide(row, a.by_G), head = at.hk * a.G + row - qi * a.G;
  const int64_t all_rows = static_cast<int64_t>(a.xcd_items) * kNumXcd * BM;
  const int64_t wrow = static_cast<int64_t>(id) * BM + in_block;
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
    for (int j = 0; j < 8; ++j) acc[j] = join(w, o[j], acc[j]);
  }
  const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
  T* const op = static_cast<T*>(a.out) + static_cast<int64_t>(p.q0 + qi) * a.so[1] +
                head * a.so[2] + c * 8;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    typename Half<T>::op4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = static_cast<T>(acc[4 * h + j] * inv);
    *reinterpret_cast<typename Half<T>::op4*>(op + 4 * h) = r;
  }
  if (a.lse && c == 0)
    a.lse[lse_at<kPacked>(a, p, head, qi)] =
        sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

template <typename T, int D>
static int launch(WindowArgs& a, hipStream_t s) {
  const int64_t items = static_cast<int64_t>(a.xcd_items) * kNumXcd;
  constexpr int64_t merges = 128 * (D / 8) / 256;
  if (items * a.n_split * 256 >= kMaxThreads || items * merges * 256 >= kMaxThreads)
    return RCSA_ERR_SHAPE;
  window_kernel<T, D, kPacked>
      <<<dim3(static_cast<unsigned>(items * a.n_split)), dim3(256), 0, s>>>(a);
  if (a.n_split > 1)
    packed_merge_kernel<T, D><<<dim3(static_cast<unsigned>(items * merges)), dim3(256), 0, s>>>(a);
  return launch_status();
}

int launch_window_packed(WindowArgs& a, int type, int64_t D, hipStream_t s) {
  if (type == 0) return D == 128 ? launch<__bf16, 128>(a, s) : launch<__bf16, 64>(a, s);
  return D == 128 ? launch<_Float16, 128>(a, s) : launch<_Float16, 64>(a, s);
}

// Row blocks of a key head of packed requests, at most; of an XCD.
static int64_t ranks_of(const int64_t* d) { return (d[1] * (d[3] / d[4])) / 128 + d[0]; }
static int64_t xcd_ranks_of(const int64_t* d) {
  return (ranks_of(d) * d[4] + kNumXcd - 1) / kNumXcd;
}

static bool packed_dims(const int64_t* d) {
  for (int i = 0; i < 6; ++i)
    if (d[i] <= 0 && !(i == 2 && d[i] == 0)) return false;
  return d[4] <= d[3] && d[3] % d[4] == 0 && d[0] < (1 << 20) && d[1] < (1 << 30) &&
         d[2] < (1 << 30) && d[3] < (1 << 16) && d[1] * (d[3] / d[4]) < (1 << 30) &&
         (d[5] == 64 || d[5] == 128) && ranks_of(d) * d[4] < (1ll << 24);
}

}  // namespace rcsa

using namespace rcsa;

// The shares of each row block's keys, in tiles' times (0.6 us of one workgroup for D 128): a
// share's tiles, or a compute unit's of all while rows see half of the keys; a share's rows
// written and merged, 1/13 a row block; the merge's launch.  One prompt of 3085 rows, 4 heads of
// D 128, in 1, 2, 3, 4, 8 shares 61, 46, 41, 41, 47 us; 6000 rows, 2 key heads of 8: 130, 111,
// 107, 120, 142; 2 of 2000 rows, 8 heads: 46, 52, 54, 58, 79.
extern "C" int rcsa_packed_attn_plan(const int64_t* dims, int64_t max_keys, int64_t* n_split) {
  if (!dims || !n_split) return RCSA_ERR_NULL;
  if (!packed_dims(dims) || max_keys < 0) return RCSA_ERR_SHAPE;
  const int64_t even = dims[2] / dims[0];  // (where the keys are spread evenly)
  const int64_t tiles = ((max_keys < even ? max_keys : even) + kTileKeys - 1) / kTileKeys;
  const int64_t cux = cus_per_xcd(), cus = (cux > 0 ? cux : 32) * kNumXcd;
  const int64_t items = ranks_of(dims) * dims[4], all = items * tiles * 2 / (5 * cus);
  *n_split = 1;
  int64_t best = tiles + 5;
  for (int64_t n = 2; n <= 16 && n * 4 <= tiles; ++n) {
    const int64_t each = (tiles + n - 1) / n;
    const int64_t cost = (each > all ? each : all) + items * n / 13 + 12;
    if (cost < best - best / 16) {
      best = cost;
      *n_split = n;
    }
  }
  return RCSA_OK;
}

extern "C" int64_t rcsa_packed_attn_workspace_bytes(const int64_t* dims, int64_t n_split) {
  if (!dims || !packed_dims(dims) || n_split < 1 || n_split > 64) return -1;
  return n_split == 1 ? 0 : n_split * xcd_ranks_of(dims) * kNumXcd * 128 * (dims[5] * 4 + 8);
}

extern "C" int rcsa_packed_attn(const void* q, const void* k, const void* v, void* out, float* lse,
                                int dtype, const int64_t* dims, const int64_t* strides,
                                const int32_t* q_offsets, const int32_t* k_offsets,
                                int64_t window, int64_t sinks, int64_t block, float sm_scale,
                                int64_t n_split, void* workspace, int64_t workspace_bytes,
                                hipStream_t stream) {
  if (!q || !k || !v || !out || !dims || !strides || !q_offsets || !k_offsets)
    return RCSA_ERR_NULL;
  if (dtype != RCSA_BF16 && dtype != RCSA_F16) return RCSA_ERR_DTYPE;
  const float scale_log2 = sm_scale * 1.4426950408889634f;
  if (!packed_dims(dims) || !(sm_scale > 0.0f && scale_log2 < INFINITY)) return RCSA_ERR_SHAPE;
  constexpr int64_t most = 1ll << 30;  // positions, windows and blocks stay far from 2^31
  if (window < 0 || sinks < 0 || block < 0) return RCSA_ERR_SHAPE;
  if (block == 0 && (window != 0 || sinks != 0)) return RCSA_ERR_SHAPE;
  for (int i = 0; i < 8; ++i)
    if (strides[i] < 0 || strides[i] % (i < 6 ? 8 : 4)) return RCSA_ERR_STRIDE;
  // (rows of keys do not overlap; the stride of a single one says nothing)
  for (int i = 2; i < 6; i += 2)
    if (strides[i] >= (1 << 25) || (dims[2] > 1 && strides[i] < dims[5])) return RCSA_ERR_STRIDE;
  if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(workspace) ||
      (reinterpret_cast<uintptr_t>(out) & 7u))
    return RCSA_ERR_ALIGN;
  const int64_t need = rcsa_packed_attn_workspace_bytes(dims, n_split);
  if (need < 0 || (need > 0 && (!workspace || workspace_bytes < need))) return RCSA_ERR_SHAPE;
  WindowArgs a{};
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.lse = lse;
  for (int i = 0; i < 2; ++i) {
    a.sq[1 + i] = strides[i];
    a.sk[1 + i] = strides[2 + i];
    a.sv[1 + i] = strides[4 + i];
    a.so[1 + i] = strides[6 + i];
  }
  if (dims[2] <= 1) a.sk[1] = a.sv[1] = dims[5];
  a.B = static_cast<int>(dims[0]);
  a.Lq = static_cast<int>(dims[1]);
  a.Lk = static_cast<int>(dims[2]);
  a.Hq = static_cast<int>(dims[3]);
  a.Hk = static_cast<int>(dims[4]);
  a.G = a.Hq / a.Hk;
  a.q_off = q_offsets;
  a.k_off = k_offsets;
  a.n_ranks = static_cast<int>(ranks_of(dims));
  a.xcd_items = static_cast<int>(xcd_ranks_of(dims));
  a.by_rblocks = divisor(static_cast<uint32_t>(a.n_ranks));
  a.window = static_cast<int>(window < most ? window : 0);
  a.sinks = static_cast<int>(sinks < most ? sinks : most);
  a.block = static_cast<int>(block < most ? block : most);
  a.scale_log2 = scale_log2;
  a.n_split = static_cast<int>(n_split);
  a.by_G = divisor(static_cast<uint32_t>(a.G));
  a.by_Hk = divisor(static_cast<uint32_t>(a.Hk));
  a.by_block = divisor(a.block > 0 ? static_cast<uint32_t>(a.block) : 1u);
  // rows without a window see more keys the later they stand
  a.descending = a.window == 0 && a.block != 0 && a.B <= kMaxRanked;
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = need ? reinterpret_cast<float2*>(a.ws_o + need / (dims[5] * 4 + 8) * dims[5])
                 : nullptr;
  return launch_window_packed(a, dtype == RCSA_BF16 ? 0 : 1, dims[5], stream);
}
