// Windowed attention, blocks of 128 rows: the dense form, the join of split blocks, plans and
// the entry points (the paged form is in a source of its own: see window_paged.hip).
#include "window_tile.h"

namespace rcsa {

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
  const ItemAt at = item_at(a, xcd, in_xcd);
  if (at.bh < 0) return;
  const int b = divide(at.bh, a.by_Hk), hk = at.bh - b * a.Hk;
  const int q_len = request_of(a, b).q_len;
  const int row = at.rblock * BM + static_cast<int>(wrow % BM);
  if (row >= q_len * a.G) return;
  const int qi = divide(row, a.by_G), head = hk * a.G + row - qi * a.G;
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
  typename Half<T>::op8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = static_cast<T>(acc[j] * inv);
  T* const op = static_cast<T*>(a.out) + b * a.so[0] + qi * a.so[1] + head * a.so[2] + c * 8;
  *reinterpret_cast<typename Half<T>::op8*>(op) = r;
  if (a.lse && c == 0)
    a.lse[(static_cast<int64_t>(b) * a.Hq + head) * a.Lq + qi] =
        sum == 0.0f ? -INFINITY : (mx + __log2f(sum)) * 0.69314718055994531f;
}

template <typename T, int D>
static int launch_window(WindowArgs& a, hipStream_t s) {
  const int64_t tail = a.xcd_items - a.xcd_whole;
  const int64_t wgs = (a.xcd_whole + tail * a.n_split) * kNumXcd;
  if (wgs * 256 >= kMaxThreads) return RCSA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(wgs));
  if (a.table) launch_window_paged(a, std::is_same<T, __bf16>::value ? 0 : 1, D, grid, s);
  else window_kernel<T, D, false><<<grid, dim3(256), 0, s>>>(a);
  if (a.n_split > 1 && tail > 0) {
    const int64_t n = (tail * kNumXcd * 128 * (D / 8) + 255) / 256;
    window_merge_kernel<T, D><<<dim3(static_cast<unsigned>(n)), dim3(256), 0, s>>>(a);
  }
  return launch_status();
}

// Blocks of rows of a key head.
static int64_t row_blocks(int64_t Lq, int64_t G) { return (Lq * G + 127) / 128; }

constexpr int64_t kMostKeys = 1ll << 30;

static bool few_rows(const int64_t* d) { return d[1] * (d[3] / d[4]) <= kFewRows; }
// Whether few rows fit a launch of a workgroup a key head, or of units and their join.
static bool group_fits(const int64_t* d) {
  return few_rows(d) && d[0] * d[4] * (64 * kGroupWaves) < kMaxThreads;
}
static bool units_fit(const int64_t* d) {
  return few_rows(d) && d[0] <= kMaxPlanned && d[0] * d[1] * d[3] * 256 < kMaxThreads;
}
// Wavefronts of few rows in units that fit at once: two (D 64: three) to a SIMD.
static int64_t units_of_round(const int64_t* d) { return (d[5] == 128 ? 8 : 12) * 256; }

// Units that a launch of few rows can have, over requests of at most `storage` keys: of their
// storage, or of the window and first keys of Lq positions; of any length the plan's (see
// chunk_of).  (A grid for any length: 16 x 32 heads x 256 keys 15.3 us, so 14.7; 64 x 512 keys
// of 8 heads 15.6 and 15.2; long ones are the same.)
static int64_t units_of_launch(const int64_t* d, int64_t storage, int64_t window, int64_t sinks) {
  int64_t tiles = (storage + kTileKeys - 1) / kTileKeys;
  if (window > 0) {
    const int64_t seen =
        (window + d[1]) / kTileKeys + 2 + (sinks + kTileKeys - 1) / kTileKeys;
    tiles = seen < tiles ? seen : tiles;
  }
  const int64_t heads = d[0] * d[4];
  const int64_t each = tiles <= kLeastTiles ? 1 : (tiles + kLeastTiles - 1) / kLeastTiles;
  const int64_t any = 4 * units_of_round(d) + heads;
  return heads * each < any ? heads * each : any;
}

// A workgroup a key head takes about 6.5 us and 0.25 a tile (the loads' latency, eight
// wavefronts) where the bandwidth does not bind; units take 11 us, their join among them, and
// their bytes at 5 TB/s (3.3 ns a tile of D 128).  Measured, us, workgroup and units:
// 8 heads x 256 keys 8.4, 11.1; 8 x 1024 13.1, 11.4; 32 x 1024 14.2, 14.7; 128 x 1024
// 18.9, 23.1; 64 x 4096 41.1, 32.6; 512 x 2048 100, 117; 2048 x 1024 205, 259.  Past 256
// tiles a single long request among short ones would hold its workgroup too long.
static bool one_group(const int64_t* d, int64_t tiles) {
  const int64_t heads = d[0] * d[4];
  return tiles <= 256 && (2500 - 33 * heads * d[5] / 128) * tiles < 45000;
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

// Few rows of a key head go to one workgroup (n_split -1) or to units of one wavefront (0),
// more to blocks of 128 rows.  Of these the ones past an XCD's whole rounds (one block to a
// compute unit) leave compute units idle: their keys go to n_split workgroups.  c =
// ceil(tail n / U) of them on a compute unit overlap a little and take c - 2/9 times as long
// as one (measured over 1210 tiles, 168 blocks: n 1 725 us, 2 526, 3 424, 4 440, 5 482, 6 448,
// 8 512); kFixed tiles for the start, as many and one a share for the join (128 blocks of 250
// tiles: n 2 95, 4 81, 6 83, 8 89; 168 of 83: n 1 57, 3 51, 5 62; 128 of 16: n 1 19, 2 26).
extern "C" int rcsa_window_attn_plan(const int64_t* dims, int64_t max_keys, int64_t* n_split) {
  if (!dims || !n_split) return RCSA_ERR_NULL;
  if (!window_dims(dims) || max_keys < 0) return RCSA_ERR_SHAPE;
  const int64_t tiles = (max_keys + kTileKeys - 1) / kTileKeys;
  const bool units = units_fit(dims);
  if (group_fits(dims) || units) {
    *n_split = group_fits(dims) && (!units || one_group(dims, tiles)) ? -1 : 0;
    return RCSA_OK;
  }
  *n_split = 1;
  const int64_t cux = xcd_cus(), items = xcd_items_of(dims);
  const int64_t tail = items % cux;
  if (tail == 0) return RCSA_OK;
  constexpr int64_t kFixed = 16;
  int64_t best = tiles + kFixed;
  for (int64_t n = 2; n <= 16 && n * 4 <= tiles; ++n) {
    const int64_t c = (tail * n + cux - 1) / cux, each = (tiles + n - 1) / n;
    const int64_t cost = (c == 1 ? each : (9 * c - 2) * each / 9) + 2 * kFixed + n;
    if (cost < best - best / 16) {
      best = cost;
      *n_split = n;
    }
  }
  return RCSA_OK;
}

extern "C" int64_t rcsa_window_attn_workspace_bytes_for(const int64_t* dims, int64_t n_split,
                                                        int64_t storage, int64_t window,
                                                        int64_t sinks) {
  if (!dims || !window_dims(dims) || n_split < -1 || n_split > 64) return -1;
  if (storage < 0 || storage > kMostKeys || window < 0 || sinks < 0) return -1;
  if (window >= kMostKeys) window = 0;
  if (sinks > kMostKeys) sinks = kMostKeys;
  const int64_t G = dims[3] / dims[4], row = dims[5] * 4 + 8;
  if (n_split < 1) {
    if (!(n_split < 0 ? group_fits(dims) : units_fit(dims))) return -1;
    return n_split < 0 ? 0
                       : units_of_launch(dims, storage, window, sinks) * dims[1] * G * row;
  }
  const int64_t items = xcd_items_of(dims);
  return n_split == 1 ? 0 : n_split * (items - xcd_whole_of(items, n_split)) * kNumXcd * 128 * row;
}

extern "C" int64_t rcsa_window_attn_workspace_bytes(const int64_t* dims, int64_t n_split) {
  return rcsa_window_attn_workspace_bytes_for(dims, n_split, kMostKeys, 0, 0);
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
  // (a masked logit is -inf before the scale; a zero one stays zero under a finite one)
  const float scale_log2 = sm_scale * 1.4426950408889634f;
  if (!window_dims(dims) || !(sm_scale > 0.0f && scale_log2 < INFINITY)) return RCSA_ERR_SHAPE;
  const int64_t most = kMostKeys;  // positions, windows and blocks stay far from 2^31
  if (dims[2] >= most || window < 0 || sinks < 0 || block < 0) return RCSA_ERR_SHAPE;
  if (block == 0 && (window != 0 || sinks != 0)) return RCSA_ERR_SHAPE;
  if (block_table && (max_pages <= 0 || n_pages <= 0 || page_size <= 0 || page_size % 16 ||
                      n_pages >= most || page_size >= most || max_pages >= most / page_size))
    return RCSA_ERR_SHAPE;
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
  const int64_t storage = block_table ? max_pages * page_size : dims[2];
  const int64_t need =
      rcsa_window_attn_workspace_bytes_for(dims, n_split, storage, window, sinks);
  if (need < 0 || (need > 0 && (!workspace || workspace_bytes < need))) return RCSA_ERR_SHAPE;
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
  if (block_table) a.by_half_page = divisor(static_cast<uint32_t>(page_size / 16));
  a.whole_tiles = page_size % kTileKeys == 0;
  a.window = static_cast<int>(window < most ? window : 0);
  a.sinks = static_cast<int>(sinks < most ? sinks : most);
  a.block = static_cast<int>(block < most ? block : most);
  a.scale_log2 = scale_log2;
  a.n_rblocks = static_cast<int>(row_blocks(a.Lq, a.G));
  a.n_items = static_cast<int64_t>(a.B) * a.Hk * a.n_rblocks;
  a.n_split = static_cast<int>(n_split);
  a.by_G = divisor(static_cast<uint32_t>(a.G));
  a.by_Hk = divisor(static_cast<uint32_t>(a.Hk));
  a.by_block = divisor(a.block > 0 ? static_cast<uint32_t>(a.block) : 1u);
  a.by_rblocks = divisor(static_cast<uint32_t>(a.n_rblocks));
  a.by_heads = divisor(static_cast<uint32_t>(a.B * a.Hk));
  a.units = n_split == 0 ? static_cast<int>(units_of_round(dims)) : 0;
  a.per_unit = a.units ? 1.0f / static_cast<float>(a.units) : 0.0f;
  const int64_t xcd_items = xcd_items_of(dims);
  if (xcd_items >= (1ll << 30)) return RCSA_ERR_SHAPE;
  a.xcd_items = static_cast<int>(xcd_items);
  a.xcd_whole = static_cast<int>(xcd_whole_of(xcd_items, n_split));
  // rows without a window see more keys the later they stand
  a.descending = a.window == 0 && a.block != 0;
  const int64_t ws_rows = need / (dims[5] * 4 + 8);
  a.ws_o = static_cast<float*>(workspace);
  a.ws_ml = need ? reinterpret_cast<float2*>(a.ws_o + ws_rows * dims[5]) : nullptr;
  if (n_split < 1)
    return launch_window_units(a, dtype == RCSA_BF16 ? 0 : 1, dims[5],
                               units_of_launch(dims, storage, a.window, a.sinks), stream);
  if (dtype == RCSA_BF16)
    return dims[5] == 128 ? launch_window<__bf16, 128>(a, stream)
                          : launch_window<__bf16, 64>(a, stream);
  return dims[5] == 128 ? launch_window<_Float16, 128>(a, stream)
                        : launch_window<_Float16, 64>(a, stream);
}
