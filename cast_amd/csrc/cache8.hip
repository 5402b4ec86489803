// Keys and values into a paged cache in 8 bits as they are written, and back.
//
// rcsa_append_cache: for a block that gets new tokens x, with a = max |x| (of finite ones) and
// s0 the block's scale if it holds tokens before them, else 0,
//   s = max(s0, scale_for(a), 2^-100),  c = nearest(x / s),
// and, where s > s0, the codes before them c = nearest(c s0 / s).  The order of calls decides
// the result, nothing else: no atomics, one workgroup a block and head.
// rcsa_read_cache: c * s in fp32, rounded once.
#include "cache8.h"
#include "packed.h"

namespace rcsa {

struct AppendArgs {
  const void* x[2];         // keys, values [B][L][H][D], or packed [L][H][D]
  int64_t sx[2][3];         // batch, token, head
  char* codes[2];           // [pages][slots][H][D]
  int64_t sc[2][3];
  float* scales[2];         // [pages][blocks][H]
  int64_t ss[2][3];
  const int32_t *offsets, *starts, *lengths, *table;  // [B + 1] (packed), [B], [B], [B][max_pages]
  int64_t table_stride;
  int B, L, H, max_pages, n_pages, page, block, runs;  // runs: of 8 channels in a head
  int64_t items;            // blocks that a request (packed: all of them) can touch
  Divisor by_heads, by_runs, by_block, by_page_blocks, by_items;
  int page_blocks;          // blocks of a page
};

// The first of the items (blocks) of packed request b: as many as its rows can touch,
// at most floor(count / block) + 2, follow.
__device__ __forceinline__ int64_t first_item(const AppendArgs& a, int b) {
  int o = a.offsets[b];
  o = o < 0 ? 0 : (o > a.L ? a.L : o);
  return divide(o, a.by_block) + 2ll * b;
}

template <typename T, bool E4M3, bool PACKED, int THREADS>
__global__ void __launch_bounds__(THREADS) append_kernel(AppendArgs a) {
  using C = Code8<E4M3>;
  using R = Run8<T>;
  typedef typename R::V V;
  constexpr int HELD = 8;  // runs of a thread that stay in registers
  const int tid = threadIdx.x, lane = tid & 63;
  const int id = static_cast<int>(blockIdx.x);
  const int at = divide(id, a.by_heads), head = id - at * a.H;
  const int kv = at & 1, all = at >> 1;
  int b, item, row0, count;
  if constexpr (PACKED) {
    b = request_at(a.B, all, lane, [&](int i) __attribute__((always_inline)) {
      return first_item(a, i);
    });
    if (b < 0) return;
    const RowsOf r = rows_of(a.offsets, b, a.L);
    row0 = r.first;
    count = r.count;
    item = static_cast<int>(all - first_item(a, b));
  } else {
    b = divide(all, a.by_items);
    item = all - b * static_cast<int>(a.items);
    row0 = 0;
    count = a.L;
    if (a.lengths != nullptr) {
      const int n = a.lengths[b];
      count = n < 0 ? 0 : (n > a.L ? a.L : n);
    }
  }
  // new tokens are indexes [lo, hi) of the request, token index - start of x
  const int64_t start = a.starts == nullptr ? 0 : a.starts[b];
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  const int64_t lo = start < 0 ? 0 : start;
  const int64_t hi = start + count < cap ? start + count : cap;
  if (lo >= hi) return;
  const int n = divide(static_cast<int>(lo), a.by_block) + item;  // the block's number
  if (item < 0 || static_cast<int64_t>(n) * a.block >= hi) return;
  const int first = n * a.block;
  const int from = lo > first ? static_cast<int>(lo) - first : 0;  // rows [from, to) are new
  const int to = hi - first < a.block ? static_cast<int>(hi - first) : a.block;
  const int col = divide(n, a.by_page_blocks), in_page = n - col * a.page_blocks;
  const int page = a.table[b * a.table_stride + col];
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.n_pages)) return;

  const T* const x = static_cast<const T*>(a.x[kv]) + (PACKED ? 0 : b * a.sx[kv][0]) +
                     head * a.sx[kv][2] + (row0 + first + from - start) * a.sx[kv][1];
  char* const codes = a.codes[kv] + page * a.sc[kv][0] + head * a.sc[kv][2] +
                      static_cast<int64_t>(in_page) * a.block * a.sc[kv][1];
  float* const scale = a.scales[kv] + page * a.ss[kv][0] + in_page * a.ss[kv][1] +
                       head * a.ss[kv][2];
  float s0 = 0.0f;
  if (from > 0) {
    s0 = *scale;
    s0 = s0 > 0.0f && s0 < INFINITY ? s0 : 0.0f;
  }

  const int64_t xs = a.sx[kv][1], cs = a.sc[kv][1];
  const int runs = (to - from) * a.runs;
  auto load = [&](int i) __attribute__((always_inline)) -> V {
    const int row = divide(i, a.by_runs);
    return *reinterpret_cast<const V*>(x + row * xs + (i - row * a.runs) * 8);
  };
  float most = 0.0f;
  auto look = [&](const V& v) __attribute__((always_inline)) {
    float f[8];
    R::floats(v, f);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float m = fabsf(f[e]);
      most = fmaxf(most, m < INFINITY ? m : 0.0f);
    }
  };
  V held[HELD];
#pragma unroll
  for (int k = 0; k < HELD; ++k)
    if (tid + k * THREADS < runs) held[k] = load(tid + k * THREADS);
#pragma unroll
  for (int k = 0; k < HELD; ++k)
    if (tid + k * THREADS < runs) look(held[k]);
  for (int i = tid + HELD * THREADS; i < runs; i += THREADS) look(load(i));
  most = wave_max(most);
  if constexpr (THREADS > kWave) {
    __shared__ float s_most[THREADS / kWave];
    if (lane == 0) s_most[tid / kWave] = most;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < THREADS / kWave; ++w) most = fmaxf(most, s_most[w]);
  }
  const float own = C::scale_for(most);
  const float s = fmaxf(fmaxf(s0, own), kLeastScale);

  const typename C::To to_code(s);
  auto store = [&](int i, const V& v) __attribute__((always_inline)) {
    const int row = divide(i, a.by_runs);
    float f[8];
    R::floats(v, f);
    *reinterpret_cast<uint2*>(codes + (from + row) * cs + (i - row * a.runs) * 8) =
        make_uint2(to_code.four(f), to_code.four(f + 4));
  };
#pragma unroll
  for (int k = 0; k < HELD; ++k)
    if (tid + k * THREADS < runs) store(tid + k * THREADS, held[k]);
  for (int i = tid + HELD * THREADS; i < runs; i += THREADS) store(i, load(i));
  if (s != s0) {  // (a block's first scale, or a larger one)
    for (int i = tid; i < from * a.runs; i += THREADS) {
      const int row = divide(i, a.by_runs);
      uint2* const p = reinterpret_cast<uint2*>(codes + row * cs + (i - row * a.runs) * 8);
      const uint2 w = *p;
      *p = make_uint2(C::again(w.x, s0, s), C::again(w.y, s0, s));
    }
    // (every thread has read the block's old scale before the barrier, or, of one wavefront,
    // before this store)
    if (tid == 0) *scale = s;
  }
}

struct ReadArgs {
  const char* codes[2];
  int64_t sc[2][3];
  const float* scales[2];
  int64_t ss[2][3];
  void* out[2];             // [B][L][H][D]
  int64_t so[2][3];
  const int32_t *starts, *lengths, *table;
  int64_t table_stride;
  int B, L, H, max_pages, n_pages, page, block, runs;  // runs: of 8 channels in a head
  Divisor by_heads, by_runs, by_L, by_page, by_block;
  int64_t total;            // runs of the keys
};

template <typename T, bool E4M3>
__global__ void __launch_bounds__(256) read_kernel(ReadArgs a) {
  using C = Code8<E4M3>;
  using R = Run8<T>;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= a.total) return;
  const int kv = static_cast<int>(blockIdx.y);
  const int row = static_cast<int>(i / (a.runs * a.H));       // b, token
  const int in_row = static_cast<int>(i - static_cast<int64_t>(row) * a.runs * a.H);
  const int head = divide(in_row, a.by_runs), run = in_row - head * a.runs;
  const int b = divide(row, a.by_L), t = row - b * a.L;
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  const int64_t start = a.starts == nullptr ? 0 : a.starts[b];
  const int64_t j = start + t, len = a.lengths[b];
  if (j < 0 || j >= len || j >= cap) return;
  const int col = divide(static_cast<int>(j), a.by_page), slot = static_cast<int>(j) - col * a.page;
  const int page = a.table[b * a.table_stride + col];
  float f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0.0f;
  if (static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages)) {
    const uint2 w = *reinterpret_cast<const uint2*>(a.codes[kv] + page * a.sc[kv][0] +
                                                    slot * a.sc[kv][1] + head * a.sc[kv][2] +
                                                    run * 8);
    const float s = a.scales[kv][page * a.ss[kv][0] + divide(slot, a.by_block) * a.ss[kv][1] +
                                 head * a.ss[kv][2]];
    C::values(w.x, f);
    C::values(w.y, f + 4);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= s;
  }
  *reinterpret_cast<typename R::V*>(static_cast<T*>(a.out[kv]) + b * a.so[kv][0] +
                                    t * a.so[kv][1] + head * a.so[kv][2] + run * 8) = R::of(f);
}

constexpr int64_t kMaxThreads8 = 1ll << 32;  // a grid's dimension holds fewer

template <typename T, bool E4M3, bool PACKED>
static int launch_append(AppendArgs& a, hipStream_t s) {
  const int64_t wgs = (PACKED ? a.items : a.items * a.B) * 2 * a.H;
  const int64_t runs = static_cast<int64_t>(a.block) * a.runs;
  const int threads = runs <= 512 ? 64 : runs <= 2048 ? 256 : 1024;
  if (wgs >= (1ll << 31) || wgs * threads >= kMaxThreads8) return RCSA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(wgs));
  if (threads == 64) append_kernel<T, E4M3, PACKED, 64><<<grid, dim3(64), 0, s>>>(a);
  else if (threads == 256) append_kernel<T, E4M3, PACKED, 256><<<grid, dim3(256), 0, s>>>(a);
  else append_kernel<T, E4M3, PACKED, 1024><<<grid, dim3(1024), 0, s>>>(a);
  return launch_status();
}

template <typename T>
static int append_type(AppendArgs& a, bool e4m3, hipStream_t s) {
  if (a.offsets)
    return e4m3 ? launch_append<T, true, true>(a, s) : launch_append<T, false, true>(a, s);
  return e4m3 ? launch_append<T, true, false>(a, s) : launch_append<T, false, false>(a, s);
}

template <typename T>
static int read_type(ReadArgs& a, bool e4m3, hipStream_t s) {
  const int64_t wgs = (a.total + 255) / 256;
  if (wgs * 256 >= kMaxThreads8) return RCSA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(wgs), 2);
  if (e4m3) read_kernel<T, true><<<grid, dim3(256), 0, s>>>(a);
  else read_kernel<T, false><<<grid, dim3(256), 0, s>>>(a);
  return launch_status();
}

// The sizes of a cache and of a call's tokens [B][L][H][D].
static bool cache_dims(const int64_t* dims, int64_t max_pages, int64_t n_pages, int64_t page,
                       int64_t block) {
  for (int i = 0; i < 4; ++i)
    if (dims[i] <= 0) return false;
  if (dims[0] >= (1 << 20) || dims[1] >= kMostSlots || dims[0] > kMostSlots / dims[1] ||
      dims[2] > 4096 || dims[3] > 1024 || dims[3] % 8)
    return false;
  return max_pages > 0 && n_pages > 0 && n_pages < kMostSlots && page > 0 && block > 0 &&
         page % block == 0 && block % 16 == 0 && block <= (1 << 16) && max_pages < kMostSlots / page;
}

// Strides of rows of 8-channel runs (elements), and their pointers.
static bool strides_ok(const int64_t* s, int n, int64_t unit) {
  for (int i = 0; i < n; ++i)
    if (s[i] < 0 || s[i] % unit) return false;
  return true;
}
static bool aligned8(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 7u) == 0; }

}  // namespace rcsa

using namespace rcsa;

static bool float_type(int dtype) {
  return dtype == RCSA_BF16 || dtype == RCSA_F16 || dtype == RCSA_F32;
}
static bool code_type(int code) { return code == RCSA_CODE_INT8 || code == RCSA_CODE_E4M3; }

extern "C" int rcsa_append_cache(const void* k, const void* v, int dtype, const int64_t* dims,
                                 const int64_t* strides, const int32_t* offsets,
                                 const int32_t* starts, const int32_t* lengths, void* k_codes,
                                 void* v_codes, int code, float* k_scales, float* v_scales,
                                 const int32_t* block_table, int64_t table_stride,
                                 int64_t max_pages, int64_t n_pages, int64_t page_size,
                                 int64_t block_size, hipStream_t stream) {
  if (!k || !v || !dims || !strides || !k_codes || !v_codes || !k_scales || !v_scales ||
      !block_table)
    return RCSA_ERR_NULL;
  if (offsets && lengths) return RCSA_ERR_SHAPE;
  if (!float_type(dtype) || !code_type(code)) return RCSA_ERR_DTYPE;
  int64_t each[4] = {offsets ? 1 : dims[0], dims[1], dims[2], dims[3]};
  if (dims[0] <= 0 || dims[0] >= (1 << 20) ||
      !cache_dims(each, max_pages, n_pages, page_size, block_size))
    return RCSA_ERR_SHAPE;
  if (!strides_ok(strides, 12, 8) || !strides_ok(strides + 12, 6, 1)) return RCSA_ERR_STRIDE;
  if (!aligned16(k) || !aligned16(v) || !aligned8(k_codes) || !aligned8(v_codes))
    return RCSA_ERR_ALIGN;
  AppendArgs a{};
  a.x[0] = k;
  a.x[1] = v;
  a.codes[0] = static_cast<char*>(k_codes);
  a.codes[1] = static_cast<char*>(v_codes);
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  for (int kv = 0; kv < 2; ++kv)
    for (int i = 0; i < 3; ++i) {
      a.sx[kv][i] = strides[3 * kv + i];
      a.sc[kv][i] = strides[6 + 3 * kv + i];
      a.ss[kv][i] = strides[12 + 3 * kv + i];
    }
  a.offsets = offsets;
  a.starts = starts;
  a.lengths = lengths;
  a.table = block_table;
  a.table_stride = table_stride;
  a.B = static_cast<int>(dims[0]);
  a.L = static_cast<int>(dims[1]);
  a.H = static_cast<int>(dims[2]);
  a.runs = static_cast<int>(dims[3] / 8);
  a.max_pages = static_cast<int>(max_pages);
  a.n_pages = static_cast<int>(n_pages);
  a.page = static_cast<int>(page_size);
  a.block = static_cast<int>(block_size);
  a.page_blocks = static_cast<int>(page_size / block_size);
  // blocks that L rows touch: one more than they fill where they start inside one
  a.items = offsets ? dims[1] / block_size + 2 * dims[0]
                    : (dims[1] + block_size - 2) / block_size + 1;
  a.by_heads = divisor(static_cast<uint32_t>(a.H));
  a.by_runs = divisor(static_cast<uint32_t>(a.runs));
  a.by_block = divisor(static_cast<uint32_t>(a.block));
  a.by_page_blocks = divisor(static_cast<uint32_t>(a.page_blocks));
  a.by_items = divisor(static_cast<uint32_t>(a.items));
  const bool e4m3 = code == RCSA_CODE_E4M3;
  if (dtype == RCSA_BF16) return append_type<__bf16>(a, e4m3, stream);
  if (dtype == RCSA_F16) return append_type<_Float16>(a, e4m3, stream);
  return append_type<float>(a, e4m3, stream);
}

extern "C" int rcsa_read_cache(const void* k_codes, const void* v_codes, int code,
                               const float* k_scales, const float* v_scales, void* k_out,
                               void* v_out, int dtype, const int64_t* dims,
                               const int64_t* strides, const int32_t* starts,
                               const int32_t* lengths, const int32_t* block_table,
                               int64_t table_stride, int64_t max_pages, int64_t n_pages,
                               int64_t page_size, int64_t block_size, hipStream_t stream) {
  if (!k_codes || !v_codes || !k_scales || !v_scales || !k_out || !v_out || !dims || !strides ||
      !lengths || !block_table)
    return RCSA_ERR_NULL;
  if (!float_type(dtype) || !code_type(code)) return RCSA_ERR_DTYPE;
  if (!cache_dims(dims, max_pages, n_pages, page_size, block_size)) return RCSA_ERR_SHAPE;
  if (!strides_ok(strides, 6, 8) || !strides_ok(strides + 6, 6, 1) ||
      !strides_ok(strides + 12, 6, 8))
    return RCSA_ERR_STRIDE;
  if (!aligned16(k_out) || !aligned16(v_out) || !aligned8(k_codes) || !aligned8(v_codes))
    return RCSA_ERR_ALIGN;
  ReadArgs a{};
  a.codes[0] = static_cast<const char*>(k_codes);
  a.codes[1] = static_cast<const char*>(v_codes);
  a.scales[0] = k_scales;
  a.scales[1] = v_scales;
  a.out[0] = k_out;
  a.out[1] = v_out;
  for (int kv = 0; kv < 2; ++kv)
    for (int i = 0; i < 3; ++i) {
      a.sc[kv][i] = strides[3 * kv + i];
      a.ss[kv][i] = strides[6 + 3 * kv + i];
      a.so[kv][i] = strides[12 + 3 * kv + i];
    }
  a.starts = starts;
  a.lengths = lengths;
  a.table = block_table;
  a.table_stride = table_stride;
  a.B = static_cast<int>(dims[0]);
  a.L = static_cast<int>(dims[1]);
  a.H = static_cast<int>(dims[2]);
  a.runs = static_cast<int>(dims[3] / 8);
  a.max_pages = static_cast<int>(max_pages);
  a.n_pages = static_cast<int>(n_pages);
  a.page = static_cast<int>(page_size);
  a.block = static_cast<int>(block_size);
  a.by_runs = divisor(static_cast<uint32_t>(a.runs));
  a.by_L = divisor(static_cast<uint32_t>(a.L));
  a.by_page = divisor(static_cast<uint32_t>(a.page));
  a.by_block = divisor(static_cast<uint32_t>(a.block));
  a.total = dims[0] * dims[1] * dims[2] * a.runs;
  const bool e4m3 = code == RCSA_CODE_E4M3;
  if (dtype == RCSA_BF16) return read_type<__bf16>(a, e4m3, stream);
  if (dtype == RCSA_F16) return read_type<_Float16>(a, e4m3, stream);
  return read_type<float>(a, e4m3, stream);
}
