// Keys and values into a paged cache in 8 bits as they are written, and back.
//
// rcsa_append_cache: for a block that gets new tokens x, with a = max |x| (of finite ones) and
// s0 the block's scale if it holds tokens before them, else 0,
//   s = max(s0, scale_for(a), 2^-100),  c = nearest(x / s),
// and, where s > s0, the codes before them c = nearest(c s0 / s).  The order of calls decides
// the result, nothing else: no atomics, one workgroup a block and head.
// rcsa_read_cache: c * s in fp32, rounded once.
//
// Both are bound by HBM, or by a launch's start and end.  An append holds a block's values in
// registers between the maximum and the codes, so that they are read once: 3520 tokens x 24 heads
// of D 128, bf16 to int8, 17.2 us for 65 MB (3.8 TB/s; with the read of the new rows 31.5, and 51
// with every value near a border divided exactly); 11 packed prompts of up to 8192 tokens x 4 heads
// of 64 in blocks of 16, fp16 to e4m3, 11.9.  64 requests' tokens 4.6 to 5.  A read of 38720 tokens
// x 24 heads of 128 takes 131 us (714 MB, 5.4 TB/s; with a place found for each run 249).
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

__device__ __forceinline__ uint32_t wave_most(uint32_t m) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint32_t other = __shfl_xor(m, o, kWave);
    m = other > m ? other : m;
  }
  return m;
}

// A workgroup takes a block's keys or values of one head (BOTH: one after the other, for
// blocks that a wavefront holds twice): one pass over them, the largest first, HELD runs of 8
// channels a thread in registers, more of them read again.
template <typename T, bool E4M3, bool PACKED, int THREADS, bool BOTH>
__global__ void __launch_bounds__(THREADS)
__attribute__((amdgpu_waves_per_eu(sizeof(T) == 2 && THREADS < 1024 ? 8 : 4, 8)))
append_kernel(AppendArgs a) {
  using C = Code8<E4M3>;
  using R = Run8<T>;
  typedef typename R::V V;
  constexpr int HELD = BOTH ? 4 : 8, KV = BOTH ? 2 : 1;
  const int tid = threadIdx.x, lane = tid & 63;
  const int id = static_cast<int>(blockIdx.x);
  const int at = divide(id, a.by_heads), head = id - at * a.H;
  const int kv0 = BOTH ? 0 : at & 1, all = BOTH ? at : at >> 1;
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

  // (the new values do not wait for the table)
  const int runs = (to - from) * a.runs;
  auto source = [&](int kv) __attribute__((always_inline)) -> const T* {
    return static_cast<const T*>(a.x[kv]) + (PACKED ? 0 : b * a.sx[kv][0]) + head * a.sx[kv][2] +
           (row0 + first + from - start) * a.sx[kv][1];
  };
  auto load = [&](int kv, const T* x, int i) __attribute__((always_inline)) -> V {
    const int row = divide(i, a.by_runs);
    return *reinterpret_cast<const V*>(x + row * a.sx[kv][1] + (i - row * a.runs) * 8);
  };
  V held[KV][HELD];
#pragma unroll
  for (int j = 0; j < KV; ++j) {
    const int kv = BOTH ? j : kv0;
    const T* const x = source(kv);
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (tid + k * THREADS < runs) held[j][k] = load(kv, x, tid + k * THREADS);
  }
  if (static_cast<uint32_t>(page) >= static_cast<uint32_t>(a.n_pages)) return;
#pragma unroll
  for (int j = 0; j < KV; ++j) {
    const int kv = BOTH ? j : kv0;
    const T* const x = source(kv);
    char* const codes = a.codes[kv] + page * a.sc[kv][0] + head * a.sc[kv][2] +
                        static_cast<int64_t>(in_page) * a.block * a.sc[kv][1];
    float* const scale = a.scales[kv] + page * a.ss[kv][0] + in_page * a.ss[kv][1] +
                         head * a.ss[kv][2];
    float s0 = 0.0f;
    if (from > 0) {
      s0 = *scale;
      s0 = s0 > 0.0f && s0 < INFINITY ? s0 : 0.0f;
    }
    uint32_t m = 0;
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (tid + k * THREADS < runs) R::most(held[j][k], m);
    for (int i = tid + HELD * THREADS; i < runs; i += THREADS) R::most(load(kv, x, i), m);
    __shared__ uint32_t s_most[2][THREADS / kWave];
    auto block_most = [&](uint32_t mine, int nth) __attribute__((always_inline)) -> uint32_t {
      uint32_t r = wave_most(mine);
      if constexpr (THREADS > kWave) {
        if (lane == 0) s_most[nth][tid / kWave] = r;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < THREADS / kWave; ++w) r = R::larger(r, s_most[nth][w]);
      }
      return r;
    };
    uint32_t bits = block_most(R::one_of(m), 0);
    const bool plain = bits < R::kInfinity;
    if (!plain) {  // the largest number beside infinities and NaN
      uint32_t f = 0;
      auto look = [&](const V& v) __attribute__((always_inline)) {
        float x8[8];
        R::floats(v, x8);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float size = fabsf(x8[e]);
          const uint32_t u = size < INFINITY ? __float_as_uint(size) : 0u;
          f = u > f ? u : f;
        }
      };
#pragma unroll
      for (int k = 0; k < HELD; ++k)
        if (tid + k * THREADS < runs) look(held[j][k]);
      for (int i = tid + HELD * THREADS; i < runs; i += THREADS) look(load(kv, x, i));
      bits = block_most(f, 1);
    }
    const float own = C::scale_for(plain ? R::value(bits) : __uint_as_float(bits));
    const float s = fmaxf(fmaxf(s0, own), kLeastScale);

    const typename C::To to_code(s);
    auto store = [&](int i, const V& v) __attribute__((always_inline)) {
      const int row = divide(i, a.by_runs);
      *reinterpret_cast<uint2*>(codes + (from + row) * a.sc[kv][1] + (i - row * a.runs) * 8) =
          to_code.template eight<R>(v, plain);
    };
#pragma unroll
    for (int k = 0; k < HELD; ++k)
      if (tid + k * THREADS < runs) store(tid + k * THREADS, held[j][k]);
    for (int i = tid + HELD * THREADS; i < runs; i += THREADS) store(i, load(kv, x, i));
    if (s != s0) {  // (a block's first scale, or a larger one)
      constexpr int U = BOTH ? 1 : 4;  // loads in flight (BOTH: values are still held)
      const int kept = from * a.runs;
      for (int i0 = tid; i0 < kept; i0 += U * THREADS) {
        uint2* p[U];
        uint2 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * THREADS;
          if (i >= kept) break;
          const int row = divide(i, a.by_runs);
          p[u] = reinterpret_cast<uint2*>(codes + row * a.sc[kv][1] + (i - row * a.runs) * 8);
          w[u] = *p[u];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i0 + u * THREADS >= kept) break;
          *p[u] = make_uint2(C::again(w[u].x, s0, s), C::again(w[u].y, s0, s));
        }
      }
      // (every thread has read the block's old scale before the barrier, or, of one
      // wavefront, before this store)
      if (tid == 0) *scale = s;
    }
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
  int tokens, groups;       // tokens of a workgroup, workgroups of a request
  int columns, side;        // runs of a token that a workgroup takes, tokens side by side
  Divisor by_runs, by_columns, by_page, by_block, by_groups;
};

constexpr int kReadTokens = 64, kReadThreads = 512;  // of a workgroup, at most

// A workgroup takes some tokens of a request, keys or values: its first threads find where the
// tokens are; then a thread goes through every `side`-th of them in one run of 8 channels, U
// at a time, so that a run's place is found once and its scale read where a block begins.
// The values pass the caches.
template <typename T, bool E4M3>
__global__ void __launch_bounds__(kReadThreads) read_kernel(ReadArgs a) {
  using C = Code8<E4M3>;
  using R = Run8<T>;
  typedef unsigned int v2i __attribute__((ext_vector_type(2)));
  constexpr int U = 4;
  __shared__ int64_t s_codes[kReadTokens], s_scale[kReadTokens];  // codes -1: no page
  const int tid = threadIdx.x, kv = static_cast<int>(blockIdx.y);
  const int b = divide(static_cast<int>(blockIdx.x), a.by_groups);
  const int t0 = (static_cast<int>(blockIdx.x) - b * a.groups) * a.tokens;
  // keys first + t, t from lo to hi - 1, are wanted and there may be some
  const int64_t first = a.starts == nullptr ? 0 : a.starts[b];
  const int64_t cap = static_cast<int64_t>(a.max_pages) * a.page;
  const int64_t len = a.lengths[b] < cap ? a.lengths[b] : cap;
  const int64_t end = len - first < a.L ? len - first : a.L;
  const int64_t from = -first > t0 ? -first : t0;
  const int64_t to = end < t0 + a.tokens ? end : t0 + a.tokens;
  if (from >= to) return;
  const int lo = static_cast<int>(from), hi = static_cast<int>(to);
  if (tid < hi - lo) {
    const int j = static_cast<int>(first + lo + tid);
    const int col = divide(j, a.by_page), slot = j - col * a.page;
    const int page = a.table[b * a.table_stride + col];
    const bool there = static_cast<uint32_t>(page) < static_cast<uint32_t>(a.n_pages);
    s_codes[tid] = there ? page * a.sc[kv][0] + slot * a.sc[kv][1] : -1;
    s_scale[tid] = page * a.ss[kv][0] + divide(slot, a.by_block) * a.ss[kv][1];
  }
  __syncthreads();
  const int beside = divide(tid, a.by_columns);
  const int c = static_cast<int>(blockIdx.z) * a.columns + tid - beside * a.columns;
  if (beside >= a.side || c >= a.runs * a.H) return;
  const int head = divide(c, a.by_runs), run = c - head * a.runs;
  const char* const codes = a.codes[kv] + head * a.sc[kv][2] + run * 8;
  const float* const scales = a.scales[kv] + head * a.ss[kv][2];
  T* const out = static_cast<T*>(a.out[kv]) + b * a.so[kv][0] + lo * a.so[kv][1] +
                 head * a.so[kv][2] + run * 8;
  const int n = hi - lo;
  int64_t had = -1;
  float s = 0.0f;
  for (int t = beside; t < n; t += U * a.side) {
    v2i w[U];
    int64_t at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tu = t + u * a.side;
      at[u] = -1;
      if (tu < n) at[u] = s_codes[tu];
      w[u] = v2i{0, 0};
      if (at[u] >= 0)
        w[u] = *reinterpret_cast<const v2i*>(codes + at[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int tu = t + u * a.side;
      if (tu >= n) break;
      if (at[u] >= 0 && s_scale[tu] != had) {
        had = s_scale[tu];
        s = scales[had];
      }
      float f[8];
      C::values(w[u][0], f);
      C::values(w[u][1], f + 4);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = at[u] >= 0 ? f[e] * s : 0.0f;
      __builtin_nontemporal_store(
          R::of(f), reinterpret_cast<typename R::V*>(out + tu * a.so[kv][1]));
    }
  }
}

constexpr int64_t kMaxThreads8 = 1ll << 32;  // a grid's dimension holds fewer

template <typename T, bool E4M3, bool PACKED>
static int launch_append(AppendArgs& a, hipStream_t s) {
  const int64_t runs = static_cast<int64_t>(a.block) * a.runs;
  const bool both = runs <= 256;
  const int64_t wgs = (PACKED ? a.items : a.items * a.B) * (both ? 1 : 2) * a.H;
  // A wavefront for small blocks; 1024 threads where large ones may get many tokens at once (5
  // tokens of 64 requests, 4 heads of D 256 in blocks of 256: 16.5 us by 1024 threads, 8.0 by 256;
  // 54 and 51 where every block's scale grows).  Packed requests: what one of them has on average
  // (the same tokens packed 15.0 by 1024 threads, 5.9 by 256; 1 of 300 requests' 65.5, 12.7; 64 of 40
  // tokens 16.0, 9.4); a longer one's blocks are gone through in rounds (one of 3000 beside 63 of
  // 5: 19.1, 28.7).
  const int64_t each = PACKED ? (a.L + a.B - 1) / a.B : a.L;
  const int64_t fresh = (each < a.block ? each : a.block) * a.runs;
  const int threads = runs <= 512 ? 64 : fresh <= 2048 ? 256 : 1024;
  if (wgs >= (1ll << 31) || wgs * threads >= kMaxThreads8) return RCSA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(wgs)), block(static_cast<unsigned>(threads));
  if (both) append_kernel<T, E4M3, PACKED, 64, true><<<grid, block, 0, s>>>(a);
  else if (threads == 64) append_kernel<T, E4M3, PACKED, 64, false><<<grid, block, 0, s>>>(a);
  else if (threads == 256) append_kernel<T, E4M3, PACKED, 256, false><<<grid, block, 0, s>>>(a);
  else append_kernel<T, E4M3, PACKED, 1024, false><<<grid, block, 0, s>>>(a);
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
  // a token's runs on whole wavefronts, tokens side by side where they are few
  const int64_t per = static_cast<int64_t>(a.runs) * a.H;
  const int64_t passes = (per + kReadThreads - 1) / kReadThreads;
  const int64_t columns = (per + passes - 1) / passes;
  const int64_t side = columns >= 256 ? 1 : (256 / columns < kReadTokens ? 256 / columns
                                                                         : kReadTokens);
  const int64_t threads = (columns * side + kWave - 1) / kWave * kWave;
  // eight tokens a thread, fewer where that leaves compute units without a workgroup
  int64_t nt = side * 8 < kReadTokens ? side * 8 : kReadTokens;
  while (nt > side && static_cast<int64_t>(a.B) * ((a.L + nt - 1) / nt) * passes * 2 < 1024)
    nt = (nt / 2 + side - 1) / side * side;
  nt = nt < threads ? nt : threads;
  a.columns = static_cast<int>(columns);
  a.side = static_cast<int>(side);
  a.tokens = static_cast<int>(nt);
  a.groups = static_cast<int>((a.L + nt - 1) / nt);
  a.by_groups = divisor(static_cast<uint32_t>(a.groups));
  a.by_columns = divisor(static_cast<uint32_t>(columns));
  const int64_t wgs = static_cast<int64_t>(a.groups) * a.B;
  if (wgs * threads >= kMaxThreads8) return RCSA_ERR_SHAPE;
  const dim3 grid(static_cast<unsigned>(wgs), 2, static_cast<unsigned>(passes));
  const dim3 block(static_cast<unsigned>(threads));
  if (e4m3) read_kernel<T, true><<<grid, block, 0, s>>>(a);
  else read_kernel<T, false><<<grid, block, 0, s>>>(a);
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

// Strides of rows (elements), a multiple of `unit`, and pointers of rows of codes.
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
// Elements of 16 bytes.
static int64_t row_unit(int dtype) { return dtype == RCSA_F32 ? 4 : 8; }
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
  if (!strides_ok(strides, 6, row_unit(dtype)) || !strides_ok(strides + 6, 6, 8) ||
      !strides_ok(strides + 12, 6, 1))
    return RCSA_ERR_STRIDE;
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
      !strides_ok(strides + 12, 6, row_unit(dtype)))
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
  a.by_page = divisor(static_cast<uint32_t>(a.page));
  a.by_block = divisor(static_cast<uint32_t>(a.block));
  const bool e4m3 = code == RCSA_CODE_E4M3;
  if (dtype == RCSA_BF16) return read_type<__bf16>(a, e4m3, stream);
  if (dtype == RCSA_F16) return read_type<_Float16>(a, e4m3, stream);
  return read_type<float>(a, e4m3, stream);
}
