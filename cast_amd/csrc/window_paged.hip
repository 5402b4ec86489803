// Windowed attention over pages, blocks of 128 rows: a source of its own for the
// memory-clause scheduler, the only one that fits D 128 into 168 VGPRs without spills (the
// dense form, built for instruction-level parallelism, is 1 to 3% slower under it).
#include "window_tile.h"

namespace rcsa {

template <typename T, int D>
static void launch(WindowArgs& a, dim3 grid, hipStream_t s) {
  window_kernel<T, D, kPaged><<<grid, dim3(256), 0, s>>>(a);
}

void launch_window_paged(WindowArgs& a, int type, int64_t D, dim3 grid, hipStream_t s) {
  if (type == 0) D == 128 ? launch<__bf16, 128>(a, grid, s) : launch<__bf16, 64>(a, grid, s);
  else D == 128 ? launch<_Float16, 128>(a, grid, s) : launch<_Float16, 64>(a, grid, s);
}

}  // namespace rcsa
