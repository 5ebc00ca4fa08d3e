// The kernel for few rows (ma_cache_attend.inc) over trees of tokens.
#include "ma_cache_attend.inc"

namespace ma {

cudaError_t launch_few_tree(AttendArgs& a, int dtype, int width, int nt, int warps, long long grid, cudaStream_t stream) {
  return launch_few_of<true>(a, dtype, width, nt, warps, grid, stream);
}

}  // namespace ma
