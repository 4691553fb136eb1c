// A tree of drafted tokens (gfx950): T <= 64 nodes a sequence, a node's parent before it.  Its
// ancestors are a 64-bit word, bit j for node j, its own among them; everything that walks a tree
// goes by these words.
#include "common.h"

namespace lollm {

constexpr int TREE_MAX = 64;

// A wave per sequence, a lane per node: ancestors by pointer doubling, 6 rounds.
__global__ __launch_bounds__(64) void tree_masks_kernel(const int32_t* parents, uint64_t* mask, int32_t* depth, int T) {
  const int b = blockIdx.x, i = threadIdx.x;
  int p = i < T ? parents[(size_t)b * T + i] : -1;
  p = p >= 0 && p < i ? p : -1;   // anything else hangs on the committed context
  uint64_t w = 1ull << i;
  for (int r = 0; r < 6; ++r) {
    const int at = p < 0 ? i : p;
    const uint32_t lo = __shfl((uint32_t)w, at, 64), hi = __shfl((uint32_t)(w >> 32), at, 64);
    const int up = __shfl(p, at, 64);
    if (p >= 0) {
      w |= (uint64_t)hi << 32 | lo;
      p = up;
    }
  }
  if (i < T) {
    mask[(size_t)b * T + i] = w;
    if (depth) depth[(size_t)b * T + i] = __popcll(w) - 1;
  }
}

}  // namespace lollm

using namespace lollm;

LOLLM_API int lollm_tree_masks(const int32_t* parents, void* mask, int32_t* depth, int B, int T, void* stream) {
  if (!parents || !mask || B <= 0 || T <= 0) return LOLLM_EINVAL;
  if ((uintptr_t)mask % 8) return LOLLM_EINVAL;
  if (T > TREE_MAX) return LOLLM_EUNSUPPORTED;
  hipLaunchKernelGGL(tree_masks_kernel, dim3(B), dim3(64), 0, (hipStream_t)stream, parents, (uint64_t*)mask, depth, T);
  return launch_status();
}
