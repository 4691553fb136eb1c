// A tree of drafted tokens (gfx950): T <= 64 nodes a sequence, a node's parent before it.  Its
// ancestors are a 64-bit word, bit j for node j, its own among them; everything that walks a tree
// goes by these words.
#include "attn_common.h"
#include "gdn_common.h"

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

// The walk of the accepted path, a wave per sequence, a lane per node: from node 0 on to the first
// child (the lowest) that is the token drawn at its parent, until there is none.
__global__ __launch_bounds__(64) void tree_accept_kernel(const int32_t* drawn, const int32_t* ids, const uint64_t* mask,
                                                         int32_t* path, int32_t* count, int32_t* next, int T) {
  const int b = blockIdx.x, i = threadIdx.x;
  const size_t at = (size_t)b * T + i;
  const uint64_t above = i < T ? mask[at] & ((1ull << i) - 1) : 0ull;
  const int parent = above ? 63 - __clzll((long long)above) : -1;
  const int id = i < T ? ids[at] : 0, want_here = i < T ? drawn[at] : 0;
  int cur = 0, n = 1, mine = i == 0 ? 0 : -1, want;
  for (;;) {
    want = __builtin_amdgcn_readlane(want_here, cur);
    const uint64_t hit = __ballot(i < T && parent == cur && id == want);
    if (!hit) break;              // (a child comes after its parent: at most T turns)
    cur = __builtin_ctzll(hit);
    if (i == n) mine = cur;
    ++n;
  }
  if (i < T) path[at] = mine;
  if (i == 0) {
    count[b] = n;
    next[b] = want;
  }
}

struct KeepArgs {
  const int32_t *path, *count;   // (B, P) nodes, increasing; (B)
  int P, T;
};

// Moves row path[i] of a sequence to row i, i < count, one 16-byte column per thread: in order, a row
// is read before it is written over (a path increases, path[i] >= i).  row(r): the address of
// row r's column, or null where there is none.
template <typename Row>
__device__ __forceinline__ void tree_keep_column(const KeepArgs& k, int b, Row row) {
  const int n = min(max(k.count[b], 0), k.P);
  for (int i = 0; i < n; ++i) {
    const int p = k.path[(size_t)b * k.P + i];
    if (p <= i || p >= k.T) continue;
    const uint4* src = row(p);
    uint4* dst = row(i);
    if (src && dst) *dst = *src;
  }
}

// K and V rows: thread 32 x + c of a workgroup column c of (sequence, KV head) x of the grid's rows.
__global__ __launch_bounds__(256) void tree_keep_kv_kernel(KeepArgs k, uint4* kc, uint4* vc, const int32_t* lengths,
                                                           const int32_t* table, long long table_stride, int width,
                                                           int n_pages, int pshift, int B, int Hkv, int max_len) {
  constexpr int COLS = AT_D * 2 / 16;
  const int x = blockIdx.x * 8 + (threadIdx.x >> 5), c = threadIdx.x & 31;
  if (x >= B * Hkv) return;
  const int b = x / Hkv, h = x - b * Hkv;
  uint4* pool = blockIdx.y ? vc : kc;
  const long long L = max(lengths[b], 0);
  tree_keep_column(k, b, [&](int r) -> uint4* {
    const long long at = L + r;
    if (!table) return at < max_len ? pool + (((long long)b * Hkv + h) * max_len + at) * COLS + c : nullptr;
    if (at >> pshift >= width) return nullptr;
    const int id = table[b * table_stride + (at >> pshift)];
    if (id < 0 || id >= n_pages) return nullptr;
    return pool + (((((long long)id * Hkv + h) << pshift) + (at & ((1 << pshift) - 1)))) * COLS + c;
  });
}

// Records (workgroups of heads' 33 columns) and window rows (of C / 8) of the half that was written.
__global__ __launch_bounds__(256) void tree_keep_gdn_kernel(KeepArgs k, uint4* rep, uint4* win, const int32_t* rec_half,
                                                            const int32_t* conv_off, int B, int Hv, int S, int W,
                                                            int cols, int Km1) {
  const int b = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
  const int records = Hv * GL_REC_U4;
  if (t < records) {
    const int h = t / GL_REC_U4, c = t - h * GL_REC_U4;
    uint4* at = rep + (((long long)b * 2 + (1 - (rec_half[b] & 1))) * Hv + h) * S * GL_REC_U4 + c;
    tree_keep_column(k, b, [&](int r) -> uint4* { return r < S ? at + (long long)r * GL_REC_U4 : nullptr; });
  } else if (t - records < cols) {
    const int base = conv_off[b] >= W ? 0 : W;
    uint4* at = win + ((long long)b * 2 * W + base + Km1) * cols + (t - records);
    tree_keep_column(k, b, [&](int r) -> uint4* { return Km1 + r < W ? at + (long long)r * cols : nullptr; });
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

LOLLM_API int lollm_tree_accept(const int32_t* drawn, const int32_t* ids, const void* mask, int32_t* path,
                                int32_t* count, int32_t* next_token, int B, int T, void* stream) {
  if (!drawn || !ids || !mask || !path || !count || !next_token || B <= 0 || T <= 0) return LOLLM_EINVAL;
  if ((uintptr_t)mask % 8) return LOLLM_EINVAL;
  if (T > TREE_MAX) return LOLLM_EUNSUPPORTED;
  hipLaunchKernelGGL(tree_accept_kernel, dim3(B), dim3(64), 0, (hipStream_t)stream, drawn, ids, (const uint64_t*)mask,
                     path, count, next_token, T);
  return launch_status();
}

LOLLM_API int lollm_tree_keep_kv(void* k, void* v, const int32_t* lengths, const int32_t* table, long long table_stride,
                                 int table_width, int n_pages, int page, const int32_t* path, const int32_t* count,
                                 int P, int B, int T, int Hkv, int D, int max_len, void* stream) {
  if (!k || !v || !lengths || !path || !count || P <= 0 || B <= 0 || T <= 0 || Hkv <= 0) return LOLLM_EINVAL;
  if (((uintptr_t)k | (uintptr_t)v) % 16) return LOLLM_EINVAL;
  if (D != AT_D || T > TREE_MAX) return LOLLM_EUNSUPPORTED;
  int pshift = 0;
  if (table) {
    if (table_width <= 0 || n_pages <= 0 || table_stride < table_width) return LOLLM_EINVAL;
    if ((pshift = attn_page_shift(page)) < 0) return LOLLM_EUNSUPPORTED;
  } else if (max_len <= 0) {
    return LOLLM_EINVAL;
  }
  if ((long long)B * Hkv > 0x7fffff00LL) return LOLLM_EUNSUPPORTED;
  const KeepArgs a = {path, count, P, T};
  hipLaunchKernelGGL(tree_keep_kv_kernel, dim3((B * Hkv + 7) / 8, 2), dim3(256), 0, (hipStream_t)stream, a, (uint4*)k,
                     (uint4*)v, lengths, table, table_stride, table_width, n_pages, pshift, B, Hkv, max_len);
  return launch_status();
}

LOLLM_API int lollm_tree_keep_gdn(void* rep, void* win, const int32_t* rec_half, const int32_t* conv_off,
                                  const int32_t* path, const int32_t* count, int P, int B, int T, int Hv, int slots,
                                  int win_rows, int conv_dim, int conv_kernel, void* stream) {
  if (!rep || !win || !rec_half || !conv_off || !path || !count || P <= 0 || B <= 0 || T <= 0 || Hv <= 0 || slots < 1)
    return LOLLM_EINVAL;
  if (((uintptr_t)rep | (uintptr_t)win) % 16 || conv_dim <= 0 || conv_dim % 8) return LOLLM_EINVAL;
  if (T > TREE_MAX || conv_kernel < 1 || conv_kernel > GL_KMAX || B > 65535) return LOLLM_EUNSUPPORTED;
  if (slots < T || win_rows < conv_kernel - 1 + T) return LOLLM_EINVAL;
  const KeepArgs a = {path, count, P, T};
  const long long cols = (long long)Hv * GL_REC_U4 + conv_dim / 8;
  if (cols > 0x3fffffff) return LOLLM_EUNSUPPORTED;
  hipLaunchKernelGGL(tree_keep_gdn_kernel, dim3((unsigned)((cols + 255) / 256), B), dim3(256), 0, (hipStream_t)stream, a,
                     (uint4*)rep, (uint4*)win, rec_half, conv_off, B, Hv, slots, win_rows, conv_dim / 8, conv_kernel - 1);
  return launch_status();
}
