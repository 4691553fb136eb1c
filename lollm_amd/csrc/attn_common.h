// Shared by the gated attention kernels: geometry, the argument block and small helpers.
#pragma once

#include "common.h"

namespace lollm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) void lds_void_t;
typedef __attribute__((address_space(3))) s16x4 lds_s16x4_t;
typedef int i32x2_t __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) i32x2_t lds_i32x2_t;

constexpr int AT_D = 256;            // head dim
constexpr int AT_ROWS = 32;          // MFMA rows per pair (n_rep x QB)

struct AttnArgs {
  const uint16_t* q;       // (B, T, Hq, D)
  const uint16_t* kc;      // K cache
  const uint16_t* vc;      // V cache
  const int32_t* kv_len;   // (B) keys per sequence, the T new ones included
  const uint16_t* gate;    // (B, T, Hq, D), strided, or null
  uint16_t* out;           // (B, T, Hq * D)
  float* ws;               // partials: (nw + pairs) x AT_PART, then the combine table
  long long seq_stride, head_stride;  // cache strides in elements
  int B, T, Hq, Hkv, n_rep, QB, qblocks, max_len, nw;
  float cl2;               // scale * log2(e)
  // strides of gate in elements: of a token, of a head (Hq * D and D where it is dense)
  long long gate_row;
  int gate_head;
  const uint64_t* tree;    // (B, T) or null: bit j of query i's word says that it sees new position j
};

struct PagedArgs {
  AttnArgs a;                 // kc, vc: the pools; max_len: the rows that the table can name
  const int32_t* table;       // (B, table_stride)
  const float* ks;            // (n_pages, Hkv) scales, 8-bit pages
  const float* vs;
  long long table_stride;
  int n_pages, pshift;        // page = 1 << pshift
  uint32_t rep_mul;           // ceil(2^16 / n_rep): r / n_rep = r * rep_mul >> 16 for r < 256
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float sigmoidf_(float x) { return 1.f / (1.f + __expf(-x)); }

// A pair of fp32 weights as bf16 hi and lo, x = hi + lo to 16 bits.  hi is cut and not rounded, so
// that lo is never negative, and lo is at least 2^-126 where hi is not 0: an infinite V then takes
// the sum of both products to infinity as a single product does, not to infinity - infinity or
// 0 x infinity.
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void at_split(float x, float y, uint32_t& hi, uint32_t& lo) {
  const uint32_t xb = __float_as_uint(x), yb = __float_as_uint(y);
  hi = __builtin_amdgcn_perm(yb, xb, 0x07060302u);   // the upper halves
  const bf16x2 l = {(__bf16)(x - __uint_as_float(xb & 0xffff0000u)), (__bf16)(y - __uint_as_float(yb & 0xffff0000u))};
  const u16x2 least = __builtin_elementwise_min(__builtin_bit_cast(u16x2, hi), u16x2{0x0080, 0x0080});
  lo = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, l), least));
}

// Eight e4m3 codes as bf16, times their scale (a power of two: exact).
__device__ __forceinline__ bf16x8 at_bf16(uint32_t w0, uint32_t w1, float scale) {
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false);
  const bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false);
  const bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
  return bf16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

// The weights of 8-bit pages are fp16 (at_f16), whose steps end at 2^-24: a weight far below its row's
// largest is held by that step and not by its own bits, while the row's sum counts it whole, and many
// light keys beside a heavy one (a first token that every query looks at) would be lost from the
// product alone.  So the row's reference has the weight 2^AT_F16_UP and moves where a block's maximum
// passes it by more than AT_F16_LAG in the exponent (weights end at 2^15 of fp16's 65504): a weight is
// off by at most 2^-11 of itself, or by 2^-25 / 2^AT_F16_UP of the row's largest.  What that costs is the
// moves, of all of O each (us, UP, LAG 0, 15 / 8, 7 / 10, 5 / 12, 3: 2 x 1999 tokens 182 / 184 / 185 / 190,
// 16 x 1 over 1000 .. 4000 keys 25.4 / 25.5 / 26.2 / 26.9).
constexpr float AT_F16_UP = 10.f, AT_F16_LAG = 5.f;

// Eight e4m3 codes as fp16, times a power of two of at most 2^7.  With 8-bit values the weights enter
// their product as fp16, 11 bits of them, in one product, where bf16 values (whose range fp16 lacks)
// take two of hi + lo bf16 weights.  So that no value leaves fp16's range, a tile of O counts in
// units of a scale that it has met: codes enter times their page's scale over that (448 * 2^7 is
// below 2^16), and O is rescaled where one comes that is more than 2^7 of it.  Scales are compared
// and divided as the bits of powers of two; 0 is no scale (an unmapped page).
__device__ __forceinline__ f16x8 at_f16(uint32_t w0, uint32_t w1, float ratio) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, ratio, false);
  const f16x2 b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w0, ratio, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, ratio, false);
  const f16x2 d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w1, ratio, true);
  return f16x8{a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}
__device__ __forceinline__ int at_units(int units, int a, int b) {   // for a block of these scales
  const int m = max(a, b);
  return units == 0 || m > units + (7 << 23) ? max(m, units) : units;
}
// a / b of two powers of two, or 1 where b is no scale; 2^-126 where it is less.
__device__ __forceinline__ float at_ratio(int a, int b) {
  return __int_as_float(b == 0 ? 0x3f800000 : max(a - b + 0x3f800000, 0x00800000));
}
__device__ __forceinline__ int at_scale_bits(float s) { return __float_as_int(s) & 0x7f800000; }

// Four columns of a finished row: acc / l (inv = 1 / l, 0 where no key was seen) times sigmoid(gate).
__device__ __forceinline__ void at_store4(uint16_t* out, const float (&acc)[4], float inv, bool gated, uint2 gate) {
  float y[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t g = e < 2 ? gate.x : gate.y;
    y[e] = acc[e] * inv;
    if (gated) y[e] *= sigmoidf_(__uint_as_float(e & 1 ? g & 0xffff0000u : g << 16));
  }
  const bf16x2 lo = {(__bf16)y[0], (__bf16)y[1]}, hi = {(__bf16)y[2], (__bf16)y[3]};
  *reinterpret_cast<uint2*>(out) = make_uint2(__builtin_bit_cast(uint32_t, lo), __builtin_bit_cast(uint32_t, hi));
}

// A tree of drafts: the T new positions are its nodes, and a query sees, of these, the ones whose bit
// its word has (itself and its ancestors); the cache before them it sees whole.
constexpr int AT_TREE_MAX = 64;   // nodes: bits of a word
// Which of the 32 keys from node `first` on (negative: cache before the tree) a word lets through, of
// those up to key `lim` of the 32 (negative: none); bit k for key k.
__device__ __forceinline__ uint32_t at_tree_keys(uint64_t word, int first, int lim) {
  const uint32_t w = first >= 0 ? (first < 64 ? (uint32_t)(word >> first) : 0u)
                                : (first > -32 ? (uint32_t)(word << -first) | ((1u << -first) - 1u) : ~0u);
  return lim < 0 ? 0u : w & (lim >= 31 ? ~0u : (2u << lim) - 1u);
}

constexpr int AW_WAVES = 4;
constexpr int AW_THREADS = 64 * AW_WAVES;
constexpr int AT_BLOCK = 128;        // keys per block
constexpr int AT_MAXB = 512;         // sequences per call (prefix table in LDS)
constexpr int AT_PART = 2 * AT_ROWS + AT_ROWS * AT_D;  // floats per partial

// Balanced split-K over 128-key blocks: helpers of the kernels that deal the blocks of all pairs
// out to a fixed grid of 4-wave workgroups.
__device__ __forceinline__ int seq_len(const AttnArgs& a, int b) {
  return min(max(a.kv_len[b], 0), a.max_len);  // never past the cache capacity
}

__device__ __forceinline__ int nblk_of(int L) { return (L + AT_BLOCK - 1) / AT_BLOCK; }

// First unit of workgroup w and the workgroup that owns unit u, for U units dealt
// out to nw workgroups in equal contiguous ranges: w owns [U w / nw, U (w+1) / nw).
__device__ __forceinline__ long long unit_begin(long long U, int w, int nw) {
  return U * w / nw;
}
__device__ __forceinline__ int unit_owner(long long U, long long u, int nw) {
  return (int)(((u + 1) * nw - 1) / U);
}

// pre[b] = blocks of sequences 0..b-1 (pre[0] = 0), for b = 0..B, and len[b] = the
// clamped key count of sequence b, built in LDS by the whole workgroup (so the main
// loop never waits on a global load to address the next block).  Returns pre[B].
__device__ __forceinline__ int build_prefix(const AttnArgs& a, int* pre, int* len, int* tmp) {
  constexpr int WAVES = AW_WAVES;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  int carry = 0;
  if (tid == 0) pre[0] = 0;
  for (int base = 0; base < a.B; base += AW_THREADS) {
    const int b = base + tid;
    const int Lb = b < a.B ? seq_len(a, b) : 0;
    if (b < a.B) len[b] = Lb;
    int v = nblk_of(Lb);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int o = __shfl_up(v, d, 64);
      if (lane >= d) v += o;
    }
    if (lane == 63) tmp[wave] = v;
    __syncthreads();
    int before = carry, all = carry;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) before += tmp[w];
      all += tmp[w];
    }
    if (b < a.B) pre[b + 1] = before + v;
    carry = all;
    __syncthreads();
  }
  return carry;
}

// Workgroup barrier after this wave's LDS accesses complete; the compiler sees a memory
// clobber (no LDS access moves across it) but no fence, so global loads and LDS DMA in
// flight are not drained.
__device__ __forceinline__ void aw_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// log2 of a cache page's rows (16, 32, 64 or 128), -1 for another size.
inline int attn_page_shift(int page) {
  for (int s = 4; s <= 7; ++s)
    if (page == 1 << s) return s;
  return -1;
}

// Sizes of a split-K call and its workspace; workgroups of the balanced grid (`grid` if positive,
// else one per CU of the current device), -1 where the device is not known.
int attn_geometry(int B, int T, int Hq, int Hkv, int D, int max_len, int* n_rep, int* QB, int* qblocks);
long long attn_ws_bytes(long long nw, long long pairs);
int attn_grid(int grid);

// Row groups per wave of the long-call kernel (attn_prefill.hip) for this geometry on a device
// with `cus` CUs, or 0 where the split-K kernels are the faster ones.
int attn_prefill_groups(int B, int T, int Hkv, int n_rep, int cus);
int attn_prefill_launch(const AttnArgs& a, int groups, hipStream_t st, const PagedArgs* paged = nullptr,
                        int parts = 1);
int attn_slab_tree(const AttnArgs& a, hipStream_t st);   // attn_paged.hip's kernels over slabs
// For pages: workgroups of 128-row tiles that share a CU, or 0 for the split-K kernels, and the
// workgroups that a tile's keys are dealt out to, with the bytes of workspace that takes.
int attn_paged_groups(int B, int T, int Hkv, int n_rep, int cus, bool f8, int* parts, bool tree = false);
long long attn_parts_bytes(int B, int T, int Hkv, int n_rep, int parts);

}  // namespace lollm
