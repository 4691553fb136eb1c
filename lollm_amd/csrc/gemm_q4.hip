// Products with 4-bit weights and group scales (gfx950): y[m, n] = sum_g s[n, g] sum_{k in g}
// x[m, k] (c[n, k] - z[n, g]), x and y bf16, c 4-bit codes, s bf16, z 8 where none is given; groups
// of 32, 64 or 128 k.  SwiGLU, silu(gate) up of the interleaved halves, in fp32, rounded once.
//
// Arithmetic.  A code q becomes the bf16 number 16 + q, exactly, with a rotation and an and-or for two
// codes (its bits are the upper mantissa bits of 16).  The products run over these; what 16 + z adds to
// every code is taken off through the accumulator: a group's chain of products starts from
// -(16 + z) sum_k x, the sum itself one more product with a constant operand that all columns of a row
// tile share (many rows: after the loop, by a product over the groups).  The group's scale then meets an
// fp32 sum, so weights are never rounded.  What the detour costs: partial sums of at most 32 sum |x| in
// fp32, 2^-24 of that against a group's typical 52 |x| is 1e-5 of it, below a bf16 output's 2^-9.  An
// x that is infinite, or so large (2^116) that these sums are, makes its row NaN.
//
// Layout (lollm_q4_pack, once per weight).  1 KB blocks of 16 rows x 128 k in operand order: lane
// 16 g + r holds row r's codes of k 32 j + 8 g .. + 8 in word j, even k in the low half and odd k in
// the high half, the word rotated left by 3, so that the first pair lies at the mantissa's place.  Then
// the scales, per block [lane group g][group][rows 4 g ..], as the accumulator holds rows, and the zeros
// in the same order.
#include <type_traits>

#include "common.h"

namespace lollm {

typedef __bf16 q4_bf16x8 __attribute__((ext_vector_type(8)));
typedef float q4_f32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int q4_u32x2 __attribute__((ext_vector_type(2)));

constexpr int Q4_STAGE = 128;       // k per block
constexpr int Q4_WAVES = 8;
constexpr int Q4_THREADS = 64 * Q4_WAVES;

struct Q4Args {
  const uint16_t* x;        // (M, K), row stride ldx
  const uint8_t* codes;     // packed
  const uint16_t* scale;
  const uint8_t* zero;      // or null: 8
  uint16_t* y;              // (M, oc), row stride ldy
  long long ldx, ldy;
  int M, N, K;
  uint16_t* sums;           // many rows: (3, M, groups padded to 32) bf16 parts of the groups' sums of x
};

// Eight codes, the k-th pair of them at bits 3 + 4 k of both halves once the word is rotated by 4 k: three
// rotations and four and-ors (whose constants are in registers: two literals do not fit the instruction).
struct Q4Const {
  uint32_t mask = 0x00780078u, base = 0x41804180u;
  __device__ __forceinline__ Q4Const() {
    asm("" : "+s"(mask));
    asm("" : "+v"(base));
  }
};
__device__ __forceinline__ q4_bf16x8 q4_frag(uint32_t w, const Q4Const& k) {
  const u32x4_t r = {(w & k.mask) | k.base, (__builtin_amdgcn_alignbit(w, w, 4) & k.mask) | k.base,
                     (__builtin_amdgcn_alignbit(w, w, 8) & k.mask) | k.base,
                     (__builtin_amdgcn_alignbit(w, w, 12) & k.mask) | k.base};
  return __builtin_bit_cast(q4_bf16x8, r);
}

__device__ __forceinline__ float q4_silu(float g) { return g / (1.f + __expf(-g)); }

__device__ __forceinline__ uint32_t q4_pack2(float a, float b) {
  return (uint32_t)f32_to_bf16(a) | ((uint32_t)f32_to_bf16(b) << 16);
}

// One output tile (16 columns x 16 rows; lane: row l16, columns 4 g4 ..): SwiGLU tiles hold 8 gate
// rows of the weight, then their 8 up rows, in lanes 32 apart.
template <bool SWIGLU>
__device__ __forceinline__ void q4_emit(const Q4Args& a, q4_f32x4 v, int t, int m, int g4) {
  if constexpr (SWIGLU) {
    float u[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __shfl_xor(v[e], 32, 64);
    if (g4 < 2 && m < a.M)
      *reinterpret_cast<uint2*>(a.y + (size_t)m * a.ldy + 8 * t + 4 * g4) =
          make_uint2(q4_pack2(q4_silu(v[0]) * u[0], q4_silu(v[1]) * u[1]),
                     q4_pack2(q4_silu(v[2]) * u[2], q4_silu(v[3]) * u[3]));
  } else if (m < a.M) {
    *reinterpret_cast<uint2*>(a.y + (size_t)m * a.ldy + 16 * t + 4 * g4) =
        make_uint2(q4_pack2(v[0], v[1]), q4_pack2(v[2], v[3]));
  }
}

// The weights of a stage for NT column tiles: codes, and of each group the scales (and zeros) of the
// lane's four rows.
template <int NT, int GPS>
struct Q4Weights {
  u32x4_t w[NT];
  q4_u32x2 s[NT][GPS];
  uint32_t z[NT][GPS];
};

// The blocks of column tiles t0 .. t0 + NT - 1: descriptors, so that a load's address is the lane's own
// offset and a scalar.
template <int NT, int GPS, bool ZERO>
struct Q4Source {
  __amdgpu_buffer_rsrc_t codes, scale, zero;
  int SK, vc, vs;
  __device__ __forceinline__ Q4Source(const Q4Args& a, int t0, int lane) {
    SK = a.K / Q4_STAGE;
    const size_t first = (size_t)t0 * SK;
    const uint32_t blocks = (uint32_t)(min(NT, a.N / 16 - t0) * SK);   // (a block's place is a scalar: none past these is asked for)
    codes = buf_rsrc(a.codes + first * 1024, blocks * 1024);
    scale = buf_rsrc(a.scale + first * (16 * GPS), blocks * (32 * GPS));
    zero = buf_rsrc(ZERO ? a.zero + first * (16 * GPS) : nullptr, ZERO ? blocks * (16 * GPS) : 0);
    vc = 16 * lane;
    vs = (lane >> 4) * GPS * 8;
  }
  // block blk of these tiles' into place j
  template <typename Weights>
  __device__ __forceinline__ void block(Weights& d, int j, int blk) const {
    d.w[j] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(codes, vc, blk * 1024, 2));
    if constexpr (GPS == 1) {
      d.s[j][0] = __builtin_bit_cast(q4_u32x2, __builtin_amdgcn_raw_buffer_load_b64(scale, vs, blk * 32, 0));
      if (ZERO) d.z[j][0] = __builtin_amdgcn_raw_buffer_load_b32(zero, vs / 2, blk * 16, 0);
    } else {
#pragma unroll
      for (int g = 0; g < GPS; g += 2) {
        const u32x4_t t = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(scale, vs + 8 * g, blk * (32 * GPS), 0));
        d.s[j][g] = {t.x, t.y};
        d.s[j][g + 1] = {t.z, t.w};
      }
      if constexpr (ZERO && GPS == 2) {
        const q4_u32x2 t = __builtin_bit_cast(q4_u32x2, __builtin_amdgcn_raw_buffer_load_b64(zero, vs / 2, blk * 32, 0));
        d.z[j][0] = t.x;
        d.z[j][1] = t.y;
      } else if constexpr (ZERO) {
        const u32x4_t t = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(zero, vs / 2, blk * 64, 0));
#pragma unroll
        for (int g = 0; g < 4; ++g) d.z[j][g] = t[g];
      }
    }
  }
  __device__ __forceinline__ void tile(Q4Weights<NT, GPS>& d, int j, int s) const { block(d, j, j * SK + s); }
  static constexpr int LOADS = 1 + (GPS == 4 ? 2 : 1) + (ZERO ? 1 : 0);   // instructions of a tile
  __device__ __forceinline__ void load(Q4Weights<NT, GPS>& d, int s) const {
#pragma unroll
    for (int j = 0; j < NT; ++j) tile(d, j, s);
  }
};

// tot += a stage's products: x holds the row tiles' operands of its four k-steps.  refill(j): tile j's
// weights are used.
template <int MT, int NT, int GPS, bool ZERO, typename Refill>
__device__ __forceinline__ void q4_stage(q4_f32x4 (&tot)[NT][MT], const Q4Weights<NT, GPS>& d, const u32x4_t (&x)[MT][4],
                                         Refill refill) {
  constexpr int KPG = 4 / GPS;      // k-steps per group
  // the constant operand: -(16 + 8), or 1 where columns have zeros of their own
  constexpr uint32_t CONST = ZERO ? 0x3f803f80u : 0xc1c0c1c0u;
  const q4_bf16x8 ones = __builtin_bit_cast(q4_bf16x8, u32x4_t{CONST, CONST, CONST, CONST});
  const Q4Const kc;
  // One tile of one group after the other: while its products run, the next one's codes are decoded and
  // the last one's sums scaled.
  float c0[MT];   // (its four are equal)
  q4_f32x4 c[2][MT];
  q4_bf16x8 w[2][KPG];
#pragma unroll
  for (int q = 0; q < KPG; ++q) w[0][q] = q4_frag(d.w[0][q], kc);
  auto scale = [&](int step) {
    const int g = step / NT, j = step % NT;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t b = d.s[j][g][e >> 1];
      const float sc = __uint_as_float(e & 1 ? b & 0xffff0000u : b << 16);
#pragma unroll
      for (int i = 0; i < MT; ++i) tot[j][i][e] = fmaf(sc, c[step & 1][i][e], tot[j][i][e]);
    }
    if (g == GPS - 1) refill(j);
  };
#pragma unroll
  for (int step = 0; step < GPS * NT; ++step) {
    const int g = step / NT, j = step % NT;
    if (j == 0) {
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        q4_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < KPG; ++q)
          v = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(q4_bf16x8, x[i][g * KPG + q]), v, 0, 0, 0);
        c0[i] = v[0];
      }
      if (MT > 1) __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float zc = ZERO ? -16.f - (float)((d.z[j][g] >> (8 * e)) & 0xffu) : 1.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) c[step & 1][i][e] = ZERO ? c0[i] * zc : c0[i];
    }
    const int gn = (step + 1) / NT, jn = (step + 1) % NT;
    if (step + 1 < GPS * NT)
#pragma unroll
      for (int q = 0; q < KPG; ++q) w[(step + 1) & 1][q] = q4_frag(d.w[jn][gn * KPG + q], kc);
#pragma unroll
    for (int q = 0; q < KPG; ++q)
#pragma unroll
      for (int i = 0; i < MT; ++i)
        c[step & 1][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            w[step & 1][q], __builtin_bit_cast(q4_bf16x8, x[i][g * KPG + q]), c[step & 1][i], 0, 0, 0);
    if (step) scale(step - 1);
    if (MT > 1) {
#pragma unroll
      for (int m = 0; m < KPG * MT; ++m) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);    // a product,
        __builtin_amdgcn_sched_group_barrier(0x2, 3, 0);    // three VALU instructions
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  scale(GPS * NT - 1);
}

// The first row of row tile i where m rows are left: the last tile ends with the last row, and computes what
// the one before has (the same bits) rather than read past the end.
__device__ __forceinline__ int q4_row_tile(int i, int m) { return min(16 * i, max(m - 16, 0)); }

// A workgroup's sums, ((w0 + w4) + (w1 + w5)) + ..: waves 4 .. 7 hand theirs to 0 .. 3, through `red`.
template <int MT, int NT, bool SWIGLU>
__device__ __forceinline__ void q4_finish(const Q4Args& a, const q4_f32x4 (&tot)[NT][MT], q4_f32x4 (*red)[NT * MT][64],
                                          int t0, int m0, int wave, int lane, int nt = NT) {
  if (wave >= Q4_WAVES / 2)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) red[wave - Q4_WAVES / 2][j * MT + i][lane] = tot[j][i];
  __syncthreads();
  if (wave < Q4_WAVES / 2)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int i = 0; i < MT; ++i) red[wave][j * MT + i][lane] = tot[j][i] + red[wave][j * MT + i][lane];
  __syncthreads();
  for (int k = wave; k < nt * MT; k += Q4_WAVES) {
    q4_f32x4 v = red[0][k][lane];
#pragma unroll
    for (int w = 1; w < Q4_WAVES / 2; ++w) v += red[w][k][lane];
    q4_emit<SWIGLU>(a, v, t0 + k / MT, m0 + q4_row_tile(k % MT, a.M - m0) + (lane & 15), lane >> 4);
  }
}

// At most 16 rows, a column tile a workgroup: its eight waves deal out the stages of K (wave w: w, w + 8, ..),
// operands straight to registers, two stages ahead; the waves' sums meet in LDS in a fixed order at the end.
// All few-row kernels share these sums' order, so that a row's bits do not depend on the number of rows.
// (Eight stages ahead cost 8% more: the code is longer, and every launch starts with it out of the cache.)
// 1 x 4096 x 12288 at groups of 64: 9.7 us, 2.6 TB/s of codes; 16 rows 15.4 us, where every workgroup fetches all of x,
// four times the weights in all, from L2.
template <int GPS, bool ZERO, bool SWIGLU>
__global__ __launch_bounds__(Q4_THREADS) void gemm_q4_kernel(Q4Args a) {
  constexpr int P = 2;
  __shared__ __attribute__((aligned(16))) q4_f32x4 red[Q4_WAVES / 2][1][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int SK = a.K / Q4_STAGE;
  const int n = SK > wave ? (SK - wave + Q4_WAVES - 1) / Q4_WAVES : 0;

  const Q4Source<1, GPS, ZERO> src(a, blockIdx.x, lane);
  const uint16_t* xr = a.x + (size_t)min(l16, a.M - 1) * a.ldx + 8 * g4;
  struct Stage : Q4Weights<1, GPS> {
    u32x4_t x[1][4];
  };
  Stage st[P];
  auto load = [&](Stage& d, int i) {
    const int s = wave + Q4_WAVES * i;
    src.load(d, s);
#pragma unroll
    for (int q = 0; q < 4; ++q) d.x[0][q] = *reinterpret_cast<const u32x4_t*>(xr + s * Q4_STAGE + 32 * q);
  };

  q4_f32x4 tot[1][1] = {{q4_f32x4{0.f, 0.f, 0.f, 0.f}}};
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (p < n) load(st[p], p);
  for (int i = 0; i < n; i += P) {
#pragma unroll
    for (int p = 0; p < P; ++p) {
      if (i + p < n) q4_stage<1, 1, GPS, ZERO>(tot, st[p], st[p].x, [](int) {});
      if (i + p + P < n) load(st[p], i + p + P);
    }
  }
  q4_finish<1, 1, SWIGLU>(a, tot, red, blockIdx.x, 0, wave, lane);
}

// At most 16 rows and several column tiles a workgroup: the rows' operands of a few stages stay in
// registers while the weights of one column tile after the other stream past them, two tiles ahead.
// (Fetched again for every tile, as above, they and their sums cost more than the weights.)
// 1 x 24576 x 4096 with SwiGLU and zeros, groups of 128: 15.5 us, 3.3 TB/s; 16 rows 18 us; 1 x 151936 x 4096
// 78 us, 4.0 TB/s.
template <int NT, int GPS, bool ZERO, bool SWIGLU>
__global__ __launch_bounds__(Q4_THREADS) void gemm_q4_wide_kernel(Q4Args a) {
  constexpr int KPG = 4 / GPS, HELD = GPS == 4 ? 2 : 4;   // (stages held)
  static_assert(NT % 2 == 0, "the weights' buffers alternate");
  __shared__ __attribute__((aligned(16))) q4_f32x4 red[Q4_WAVES / 2][NT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int t0 = blockIdx.x * NT, nt = min(NT, a.N / 16 - t0);
  const int SK = a.K / Q4_STAGE;
  const int n = SK > wave ? (SK - wave + Q4_WAVES - 1) / Q4_WAVES : 0;
  const Q4Source<NT, GPS, ZERO> src(a, t0, lane);
  const uint16_t* xr = a.x + (size_t)min(l16, a.M - 1) * a.ldx + 8 * g4;
  constexpr uint32_t CONST = ZERO ? 0x3f803f80u : 0xc1c0c1c0u;
  const q4_bf16x8 ones = __builtin_bit_cast(q4_bf16x8, u32x4_t{CONST, CONST, CONST, CONST});
  const Q4Const kc;
  q4_f32x4 tot[NT];
#pragma unroll
  for (int j = 0; j < NT; ++j) tot[j] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
  Q4Weights<HELD, GPS> st[2];   // (of a tile's HELD stages)
  auto load = [&](Q4Weights<HELD, GPS>& d, int c, int j) {   // (past the last tile or stage: nothing)
#pragma unroll
    for (int h = 0; h < HELD; ++h)
      if (j < nt && c + h < n) src.block(d, h, j * SK + wave + Q4_WAVES * (c + h));
  };
  if (n > 0) {
    load(st[0], 0, 0);
    load(st[1], 0, 1);
  }
  u32x4_t x[HELD][4];
  float c0[HELD][GPS];
  // column tile j with COUNT of the held stages: their chains of products side by side
  auto tile = [&](const Q4Weights<HELD, GPS>& d, int j, auto count) {
    constexpr int COUNT = decltype(count)::value;
    q4_f32x4 v[COUNT][GPS];
#pragma unroll
    for (int h = 0; h < COUNT; ++h)
#pragma unroll
      for (int g = 0; g < GPS; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[h][g][e] = ZERO ? c0[h][g] * (-16.f - (float)((d.z[h][g] >> (8 * e)) & 0xffu)) : c0[h][g];
#pragma unroll
    for (int q = 0; q < KPG; ++q)
#pragma unroll
      for (int h = 0; h < COUNT; ++h)
#pragma unroll
        for (int g = 0; g < GPS; ++g)
          v[h][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(q4_frag(d.w[h][g * KPG + q], kc),
                                                            __builtin_bit_cast(q4_bf16x8, x[h][g * KPG + q]), v[h][g], 0, 0, 0);
#pragma unroll
    for (int h = 0; h < COUNT; ++h)   // (a stage's groups, then the next one's: the order of all few-row kernels)
#pragma unroll
      for (int g = 0; g < GPS; ++g)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b = d.s[h][g][e >> 1];
          tot[j][e] = fmaf(__uint_as_float(e & 1 ? b & 0xffff0000u : b << 16), v[h][g][e], tot[j][e]);
        }
  };
  for (int c = 0; c < n; c += HELD) {
#pragma unroll
    for (int h = 0; h < HELD; ++h) {
      const int s = wave + Q4_WAVES * min(c + h, n - 1);
#pragma unroll
      for (int q = 0; q < 4; ++q) x[h][q] = *reinterpret_cast<const u32x4_t*>(xr + s * Q4_STAGE + 32 * q);
    }
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      q4_f32x4 v[HELD];
#pragma unroll
      for (int q = 0; q < KPG; ++q)
#pragma unroll
        for (int h = 0; h < HELD; ++h)
          v[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(q4_bf16x8, x[h][g * KPG + q]),
                                                         q ? v[h] : q4_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
      for (int h = 0; h < HELD; ++h) c0[h][g] = v[h][0];
    }
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      Q4Weights<HELD, GPS>& d = st[j & 1];
      if (c + HELD <= n) {
        tile(d, j, std::integral_constant<int, HELD>{});
      } else {
        // (stages in turn, as in a whole set: a row's bits do not tell them apart)
        const int left = n - c;
        if (left == 1) tile(d, j, std::integral_constant<int, 1>{});
        if (HELD > 2 && left == 2) tile(d, j, std::integral_constant<int, (HELD > 2 ? 2 : 1)>{});
        if (HELD > 2 && left == 3) tile(d, j, std::integral_constant<int, (HELD > 2 ? 3 : 1)>{});
      }
      // the step after next: tile j + 2 of these stages, or j + 2 - NT of the next ones
      if (j + 2 < NT) load(d, c, j + 2);
      else load(d, c + HELD, j + 2 - NT);
    }
  }
  q4_f32x4 t1[NT][1];
#pragma unroll
  for (int j = 0; j < NT; ++j) t1[j][0] = tot[j];
  q4_finish<1, NT, SWIGLU>(a, t1, red, t0, 0, wave, lane, nt);
}

// 17 .. 64 rows a tile (MT 2 or 4): the same division of K, but a wave's rows of a stage come by LDS DMA,
// whole 256-byte lines of four rows an instruction, into a buffer of its own (the 16-byte chunk c of row r
// at c ^ (r & 15)), and from there as operands: read in the operand's order from memory, 64 bytes of
// 16 rows at a time, they cost twice as much.  All of a stage's operands lie in registers before its
// products, so the next stage's rows are on their way into the same buffer meanwhile.
// 61 x 12352 x 4096 with zeros, groups of 128: 19 us, 1.3 TB/s, 316 TF: bound by the rows' way from L2 to LDS,
// once for each 64 columns (without it two thirds of the time remain), and by products behind their decoding.
// Four column tiles of 64 rows with zeros spill 6 registers (2.4 MB written for these 61 rows).
typedef __attribute__((address_space(3))) void q4_lds_t;

template <int MT, int NT, int P, int GPS, bool ZERO, bool SWIGLU>
__global__ __launch_bounds__(Q4_THREADS) void gemm_q4_lds_kernel(Q4Args a) {
  constexpr int TILE = 16 * MT * 256;           // bytes of a wave's rows of a stage
  constexpr int RED = Q4_WAVES / 2 * NT * MT * 1024;
  constexpr int BYTES = Q4_WAVES * TILE > RED ? Q4_WAVES * TILE : RED;
  __shared__ __attribute__((aligned(1024))) unsigned char lds[BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int t0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
  const int SK = a.K / Q4_STAGE;
  const int n = SK > wave ? (SK - wave + Q4_WAVES - 1) / Q4_WAVES : 0;
  unsigned char* buf = lds + wave * TILE;

  const int m = a.M - m0;   // rows from here on
  const uint32_t pitch = (uint32_t)(2 * a.ldx);
  const __amdgpu_buffer_rsrc_t rows =
      buf_rsrc(a.x + (size_t)m0 * a.ldx, (uint32_t)(min(16 * MT, m) - 1) * pitch + (uint32_t)(2 * a.K));
  uint32_t vx[4];   // rows 4 d + g4 of 16, their chunks swizzled
#pragma unroll
  for (int d = 0; d < 4; ++d) vx[d] = min(4 * d + g4, m - 1) * pitch + 16 * (l16 ^ (4 * d + g4));
  auto issue_x = [&](int i) {
    const uint32_t k0 = (uint32_t)(wave + Q4_WAVES * i) * (2 * Q4_STAGE);
#pragma unroll
    for (int d = 0; d < 4 * MT; ++d)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (q4_lds_t*)(buf + 1024 * d), 16, vx[d & 3],
                                               q4_row_tile(d >> 2, m) * pitch + k0, 0, 0);
  };
  const Q4Source<NT, GPS, ZERO> src(a, t0, lane);
  Q4Weights<NT, GPS> st[P];
  q4_f32x4 tot[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) tot[j][i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};

  constexpr int NW = NT * Q4Source<NT, GPS, ZERO>::LOADS;   // loads of a stage's weights
  if (n > 0) {
    issue_x(0);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p < n) src.load(st[p], wave + Q4_WAVES * p);
    for (int i = 0; i < n; i += P) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (i + p >= n) break;
        // this stage's rows have landed: after them the weights of a later stage were asked for, if there is one
        if (i + p == 0 ? n >= P : i + p - 1 + P < n) {
          if (p == 0 && i == 0) asm volatile("s_waitcnt vmcnt(%0)" ::"n"((P * NW < 63 ? P * NW : 63)) : "memory");
          else asm volatile("s_waitcnt vmcnt(%0)" ::"n"(NW) : "memory");
        } else {
          asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        u32x4_t x[MT][4];
#pragma unroll
        for (int i2 = 0; i2 < MT; ++i2)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            x[i2][q] = *reinterpret_cast<const u32x4_t*>(buf + (16 * i2 + l16) * 256 + (((4 * q + g4) ^ l16) * 16));
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // before the buffer is filled again
        if (i + p + 1 < n) issue_x(i + p + 1);
        __builtin_amdgcn_sched_barrier(0);
        q4_stage<MT, NT, GPS, ZERO>(tot, st[p], x, [&](int j) {
          if (i + p + P < n) src.tile(st[p], j, wave + Q4_WAVES * (i + p + P));
        });
      }
    }
  }
  __syncthreads();   // every wave is done with the buffers
  q4_finish<MT, NT, SWIGLU>(a, tot, reinterpret_cast<q4_f32x4(*)[NT * MT][64]>(lds), t0, m0, wave, lane);
}

// ---- many rows ----
// A workgroup of eight waves, 2 x 4, owns 128 rows x 256 columns, a wave 64 x 64 of them; K goes by in its
// stages of 128 through three LDS slots, rows and codes, filled by DMA two stages ahead, one barrier a
// stage.  What 16 + z adds is here taken off at the end, by a product over the groups: sum_g s (16 + z)
// times the group's sum of x, which a first kernel has formed (each as three bf16 numbers, 24 bits, so
// that nothing is lost; s (16 + z) has 13 bits and needs two).  In the loop that leaves the decoding
// (7 instructions for 8 codes), the products and, a group's end, its scale: 192 VALU instructions a stage
// beside 64 products of 16 cycles.
// 1999 x 18432 x 4096, groups of 128: 300 to 316 us by the card, 955 to 1000 TF (64: 379, 32: 454), 63% of what a bf16 product of 8192^3
// reaches here.  The decoding is what is left: it and the products of two waves share a SIMD's issue.
// (Groups of 64 spill 5 or 6 registers.)
constexpr int QR_BM = 128, QR_BN = 256;
constexpr int QR_CODES = QR_BM * 256, QR_SCALES = QR_CODES + QR_BN * 64;   // a slot: rows, codes, scales

// 16 bytes a lane from a buffer to 1 KB of LDS at `to`, without the compiler's knowledge: it cannot tell slots
// apart for long, and then waits for all DMA before it reads any slot.  Waits and barriers are written out.
__device__ __forceinline__ void q4_dma(uint32_t to, uint32_t voff, u32x4_t rsrc, uint32_t soff) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds"
               ::"s"(to), "v"(voff), "s"(rsrc), "s"(soff) : "memory");
}
__device__ __forceinline__ u32x4_t q4_rsrc(const void* base, uint32_t bytes) {
  const uint64_t p = (uint64_t)base;
  return u32x4_t{(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)p),
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(p >> 32)) & 0xffffu,
                 (uint32_t)__builtin_amdgcn_readfirstlane((int)bytes), 0x00020000u};
}

__global__ __launch_bounds__(256) void q4_sums_kernel(const uint16_t* __restrict__ x, long long ldx, uint16_t* sums, int M,
                                                      int groups, int padded, int G, float factor) {
  const long long id = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);   // 16 threads a (row, group)
  const int l = threadIdx.x & 15;
  const int m = (int)(id / padded), g = (int)(id % padded);
  if (m >= M) return;
  float v = 0.f;
  if (g < groups) {
    const uint16_t* p = x + (size_t)m * ldx + (size_t)g * G + l * (G / 16);
    u32x4_t w = {0, 0, 0, 0};   // the thread's 8, 4 or 2 values
    if (G == 128) w = *reinterpret_cast<const u32x4_t*>(p);
    else if (G == 64) { const uint2 t = *reinterpret_cast<const uint2*>(p); w.x = t.x; w.y = t.y; }
    else w.x = *reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int i = 0; i < 4; ++i) v += __uint_as_float(w[i] << 16) + __uint_as_float(w[i] & 0xffff0000u);
  }
  v = sum_lanes16(v) * factor;
  if (l < 3) {
    const float hi = round_bf16(v), mid = round_bf16(v - hi);
    sums[(size_t)l * M * padded + id] = f32_to_bf16(l == 0 ? hi : (l == 1 ? mid : v - hi - mid));
  }
}

template <int GPS, bool ZERO, bool SWIGLU>
__global__ __launch_bounds__(512, 1) void gemm_q4_rows_kernel(Q4Args a) {
  constexpr int KPG = 4 / GPS;
  constexpr int SLOT = QR_SCALES + 1024 * (GPS == 4 ? 2 : 1);
  __shared__ __attribute__((aligned(1024))) unsigned char lds[3 * SLOT];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int wm = wave & 1, wn = wave >> 1;
  const int n = a.K / Q4_STAGE;
  const int mt = (a.M + QR_BM - 1) / QR_BM, nt = (a.N + QR_BN - 1) / QR_BN;
  // an XCD (workgroups i, i + 8, ..) takes a contiguous run of the tiles, in bands of 8 row tiles
  int m0, t0;
  {
    const int ntiles = mt * nt, v = blockIdx.x, xcd = v & 7;
    const int u = xcd * (ntiles / 8) + min(xcd, ntiles % 8) + (v >> 3);
    const int band = u / (8 * nt), r = u - band * 8 * nt, hb = min(8, mt - 8 * band);
    m0 = (8 * band + r % hb) * QR_BM;
    t0 = (r / hb) * (QR_BN / 16);
  }
  // DMA of a stage, 6 KB a wave: rows 16 w .. + 15 of the tile's 128 (chunk c of row r at c ^ (r & 15); past M
  // they read as zeros) and column tiles 2 w, 2 w + 1 (past N too)
  const uint32_t pitch = (uint32_t)(2 * a.ldx);
  const u32x4_t rows =
      q4_rsrc(a.x + (size_t)m0 * a.ldx, (uint32_t)(min(QR_BM, a.M - m0) - 1) * pitch + (uint32_t)(2 * a.K));
  const int tiles = min(QR_BN, a.N - 16 * t0) / 16;
  const u32x4_t codes = q4_rsrc(a.codes + (size_t)t0 * n * 1024, (uint32_t)(tiles * n) * 1024u);
  const u32x4_t scale = q4_rsrc(a.scale + (size_t)t0 * n * (16 * GPS), (uint32_t)(tiles * n) * (32u * GPS));
  uint32_t vx[4];
#pragma unroll
  for (int d = 0; d < 4; ++d) vx[d] = (16 * wave + 4 * d + g4) * pitch + 16 * (l16 ^ (4 * d + g4));
  const uint32_t vc[2] = {(uint32_t)(2 * wave * n) * 1024u + 16u * lane, (uint32_t)((2 * wave + 1) * n) * 1024u + 16u * lane};
  // (scales of a column tile, 32 GPS bytes, by 2 GPS lanes: 1 KB takes 32 / GPS tiles.  Every wave asks for
  // them and all write the same, so that their counts agree.)
  uint32_t vt[GPS == 4 ? 2 : 1];
#pragma unroll
  for (int d = 0; d < (GPS == 4 ? 2 : 1); ++d)
    vt[d] = (uint32_t)((64 * d + lane) / (2 * GPS) * n) * (32u * GPS) + 16u * (lane % (2 * GPS));
  const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)lds;
  constexpr int DMA = GPS == 4 ? 8 : 7;   // instructions of a wave's stage
  auto issue = [&](int slot, int st) {
    const uint32_t to = base + slot * SLOT;
#pragma unroll
    for (int d = 0; d < 4; ++d) q4_dma(to + 4096 * wave + 1024 * d, vx[d], rows, st * 256);
#pragma unroll
    for (int d = 0; d < 2; ++d) q4_dma(to + QR_CODES + 1024 * (2 * wave + d), vc[d], codes, st * 1024);
#pragma unroll
    for (int d = 0; d < (GPS == 4 ? 2 : 1); ++d) q4_dma(to + QR_SCALES + 1024 * d, vt[d], scale, st * (32 * GPS));
  };
  const int tw = t0 + 4 * wn;          // the wave's column tiles
  const bool there = 4 * wn < tiles;   // (N comes in 64s: the four exist or not)
  q4_u32x2 sc[4][GPS];
  const Q4Const kc;
  q4_f32x4 tot[4][4], c[4][4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) tot[j][i] = c[j][i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int g = 0; g < GPS; ++g) sc[j][g] = {0, 0};
  auto take_tile = [&](int j, int g) {   // a finished group's sums, with its scales
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t b = sc[j][g][e >> 1];
      const float f = __uint_as_float(e & 1 ? b & 0xffff0000u : b << 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) tot[j][i][e] = fmaf(f, c[j][i][e], tot[j][i][e]);
    }
  };
  auto take = [&](int g) {
#pragma unroll
    for (int j = 0; j < 4; ++j) take_tile(j, g);
  };
  const int ar = (64 * wm + l16) * 256;
  auto stage = [&](auto at, int st) {
    constexpr int SL = decltype(at)::value;
    const unsigned char* slot = lds + SL * SLOT;
    // this stage has landed (the next one's DMA may be on its way), every wave is done with the last one's slot
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(DMA) : "memory");
    issue((SL + 2) % 3, min(st + 2, n - 1));   // (always, for that count; past the end into a free slot)
    u32x4_t w[4], x[2][4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = *reinterpret_cast<const u32x4_t*>(slot + QR_CODES + 1024 * (4 * wn + j) + 16 * lane);
#pragma unroll
    for (int i = 0; i < 4; ++i) x[0][i] = *reinterpret_cast<const u32x4_t*>(slot + ar + 4096 * i + 16 * (g4 ^ l16));
    take(GPS - 1);   // the last stage's last group, while these are on their way
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int g = 0; g < GPS; ++g)
        sc[j][g] = *reinterpret_cast<const q4_u32x2*>(slot + QR_SCALES + (4 * wn + j) * (32 * GPS) + (g4 * GPS + g) * 8);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (q < 3)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          x[(q + 1) & 1][i] = *reinterpret_cast<const u32x4_t*>(slot + ar + 4096 * i + 16 * ((4 * (q + 1) + g4) ^ l16));
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (q && q % KPG == 0) take_tile(j, q / KPG - 1);   // (while the last tile's products run)
        const q4_bf16x8 f = q4_frag(w[j][q], kc);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          c[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, __builtin_bit_cast(q4_bf16x8, x[q & 1][i]),
                                                            q % KPG ? c[j][i] : q4_f32x4{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
      }
    }
  };
  issue(0, 0);
  issue(1, min(1, n - 1));
  for (int st = 0; st < n; st += 3) {
    stage(std::integral_constant<int, 0>{}, st);
    if (st + 1 < n) stage(std::integral_constant<int, 1>{}, st + 1);
    if (st + 2 < n) stage(std::integral_constant<int, 2>{}, st + 2);
  }
  take(GPS - 1);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // (no DMA into a workgroup that has ended)
  if (!there) return;
  // what 16 + z added: groups 32 k + 8 g4 + e of the lane's row
  const int groups = n * GPS, padded = (groups + 31) / 32 * 32;
  for (int k = 0; k < padded; k += 32) {
    q4_bf16x8 xs[3][4];
#pragma unroll
    for (int p = 0; p < 3; ++p)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int m = min(m0 + 64 * wm + 16 * i + l16, a.M - 1);
        xs[p][i] = __builtin_bit_cast(q4_bf16x8, *reinterpret_cast<const u32x4_t*>(
                                                     a.sums + ((size_t)p * a.M + m) * padded + k + 8 * g4));
      }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      q4_bf16x8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int g = min(k + 8 * g4 + e, groups - 1);   // (the sums of padding are zeros)
        const size_t at = ((size_t)(tw + j) * n + g / GPS) * (16 * GPS) + (l16 >> 2) * (4 * GPS) + g % GPS * 4 + (l16 & 3);
        float v = -bf16_to_f32(a.scale[at]);
        if constexpr (ZERO) v *= 16.f + (float)a.zero[at];
        hi[e] = (__bf16)v;
        lo[e] = (__bf16)(v - (float)(__bf16)v);
      }
#pragma unroll
      for (int p = 0; p < 3; ++p)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          tot[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(hi, xs[p][i], tot[j][i], 0, 0, 0);
          if (ZERO) tot[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(lo, xs[p][i], tot[j][i], 0, 0, 0);
        }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) q4_emit<SWIGLU>(a, tot[j][i], tw + j, m0 + 64 * wm + 16 * i + l16, g4);
}

// Row `src` of the (N, K) weight behind row r of tile t.
__device__ __forceinline__ int q4_src_row(int t, int r, int N, int swiglu) {
  return swiglu ? (r < 8 ? 0 : N / 2) + 8 * t + (r & 7) : 16 * t + r;
}

// Block blockIdx.x of the packed weight: thread 4 L + j writes lane L's word j.
__global__ __launch_bounds__(256) void q4_pack_kernel(const uint8_t* __restrict__ codes,
                                                      const uint16_t* __restrict__ scale,
                                                      const uint8_t* __restrict__ zero, uint32_t* pc, uint16_t* ps,
                                                      uint8_t* pz, int N, int K, int gps, int swiglu) {
  const int SK = K / Q4_STAGE, tid = threadIdx.x;
  const size_t blk = blockIdx.x;
  const int t = (int)(blk / SK), s = (int)(blk % SK);
  const int L = tid >> 2, j = tid & 3, r = L & 15, g = L >> 4;
  const uint32_t v = *reinterpret_cast<const uint32_t*>(codes + (size_t)q4_src_row(t, r, N, swiglu) * (K / 2) +
                                                        (Q4_STAGE * s + 32 * j + 8 * g) / 2);
  uint32_t w = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    w |= ((v >> (8 * e)) & 15u) << (4 * e) | ((v >> (8 * e + 4)) & 15u) << (16 + 4 * e);
  pc[blk * 256 + tid] = w << 3 | w >> 29;
  if (tid < 16 * gps) {   // element (g4, group, row 4 g4 + e)
    const int g4 = tid / (4 * gps), grp = tid / 4 % gps, e = tid & 3;
    const size_t src = (size_t)q4_src_row(t, 4 * g4 + e, N, swiglu) * (SK * gps) + s * gps + grp;
    ps[blk * (16 * gps) + tid] = scale[src];
    if (zero) pz[blk * (16 * gps) + tid] = zero[src];
  }
}

// Round to nearest: 32 threads a group.  With zeros: 16 levels from min(x, 0) to max(x, 0), the
// scale rounded to bf16 first; without: levels -8 .. 7 of max |x| / 7.5.  A group of zeros, or one
// whose range is no finite number, gets scale 0 or what it has.
__global__ __launch_bounds__(256) void q4_quantize_kernel(const uint16_t* __restrict__ w, uint8_t* codes,
                                                          uint16_t* scale, uint8_t* zero, long long groups, int G) {
  const long long g = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (g >= groups) return;      // (32 lanes at a time, whose exchanges below stay among them)
  const int l = threadIdx.x & 31, per = G / 32;
  const uint16_t* p = w + g * G + l * per;
  float v[4], lo = 0.f, hi = 0.f;
  for (int i = 0; i < per; ++i) {
    v[i] = bf16_to_f32(p[i]);
    lo = fminf(lo, v[i]);
    hi = fmaxf(hi, v[i]);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor(lo, o, 32));
    hi = fmaxf(hi, __shfl_xor(hi, o, 32));
  }
  const float s = round_bf16(zero ? (hi - lo) / 15.f : fmaxf(hi, -lo) / 7.5f);
  // (a scale below 2^-128 has no finite reciprocal: it and the values are then taken 2^100 times)
  const float up = s < 0x1p-100f ? 0x1p100f : 1.f, inv = s > 0.f ? 1.f / (s * up) : 0.f;
  const float z = zero ? fminf(fmaxf(rintf(-lo * up * inv), 0.f), 15.f) : 8.f;
  if (l == 0) {
    scale[g] = f32_to_bf16(s);
    if (zero) zero[g] = (uint8_t)z;
  }
  // a thread's 1, 2 or 4 codes: bytes of two; with one each, the even lanes write
  uint32_t c = 0;
  for (int i = 0; i < per; ++i) c |= (uint32_t)fminf(fmaxf(rintf(v[i] * up * inv) + z, 0.f), 15.f) << (4 * i);
  uint8_t* d = codes + (g * G + l * per) / 2;
  if (per == 1) {
    const uint32_t o = __shfl_down(c, 1, 32);
    if (!(l & 1)) *d = (uint8_t)(c | o << 4);
  } else {
    for (int i = 0; i < per / 2; ++i) d[i] = (uint8_t)(c >> (8 * i));
  }
}

template <int MT, int NT, int P, int GPS, bool ZERO, bool SWIGLU>
static void q4_start(const Q4Args& a, hipStream_t st) {
  hipLaunchKernelGGL((gemm_q4_lds_kernel<MT, NT, P, GPS, ZERO, SWIGLU>), dim3(a.N / (16 * NT), (a.M + 16 * MT - 1) / (16 * MT)),
                     dim3(Q4_THREADS), 0, st, a);
}

template <int NT, int GPS, bool ZERO, bool SWIGLU>
static void q4_wide(const Q4Args& a, hipStream_t st) {
  hipLaunchKernelGGL((gemm_q4_wide_kernel<NT, GPS, ZERO, SWIGLU>), dim3((a.N / 16 + NT - 1) / NT), dim3(Q4_THREADS), 0, st, a);
}

// Few rows.  As many column tiles a workgroup as still leave one for every CU: the rows' operands are then fetched
// less often.  (Up to 16 rows an even number, of which the last workgroup may have fewer.)
template <int GPS, bool ZERO, bool SWIGLU>
static void q4_few(const Q4Args& a, int cus, hipStream_t st) {
  const int mt = a.M <= 16 ? 1 : (a.M <= 32 ? 2 : 4);
  const long long tiles = (long long)((a.M + 16 * mt - 1) / (16 * mt)) * (a.N / 16);
  if (mt == 1) {
    const long long per = (tiles + cus - 1) / cus;
    if (per <= 1) hipLaunchKernelGGL((gemm_q4_kernel<GPS, ZERO, SWIGLU>), dim3(a.N / 16), dim3(Q4_THREADS), 0, st, a);
    else if (per <= 2) q4_wide<2, GPS, ZERO, SWIGLU>(a, st);
    else if (per <= 4) q4_wide<4, GPS, ZERO, SWIGLU>(a, st);
    else if (per <= 6) q4_wide<6, GPS, ZERO, SWIGLU>(a, st);
    else q4_wide<8, GPS, ZERO, SWIGLU>(a, st);
    return;
  }
  // (four tiles where their weights and sums fit the registers)
  const int nt = tiles >= 3LL * cus ? 4 : tiles >= 3LL * cus / 2 ? 2 : 1;
  if (mt == 2) {
    if constexpr (GPS < 4)
      if (nt == 4) return q4_start<2, 4, GPS == 1 ? 2 : 1, GPS, ZERO, SWIGLU>(a, st);
    if (nt >= 2) q4_start<2, 2, 2, GPS, ZERO, SWIGLU>(a, st);
    else q4_start<2, 1, 2, GPS, ZERO, SWIGLU>(a, st);
  } else {
    if constexpr (GPS == 1)
      if (nt == 4) return q4_start<4, 4, 1, GPS, ZERO, SWIGLU>(a, st);
    if (nt >= 2) q4_start<4, 2, GPS == 4 ? 1 : 2, GPS, ZERO, SWIGLU>(a, st);
    else q4_start<4, 1, 4, GPS, ZERO, SWIGLU>(a, st);
  }
}

template <int GPS, bool ZERO, bool SWIGLU>
static void q4_rows(const Q4Args& a, hipStream_t st) {
  const int groups = a.K / Q4_STAGE * GPS, padded = (groups + 31) / 32 * 32;
  const long long sums = (long long)a.M * padded;
  hipLaunchKernelGGL(q4_sums_kernel, dim3((unsigned)((sums + 15) / 16)), dim3(256), 0, st, a.x, a.ldx, a.sums, a.M, groups,
                     padded, Q4_STAGE / GPS, ZERO ? 1.f : 24.f);
  const int tiles = (a.M + QR_BM - 1) / QR_BM * ((a.N + QR_BN - 1) / QR_BN);
  hipLaunchKernelGGL((gemm_q4_rows_kernel<GPS, ZERO, SWIGLU>), dim3(tiles), dim3(512), 0, st, a);
}

// Whether the 128 x 256 tiles are the faster ones: their rounds of the chip at 1.8 us a stage against those
// of 64 x 64 tiles at 0.4 us a stage (eight waves share them) and 3 us each, the costs of groups of 128.  Smaller
// groups raise both alike, so one rule serves all (us, large / small tiles, at groups of 128; 64; 32: 129 x 4096 x
// 4096 59 / 17; 72 / 22; 88 / 25, 512 x 4096 x 4096 59 / 31; 75 / 45; 91 / 51, 700 x 4096 x 8192 114 / 80; 144 / 114;
// 179 / 133, 1000 x 4096 x 12288 167 / 156; 215 / 223; 271 / 258; but 300 x 12352 x 4096 60 / 64; 76 / 87; 92 / 100,
// 512 x 18432 x 4096 120 / 140; 151 / 193; 181 / 225, 1000 x 24576 x 4096 189 / 365; 234 / 503; 281 / 585.  With
// zeros 1000 x 4096 x 12288 170 / 174 and 278 / 272 at 128 and 32: where the rule errs it is a tie).
static bool q4_many_rows(int M, int N, int K, int cus) {
  if (M <= 64) return false;
  const long long large = (long long)((M + QR_BM - 1) / QR_BM) * ((N + QR_BN - 1) / QR_BN);
  const long long small = (long long)((M + 63) / 64) * (N / 64);
  const int n = K / Q4_STAGE;
  return (large + cus - 1) / cus * 18 * n < (small + cus - 1) / cus * (4 * n + 30);
}

template <int GPS>
static void q4_dispatch(const Q4Args& a, bool swiglu, int cus, hipStream_t st) {
  if (q4_many_rows(a.M, a.N, a.K, cus)) {
    if (a.zero) swiglu ? q4_rows<GPS, true, true>(a, st) : q4_rows<GPS, true, false>(a, st);
    else swiglu ? q4_rows<GPS, false, true>(a, st) : q4_rows<GPS, false, false>(a, st);
    return;
  }
  if (a.zero) swiglu ? q4_few<GPS, true, true>(a, cus, st) : q4_few<GPS, true, false>(a, cus, st);
  else swiglu ? q4_few<GPS, false, true>(a, cus, st) : q4_few<GPS, false, false>(a, cus, st);
}

static bool q4_shape_ok(int N, int K, int group) {
  return N > 0 && K > 0 && N % 64 == 0 && K % Q4_STAGE == 0 && (group == 32 || group == 64 || group == 128);
}

}  // namespace lollm

using namespace lollm;

LOLLM_API long long lollm_q4_packed_bytes(int N, int K, int group, int zeros) {
  if (!q4_shape_ok(N, K, group)) return -1;
  const long long groups = (long long)N * (K / group);
  return (long long)N * K / 2 + groups * (zeros ? 3 : 2);
}

LOLLM_API int lollm_q4_pack(const void* codes, const void* scales, const void* zeros, void* packed, int N, int K,
                            int group, int epilogue, void* stream) {
  if (!codes || !scales || !packed || epilogue < 0 || epilogue > 1) return LOLLM_EINVAL;
  if (!q4_shape_ok(N, K, group)) return LOLLM_EUNSUPPORTED;
  if ((uintptr_t)packed % 16 || (uintptr_t)codes % 4 || (uintptr_t)scales % 2) return LOLLM_EINVAL;
  const long long blocks = (long long)(N / 16) * (K / Q4_STAGE);
  if (blocks > 0x7fffffffLL) return LOLLM_EUNSUPPORTED;
  uint8_t* pc = (uint8_t*)packed;
  uint16_t* ps = (uint16_t*)(pc + (size_t)N * K / 2);
  uint8_t* pz = (uint8_t*)(ps + (size_t)N * (K / group));
  hipLaunchKernelGGL(q4_pack_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, (const uint8_t*)codes,
                     (const uint16_t*)scales, (const uint8_t*)zeros, (uint32_t*)pc, ps, pz, N, K, Q4_STAGE / group,
                     epilogue);
  return launch_status();
}

LOLLM_API int lollm_q4_quantize(const void* weight, void* codes, void* scales, void* zeros, int N, int K, int group,
                                void* stream) {
  if (!weight || !codes || !scales) return LOLLM_EINVAL;
  if (!q4_shape_ok(N, K, group)) return LOLLM_EUNSUPPORTED;
  const long long groups = (long long)N * (K / group);
  if ((groups + 7) / 8 > 0x7fffffffLL) return LOLLM_EUNSUPPORTED;
  hipLaunchKernelGGL(q4_quantize_kernel, dim3((unsigned)((groups + 7) / 8)), dim3(256), 0, (hipStream_t)stream,
                     (const uint16_t*)weight, (uint8_t*)codes, (uint16_t*)scales, (uint8_t*)zeros, groups, group);
  return launch_status();
}

static int q4_cus() {
  int dev = 0, cus = 0;
  if (hipGetDevice(&dev) != hipSuccess) return -1;
  if (hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return -1;
  return cus > 0 ? cus : -1;
}

static long long q4_workspace(int M, int N, int K, int group, int cus) {
  return q4_many_rows(M, N, K, cus) ? 6LL * M * ((K / group + 31) / 32 * 32) : 0;
}

LOLLM_API long long lollm_gemm_q4_workspace_bytes(int M, int N, int K, int group) {
  if (M <= 0 || !q4_shape_ok(N, K, group)) return -1;
  const int cus = q4_cus();
  return cus > 0 ? q4_workspace(M, N, K, group, cus) : -1;
}

LOLLM_API int lollm_gemm_q4(const void* A, long long lda, const void* packed, int zeros, void* C, long long ldc,
                            void* workspace, long long workspace_bytes, int M, int N, int K, int group, int epilogue,
                            void* stream) {
  if (!A || !packed || !C || M <= 0 || epilogue < 0 || epilogue > 1) return LOLLM_EINVAL;
  if (!q4_shape_ok(N, K, group)) return LOLLM_EUNSUPPORTED;
  if (lda < K || lda % 8 || ldc % 4 || ldc < (epilogue ? N / 2 : N)) return LOLLM_EINVAL;
  if (((uintptr_t)A | (uintptr_t)packed) % 16 || (uintptr_t)C % 8) return LOLLM_EINVAL;
  // 32-bit byte offsets inside a tile's rows of A and columns of W; the grids' sizes
  if (256LL * lda >= (1LL << 31) || 128LL * K >= (1LL << 31) || M > 65535 * 64) return LOLLM_EUNSUPPORTED;
  const int cus = q4_cus();
  if (cus < 0) return LOLLM_EUNSUPPORTED;
  const long long need = q4_workspace(M, N, K, group, cus);
  if (need && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16)) return LOLLM_EINVAL;
  if ((long long)((M + QR_BM - 1) / QR_BM) * ((N + QR_BN - 1) / QR_BN) > 0x7fffffffLL || need / 6 > 0x7fffffff0LL)
    return LOLLM_EUNSUPPORTED;
  Q4Args a;
  a.x = (const uint16_t*)A; a.y = (uint16_t*)C; a.ldx = lda; a.ldy = ldc;
  a.codes = (const uint8_t*)packed;
  a.scale = (const uint16_t*)(a.codes + (size_t)N * K / 2);
  a.zero = zeros ? (const uint8_t*)(a.scale + (size_t)N * (K / group)) : nullptr;
  a.M = M; a.N = N; a.K = K;
  a.sums = (uint16_t*)workspace;
  const hipStream_t st = (hipStream_t)stream;
  if (group == 128) q4_dispatch<1>(a, epilogue != 0, cus, st);
  else if (group == 64) q4_dispatch<2>(a, epilogue != 0, cus, st);
  else q4_dispatch<4>(a, epilogue != 0, cus, st);
  return launch_status();
}
