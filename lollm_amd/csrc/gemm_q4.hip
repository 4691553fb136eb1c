// Products with 4-bit weights and group scales (gfx950): y[m, n] = sum_g s[n, g] sum_{k in g}
// x[m, k] (c[n, k] - z[n, g]), x and y bf16, c 4-bit codes, s bf16, z 8 where none is given; groups
// of 32, 64 or 128 k.  SwiGLU, silu(gate) up of the interleaved halves, in fp32, rounded once.
//
// Arithmetic.  A code q becomes the bf16 number 16 + q, exactly, with one shift and one
// v_and_or_b32 for two codes (its bits are the upper mantissa bits of 16).  The products run over
// these; what 16 + z adds to every code is taken off through the accumulator: a group's chain of
// products starts from -(16 + z) sum_k x, the sum itself one more product with a constant operand
// that all columns of a row tile share.  The group's scale then meets an fp32 sum, so weights are
// never rounded.  What the detour costs: partial sums of at most 32 sum |x| in fp32, 2^-24 of that
// against a group's typical 52 |x| is 1e-5 of it, below a bf16 output's 2^-9.  An infinite x gives
// NaN in its row.
//
// Layout (lollm_q4_pack, once per weight).  1 KB blocks of 16 rows x 128 k in operand order: lane
// 16 g + r holds row r's codes of k 32 j + 8 g .. + 8 in word j, even k in the low half and odd k in
// the high half.  Then the scales, per block [lane group g][group][rows 4 g ..], as the
// accumulator holds rows, and the zeros in the same order.
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
};

__device__ __forceinline__ q4_bf16x8 q4_frag(uint32_t w) {
  constexpr uint32_t MASK = 0x00780078u, BASE = 0x41804180u;
  const u32x4_t r = {((w << 3) & MASK) | BASE, ((w >> 1) & MASK) | BASE, ((w >> 5) & MASK) | BASE,
                     ((w >> 9) & MASK) | BASE};
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

// Few rows: a workgroup owns NT column tiles and MT row tiles, its eight waves deal out the stages
// of K (wave w: w, w + 8, ..), operands straight to registers, P stages ahead; the waves' sums meet
// in LDS in a fixed order at the end, so a row's bits depend on neither MT nor NT.
template <int MT, int NT, int P, int GPS, bool ZERO, bool SWIGLU>
__global__ __launch_bounds__(Q4_THREADS) void gemm_q4_kernel(Q4Args a) {
  constexpr int KPG = 4 / GPS;      // k-steps per group
  __shared__ __attribute__((aligned(16))) q4_f32x4 red[Q4_WAVES / 2][NT * MT][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int t0 = blockIdx.x * NT, m0 = blockIdx.y * (16 * MT);
  const int SK = a.K / Q4_STAGE;
  const int n = SK > wave ? (SK - wave + Q4_WAVES - 1) / Q4_WAVES : 0;

  const uint16_t* xr[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) xr[i] = a.x + (size_t)min(m0 + 16 * i + l16, a.M - 1) * a.ldx + 8 * g4;

  struct Stage {
    u32x4_t w[NT], x[MT][4];
    q4_u32x2 s[NT][GPS];
    uint32_t z[NT][GPS];
  };
  Stage st[P];
  auto load = [&](Stage& d, int i) {
    const int s = wave + Q4_WAVES * i;
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const size_t blk = (size_t)(t0 + j) * SK + s;
      d.w[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(a.codes + blk * 1024 + 16 * lane));
#pragma unroll
      for (int g = 0; g < GPS; ++g) {
        d.s[j][g] = *reinterpret_cast<const q4_u32x2*>(a.scale + blk * (16 * GPS) + (g4 * GPS + g) * 4);
        if (ZERO) d.z[j][g] = *reinterpret_cast<const uint32_t*>(a.zero + blk * (16 * GPS) + (g4 * GPS + g) * 4);
      }
    }
#pragma unroll
    for (int i2 = 0; i2 < MT; ++i2)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        d.x[i2][q] = *reinterpret_cast<const u32x4_t*>(xr[i2] + s * Q4_STAGE + 32 * q);
  };

  q4_f32x4 tot[NT][MT];
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int i = 0; i < MT; ++i) tot[j][i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
  // the constant operand: -(16 + 8), or 1 where columns have zeros of their own
  constexpr uint32_t CONST = ZERO ? 0x3f803f80u : 0xc1c0c1c0u;
  const q4_bf16x8 ones = __builtin_bit_cast(q4_bf16x8, u32x4_t{CONST, CONST, CONST, CONST});

  auto compute = [&](const Stage& d) {
#pragma unroll
    for (int g = 0; g < GPS; ++g) {
      q4_f32x4 c0[MT];
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        c0[i] = q4_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int q = 0; q < KPG; ++q)
          c0[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, __builtin_bit_cast(q4_bf16x8, d.x[i][g * KPG + q]),
                                                          c0[i], 0, 0, 0);
      }
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        q4_bf16x8 w[KPG];
#pragma unroll
        for (int q = 0; q < KPG; ++q) w[q] = q4_frag(d.w[j][g * KPG + q]);
        float sc[4], zc[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t b = d.s[j][g][e >> 1];
          sc[e] = __uint_as_float(e & 1 ? b & 0xffff0000u : b << 16);
          if (ZERO) zc[e] = -16.f - (float)((d.z[j][g] >> (8 * e)) & 0xffu);
        }
#pragma unroll
        for (int i = 0; i < MT; ++i) {
          q4_f32x4 c = c0[i];
          if (ZERO)
#pragma unroll
            for (int e = 0; e < 4; ++e) c[e] *= zc[e];
#pragma unroll
          for (int q = 0; q < KPG; ++q)
            c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[q], __builtin_bit_cast(q4_bf16x8, d.x[i][g * KPG + q]), c,
                                                        0, 0, 0);
#pragma unroll
          for (int e = 0; e < 4; ++e) tot[j][i][e] = fmaf(sc[e], c[e], tot[j][i][e]);
        }
      }
    }
  };

  if (n > 0) {
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (p < n) load(st[p], p);
    for (int i = 0; i < n; i += P) {
#pragma unroll
      for (int p = 0; p < P; ++p) {
        if (i + p < n) compute(st[p]);
        if (i + p + P < n) load(st[p], i + p + P);
      }
    }
  }
  // ((w0 + w4) + (w1 + w5)) + ..: waves 4 .. 7 hand theirs to 0 .. 3
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
  for (int k = wave; k < NT * MT; k += Q4_WAVES) {
    q4_f32x4 v = red[0][k][lane];
#pragma unroll
    for (int w = 1; w < Q4_WAVES / 2; ++w) v += red[w][k][lane];
    q4_emit<SWIGLU>(a, v, t0 + k / MT, m0 + 16 * (k % MT) + l16, g4);
  }
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
  pc[blk * 256 + tid] = w;
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
  const float inv = s > 0.f ? 1.f / s : 0.f;
  const float z = zero ? fminf(fmaxf(rintf(-lo * inv), 0.f), 15.f) : 8.f;
  if (l == 0) {
    scale[g] = f32_to_bf16(s);
    if (zero) zero[g] = (uint8_t)z;
  }
  // a thread's 1, 2 or 4 codes: bytes of two; with one each, the even lanes write
  uint32_t c = 0;
  for (int i = 0; i < per; ++i) c |= (uint32_t)fminf(fmaxf(rintf(v[i] * inv) + z, 0.f), 15.f) << (4 * i);
  uint8_t* d = codes + (g * G + l * per) / 2;
  if (per == 1) {
    const uint32_t o = __shfl_down(c, 1, 32);
    if (!(l & 1)) *d = (uint8_t)(c | o << 4);
  } else {
    for (int i = 0; i < per / 2; ++i) d[i] = (uint8_t)(c >> (8 * i));
  }
}

template <int MT, int NT, int P, int GPS>
static void q4_start(const Q4Args& a, bool swiglu, hipStream_t st) {
  const dim3 g(a.N / (16 * NT), (a.M + 16 * MT - 1) / (16 * MT)), b(Q4_THREADS);
  if (a.zero) {
    if (swiglu) hipLaunchKernelGGL((gemm_q4_kernel<MT, NT, P, GPS, true, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((gemm_q4_kernel<MT, NT, P, GPS, true, false>), g, b, 0, st, a);
  } else {
    if (swiglu) hipLaunchKernelGGL((gemm_q4_kernel<MT, NT, P, GPS, false, true>), g, b, 0, st, a);
    else hipLaunchKernelGGL((gemm_q4_kernel<MT, NT, P, GPS, false, false>), g, b, 0, st, a);
  }
}

template <int GPS>
static void q4_dispatch(const Q4Args& a, bool swiglu, hipStream_t st) {
  if (a.M <= 16) q4_start<1, 1, 4, GPS>(a, swiglu, st);
  else if (a.M <= 32) q4_start<2, 2, 2, GPS>(a, swiglu, st);
  else q4_start<4, 2, 1, GPS>(a, swiglu, st);
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

LOLLM_API int lollm_gemm_q4(const void* A, long long lda, const void* packed, int zeros, void* C, long long ldc, int M,
                            int N, int K, int group, int epilogue, void* stream) {
  if (!A || !packed || !C || M <= 0 || epilogue < 0 || epilogue > 1) return LOLLM_EINVAL;
  if (!q4_shape_ok(N, K, group)) return LOLLM_EUNSUPPORTED;
  if (lda < K || lda % 8 || ldc % 4 || ldc < (epilogue ? N / 2 : N)) return LOLLM_EINVAL;
  if (((uintptr_t)A | (uintptr_t)packed) % 16 || (uintptr_t)C % 8) return LOLLM_EINVAL;
  if (M > 65535 * 16) return LOLLM_EUNSUPPORTED;
  Q4Args a;
  a.x = (const uint16_t*)A; a.y = (uint16_t*)C; a.ldx = lda; a.ldy = ldc;
  a.codes = (const uint8_t*)packed;
  a.scale = (const uint16_t*)(a.codes + (size_t)N * K / 2);
  a.zero = zeros ? (const uint8_t*)(a.scale + (size_t)N * (K / group)) : nullptr;
  a.M = M; a.N = N; a.K = K;
  const hipStream_t st = (hipStream_t)stream;
  if (group == 128) q4_dispatch<1>(a, epilogue != 0, st);
  else if (group == 64) q4_dispatch<2>(a, epilogue != 0, st);
  else q4_dispatch<4>(a, epilogue != 0, st);
  return launch_status();
}
