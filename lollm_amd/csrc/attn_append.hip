// Appending keys and values to a paged KV cache, with QK-norm and the position rotation on the
// way (gfx950): the attention prologue (fused_ops.hip) of the paged cache.
//
// Math, per token t of sequence b with cache row r = lengths[b] + t and position p:
//   n(x) = x rsqrt(mean x^2 + eps) (1 + w)               over the head's 256 values
//   rot(x)_i = x_i cos(p f_i) - x_{i+h} sin(p f_i),  rot(x)_{i+h} = x_{i+h} cos(p f_i) + x_i sin(p f_i)
//              for i < h = rotary_dim / 2, the other values as they are
//   q = rot(n(q)),  k = rot(n(k)),  v as it is; row r % page of page table[b][r / page].
// All of it in fp32, rounded once where it is stored; the angle in 64 bits, as turns reduced to
// half a turn (an fp32 angle at position 250000 is off by 0.01).  The gate is not copied: the
// attention reads it where the projection wrote it.
//
// 8-bit pages (e4m3 codes c, value c s) have one scale s for each (page, KV head) of K and of V,
// a power of two: the least with amax <= 448 s over the finite values of the page's new rows, and
// no less than the page's scale while it keeps rows of earlier calls (a call whose first row is
// not the page's first).  As s is a power of two, a larger one leaves the kept rows their values,
// but for codes that become subnormal, which are rounded again.  Values that are not finite
// become NaN.
//
// One workgroup per (sequence, page touched, KV head, K or V) for 8-bit pages, whose scale it
// owns, per 16 or 32 rows of a bf16 page; up to 4 rows per half-wave, 8 values a lane, 16-byte
// loads.  An 8-bit page's rows stay in registers as they came and are formed twice, for their
// maximum and for their rounding (in fp32 they would take the registers of two waves in three).
// Query heads: a workgroup per token and as many heads as its half-waves take at once where
// tokens are few, up to 32 heads otherwise.
//
// What bounds it: memory for prompts (32 / 4 heads, three inputs in turn, us and TB/s: 3 x 1500 tokens
// into bf16 pages 35, 5.3; 2 x 1999 32, 5.2; into 8-bit pages of 16 / 64 / 128 rows 34 / 39 / 43, 4.5 /
// 4.0 / 3.6, as the rows that a workgroup holds take its registers; one input again and again, part of
// it still in the chip's last cache, 31, 28 and 31 / 33 / 38), the launch for few tokens (4 to 5 us at
// 1 to 64).
#include "attn_common.h"

namespace lollm {

struct AppendArgs {
  const uint16_t* qkv;       // (B, T, Hq * 2 D + 2 Hkv D)
  const uint16_t* qw;        // QK-norm weights (D)
  const uint16_t* kw;
  const float* inv_freq;     // (rd / 2)
  const int32_t* lengths;    // (B)
  const int32_t* rope_pos;   // null, (B) or (B, T)
  const int32_t* table;      // (B, table_stride)
  uint16_t* q_out;           // (B, T, Hq, D)
  void* kp;                  // pools (n_pages, Hkv, page, D)
  void* vp;
  float* ks;                 // (n_pages, Hkv), 8-bit pages
  float* vs;
  long long table_stride;
  int per_token, T, Hq, Hkv, rd, table_width, n_pages, pshift;
  int gshift;                // rows of a workgroup's piece of a page: 1 << gshift
  int npg;                   // pieces that T rows can touch
  int kv_items, q_chunks;    // workgroups of K and V; query-head chunks of a token
  int chunk_heads;           // heads of a chunk
  float eps;
};

constexpr int AA_CHUNK = 32;                 // query heads of a workgroup at most

__device__ __forceinline__ void aa_unpack(u32x4_t w, float (&x)[8]) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[2 * e] = __uint_as_float(w[e] << 16);
    x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
  }
}

__device__ __forceinline__ u32x4_t aa_pack(const float (&y)[8]) {
  u32x4_t o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const bf16x2 t = {(__bf16)y[2 * e], (__bf16)y[2 * e + 1]};
    o[e] = __builtin_bit_cast(uint32_t, t);
  }
  return o;
}

// cos and sin of position p's angles into the half-wave's (or workgroup's) LDS rows, by `lanes`
// lanes of which this is `l`.
__device__ __forceinline__ void aa_angles(const float* inv_freq, int half, int p, int l, int lanes, float* cs,
                                          float* sn) {
  for (int f = l; f < half; f += lanes) {
    double turns = (double)p * (double)inv_freq[f] * 0.15915494309189533577;
    turns -= __builtin_rint(turns);
    cs[f] = __builtin_amdgcn_cosf((float)turns);
    sn[f] = __builtin_amdgcn_sinf((float)turns);
  }
}

// The half-wave's head vector (8 values a lane) normalised, w1 = 1 + w, and rotated; xs: 256 floats
// of its own.
__device__ __forceinline__ void aa_norm_rotate(float (&x)[8], const float (&w1)[8], int rd, float eps, int l,
                                               const float* cs, const float* sn, float* xs) {
  float ss = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) ss += x[e] * x[e];
  ss = sum_lanes16(ss);
  ss += __shfl_xor(ss, 16, 64);
  const float r = rsqrtf(ss / (float)AT_D + eps);
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = x[e] * r * w1[e];
  const int half = rd / 2;
  if (8 * l < rd) {
#pragma unroll
    for (int u = 0; u < 2; ++u)
      *reinterpret_cast<float4*>(xs + 8 * l + 4 * u) = make_float4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]);
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read by the same wave
  if (half % 8 == 0) {   // the lane's partners, cosines and sines are 8 in a row
    if (8 * l < rd) {
      const int f = 8 * l < half ? 8 * l : 8 * l - half, at = 8 * l < half ? 8 * l + half : f;
      float o[8], c[8], s[8];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        *reinterpret_cast<float4*>(o + 4 * u) = *reinterpret_cast<const float4*>(xs + at + 4 * u);
        *reinterpret_cast<float4*>(c + 4 * u) = *reinterpret_cast<const float4*>(cs + f + 4 * u);
        *reinterpret_cast<float4*>(s + 4 * u) = *reinterpret_cast<const float4*>(sn + f + 4 * u);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = x[e] * c[e] + (8 * l < half ? -o[e] : o[e]) * s[e];
    }
  } else if (8 * l < rd) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = 8 * l + e;
      if (d < rd) {
        const int f = d < half ? d : d - half;
        const float o = d < half ? -xs[d + half] : xs[f];
        x[e] = x[e] * cs[f] + o * sn[f];
      }
    }
  }
  asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // before the next vector takes xs
}

__device__ __forceinline__ float aa_scale_for(float amax) {
  const uint32_t u = __float_as_uint(amax);
  const int x = (int)(u >> 23) - 127 - ((u & 0x7fffffu) <= 0x600000u ? 8 : 7);   // 448 = 1.75 * 2^8
  return __uint_as_float((uint32_t)(max(x, -64) + 127) << 23);
}

__device__ __forceinline__ uint2 aa_codes(const float (&y)[8], float inv) {
  int lo = 0, hi = 0;
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0] * inv, y[1] * inv, lo, false);
  lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2] * inv, y[3] * inv, lo, true);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4] * inv, y[5] * inv, hi, false);
  hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6] * inv, y[7] * inv, hi, true);
  return make_uint2((uint32_t)lo, (uint32_t)hi);
}

// Query heads of item `item`: a token and a chunk of its heads.
template <int THREADS>
__device__ __forceinline__ void aa_queries(const AppendArgs& a, int item, float (&xs)[THREADS / 32][AT_D],
                                           float* cs, float* sn) {
  constexpr int D = AT_D, HALVES = THREADS / 32, QN = AA_CHUNK / HALVES;   // query heads per half-wave
  const int tid = threadIdx.x, l = tid & 31, hw = tid >> 5;
  const int bt = item / a.q_chunks, b = bt / a.T, t = bt - b * a.T;
  const long long row_w = (long long)a.Hq * 2 * D + 2LL * a.Hkv * D;
  const int h0 = (item - bt * a.q_chunks) * a.chunk_heads, h1 = min(h0 + a.chunk_heads, a.Hq);
  const int p = a.per_token ? a.rope_pos[bt] : (a.rope_pos ? a.rope_pos[b] : a.lengths[b]) + t;
  u32x4_t raw[QN];   // the half-wave's heads, on their way together
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int hd = h0 + hw + HALVES * i;
    raw[i] = u32x4_t{0, 0, 0, 0};
    if (hd < h1) raw[i] = reinterpret_cast<const u32x4_t*>(a.qkv + bt * row_w + (long long)hd * 2 * D)[l];
  }
  float w1[8];
  aa_unpack(reinterpret_cast<const u32x4_t*>(a.qw)[l], w1);
#pragma unroll
  for (int e = 0; e < 8; ++e) w1[e] += 1.f;
  aa_angles(a.inv_freq, a.rd / 2, p, tid, THREADS, cs, sn);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < QN; ++i) {
    const int hd = h0 + hw + HALVES * i;
    if (h0 + HALVES * i >= h1) break;
    float x[8];
    aa_unpack(raw[i], x);
    aa_norm_rotate(x, w1, a.rd, a.eps, l, cs, sn, xs[hw]);
    if (hd < h1) reinterpret_cast<u32x4_t*>(a.q_out + ((long long)bt * a.Hq + hd) * D)[l] = aa_pack(x);
  }
}

// RPH: rows of a piece per half-wave.
template <bool F8, int THREADS, int RPH>
__global__ __launch_bounds__(THREADS, THREADS == 512 ? 6 : 5) void attn_append_kernel(AppendArgs a) {
  constexpr int D = AT_D;
  constexpr int AA_THREADS = THREADS, AA_HALVES = THREADS / 32;   // head vectors at a time
  __shared__ __attribute__((aligned(16))) float xs[AA_HALVES][D];
  __shared__ __attribute__((aligned(16))) float cs[AA_HALVES][D / 2], sn[AA_HALVES][D / 2];
  __shared__ float red[AA_THREADS / 64];
  const int tid = threadIdx.x, l = tid & 31, hw = tid >> 5;
  const long long row_w = (long long)a.Hq * 2 * D + 2LL * a.Hkv * D;
  const int half = a.rd / 2;

  if ((int)blockIdx.x >= a.kv_items) {
    aa_queries<THREADS>(a, blockIdx.x - a.kv_items, xs, cs[0], sn[0]);
    return;
  }

  // K or V of one KV head in a piece of a page
  int item = blockIdx.x;
  const bool is_k = !(item & 1);
  item >>= 1;
  const int kvh = item % a.Hkv;
  item /= a.Hkv;
  const int b = item / a.npg, pi = item - b * a.npg;
  const long long len = a.lengths[b];
  const long long piece = (max(len, 0LL) >> a.gshift) + pi, idx = (piece << a.gshift) >> a.pshift;
  const long long lo = max(max(len, 0LL), piece << a.gshift), hi = min(len + a.T, (piece + 1) << a.gshift);
  if (lo >= hi || idx >= a.table_width) return;
  const int id = a.table[b * a.table_stride + idx];
  if (id < 0 || id >= a.n_pages) return;
  const int s0 = (int)(lo - (idx << a.pshift)), s1 = (int)(hi - (idx << a.pshift));   // slots
  const long long t0 = lo - len;                                                     // token of slot s0
  const long long first_row = ((long long)id * a.Hkv + kvh) << a.pshift;
  const uint16_t* src = a.qkv + ((long long)b * a.T + t0) * row_w + (long long)a.Hq * 2 * D +
                        (is_k ? 0 : a.Hkv * D) + kvh * D;
  u32x4_t raw[RPH];
#pragma unroll
  for (int i = 0; i < RPH; ++i) {
    const int s = hw + AA_HALVES * i;   // the row's place among the new ones
    raw[i] = u32x4_t{0, 0, 0, 0};
    if (s < s1 - s0) raw[i] = reinterpret_cast<const u32x4_t*>(src + s * row_w)[l];
  }
  float w1[8];
  aa_unpack(reinterpret_cast<const u32x4_t*>(a.kw)[l], w1);
#pragma unroll
  for (int e = 0; e < 8; ++e) w1[e] += 1.f;
  const int start = a.rope_pos && !a.per_token ? a.rope_pos[b] : (int)len;
  auto form = [&](int i, float (&x)[8]) {   // row i's values, in fp32
    const int s = hw + AA_HALVES * i;
    aa_unpack(raw[i], x);
    if (is_k) {   // (uniform; rows past the last are zeros and stay so)
      const int t = (int)t0 + min(s, s1 - s0 - 1);
      const int p = a.per_token ? a.rope_pos[(long long)b * a.T + t] : start + t;
      aa_angles(a.inv_freq, half, p, l, 32, cs[hw], sn[hw]);
      aa_norm_rotate(x, w1, a.rd, a.eps, l, cs[hw], sn[hw], xs[hw]);
    }
  };
  if constexpr (!F8) {
    uint16_t* dst = (uint16_t*)(is_k ? a.kp : a.vp) + (first_row + s0) * D;
#pragma unroll
    for (int i = 0; i < RPH; ++i) {
      const int s = hw + AA_HALVES * i;
      if (AA_HALVES * i >= s1 - s0) break;
      float x[8];
      form(i, x);
      if (s < s1 - s0) reinterpret_cast<u32x4_t*>(dst + (long long)s * D)[l] = aa_pack(x);
    }
  } else {
    float* scale = (is_k ? a.ks : a.vs) + (long long)id * a.Hkv + kvh;
    const float old = s0 > 0 ? *scale : 0.f;
    float amax = 0.f;
#pragma unroll
    for (int i = 0; i < RPH; ++i) {
      if (AA_HALVES * i >= s1 - s0) break;
      float y[8];
      form(i, y);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float m = fabsf(y[e]);
        amax = fmaxf(amax, m < INFINITY ? m : 0.f);
      }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    if ((tid & 63) == 0) red[tid >> 6] = amax;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < AA_THREADS / 64; ++w) amax = fmaxf(amax, red[w]);
    const float now = fmaxf(old, aa_scale_for(amax));
    const float inv = 1.f / now;   // (exact: a power of two)
    uint8_t* page = (uint8_t*)(is_k ? a.kp : a.vp) + first_row * D;
    if (old > 0.f && now > old) {   // kept rows under the larger scale
      const float f = old * inv;
      for (int s = hw; s < s0; s += AA_HALVES) {
        uint2* at = reinterpret_cast<uint2*>(page + s * D) + l;
        const uint2 c = *at;
        float z[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const int cw = (int)(u ? c.y : c.x);
          const auto a0 = __builtin_amdgcn_cvt_pk_f32_fp8(cw, false), a1 = __builtin_amdgcn_cvt_pk_f32_fp8(cw, true);
          z[4 * u] = a0[0]; z[4 * u + 1] = a0[1]; z[4 * u + 2] = a1[0]; z[4 * u + 3] = a1[1];
        }
        *at = aa_codes(z, f);
      }
    }
#pragma unroll
    for (int i = 0; i < RPH; ++i) {
      const int s = hw + AA_HALVES * i;
      if (AA_HALVES * i >= s1 - s0) break;
      float y[8];
      form(i, y);   // again: the rows as they came are half of what they are in fp32
      if (s < s1 - s0) reinterpret_cast<uint2*>(page + (s0 + s) * D)[l] = aa_codes(y, inv);
    }
    if (tid == 0) *scale = now;
  }
}

}  // namespace lollm

using namespace lollm;

template <bool F8, int THREADS, int RPH>
static void append_start(AppendArgs a, int B, int* too_many, hipStream_t st) {
  constexpr int halves = THREADS / 32;
  static_assert(halves * RPH >= 16, "a piece of 16 rows or more");
  a.npg = (int)(((long long)a.T + (1 << a.gshift) - 2) >> a.gshift) + 1;
  // few tokens: no half-wave has a second head to wait for
  a.chunk_heads = (long long)B * a.T < 1024 ? halves : AA_CHUNK;
  a.q_chunks = (a.Hq + a.chunk_heads - 1) / a.chunk_heads;
  const long long kv = 2LL * B * a.npg * a.Hkv, n = kv + (long long)B * a.T * a.q_chunks;
  if ((*too_many = n > 0x7fffffffLL)) return;
  a.kv_items = (int)kv;
  hipLaunchKernelGGL((attn_append_kernel<F8, THREADS, RPH>), dim3((unsigned)n), dim3(THREADS), 0, st, a);
}

LOLLM_API int lollm_attn_append(const void* qkv, const void* q_norm_w, const void* k_norm_w,
                                const float* inv_freq, const int32_t* lengths, const int32_t* rope_pos,
                                int rope_per_token, const int32_t* table, long long table_stride,
                                int table_width, int n_pages, int page, int kv_dtype, int B, int T, int Hq,
                                int Hkv, int D, int rotary_dim, float eps, void* q_out, void* k_pages,
                                void* v_pages, float* k_scale, float* v_scale, void* stream) {
  if (!qkv || !q_norm_w || !k_norm_w || !lengths || !table || !q_out || !k_pages || !v_pages)
    return LOLLM_EINVAL;
  if (rope_per_token && !rope_pos) return LOLLM_EINVAL;
  if (B <= 0 || T <= 0 || Hq <= 0 || Hkv <= 0) return LOLLM_EINVAL;
  if (table_width <= 0 || n_pages <= 0 || table_stride < table_width) return LOLLM_EINVAL;
  if (Hq > 32 * 65535 || Hkv > 65535) return LOLLM_EUNSUPPORTED;   // (32-bit offsets in a token)
  if (D != AT_D || rotary_dim < 0 || rotary_dim > D || rotary_dim % 2) return LOLLM_EUNSUPPORTED;
  if (rotary_dim > 0 && !inv_freq) return LOLLM_EINVAL;
  if (kv_dtype != LOLLM_BF16 && kv_dtype != LOLLM_F8) return LOLLM_EUNSUPPORTED;
  if (kv_dtype == LOLLM_F8 && (!k_scale || !v_scale)) return LOLLM_EINVAL;
  const int pshift = attn_page_shift(page);
  if (pshift < 0 || ((long long)table_width << pshift) > 0x7fffff00LL) return LOLLM_EUNSUPPORTED;
  AppendArgs a;
  a.qkv = (const uint16_t*)qkv; a.qw = (const uint16_t*)q_norm_w; a.kw = (const uint16_t*)k_norm_w;
  a.inv_freq = inv_freq; a.lengths = lengths; a.rope_pos = rope_pos; a.table = table;
  a.q_out = (uint16_t*)q_out; a.kp = k_pages; a.vp = v_pages; a.ks = k_scale; a.vs = v_scale;
  a.table_stride = table_stride; a.per_token = rope_per_token ? 1 : 0;
  a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.rd = rotary_dim; a.table_width = table_width; a.n_pages = n_pages;
  a.pshift = pshift; a.eps = eps;
  const bool f8 = kv_dtype == LOLLM_F8;
  a.gshift = f8 || pshift < 5 ? pshift : 5;
  int too_many = 0;
  hipStream_t st = (hipStream_t)stream;
  // New rows of a page at most: as many threads as bring it to 4 rows a half-wave.  A page of 128
  // takes 1024, which leave the query heads, most of the work of many tokens, a CU half empty: from
  // 2560 tokens on 512 with 8 rows (us, 1024 / 512 threads: 512 tokens 13 / 21, 1800 22 / 27, 3998
  // 42 / 37; a second launch for the query heads costs 5).
  const int rows = T < page ? T : page;
  if (f8) {
    if (rows <= 16) append_start<true, 256, 2>(a, B, &too_many, st);
    else if (rows <= 32) append_start<true, 256, 4>(a, B, &too_many, st);
    else if (rows <= 64) append_start<true, 512, 4>(a, B, &too_many, st);
    else if ((long long)B * T < 2560) append_start<true, 1024, 4>(a, B, &too_many, st);
    else append_start<true, 512, 8>(a, B, &too_many, st);
  } else if (rows <= 16) {
    append_start<false, 256, 2>(a, B, &too_many, st);
  } else {
    append_start<false, 256, 4>(a, B, &too_many, st);
  }
  return too_many ? LOLLM_EUNSUPPORTED : launch_status();
}
