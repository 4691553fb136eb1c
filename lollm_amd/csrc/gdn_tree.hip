// The Gated DeltaNet layer over a tree of drafted tokens (gfx950): gdn_layer.hip's short call, whose T
// positions are the nodes of a tree.  Node i continues from its parent: its convolution reads its three
// nearest ancestors and, above the tree, the window; its state is its parent's after one step of the
// delta rule.
//
// Mathematics.  With g the log-decays, G_i their sum over the path from the root to i, E = exp(G),
// k^ = k / |k|, q^ = q / (|q| sqrt(128)), S0 the committed state and j -> i for an ancestor,
//   u_i + beta_i sum_{j -> i, j != i} e^(G_i - G_j) (k^_i . k^_j) u_j = beta_i (v_i - E_i S0^T k^_i)
//   o_i = E_i S0^T q^_i + sum_{j -> i, or i} e^(G_i - G_j) (q^_i . k^_j) u_j:
// no node's state is ever formed, and S0, the call's largest operand, is read once for all nodes.
// The left side is a unit lower triangular matrix (a parent comes before its node): 16 x 16
// blocks on its diagonal are inverted by the recurrence, the rest is block substitution in fp32 MFMA.
// The products with S0 are bf16 MFMAs of the rows (bf16 as they are: q, k and v are bf16 tensors, which
// the records hold) with S0 as three bf16 parts, all of its bits: queries that cancel most of a state, and a norm
// behind them that scales the rest up, leave none to spare (with two parts outputs were off by 2^-17 of the terms).
// All sums are fp32, those of the decays 64 bits, as their differences count.
//
// One workgroup of eight waves per (sequence, v-head).  Wave w owns value columns 16 w ..: its part of S0
// lies in registers in the order in which the MFMA takes it as operand (lane 16 g + c: rows 32 s + 8 g
// + e, column 16 w + c), the triangular solve and the outputs of its columns never leave its
// accumulators, which hold rows in the order that the next product contracts over.
//
// Measured: 8 x 63 nodes, 32 v-heads 30 us, 16 x 16 26 us, 1 x 7 with 16 heads 11 us; the bytes (states in and
// out, rows, records) take 12.5, 16 and 0.5 at a large copy's rate.  With one workgroup a CU (63 nodes: 108 KB of
// LDS) its phases follow each other: of 50,000 cycles 13,000 each are the loads' way and the last products
// (fp32 MFMAs of a 64 x 64 triangle, a chain), 7,700 the convolution (exponentials), 5,500 the two matrices.
// Four waves of 32 columns took 36 us: each phase had half the waves to hide its latencies.
#include "gdn_common.h"

namespace lollm {

typedef float gt_f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 gt_bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 gt_bf16x2 __attribute__((ext_vector_type(2)));

constexpr int GT_MAX = 64;            // nodes
constexpr int GT_WAVES = 8, GT_THREADS = 64 * GT_WAVES;
constexpr int GT_K = 4;               // taps of the convolution
constexpr int GT_PW = GL_DK + 8;      // bf16 pitch of 128-wide rows

struct GtArgs {
  GdnLayerArgs l;
  const uint64_t* tree;   // (B, T) words of ancestors
};

template <int MT>
struct GtShared {
  static constexpr int TP = 16 * MT, PA = TP + 4;
  union {
    uint16_t raw[GT_K - 1 + TP][GL_CH];      // window rows, then the nodes' inputs
    struct {
      float am[TP][PA];                      // minus the triangular matrix below its diagonal
      float qk[TP][PA];                      // e^(G_i - G_j) q^_i . k^_j
      float tinv[MT][16][20];                // inverses of the diagonal blocks
    } m;
  };
  uint16_t q[TP][GT_PW], k[TP][GT_PW], v[TP][GT_PW];
  uint16_t cw[GL_CH][GT_K];
  uint64_t word[TP];                         // ancestors, without the node itself
  double G[TP];
  float beta[TP], rk[TP], rq[TP], E[TP];
  float ss[GT_WAVES][TP], rn[TP];
  uint8_t up[TP][4];                         // rows of raw behind the taps 2, 1, 0
};

__device__ __forceinline__ float gt_lo(uint32_t x) { return __uint_as_float(x << 16); }
__device__ __forceinline__ float gt_hi(uint32_t x) { return __uint_as_float(x & 0xffff0000u); }
__device__ __forceinline__ uint32_t gt_pack(float a, float b) {
  const gt_bf16x2 t = {(__bf16)a, (__bf16)b};
  return __builtin_bit_cast(uint32_t, t);
}
// Sum over the four lanes 16 apart, in each of them.
__device__ __forceinline__ float gt_sum_groups(float v) {
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
  const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
__device__ __forceinline__ float gt_dot2(uint32_t a, uint32_t b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(gt_bf16x2, a), __builtin_bit_cast(gt_bf16x2, b), c, false);
}
__device__ __forceinline__ gt_bf16x8 gt_row8(const uint16_t* p) {
  return __builtin_bit_cast(gt_bf16x8, *reinterpret_cast<const u32x4_t*>(p));
}

struct GtRecord {   // of a committed token: k in the lane's rows, v of its column; decay, beta, 1 / |k|
  u32x4_t k[4];
  uint16_t v;
  float4 sc;
};

template <int MT>
__global__ __launch_bounds__(GT_THREADS, MT < 4 ? 4 : 2) void gdn_tree_kernel(GtArgs ga) {
  using Sh = GtShared<MT>;
  constexpr int TP = Sh::TP;
  __shared__ __attribute__((aligned(16))) Sh sh;
  const GdnLayerArgs& a = ga.l;
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int c16 = lane & 15, g4 = lane >> 4;
  const int b = blockIdx.x / a.Hv, h = blockIdx.x % a.Hv;
  const int vpk = a.Hv / a.Hk, hk = h / vpk;
  const bool write_qk = (h % vpk) == 0;  // q/k window channels are shared by vpk heads
  const int T = a.T;
  constexpr int Km1 = GT_K - 1;
  constexpr size_t SS = (size_t)GL_DK * GL_DK;
  int off = a.conv_off[b];
  off = off < 0 ? 0 : (off > 2 * a.W - Km1 ? 2 * a.W - Km1 : off);  // never out of range
  const int wbase = off >= a.W ? 0 : a.W;          // window half written by this call
  const int half = a.rec_half[b] & 1, other = half ^ 1;
  int n = a.fresh ? 0 : a.replay[b];
  n = n < 0 ? 0 : (n > a.S ? a.S : n);
  const size_t hin = (size_t)(b * 2 + half) * a.Hv + h, hout = (size_t)(b * 2 + other) * a.Hv + h;
  const size_t win_b = (size_t)b * 2 * a.W;
  auto gbase = [&](int gi) {   // channel group (q, k, v) -> first global conv channel
    return gi == 0 ? hk * GL_DK : (gi == 1 ? a.key_dim + hk * GL_DK : 2 * a.key_dim + h * GL_DK);
  };

  // ---- 1. one batch of loads: the convolution's inputs and weights, the gates; the state last ----
  constexpr int NX = ((Km1 + TP) * 48 + GT_THREADS - 1) / GT_THREADS;
  const int nx = (Km1 + T) * 48;
  uint4 xv[NX];
#pragma unroll
  for (int it = 0; it < NX; ++it) {
    const int id = it * GT_THREADS + tid;
    xv[it] = make_uint4(0, 0, 0, 0);
    if (id < nx) {
      const int r = id / 48, gi = (id / 16) % 3, part = id % 16;
      const int c = gbase(gi) + part * 8;
      xv[it] = *reinterpret_cast<const uint4*>(r < Km1 ? a.win + (win_b + off + r) * a.C + c
                                                       : a.proj + ((size_t)b * T + r - Km1) * a.P + c);
    }
  }
  uint4 cwv = make_uint4(0, 0, 0, 0);
  if (tid < 192) cwv = *reinterpret_cast<const uint4*>(a.conv_w + (size_t)gbase(tid / 64) * GT_K + (tid % 64) * 8);
  const size_t base_ba = ((size_t)b * T + (lane < T ? lane : T - 1)) * a.P + a.C + a.value_dim;
  const uint16_t bb_raw = a.proj[base_ba + h], aa_raw = a.proj[base_ba + a.Hv + h];
  const uint64_t word_raw = ga.tree[(size_t)b * T + (lane < T ? lane : T - 1)];
  const float a_log = a.A_log[h], dtb = a.dt_bias[h];
  // the first two records, later the next two while one is applied: each in turn from memory costs its way there
  const uint8_t* rp = a.rep + hin * a.S * GL_REC_BYTES;
  GtRecord rec2[2];
  const int col = 16 * wave + c16;
  auto load_rec = [&](GtRecord& r, int j) {
    const uint8_t* p = rp + (size_t)min(j, a.S - 1) * GL_REC_BYTES;
#pragma unroll
    for (int s = 0; s < 4; ++s) r.k[s] = *reinterpret_cast<const u32x4_t*>(p + 2 * (32 * s + 8 * g4));
    r.v = *reinterpret_cast<const uint16_t*>(p + 2 * GL_DK + 2 * col);
    r.sc = *reinterpret_cast<const float4*>(p + 4 * GL_DK);
  };
#pragma unroll
  for (int j = 0; j < 2; ++j)
    if (j < n) load_rec(rec2[j], j);
  float S[4][8];
  {
    const __amdgpu_buffer_rsrc_t rs = buf_rsrc(a.rec + hin * SS, a.fresh ? 0u : (uint32_t)(SS * sizeof(float)));
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        S[s][e] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(
            rs, (uint32_t)(((32 * s + 8 * g4 + e) * GL_DK + col) * 4), 0, 2));
  }
  __builtin_amdgcn_sched_barrier(0);   // nothing that waits on a load moves above the state loads

  // ---- 2. to LDS, the new conv window to the other half; words, gates and path sums ----
#pragma unroll
  for (int it = 0; it < NX; ++it) {
    const int id = it * GT_THREADS + tid;
    if (id < (Km1 + TP) * 48) {
      const int r = id / 48, gi = (id / 16) % 3, part = id % 16;
      *reinterpret_cast<uint4*>(&sh.raw[r][gi * GL_DK + part * 8]) = xv[it];   // (zeros past the last node)
      if (id < nx && (gi == 2 || write_qk))
        *reinterpret_cast<uint4*>(a.win + (win_b + wbase + r) * a.C + gbase(gi) + part * 8) = xv[it];
    }
  }
  if (tid < 192) *reinterpret_cast<uint4*>(&sh.cw[(tid / 64) * GL_DK + (tid % 64) * 2][0]) = cwv;
  if (wave == 0) {
    const uint64_t above = lane < T ? word_raw & ((1ull << lane) - 1) : 0ull;
    const float g = lane < T ? -__expf(a_log) * softplus_g(bf16_to_f32(aa_raw) + dtb) : 0.f;
    const float beta = lane < T ? 1.f / (1.f + __expf(-bf16_to_f32(bb_raw))) : 0.f;
    // the path's sum by doubling: from the parent, its sum so far and its own.  In 64 bits: the weights are
    // differences of these sums, and a strong decay above both nodes (of 10^6 half a unit of the last place in 32
    // bits is 0.03) cancels in them.  Past 10^6, infinity among them, e^g is 0 all the same.
    double G = g < -1e6f ? -1e6f : g;
    int p = above ? 63 - __clzll((long long)above) : -1;
    for (int d = 1; d < T; d <<= 1) {
      const double Gp = __shfl(G, max(p, 0), 64);
      const int pp = __shfl(p, max(p, 0), 64);
      G += p >= 0 ? Gp : 0.;
      p = p >= 0 ? pp : -1;
    }
    if (lane < TP) {
      sh.word[lane] = above;
      sh.G[lane] = G;
      sh.E[lane] = lane < T ? __expf((float)G) : 0.f;
      sh.beta[lane] = beta;
      // the rows of the last three inputs before the node's own: nearest ancestors, then the window's
      uint64_t m = above;
      int row = Km1 - 1;
#pragma unroll
      for (int tap = 0; tap < Km1; ++tap) {
        const int p = m ? 63 - __clzll((long long)m) : -1;
        sh.up[lane][tap] = (uint8_t)(p >= 0 ? Km1 + p : row--);
        m = p >= 0 ? m & ~(1ull << p) : 0ull;
      }
    }
    if (lane < T) {   // decay and beta of the record (1 / |k| follows)
      float* rec = reinterpret_cast<float*>(a.rep + (hout * a.S + lane) * GL_REC_BYTES + 4 * GL_DK);
      rec[0] = __expf(g);
      rec[1] = beta;
    }
  }
  lds_only_barrier();
  // ---- 3. conv + SiLU: channels 8 o .. of the head's 384, nodes i, i + 10, .. ----
  if (tid < 480) {
    const int o = tid % 48;
    uint16_t* dst = o < 16 ? &sh.q[0][8 * o] : (o < 32 ? &sh.k[0][8 * o - GL_DK] : &sh.v[0][8 * o - 2 * GL_DK]);
    uint2 w[8];   // a channel's taps in pairs
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = *reinterpret_cast<const uint2*>(&sh.cw[8 * o + e][0]);
    for (int i = tid / 48; i < TP; i += 10) {
      const uint32_t up = *reinterpret_cast<const uint32_t*>(&sh.up[i][0]);
      const int rows[GT_K] = {(int)(up >> 16 & 255), (int)(up >> 8 & 255), (int)(up & 255), Km1 + i};
      u32x4_t x[GT_K];
#pragma unroll
      for (int tap = 0; tap < GT_K; ++tap) x[tap] = *reinterpret_cast<const u32x4_t*>(&sh.raw[rows[tap]][8 * o]);
      float acc[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t sel = e & 1 ? 0x07060302u : 0x05040100u;   // the same half of two rows
        acc[e] = gt_dot2(__builtin_amdgcn_perm(x[1][e >> 1], x[0][e >> 1], sel), w[e].x, 0.f);
        acc[e] = gt_dot2(__builtin_amdgcn_perm(x[3][e >> 1], x[2][e >> 1], sel), w[e].y, acc[e]);
      }
      u32x4_t y;
#pragma unroll
      for (int e = 0; e < 4; ++e) y[e] = i < T ? gt_pack(silu_g(acc[2 * e]), silu_g(acc[2 * e + 1])) : 0u;
      *reinterpret_cast<u32x4_t*>(dst + i * GT_PW) = y;
    }
  }
  lds_only_barrier();
  // ---- 4. norms, records ----
  {
    constexpr int PER = TP < 64 ? 16 : 8, CH = GL_DK / PER;   // threads of a node, values of a thread
    const int i = min(tid / PER, TP - 1), part = tid % PER;   // (16 nodes take half the threads)
    float sq = 0.f, sk = 0.f;
#pragma unroll
    for (int e = 0; e < CH; e += 8) {
      const u32x4_t q = *reinterpret_cast<const u32x4_t*>(&sh.q[i][CH * part + e]);
      const u32x4_t k = *reinterpret_cast<const u32x4_t*>(&sh.k[i][CH * part + e]);
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        sq = gt_dot2(q[x], q[x], sq);
        sk = gt_dot2(k[x], k[x], sk);
      }
    }
#pragma unroll
    for (int o = 1; o < PER; o <<= 1) {
      sq += __shfl_xor(sq, o, 64);
      sk += __shfl_xor(sk, o, 64);
    }
    if (part == 0 && tid < TP * PER) {
      const float rk = rsqrtf(sk + 1e-6f);
      sh.rk[i] = i < T ? rk : 0.f;
      sh.rq[i] = i < T ? rsqrtf(sq + 1e-6f) * rsqrtf((float)GL_DK) : 0.f;
      if (i < T) {
        float* rec = reinterpret_cast<float*>(a.rep + (hout * a.S + i) * GL_REC_BYTES + 4 * GL_DK);
        rec[2] = rk;
        rec[3] = 0.f;
      }
    }
    for (int id = tid; id < T * 32; id += GT_THREADS) {
      const int r = id / 32, p = id % 32;
      const uint16_t* src = p < 16 ? &sh.k[r][8 * p] : &sh.v[r][8 * p - GL_DK];
      *reinterpret_cast<uint4*>(a.rep + (hout * a.S + r) * GL_REC_BYTES + 16 * p) = *reinterpret_cast<const uint4*>(src);
    }
  }
  lds_only_barrier();
  // ---- 5. the two T x T matrices (block rows I, columns J <= I), the diagonal blocks' inverses ----
  {
    constexpr int NT = MT * (MT + 1) / 2;
    for (int t = wave; t < 2 * NT; t += GT_WAVES) {
      const bool qs = t >= NT;
      int I = 0, J = qs ? t - NT : t;
      while (J > I) J -= ++I;
      gt_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s)
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
            gt_row8(qs ? &sh.q[16 * I + c16][32 * s + 8 * g4] : &sh.k[16 * I + c16][32 * s + 8 * g4]),
            gt_row8(&sh.k[16 * J + c16][32 * s + 8 * g4]), acc, 0, 0, 0);
      const int j = 16 * J + c16;
      const double Gj = sh.G[j];
      const float rkj = sh.rk[j];
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int i = 16 * I + 4 * g4 + r;
        const uint64_t w = sh.word[i];
        const bool on = ((w >> j) & 1) || (qs && i == j);
        // (of a tree's words G_i <= G_j)
        const float f = on ? __expf(fminf((float)(sh.G[i] - Gj), 0.f)) * rkj * (qs ? sh.rq[i] : -sh.beta[i] * sh.rk[i]) : 0.f;
        (qs ? sh.m.qk : sh.m.am)[i][j] = on ? acc[r] * f : 0.f;
      }
    }
  }
  lds_only_barrier();
  if (wave < MT && lane < 16) {   // column `lane` of block `wave`'s inverse: x_i = [i = c] + sum_{j < i} am_ij x_j
    float x[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      float y = i == lane ? 1.f : 0.f;
#pragma unroll
      for (int j = 0; j < i; ++j) y = fmaf(sh.m.am[16 * wave + i][16 * wave + j], x[j], y);
      x[i] = y;
      sh.m.tinv[wave][i][lane] = y;
      if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (or all of the block waits in registers)
    }
  }
  // ---- 6. the committed state: n records on the stored one, to the other half ----
  auto apply = [&](const GtRecord& r) {
    float p[2] = {0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) p[s & 1] = fmaf(S[s][e], e & 1 ? gt_hi(r.k[s][e >> 1]) : gt_lo(r.k[s][e >> 1]), p[s & 1]);
    const float d = (bf16_to_f32(r.v) - r.sc.x * gt_sum_groups(p[0] + p[1]) * r.sc.z) * r.sc.y, kd = d * r.sc.z;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        S[s][e] = fmaf(e & 1 ? gt_hi(r.k[s][e >> 1]) : gt_lo(r.k[s][e >> 1]), kd, r.sc.x * S[s][e]);
  };
  for (int j = 0; j < n; j += 2) {
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      if (j + x >= n) break;
      apply(rec2[x]);
      if (j + x + 2 < n) load_rec(rec2[x], j + x + 2);
    }
  }
  {
    float* so = a.rec + hout * SS;
#pragma unroll
    for (int s = 0; s < 4; ++s)
#pragma unroll
      for (int e = 0; e < 8; ++e) __builtin_nontemporal_store(S[s][e], so + (32 * s + 8 * g4 + e) * GL_DK + col);
  }
  gt_bf16x8 S3[3][4];   // (each the rest of what is before it: together all of S0's 24 bits)
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      S3[0][s][e] = (__bf16)S[s][e];
      const float rest = S[s][e] - (float)S3[0][s][e];
      S3[1][s][e] = (__bf16)rest;
      S3[2][s][e] = (__bf16)(rest - (float)S3[1][s][e]);
    }
  // ---- 7. u and o, block row by block row; the gate's z on its way ----
  lds_only_barrier();   // the inverses
  uint16_t z[MT][4];
#pragma unroll
  for (int I = 0; I < MT; ++I)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = min(16 * I + 4 * g4 + r, T - 1);
      z[I][r] = a.proj[((size_t)b * T + i) * a.P + a.C + (size_t)h * GL_DK + col];
    }
  // the products with the state of all rows first: the chain below waits for none of them
  gt_f32x4 U[MT], O[MT];   // (U: the right sides until solved)
#pragma unroll
  for (int I = 0; I < MT; ++I) {
    gt_f32x4 ks[2], qs[2];   // with the state's first part, with the others
#pragma unroll
    for (int t = 0; t < 2; ++t) ks[t] = qs[t] = gt_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const gt_bf16x8 kr = gt_row8(&sh.k[16 * I + c16][32 * s + 8 * g4]), qr = gt_row8(&sh.q[16 * I + c16][32 * s + 8 * g4]);
#pragma unroll
      for (int t = 0; t < 3; ++t) {
        ks[t > 0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kr, S3[t][s], ks[t > 0], 0, 0, 0);
        qs[t > 0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(qr, S3[t][s], qs[t > 0], 0, 0, 0);
      }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * I + 4 * g4 + r;
      const float E = sh.E[i];
      U[I][r] = sh.beta[i] * (bf16_to_f32(sh.v[i][col]) - E * sh.rk[i] * (ks[0][r] + ks[1][r]));
      O[I][r] = E * sh.rq[i] * (qs[0][r] + qs[1][r]);
    }
  }
#pragma unroll
  for (int I = 0; I < MT; ++I) {
    gt_f32x4 rhs = U[I];
#pragma unroll
    for (int J = 0; J < I; ++J) {
      const float4 m = *reinterpret_cast<const float4*>(&sh.m.am[16 * I + c16][16 * J + 4 * g4]);
      const float mm[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
      for (int s = 0; s < 4; ++s) rhs = __builtin_amdgcn_mfma_f32_16x16x4f32(mm[s], U[J][s], rhs, 0, 0, 0);
    }
    {
      const float4 m = *reinterpret_cast<const float4*>(&sh.m.tinv[I][c16][4 * g4]);
      const float mm[4] = {m.x, m.y, m.z, m.w};
      U[I] = gt_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int s = 0; s < 4; ++s) U[I] = __builtin_amdgcn_mfma_f32_16x16x4f32(mm[s], rhs[s], U[I], 0, 0, 0);
    }
#pragma unroll
    for (int J = 0; J <= I; ++J) {
      const float4 m = *reinterpret_cast<const float4*>(&sh.m.qk[16 * I + c16][16 * J + 4 * g4]);
      const float mm[4] = {m.x, m.y, m.z, m.w};
#pragma unroll
      for (int s = 0; s < 4; ++s) O[I] = __builtin_amdgcn_mfma_f32_16x16x4f32(mm[s], U[J][s], O[I], 0, 0, 0);
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float s = sum_lanes16(O[I][r] * O[I][r]);
      if (c16 == 0) sh.ss[wave][16 * I + 4 * g4 + r] = s;
    }
  }
  lds_only_barrier();
  // ---- 8. gated RMSNorm ----
  if (tid < TP) {
    float ss = 0.f;
#pragma unroll
    for (int w = 0; w < GT_WAVES; ++w) ss += sh.ss[w][tid];
    sh.rn[tid] = rsqrtf(ss / (float)GL_DK + a.eps);
  }
  lds_only_barrier();
  const float nw = bf16_to_f32(a.norm_w[col]);
#pragma unroll
  for (int I = 0; I < MT; ++I)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int i = 16 * I + 4 * g4 + r;
      const float y = O[I][r] * sh.rn[i] * nw * silu_g(bf16_to_f32(z[I][r]));
      if (i < T) a.out[((size_t)b * T + i) * a.value_dim + (size_t)h * GL_DK + col] = f32_to_bf16(y);
    }
}

}  // namespace lollm

using namespace lollm;

LOLLM_API int lollm_gdn_layer_tree(const void* proj, long long proj_stride, const void* conv_w, const float* A_log,
                                   const float* dt_bias, const void* norm_w, void* win, const int32_t* conv_off,
                                   int win_rows, float* rec, const int32_t* rec_half, void* rep, const int32_t* replay,
                                   int slots, int fresh, const void* tree, void* out, int B, int T, int Hk, int Hv,
                                   int Dk, int Dv, int conv_kernel, float eps, void* stream) {
  if (!proj || !conv_w || !A_log || !dt_bias || !norm_w || !win || !conv_off || !rec || !rec_half || !rep ||
      !replay || !tree || !out)
    return LOLLM_EINVAL;
  if (B <= 0 || T <= 0 || Hk <= 0 || Hv <= 0 || Hv % Hk) return LOLLM_EINVAL;
  if (Dk != GL_DK || Dv != GL_DK || conv_kernel != GT_K || T > GT_MAX) return LOLLM_EUNSUPPORTED;
  if (slots < T || win_rows < conv_kernel - 1 + T) return LOLLM_EINVAL;   // a record and a window row a node
  const int key_dim = Hk * Dk, value_dim = Hv * Dv, C = 2 * key_dim + value_dim;
  if (proj_stride < (long long)C + value_dim + 2 * Hv || proj_stride % 8) return LOLLM_EINVAL;
  if (((uintptr_t)proj | (uintptr_t)conv_w | (uintptr_t)win | (uintptr_t)rec | (uintptr_t)rep | (uintptr_t)norm_w |
       (uintptr_t)out) % 16 || (uintptr_t)tree % 8)
    return LOLLM_EINVAL;
  GtArgs ga;
  GdnLayerArgs& a = ga.l;
  a.proj = (const uint16_t*)proj; a.conv_w = (const uint16_t*)conv_w; a.A_log = A_log;
  a.dt_bias = dt_bias; a.norm_w = (const uint16_t*)norm_w; a.win = (uint16_t*)win;
  a.conv_off = conv_off; a.rec = rec; a.rec_half = rec_half; a.rep = (uint8_t*)rep;
  a.replay = replay; a.out = (uint16_t*)out;
  a.P = proj_stride; a.T = T; a.Hk = Hk; a.Hv = Hv; a.C = C; a.key_dim = key_dim;
  a.value_dim = value_dim; a.K = conv_kernel; a.W = win_rows; a.S = slots; a.fresh = fresh ? 1 : 0;
  a.eps = eps;
  ga.tree = (const uint64_t*)tree;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 g(B * Hv), t(GT_THREADS);
  if (T <= 16) hipLaunchKernelGGL(gdn_tree_kernel<1>, g, t, 0, st, ga);
  else if (T <= 32) hipLaunchKernelGGL(gdn_tree_kernel<2>, g, t, 0, st, ga);
  else hipLaunchKernelGGL(gdn_tree_kernel<4>, g, t, 0, st, ga);
  return launch_status();
}
