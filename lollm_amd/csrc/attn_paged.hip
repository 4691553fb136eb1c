// Gated GQA attention over a paged KV cache, pages in bf16 or in 8 bits (gfx950).
//
// Math: as attn_verify.hip (offset-causal GQA, query i of the T new positions of sequence b at
// position kv_len[b] - T + i, output o * sigmoid(gate)), with key j of sequence b in row
// j % page of page table[b][j / page]: rows of D values, (n_pages, Hkv, page, D).  A key whose
// page is unmapped (an entry < 0 or >= n_pages) does not exist.  8-bit pages hold e4m3 codes c
// and one power-of-two scale s for each (page, KV head) of K and of V: the value is c s, which
// bf16 holds exactly.
//
// Work decomposition: attn_verify.hip's balanced split-K (128-key blocks of all (sequence, KV
// head x query block) pairs dealt out evenly, one partial per workgroup and pair, the combine
// kernel).  What differs is how a wave finds its rows.  Each of the four waves owns 32
// consecutive keys of a block, which lie in one page, or in two pages of 16.  Every 64 blocks
// each lane looks up one block of the range ahead -- its sequence and pair by binary search, its
// page ids, its scales -- and the loop takes them with readlane two blocks before it needs them,
// so no load of a page waits for a load of the table.
//   K: 16 bytes a lane straight into the S MFMA A operand (64-bit addresses: a pool may pass
//      4 GB).  Without a page it is masked, and the lanes read the pool's first line.
//   V: LDS DMA through a descriptor of the page's valid rows; the others become zeros, so that
//      nothing that an unmapped or unwritten row holds meets a weight of 0.
//   8 bits: a lane's 16 bytes of K are two k-steps (Q's columns are read in the same order) and
//      become bf16 with v_cvt_scalef32_pk_bf16_fp8, which applies the scale; V is read with the
//      transposing 8-bit LDS read and becomes fp16 (at_f16).
// Weights enter the product with V as hi + lo bf16 (attn_prefill.hip), with 8-bit V as fp16.
//
// What bounds it: the KV stream from some ten blocks a workgroup on, a fixed 12 us before.  16 x 4
// tokens, 32 / 4 heads, inputs in turn (us, TB/s of K and V): 128 keys 17 (8 bits 14.3), 1024 25.8, 2.6
// (22.6, 1.5), 4096 56, 4.8 (36, 3.7), 16384 172, 6.2 (102, 5.3), 65536 638, 6.7 (350, 6.1); pages of 16
// to 128 rows alike.  Of the fixed part the two launches are 5, lengths and table before the first
// load 1.5, the last block's products 1.5, the merge of the waves 1.8.  8-bit blocks
// are half the bytes: K is asked for two blocks ahead, of bf16 one, as a wave has at most 63 loads on
// its way.
#include <type_traits>

#include "attn_common.h"

namespace lollm {

constexpr int PG_WKEYS = AT_BLOCK / AW_WAVES;   // 32 keys of each block per wave
constexpr int PG_QROW = AT_D * 2 + 16;          // padded Q row in LDS
constexpr int PG_DUMP = AW_WAVES * AT_ROWS * (AT_D / 2 + 4) * 4;   // half of a pair's O of four waves

template <bool F8>
struct PagedSet {   // the V rows of a block in LDS
  static constexpr int ROW = F8 ? AT_D : AT_D * 2;
  // bf16: two rows (one DMA) + 64 bytes, so that the transposing reads of 8 rows touch every bank
  // at most twice; 8 bits: four rows a DMA, the 16-byte chunk c of row r at c ^ (r % 16)
  static constexpr int PAIR = F8 ? 2 * AT_D : 2 * AT_D * 2 + 64;
  static constexpr int WAVE = PG_WKEYS / 2 * PAIR;
  static constexpr int SET = AW_WAVES * WAVE;
};

// One block of a workgroup's range, uniform across the wave.
struct PgUnit {
  int b, ph, j, L;
  int page[2];                // of the wave's keys 0..15 and 16..31, -1 unmapped or past the end
  float ks[2];
  int vs[2];                  // bits of V's scales, 0 unmapped
};

__device__ __forceinline__ uint32_t lds_at(const unsigned char* p) {
  return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) unsigned char*)p;
}

// A wave's V operands of a block by transposing reads, landed when they return.  8 bits: column
// tile d at `at` with the chunk bits (5 .. 7: rows begin at multiples of 256) flipped by 2 d, keys
// 16 .. 31 4 KB further.
__device__ __forceinline__ void pg_read_codes(uint32_t at, i32x2_t (&v)[16]) {
#define RD2(i, j, a) "ds_read_b64_tr_b8 %" #i ", %" #a "\n\tds_read_b64_tr_b8 %" #j ", %" #a " offset:4096\n\t"
  asm volatile(RD2(0, 1, 16) RD2(2, 3, 17) RD2(4, 5, 18) RD2(6, 7, 19) RD2(8, 9, 20) RD2(10, 11, 21) RD2(12, 13, 22)
                   RD2(14, 15, 23) "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]),
                 "=&v"(v[7]), "=&v"(v[8]), "=&v"(v[9]), "=&v"(v[10]), "=&v"(v[11]), "=&v"(v[12]), "=&v"(v[13]),
                 "=&v"(v[14]), "=&v"(v[15])
               : "v"(at), "v"(at ^ 32u), "v"(at ^ 64u), "v"(at ^ 96u), "v"(at ^ 128u), "v"(at ^ 160u), "v"(at ^ 192u),
                 "v"(at ^ 224u)
               : "memory");
#undef RD2
}

// bf16: two column tiles 64 bytes apart, rows in pairs of PAIR bytes.
template <int PAIR>
__device__ __forceinline__ void pg_read_rows(uint32_t at, u32x2_t (&v)[8]) {
#define RD(i, off) "ds_read_b64_tr_b16 %" #i ", %8 offset:%" #off "\n\t"
  asm volatile(RD(0, 9) RD(1, 10) RD(2, 11) RD(3, 12) RD(4, 13) RD(5, 14) RD(6, 15) RD(7, 16)
               "s_waitcnt lgkmcnt(0)"
               : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
               : "v"(at), "n"(0), "n"(4 * PAIR), "n"(8 * PAIR), "n"(12 * PAIR), "n"(64), "n"(64 + 4 * PAIR),
                 "n"(64 + 8 * PAIR), "n"(64 + 12 * PAIR)
               : "memory");
#undef RD
}

template <bool F8>
__global__ __launch_bounds__(AW_THREADS, 1) void attn_paged_kernel(PagedArgs p) {
  using Set = PagedSet<F8>;
  const AttnArgs& a = p.a;
  __shared__ __attribute__((aligned(256))) unsigned char vs0[Set::SET];   // V of even blocks
  __shared__ __attribute__((aligned(256))) unsigned char vs1[Set::SET];   // V of odd blocks
  __shared__ __attribute__((aligned(16))) unsigned char own_dump[F8 ? PG_DUMP : 16];
  __shared__ __attribute__((aligned(16))) unsigned char qs[AT_ROWS * PG_QROW];   // Q of the pair
  __shared__ float mx[AW_WAVES][32], lx[AW_WAVES][32], vx[AW_WAVES];
  __shared__ int pre[AT_MAXB + 1], len[AT_MAXB], tmp[AW_WAVES];
  static_assert(F8 || PG_DUMP <= Set::SET, "the O dump fits a V set");

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  const int w = blockIdx.x;
  const int PH = a.Hkv * a.qblocks;

  // All pairs' blocks, dealt out in equal ranges, the first `more` of them one block longer (the
  // host keeps U below 2^31); one block a workgroup where there are fewer blocks, so that no
  // workgroup between a pair's has none.
  const uint32_t U = (uint32_t)PH * (uint32_t)__builtin_amdgcn_readfirstlane(build_prefix(a, pre, len, tmp));
  const uint32_t nw = min((uint32_t)a.nw, U), each = U / max(nw, 1u), more = U - each * nw;
  auto owner = [&](uint32_t u) {
    const uint32_t cut = more * (each + 1);
    return (int)(u < cut ? u / (each + 1) : more + (u - cut) / each);
  };
  const uint32_t u0 = min((uint32_t)w, nw) * each + min((uint32_t)w, more);
  const uint32_t u1 = (uint32_t)w < nw ? u0 + each + ((uint32_t)w < more) : u0;
  auto build_table = [&]() {
    const int npairs = a.B * PH;
    int2* tab = reinterpret_cast<int2*>(a.ws + (size_t)(a.nw + npairs) * AT_PART);
    for (int pr = w * AW_THREADS + tid; pr < npairs; pr += (U ? (int)nw : a.nw) * AW_THREADS) {
      const int pb = pr / PH, pph = pr % PH, pnb = pre[pb + 1] - pre[pb];
      int wf = -1, wl = -1;
      if (pnb > 0) {
        const uint32_t first = (uint32_t)PH * pre[pb] + (uint32_t)pph * pnb;
        wf = owner(first);
        wl = owner(first + pnb - 1);
      }
      tab[pr] = make_int2(wf, wl);
    }
  };
  if (u0 >= u1) {   // no work for this one; with no keys at all the table says so
    if (U == 0) build_table();
    return;
  }

  // The lane's block of the 64 from tbase on.
  uint32_t tbase = u0;
  int tb = 0, tph = 0, tj = 0, tL = 0, tp[2];
  float tks[2] = {1.f, 1.f}, tvs[2] = {1.f, 1.f};
  auto look_up = [&]() {
    const uint32_t u = min(tbase + lane, u1 - 1);
    int lo = 0, hi = a.B - 1;   // the last sequence that begins at or before u: not an empty one
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if ((uint32_t)PH * pre[mid] <= u) lo = mid; else hi = mid - 1;
    }
    const uint32_t nb = pre[lo + 1] - pre[lo], r = u - (uint32_t)PH * pre[lo];
    tb = lo;
    tph = (int)(r / nb);
    tj = (int)(r - tph * nb);
    tL = len[lo];
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = tj * AT_BLOCK + PG_WKEYS * wave + 16 * g;
      const bool in = key >= 0 && key < tL;   // (a table of 2^31 rows: a last block's keys may wrap)
      const int id = in ? p.table[(long long)lo * p.table_stride + (key >> p.pshift)] : -1;
      tp[g] = id >= 0 && id < p.n_pages ? id : -1;
    }
  };
  auto look_up_scales = [&]() {
    if constexpr (F8) {
      const int kvh = tph / a.qblocks;
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const size_t s = (size_t)max(tp[g], 0) * a.Hkv + kvh;
        tks[g] = p.ks[s];
        tvs[g] = p.vs[s];
      }
    }
  };
  // (an unmapped page's scale is not there: whatever lies in page 0's may not meet its zeros)
  auto unit_scales = [&](PgUnit& X, uint32_t u) {
    const int i = (int)(u - tbase);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int k = __builtin_amdgcn_readlane(__float_as_int(tks[g]), i);
      const int v = __builtin_amdgcn_readlane(__float_as_int(tvs[g]), i);
      X.ks[g] = __int_as_float(X.page[g] >= 0 ? k : 0x3f800000);
      X.vs[g] = X.page[g] >= 0 ? v & 0x7f800000 : 0;
    }
  };
  auto unit = [&](uint32_t u) {
    const int i = (int)(u - tbase);
    const bool live = u < u1;
    PgUnit X;
    X.b = __builtin_amdgcn_readlane(tb, i);
    X.ph = __builtin_amdgcn_readlane(tph, i);
    X.j = __builtin_amdgcn_readlane(tj, i);
    X.L = __builtin_amdgcn_readlane(tL, i);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      X.page[g] = live ? __builtin_amdgcn_readlane(tp[g], i) : -1;
      X.ks[g] = 1.f;
      X.vs[g] = 0;
    }
    return X;
  };

  // Loads of a block (all unconditional; past the range no page is mapped).
  constexpr int KL = Set::ROW / 32;   // 16-byte loads of a key's row per lane (two lanes a row)
  constexpr int KAHEAD = F8 ? 2 : 1;  // blocks that K is asked for ahead of its products
  u32x4_t kr[KAHEAD][KL], qr[4];
  const int pmask = (1 << p.pshift) - 1;
  auto row_of = [&](const PgUnit& X, int page, int key) {   // the pool's row of a key in that page
    const int kvh = X.ph / a.qblocks;
    return (((long long)page * a.Hkv + kvh) << p.pshift) + (key & pmask);
  };
  auto issue_k = [&](u32x4_t (&to)[KL], const PgUnit& X) {
    const int key0 = X.j * AT_BLOCK + PG_WKEYS * wave;
    const long long r0 = row_of(X, max(X.page[0], 0), key0), r1 = row_of(X, max(X.page[1], 0), key0 + 16);
    // (without a page all lanes read the pool's first bytes, one line an instruction)
    const long long at = (l32 < 16 ? r0 : r1) * Set::ROW + (l32 & 15) * Set::ROW + 16 * h;
    const unsigned char* src =
        reinterpret_cast<const unsigned char*>(a.kc) + ((l32 < 16 ? X.page[0] : X.page[1]) >= 0 ? at : 0);
#pragma unroll
    for (int i = 0; i < KL; ++i) to[i] = *reinterpret_cast<const u32x4_t*>(src + 32 * i);
  };
  auto issue_v = [&](unsigned char* vset, const PgUnit& X) {
    unsigned char* dst = vset + wave * Set::WAVE;
    const int key0 = X.j * AT_BLOCK + PG_WKEYS * wave;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      const int key = key0 + 16 * g;
      const int rows = X.page[g] >= 0 ? min(X.L - key, 16) : 0;   // (a mapped group begins before L)
      const __amdgpu_buffer_rsrc_t rs =
          buf_rsrc(reinterpret_cast<const unsigned char*>(a.vc) + row_of(X, max(X.page[g], 0), key) * Set::ROW,
                   (uint32_t)(rows * Set::ROW));
      if constexpr (F8) {
        // four rows a DMA: lane -> row 4 i + lane / 16, chunk (lane % 16) ^ row
        const uint32_t vo = 256u * (lane >> 4) + 16u * ((lane & 15) ^ (lane >> 4));
#pragma unroll
        for (int i = 0; i < 4; ++i)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(dst + 4096 * g + 1024 * i), 16,
                                                   1024u * i + (vo ^ (64u * i)), 0, 0, 2);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(dst + Set::PAIR * (8 * g + i)), 16,
                                                   1024u * i + 16u * lane, 0, 0, 2);
      }
    }
  };
  // Row r of a pair is position r / n_rep of its query block, head r % n_rep; this thread's rows
  // tid / 32 + 8 i of Q, 16 bytes each.
  uint32_t qoff[4];
  int qi[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = (tid >> 5) + 8 * i;
    qi[i] = (int)(((uint32_t)r * p.rep_mul) >> 16);
    qoff[i] = ((uint32_t)qi[i] * a.Hq + (r - qi[i] * a.n_rep)) * (AT_D * 2) + 16u * (tid & 31);
  }
  auto issue_q = [&](const PgUnit& X) {
    const int kvh = X.ph / a.qblocks, q0 = (X.ph - kvh * a.qblocks) * a.QB, QB = min(a.QB, a.T - q0);
    const uint16_t* base = a.q + (((size_t)X.b * a.T + q0) * a.Hq + kvh * a.n_rep) * AT_D;
    const __amdgpu_buffer_rsrc_t rs = buf_rsrc(base, (uint32_t)((QB - 1) * a.Hq + a.n_rep) * (AT_D * 2));
#pragma unroll
    for (int i = 0; i < 4; ++i)
      qr[i] = __builtin_bit_cast(u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                                              rs, qi[i] < QB ? qoff[i] : 0x80000000u, 0, 0));
  };

  look_up();
  PgUnit C = unit(u0), X1 = unit(u0 + 1), X2 = unit(u0 + 2);
  look_up_scales();   // before the rows: here when these are
  issue_q(C);
  // (in the loop's own order, for the counts of its waits)
  if constexpr (F8) issue_k(kr[0], C);
  issue_v(vs0, C);
  issue_k(kr[KAHEAD - 1], F8 ? X1 : C);
  issue_v(vs1, X1);
  if constexpr (F8) {
    unit_scales(C, u0);
    unit_scales(X1, u0 + 1);
    unit_scales(X2, u0 + 2);
  }
  build_table();

  f32x16 O[8];            // O^T: d-tile dt (32 columns) x the 32 rows; lane row = l32
  float m_ref = -INFINITY, l_s = 0.f;
  int v_ref = 0;          // 8 bits: O counts in units of this scale (bits), at_f16
  constexpr float LAG = F8 ? AT_F16_LAG : 16.f, UP = F8 ? AT_F16_UP : 0.f;
  const int lq = (int)(((uint32_t)l32 * p.rep_mul) >> 16);   // the lane's position in its query block
  int qpos = 0, rows = 0;

  for (uint32_t ub = u0; ub < u1; ub += 2) {
#pragma unroll
    for (int set = 0; set < 2; ++set) {   // (ended from the inside)
      unsigned char* vset = set ? vs1 : vs0;
      const uint32_t u = ub + set;
      const bool any = (C.page[0] & C.page[1]) != -1;   // keys of this wave to look at
      const int nb = nblk_of(C.L);
      const bool seg_first = u == u0 || C.j == 0;
      const bool seg_last = u == u1 - 1 || C.j == nb - 1;
      if (seg_first) {
        const int q0 = (C.ph % a.qblocks) * a.QB;
        qpos = C.L - a.T + q0 + lq;
        rows = a.n_rep * min(a.QB, a.T - q0);
#pragma unroll
        for (int dt = 0; dt < 8; ++dt)
#pragma unroll
          for (int r = 0; r < 16; ++r) O[dt][r] = 0.f;
        m_ref = -INFINITY;
        l_s = 0.f;
        v_ref = 0;
        // (the previous pair's last block ended with barriers: no wave still reads qs)
#pragma unroll
        for (int ii = 0; ii < 4; ++ii)
          *reinterpret_cast<u32x4_t*>(qs + ((tid >> 5) + 8 * ii) * PG_QROW + 16 * (tid & 31)) = qr[ii];
        aw_barrier();
      }
      // S^T (32 keys x 32 rows) = K Q^T
      f32x16 S, S1;   // two chains: a product waits for the one before the last
#pragma unroll
      for (int r = 0; r < 16; ++r) S[r] = S1[r] = 0.f;
      if (any) {
        if constexpr (F8) {
          const float sc = l32 < 16 ? C.ks[0] : C.ks[1];
          const unsigned char* qp = qs + l32 * PG_QROW + 32 * h;   // columns 32 i + 16 h ..
#pragma unroll
          for (int i = 0; i < KL; ++i) {
            const u32x4_t c = kr[set][i];
            const bf16x8 k0 = at_bf16(c.x, c.y, sc), k1 = at_bf16(c.z, c.w, sc);
            S = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k0, *reinterpret_cast<const bf16x8*>(qp + 64 * i), S, 0, 0, 0);
            S1 = __builtin_amdgcn_mfma_f32_32x32x16_bf16(k1, *reinterpret_cast<const bf16x8*>(qp + 64 * i + 16), S1, 0, 0, 0);
          }
        } else {
#pragma unroll
          for (int i = 0; i < KL; ++i) {
            const bf16x8 qv = *reinterpret_cast<const bf16x8*>(qs + l32 * PG_QROW + 16 * h + 32 * i);
            f32x16& s = i & 1 ? S1 : S;
            s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kr[0][i]), qv, s, 0, 0, 0);
          }
        }
      }
      // Q of the next block's pair (staged at that block's start)
      if (u + 1 < u1 && X1.j == 0) issue_q(X1);
      // K into the registers S consumed, V of this block landed: after it at least V of the next
      // block and K of the next KAHEAD were asked for.  (Counted here and V read by hand: where
      // the compiler cannot tell the sets apart it waits for both, and nothing is on its way while
      // the products run.)
      if constexpr (F8) {
        issue_k(kr[set], X2);
        asm volatile("s_waitcnt vmcnt(24)" ::: "memory");
      } else {
        issue_k(kr[0], X1);
        asm volatile("s_waitcnt vmcnt(32)" ::: "memory");
      }
      static_assert(KAHEAD * KL + PG_WKEYS * Set::ROW / 1024 == (F8 ? 24 : 32), "the counts above");

      if (any) {
        // mask: acc r holds key 32 wave + 8 (r / 4) + 4 h + r % 4 of the block
        const int kb = C.j * AT_BLOCK + PG_WKEYS * wave + 4 * h;
        const int lim = min(C.L - 1, qpos) - kb;
        const int lim0 = C.page[0] >= 0 ? lim : -1, lim1 = C.page[1] >= 0 ? lim : -1;
        float bm = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int kk = 8 * (r >> 2) + (r & 3);
          S[r] = kk <= (r < 8 ? lim0 : lim1) ? S[r] + S1[r] : -INFINITY;
          bm = fmaxf(bm, S[r]);
        }
        bm = fmaxf(bm, __shfl_xor(bm, 32, 64));
        // the reference max moves (and l, O are rescaled) only when a row's block max exceeds it
        // by more than LAG in the exponent: attn_verify's rule, each row's own decision
        const bool big = (bm - m_ref) * a.cl2 > LAG;
        const bool had = m_ref != -INFINITY;   // (nothing to rescale at a row's first block)
        const int v_now = F8 ? at_units(v_ref, C.vs[0], C.vs[1]) : 0;
        const bool units = F8 && v_ref != 0 && v_now != v_ref;
        if (__builtin_amdgcn_readfirstlane((int)(__ballot(big && had) != 0 || units))) {
          float alpha = big && had ? fast_exp2((m_ref - bm) * a.cl2) : 1.f;
          l_s *= alpha;
          if (units) alpha *= at_ratio(v_ref, v_now);
#pragma unroll
          for (int dt = 0; dt < 8; ++dt) {
            // (O stays in accumulator registers but for the tile at hand: without the pins the
            // compiler copies all of it to vector registers and back in every block)
            asm volatile("" : "+a"(O[dt]));
            O[dt] *= alpha;
            asm volatile("" : "+a"(O[dt]));
            __builtin_amdgcn_sched_barrier(0);
          }
        }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) asm volatile("" : "+a"(O[dt]));
        m_ref = big ? bm : m_ref;
        v_ref = v_now;
        const float base = m_ref == -INFINITY ? 0.f : m_ref * a.cl2 - UP;
        float e[16];
#pragma unroll
        for (int r = 0; r < 16; ++r) e[r] = fast_exp2(__builtin_fmaf(S[r], a.cl2, -base));
        float ps = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) ps += e[r];
        l_s += ps;
        bf16x8 Ph[2], Pl[2];
        f16x8 Pf[2];
        if constexpr (F8) {
#pragma unroll
          for (int r = 0; r < 16; ++r) Pf[r >> 3][r & 7] = (_Float16)e[r];
        } else
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
          u32x4_t hw, lw;
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            uint32_t hi, lo;
            at_split(e[8 * k2 + 2 * q], e[8 * k2 + 2 * q + 1], hi, lo);
            hw[q] = hi;
            lw[q] = lo;
          }
          Ph[k2] = __builtin_bit_cast(bf16x8, hw);
          Pl[k2] = __builtin_bit_cast(bf16x8, lw);
        }

        // O^T += V^T P^T: A = V^T from LDS by transposing reads (lane: column 32 dt + l32, keys
        // 16 ks + 4 h + 0..3 and 16 ks + 8 + 4 h + 0..3, the order P holds them in)
        const uint32_t set_at = lds_at(vset) + (uint32_t)(wave * Set::WAVE);
        if constexpr (F8) {
          // the 16 lanes of a group read 8 rows x 16 bytes: lane i row i / 2 of the order above,
          // bytes 8 (i % 2) of the group's chunk 2 dt + (group % 2), swizzled by the row
          const int i2 = (lane & 15) >> 1, key = (i2 & 3) + 4 * h + 8 * (i2 >> 2);
          const uint32_t at = set_at + (uint32_t)(256 * key + 16 * (((lane >> 4) & 1) ^ key) + 8 * (lane & 1));
          const float ratio[2] = {at_ratio(C.vs[0], v_ref), at_ratio(C.vs[1], v_ref)};
          i32x2_t v[16];   // column tile i / 2, keys 16 (i % 2) ..
          pg_read_codes(at, v);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const f16x8 vA = at_f16((uint32_t)v[i].x, (uint32_t)v[i].y, ratio[i & 1]);
            O[i >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vA, Pf[i & 1], O[i >> 1], 0, 0, 0);
          }
        } else {
          const int x = 4 * h + ((lane & 15) >> 2);
          const uint32_t at = set_at + (uint32_t)((x >> 1) * Set::PAIR + (x & 1) * (AT_D * 2) +
                                                  32 * ((lane >> 4) & 1) + 8 * (lane & 3));
#pragma unroll
          for (int two = 0; two < 4; ++two) {
            u32x2_t v[8];   // column tile 2 two + i / 4, keys 16 (i / 2 % 2) + 8 (i % 2) ..
            pg_read_rows<Set::PAIR>(at + 128 * two, v);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const bf16x8 vA = __builtin_bit_cast(bf16x8, u32x4_t{v[2 * i].x, v[2 * i].y, v[2 * i + 1].x, v[2 * i + 1].y});
              const int dt = 2 * two + (i >> 1);
              O[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vA, Ph[i & 1], O[dt], 0, 0, 0);
              O[dt] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vA, Pl[i & 1], O[dt], 0, 0, 0);
            }
          }
        }
      }

      if (seg_last) {
        // merge the four waves' (m, l, O) of this pair into the workgroup's piece: each wave dumps
        // its O straight from the accumulators, then every thread sums 16 columns of a row with
        // the waves' weights exp(m_w - M).  Up to 16 rows (few tokens have no more) go in one
        // turn, more in two turns of half the columns.
        const float lrow = l_s + __shfl_xor(l_s, 32, 64);
        aw_barrier();   // every wave is done reading this set
        if (h == 0) {
          mx[wave][l32] = m_ref;
          lx[wave][l32] = lrow;
          if (F8 && l32 == 0) vx[wave] = __int_as_float(v_ref);
        }
        float* part = a.ws + ((size_t)w + C.b * PH + C.ph) * AT_PART;
        float* dump = reinterpret_cast<float*>(F8 ? own_dump : vset);
        // columns D0 .. of the rows that the wave has, WIDE of them, then their sum
        auto turn = [&](auto first, auto wide) {
          constexpr int D0 = decltype(first)::value, WIDE = decltype(wide)::value;
          constexpr int ROWS = WIDE == AT_D ? 16 : AT_ROWS, OROW = WIDE + 4, TPR = AW_THREADS / ROWS;
          static_assert(AW_WAVES * ROWS * OROW * 4 <= PG_DUMP, "a turn fits the dump");
          if (l32 < rows) {
#pragma unroll
            for (int dt = 0; dt < WIDE / 32; ++dt)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const f32x16& o = O[D0 / 32 + dt];
                *reinterpret_cast<float4*>(dump + (wave * ROWS + l32) * OROW + 32 * dt + 8 * q + 4 * h) =
                    make_float4(o[4 * q], o[4 * q + 1], o[4 * q + 2], o[4 * q + 3]);
              }
          }
          aw_barrier();
          const int row = tid / TPR, c4 = 4 * (tid % TPR);
          if (row < rows) {
            float M = mx[0][row], Lsum = 0.f, wgt[AW_WAVES];
#pragma unroll
            for (int ww = 1; ww < AW_WAVES; ++ww) M = fmaxf(M, mx[ww][row]);
#pragma unroll
            for (int ww = 0; ww < AW_WAVES; ++ww) {
              const float mw = mx[ww][row];
              wgt[ww] = mw == -INFINITY ? 0.f : fast_exp2((mw - M) * a.cl2);
              Lsum += lx[ww][row] * wgt[ww];
              if constexpr (F8) wgt[ww] *= vx[ww];
            }
            if (D0 == 0 && c4 == 0) {
              part[row] = M;
              part[AT_ROWS + row] = Lsum;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int c = c4 + 4 * TPR * k;
              float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
              for (int ww = 0; ww < AW_WAVES; ++ww) {
                const float4 v = *reinterpret_cast<const float4*>(dump + (ww * ROWS + row) * OROW + c);
                acc.x += wgt[ww] * v.x; acc.y += wgt[ww] * v.y; acc.z += wgt[ww] * v.z; acc.w += wgt[ww] * v.w;
              }
              *reinterpret_cast<float4*>(part + 2 * AT_ROWS + row * AT_D + D0 + c) = acc;
            }
          }
          aw_barrier();   // the dump is read before it is overwritten (and the set refilled)
        };
        if (rows <= 16) {
          turn(std::integral_constant<int, 0>{}, std::integral_constant<int, AT_D>{});
        } else {
          turn(std::integral_constant<int, 0>{}, std::integral_constant<int, AT_D / 2>{});
          turn(std::integral_constant<int, AT_D / 2>{}, std::integral_constant<int, AT_D / 2>{});
        }
      }
      // The last block: nothing is to come.  (By hand: as a branch of the compiler's this is an edge
      // over which no V follows K, and its waits for K in the next block then wait for all.)
      asm volatile("s_cmp_lt_u32 %0, %1\n\ts_cbranch_scc1 1f\n\ts_endpgm\n1:" ::"s"(u + 1), "s"(u1) : "scc", "memory");
      // V of block u + 2 into this set
      issue_v(vset, X2);
      C = X1;
      X1 = X2;
      if (set && u + 4 - tbase >= 64) {   // the lanes' blocks are used up
        tbase = u + 1;
        look_up();
        look_up_scales();
        // (waited for here: else the compiler drains the loop's loads where it reads these)
        asm volatile("" : "+v"(tp[0]), "+v"(tp[1]), "+v"(tks[0]), "+v"(tks[1]), "+v"(tvs[0]), "+v"(tvs[1]));
      }
      X2 = unit(u + 3);
      if constexpr (F8) unit_scales(X2, u + 3);
    }
  }
}

// Merges the pieces of pair blockIdx.y for its rows 4 blockIdx.x .., a wave per row with 4 columns a
// lane, and applies the gate.  The pieces are those of workgroups wf .. wl of the table, in that
// order; the weights of 64 of them are formed in the lanes while the first columns are on their way.
__global__ __launch_bounds__(256) void attn_paged_combine_kernel(PagedArgs p) {
  const AttnArgs& a = p.a;
  const int r = 4 * blockIdx.x + (threadIdx.x >> 6), pair = blockIdx.y, lane = threadIdx.x & 63;
  const int PH = a.Hkv * a.qblocks;
  const int2 te = reinterpret_cast<const int2*>(a.ws + (size_t)(a.nw + a.B * PH) * AT_PART)[pair];
  const int b = pair / PH, ph = pair - b * PH, kvh = ph / a.qblocks;
  const int q0 = (ph - kvh * a.qblocks) * a.QB;
  const int i = (int)(((uint32_t)r * p.rep_mul) >> 16), h = kvh * a.n_rep + r - i * a.n_rep;
  if (i >= min(a.QB, a.T - q0)) return;
  const size_t bt = (size_t)b * a.T + q0 + i;
  uint2 gv = make_uint2(0, 0);
  if (a.gate) gv = *reinterpret_cast<const uint2*>(a.gate + bt * a.gate_row + (size_t)h * a.gate_head + 4 * lane);
  const int wf = te.x, np = wf < 0 ? 0 : te.y - wf + 1;
  const float* base = a.ws + ((size_t)max(wf, 0) + pair) * AT_PART;
  const float* col = base + 2 * AT_ROWS + r * AT_D + 4 * lane;
  constexpr int AHEAD = 6;
  float M = -INFINITY, l = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int c = 0; c < np; c += 64) {
    const int n = min(np - c, 64);
    const float* piece = base + (size_t)(c + min(lane, n - 1)) * AT_PART;
    float m = piece[r], ls = piece[AT_ROWS + r];
    float4 v[AHEAD];
#pragma unroll
    for (int s = 0; s < AHEAD; ++s)
      v[s] = *reinterpret_cast<const float4*>(col + (size_t)(c + min(s, n - 1)) * AT_PART);
    if (lane >= n) {
      m = -INFINITY;
      ls = 0.f;
    }
    float mn = m;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor(mn, o, 64));
    mn = fmaxf(mn, M);
    const float shrink = M == -INFINITY ? 0.f : fast_exp2((M - mn) * a.cl2);
    const float wgt = m == -INFINITY ? 0.f : fast_exp2((m - mn) * a.cl2);
    ls *= wgt;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o, 64);
    l = l * shrink + ls;
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] *= shrink;
    M = mn;
    for (int s = 0; s < n; s += AHEAD) {
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        if (s + e < n) {
          const float x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wgt), s + e));
          acc[0] += x * v[e].x; acc[1] += x * v[e].y; acc[2] += x * v[e].z; acc[3] += x * v[e].w;
        }
      }
      if (s + AHEAD < n) {
#pragma unroll
        for (int e = 0; e < AHEAD; ++e)
          v[e] = *reinterpret_cast<const float4*>(col + (size_t)(c + min(s + AHEAD + e, n - 1)) * AT_PART);
      }
    }
  }
  at_store4(a.out + (bt * a.Hq + h) * AT_D + 4 * lane, acc, l == 0.f ? 0.f : 1.f / l, a.gate != nullptr, gv);
}

}  // namespace lollm

using namespace lollm;

// Workspace of a call: the split-K's pieces, or the parts' of query tiles.
static long long paged_ws_bytes(int B, int T, int Hkv, int n_rep, int qblocks, int nw, int groups, int parts) {
  const long long n = groups ? attn_parts_bytes(B, T, Hkv, n_rep, parts) : attn_ws_bytes(nw, (long long)B * Hkv * qblocks);
  return n > 16 ? n : 16;
}

LOLLM_API long long lollm_attn_paged_workspace_bytes(int B, int T, int Hq, int Hkv, int D, int kv_dtype,
                                                     int grid) {
  int n_rep, QB, qblocks, parts = 1;
  if (attn_geometry(B, T, Hq, Hkv, D, 1, &n_rep, &QB, &qblocks)) return -1;
  const int nw = attn_grid(grid);
  if (nw <= 0 || nw > 1024 || (kv_dtype != LOLLM_BF16 && kv_dtype != LOLLM_F8)) return -1;
  const int groups = grid == 0 ? attn_paged_groups(B, T, Hkv, n_rep, nw, kv_dtype == LOLLM_F8, &parts) : 0;
  return paged_ws_bytes(B, T, Hkv, n_rep, qblocks, nw, groups, parts);
}

LOLLM_API int lollm_attn_paged(const void* q, const void* k_pages, const void* v_pages,
                               const float* k_scale, const float* v_scale, int kv_dtype,
                               const int32_t* table, long long table_stride, int table_width, int n_pages,
                               int page, const int32_t* kv_len, const void* gate, long long gate_row,
                               int gate_head, void* out, void* workspace, long long workspace_bytes, int B,
                               int T, int Hq, int Hkv, int D, int grid, float scale, void* stream) {
  if (!q || !k_pages || !v_pages || !table || !kv_len || !out) return LOLLM_EINVAL;
  if (kv_dtype != LOLLM_BF16 && kv_dtype != LOLLM_F8) return LOLLM_EUNSUPPORTED;
  const bool f8 = kv_dtype == LOLLM_F8;
  if (f8 && (!k_scale || !v_scale)) return LOLLM_EINVAL;
  if (table_width <= 0 || n_pages <= 0 || table_stride < table_width) return LOLLM_EINVAL;
  const int pshift = attn_page_shift(page);
  if (pshift < 0) return LOLLM_EUNSUPPORTED;
  const long long rows = (long long)table_width << pshift;
  if (rows > 0x7fffff00LL) return LOLLM_EUNSUPPORTED;
  int n_rep, QB, qblocks;
  int rc = attn_geometry(B, T, Hq, Hkv, D, (int)rows, &n_rep, &QB, &qblocks);
  if (rc) return rc;
  if (Hkv > 65535) return LOLLM_EUNSUPPORTED;        // 32-bit offsets in a query block's tokens
  if (!(scale > 0.f) || !(scale < INFINITY)) return LOLLM_EINVAL;   // the maxima are of unscaled scores
  if (grid < 0 || grid > 1024) return LOLLM_EINVAL;  // pieces per pair <= combine table
  if (gate && (gate_head < D || gate_row < (Hq - 1LL) * gate_head + D)) return LOLLM_EINVAL;
  if (gate && (gate_row % 8 || gate_head % 8)) return LOLLM_EINVAL;
  const long long pairs = (long long)B * Hkv * qblocks;
  const int nw = attn_grid(grid);
  if (nw <= 0 || nw > 1024) return LOLLM_EUNSUPPORTED;
  int parts = 1;
  const int groups = grid == 0 ? attn_paged_groups(B, T, Hkv, n_rep, nw, f8, &parts) : 0;
  if (!groups && pairs > 65535) return LOLLM_EUNSUPPORTED;                        // the combine's grid
  if (!groups && pairs * (rows / AT_BLOCK + 1) > 0x7fffffffLL) return LOLLM_EUNSUPPORTED;   // 32-bit block numbers
  if (!workspace || workspace_bytes < paged_ws_bytes(B, T, Hkv, n_rep, qblocks, nw, groups, parts)) return LOLLM_EINVAL;
  PagedArgs p;
  AttnArgs& a = p.a;
  a.q = (const uint16_t*)q; a.kc = (const uint16_t*)k_pages; a.vc = (const uint16_t*)v_pages;
  a.kv_len = kv_len; a.gate = (const uint16_t*)gate; a.out = (uint16_t*)out;
  a.ws = (float*)workspace; a.seq_stride = 0; a.head_stride = 0;
  a.B = B; a.T = T; a.Hq = Hq; a.Hkv = Hkv; a.n_rep = n_rep; a.QB = QB; a.qblocks = qblocks;
  a.max_len = (int)rows; a.nw = nw;
  a.cl2 = scale * 1.4426950408889634f;
  a.gate_row = gate_row; a.gate_head = gate_head;
  p.table = table; p.ks = k_scale; p.vs = v_scale; p.table_stride = table_stride;
  p.n_pages = n_pages; p.pshift = pshift;
  p.rep_mul = (uint32_t)((65536 + n_rep - 1) / n_rep);
  hipStream_t st = (hipStream_t)stream;
  if (groups) return attn_prefill_launch(a, groups, st, &p, parts);
  if (f8)
    hipLaunchKernelGGL(attn_paged_kernel<true>, dim3(nw), dim3(AW_THREADS), 0, st, p);
  else
    hipLaunchKernelGGL(attn_paged_kernel<false>, dim3(nw), dim3(AW_THREADS), 0, st, p);
  if ((rc = launch_status())) return rc;
  hipLaunchKernelGGL(attn_paged_combine_kernel, dim3((n_rep * QB + 3) / 4, (unsigned)pairs), dim3(256), 0, st, p);
  return launch_status();
}
