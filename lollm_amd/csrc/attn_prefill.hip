// Gated GQA attention of a long call (prefill: many new positions per sequence), gfx950.
//
// Same math and operands as attn_verify.hip (src/qwen3_5/blocks.py:226-235 +
// src/attention.py:43-51: offset-causal GQA over the cache, output o * sigmoid(gate)),
// for calls whose query rows alone fill the chip, where splitting keys between workgroups
// (and the fp32 pieces and the second launch that go with it) buys nothing; and for long calls
// over pages at any number of tiles.
//
// Tile.  A workgroup owns 128 RG query rows of one (sequence, KV head): the n_rep query
// heads x QB consecutive positions, packed position-major (row r = position r / n_rep,
// head r % n_rep), so every K / V byte staged serves all the heads that share it and a
// tile's causal edge is only QB positions wide.  It walks the keys in blocks of 32: K and
// V rows arrive by LDS DMA (three sets each, K three and V two blocks ahead, one barrier
// per block) and are read by all four waves; wave w owns rows 32 RG w .. of the tile with
// its Q in registers and its O^T in accumulator registers.
//
// Precision.  One running maximum serves a row where the split-K kernels have one per wave and
// piece, whose largest weights are 1 and lose nothing as bf16; so weights enter the product with
// V as hi + lo bf16 (16 bits) and the row sum as they are, fp32.  Relative error against 64 bits
// (2 x 1999 tokens, normal q, k, v): split-K 2.07e-3, weights in bf16 here 2.12e-3, hi + lo
// 1.66e-3, which is the output's own rounding to bf16.  It costs a third of the products: 185 ->
// 221 us.
//
// What bounds it: operand reads and the softmax beside the products.  A 32x32x16 MFMA
// (32 cycles) takes a 1 KB operand from LDS, and the four waves of a CU then need 128 B per
// cycle, the LDS peak.  With RG = 2 a wave reuses each K / V operand for two row groups and
// needs half of that, at one wave per SIMD: O^T of 64 rows takes all 256 accumulator
// registers, Q half of the vector registers.  A lone wave overlaps nothing by itself, so the
// exponentials of block j + 1 are placed between the products of V with block j.
//
// Measured (us, causal, T = kv length, split-K kernels / RG = 1 / RG = 2): 2 x 1999,
// 32 q / 4 kv heads 1020 / 247 / 222 (591 TFLOP/s); 1 x 4096 1822 / 407 / 372 (740 TFLOP/s);
// 3 x 1500 1110 / 216 / 217; 32 x 128 over 1128 keys 903 / 260 / 244.
//
// Pages (attn_paged.hip).  A block's rows lie in one page, or two of 16 rows; a wave's eight in one,
// which a descriptor of their own covers.  Page ids and scales are the same for every lane and come
// through the scalar cache, a block ahead of the loads that need them.  8 bits: K becomes bf16 and V
// fp16 as they are read, and weights are fp16, one product in the place of two.  Tiles of 128 rows
// only, where they can two workgroups a CU: 256 registers a wave, for which bf16 pages leave four of
// Q's 16 operands in LDS and have two sets of rows (80 KB), and O leaves through the sets.  2 x 1999
// tokens: bf16 pages 223 us (588 TFLOP/s; one workgroup of 256 rows a CU 240, slabs that way 219), 8
// bits 189 (694; 183 and 197 while a row's reference had the weight 1, at_f16).  1024 tokens over 9024
// keys: 383 us (745; 433), 8 bits 317 (901; 412).  What
// bounds it is the instructions beside the products: 240 of the VALU and 80 of the scalar unit a
// block and wave of 8-bit pages, half of the former conversions, beside 32 products of 32 cycles.
// Where tiles are fewer than the chip holds, a tile's keys are dealt out to `parts` workgroups, whose
// pieces a second kernel merges (512 tokens over 8289 keys, 128 tiles in four parts: 203 us, of
// which the merge 15; 418 on the split-K kernel).
//
// Rows of K and V are 512 bytes in LDS with no padding (the DMA writes 1 KB runs); the
// 16-byte chunk c of row r sits at c ^ (r & 15) for K and c ^ (2 (r & 7)) for V, so the
// operand reads (32 rows at one chunk; 8 rows x 4 chunks for the transposing V read) touch
// every bank equally.
#include <type_traits>

#include "attn_common.h"

namespace lollm {

constexpr int AP_WAVES = 4;
constexpr int AP_MIN_T = 16;                   // new positions per sequence
constexpr int AP_FEW_ROWS = 64;                // tokens of a call that keeps the split-K kernels
constexpr int AP_KEYS = 32;                    // keys per block
constexpr int AP_AHEAD = 3;                    // operands read ahead of their products
constexpr int AP_PART_BLOCKS = 8;              // blocks of a part of a tile's keys at least
constexpr int AP_MAX_PARTS = 64;
constexpr int AP_PIECE = 2 * 128 + 128 * AT_D; // floats: maxima, sums and O of a part of a 128-row tile

// Where the keys are: AP_ROWS one slab per (sequence, KV head); AP_PAGES, AP_PAGES8 pages that a
// table names (attn_paged.hip), in bf16 or as e4m3 codes with scales.
enum { AP_ROWS, AP_PAGES, AP_PAGES8 };

struct ApArgs {
  const uint16_t* q;       // (B, T, Hq, D)
  const uint16_t* kc;      // K cache
  const uint16_t* vc;      // V cache
  const int32_t* kv_len;   // (B) keys per sequence, the T new ones included
  const uint16_t* gate;    // (B, T, Hq, D), strided, or null
  uint16_t* out;           // (B, T, Hq * D)
  long long seq_stride, head_stride;
  int B, T, Hq, Hkv, n_rep, QB, qtiles, max_len;
  const int32_t* table;    // pages: (B, table_stride)
  const float* ks;         // 8-bit pages: (n_pages, Hkv) scales
  const float* vs;
  long long table_stride, gate_row;
  float* ws;               // pieces of tiles whose keys are dealt out to several workgroups
  int gate_head, n_pages, pshift, parts;
  uint32_t rep_mul;        // ceil(2^16 / n_rep): r / n_rep = r * rep_mul >> 16 for r < 256
  float cl2;
};

// S += K Q^T with S in vector registers.  O of 64 rows takes all 256 accumulator registers,
// and the compiler, which gives every MFMA of a kernel one register class, would move parts of
// O out and back for each S.  (The nop: a VALU write may precede; the matrix pipe is busy for
// longer than that with the previous product.)
__device__ __forceinline__ void ap_mfma_first(f32x16& s, bf16x8 k, bf16x8 q) {
  asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, 0" : "=&v"(s) : "v"(k), "v"(q));
}
__device__ __forceinline__ void ap_mfma(f32x16& s, bf16x8 k, bf16x8 q) {
  asm("s_nop 1\n\tv_mfma_f32_32x32x16_bf16 %0, %1, %2, %0" : "+v"(s) : "v"(k), "v"(q));
}
// the wait states between the last product and the first VALU access of its result
__device__ __forceinline__ void ap_mfma_done(f32x16& s) { asm volatile("s_nop 15\n\ts_nop 7" : "+v"(s)); }

__device__ __forceinline__ int ap_div(int r, uint32_t mul) { return (int)(((uint32_t)r * mul) >> 16); }

// A value that every lane loads from the same address, through the scalar cache: nothing that the
// kernel writes is read so.
template <typename T>
__device__ __forceinline__ T ap_sload(const T* p, long long i) {
  return ((const __attribute__((address_space(4))) T*)p)[i];
}

// SETS: of K and V rows in LDS.  Two for bf16 pages where two workgroups share a CU (K two blocks
// ahead, V one), else three.
template <int RG, int KV, int SETS>
__global__ __launch_bounds__(64 * AP_WAVES, KV == AP_PAGES8 || SETS == 2 ? 2 : 1) void attn_prefill_kernel(ApArgs a) {
  constexpr bool F8 = KV == AP_PAGES8;
  constexpr int ROW = F8 ? AT_D : AT_D * 2;      // bytes of a key's row
  constexpr int AP_SET = AP_KEYS * ROW;          // K or V rows of a block
  // separate arrays, so that the reads of one set are not ordered after the DMA into another
  constexpr int AHEAD = SETS == 2 ? 2 : AP_AHEAD;
  constexpr int THIRD = SETS == 3 ? AP_SET : 16;
  __shared__ __attribute__((aligned(16))) unsigned char ks0[AP_SET], ks1[AP_SET], ks2[THIRD];
  __shared__ __attribute__((aligned(16))) unsigned char vs0[AP_SET], vs1[AP_SET], vs2[THIRD];

  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l32 = lane & 31, h = lane >> 5;
  // the longest tiles first (they end last), (sequence, KV head) fastest: with a multiple of
  // 8 pairs, one pair's tiles all run on one XCD and share its L2
  const int pairs = a.B * a.Hkv;
  constexpr bool PARTS = KV != AP_ROWS;   // a tile's keys may go to a.parts workgroups
  const int turn_ = blockIdx.x / pairs, pair = blockIdx.x % pairs;
  const int part = PARTS ? turn_ % a.parts : 0;
  const int qt = a.qtiles - 1 - (PARTS ? turn_ / a.parts : turn_);
  const int b = pair / a.Hkv, kvh = pair % a.Hkv;
  const int q0 = qt * a.QB, QB = min(a.QB, a.T - q0);
  const int L = min(max(a.kv_len[b], 0), a.max_len);
  const int p0 = L - a.T + q0;                       // position of the tile's first query
  const int keys = min(max(p0 + QB, 0), L);          // keys any row of the tile sees
  const int nall = (keys + AP_KEYS - 1) / AP_KEYS;

  // The blocks of this workgroup: from the first page that is mapped on (a window leaves none
  // before it), and of these one of `parts` equal parts.  Parts of 8 blocks (10 us) or more, from
  // 24 blocks on: what a division saves has to pay for the pieces and their merge, some 10 us.
  int j0 = 0, nblk = nall, parts = 1;
  if constexpr (KV != AP_ROWS) {
    const int32_t* row = a.table + b * a.table_stride;
    const int entries = (int)(((long long)keys + (1 << a.pshift) - 1) >> a.pshift);
    if (entries > 0 && (uint32_t)ap_sload(row, 0) >= (uint32_t)a.n_pages) {
      int e = entries;
      for (int at = 0; at < entries; at += 64) {
        const bool there = at + lane < entries && (uint32_t)row[at + lane] < (uint32_t)a.n_pages;
        const uint64_t m = __ballot(there);
        if (m) {
          e = at + __builtin_ctzll(m);
          break;
        }
      }
      j0 = min((int)(((long long)e << a.pshift) / AP_KEYS), nall);
    }
    if constexpr (PARTS) {
      const int n = nall - j0;
      parts = n < 3 * AP_PART_BLOCKS ? 1 : min(a.parts, n / AP_PART_BLOCKS);
      if (part >= parts) return;
      nblk = j0 + (int)((long long)n * (part + 1) / parts);
      j0 += (int)((long long)n * part / parts);
    }
  }
  const int Lend = (int)min((long long)L, (long long)nblk * AP_KEYS);

  // Loads of a block: wave w brings rows 8 w .. 8 w + 7 of K and of V, two rows (1 KB) per
  // instruction; the lane's source chunk undoes the swizzle of the place it writes.  Rows
  // past the sequence's end touch no memory.
  // Pages: the wave's 8 rows of a block lie in one page, which a descriptor of their own covers
  // (none of its bytes where the page is unmapped: zeros).  Page ids come through the scalar
  // cache a block before they are needed, and two bits a block say which halves are mapped.
  constexpr int WR = AP_KEYS / AP_WAVES;
  static_assert(WR == 8, "the swizzles below take the row of the wave's 8");
  const size_t cbase = KV == AP_ROWS ? (size_t)b * a.seq_stride + (size_t)kvh * a.head_stride : 0;
  const __amdgpu_buffer_rsrc_t krs = buf_rsrc(a.kc + cbase, KV == AP_ROWS ? (uint32_t)L * (AT_D * 2) : 0u);
  const __amdgpu_buffer_rsrc_t vrs = buf_rsrc(a.vc + cbase, KV == AP_ROWS ? (uint32_t)L * (AT_D * 2) : 0u);
  // page of keys 16 g .. of block j, -1: unmapped or past this workgroup's blocks
  auto entry = [&](int j, int g) {   // (no branch: O lives in all of them)
    const uint32_t key = (uint32_t)(j * AP_KEYS + 16 * g);
    return ap_sload(a.table, b * a.table_stride + (min(key, (uint32_t)max(L - 1, 0)) >> a.pshift));
  };
  auto page_of = [&](int id, int j, int g) {
    return (uint32_t)(j * AP_KEYS + 16 * g) < (uint32_t)Lend && (uint32_t)id < (uint32_t)a.n_pages ? id : -1;
  };
  struct Rows { long long at; uint32_t bytes; };   // the wave's rows of a block, the same in both pools
  auto rows_of = [&](int id, int j) {
    const int key = j * AP_KEYS + WR * wave;
    const long long row = (((long long)max(id, 0) * a.Hkv + kvh) << a.pshift) + (key & ((1 << a.pshift) - 1));
    return Rows{row * ROW, id >= 0 ? (uint32_t)(min(max(L - key, 0), WR) * ROW) : 0u};
  };
  // 8 bits: four rows a load, the 16-byte chunk c of row r at c ^ (r & 15)
  const uint32_t l8 = 256u * (lane >> 4) + 16u * ((lane & 15) ^ (8 * (wave & 1) + (lane >> 4)));
  auto issue_page = [&](unsigned char* d, const uint16_t* pool, const Rows& r, uint32_t x, uint32_t swz) {
    asm volatile("" : "+v"(x));
    const __amdgpu_buffer_rsrc_t rs = buf_rsrc((const unsigned char*)pool + r.at, r.bytes);
    // (the instruction's own offset moves both the row's address and its place)
    auto load = [&](auto at) {
      constexpr int I = decltype(at)::value;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_void_t*)(d + ROW * WR * wave), 16, x ^ (swz * I), 0, 1024 * I, 0);
    };
    load(std::integral_constant<int, 0>{});
    load(std::integral_constant<int, 1>{});
    if constexpr (!F8) {
      load(std::integral_constant<int, 2>{});
      load(std::integral_constant<int, 3>{});
    }
  };
  // (row = 8 w + 2 i + h: its swizzle is the lane's part ^ that of 2 i; one register per cache,
  // the rest formed per load -- registers are what this kernel is short of)
  const uint32_t rl = (uint32_t)(WR * wave + h) * (AT_D * 2);
  const uint32_t kl = 16u * (l32 ^ (8 * (wave & 1) + h)), vl = 16u * (l32 ^ (2 * h));
  auto issue_k = [&](unsigned char* kd, int j) {
    uint32_t x = kl;
    asm volatile("" : "+v"(x));
    const uint32_t blk = (uint32_t)(j * AP_KEYS) * (AT_D * 2) + rl;
#pragma unroll
    for (int i = 0; i < WR / 2; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(krs, (lds_void_t*)(kd + 512 * WR * wave + 1024 * i), 16,
                                               blk + 1024u * i + (x ^ (32u * i)), 0, 0, 0);
  };
  auto issue_v = [&](unsigned char* vd, int j) {
    uint32_t x = vl;
    asm volatile("" : "+v"(x));
    const uint32_t blk = (uint32_t)(j * AP_KEYS) * (AT_D * 2) + rl;
#pragma unroll
    for (int i = 0; i < WR / 2; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(vrs, (lds_void_t*)(vd + 512 * WR * wave + 1024 * i), 16,
                                               blk + 1024u * i + (x ^ (64u * i)), 0, 0, 0);
  };
  auto load_k = [&](unsigned char* kd, const Rows& r, int j) {
    if constexpr (KV == AP_ROWS) issue_k(kd, j);
    else if constexpr (F8) issue_page(kd, a.kc, r, l8, 64u);
    else issue_page(kd, a.kc, r, kl + (uint32_t)(ROW * h), 32u);
  };
  auto load_v = [&](unsigned char* vd, const Rows& r, int j) {
    if constexpr (KV == AP_ROWS) issue_v(vd, j);
    else if constexpr (F8) issue_page(vd, a.vc, r, l8, 64u);
    else issue_page(vd, a.vc, r, vl + (uint32_t)(ROW * h), 64u);
  };
  // this wave's loads up to the last N have landed and its LDS accesses are complete, then
  // every wave's
#define AP_BARRIER(N) asm volatile("s_waitcnt vmcnt(" #N ") lgkmcnt(0)\n\ts_barrier" ::: "memory")

  // Finite contents everywhere: rows past a sequence's end are never loaded, and P = 0
  // multiplies what they hold.
  for (int i = tid; i < AP_SET / 16; i += 64 * AP_WAVES) {
    *reinterpret_cast<uint4*>(vs0 + 16 * i) = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(vs1 + 16 * i) = make_uint4(0, 0, 0, 0);
    if constexpr (SETS == 3) *reinterpret_cast<uint4*>(vs2 + 16 * i) = make_uint4(0, 0, 0, 0);
  }
  // Q's last QL operands wait in LDS where the registers of two waves a SIMD do not hold them.
  constexpr int QL = SETS == 2 ? 4 : 0;
  __shared__ __attribute__((aligned(16))) unsigned char qlate[QL ? AP_WAVES * QL * 1024 : 16];
  unsigned char* const ql = qlate + (QL ? 1024 * QL * wave + 16 * lane : 0);
  // this lane's rows: position q0 + qi, query head kvh n_rep + hr
  int qpos[RG];
  bf16x8 Q[RG][16];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    const int r = 32 * (RG * wave + rg) + l32, qi = ap_div(r, a.rep_mul), hr = r - qi * a.n_rep;
    const bool live = qi < QB;
    qpos[rg] = live ? p0 + qi : -1;
    const uint16_t* src = a.q + (((size_t)b * a.T + q0 + (live ? qi : 0)) * a.Hq + kvh * a.n_rep + hr) * AT_D;
#pragma unroll
    for (int ks = 0; ks < 16; ++ks)   // (8 bits: a lane's 16 codes of K are two k-steps)
      Q[rg][ks] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_t*>(
                                                 src + (F8 ? 32 * (ks >> 1) + 16 * h + 8 * (ks & 1) : 16 * ks + 8 * h)));
#pragma unroll
    for (int i = 0; i < QL; ++i) *reinterpret_cast<bf16x8*>(ql + 1024 * i) = Q[rg][16 - QL + i];
  }
  // Pages (two halves of a block): of blocks j + 1, j + 2 and j + 3 before step j, and the entry of
  // block j + 4; the scales of block j + 1's K and of block j's V.  What a step asks the scalar
  // cache for, the next one uses.
  // the half of a block that holds the wave's rows (a choice: an index is a search of all of them)
  auto mine = [&](const int (&id)[2]) { return wave >> 1 ? id[1] : id[0]; };
  int pg[3][2], raw[2] = {-1, -1}, pg0[2] = {-1, -1};
  float ksc[2] = {0.f, 0.f};
  int vsc[2] = {0, 0}, v_ref = 0;      // (bits; v_ref: the units of O, at_f16)
  constexpr float LAG = F8 ? AT_F16_LAG : 16.f, UP = F8 ? AT_F16_UP : 0.f;
  auto scale_at = [&](const float* sc, int id) {
    const float s = ap_sload(sc, (long long)max(id, 0) * a.Hkv + kvh);
    return id >= 0 ? s : 0.f;
  };
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    pg[0][g] = pg[1][g] = pg[2][g] = -1;
    if constexpr (KV != AP_ROWS) {
      pg0[g] = page_of(entry(j0, g), j0, g);
#pragma unroll
      for (int n = 0; n < 3; ++n) pg[n][g] = page_of(entry(j0 + 1 + n, g), j0 + 1 + n, g);
      raw[g] = entry(j0 + 4, g);
    }
  }
  auto both = [&](const int (&id)[2]) {   // mapped halves
    return KV == AP_ROWS ? 3u : (id[0] >= 0 ? 1u : 0u) | (id[1] >= 0 ? 2u : 0u);
  };
  AP_BARRIER(0);   // the zeroed sets, before any DMA into them (and Q: the counts below are the DMA's)
  const Rows first = rows_of(mine(pg0), j0), second = rows_of(mine(pg[0]), j0 + 1);
  Rows coming = rows_of(mine(pg[1]), j0 + 2);   // of block j + 2 before step j
  load_k(ks0, first, j0);
  load_k(ks1, second, j0 + 1);
  load_v(vs0, first, j0);
  if constexpr (SETS == 3) {
    load_k(ks2, coming, j0 + 2);
    load_v(vs1, second, j0 + 1);
  }

  // the positions this wave's rows span: the key blocks it sees, and which need a mask
  const int wq0 = ap_div(32 * RG * wave, a.rep_mul);
  const int wq1 = min(ap_div(32 * RG * wave + 32 * RG - 1, a.rep_mul), QB - 1);
  const int wmin = p0 + wq0, wmax = wq0 < QB ? p0 + wq1 : -1;
  const int wblk = min(wmax < 0 ? 0 : wmax / AP_KEYS + 1, KV == AP_ROWS ? INT32_MAX : nblk);

  // LDS offsets of the operand reads: K row l32 at chunk 2 ks + h, V row x = 4 h + (lane % 16) / 4
  // at chunk 4 dt + 2 ((lane / 16) % 2) + (lane % 4) / 2; the k-step and the column tile
  // enter by xor.  8 bits: V row 4 h + (r & 3) + 8 (r >> 2), r = (lane % 16) / 2, at chunk
  // 2 dt + (lane / 16) % 2
  const int ko = l32 * ROW + 16 * (h ^ (l32 & 15));
  const int vxr = F8 ? 4 * h + ((lane & 7) >> 1) + (lane & 8) : 4 * h + ((lane & 15) >> 2);
  const int vo = F8 ? vxr * ROW + 16 * (((lane >> 4) & 1) ^ vxr) + 8 * (lane & 1)
                    : vxr * (AT_D * 2) + 16 * ((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ (2 * vxr)) + 8 * (lane & 1);

  f32x16 O[RG][8];   // O^T: 32 columns x 32 rows per tile; lane's row = l32
  float m_ref[RG], l_s[RG];
  // exp of the block whose V comes next: hi and lo bf16, or fp16
  bf16x8 P[RG][2], Pl[RG][2];
  f16x8 Pf[RG][2];
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    m_ref[rg] = -INFINITY;
    l_s[rg] = 0.f;
#pragma unroll
    for (int dt = 0; dt < 8; ++dt)
#pragma unroll
      for (int r = 0; r < 16; ++r) O[rg][dt][r] = 0.f;
  }

  f32x16 S[RG];
  float base[RG], alpha[RG];
  bool moved;
  // S^T (32 keys x 32 rows) = K Q^T of block j, masked, and the row maxima
  auto scores = [&](const unsigned char* kset, int j, uint32_t there) {
    int kof = ko;
    asm volatile("" : "+v"(kof));
    if constexpr (F8) {
      const float sc = l32 < 16 ? ksc[0] : ksc[1];   // (0, an exponent like any, where K is masked)
      u32x4_t kw[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) kw[i] = *reinterpret_cast<const u32x4_t*>(kset + (kof ^ (32 * i)));
#pragma unroll
      for (int ks = 0; ks < 16; ++ks) {
        const u32x4_t c = kw[(ks >> 1) & 1];
        const bf16x8 kf = ks & 1 ? at_bf16(c.z, c.w, sc) : at_bf16(c.x, c.y, sc);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg)
          if (ks == 0) ap_mfma_first(S[rg], kf, Q[rg][0]); else ap_mfma(S[rg], kf, Q[rg][ks]);
        const int kn = (ks >> 1) + 2;
        if ((ks & 1) && kn < 8) kw[kn & 1] = *reinterpret_cast<const u32x4_t*>(kset + (kof ^ (32 * kn)));
        __builtin_amdgcn_sched_barrier(0);
      }
    } else {
    bf16x8 kf[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      kf[i] = *reinterpret_cast<const bf16x8*>(kset + (kof ^ (32 * (i & 7))) + 256 * (i >> 3));
    bf16x8 qn;
#pragma unroll
    for (int ks = 0; ks < 16; ++ks) {
      const bf16x8 qv = qn;
      if (QL && ks + 1 >= 16 - QL && ks + 1 < 16) qn = *reinterpret_cast<const bf16x8*>(ql + 1024 * (ks + 1 - (16 - QL)));
#pragma unroll
      for (int rg = 0; rg < RG; ++rg)
        if (ks == 0) ap_mfma_first(S[rg], kf[0], Q[rg][0]);
        else ap_mfma(S[rg], kf[ks % AHEAD], QL && ks >= 16 - QL ? qv : Q[rg][ks]);
      const int kn = ks + AHEAD;
      if (QL && kn == 8) asm volatile("" : "+v"(kof));   // (or all 8 addresses wait in registers)
      if (kn < 16)
        kf[ks % AHEAD] = *reinterpret_cast<const bf16x8*>(kset + (kof ^ (32 * (kn & 7))) + 256 * (kn >> 3));
      __builtin_amdgcn_sched_barrier(0);   // no more operands ahead than the registers hold
    }
    }
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) ap_mfma_done(S[rg]);
    const int key0 = j * AP_KEYS;
    if (key0 + AP_KEYS - 1 > wmin || (KV != AP_ROWS && there != 3)) {   // acc r holds key 8 (r / 4) + 4 h + r % 4
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const int lim = qpos[rg] - key0 - 4 * h;
#pragma unroll
        for (int r = 0; r < 16; ++r)
          S[rg][r] = 8 * (r >> 2) + (r & 3) <= (KV == AP_ROWS || there & (r < 8 ? 1u : 2u) ? lim : -1) ? S[rg][r] : -INFINITY;
      }
    }
    bool any = false;
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      float bm = -INFINITY;
#pragma unroll
      for (int r = 0; r < 16; ++r) bm = fmaxf(bm, S[rg][r]);
      const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(bm), __float_as_uint(bm), false, false);
      bm = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1]));
      // the reference max moves (and l, O are rescaled) only when a row's block max exceeds it
      // by more than LAG in the exponent: attn_verify's rule, each row's own decision
      const bool big = (bm - m_ref[rg]) * a.cl2 > LAG;
      // (8 bits, whose LAG is small: with one row every row moves that can, as all of O is rescaled
      // anyway; alone 195 us for 2 x 1999, so 185)
      const bool move = F8 ? __ballot(big) != 0 && bm > m_ref[rg] : big;
      const float mn = move ? fmaxf(m_ref[rg], bm) : m_ref[rg];
      alpha[rg] = (!move || mn == -INFINITY) ? 1.f : fast_exp2((m_ref[rg] - mn) * a.cl2);
      m_ref[rg] = mn;
      l_s[rg] *= alpha[rg];
      base[rg] = mn == -INFINITY ? 0.f : mn * a.cl2 - UP;
      any = any || big;
    }
    moved = __builtin_amdgcn_readfirstlane((int)(__ballot(any) != 0)) != 0;
  };
  // (factor: of the units of O, by which the next block's V counts)
  auto rescale = [&](float factor, bool units) {
    if (moved || units) {
#pragma unroll
      for (int rg = 0; rg < RG; ++rg)
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
          // (O stays in accumulator registers but for the tile at hand: without the pins the
          // compiler copies all of it to vector registers around this branch)
          asm volatile("" : "+a"(O[rg][dt]));
          O[rg][dt] *= F8 ? alpha[rg] * factor : alpha[rg];
          asm volatile("" : "+a"(O[rg][dt]));
          __builtin_amdgcn_sched_barrier(0);
        }
    }
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int dt = 0; dt < 8; ++dt) asm volatile("" : "+a"(O[rg][dt]));
  };
  // One block: scores of block j + 1, then O^T += V^T P^T of block j with the exponentials of
  // block j + 1 between its products (the matrix pipe is busy 32 cycles per product, the
  // wave's VALU work of one product about as long).  Past the wave's last block the scores
  // are all masked.
  auto step = [&](const unsigned char* knext, const unsigned char* vset, int j, const int (&v_coming)[2]) {
    if (j >= wblk) return;
    scores(knext, j + 1, both(pg[0]));
    int vof = vo;
    asm volatile("" : "+v"(vof));
    auto read_v = [&](int n) {   // operand n = 2 dt + k2, by transposing reads (attn_verify's key order)
      const int dt = n >> 1, k2 = n & 1;
      if constexpr (F8) {   // 8 codes, converted when their product comes
        const i32x2_t v = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
            (lds_i32x2_t*)(vset + (vof ^ (32 * dt)) + 16 * ROW * k2));
        return __builtin_bit_cast(u32x2_t, v);
      } else {
      const unsigned char* vp = vset + (vof ^ (64 * (dt & 3))) + 256 * (dt >> 2) + 16 * (AT_D * 2) * k2;
      const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)vp);
      const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t*)(vp + 8 * (AT_D * 2)));
      const u32x2_t w0 = __builtin_bit_cast(u32x2_t, v0), w1 = __builtin_bit_cast(u32x2_t, v1);
      return __builtin_bit_cast(bf16x8, u32x4_t{w0.x, w0.y, w1.x, w1.y});
      }
    };
    decltype(read_v(0)) vf[AHEAD];
    u32x4_t Pn[RG][2], Pm[RG][2];
    float pe[RG];
    const float ratio[2] = {at_ratio(vsc[0], v_ref), at_ratio(vsc[1], v_ref)};   // (8 bits)
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) vf[i] = read_v(i);
#pragma unroll
    for (int n = 0; n < 16; ++n) {
      if constexpr (F8) {
        const f16x8 vA = at_f16(vf[n % AHEAD].x, vf[n % AHEAD].y, ratio[n & 1]);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg)
          O[rg][n >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(vA, Pf[rg][n & 1], O[rg][n >> 1], 0, 0, 0);
      } else {
#pragma unroll
        for (int rg = 0; rg < RG; ++rg)
          O[rg][n >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n % AHEAD], P[rg][n & 1], O[rg][n >> 1], 0, 0, 0);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg)
          O[rg][n >> 1] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[n % AHEAD], Pl[rg][n & 1], O[rg][n >> 1], 0, 0, 0);
      }
      if (QL && n + AHEAD == 8) asm volatile("" : "+v"(vof));
      if (n + AHEAD < 16) vf[n % AHEAD] = read_v(n + AHEAD);
#pragma unroll
      for (int rg = 0; rg < RG; ++rg) {
        const float p = fast_exp2(__builtin_fmaf(S[rg][n], a.cl2, -base[rg]));
        if (n & 1) {   // (pinned here: the compiler would sink them all past the rescale)
          uint32_t hi, lo = 0;
          if constexpr (F8) hi = __builtin_bit_cast(uint32_t, f16x2{(_Float16)pe[rg], (_Float16)p});
          else at_split(pe[rg], p, hi, lo);
          l_s[rg] += pe[rg] + p;
          asm volatile("" : "+v"(hi), "+v"(lo), "+v"(l_s[rg]));
          Pn[rg][n >> 3][(n & 7) >> 1] = hi;
          Pm[rg][n >> 3][(n & 7) >> 1] = lo;
        } else {
          pe[rg] = p;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int rg = 0; rg < RG; ++rg)
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        if constexpr (F8) {
          Pf[rg][k2] = __builtin_bit_cast(f16x8, Pn[rg][k2]);
        } else {
          P[rg][k2] = __builtin_bit_cast(bf16x8, Pn[rg][k2]);
          Pl[rg][k2] = __builtin_bit_cast(bf16x8, Pm[rg][k2]);
        }
      }
    const int v_next = F8 ? at_units(v_ref, v_coming[0], v_coming[1]) : 0;
    rescale(F8 ? at_ratio(v_ref, v_next) : 1.f, F8 && v_next != v_ref);
    if constexpr (F8) v_ref = v_next;
  };

  if constexpr (F8) {
#pragma unroll
    for (int g = 0; g < 2; ++g) ksc[g] = scale_at(a.ks, pg0[g]);
    AP_BARRIER(8);    // block 0 of K, the first 2 of the 10 loads
  } else if constexpr (SETS == 2) {
    AP_BARRIER(8);    // the first 4 of 12
  } else {
    AP_BARRIER(16);   // block 0 of K, the first 4 of the 20 loads
  }
  if (wblk > j0) {
    scores(ks0, j0, both(pg0));
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
      u32x4_t Pn[2], Pm[2];
#pragma unroll
      for (int r = 0; r < 16; r += 2) {
        const float p0 = fast_exp2(__builtin_fmaf(S[rg][r], a.cl2, -base[rg]));
        const float p1 = fast_exp2(__builtin_fmaf(S[rg][r + 1], a.cl2, -base[rg]));
        uint32_t hi, lo = 0;
        if constexpr (F8) hi = __builtin_bit_cast(uint32_t, f16x2{(_Float16)p0, (_Float16)p1});
        else at_split(p0, p1, hi, lo);
        l_s[rg] += p0 + p1;
        Pn[r >> 3][(r & 7) >> 1] = hi;
        Pm[r >> 3][(r & 7) >> 1] = lo;
      }
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2) {
        if constexpr (F8) {
          Pf[rg][k2] = __builtin_bit_cast(f16x8, Pn[k2]);
        } else {
          P[rg][k2] = __builtin_bit_cast(bf16x8, Pn[k2]);
          Pl[rg][k2] = __builtin_bit_cast(bf16x8, Pm[k2]);
        }
      }
    }
    rescale(1.f, false);
  }
  // Barrier before step j: blocks j + 1 of K and j of V have landed (the 8 loads after them, 4 of
  // 8-bit pages, may be in flight), and every wave is done with K of block j and V of block j - 1,
  // whose sets the loads of blocks j + 3 and j + 2 take.  With two sets nothing is in flight, and they
  // are those of blocks j + 2 and j + 1.
  if constexpr (F8) {
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      ksc[g] = scale_at(a.ks, pg[0][g]);
      vsc[g] = at_scale_bits(scale_at(a.vs, pg0[g]));
    }
    v_ref = max(vsc[0], vsc[1]);
  }
  auto turn = [&](unsigned char* kfree, unsigned char* vfree, const unsigned char* knext, const unsigned char* vset,
                  int j) {
    if constexpr (SETS == 2) {
      AP_BARRIER(0);
      load_k(kfree, rows_of(mine(pg[1]), j + 2), j + 2);
      load_v(vfree, rows_of(mine(pg[0]), j + 1), j + 1);
    } else {
      if constexpr (F8) AP_BARRIER(4); else AP_BARRIER(8);
      const Rows next = rows_of(mine(pg[2]), j + 3);
      load_k(kfree, next, j + 3);
      load_v(vfree, F8 ? coming : rows_of(mine(pg[1]), j + 2), j + 2);
      coming = next;
    }
    float kn[2] = {0.f, 0.f};
    int vn[2] = {0, 0}, rn[2] = {-1, -1};
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      if constexpr (KV != AP_ROWS) rn[g] = entry(j + 5, g);
      if constexpr (F8) {
        kn[g] = scale_at(a.ks, pg[1][g]);
        vn[g] = at_scale_bits(scale_at(a.vs, pg[0][g]));
      }
    }
    step(knext, vset, j, vn);
#pragma unroll
    for (int g = 0; g < 2; ++g) {
      pg[0][g] = pg[1][g];
      pg[1][g] = pg[2][g];
      if constexpr (KV != AP_ROWS) pg[2][g] = page_of(raw[g], j + 4, g);
      raw[g] = rn[g];
      ksc[g] = kn[g];
      vsc[g] = vn[g];
    }
  };
  for (int j = j0; j < nblk; j += SETS) {
    if constexpr (SETS == 2) {
      turn(ks0, vs1, ks1, vs0, j);
      turn(ks1, vs0, ks0, vs1, j + 1);
    } else {
      turn(ks0, vs2, ks1, vs0, j);
      turn(ks1, vs0, ks2, vs1, j + 1);
      turn(ks2, vs1, ks0, vs2, j + 2);
    }
  }
  AP_BARRIER(0);   // no load in flight, every wave done with the sets: the dumps take them
#undef AP_BARRIER

  // Epilogue in two or four parts of the columns: O / l through a set as the wave's own (fp32, chunk
  // c of row r at c ^ (r & 15)), then runs of whole rows with the gate: 8 columns per lane, 16-byte
  // loads and stores.
  constexpr int COLS = AP_SET / 128, LPR = COLS / 8, RPI = 64 / LPR;   // lanes of a row, rows at a time
  unsigned char* dump = wave == 0 ? ks0 : (wave == 1 ? ks1 : (wave == 2 ? (SETS == 3 ? ks2 : vs1) : vs0));
#pragma unroll
  for (int rg = 0; rg < RG; ++rg) {
    const auto sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(l_s[rg]), __float_as_uint(l_s[rg]), false, false);
    const float l = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    const bool whole = !PARTS || parts == 1;
    float inv = !whole ? 1.f : (l == 0.f ? 0.f : 1.f / l);   // no key seen: zeros
    if constexpr (F8) inv *= __int_as_float(v_ref);
    float* piece = nullptr;
    if constexpr (PARTS) {
      if (!whole) {
        const int tile = qt * pairs + pair;
        piece = a.ws + ((size_t)tile * a.parts + part) * AP_PIECE;
        if (h == 0) {
          piece[32 * wave + l32] = m_ref[0];
          piece[128 + 32 * wave + l32] = l;
        }
      }
      if (tid == 0 && part == 0 && a.parts > 1)
        reinterpret_cast<int*>(a.ws + (size_t)a.qtiles * pairs * a.parts * AP_PIECE)[qt * pairs + pair] = parts;
    }
#pragma unroll
    for (int cp = 0; cp < AT_D / COLS; ++cp) {
      // this lane's rows RPI it + lane / LPR, columns 8 (lane % LPR) ..; gates first
      const int c8 = lane & (LPR - 1);
      u32x4_t g[32 / RPI];
      size_t oo[32 / RPI];
      bool live[32 / RPI];
#pragma unroll
      for (int it = 0; it < 32 / RPI; ++it) {
        const int r = 32 * (RG * wave + rg) + RPI * it + lane / LPR, qi = ap_div(r, a.rep_mul), hr = r - qi * a.n_rep;
        live[it] = qi < QB;
        oo[it] = (((size_t)b * a.T + q0 + (live[it] ? qi : 0)) * a.Hq + kvh * a.n_rep + hr) * AT_D + COLS * cp + 8 * c8;
        if (a.gate && whole)
          g[it] = *reinterpret_cast<const u32x4_t*>(a.gate + ((size_t)b * a.T + q0 + (live[it] ? qi : 0)) * a.gate_row +
                                                    (size_t)(kvh * a.n_rep + hr) * a.gate_head + COLS * cp + 8 * c8);
      }
#pragma unroll
      for (int dt = 0; dt < COLS / 32; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int c = (8 * dt + 2 * q + h) ^ (l32 & 15);
          const f32x16& o = O[rg][COLS / 32 * cp + dt];
          *reinterpret_cast<float4*>(dump + l32 * (COLS * 4) + 16 * c) =
              make_float4(o[4 * q] * inv, o[4 * q + 1] * inv, o[4 * q + 2] * inv, o[4 * q + 3] * inv);
        }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the wave's own dump, read by the wave only
#pragma unroll
      for (int it = 0; it < 32 / RPI; ++it) {
        const int rr = RPI * it + lane / LPR;
        float y[8];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float4 f = *reinterpret_cast<const float4*>(dump + rr * (COLS * 4) + 16 * ((2 * c8 + u) ^ (rr & 15)));
          y[4 * u] = f.x; y[4 * u + 1] = f.y; y[4 * u + 2] = f.z; y[4 * u + 3] = f.w;
        }
        if (!whole) {
          if (live[it]) {
            float* to = piece + 256 + (32 * wave + rr) * AT_D + COLS * cp + 8 * c8;
            *reinterpret_cast<float4*>(to) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4*>(to + 4) = make_float4(y[4], y[5], y[6], y[7]);
          }
          continue;
        }
        if (a.gate) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            y[2 * e] *= sigmoidf_(__uint_as_float(g[it][e] << 16));
            y[2 * e + 1] *= sigmoidf_(__uint_as_float(g[it][e] & 0xffff0000u));
          }
        }
        u32x4_t w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const bf16x2 t = {(__bf16)y[2 * e], (__bf16)y[2 * e + 1]};
          w[e] = __builtin_bit_cast(uint32_t, t);
        }
        if (live[it]) *reinterpret_cast<u32x4_t*>(a.out + oo[it]) = w;
      }
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // read before the next dump
    }
  }
}

// Merges the parts of a tile, a wave per row (4 columns a lane), with the gate; tiles of one part
// are finished already.
__global__ __launch_bounds__(256) void attn_parts_combine_kernel(ApArgs a) {
  const int pairs = a.B * a.Hkv, tile = blockIdx.x >> 5, lane = threadIdx.x & 63;
  const int r = 4 * (blockIdx.x & 31) + (threadIdx.x >> 6);
  const int n = reinterpret_cast<const int*>(a.ws + (size_t)a.qtiles * pairs * a.parts * AP_PIECE)[tile];
  if (n == 1) return;
  const int qt = tile / pairs, pair = tile - qt * pairs, b = pair / a.Hkv, kvh = pair - b * a.Hkv;
  const int qi = ap_div(r, a.rep_mul), q0 = qt * a.QB;
  if (qi >= min(a.QB, a.T - q0)) return;
  const int head = kvh * a.n_rep + r - qi * a.n_rep;
  const size_t bt = (size_t)b * a.T + q0 + qi;
  const float* piece = a.ws + (size_t)tile * a.parts * AP_PIECE;
  const float* mine = piece + (size_t)min(lane, n - 1) * AP_PIECE;
  const float m = mine[r], ls = lane < n ? mine[128 + r] : 0.f;
  const float* col = piece + 256 + r * AT_D + 4 * lane;
  float4 v[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = *reinterpret_cast<const float4*>(col + (size_t)min(e, n - 1) * AP_PIECE);
  uint2 gv = make_uint2(0, 0);
  if (a.gate)
    gv = *reinterpret_cast<const uint2*>(a.gate + bt * a.gate_row + (size_t)head * a.gate_head + 4 * lane);
  float M = m;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
  const float wgt = m == -INFINITY ? 0.f : fast_exp2((m - M) * a.cl2);
  float l = ls * wgt;
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) l += __shfl_xor(l, o, 64);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < n; s += 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (s + e < n) {
        const float x = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(wgt), s + e));
        acc[0] += x * v[e].x; acc[1] += x * v[e].y; acc[2] += x * v[e].z; acc[3] += x * v[e].w;
      }
    }
    if (s + 4 < n) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = *reinterpret_cast<const float4*>(col + (size_t)min(s + 4 + e, n - 1) * AP_PIECE);
    }
  }
  at_store4(a.out + (bt * a.Hq + head) * AT_D + 4 * lane, acc, l == 0.f ? 0.f : 1.f / l, a.gate != nullptr, gv);
}

int attn_prefill_groups(int B, int T, int Hkv, int n_rep, int cus) {
  // A sequence's numbers do not depend on how its tokens are divided into calls of up to 64 (the
  // few-row GEMMs' limit): those keep the split-K kernels, whose rows do not depend on T.  Nor do
  // they depend on the cache's capacity, so the lines below go by the queries alone.
  if (T < AP_MIN_T || (long long)B * T <= AP_FEW_ROWS) return 0;
  const long long rows = (long long)T * n_rep, pairs = (long long)B * Hkv;
  // 256-row tiles cost 1.7 of a 128-row tile's time; worth it from one and a half rounds of them
  // (us, RG = 1 / 2: 384 tiles of 3072 keys 256 / 242, 400 of 1600 161 / 150, 512 of 4096 407 /
  // 372; 128 tiles of 8256 keys 368 / 521)
  if (2 * pairs * ((rows + 255) / 256) >= 3LL * cus) return 2;
  // A lone tile walks its keys at 0.038 us each; the split kernels take 0.00048 us per key and
  // tile: from 80 tiles on this kernel is the faster one whatever the length (us, long / split:
  // 128 tiles of 500 keys 33 / 75; 64 of 1024 51 / 54, of 2000 84 / 83, of 4000 153 / 124; 56
  // of 4000 153 / 110)
  if (16 * pairs * ((rows + 127) / 128) >= 5LL * cus) return 1;
  return 0;
}

static int prefill_tiles(int B, int T, int Hkv, int n_rep, int rg, int* QB) {
  *QB = 128 * rg / n_rep < T ? 128 * rg / n_rep : T;
  return (T + *QB - 1) / *QB;
}

int attn_paged_groups(int B, int T, int Hkv, int n_rep, int cus, bool f8, int* parts) {
  *parts = 1;
  if (T < AP_MIN_T || (long long)B * T <= AP_FEW_ROWS) return 0;
  const long long pairs = (long long)B * Hkv;
  // Query tiles, whatever their number (us, tiles / split-K, bf16: 20 tiles of 2070 keys 35 / 38, of
  // 30000 134 / 308; 64 of 8256 123 / 220; 128 of 8289 203 / 418; but 32 of 256 28 / 20), but for few
  // tiles of 8-bit pages, whose codes a tile converts for 32 rows at a time as the split-K does,
  // without its depth of loads: from 64 full tiles on (32 of 1128 33 / 32, of 4128 55 / 54; 64 of
  // 1256 47 / 39, of 4256 71 / 81, of 16256 171 / 246; 128 of 512 49 / 44, of 8289 168 / 264).
  if (f8 && 4 * pairs * T * n_rep < 128LL * cus) return 0;
  int QB;
  const long long tiles = prefill_tiles(B, T, Hkv, n_rep, 1, &QB) * pairs;
  // Workgroups of a CU: a wave alone on its SIMD issues a VALU instruction every 8 cycles, two share
  // it at 4.  8-bit pages have the LDS for two with three sets; bf16 pages with two, which leave a
  // block's rows one step to arrive: for half as many tiles as CUs and 256 tokens a sequence (us, one / two
  // a CU: 128 tiles of 8289 keys 237 / 203, 160 of 4640 185 / 151, 256 of 9024 433 / 383; but 32 of
  // 1128 37 / 43, 128 of 17 20 / 27).
  const int per_cu = f8 || (2 * tiles >= cus && T >= 256) ? 2 : 1;
  const int slots = per_cu * cus;
  // Fewer tiles than these divide their keys: as many parts as the chip holds at once, or a few more
  // where their rounds come out a tenth shorter (160 tiles: 3 parts take 2 rounds of a third).
  if (tiles < slots) {
    int best = slots / (int)tiles;
    best = best > AP_MAX_PARTS ? AP_MAX_PARTS : best;
    double cost = 0.9 / best;   // (one round)
    for (int n = best + 1; n <= best + 4 && n <= AP_MAX_PARTS; ++n) {
      const double c = (double)((tiles * n + slots - 1) / slots) / n;
      if (c < cost) {
        cost = c;
        best = n;
      }
    }
    *parts = best;
  }
  return per_cu;
}

long long attn_parts_bytes(int B, int T, int Hkv, int n_rep, int parts) {
  int QB;
  if (parts <= 1) return 0;
  const long long tiles = (long long)prefill_tiles(B, T, Hkv, n_rep, 1, &QB) * B * Hkv;
  return tiles * parts * AP_PIECE * (long long)sizeof(float) + tiles * 4;
}

template <int RG, int KV, int SETS>
static void prefill_start(const ApArgs& a, unsigned n, hipStream_t st) {
  hipLaunchKernelGGL((attn_prefill_kernel<RG, KV, SETS>), dim3(n), dim3(256), 0, st, a);
}

int attn_prefill_launch(const AttnArgs& v, int groups, hipStream_t st, const PagedArgs* paged, int parts) {
  ApArgs a;
  a.q = v.q; a.kc = v.kc; a.vc = v.vc; a.kv_len = v.kv_len; a.gate = v.gate; a.out = v.out;
  a.seq_stride = v.seq_stride; a.head_stride = v.head_stride;
  a.gate_row = v.gate_row; a.gate_head = v.gate_head;
  a.B = v.B; a.T = v.T; a.Hq = v.Hq; a.Hkv = v.Hkv; a.n_rep = v.n_rep; a.max_len = v.max_len;
  a.cl2 = v.cl2;
  a.rep_mul = (uint32_t)((65536 + v.n_rep - 1) / v.n_rep);
  a.qtiles = prefill_tiles(v.B, v.T, v.Hkv, v.n_rep, paged ? 1 : groups, &a.QB);
  a.parts = parts; a.ws = v.ws;
  a.table = nullptr; a.ks = a.vs = nullptr; a.table_stride = 0; a.n_pages = a.pshift = 0;
  const long long n = (long long)a.qtiles * v.B * v.Hkv * parts;
  if (n > 0x7fffffffLL) return LOLLM_EUNSUPPORTED;
  if (paged) {
    a.table = paged->table; a.ks = paged->ks; a.vs = paged->vs; a.table_stride = paged->table_stride;
    a.n_pages = paged->n_pages; a.pshift = paged->pshift;
  }
  if (paged && paged->ks) prefill_start<1, AP_PAGES8, 3>(a, (unsigned)n, st);
  else if (paged && groups == 2) prefill_start<1, AP_PAGES, 2>(a, (unsigned)n, st);
  else if (paged) prefill_start<1, AP_PAGES, 3>(a, (unsigned)n, st);
  else if (groups == 2) prefill_start<2, AP_ROWS, 3>(a, (unsigned)n, st);
  else prefill_start<1, AP_ROWS, 3>(a, (unsigned)n, st);
  if (parts > 1) {
    const int rc = launch_status();
    if (rc) return rc;
    hipLaunchKernelGGL(attn_parts_combine_kernel, dim3((unsigned)(n / parts) * 32), dim3(256), 0, st, a);
  }
  return launch_status();
}

}  // namespace lollm
