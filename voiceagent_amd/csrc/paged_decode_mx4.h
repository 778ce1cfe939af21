// Paged-KV decode attention over MXFP4 pools (mx4.h) on CDNA4 matrix cores.
//
// The mathematics, partitions and merge are those of paged_decode_mfma.h: for
// each (sequence, kv head) the G query heads of the group attend the tokens
// j < L that the mask leaves, by an online softmax in the exp2 domain.  What
// differs is that a row is 17 D / 32 bytes (68 at head_dim 128), so a CU's
// share of the HBM rate is a row every ~7 cycles and the work between the load
// and the matrix cores is what has to be kept small:
//
//   * S^T = K Q^T takes K in 16 bits, which hold its values exactly, and sums
//     the products in fp32, as over the other pools.  A lane reads 32
//     neighbouring codes of a row, one scale's (16 at head_dim 64), and converts
//     them two an instruction; the query's operand has the same order of k.
//     (Codes as they are, on scaled 16x16x128 products against a query cut into
//     e4m3 terms: that instruction aligns neighbouring products to 13 bits
//     before adding.  Two query channels of 256 times the others' size, whose
//     products cancel, put the output off by 0.6%, of 4096 times by 5.7%; fp32
//     sums 0.16% at any size, which is P's and the output's rounding.)
//   * O^T += V^T P^T takes V in 16 bits too.  A lane reads D / 16 neighbouring
//     elements of eight tokens, converts them with their scales (two elements
//     an instruction) and pairs tokens with v_perm: no transposing read.  P^T
//     is the S^T accumulator packed in place, rounded to the rows' type (the
//     type of the matrix product; its row sum adds the unrounded values).
//
// A workgroup is W waves; wave w takes the partition's 32-token steps w, w + W,
// ... with no barrier, through a ring of S steps in LDS of its own that DMA
// fills S - 1 steps ahead.  (Loads to registers made the compiler wait for each
// at the joins of the branches behind them.)  The waves merge through LDS at
// the end.  In the four-wave instances at head_dim 128, held to 128 registers so
// that four workgroups share a CU, the ring does less: the compiler keeps 5-11
// registers in scratch (not at group 8 with the prologue, where LDS admits
// three), the lane's scale address among them, and its reload between a step's
// requests waits for those already in flight.
#pragma once

#include "mx4.h"
#include "paged_decode_mfma.h"

namespace va {

struct DecodeMx4Params : DecodeParams {
  char* ks;  // scale bytes
  char* vs;
  int64_t sc_blk, sc_slot, sc_head;  // bytes
  int32_t num_seqs;
  int32_t by_token;  // the grid keeps a sequence's heads together (see the kernel)
  FastDiv hkv_div, seq_div;
  int32_t head_pairs;  // a workgroup serves two kv heads (see the kernel)
  int32_t min_part;  // dyn_split: fewest tokens of a partition
};

constexpr int kMx4Step = 32;  // tokens a wave reduces at a time: two 16-token tiles

// Tokens of a context partition: fixed, or with dyn_split an even share of the
// context's L tokens, in whole tiles.
__device__ inline int mx4_partition(const DecodeMx4Params& p, int L) {
  if (!p.dyn_split) return p.split_tokens;
  int P = (L + p.max_parts - 1) / p.max_parts;
  P = (P + kChunk - 1) / kChunk * kChunk;
  return P > p.min_part ? P : p.min_part;
}

// O^T += V^T P^T over 32 tokens, 16-bit.
template <typename ET>
__device__ inline mf_f32x4 mx4_pv(uint4 v, uint4 p, mf_f32x4 c) {
  return DecodeMma<ET>::qk(v, p, c);
}

template <int D>
struct Mx4DecodeShape {
  static constexpr int ROWB = D / 2;                 // bytes of a row's codes
  static constexpr int CPR = ROWB / 16;              // 16-byte chunks of a row
  static constexpr int CH = D <= 128 ? 1 : D / 128;  // 128-element chunks of a row
  static constexpr int NV = D / 16;                  // V elements of a lane and token
  static constexpr int SCW = D <= 128 ? 4 : 8;       // staged bytes of a row's scales
  using V = std::conditional_t<D == 64, uint16_t, std::conditional_t<D == 128, uint32_t, uint2>>;
};

// LDS place of a staged tile's token and of a row's chunk.  Tokens 4 c + r lie
// at row 4 r + c, so that the V reads of one r (four rows, each read whole by
// 16 lanes) are consecutive, and a row's chunks are XORed so that the K reads
// (one chunk of 16 rows) cover all banks.  kPair: a row is two heads' (see the
// kernel), whose V reads are half of each of four rows.
__device__ inline int mx4_slot(int token) { return (token & 3) * 4 + (token >> 2); }
template <int D, bool kPair>
__device__ inline int mx4_swz(int slot) {
  if constexpr (kPair) return ((slot >> 2) & 3) | ((slot & 2) << 1);
  return (slot / (256 / Mx4DecodeShape<D>::ROWB)) & (Mx4DecodeShape<D>::CPR - 1);
}

// One 4-byte global -> LDS copy per lane (lane l's word lands at lds + 4 l).
__device__ inline void dma4(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "{m0}"(lds) : "memory");
}

template <typename ET, int D, int G, bool kProlog, bool kMask, int W, int S, int HP>
__global__ __launch_bounds__(W * 64, W == 4 && D <= 128 ? 4 : 2) void paged_decode_mx4_kernel(DecodeMx4Params p) {
  using Sh = Mx4DecodeShape<D>;
  using M = DecodeMma<ET>;
  using VT = typename Sh::V;
  constexpr int CH = Sh::CH, NV = Sh::NV, CPR = Sh::CPR, ROWB = Sh::ROWB, SCW = Sh::SCW;
  constexpr int NT = W * 64, ROW16 = D * 2;
  constexpr int KP = D == 64 ? 2 : 4;               // products per chunk: 8 elements a lane each
  constexpr int LPR = D / 8, RPL = 64 / LPR, E = 8;  // the row layout of prologue.h
  constexpr int QROWS = (G + RPL - 1) / RPL;
  constexpr int LPS = kMx4Group / NV;  // lanes that share a V scale
  constexpr bool kPair = HP == 2;
  constexpr int TW = W / HP, HG = HP * G;  // a head's waves; the workgroup's query heads
  static_assert(TW % 4 == 0, "the wave merge reads (m, l) of four waves at a time");
  static_assert(HP == 1 || (kPair && D == 128), "a line holds two heads' 64 bytes");
  // A stage: K codes of both tiles, V codes, K scales, V scales.
  constexpr int PITCH = HP * ROWB, SCP = HP * SCW;  // of a staged row of codes, of scales
  constexpr int TILE_B = 16 * PITCH;
  constexpr int V_OFF = 2 * TILE_B, KS_OFF = 4 * TILE_B, VS_OFF = KS_OFF + 32 * SCP;
  constexpr int STAGE_B = VS_OFF + 32 * SCP;
  // Requests of a wave for a step (of a pair's, half).
  constexpr int NDMA = kPair ? 5 : 4 * TILE_B / 1024 + 2 * 32 * SCW / 256;
  constexpr int RING_B = TW * S * STAGE_B;

  // The waves' partial results: o [W][G][D], then m and l [G][W]; in LDS of
  // their own where two workgroups a CU have room for it, else in the ring.
  constexpr int MERGE_B = W * G * D * 4 + 2 * G * W * 4;
  constexpr int Q_B = kProlog ? W * (G + 1) * ROW16 : 16;
  constexpr bool kOwnMerge = RING_B + MERGE_B + Q_B <= (D == 256 ? 80 : W == 4 ? 40 : 160) * 1024;
  static_assert(kOwnMerge || MERGE_B <= RING_B, "merge scratch");
  __shared__ __align__(1024) char s_ring[RING_B];
  __shared__ __align__(16) char s_mrg[kOwnMerge ? MERGE_B : 16];
  // kProlog: each wave's processed query rows and current key row.
  __shared__ __align__(16) char s_q[Q_B];

  // Workgroup i runs on XCD i % 8.  Grid (kv head, sequence, partition), as the
  // other decode kernels', gives each XCD its heads of every sequence.  Where a
  // token's heads are neighbours (NHD pools), that would have every XCD read
  // every 128-byte line: a head's 64 bytes of codes are half of one, its 4 bytes
  // of scales a small part.  There (by_token) the heads of a (sequence,
  // partition) pair u follow one another on XCD u % 8 (32 contexts of 7000 tokens:
  // 92 -> 66 us; the requests to HBM then equal an HND pool's).
  //
  // That leaves each line going to two CUs, 2.2 times the requests of an HND
  // pool from L2.  With HP = 2 a workgroup serves two heads, wave w and w + W / 2
  // the same tokens for one head each, through a ring that they share: a request
  // takes 8 whole lines, half of a tile's for both, and a barrier a step says
  // that the halves are there (66 -> 59 us, against 53 over an HND pool).  Two
  // heads a workgroup with rings of their own did not help (87: the second
  // request for a line finds it in L2, not in the CU).
  int b = blockIdx.y, h = blockIdx.x, part = blockIdx.z;
  if (p.by_token) {
    const uint32_t j = blockIdx.x >> 3, r = fast_div(j, p.hkv_div);
    const uint32_t u = r * 8 + (blockIdx.x & 7);
    h = (int)(j - r * p.hkv_div.d);
    part = (int)fast_div(u, p.seq_div);
    b = (int)(u - (uint32_t)part * p.seq_div.d);
    if (part >= p.max_parts) return;
  }
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int tw = kPair ? wave % TW : wave;
  const int h0 = h * HP;  // the workgroup's first kv head
  const int hd = kPair ? wave / TW : 0;
  h = h0 + hd;
  const int lane = tid & 63;
  const int r16 = lane & 15, c4 = lane >> 4;
  const int rg = lane / LPR, col = lane % LPR;
  const int64_t table_row = (int64_t)b * p.t_sb;
  int P = p.split_tokens;  // a placeholder with dyn_split, fixed below from L
  int start = part * P;
  const bool last_part = part == p.max_parts - 1;

  // ---- independent loads, all requested before the first wait: block ids,
  // the query, the current row, the mask, the length and the slot ----
  // Lane l holds tile l % 2 of the wave's step 32 i + l / 2: the block id, from
  // which its byte offsets are formed 32 steps at a time.
  const uint32_t* const tabw = reinterpret_cast<const uint32_t*>(p.table);
  auto tile_tok = [&](int k0) {
    return start + kMx4Step * (tw + TW * (k0 + (lane >> 1))) + 16 * (lane & 1);
  };
  uint2 ids = make_uint2(0u, 0u);  // raw words of a block id
  auto load_ids = [&](int k0, int limit) {
    const int tok = tile_tok(k0);
    const int idx = (int)fast_div((uint32_t)tok, p.bs_div);
    ids = make_uint2(0u, 0u);  // columns past the table read as block 0
    if (tok < limit && idx < p.table_width) {
      const int64_t at = (table_row + idx) << p.table_i64;
      ids.x = tabw[at];
      ids.y = tabw[at + p.table_i64];
    }
  };
  const bool early = !p.dyn_split;
  const int early_limit = last_part ? INT32_MAX : start + P;
  if (early) load_ids(0, early_limit);
  // Queries in the order of the products' B operand, K's: lane (r16, c4) holds
  // elements 128 c + 8 KP c4 + 8 i .. + 7 of head r16; with the prologue as rows
  // first.
  uint4 qreg[CH][KP];
  uint4 qrow[QROWS];
  constexpr int QL = 16 * KP;  // bytes of a lane's elements of a chunk
  if constexpr (!kProlog) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        // Columns past the group read head 0's row; their scores are unused.
        const int g = r16 < G ? r16 : 0;
        qreg[c][i] = ld16(p.q + b * p.q_sb + (int64_t)(h * G + g) * p.q_sh + 256 * c + QL * c4 + 16 * i);
      }
  } else {
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
      const int g = rg + RPL * i;
      qrow[i] = ld16(p.q + b * p.q_sb + (int64_t)(h * G + (g < G ? g : 0)) * p.q_sh + col * 16);
    }
  }
  // key_valid_mask: lane l holds its tile's 16 tokens as bits (the words that
  // cover its bytes; see paged_decode_mfma.h, which reads them the same way).
  const int mlen = kMask ? p.valid_len : 0;
  const uint8_t* const mrow = p.valid + (kMask ? (int64_t)b * p.valid_sb : 0);
  const int moff = (int)((uintptr_t)mrow & 3);
  const uint32_t* const mwords = reinterpret_cast<const uint32_t*>(mrow - moff);
  uint32_t mraw[5] = {~0u, ~0u, ~0u, ~0u, ~0u};
  int mtb = 0;
  auto mask_load = [&](int k0) {
    mtb = tile_tok(k0);
#pragma unroll
    for (int j = 0; j < 5; ++j) {
      const int rb = mtb + 4 * j - moff;
      mraw[j] = rb < mlen && (j < 4 || moff != 0) ? mwords[(mtb >> 2) + j] : 0xffffffffu;
    }
  };
  auto mask_bits = [&]() -> uint32_t {
    uint32_t bits = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t x = __builtin_amdgcn_alignbyte(mraw[j + 1], mraw[j], (uint32_t)moff);
      x |= x >> 4;
      x |= x >> 2;
      x |= x >> 1;
      x &= 0x01010101u;
      bits |= ((x * 0x01020408u) >> 24) << (4 * j);
    }
    const int rem = mlen - mtb;
    if (rem < 16) bits |= rem <= 0 ? 0xffffu : (0xffffu << rem) & 0xffffu;
    return bits;
  };
  uint32_t mbits = 0xffffu;
  if (kMask && early) mask_load(0);
  const uint32_t* const lensw = reinterpret_cast<const uint32_t*>(p.lens);
  const uint32_t len_hi = lensw[(int64_t)(b + p.lens_cum) << p.lens_i64];
  const uint32_t len_lo = lensw[(int64_t)b << p.lens_i64];
  uint32_t slot_lo = ~0u, slot_hi = ~0u;  // new_slots[b] (-1 without one)
  if (p.new_slots != nullptr) {
    const uint32_t* const sw = reinterpret_cast<const uint32_t*>(p.new_slots);
    slot_lo = sw[(int64_t)b << p.new_slots_i64];
    slot_hi = sw[((int64_t)b << p.new_slots_i64) + p.new_slots_i64];
  }

  // ---- the wave's (the pair's) ring: S stages of a step each, filled by DMA ----
  char* const s_wave = s_ring + tw * S * STAGE_B;
  const uint32_t lds_wave = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_wave);
  // Codes: request i of a tile fills LDS rows i RPI ..; lane l's chunk is
  // position l % CPR of row i RPI + l / CPR.  At head_dim 64 one request takes
  // both tiles, 32 lanes each.
  // A pair's wave hd takes LDS rows 8 hd .. of each tile.
  constexpr int RPI = 1024 / PITCH, CPP = PITCH / 16;
  constexpr int NI = kPair || TILE_B < 1024 ? 1 : TILE_B / 1024;
  uint32_t loff[NI];
  auto swz = [](int slot) { return mx4_swz<D, kPair>(slot); };
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int slot = ((kPair ? hd : i) * RPI + lane / CPP) & 15, pos = lane % CPP;
    const int token = (slot & 3) * 4 + (slot >> 2);
    loff[i] = (uint32_t)(token * (int)p.s_slot) + (uint32_t)((pos ^ swz(slot)) << 4);
  }
  const int64_t head_off = (int64_t)h * p.s_head, head_sc = (int64_t)h * p.sc_head;
  const int64_t ring_off = (int64_t)h0 * p.s_head, ring_sc = (int64_t)h0 * p.sc_head;
  int64_t toff = ring_off, tsc = ring_sc;  // of the lane's tile (block 0 where there is none)
  uint64_t tiles_ok = 0;                   // bit l: lane l's tile has a block of the pool
  auto take_ids = [&](int k0) {
    const int64_t bid = p.table_i64 ? (int64_t)(((uint64_t)ids.y << 32) | ids.x)
                                    : (int64_t)(int32_t)ids.x;
    const bool ok = bid >= 0 && bid < p.num_blocks;
    const int in = ok ? (int)fast_mod((uint32_t)tile_tok(k0), p.bs_div) : 0;
    toff = (ok ? bid : 0) * p.s_blk + (int64_t)in * p.s_slot + ring_off;
    tsc = (ok ? bid : 0) * p.sc_blk + (int64_t)in * p.sc_slot + ring_sc;
    tiles_ok = __builtin_amdgcn_ballot_w64(ok);
  };
  auto lane64 = [&](int64_t x, int l) -> int64_t {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)x, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  };
  // Requests step k (of the 32 whose offsets the lanes hold) into stage k % S.
  auto issue = [&](int k) {
    const uint32_t dst = lds_wave + (uint32_t)((k % S) * STAGE_B);
    const int l = 2 * (k & 31);
    const int64_t o0 = lane64(toff, l), o1 = lane64(toff, l + 1);
    const int64_t c0 = lane64(tsc, l), c1 = lane64(tsc, l + 1);
    if constexpr (kPair) {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const uint32_t at = dst + t * TILE_B + hd * 1024;
        dma16_nt(loff[0], uniform_ptr(p.kp + (t ? o1 : o0)), at);
        dma16_nt(loff[0], uniform_ptr(p.vp + (t ? o1 : o0)), at + V_OFF);
      }
    } else if constexpr (D == 64) {
      const int64_t o = (lane < 32 ? o0 : o1) + loff[0];
      dma16_nt(p.kp + o, dst);
      dma16_nt(p.vp + o, dst + V_OFF);
    } else {
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const char* const kb = uniform_ptr(p.kp + (t ? o1 : o0));
        const char* const vb = uniform_ptr(p.vp + (t ? o1 : o0));
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          // Lines that other heads share stay in L2; others stream past it (32
          // contexts of 7000, us: NHD 66.9 / 69.6, HND 55.9 / 52.0 without / with nt).
          if (p.by_token) {
            dma16(loff[i], kb, dst + t * TILE_B + i * 1024);
            dma16(loff[i], vb, dst + V_OFF + t * TILE_B + i * 1024);
          } else {
            dma16_nt(loff[i], kb, dst + t * TILE_B + i * 1024);
            dma16_nt(loff[i], vb, dst + V_OFF + t * TILE_B + i * 1024);
          }
        }
      }
    }
    // Scales, a word a lane: at head_dim 64 the aligned word that holds the
    // row's two.  A pair's wave 0 takes both heads' K scales, wave 1 the V's.
    if constexpr (kPair) {
      const int64_t at = (lane < 32 ? c0 : c1) + (int64_t)((lane >> 1) & 15) * p.sc_slot +
                         (lane & 1) * p.sc_head;
      dma4((hd ? p.vs : p.ks) + at, dst + (hd ? VS_OFF : KS_OFF));
    } else if constexpr (D <= 128) {
      const char* src = (lane < 32 ? p.ks : p.vs) + ((lane & 16) ? c1 : c0) +
                        (int64_t)r16 * p.sc_slot;
      if constexpr (D == 64) src = (const char*)((uintptr_t)src & ~(uintptr_t)3);
      dma4(src, dst + KS_OFF);
    } else {
      const int64_t at = (lane < 32 ? c0 : c1) + (int64_t)((lane >> 1) & 15) * p.sc_slot + (lane & 1) * 4;
      dma4(p.ks + at, dst + KS_OFF);
      dma4(p.vs + at, dst + VS_OFF);
    }
  };

  // With fixed partitions the first steps are requested before the length is
  // known, once what was loaded above is there (a wait left to a first use
  // behind the DMA would wait for the DMA too).  Tokens past the context are
  // masked.
  if (early) {
    asm volatile("" ::"v"(ids.x), "v"(ids.y));
    take_ids(0);
    if constexpr (!kProlog) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < KP; ++i)
          asm volatile("" ::"v"(qreg[c][i].x), "v"(qreg[c][i].y), "v"(qreg[c][i].z), "v"(qreg[c][i].w));
    }
    if constexpr (kMask)
      asm volatile("" ::"v"(mraw[0]), "v"(mraw[1]), "v"(mraw[2]), "v"(mraw[3]), "v"(mraw[4]));
    if (p.num_blocks > 0)
      for (int k = 0; k < S - kPair; ++k)
        if (last_part || (tw + TW * k) * kMx4Step < P) issue(k);
  }

  // ---- the length and the partition ----
  int L = __builtin_amdgcn_readfirstlane((int)(p.lens_cum ? len_hi - len_lo : len_lo));
  const int Lr = L;
  L = attend_len(p, L);
  if (p.num_blocks <= 0) L = 0;
  const int col_new = Lr >= 1 ? (int)fast_div((uint32_t)(Lr - 1), p.bs_div) : 0;
  const bool detached = current_row_detached(p, Lr, L, col_new);
  const int64_t new_slot = p.new_slots_i64 ? (int64_t)(((uint64_t)slot_hi << 32) | slot_lo)
                                           : (int64_t)(int32_t)slot_lo;
  if (p.dyn_split) {
    P = mx4_partition(p, L > 0 ? L : 1);
    start = part * P;
  }
  const int end = L <= 0 ? 0 : (last_part ? L : min(start + P, L));
  const bool writes_row = detached && part == 0;  // this workgroup writes the detached row
  if (start >= L && !writes_row && !(part == 0 && L <= 0)) {
    wait_vmcnt<0>();  // early steps land before the workgroup's LDS is released
    return;
  }
  int nparts = L > 0 ? (L + P - 1) / P : 1;
  if (nparts > p.max_parts) nparts = p.max_parts;  // the last partition absorbs the rest
  const int nsteps = end > start ? (end - start + kMx4Step - 1) / kMx4Step : 0;
  const int ntw = nsteps > tw ? (nsteps - tw + TW - 1) / TW : 0;  // steps of this wave
  const int new_tok =
      (!detached && p.new_k != nullptr && L - 1 >= start && L - 1 < end) ? L - 1 : -1;
  const int new_step = new_tok >= 0 ? (new_tok - start) / kMx4Step : -1;
  const bool owns_new = new_step >= 0 && new_step % TW == tw;
  const int64_t cap = (int64_t)p.num_blocks * p.block_size;
  const bool has_new = p.new_k != nullptr && (owns_new || (writes_row && tw == 0));
  if (!early && ntw > 0) {
    load_ids(0, end);
    if (kMask) mask_load(0);
    asm volatile("" ::"v"(ids.x), "v"(ids.y));
    if constexpr (kMask)
      asm volatile("" ::"v"(mraw[0]), "v"(mraw[1]), "v"(mraw[2]), "v"(mraw[3]), "v"(mraw[4]));
    take_ids(0);
    for (int k = 0; k < S - kPair; ++k)
      if (k < ntw) issue(k);
  }
  if (kMask) mbits = mask_bits();
  uint32_t mbits_k = mbits;   // of the step being reduced; the others are of the step requested
  uint64_t tiles_ok_k = tiles_ok;
  uint32_t tsc_k = (uint32_t)tsc;

  if constexpr (kProlog) {
    // Rows in the row layout, then through LDS (the wave's own part of it).
    int64_t pos = load_index(p.pro.pos, b, p.pro.pos_i64);
    pos = pos < 0 ? 0 : (pos >= p.pro.max_pos ? p.pro.max_pos - 1 : pos);
    float pro_c[E], pro_s[E];
    load_rotary<E, LPR>(p.pro, pos, col, D, pro_c, pro_s);
    char* const s_w = s_q + wave * (G + 1) * ROW16;
    float w[E], x[E];
    convert_weights<E>(load_weights_raw<E>(p.pro.q_w, p.pro.w_dtype, col * E), p.pro.w_dtype, w);
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
      const int g = rg + RPL * i;
      ET::unpack(qrow[i], x);
      qk_prologue<ET, LPR, E>(x, w, p.pro.eps, D, pro_c, pro_s);
      if (g < G) st16(s_w + g * ROW16 + col * 16, ET::pack(x));
    }
    if (has_new) {
      convert_weights<E>(load_weights_raw<E>(p.pro.k_w, p.pro.w_dtype, col * E), p.pro.w_dtype, w);
      ET::unpack(ld16(p.new_k + b * p.nk_sb + h * p.nk_sh + col * 16), x);
      qk_prologue<ET, LPR, E>(x, w, p.pro.eps, D, pro_c, pro_s);
      if (rg == 0) st16(s_w + G * ROW16 + col * 16, ET::pack(x));
    }
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < KP; ++i)
        qreg[c][i] = *reinterpret_cast<const uint4*>(s_w + (r16 < G ? r16 : 0) * ROW16 + 256 * c +
                                                     QL * c4 + 16 * i);
  }

  // ---- the current row, quantised: lane (., c4) the K group its step
  // operand holds (per chunk), lane (r16, .) its V elements ----
  uint4 kq[CH];
  uint32_t kqs[CH];
  VT vq{};
  uint32_t vqs = 0;  // scale of the lane's V elements
  if (has_new) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int g = D == 64 ? (c4 & 1) : 4 * c + c4;  // the row's group
      uint4 u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if constexpr (kProlog)
          u[i] = *reinterpret_cast<const uint4*>(s_q + (wave * (G + 1) + G) * ROW16 + g * 64 +
                                                 16 * i);
        else
          u[i] = ld16(p.new_k + b * p.nk_sb + h * p.nk_sh + g * 64 + 16 * i);
      }
      uint32_t mag = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint32_t m8 = mx4_absmax8(u[i]);
        mag = mag > m8 ? mag : m8;
      }
      kqs[c] = mx4_scale<ET>(mag);
      kq[c] = make_uint4(mx4_codes8<ET>(u[0], kqs[c]), mx4_codes8<ET>(u[1], kqs[c]),
                         mx4_codes8<ET>(u[2], kqs[c]), mx4_codes8<ET>(u[3], kqs[c]));
    }
    // V: the lane's NV elements; a group is 32 / NV neighbouring lanes.
    const char* const src = p.new_v + b * p.nv_sb + h * p.nv_sh + r16 * NV * 2;
    uint4 u[2] = {};
    if constexpr (D == 64) {
      const uint2 x = *reinterpret_cast<const uint2*>(src);
      u[0] = make_uint4(x.x, x.y, 0, 0);
    } else {
      u[0] = ld16(src);
      if constexpr (D == 256) u[1] = ld16(src + 16);
    }
    uint32_t mag = mx4_absmax8(u[0]);
    if constexpr (D == 256) {
      const uint32_t m1 = mx4_absmax8(u[1]);
      mag = mag > m1 ? mag : m1;
    }
#pragma unroll
    for (int i = 1; i < kMx4Group / NV; i *= 2) {
      const uint32_t o = (uint32_t)__shfl_xor((int)mag, i, 64);
      mag = mag > o ? mag : o;
    }
    vqs = mx4_scale<ET>(mag);
    if constexpr (D == 64)
      vq = (VT)mx4_codes8<ET>(u[0], vqs);
    else if constexpr (D == 128)
      vq = mx4_codes8<ET>(u[0], vqs);
    else
      vq = make_uint2(mx4_codes8<ET>(u[0], vqs), mx4_codes8<ET>(u[1], vqs));
  }
  // Where it is stored: new_slots[b], or position Lr - 1 through the table
  // (the attended tile's entry, or the table's own for a detached row).
  int64_t dst_off = INT64_MIN, dst_sc = 0;
  if (has_new) {
    int64_t slot = new_slot;
    if (p.new_slots == nullptr) {
      const int width = detached ? p.table_width_full : p.table_width;
      const int64_t blk = col_new < width ? load_index(p.table, table_row + col_new, p.table_i64) : 0;
      slot = blk >= 0 && blk < p.num_blocks
                 ? blk * p.block_size + (int)fast_mod((uint32_t)(Lr - 1), p.bs_div)
                 : -1;
    }
    if (slot >= 0 && slot < cap) {
      const int64_t sb = slot / p.block_size;
      const int64_t in = slot - sb * p.block_size;
      dst_off = sb * p.s_blk + in * p.s_slot + head_off;
      dst_sc = sb * p.sc_blk + in * p.sc_slot + head_sc;
    }
  }
  auto store_row = [&]() {
    if (dst_off == INT64_MIN) return;
    if (r16 == 0 && (D > 64 || c4 < 2)) {
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        st16(p.kp + dst_off + 64 * c + 16 * c4, kq[c]);
        p.ks[dst_sc + 4 * c + c4] = (char)kqs[c];
      }
    }
    if (c4 == 0) {
      *reinterpret_cast<VT*>(p.vp + dst_off + r16 * (NV / 2)) = vq;
      if (r16 % (kMx4Group / NV) == 0) p.vs[dst_sc + r16 * NV / kMx4Group] = (char)vqs;
    }
  };
  if (writes_row && tw == 0) store_row();
  if (L <= 0) {
    // Nothing to attend: the output is defined as 0.
    if (part == 0) {
      for (int idx = tid; idx < HG * D / E; idx += NT) {
        const int g = idx / (D / E), d = (idx % (D / E)) * E;
        st16(p.out + b * p.o_sb + (int64_t)(h0 * G + g) * p.o_sh + d * 2, make_uint4(0, 0, 0, 0));
      }
    }
    wait_vmcnt<0>();
    return;
  }
  if (start >= L) {
    wait_vmcnt<0>();
    return;
  }

  // A query row with an infinity or a NaN scores NaN, whatever the keys are: its
  // scores start there.
  float score0 = 0.f;
  {
    uint32_t mag = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < KP; ++i) {
        const uint32_t m8 = mx4_absmax8(qreg[c][i]);
        mag = mag > m8 ? mag : m8;
      }
    const uint32_t m16 = (uint32_t)__shfl_xor((int)mag, 16, 64);
    mag = mag > m16 ? mag : m16;
    const uint32_t m32 = (uint32_t)__shfl_xor((int)mag, 32, 64);
    mag = mag > m32 ? mag : m32;
    if (mag >= (ET::kIsBF16 ? 0x7f80u : 0x7c00u)) score0 = __builtin_nanf("");
  }

  float m = kNegBig, l = 0.f;
  mf_f32x4 o[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) o[i] = mf_f32x4{0.f, 0.f, 0.f, 0.f};

  // Byte offsets of the lane's reads inside a stage (K: its 16 bytes of a chunk, or
  // at head_dim 64 8, half a scale's).
  typedef uint32_t KT __attribute__((ext_vector_type(KP)));
  const int kslot = mx4_slot(r16);
  const int hc = CPR * hd, hs = SCW * hd;  // the head's chunks and scales of a staged row
  const int koff = D == 64 ? kslot * PITCH + (((c4 >> 1) ^ swz(kslot)) << 4) + 8 * (c4 & 1)
                           : kslot * PITCH + (((hc + c4) ^ swz(kslot)) << 4);
  const int ksoff = KS_OFF + r16 * SCP + hs + (D == 64 ? c4 >> 1 : c4);
  int voff[4];  // of token 4 c4 + i
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int slot = 4 * i + c4, byte = r16 * (NV / 2);
    voff[i] = V_OFF + slot * PITCH + (((hc + (byte >> 4)) ^ swz(slot)) << 4) + (byte & 15);
  }
  const int vsoff = VS_OFF + 4 * c4 * SCP + hs + r16 / LPS;

  const int nloop = kPair ? (nsteps + TW - 1) / TW : ntw;
  for (int k = 0; k < nloop; ++k) {
    constexpr int kAhead = S - 1 - kPair;  // steps that may stay in flight
    if (k + kAhead < ntw)
      wait_vmcnt<NDMA * kAhead>();
    else
      wait_vmcnt<0>();
    if constexpr (kPair) {
      // Both waves' halves of step k are there, and both are done with the
      // stage before it, which takes step k + S - 1 below.
      asm volatile("s_barrier" ::: "memory");
      if (k >= ntw) continue;
    }
    if (k > 0 && (k & 31) == 0) {
      tiles_ok_k = tiles_ok;
      mbits_k = mbits;
      tsc_k = (uint32_t)tsc;
    }
    char* const st = s_wave + (k % S) * STAGE_B;
    const int c = tw + TW * k;
    const int tb = start + kMx4Step * c;
    uint32_t tpar[2] = {0u, 0u};
    if constexpr (D == 64) {
#pragma unroll
      for (int t = 0; t < 2; ++t)
        tpar[t] = (uint32_t)__builtin_amdgcn_readlane((int)tsc_k, 2 * (k & 31) + t);
    }
    // Byte offset (0 or 2) of row `row`'s scales in its staged word.
    auto half = [&](int t, const char* base, int row) -> int {
      return D == 64 ? (int)((uint32_t)(uintptr_t)base + tpar[t] + (uint32_t)(row * (int)p.sc_slot)) & 2 : 0;
    };
    if (c == new_step && dst_off != INT64_MIN) {
      // The current row in place of the pool's.
      const int t = (new_tok - tb) >> 4, r = (new_tok - tb) & 15, slot = mx4_slot(r);
      if (r16 == 0 && (D > 64 || c4 < 2)) {
#pragma unroll
        for (int cc = 0; cc < CH; ++cc) {
          *reinterpret_cast<uint4*>(st + t * TILE_B + slot * PITCH +
                                    (((4 * cc + hc + c4) ^ swz(slot)) << 4)) = kq[cc];
          st[KS_OFF + (t * 16 + r) * SCP + hs + half(t, p.ks, r) + 4 * cc + c4] = (char)kqs[cc];
        }
      }
      if (c4 == 0) {
        const int byte = r16 * (NV / 2);
        *reinterpret_cast<VT*>(st + V_OFF + t * TILE_B + slot * PITCH +
                               (((hc + (byte >> 4)) ^ swz(slot)) << 4) + (byte & 15)) = vq;
        if (r16 % LPS == 0)
          st[VS_OFF + (t * 16 + r) * SCP + hs + half(t, p.vs, r) + r16 / LPS] = (char)vqs;
      }
      __builtin_amdgcn_wave_barrier();
    }
    // S^T: the lane's scores are tokens 4 c4 + i of both tiles, head r16.
    KT kk[2][CH];
    uint32_t kks[2][CH];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int cc = 0; cc < CH; ++cc) {
        // (a row's chunks 4 .. 7 are its chunks 0 .. 3 with the third bit flipped)
        kk[t][cc] = *reinterpret_cast<const KT*>(st + t * TILE_B + (koff ^ (cc << 6)));
        kks[t][cc] = (uint8_t)st[ksoff + t * 16 * SCP + 4 * cc + half(t, p.ks, r16)];
      }
    VT vv[8];
    uint32_t vb[8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        vv[4 * t + i] = *reinterpret_cast<const VT*>(st + t * TILE_B + voff[i]);
        vb[4 * t + i] = (uint8_t)st[vsoff + (t * 16 + i) * SCP + half(t, p.vs, 4 * c4 + i)];
      }
    mf_f32x4 sc[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = mf_f32x4{score0, score0, score0, score0};
#pragma unroll
      for (int cc = 0; cc < CH; ++cc)
#pragma unroll
        for (int i = 0; i < KP; ++i)
          sc[t] = M::qk(mx4_values8<ET>(kk[t][cc][i], kks[t][cc]), qreg[cc][i], sc[t]);
    }
    // The stage has been read: it takes the wave's step k + S (a pair's, once
    // both have read it: the stage before it takes step k + S - 1).
    wait_lgkmcnt0();
    if (const int n = k + S - kPair; n < ntw) {
      if ((n & 31) == 0) {
        // The offsets of the next 32 steps.
        load_ids(n, end);
        if (kMask) mask_load(n);
        asm volatile("" ::"v"(ids.x), "v"(ids.y));
        take_ids(n);
        if (kMask) mbits = mask_bits();
      }
      issue(n);
    }
    float sv[8];
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) sv[4 * t + i] = sc[t][i];
    const uint32_t ok = (uint32_t)(tiles_ok_k >> (2 * (k & 31))) & 3u;
    if (kMask || ok != 3u || end - tb < kMx4Step) {
      // Tokens that are not attended: their scores are -inf, and their V
      // scales 0, so that nothing their rows may hold (a NaN scale) meets
      // their P of 0.
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        const int rel = (ok >> t) & 1u ? end - tb - 16 * t - 4 * c4 : 0;
        uint32_t live = rel >= 4 ? 15u : (rel <= 0 ? 0u : (1u << rel) - 1u);
        if constexpr (kMask)
          live &= (uint32_t)__builtin_amdgcn_readlane((int)mbits_k, 2 * (k & 31) + t) >> (4 * c4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool on = (live >> i) & 1u;
          sv[4 * t + i] = on ? sv[4 * t + i] : -INFINITY;
          vb[4 * t + i] = on ? vb[4 * t + i] : 0u;
        }
      }
    }
    float mx = sv[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, sv[i]);
    mx = max_xor16(mx);
    mx = max_xor32(mx);
    const float mxs = mx * p.scale_log2;
    if (__builtin_amdgcn_ballot_w64(mxs > m + kDecLazy) != 0) {
      const float mnew = fmaxf(m, mxs);
      const float alpha = fast_exp2(m - mnew);
      m = mnew;
      l *= alpha;
#pragma unroll
      for (int i = 0; i < NV; ++i) o[i] *= alpha;
    }
    float pr[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      pr[i] = fast_exp2(fmaf(sv[i], p.scale_log2, -m));
      l += pr[i];
    }
    const uint4 pb = make_uint4(M::pack2(pr[0], pr[1]), M::pack2(pr[2], pr[3]),
                                M::pack2(pr[4], pr[5]), M::pack2(pr[6], pr[7]));
    // O^T += V^T P^T, two d's at a time: eight tokens' pairs, then the tokens
    // of each d together.
    auto word = [&](const VT& v, int i) -> uint32_t {  // codes 8 i .. of the lane's elements
      if constexpr (D == 256)
        return i == 0 ? v.x : v.y;
      else
        return v;
    };
    auto product = [&](auto BB, int i) {
      constexpr int B = decltype(BB)::value;
      uint32_t x[8];
#pragma unroll
      for (int j = 0; j < 8; ++j)
        x[j] = mx4_pair<ET, B>(word(vv[j], i), __uint_as_float(vb[j] << 23));
      const uint4 lo = make_uint4(__builtin_amdgcn_perm(x[1], x[0], 0x05040100u),
                                  __builtin_amdgcn_perm(x[3], x[2], 0x05040100u),
                                  __builtin_amdgcn_perm(x[5], x[4], 0x05040100u),
                                  __builtin_amdgcn_perm(x[7], x[6], 0x05040100u));
      const uint4 hi = make_uint4(__builtin_amdgcn_perm(x[1], x[0], 0x07060302u),
                                  __builtin_amdgcn_perm(x[3], x[2], 0x07060302u),
                                  __builtin_amdgcn_perm(x[5], x[4], 0x07060302u),
                                  __builtin_amdgcn_perm(x[7], x[6], 0x07060302u));
      const int n = 8 * i + 2 * B;
      o[n] = mx4_pv<ET>(lo, pb, o[n]);
      o[n + 1] = mx4_pv<ET>(hi, pb, o[n + 1]);
    };
#pragma unroll
    for (int i = 0; i < (NV + 7) / 8; ++i) {
      product(std::integral_constant<int, 0>{}, i);
      product(std::integral_constant<int, 1>{}, i);
      if constexpr (NV >= 8) {
        product(std::integral_constant<int, 2>{}, i);
        product(std::integral_constant<int, 3>{}, i);
      }
    }
  }
  wait_vmcnt<0>();  // steps requested early past the wave's last one

  // ---- merge the waves through LDS ----
  l = sum_xor16(l);
  l = sum_xor32(l);
  if constexpr (!kOwnMerge) __syncthreads();  // every wave is done with its stages
  float* const s_o = reinterpret_cast<float*>(kOwnMerge ? s_mrg : s_ring);  // [TW][HG][D]
  float* const s_m = s_o + W * G * D;                                        // [HG][TW]
  float* const s_l = s_m + G * W;                                            // [HG][TW]
  const int row0 = hd * G;  // the wave's first row of HG
  if (r16 < G) {
    // Lane (r16, c4) holds o of head r16 at d = NV (4 c4 + r) + i.
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < NV; i += 4)
        *reinterpret_cast<mf_f32x4*>(s_o + (tw * HG + row0 + r16) * D + NV * (4 * c4 + r) + i) =
            mf_f32x4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
    if (c4 == 0) {
      s_m[(row0 + r16) * TW + tw] = ntw > 0 ? m : kNegBig;
      s_l[(row0 + r16) * TW + tw] = ntw > 0 ? l : 0.f;
    }
  }
  __syncthreads();
  for (int qd = tid; qd < HG * D / 4; qd += NT) {
    const int g = qd / (D / 4), d = (qd % (D / 4)) * 4;
    float mw[TW], lw[TW];
#pragma unroll
    for (int w = 0; w < TW; w += 4) {
      const mf_f32x4 mv = *reinterpret_cast<const mf_f32x4*>(s_m + g * TW + w);
      const mf_f32x4 lv = *reinterpret_cast<const mf_f32x4*>(s_l + g * TW + w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mw[w + i] = mv[i];
        lw[w + i] = lv[i];
      }
    }
    float Mx = kNegBig;
#pragma unroll
    for (int w = 0; w < TW; ++w) Mx = fmaxf(Mx, mw[w]);
    float Lt = 0.f;
    mf_f32x4 acc = mf_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < TW; ++w) {
      const float f = fast_exp2(mw[w] - Mx);
      Lt += lw[w] * f;
      acc += f * *reinterpret_cast<const mf_f32x4*>(s_o + (w * HG + g) * D + d);
    }
    if (nparts == 1) {
      const float inv = Lt > 0.f ? 1.0f / Lt : (Lt == 0.f ? 0.f : Lt);  // a NaN stays one
      uint2 u;
      u.x = M::pack2(acc[0] * inv, acc[1] * inv);
      u.y = M::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2*>(p.out + b * p.o_sb + (int64_t)(h0 * G + g) * p.o_sh + d * 2) = u;
    } else {
      const int64_t pair = (int64_t)b * p.num_kv_heads + h0 + g / G;
      const int64_t slot = (pair * p.max_parts + part) * G + g % G;
      *reinterpret_cast<mf_f32x4*>(p.part_o + slot * D + d) = acc;
      if (d == 0) {
        p.part_ml[slot * 2] = Mx;
        p.part_ml[slot * 2 + 1] = Lt;
      }
    }
  }
  if (owns_new) store_row();
}

// Merge of a split launch's partitions: one workgroup for each query head of a
// sequence, 4 outputs a lane, the partitions dealt to the NG = 1024 / D groups
// of D / 4 lanes, which meet in LDS.  (One workgroup for a whole group of
// heads, each wave going through every partition, took 25 us over 64 heads'
// worth of partitions at group 8.)  The first kFirst partitions of a group are
// requested before the length is known.
//   out = sum_q 2^(m_q - M) o_q / sum_q 2^(m_q - M) l_q,  M = max_q m_q.
template <typename ET, int D>
__global__ __launch_bounds__(256) void paged_decode_mx4_merge_kernel(DecodeMx4Params p, int G) {
  constexpr int LPO = D / 4, NG = 256 / LPO, kFirst = 4;
  __shared__ __align__(16) float s_o[NG * D];
  __shared__ float s_m[NG], s_l[NG];
  const int b = blockIdx.y, hq = blockIdx.x;
  const int col = threadIdx.x % LPO, grp = threadIdx.x / LPO;
  const int64_t slot0 = ((int64_t)b * p.num_kv_heads + hq / G) * p.max_parts * G + hq % G;
  const uint32_t* const lensw = reinterpret_cast<const uint32_t*>(p.lens);
  const uint32_t len_hi = lensw[(int64_t)(b + p.lens_cum) << p.lens_i64];
  const uint32_t len_lo = lensw[(int64_t)b << p.lens_i64];
  mf_f32x4 oq[kFirst];
  float2 ml[kFirst];
  auto request = [&](int q0) {  // partitions q0 + grp + NG j (past the last: the last)
#pragma unroll
    for (int j = 0; j < kFirst; ++j) {
      const int q = q0 + grp + NG * j;
      const int64_t slot = slot0 + (int64_t)(q < p.max_parts ? q : p.max_parts - 1) * G;
      ml[j] = *reinterpret_cast<const float2*>(p.part_ml + slot * 2);
      oq[j] = *reinterpret_cast<const mf_f32x4*>(p.part_o + slot * D + 4 * col);
    }
  };
  request(0);
  int L = (int)(p.lens_cum ? len_hi - len_lo : len_lo);
  L = attend_len(p, __builtin_amdgcn_readfirstlane(L));
  if (L <= 0 || p.num_blocks <= 0) return;
  const int P = mx4_partition(p, L);
  int nparts = (L + P - 1) / P;
  if (nparts > p.max_parts) nparts = p.max_parts;
  if (nparts <= 1) return;  // the attention kernel wrote the output itself
  float M = kNegBig, Lt = 0.f;
  mf_f32x4 acc = mf_f32x4{0.f, 0.f, 0.f, 0.f};
  for (int q0 = 0; q0 < nparts; q0 += NG * kFirst) {
    if (q0 > 0) request(q0);
#pragma unroll
    for (int j = 0; j < kFirst; ++j) {
      if (q0 + grp + NG * j < nparts) {
        const float mn = fmaxf(M, ml[j].x);
        const float a = fast_exp2(M - mn), c = fast_exp2(ml[j].x - mn);
        acc = acc * a + oq[j] * c;
        Lt = Lt * a + ml[j].y * c;
        M = mn;
      }
    }
  }
  *reinterpret_cast<mf_f32x4*>(s_o + grp * D + 4 * col) = acc;
  if (col == 0) {
    s_m[grp] = M;
    s_l[grp] = Lt;
  }
  __syncthreads();
  if (grp != 0) return;
  M = kNegBig;
#pragma unroll
  for (int g = 0; g < NG; ++g) M = fmaxf(M, s_m[g]);
  Lt = 0.f;
  acc = mf_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int g = 0; g < NG; ++g) {
    const float f = fast_exp2(s_m[g] - M);
    Lt += s_l[g] * f;
    acc += f * *reinterpret_cast<const mf_f32x4*>(s_o + g * D + 4 * col);
  }
  const float inv = Lt > 0.f ? 1.0f / Lt : (Lt == 0.f ? 0.f : Lt);  // a NaN stays one
  uint2 u;
  u.x = DecodeMma<ET>::pack2(acc[0] * inv, acc[1] * inv);
  u.y = DecodeMma<ET>::pack2(acc[2] * inv, acc[3] * inv);
  *reinterpret_cast<uint2*>(p.out + b * p.o_sb + (int64_t)hq * p.o_sh + col * 8) = u;
}

// ------------------------------------------------------------- launching
template <typename ET, int D, int G, int W, int S, int HP = 1>
static void launch_decode_mx4_w(const DecodeMx4Params& p, dim3 grid, hipStream_t s) {
  if (p.by_token) {
    const int64_t units = (int64_t)p.num_seqs * p.max_parts;
    grid = dim3((unsigned)((units + 7) / 8 * 8 * (p.num_kv_heads / HP)));
  }
  const dim3 nt(W * 64);
  const bool mask = p.valid != nullptr && p.valid_len > 0;
  if (p.has_pro && mask)
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, true, true, W, S, HP>), grid, nt, 0, s, p);
  else if (p.has_pro)
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, true, false, W, S, HP>), grid, nt, 0, s, p);
  else if (mask)
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, false, true, W, S, HP>), grid, nt, 0, s, p);
  else
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, false, false, W, S, HP>), grid, nt, 0, s, p);
}

template <typename ET, int D, int G>
static void launch_decode_mx4(const DecodeMx4Params& p, dim3 grid, hipStream_t s) {
  if constexpr (D == 256) {
    launch_decode_mx4_w<ET, D, G, 4, 2>(p, grid, s);
  } else {
    if (p.head_pairs) {
      if constexpr (D == 128) launch_decode_mx4_w<ET, D, G, 8, 3, 2>(p, grid, s);
    } else if (p.waves == 4)
      launch_decode_mx4_w<ET, D, G, 4, 2>(p, grid, s);
    else
      launch_decode_mx4_w<ET, D, G, 8, 3>(p, grid, s);
  }
  if (p.max_parts > 1)
    hipLaunchKernelGGL((paged_decode_mx4_merge_kernel<ET, D>), dim3(grid.x * G, grid.y), dim3(256),
                       0, s, p, G);
}

template <typename ET, int D>
static bool dispatch_mx4_g(int G, const DecodeMx4Params& p, dim3 grid, hipStream_t s) {
  switch (G) {
    case 1: launch_decode_mx4<ET, D, 1>(p, grid, s); return true;
    case 2: launch_decode_mx4<ET, D, 2>(p, grid, s); return true;
    case 4: launch_decode_mx4<ET, D, 4>(p, grid, s); return true;
    case 8: launch_decode_mx4<ET, D, 8>(p, grid, s); return true;
    default: return false;
  }
}

template <typename ET>
static bool dispatch_mx4_d(int D, int G, const DecodeMx4Params& p, dim3 grid, hipStream_t s) {
  switch (D) {
    case 64: return dispatch_mx4_g<ET, 64>(G, p, grid, s);
    case 128: return dispatch_mx4_g<ET, 128>(G, p, grid, s);
    case 256: return dispatch_mx4_g<ET, 256>(G, p, grid, s);
    default: return false;
  }
}

// Launch the decode (and, when partitioned, the merge) for one element type,
// instantiated in paged_decode_<type>_mx4.hip; grid (kv heads, sequences,
// partitions).  False for an unsupported (head_dim, group) pair.
template <typename ET>
bool launch_paged_decode_mx4(int D, int G, const DecodeMx4Params& p, dim3 grid, hipStream_t s);

}  // namespace va
