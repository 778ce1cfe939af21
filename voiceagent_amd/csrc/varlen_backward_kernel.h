// The gradient of variable-length attention over packed sequences (16-bit
// rows, no pool), on CDNA4 bf16/f16 MFMA.
//
// With c = scale, P = softmax(c q k^T) over the visible keys (the forward's
// masks, varlen_kernel.h), and the query heads of a group sharing a kv head:
//     delta_i = sum_d dout_i out_i
//     dS_ij   = P_ij (dout_i . v_j - delta_i)
//     dq_i = c sum_j dS_ij k_j,   dk_j = c sum_i dS_ij q_i,   dv_j = sum_i P_ij dout_i
// P is recomputed from q and k: nothing of the forward pass is kept but out.
//
// Two launches, or three (or one, for short sequences: varlen_window_kernel), none
// with atomics, so that every call repeats bit for bit:
//   1. varlen_dq_kernel: a workgroup per 128 (or 64) queries of one head, one pass
//      over their keys.  delta is known from out, so dq needs no softmax statistics
//      beforehand: with a running maximum m, dq gathers 2^(s c - m) (dP - delta) k
//      and is divided by the sum at the end, rescaled where m rises.  It leaves
//      lse_i = log2 sum_j 2^(c log2 e s_ij) and -delta_i for the second launch.
//   2. varlen_dkv_kernel: a workgroup per 64 keys of one kv head, over the queries
//      that see them in every head of the group; or several, with a part of the
//      queries each.
//   3. varlen_dkv_sum_kernel: adds up the parts, where there are several.
// A wave holds 32 queries (keys): their rows are B operands in registers for the
// whole loop, their gradients accumulators.  The other side streams through LDS in
// 64-row tiles, two stages filled by DMA, swizzled.  S^T and dP^T (or S and dP)
// come from 32x32x16 MFMAs with the tile's rows as A operands; their accumulators,
// rounded to 16 bits, are in place the B operands of the gradients' products, whose
// A operands are the same tile rows transposed by ds_read_b64_tr_b16.
// That rounding (half a step of the type, of each P and dS) is the price of the matrix
// cores, whose 16-bit products run at some 16 times the rate of fp32 ones: against
// float64 the gradients are off by 0.0024 of their size in bf16 and 0.0003 in f16 (root
// mean square), and by 0.0017 and 0.00021 if only the results are rounded.  The forward
// rounds P in the same way.
#pragma once

#include <algorithm>

#include "varlen_kernel.h"

namespace va {

typedef float f32x16_t __attribute__((ext_vector_type(16)));

struct VarlenBwdParams {
  const char* q;
  int64_t q_st, q_sh;  // bytes
  const char* k;
  int64_t k_st, k_sh;
  const char* v;
  int64_t v_st, v_sh;
  const char* out;
  int64_t o_st, o_sh;
  const char* dout;
  int64_t do_st, do_sh;
  char* dq;
  int64_t dq_st, dq_sh;
  char* dk;
  int64_t dk_st, dk_sh;
  char* dv;
  int64_t dv_st, dv_sh;
  const int32_t* cu_q;
  const int32_t* cu_k;
  float scale, scale_log2;  // c, c log2 e
  int32_t causal;
  int32_t num_seqs, total_q, total_k, num_heads, num_kv_heads;
  int32_t q_tiles, k_tiles;  // workgroups per head of the two launches (and part)
  int32_t q_rows;            // queries of a workgroup of the first launch
  int32_t window;            // > 0: one launch, no sequence is longer than this
  int32_t parts;             // workgroups that share a block of keys' queries
  float* part;               // parts > 1: their sums, [block][part][kv head][wave][D / 8][64] x 4
  float* lse;                // [num_heads][total_q]: log2 sum 2^(c log2 e s), f16: - kF16Lift
  float* delta;              // [num_heads][total_q]: -delta
  float* top;                // f16: [num_heads][total_q], largest |dout| of the row (held_top)
};

constexpr int kBwdThreads = 256;

template <bool kBF16>
__device__ inline f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
  if constexpr (kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// One 4-byte global -> LDS copy per lane (lane l's word lands at lds + 4 l);
// wait states as in dma16.
__device__ inline void dma4(uint32_t off, const void* base, uint32_t lds) {
  asm volatile("s_nop 4\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(base), "{m0}"(lds)
               : "memory");
}

// In front of a loop with copies under way: the compiler has to see that the
// registers loaded before it are there.  It does not know of the waits in inline
// assembly, and puts its own in front of their first use, in the loop, where every
// turn waits for the copies just requested (dk and dv of 4 sequences of 600 to 2000
// rows, 32 heads over 4 of 64, 153 us; 145 to 152 so).
__device__ inline void loads_done() {
  asm volatile("" ::: "memory");
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0) alone
  __builtin_amdgcn_sched_barrier(0);
}

// A sequence's rows [row, row + len) of `total` packed rows: what cu says (a and
// b, its ends), held to rows that there are.
struct SeqRows {
  int row, len;
};
__device__ inline SeqRows seq_rows(int a, int b, int total) {
  a = min(max(a, 0), total);
  return {a, min(max(b, a), total) - a};
}

// Orders of a launch's blocks.  kInTurn: sequence after sequence.  The others, up to
// 128 sequences, are by the work under a causal mask, the most first, so that no
// long block starts late: a sequence's n-th block has the keys of n blocks
// (kByIndex: dq), and its n-th from the end the queries of n (kFromEnd: dk, dv).  32
// sequences of 50 to 450 rows take 46 us for dk and dv so and 53.5 in turn; 4 of 600
// to 2000 in f16 107 for dq and 119 (with a sequence's last block first).
enum BwdOrder { kInTurn, kByIndex, kFromEnd };

// The `tile`-th block of kRows rows of one side in that order, with its sequence's
// rows on both.  found: there is one; otherwise `blocks` is how many there are.  The
// ends of 128 sequences, both sides', are requested at once (64 in turn, and the
// found sequence's again, took 160 sequences of 14 heads 27.1 us for dq and 30.9
// for dk and dv instead of 26.3 and 29.2).
struct BwdBlock {
  bool found;
  int index;   // of the block in its sequence
  int blocks;
  int place;   // found: its number in turn
  SeqRows rows, other;
};
template <int kRows, BwdOrder kOrder>
__device__ inline BwdBlock find_block(const int32_t* cu, const int32_t* cu_other, int num_seqs,
                                      int total, int total_other, int tile) {
  const int lane = threadIdx.x & 63;
  auto pick = [](int x, int at) { return __builtin_amdgcn_readlane(x, at); };
  int before = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += 128) {
    int end[2][4], nb[2], upto[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const int s = min(s0 + 64 * n + lane, num_seqs - 1);
      end[n][0] = cu[s];
      end[n][1] = cu[s + 1];
      end[n][2] = cu_other[s];
      end[n][3] = cu_other[s + 1];
    }
    SeqRows mine[2], theirs[2];
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      mine[n] = seq_rows(end[n][0], end[n][1], total);
      theirs[n] = seq_rows(end[n][2], end[n][3], total_other);
      nb[n] = s0 + 64 * n + lane < num_seqs ? (mine[n].len + kRows - 1) / kRows : 0;
      upto[n] = wave_scan(nb[n]);
    }
    const int c0 = pick(upto[0], 63), here = c0 + pick(upto[1], 63);
    if (tile >= before + here) {
      before += here;
      continue;
    }
    int left = tile - before, n, at, index;
    if (kOrder == kInTurn || num_seqs > 128) {
      n = left >= c0;
      left -= n ? c0 : 0;
      at = __builtin_ctzll(__builtin_amdgcn_ballot_w64((n ? upto[1] : upto[0]) > left));
      index = left - pick(n ? upto[1] : upto[0], at) + pick(n ? nb[1] : nb[0], at);
    } else {
      // Level by level of blocks that sequences have, those with the same sequences
      // at once.
      // (Floats hold the counts: 2^24 blocks of a sequence are 2^30 rows.)
      int level = __builtin_amdgcn_readfirstlane((int)group_max<64>((float)max(nb[0], nb[1])));
      uint64_t m[2];
      int c[2];
      while (true) {
        int under = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          m[i] = __builtin_amdgcn_ballot_w64(nb[i] >= level);
          c[i] = __builtin_popcountll(m[i]);
          under = max(under, nb[i] < level ? nb[i] : 0);
        }
        under = __builtin_amdgcn_readfirstlane((int)group_max<64>((float)under));
        const int run = (c[0] + c[1]) * (level - under);
        if (left < run) break;
        left -= run;
        level = under;
      }
      level -= left / (c[0] + c[1]);
      left %= c[0] + c[1];
      n = left >= c[0];
      left -= n ? c[0] : 0;
      const uint64_t in = n ? m[1] : m[0];
      const int rank = __builtin_amdgcn_mbcnt_hi((uint32_t)(in >> 32),
                                                 __builtin_amdgcn_mbcnt_lo((uint32_t)in, 0));
      at = __builtin_ctzll(__builtin_amdgcn_ballot_w64((in >> lane & 1) != 0 && rank == left));
      index = kOrder == kByIndex ? level - 1 : pick(n ? nb[1] : nb[0], at) - level;
    }
    const SeqRows& a = n ? mine[1] : mine[0];
    const SeqRows& b = n ? theirs[1] : theirs[0];
    return {true, index, 0,
            before + (n ? c0 : 0) + pick(n ? upto[1] : upto[0], at) - pick(n ? nb[1] : nb[0], at) + index,
            {pick(a.row, at), pick(a.len, at)}, {pick(b.row, at), pick(b.len, at)}};
  }
  return {false, 0, before, 0, {}, {}};
}

// Zeros for one head of the rows that belong to no sequence (in front of the
// first and behind the last), shared among the workgroups that found no block.
template <int D, int kThreads>
__device__ inline void zero_rest(const int32_t* cu, int num_seqs, int total, char* g, int64_t st,
                                 int64_t off, int nth, int of) {
  const int lo = num_seqs > 0 ? min(max(cu[0], 0), total) : 0;
  const int hi = num_seqs > 0 ? min(max(cu[num_seqs], lo), total) : 0;
  const int rest = lo + total - hi;
  constexpr int CPR = D / 8, RPB = kThreads / CPR;
  for (int64_t i = (int64_t)nth * RPB + threadIdx.x / CPR; i < rest; i += (int64_t)of * RPB) {
    const int64_t row = i < lo ? i : hi + (i - lo);
    st16(g + row * st + off + (threadIdx.x % CPR) * 16, make_uint4(0, 0, 0, 0));
  }
}

// The tiles' swizzle: the 16-byte chunk c of row r sits at chunk c ^ this.  Both
// kinds of reads below find their 256 bytes a cycle in distinct banks: 16 rows of
// one chunk (A operands), and 4 rows of 4 chunks (transposed; with the forward
// kernel's swizzle these take two cycles).  Depends on r % 16 only.
template <int D>
__device__ inline int bwd_swz(int r) {
  if constexpr (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
  return ((r & 2) << 1) | ((r >> 1) & 2) | ((r >> 3) & 1);
}

// A wave's share of the copies of kRows rows of one tensor into an LDS tile: NI
// copies of 1 KiB.  A copy holds up its wave for some 70 cycles (more when all of
// a CU's waves issue theirs at once: 64 bytes a cycle go to a CU), so a step's are
// spread among its matrix products.  Rows past the sequence's last repeat it; what
// they make is masked.  Lane offsets are 32-bit, what is left of an address is
// uniform (64-bit lane addresses, formed for each copy, took 300 cycles a step).
template <int D, int kWaves, int kRows>
struct TileCopy {
  static constexpr int CPR = D / 8, RPI = 64 / CPR;
  static constexpr int NI = kRows * D * 2 / 1024 / kWaves;
  static_assert(NI >= 1 && NI <= 4, "a wave copies 1 to 4 KiB");
  uint32_t chunk;  // the lane's, in bytes, in copy 0; copy i's differs by exactly i chunks' bits
  int row;         // its row in copy 0
  __device__ inline TileCopy(int wave, int lane) {
    row = wave * NI * RPI + lane / CPR;
    chunk = (uint32_t)(((lane % CPR) ^ bwd_swz<D>(row)) << 4);
  }
  // Copy i of the tile whose row 0 is at src (rows st bytes apart, row `last` the
  // last one there is; row_st is row * st).
  __device__ inline void one(int i, const char* src, uint32_t st, uint32_t row_st, int last,
                             uint32_t lds, int wave) const {
    if (last >= kRows - 1) {
      dma16(row_st + (chunk ^ (i << 4)), src + (uint32_t)(i * RPI) * st,
            lds + (uint32_t)((wave * NI + i) * 1024));
    } else {
      const uint32_t r = (uint32_t)min(row + i * RPI, last);
      dma16(r * st + (chunk ^ (i << 4)), src, lds + (uint32_t)((wave * NI + i) * 1024));
    }
  }
};

// A wave's LDS offsets in a tile: of row l % 32's chunk for 8 elements of the
// l / 32 half (A rows), and of the transposed reads.
template <int D>
struct TileAt {
  int row, row0;  // row % 32 in bytes; first chunk, swizzled
  int tr, tr0;    // the same of the transposed read (rows 4 (l / 32) + ...)
  __device__ inline explicit TileAt(int lane) {
    constexpr int ROWB = D * 2;
    const int r = lane & 31, h = lane >> 5, r16 = lane & 15, g = lane >> 4;
    row = r * ROWB;
    row0 = (h ^ bwd_swz<D>(r)) << 4;
    const int t = 4 * h + (r16 >> 2);
    tr = t * ROWB + ((r16 & 1) << 3);
    tr0 = ((2 * (g & 1) + ((r16 >> 1) & 1)) ^ bwd_swz<D>(t)) << 4;
  }
  // Keeps what the reads below add to these from being held in registers through
  // a loop, where it makes the compiler spill.
  __device__ inline void rebuild() { asm volatile("" : "+v"(row0), "+v"(tr0), "+v"(row), "+v"(tr)); }
  // Rows 32 sub + l % 32, elements 16 step + 8 (l / 32) ... + 7.
  __device__ inline uint4 a(const char* tile, int sub, int step) const {
    return lds_read16(tile, sub * 32 * D * 2 + row + (row0 ^ (step << 5)));
  }
  // Element 32 dt + l % 32 of rows 32 sub + 16 half + {0-3, 8-11} + 4 (l / 32).
  __device__ inline uint4 at(const char* tile, int sub, int half, int dt) const {
    const int off = (sub * 32 + half * 16) * D * 2 + tr;
    const uint2 lo = __builtin_bit_cast(uint2, lds_read_tr(tile, off + (tr0 ^ (dt << 6))));
    const uint2 hi =
        __builtin_bit_cast(uint2, lds_read_tr(tile, off + 8 * D * 2 + (tr0 ^ (D == 128 ? 32 : 16) ^ (dt << 6))));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
};

// Two floats to a pair of 16-bit elements, rounded to nearest even, in one
// instruction (f16 too).
template <bool kBF16>
__device__ inline uint32_t pack_pair(float lo, float hi) {
  if constexpr (kBF16) {
    return Mma<true>::pack2(lo, hi);
  } else {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2{lo, hi}), f16x2_t));
  }
}

// Eight accumulator values of one lane (rows 16 half + {0-3, 8-11} + 4 (l / 32))
// as a B operand.
template <bool kBF16>
__device__ inline uint4 pack_b(const f32x16_t& x, int half) {
  return make_uint4(pack_pair<kBF16>(x[8 * half], x[8 * half + 1]),
                    pack_pair<kBF16>(x[8 * half + 2], x[8 * half + 3]),
                    pack_pair<kBF16>(x[8 * half + 4], x[8 * half + 5]),
                    pack_pair<kBF16>(x[8 * half + 6], x[8 * half + 7]));
}

// A wave's accumulators to LDS, 16 bytes a lane at a time, and a weighted sum with
// what lies there.
template <int DT>
__device__ inline void put_acc(const f32x16_t (&acc)[DT], char* s, int lane) {
#pragma unroll
  for (int n = 0; n < 4 * DT; ++n) {
    const f32x16_t& x = acc[n / 4];
    const int i = n % 4 * 4;
    *reinterpret_cast<f32x4_t*>(s + (n * 64 + lane) * 16) = f32x4_t{x[i], x[i + 1], x[i + 2], x[i + 3]};
  }
}
template <int DT>
__device__ inline void add_acc(f32x16_t (&acc)[DT], float mine, const char* s, float theirs,
                               int lane) {
#pragma unroll
  for (int n = 0; n < 4 * DT; ++n) {
    const f32x4_t x = *reinterpret_cast<const f32x4_t*>(s + (n * 64 + lane) * 16);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      acc[n / 4][n % 4 * 4 + i] = fmaf(x[i], theirs, acc[n / 4][n % 4 * 4 + i] * mine);
  }
}

// Writes a wave's gradient, accumulators [D][32 rows] times `mul`, as rows of
// 16 bits: through the wave's own 32 rows of LDS, so that each store
// instruction writes whole rows.
template <bool kBF16, int D>
__device__ inline void write_rows(const f32x16_t (&acc)[D / 32], float mul, char* s, char* dst,
                                  int64_t st, int row0, int rows, int lane) {
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPS = 64 / CPR;
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint2 w = make_uint2(pack_pair<kBF16>(acc[dt][4 * j] * mul, acc[dt][4 * j + 1] * mul),
                                 pack_pair<kBF16>(acc[dt][4 * j + 2] * mul, acc[dt][4 * j + 3] * mul));
      *reinterpret_cast<uint2*>(s + r * ROWB + (((4 * dt + j) ^ (r % CPR)) << 4) + h * 8) = w;
    }
  __builtin_amdgcn_wave_barrier();
#pragma unroll 4
  for (int i = 0; i < 32 / RPS; ++i) {
    const int rw = i * RPS + lane / CPR, c = lane % CPR;
    const uint4 x = lds_read16(s, rw * ROWB + ((c ^ (rw % CPR)) << 4));
    if (row0 + rw < rows) st16_nt(dst + (int64_t)(row0 + rw) * st + c * 16, x);
  }
}

// 2^e with e the exponent of x, 1 for 0, infinities and NaN; held to exponents
// whose inverse and square are representable.
__device__ inline int top_exponent(float x) {
  const int e = (int)(__float_as_uint(x) >> 23 & 255);
  return e == 0 || e == 255 ? 0 : min(max(e - 127, -40), 40);
}
__device__ inline float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// f16 holds 2^-24 .. 65504: P times this in dv's product keeps the small
// probabilities of long contexts out of its subnormals.
constexpr int kF16Lift = 14;

// f16: dS is held as P (dP - delta) 2^-e, e the exponent of the row's largest |dout|.
// Values of v in the ten thousands would take that past 65504, to infinity, and a
// finite gradient with it.  So |dP - delta| 2^-e is held below 2^15: where `big`, the
// largest one a lane has met, is not, e is raised, as the maximum is; masked keys do not
// count.  (The test takes 4 sequences of 600 to 2000 rows, 32 heads over 4 of 64, from
// 239.5 to 244.5 us a gradient.)
__device__ inline bool out_of_range(float big, int e) { return big >= pow2(e + 15); }
__device__ inline int raised(float big, int e) { return max(e, top_exponent(max_xor32(big)) - 14); }
// What stands for the row's largest |dout| where the exponent was raised.
__device__ inline float held_top(float top, int e) { return e > top_exponent(top) ? pow2(e) : top; }

// ---------------------------------------------------------------------- dq
// f16 (as for dk): dS is rounded to 16 bits, and a gradient of 1e-4 spread over
// a thousand keys would fall among f16's subnormals.  So P is scaled by 2^-e, e
// the exponent of the row's largest |dout| (or more: out_of_range), through the
// exponential's argument, and the maximum is followed without slack, which keeps dS
// near v's size.
//
// kSplit: a wave takes 32 keys of each tile for its 32 queries, its neighbour the
// other 32, and their sums meet in LDS at the end: launches whose blocks of 128
// queries would leave the chip half idle take blocks of 64 in less time.
template <bool kBF16, int D, bool kSplit>
__global__ __launch_bounds__(kBwdThreads, D == 64 ? 3 : 2) void varlen_dq_kernel(VarlenBwdParams p) {
  constexpr int kTile = 64;  // keys
  constexpr int kRows = kSplit ? 64 : 128;  // queries of a workgroup, 32 a wave
  constexpr int ROWB = D * 2, TILE_B = kTile * ROWB, DS = D / 16, DT = D / 32;
  __shared__ __align__(1024) char s_kv[2 * 2 * TILE_B];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  // Consecutive workgroups, which run on different XCDs, take different kv heads.
  const int tile = (int)(blockIdx.x / (unsigned)p.num_heads);
  const int pick = (int)(blockIdx.x % (unsigned)p.num_heads);
  const int group = p.num_heads / p.num_kv_heads;
  const int kv = pick % p.num_kv_heads, head = kv * group + pick / p.num_kv_heads;
  const BwdBlock blk = find_block<kRows, kByIndex>(p.cu_q, p.cu_k, p.num_seqs, p.total_q, p.total_k, tile);
  if (!blk.found) {
    zero_rest<D, kBwdThreads>(p.cu_q, p.num_seqs, p.total_q, p.dq, p.dq_st, head * p.dq_sh,
                              tile - blk.blocks, p.q_tiles - blk.blocks);
    return;
  }
  const SeqRows qs = blk.rows, ks = blk.other;
  const int i0 = blk.index * kRows;  // the block's first query
  const int ahead = ks.len - qs.len;         // causal: query i sees keys j <= i + ahead
  const int kend = p.causal ? min(max(ahead + min(i0 + kRows, qs.len), 0), ks.len) : ks.len;
  const int tiles = (kend + kTile - 1) / kTile;
  const char* const kp = p.k + (int64_t)ks.row * p.k_st + kv * p.k_sh;
  const char* const vp = p.v + (int64_t)ks.row * p.v_st + kv * p.v_sh;
  const uint32_t lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_kv);
  using Copy = TileCopy<D, 4, kTile>;
  const Copy copy(wave, lane);
  const uint32_t k_row = (uint32_t)copy.row * (uint32_t)p.k_st;
  const uint32_t v_row = (uint32_t)copy.row * (uint32_t)p.v_st;
  // Copy n of tile t: K's, then V's.
  auto issue = [&](int t, int n) {
    const uint32_t to = lds + (uint32_t)((t & 1) * 2 * TILE_B);
    const int last = ks.len - 1 - t * kTile;
    if (n < Copy::NI)
      copy.one(n, kp + (int64_t)(t * kTile) * p.k_st, (uint32_t)p.k_st, k_row, last, to, wave);
    else
      copy.one(n - Copy::NI, vp + (int64_t)(t * kTile) * p.v_st, (uint32_t)p.v_st, v_row, last,
               to + TILE_B, wave);
  };
  if (tiles > 0) {
#pragma unroll
    for (int n = 0; n < 2 * Copy::NI; ++n) issue(0, n);
  }

  // The wave's 32 queries (rows past the sequence repeat its last).
  const int wrow = i0 + 32 * (kSplit ? wave >> 1 : wave);
  const int row = wrow + l32, at = qs.row + min(row, qs.len - 1);
  uint4 qreg[DS], doreg[DS];
  float delta = 0.f, top = 0.f;
  int e = 0;
  {
    const char* const qp = p.q + at * p.q_st + head * p.q_sh + half * 16;
    const char* const dp = p.dout + at * p.do_st + head * p.do_sh + half * 16;
    const char* const op = p.out + at * p.o_st + head * p.o_sh + half * 16;
    uint4 oreg[DS];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) doreg[ds] = ld16(dp + ds * 32);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) oreg[ds] = ld16(op + ds * 32);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qreg[ds] = ld16(qp + ds * 32);
    // Tensor after tensor, so that the four loads that share a row's lines follow one
    // another (in turn: 54 us for 32 sequences of 50 to 450 rows instead of 50), and
    // all of them now (left to itself the compiler requests q once delta is done).
    __builtin_amdgcn_sched_barrier(0);
    using ET = std::conditional_t<kBF16, BF16, F16>;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      float a[8], b[8];
      ET::unpack(doreg[ds], a);
      ET::unpack(oreg[ds], b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        delta = fmaf(a[i], b[i], delta);
        if constexpr (!kBF16) top = fmaxf(top, fabsf(a[i]));
      }
    }
    delta = sum_xor32(delta);
    if constexpr (!kBF16) {
      top = max_xor32(top);
      e = top_exponent(top);
    }
  }

  TileAt<D> ta(lane);
  const int lim = p.causal ? min(ks.len, ahead + row + 1) : ks.len;  // keys the lane's query sees
  const int lim_lo = p.causal ? min(ks.len, ahead + wrow + 1) : ks.len;
  const int lim_hi = p.causal ? min(ks.len, ahead + wrow + 32) : ks.len;
  constexpr float kSlack = kBF16 ? kLazy : 0.f;
  float m = -1.0e30f, l = 0.f;
  f32x16_t acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16_t{};

  loads_done();
  for (int t = 0; t < tiles; ++t) {
    wait_vmcnt<0>();
    __syncthreads();
    const bool more = t + 1 < tiles;
    const char* const sk = s_kv + (t & 1) * 2 * TILE_B;
    const char* const sv = sk + TILE_B;
#pragma unroll
    for (int turn = 0; turn < (kSplit ? 1 : 2); ++turn) {
      const int sub = kSplit ? wave & 1 : turn;
      constexpr int kTurnCopies = kSplit ? 2 * Copy::NI : Copy::NI;
      const int j0 = t * kTile + 32 * sub;
      if (j0 >= lim_hi) {  // no query of the wave sees these
        if (more) {
#pragma unroll
          for (int n = 0; n < kTurnCopies; ++n) issue(t + 1, turn * Copy::NI + n);
        }
        continue;
      }
      ta.rebuild();
      // S and dP in turn, operands requested kAhead products before their own, the
      // next tile's copies (K's beside the first 32 keys, V's beside the others)
      // between them.
      constexpr int kAhead = 4;
      uint4 op[kAhead];
      auto request = [&](int n) {
        if (n < 2 * DS) op[n % kAhead] = ta.a(n & 1 ? sv : sk, sub, n / 2);
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) request(n);
      f32x16_t s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = -delta;
      // (The products ahead of the exponentials of the SIMD's other waves: a sequence of
      // 8192 rows 388 us instead of 402, and 550 instead of 578 for dk and dv.)
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int n = 0; n < 2 * DS; ++n) {
        if (n & 1)
          dp = mfma32<kBF16>(op[n % kAhead], doreg[n / 2], dp);
        else
          s = mfma32<kBF16>(op[n % kAhead], qreg[n / 2], s);
        request(n + kAhead);
        constexpr int kEvery = 2 * DS / kTurnCopies;
        if (n % kEvery == kEvery - 1 && more) issue(t + 1, turn * Copy::NI + n / kEvery);
      }
      __builtin_amdgcn_s_setprio(0);
      if (j0 + 32 > lim_lo) {
        const int rel = lim - j0 - 4 * half;  // key 8 (i / 4) + i % 4 of the lane is seen iff < rel
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 >= rel) {
            s[i] = -INFINITY;
            if constexpr (!kBF16) dp[i] = 0.f;
          }
      }
      float mx = s[0], big = 0.f;
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      mx = max_xor32(mx) * p.scale_log2;
      bool up = mx > m + kSlack;
      if constexpr (!kBF16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(dp[i]));
        up = up || out_of_range(big, e);
      }
      if (__builtin_amdgcn_ballot_w64(up) != 0) {
        const float mn = fmaxf(m, mx);
        float alpha = m - mn;
        m = mn;
        if constexpr (!kBF16) {
          const int en = raised(big, e);
          alpha += (float)(e - en);
          e = en;
        }
        alpha = fast_exp2(alpha);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      const float base = kBF16 ? m : m + (float)e;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = fast_exp2(fmaf(s[i], p.scale_log2, -base));
        l += s[i];
        dp[i] *= s[i];
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint4 b = pack_b<kBF16>(dp, hf);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] = mfma32<kBF16>(ta.at(sk, sub, hf, dt), b, acc[dt]);
      }
    }
  }
  l = sum_xor32(l);
  __syncthreads();  // every wave is done with the tiles
  float base = kBF16 ? m : m + (float)e;  // what the sums are relative to
  // Where the wave's rows go out from, and in a split block its neighbour's sums lie.
  char* const s_x = s_kv + (kSplit ? (wave >> 1) * (DT * 4 + 1) * 1024 : wave * 32 * ROWB);
  if constexpr (kSplit) {
    float4* const s_ml = reinterpret_cast<float4*>(s_x + DT * 4 * 1024);
    if (wave & 1) {
      put_acc<DT>(acc, s_x, lane);
      s_ml[lane] = make_float4(base, l, __int_as_float(e), 0.f);
    }
    __syncthreads();
    if (wave & 1) return;
    const float4 o = s_ml[lane];
    const float mn = fmaxf(base, o.x), mine = fast_exp2(base - mn), theirs = fast_exp2(o.x - mn);
    base = mn;
    l = l * mine + o.y * theirs;
    e = max(e, __float_as_int(o.z));
    add_acc<DT>(acc, mine, s_x, theirs, lane);
  }
  if (half == 0 && row < qs.len) {
    const int64_t w = (int64_t)head * p.total_q + at;
    p.lse[w] = l > 0.f ? base + __builtin_amdgcn_logf(l) - (kBF16 ? 0.f : (float)kF16Lift) : INFINITY;
    p.delta[w] = -delta;
    if constexpr (!kBF16) p.top[w] = held_top(top, e);
  }
  write_rows<kBF16, D>(acc, l > 0.f ? p.scale / l : 0.f, s_x,
                       p.dq + (int64_t)qs.row * p.dq_st + head * p.dq_sh, p.dq_st, wrow, qs.len,
                       lane);
}

// ------------------------------------------------------------------- dk, dv
// A wave's 32 keys of dv (role 0) or dk.
template <bool kBF16, int D>
__device__ inline void write_dkv(const VarlenBwdParams& p, const f32x16_t (&acc)[D / 32], float mul,
                                 char* s, int role, const SeqRows& ks, int kv, int key, int lane) {
  if (role == 0)
    write_rows<kBF16, D>(acc, mul, s, p.dv + (int64_t)ks.row * p.dv_st + kv * p.dv_sh, p.dv_st, key,
                         ks.len, lane);
  else
    write_rows<kBF16, D>(acc, mul, s, p.dk + (int64_t)ks.row * p.dk_st + kv * p.dk_sh, p.dk_st, key,
                         ks.len, lane);
}

// A workgroup's share of the gradients of a block of 64 keys of one kv head: the
// tiles of 64 queries, head by head of the group, that see some of them.
constexpr int kDkvKeys = 64;
constexpr int kDkvTile = 64;
struct DkvBlock {
  bool found;
  SeqRows qs, ks;
  int j0;      // the block's first key
  int t0, nt;  // tiles of queries that see it
  int steps;   // nt, for every head of the group
  int empty;   // not found: the tiles that are there
  int place;   // its number in turn
};
template <BwdOrder kOrder>
__device__ inline DkvBlock dkv_block(const VarlenBwdParams& p, int tile) {
  const BwdBlock blk =
      find_block<kDkvKeys, kOrder>(p.cu_k, p.cu_q, p.num_seqs, p.total_k, p.total_q, tile);
  DkvBlock b{};
  b.found = blk.found;
  b.empty = blk.blocks;
  b.place = blk.place;
  if (!blk.found) return b;
  b.qs = blk.other;
  b.ks = blk.rows;
  b.j0 = blk.index * kDkvKeys;
  b.t0 = p.causal ? max(b.j0 - (b.ks.len - b.qs.len), 0) / kDkvTile : 0;
  b.nt = max((b.qs.len + kDkvTile - 1) / kDkvTile - b.t0, 0);
  b.steps = b.nt * (p.num_heads / p.num_kv_heads);
  return b;
}
// The first step of part n of `parts`.
__device__ inline int part_begin(int steps, int n, int parts) {
  return (int)((int64_t)steps * n / parts);
}
// Zeros for the rows outside the sequences, by the workgroups without a block.
template <int D>
__device__ inline void zero_rest_kv(const VarlenBwdParams& p, int kv, int nth, int of) {
  zero_rest<D, 256>(p.cu_k, p.num_seqs, p.total_k, p.dk, p.dk_st, kv * p.dk_sh, nth, of);
  zero_rest<D, 256>(p.cu_k, p.num_seqs, p.total_k, p.dv, p.dv_st, kv * p.dv_sh, nth, of);
}

// Two pairs of waves, 32 keys a pair.  Of a tile the first wave of a pair forms P
// and dS of the first 32 queries, the second of the others; they exchange through
// LDS what the other one needs, and the first adds up dv of all 64, the second dk.
// So a wave holds one gradient beside its K and V operands and has registers left
// for the operands ahead.  (A wave that adds up both has none at head_dim 128: its
// step of 32 queries took 3600 cycles for 1024 of matrix work.)  Eight waves that
// add up both gradients of 128 keys, two for each 32 keys, are faster on one long
// sequence and slower where there are few blocks: 8192 rows 530 us against 578 (550
// with the priorities below), windows of 104 rows 56 against 30, one sequence of 420
// rows 31 against 25.
//
// kParts: the block's steps are shared among several workgroups, whose sums a
// third launch adds up (varlen_dkv_sum_kernel).
template <bool kBF16, int D, bool kParts>
__global__ __launch_bounds__(256, D == 64 ? 3 : 2) void varlen_dkv_kernel(VarlenBwdParams p) {
  constexpr int kWaves = 4, kThreads = 256;
  constexpr int kTile = kDkvTile, ROWB = D * 2, TILE_B = kTile * ROWB, DS = D / 16, DT = D / 32;
  constexpr int kAhead = D == 128 ? 6 : 4;
  __shared__ __align__(1024) char s_qd[2 * 2 * TILE_B];
  __shared__ __align__(16) float s_st[2 * 2 * kTile];  // a stage's lse, delta
  __shared__ __align__(16) char s_ex[kWaves * 2048];   // what a wave hands over
  __shared__ float s_top[kWaves];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int pair = wave >> 1, role = wave & 1;  // role 0: first 32 queries, dv
  const int kv = (int)(blockIdx.x % (unsigned)p.num_kv_heads);
  const int unit = (int)(blockIdx.x / (unsigned)p.num_kv_heads);
  const int parts = kParts ? p.parts : 1;
  const int tile = unit / parts, part = unit % parts;
  const int group = p.num_heads / p.num_kv_heads;
  const DkvBlock blk = dkv_block<kFromEnd>(p, tile);
  if (!blk.found) {
    if constexpr (!kParts) zero_rest_kv<D>(p, kv, tile - blk.empty, p.k_tiles - blk.empty);
    return;
  }
  const SeqRows qs = blk.qs, ks = blk.ks;
  const int j0 = blk.j0, t0 = blk.t0, nt = blk.nt;
  const int ahead = ks.len - qs.len;
  const int begin = kParts ? part_begin(blk.steps, part, parts) : 0;
  const int steps = (kParts ? part_begin(blk.steps, part + 1, parts) : blk.steps) - begin;
  // (Lengths that fall and rise again make more blocks than there is room for.)
  if (kParts && (steps == 0 || blk.place >= p.k_tiles)) return;

  const uint32_t lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_qd);
  const uint32_t lds_st = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_st);
  using Copy = TileCopy<D, kWaves, kTile>;
  constexpr int kCopies = 2 * Copy::NI + 1;
  const Copy copy(wave, lane);
  const uint32_t q_row = (uint32_t)copy.row * (uint32_t)p.q_st;
  const uint32_t do_row = (uint32_t)copy.row * (uint32_t)p.do_st;
  // The tile requested next: its number, the rows behind its first, its sources.
  int ti = nt > 0 ? begin % nt : 0, last = 0;
  const char *next_q, *next_do;
  const float* next_st;  // lse (wave 0) or delta
  {
    const int head = kv * group + (nt > 0 ? begin / nt : 0), base = qs.row + (t0 + ti) * kTile;
    next_q = p.q + (int64_t)base * p.q_st + head * p.q_sh;
    next_do = p.dout + (int64_t)base * p.do_st + head * p.do_sh;
    next_st = (wave == 0 ? p.lse : p.delta) + (int64_t)head * p.total_q + base;
    last = qs.len - 1 - (t0 + ti) * kTile;
  }
  const int64_t q_step = kTile * p.q_st, do_step = kTile * p.do_st;
  const int64_t q_head = p.q_sh - (nt - 1) * q_step, do_head = p.do_sh - (nt - 1) * do_step;
  const int64_t st_head = (int64_t)p.total_q - (int64_t)(nt - 1) * kTile;
  auto next_tile = [&]() {  // (behind a tile's copies)
    const bool wrap = ++ti == nt;  // on to the next head's first tile
    next_q += wrap ? q_head : q_step;
    next_do += wrap ? do_head : do_step;
    next_st += wrap ? st_head : kTile;
    last = wrap ? qs.len - 1 - t0 * kTile : last - kTile;
    ti = wrap ? 0 : ti;
  };
  // Its copy n: lse (wave 0) or delta (wave 1), Q's, dO's.
  auto issue = [&](int stage, int n) {
    const uint32_t to = lds + (uint32_t)(stage * 2 * TILE_B);
    if (n == 0) {
      if (wave < 2)
        dma4((uint32_t)min(lane, last) * 4, next_st,
             lds_st + (uint32_t)((stage * 2 + wave) * kTile * 4));
    } else if (n <= Copy::NI) {
      copy.one(n - 1, next_q, (uint32_t)p.q_st, q_row, last, to, wave);
    } else {
      copy.one(n - 1 - Copy::NI, next_do, (uint32_t)p.do_st, do_row, last, to + TILE_B, wave);
    }
  };
  if (steps > 0) {
#pragma unroll
    for (int n = 0; n < kCopies; ++n) issue(0, n);
  }

  const int wkey = j0 + 32 * pair, key = wkey + l32;
  const int at = ks.row + min(key, ks.len - 1);
  uint4 kreg[DS], vreg[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds)
    kreg[ds] = ld16(p.k + at * p.k_st + kv * p.k_sh + half * 16 + ds * 32);
#pragma unroll
  for (int ds = 0; ds < DS; ++ds)
    vreg[ds] = ld16(p.v + at * p.v_st + kv * p.v_sh + half * 16 + ds * 32);
  // f16: dS is scaled by the largest |dout| of the queries (see above).
  float lift = 1.f, lower = 1.f;
  if constexpr (!kBF16) {
    float top = 0.f;
    for (int g = 0; g < group; ++g)
      for (int i = threadIdx.x; i < qs.len; i += kThreads)
        top = fmaxf(top, p.top[(int64_t)(kv * group + g) * p.total_q + qs.row + i]);
    top = group_max<64>(top);
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kWaves; ++w) top = fmaxf(top, s_top[w]);
    const int e = top_exponent(top);
    lift = pow2(-e - kF16Lift);
    lower = pow2(e);
  }

  // The lane's LDS addresses: of the 8 elements of step n of S's rows (dO's for dP
  // lie TILE_B further on), and of the transposed reads for the wave's gradient
  // (role 0: dO, dv), whose other 32 rows differ in one bit.  In registers, with a
  // stage's offset in the instruction: formed for each read they took 600 cycles
  // of a step.
  static_assert((32 * ROWB & (32 * ROWB - 1)) == 0 && 64 * ROWB <= TILE_B, "the rows' bit");
  int a_at[DS], t_lo[DT], t_hi[DT];
  {
    const TileAt<D> ta(lane);
#pragma unroll
    for (int n = 0; n < DS; ++n) a_at[n] = role * 32 * ROWB + ta.row + (ta.row0 ^ (n << 5));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
      const int of = role * 32 * ROWB + (role == 0 ? TILE_B : 0);
      t_lo[dt] = of + ta.tr + (ta.tr0 ^ (dt << 6));
      t_hi[dt] = of + ta.tr + 8 * ROWB + (ta.tr0 ^ (D == 128 ? 32 : 16) ^ (dt << 6));
    }
  }
  f32x16_t acc[DT];  // dv (role 0) or dk
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16_t{};
  int tq = nt > 0 ? begin % nt : 0;  // the step's tile of queries, from t0
  const int st_at = 32 * role + 4 * half;
  auto step = [&](auto stage_c, int it) {
    constexpr int kStage = decltype(stage_c)::value;
    constexpr int kAt = kStage * 2 * TILE_B;
    wait_vmcnt<0>();
    __syncthreads();
    const bool more = it + 1 < steps;
    if (more) next_tile();
    const int base = (t0 + tq) * kTile;
    if (++tq == nt) tq = 0;
    // Whether any of 32 queries sees a key of the pair.
    auto seen = [&](int r) {
      return base + 32 * r < qs.len && (!p.causal || base + 32 * r + 31 + ahead >= wkey);
    };
    uint4 op[kAhead];  // A operands requested ahead
    auto sums = [&](int n, int other) {  // operand n of the sum over 32 queries
      const int x = other * 32 * ROWB;
      const uint2 lo = __builtin_bit_cast(uint2, lds_read_tr(s_qd + kAt + n / DT * 16 * ROWB, t_lo[n % DT] ^ x));
      const uint2 hi = __builtin_bit_cast(uint2, lds_read_tr(s_qd + kAt + n / DT * 16 * ROWB, t_hi[n % DT] ^ x));
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };
    uint4 own[2];  // P (role 0) or dS of the wave's own queries, as B operands
    const bool mine = seen(role);
    if (mine) {
      const int i0 = base + 32 * role;
      const float* const st = s_st + kStage * 2 * kTile + st_at;
      // S and dP in turn, the next tile's copies between them.
      auto request = [&](int n) {
        if (n < 2 * DS) op[n % kAhead] = lds_read16(s_qd + kAt + (n & 1) * TILE_B, a_at[n / 2]);
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) request(n);
      f32x16_t s = {}, dp;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4_t d = *reinterpret_cast<const f32x4_t*>(st + kTile + 8 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) dp[4 * j + i] = d[i];
      }
      __builtin_amdgcn_s_setprio(1);
#pragma unroll
      for (int n = 0; n < 2 * DS; ++n) {
        if (n & 1)
          dp = mfma32<kBF16>(op[n % kAhead], vreg[n / 2], dp);
        else
          s = mfma32<kBF16>(op[n % kAhead], kreg[n / 2], s);
        request(n + kAhead);
        constexpr int kEvery = (2 * DS) / (kCopies - 1);
        if (more) {
          if (n == 0) issue(kStage ^ 1, 0);
          if (n % kEvery == kEvery - 1) issue(kStage ^ 1, 1 + n / kEvery);
        }
      }
      __builtin_amdgcn_s_setprio(0);
      // The first operands of the sums, past the exponentials.
#pragma unroll
      for (int n = 0; n < kAhead && n < 2 * DT; ++n) op[n] = sums(n, 0);
      const bool edge = p.causal && i0 + ahead < wkey + 31;
      if (edge || i0 + 32 > qs.len) {
        // Query 8 (i / 4) + i % 4 sees the lane's key iff >= rel, and is there iff < end.
        const int rel = edge ? key - ahead - i0 - 4 * half : 0, end = qs.len - i0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int c = 8 * (i / 4) + i % 4;
          if (c < rel || c >= end) s[i] = -INFINITY;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const f32x4_t lse = *reinterpret_cast<const f32x4_t*>(st + 8 * j);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          s[4 * j + i] = fast_exp2(fmaf(s[4 * j + i], p.scale_log2, -lse[i]));
          dp[4 * j + i] *= kBF16 ? s[4 * j + i] : s[4 * j + i] * lift;
        }
      }
#pragma unroll
      for (int hf = 0; hf < 2; ++hf) {
        const uint4 pb = pack_b<kBF16>(s, hf), db = pack_b<kBF16>(dp, hf);
        uint4* const over = reinterpret_cast<uint4*>(s_ex + wave * 2048 + hf * 1024 + lane * 16);
        if (role == 0) {
          own[hf] = pb;
          *over = db;
        } else {
          own[hf] = db;
          *over = pb;
        }
      }
    } else if (more) {
#pragma unroll
      for (int n = 0; n < kCopies; ++n) issue(kStage ^ 1, n);
    }
    __syncthreads();
    // The wave's own 32 queries, then its neighbour's.
    if (mine) {
#pragma unroll
      for (int n = 0; n < 2 * DT; ++n) {
        acc[n % DT] = mfma32<kBF16>(op[n % kAhead], own[n / DT], acc[n % DT]);
        if (n + kAhead < 2 * DT) op[n % kAhead] = sums(n + kAhead, 0);
      }
    }
    if (seen(role ^ 1)) {
      uint4 b[2];
#pragma unroll
      for (int hf = 0; hf < 2; ++hf)
        b[hf] = lds_read16(s_ex, (wave ^ 1) * 2048 + hf * 1024 + lane * 16);
#pragma unroll
      for (int n = 0; n < kAhead && n < 2 * DT; ++n) op[n] = sums(n, 1);
#pragma unroll
      for (int n = 0; n < 2 * DT; ++n) {
        acc[n % DT] = mfma32<kBF16>(op[n % kAhead], b[n / DT], acc[n % DT]);
        if (n + kAhead < 2 * DT) op[n % kAhead] = sums(n + kAhead, 1);
      }
    }
  };
  loads_done();
  for (int it = 0; it < steps; it += 2) {
    step(std::integral_constant<int, 0>{}, it);
    if (it + 1 < steps) step(std::integral_constant<int, 1>{}, it + 1);
  }
  const float mul = role == 1 ? p.scale * lower : kBF16 ? 1.f : pow2(-kF16Lift);
  if constexpr (kParts) {
    float* const to =
        p.part + ((((int64_t)blk.place * parts + part) * p.num_kv_heads + kv) * kWaves + wave) * (32 * D);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int j = 0; j < 4; ++j)
        *reinterpret_cast<f32x4_t*>(to + ((dt * 4 + j) * 64 + lane) * 4) =
            f32x4_t{acc[dt][4 * j] * mul, acc[dt][4 * j + 1] * mul, acc[dt][4 * j + 2] * mul,
                    acc[dt][4 * j + 3] * mul};
    return;
  }
  __syncthreads();  // every wave is done with the tiles
  write_dkv<kBF16, D>(p, acc, mul, s_qd + wave * 32 * ROWB, role, ks, kv, wkey, lane);
}

// Adds up the parts of a block's gradients, in their order: a thread 4 elements of
// one key's dk or dv (256 of a wave's a workgroup; blockIdx.y counts them).
template <bool kBF16, int D>
__global__ __launch_bounds__(256) void varlen_dkv_sum_kernel(VarlenBwdParams p) {
  const int kv = (int)(blockIdx.x % (unsigned)p.num_kv_heads);
  const int tile = (int)(blockIdx.x / (unsigned)p.num_kv_heads);
  const DkvBlock blk = dkv_block<kInTurn>(p, tile);
  if (!blk.found) {
    if (blockIdx.y == 0) zero_rest_kv<D>(p, kv, tile - blk.empty, p.k_tiles - blk.empty);
    return;
  }
  const int at = blockIdx.y * 256 + threadIdx.x;  // of the block's 4 waves x D / 8 x 64
  const int wave = at / (D * 8), dt = at / 256 % (D / 32), j = at / 64 % 4, lane = at % 64;
  const int key = blk.j0 + 32 * (wave >> 1) + lane % 32;
  if (key >= blk.ks.len) return;
  const int64_t unit = (int64_t)p.num_kv_heads * 4 * 32 * D;  // floats from part to part
  const float* const from = p.part + (int64_t)tile * p.parts * unit + (int64_t)kv * 4 * 32 * D + at * 4;
  f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
  for (int n0 = 0; n0 < p.parts; n0 += 4) {
    f32x4_t x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      // (A part without steps wrote nothing.)
      const int n = n0 + i;
      const bool any = n < p.parts && part_begin(blk.steps, n, p.parts) < part_begin(blk.steps, n + 1, p.parts);
      x[i] = any ? *reinterpret_cast<const f32x4_t*>(from + n * unit) : f32x4_t{0.f, 0.f, 0.f, 0.f};
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) acc += x[i];
  }
  const bool is_k = wave & 1;
  char* const to = is_k ? p.dk + (int64_t)(blk.ks.row + key) * p.dk_st + kv * p.dk_sh
                        : p.dv + (int64_t)(blk.ks.row + key) * p.dv_st + kv * p.dv_sh;
  *reinterpret_cast<uint2*>(to + (32 * dt + 8 * j + 4 * (lane / 32)) * 2) =
      make_uint2(pack_pair<kBF16>(acc[0], acc[1]), pack_pair<kBF16>(acc[2], acc[3]));
}

// ------------------------------------------------------- short sequences, at once
// Sequences of at most kWindowMost rows (an encoder's windows) at head_dim 64, a kv
// head to each query head: one workgroup takes a sequence's head whole.  q, dout, k
// and v come to LDS once, in as many rows as the longest sequence has (104 rows let
// three workgroups share a CU); every wave forms dq of 32 queries, leaves lse and
// -delta in LDS, and then dk and dv of 32 keys.  The launches above read the four
// twice, and a launch waits for the other: 160 windows of 13 to 104 rows and 14 heads
// take 36 us at once (134 MB, 3.7 TB/s) and 54 in two launches, 4 windows 10.9 and
// 13.1.  What bounds many windows is HBM and each workgroup's own length, some 10 us
// with three to a CU; few windows, that length alone.  Rows past the sequence's last
// are never in LDS: what stands for them is the last row, and is masked.
constexpr int kWindowMost = 128;
constexpr int kWindowStats = 2 * kWindowMost * 4 + 4 * 4;  // bytes: lse, -delta, f16: largest |dout|s
inline size_t window_lds(int rows) {
  const size_t tile = (size_t)((rows + 7) / 8 * 8) * 128;
  return std::max(4 * tile, 2 * tile + kWindowStats + 4 * 32 * 128);
}
constexpr int kWindowExtra = 2048;  // rows outside the sequences to a workgroup and head

// LDS offsets in a tile of 64-element rows: of row r's chunk for the lane's half (8
// elements from 16 step + 8 half: ^ step << 5), and of the transposed read of row r
// (32 elements from 32 dt: ^ dt << 6).
__device__ inline int window_row(int r, int half) { return r * 128 + ((half ^ bwd_swz<64>(r)) << 4); }
__device__ inline int window_tr(int r, int lane) {
  const int c = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  return r * 128 + ((lane & 1) << 3) + ((c ^ bwd_swz<64>(r)) << 4);
}

// Adds to acc the products of a tile's rows r0 ... r0 + 31 (transposed) and x.
template <bool kBF16>
__device__ inline void window_sum(f32x16_t (&acc)[2], const f32x16_t& x, const char* tile, int r0,
                                  int last, int lane) {
#pragma unroll
  for (int hf = 0; hf < 2; ++hf) {
    const int r = r0 + 16 * hf + 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int lo = window_tr(min(r, last), lane), hi = window_tr(min(r + 8, last), lane);
    const uint4 b = pack_b<kBF16>(x, hf);
#pragma unroll
    for (int dt = 0; dt < 2; ++dt) {
      const uint2 a = __builtin_bit_cast(uint2, lds_read_tr(tile, lo ^ (dt << 6)));
      const uint2 c = __builtin_bit_cast(uint2, lds_read_tr(tile, hi ^ (dt << 6)));
      acc[dt] = mfma32<kBF16>(make_uint4(a.x, a.y, c.x, c.y), b, acc[dt]);
    }
  }
}

template <bool kBF16>
__global__ __launch_bounds__(kBwdThreads, 3) void varlen_window_kernel(VarlenBwdParams p) {
  constexpr int D = 64, ROWB = D * 2, DS = D / 16, DT = D / 32, kAhead = 4;
  extern __shared__ __align__(16) char s_all[];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  const int seq = (int)(blockIdx.x / (unsigned)p.num_heads);
  const int head = (int)(blockIdx.x % (unsigned)p.num_heads);
  if (seq >= p.num_seqs) {
    const int nth = seq - p.num_seqs, of = (int)(gridDim.x / (unsigned)p.num_heads) - p.num_seqs;
    zero_rest<D, kBwdThreads>(p.cu_q, p.num_seqs, p.total_q, p.dq, p.dq_st, head * p.dq_sh, nth, of);
    zero_rest_kv<D>(p, head, nth, of);
    return;
  }
  const SeqRows qs = seq_rows(p.cu_q[seq], p.cu_q[seq + 1], p.total_q);
  const SeqRows ks = seq_rows(p.cu_k[seq], p.cu_k[seq + 1], p.total_k);
  char* const dq = p.dq + (int64_t)qs.row * p.dq_st + head * p.dq_sh;
  char* const dk = p.dk + (int64_t)ks.row * p.dk_st + head * p.dk_sh;
  char* const dv = p.dv + (int64_t)ks.row * p.dv_st + head * p.dv_sh;
  if (max(qs.len, ks.len) > p.window) {  // longer than the caller said: NaN, not some of it
    const uint4 nan = make_uint4(0x7fff7fff, 0x7fff7fff, 0x7fff7fff, 0x7fff7fff);
    for (int i = threadIdx.x / 8; i < max(qs.len, ks.len); i += kBwdThreads / 8) {
      const int at = threadIdx.x % 8 * 16;
      if (i < qs.len) st16(dq + i * p.dq_st + at, nan);
      if (i < ks.len) st16(dk + i * p.dk_st + at, nan);
      if (i < ks.len) st16(dv + i * p.dv_st + at, nan);
    }
    return;
  }
  const int ahead = ks.len - qs.len;
  const int tile_b = (p.window + 7) / 8 * 8 * ROWB;
  char* const sq = s_all;
  char* const sd = sq + tile_b;
  char* const sk = sd + tile_b;
  char* const sv = sk + tile_b;
  // In K's and V's place, once every wave has its keys in registers.
  float* const s_lse = reinterpret_cast<float*>(sk);
  float* const s_delta = s_lse + kWindowMost;
  float* const s_top = s_delta + kWindowMost;
  char* const s_out = sk + kWindowStats + wave * 32 * ROWB;  // the wave's rows on their way out
  const uint32_t lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_all);
  // 8 rows a copy, the waves in turn.
  auto fetch = [&](const char* src, int64_t st, int len, int n) {
    const int in8 = lane / 8;
    for (int r0 = wave * 8; r0 < len; r0 += 32) {
      const int r = r0 + in8;
      const uint32_t chunk = (uint32_t)(((lane % 8) ^ bwd_swz<D>(r)) << 4);
      dma16((uint32_t)min(in8, len - 1 - r0) * (uint32_t)st + chunk, src + r0 * st,
            lds + (uint32_t)(n * tile_b + r0 * ROWB));
    }
  };
  fetch(p.q + (int64_t)qs.row * p.q_st + head * p.q_sh, p.q_st, qs.len, 0);
  fetch(p.dout + (int64_t)qs.row * p.do_st + head * p.do_sh, p.do_st, qs.len, 1);
  fetch(p.k + (int64_t)ks.row * p.k_st + head * p.k_sh, p.k_st, ks.len, 2);
  fetch(p.v + (int64_t)ks.row * p.v_st + head * p.v_sh, p.v_st, ks.len, 3);
  const int first = 32 * wave, row = first + l32;  // the wave's queries, then its keys
  uint4 oreg[DS] = {};
  if (first < qs.len) {
    const char* const op =
        p.out + (int64_t)(qs.row + min(row, qs.len - 1)) * p.o_st + head * p.o_sh + half * 16;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) oreg[ds] = ld16(op + ds * 32);
  }
  wait_vmcnt<0>();
  __syncthreads();

  float top = 0.f, lse = 0.f, delta = 0.f, mul = 0.f;
  f32x16_t acc[DT];  // dq
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16_t{};
  if (first < qs.len) {
    uint4 qreg[DS], doreg[DS];
    const int own = window_row(min(row, qs.len - 1), half);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      qreg[ds] = lds_read16(sq, own ^ (ds << 5));
      doreg[ds] = lds_read16(sd, own ^ (ds << 5));
    }
    using ET = std::conditional_t<kBF16, BF16, F16>;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      float a[8], b[8];
      ET::unpack(doreg[ds], a);
      ET::unpack(oreg[ds], b);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        delta = fmaf(a[i], b[i], delta);
        if constexpr (!kBF16) top = fmaxf(top, fabsf(a[i]));
      }
    }
    delta = sum_xor32(delta);
    int e = 0;
    if constexpr (!kBF16) {
      top = max_xor32(top);
      e = top_exponent(top);
    }
    const int lim = p.causal ? min(ks.len, ahead + row + 1) : ks.len;
    const int lim_lo = p.causal ? min(ks.len, ahead + first + 1) : ks.len;
    const int lim_hi = p.causal ? min(ks.len, ahead + min(first + 32, qs.len)) : ks.len;
    constexpr float kSlack = kBF16 ? kLazy : 0.f;
    float m = -1.0e30f, l = 0.f;
    for (int j0 = 0; j0 < lim_hi; j0 += 32) {
      const int ra = window_row(min(j0 + l32, ks.len - 1), half);
      uint4 op[kAhead];
      auto request = [&](int n) {
        if (n < 2 * DS) op[n % kAhead] = lds_read16(n & 1 ? sv : sk, ra ^ (n / 2 << 5));
      };
#pragma unroll
      for (int n = 0; n < kAhead; ++n) request(n);
      f32x16_t s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = -delta;
#pragma unroll
      for (int n = 0; n < 2 * DS; ++n) {
        if (n & 1)
          dp = mfma32<kBF16>(op[n % kAhead], doreg[n / 2], dp);
        else
          s = mfma32<kBF16>(op[n % kAhead], qreg[n / 2], s);
        request(n + kAhead);
      }
      if (j0 + 32 > lim_lo) {
        const int rel = lim - j0 - 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 >= rel) {
            s[i] = -INFINITY;
            if constexpr (!kBF16) dp[i] = 0.f;
          }
      }
      float mx = s[0], big = 0.f;
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      mx = max_xor32(mx) * p.scale_log2;
      bool up = mx > m + kSlack;
      if constexpr (!kBF16) {
#pragma unroll
        for (int i = 0; i < 16; ++i) big = fmaxf(big, fabsf(dp[i]));
        up = up || out_of_range(big, e);
      }
      if (__builtin_amdgcn_ballot_w64(up) != 0) {
        const float mn = fmaxf(m, mx);
        float alpha = m - mn;
        m = mn;
        if constexpr (!kBF16) {
          const int en = raised(big, e);
          alpha += (float)(e - en);
          e = en;
        }
        alpha = fast_exp2(alpha);
        l *= alpha;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[dt] *= alpha;
      }
      const float base = kBF16 ? m : m + (float)e;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[i] = fast_exp2(fmaf(s[i], p.scale_log2, -base));
        l += s[i];
        dp[i] *= s[i];
      }
      window_sum<kBF16>(acc, dp, sk, j0, ks.len - 1, lane);
    }
    l = sum_xor32(l);
    lse = l > 0.f ? (kBF16 ? m : m + (float)e) + __builtin_amdgcn_logf(l) -
                        (kBF16 ? 0.f : (float)kF16Lift)
                  : INFINITY;
    mul = l > 0.f ? p.scale / l : 0.f;
    if constexpr (!kBF16) top = held_top(top, e);
  }
  __syncthreads();  // every wave has been through K and V
  uint4 kreg[DS] = {}, vreg[DS] = {};
  if (first < ks.len) {
    const int own = window_row(min(row, ks.len - 1), half);
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      kreg[ds] = lds_read16(sk, own ^ (ds << 5));
      vreg[ds] = lds_read16(sv, own ^ (ds << 5));
    }
  }
  __syncthreads();
  if constexpr (!kBF16) {
    top = group_max<64>(top);
    if (lane == 0) s_top[wave] = top;
  }
  if (first < qs.len) {
    // Rows past the sequence's last, too: the queries' blocks below read them.
    if (half == 0) {
      s_lse[row] = lse;
      s_delta[row] = -delta;
    }
    write_rows<kBF16, D>(acc, mul, s_out, dq, p.dq_st, first, qs.len, lane);
  }
  __syncthreads();
  if (first >= ks.len) return;
  float lift = 1.f, lower = 1.f;
  if constexpr (!kBF16) {
    const int e = top_exponent(fmaxf(fmaxf(s_top[0], s_top[1]), fmaxf(s_top[2], s_top[3])));
    lift = pow2(-e - kF16Lift);
    lower = pow2(e);
  }

  f32x16_t acc_k[DT], acc_v[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc_k[dt] = acc_v[dt] = f32x16_t{};
  // The first 32 queries of which one sees a key of the wave.
  for (int i0 = p.causal ? max(first - ahead, 0) / 32 * 32 : 0; i0 < qs.len; i0 += 32) {
    const int ra = window_row(min(i0 + l32, qs.len - 1), half);
    uint4 op[kAhead];
    auto request = [&](int n) {
      if (n < 2 * DS) op[n % kAhead] = lds_read16(n & 1 ? sd : sq, ra ^ (n / 2 << 5));
    };
#pragma unroll
    for (int n = 0; n < kAhead; ++n) request(n);
    f32x16_t s = {}, dp;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t d = *reinterpret_cast<const f32x4_t*>(s_delta + i0 + 4 * half + 8 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) dp[4 * j + i] = d[i];
    }
#pragma unroll
    for (int n = 0; n < 2 * DS; ++n) {
      if (n & 1)
        dp = mfma32<kBF16>(op[n % kAhead], vreg[n / 2], dp);
      else
        s = mfma32<kBF16>(op[n % kAhead], kreg[n / 2], s);
      request(n + kAhead);
    }
    const bool edge = p.causal && i0 + ahead < first + 31;
    if (edge || i0 + 32 > qs.len) {
      // Query 8 (i / 4) + i % 4 sees the lane's key iff >= rel, and is there iff < end.
      const int rel = edge ? row - ahead - i0 - 4 * half : 0, end = qs.len - i0 - 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int c = 8 * (i / 4) + i % 4;
        if (c < rel || c >= end) s[i] = -INFINITY;
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t at = *reinterpret_cast<const f32x4_t*>(s_lse + i0 + 4 * half + 8 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        s[4 * j + i] = fast_exp2(fmaf(s[4 * j + i], p.scale_log2, -at[i]));
        dp[4 * j + i] *= kBF16 ? s[4 * j + i] : s[4 * j + i] * lift;
      }
    }
    window_sum<kBF16>(acc_v, s, sd, i0, qs.len - 1, lane);
    window_sum<kBF16>(acc_k, dp, sq, i0, qs.len - 1, lane);
  }
  write_rows<kBF16, D>(acc_v, kBF16 ? 1.f : pow2(-kF16Lift), s_out, dv, p.dv_st, first, ks.len, lane);
  write_rows<kBF16, D>(acc_k, p.scale * lower, s_out, dk, p.dk_st, first, ks.len, lane);
}

// The launches for one 16-bit type and head_dim, instantiated in
// varlen_backward_<type>.hip.
template <bool kBF16, int D>
void launch_varlen_backward(const VarlenBwdParams& p, hipStream_t st);

template <bool kBF16, int D>
static void launch_varlen_backward_d(const VarlenBwdParams& p, hipStream_t st) {
  if constexpr (D == 64) {
    if (p.window > 0) {
      const unsigned items = (unsigned)p.num_seqs + 1 + std::max(p.total_q, p.total_k) / kWindowExtra;
      hipLaunchKernelGGL((varlen_window_kernel<kBF16>), dim3(items * p.num_heads),
                         dim3(kBwdThreads), window_lds(p.window), st, p);
      return;
    }
  }
  const dim3 q_grid((unsigned)p.q_tiles * p.num_heads);
  if (p.q_rows == 64)
    hipLaunchKernelGGL((varlen_dq_kernel<kBF16, D, true>), q_grid, dim3(kBwdThreads), 0, st, p);
  else
    hipLaunchKernelGGL((varlen_dq_kernel<kBF16, D, false>), q_grid, dim3(kBwdThreads), 0, st, p);
  const dim3 grid((unsigned)p.k_tiles * p.parts * p.num_kv_heads);
  if (p.parts == 1) {
    hipLaunchKernelGGL((varlen_dkv_kernel<kBF16, D, false>), grid, dim3(256), 0, st, p);
    return;
  }
  hipLaunchKernelGGL((varlen_dkv_kernel<kBF16, D, true>), grid, dim3(256), 0, st, p);
  hipLaunchKernelGGL((varlen_dkv_sum_kernel<kBF16, D>),
                     dim3((unsigned)p.k_tiles * p.num_kv_heads, D / 8), dim3(256), 0, st, p);
}

template <>
void launch_varlen_backward<true, 64>(const VarlenBwdParams&, hipStream_t);
template <>
void launch_varlen_backward<true, 128>(const VarlenBwdParams&, hipStream_t);
template <>
void launch_varlen_backward<false, 64>(const VarlenBwdParams&, hipStream_t);
template <>
void launch_varlen_backward<false, 128>(const VarlenBwdParams&, hipStream_t);

}  // namespace va
