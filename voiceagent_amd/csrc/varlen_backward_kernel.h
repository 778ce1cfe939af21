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
// Two launches, neither with atomics, so that every call repeats bit for bit:
//   1. varlen_dq_kernel: a workgroup per 128 queries of one head, one pass over
//      their keys.  delta is known from out, so dq needs no softmax statistics
//      beforehand: with a running maximum m, dq gathers 2^(s c - m) (dP - delta) k
//      and is divided by the sum at the end, rescaled where m rises.  It leaves
//      lse_i = log2 sum_j 2^(c log2 e s_ij) and delta_i for the second launch.
//   2. varlen_dkv_kernel: a workgroup per 128 keys of one kv head, over the
//      queries that see them in every head of the group.
// Each wave holds 32 queries (keys): their rows are B operands in registers
// for the whole loop, their gradients accumulators.  The other side streams
// through LDS in 64-row tiles, two stages filled by DMA, swizzled as in the
// forward kernel.  S^T and dP^T (or S and dP) come from 32x32x16 MFMAs with the
// tile's rows as A operands; their accumulators, rounded to 16 bits, are in
// place the B operands of the gradients' products, whose A operands are the
// same tile rows transposed by ds_read_b64_tr_b16.
#pragma once

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
  int32_t q_tiles, k_tiles;  // workgroups per head of the two launches
  float* lse;                // [num_heads][total_q]
  float* delta;              // [num_heads][total_q]
  float* top;                // f16: [num_heads][total_q], largest |dout| of the row
};

constexpr int kBwdThreads = 256;
constexpr int kBwdRows = 128;  // queries (keys) of a workgroup, 32 a wave
constexpr int kBwdTile = 64;   // rows of the other side staged at a time

template <bool kBF16>
__device__ inline f32x16_t mfma32(uint4 a, uint4 b, f32x16_t c) {
  if constexpr (kBF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                   __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                                  __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// The lse of a staged row that is not there: its P is 2^-inf = 0.
__device__ const float kInfRow = INFINITY;

// One 4-byte global -> LDS copy per lane (lane l's word lands at lds + 4 l);
// wait states as in dma16.
__device__ inline void dma4(const void* src, uint32_t lds) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %0, off" ::"v"(src), "{m0}"(lds) : "memory");
}

// Sequence s's rows [row, row + len) of `total` packed rows: what cu says, held
// to rows that there are.
struct SeqRows {
  int row, len;
};
__device__ inline SeqRows seq_rows(const int32_t* cu, int s, int total) {
  const int a = min(max(cu[s], 0), total);
  return {a, min(max(cu[s + 1], a), total) - a};
}

// The `tile`-th block of kBwdRows rows, counting every sequence's blocks in
// turn.  found: there is one; otherwise first is the number of blocks there are.
struct BwdBlock {
  bool found;
  int seq, first;  // first: tile number of the sequence's first block
};
__device__ inline BwdBlock find_block(const int32_t* cu, int num_seqs, int total, int tile) {
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int s0 = 0; s0 < num_seqs; s0 += 64) {
    int nb = 0;
    if (s0 + lane < num_seqs) nb = (seq_rows(cu, s0 + lane, total).len + kBwdRows - 1) / kBwdRows;
    const int upto = wave_scan(nb);
    const uint64_t past = __builtin_amdgcn_ballot_w64(before + upto > tile);
    if (past != 0) {
      const int at = __builtin_ctzll(past);
      return {true, s0 + at,
              before + __builtin_amdgcn_readlane(upto, at) - __builtin_amdgcn_readlane(nb, at)};
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return {false, 0, before};
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

// Copies 64 rows of one tensor into an LDS tile, wave w's share of kWaves: row r
// of the tile is row base + r of the sequence, zeros past `len`.
template <int D, int kWaves>
__device__ inline void stage_rows(const char* src, int64_t st, int base, int len, uint32_t lds,
                                  int wave, int lane) {
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPI = 64 / CPR;
  constexpr int NI = kBwdTile * ROWB / 1024 / kWaves;
  static_assert(NI >= 1, "a wave copies at least 1 KiB");
#pragma unroll
  for (int i = 0; i < NI; ++i) {
    const int r = (wave * NI + i) * RPI + lane / CPR;
    const int chunk = (lane % CPR) ^ swz<D>(r);
    const char* const at = src + (int64_t)(base + r) * st + chunk * 16;
    dma16(base + r < len ? at : reinterpret_cast<const char*>(&kZeroRow),
          lds + (uint32_t)((wave * NI + i) * 1024));
  }
}

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
    row0 = (h ^ swz<D>(r)) << 4;
    const int t = 4 * h + (r16 >> 2);
    tr = t * ROWB + ((r16 & 1) << 3);
    tr0 = ((2 * (g & 1) + ((r16 >> 1) & 1)) ^ swz<D>(t)) << 4;
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
        __builtin_bit_cast(uint2, lds_read_tr(tile, off + 8 * D * 2 + (tr0 ^ 16 ^ (dt << 6))));
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
};

// Eight accumulator values of one lane (rows 16 half + {0-3, 8-11} + 4 (l / 32))
// as a B operand.
template <bool kBF16>
__device__ inline uint4 pack_b(const f32x16_t& x, int half) {
  using M = Mma<kBF16>;
  return make_uint4(M::pack2(x[8 * half], x[8 * half + 1]), M::pack2(x[8 * half + 2], x[8 * half + 3]),
                    M::pack2(x[8 * half + 4], x[8 * half + 5]), M::pack2(x[8 * half + 6], x[8 * half + 7]));
}

// Writes a wave's gradient, accumulators [D][32 rows] times `mul`, as rows of
// 16 bits: through the wave's own 32 rows of LDS, so that each store
// instruction writes whole rows.
template <bool kBF16, int D>
__device__ inline void write_rows(const f32x16_t (&acc)[D / 32], float mul, char* s, char* dst,
                                  int64_t st, int row0, int rows, int lane) {
  using M = Mma<kBF16>;
  constexpr int ROWB = D * 2, CPR = ROWB / 16, RPS = 64 / CPR;
  const int r = lane & 31, h = lane >> 5;
#pragma unroll
  for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint2 w = make_uint2(M::pack2(acc[dt][4 * j] * mul, acc[dt][4 * j + 1] * mul),
                                 M::pack2(acc[dt][4 * j + 2] * mul, acc[dt][4 * j + 3] * mul));
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

// ---------------------------------------------------------------------- dq
// f16 (as for dk): dS is rounded to 16 bits, and a gradient of 1e-4 spread over
// a thousand keys would fall among f16's subnormals.  So P is scaled by 2^-e, e
// the exponent of the row's largest |dout|, through the exponential's argument,
// and the maximum is followed without slack, which keeps dS near v's size.
template <bool kBF16, int D>
__global__ __launch_bounds__(kBwdThreads, 2) void varlen_dq_kernel(VarlenBwdParams p) {
  constexpr int ROWB = D * 2, TILE_B = kBwdTile * ROWB, DS = D / 16, DT = D / 32;
  __shared__ __align__(1024) char s_kv[2 * 2 * TILE_B];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  // Tiles run from the last to the first: under a causal mask a sequence's
  // later blocks have more keys.  Consecutive workgroups, which run on
  // different XCDs, take different kv heads.
  const int tile = p.q_tiles - 1 - (int)(blockIdx.x / (unsigned)p.num_heads);
  const int pick = (int)(blockIdx.x % (unsigned)p.num_heads);
  const int group = p.num_heads / p.num_kv_heads;
  const int kv = pick % p.num_kv_heads, head = kv * group + pick / p.num_kv_heads;
  const BwdBlock blk = find_block(p.cu_q, p.num_seqs, p.total_q, tile);
  if (!blk.found) {
    zero_rest<D, kBwdThreads>(p.cu_q, p.num_seqs, p.total_q, p.dq, p.dq_st, head * p.dq_sh, tile - blk.first,
                 p.q_tiles - blk.first);
    return;
  }
  const SeqRows qs = seq_rows(p.cu_q, blk.seq, p.total_q);
  const SeqRows ks = seq_rows(p.cu_k, blk.seq, p.total_k);
  const int i0 = (tile - blk.first) * kBwdRows;  // the block's first query
  const int ahead = ks.len - qs.len;             // causal: query i sees keys j <= i + ahead
  const int kend =
      p.causal ? min(max(ahead + min(i0 + kBwdRows, qs.len), 0), ks.len) : ks.len;
  const int tiles = (kend + kBwdTile - 1) / kBwdTile;
  const char* const kp = p.k + (int64_t)ks.row * p.k_st + kv * p.k_sh;
  const char* const vp = p.v + (int64_t)ks.row * p.v_st + kv * p.v_sh;
  const uint32_t lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_kv);
  auto issue = [&](int t) {
    const uint32_t to = lds + (uint32_t)((t & 1) * 2 * TILE_B);
    stage_rows<D, 4>(kp, p.k_st, t * kBwdTile, ks.len, to, wave, lane);
    stage_rows<D, 4>(vp, p.v_st, t * kBwdTile, ks.len, to + TILE_B, wave, lane);
  };
  if (tiles > 0) issue(0);

  // The wave's 32 queries (rows past the sequence repeat its last).
  const int wrow = i0 + 32 * wave;
  const int row = wrow + l32, at = qs.row + min(row, qs.len - 1);
  uint4 qreg[DS], doreg[DS];
  float delta = 0.f;
  int e = 0;
  {
    const char* const qp = p.q + at * p.q_st + head * p.q_sh + half * 16;
    const char* const dp = p.dout + at * p.do_st + head * p.do_sh + half * 16;
    const char* const op = p.out + at * p.o_st + head * p.o_sh + half * 16;
    uint4 oreg[DS];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) {
      qreg[ds] = ld16(qp + ds * 32);
      doreg[ds] = ld16(dp + ds * 32);
      oreg[ds] = ld16(op + ds * 32);
    }
    using ET = std::conditional_t<kBF16, BF16, F16>;
    float top = 0.f;
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
      if (half == 0 && row < qs.len) p.top[(int64_t)head * p.total_q + at] = top;
    }
  }

  const TileAt<D> ta(lane);
  const int lim = p.causal ? min(ks.len, ahead + row + 1) : ks.len;  // keys the lane's query sees
  const int lim_lo = p.causal ? min(ks.len, ahead + wrow + 1) : ks.len;
  const int lim_hi = p.causal ? min(ks.len, ahead + wrow + 32) : ks.len;
  constexpr float kSlack = kBF16 ? kLazy : 0.f;
  float m = -1.0e30f, l = 0.f;
  f32x16_t acc[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x16_t{};

  for (int t = 0; t < tiles; ++t) {
    wait_vmcnt<0>();
    __syncthreads();
    if (t + 1 < tiles) issue(t + 1);
    const char* const sk = s_kv + (t & 1) * 2 * TILE_B;
    const char* const sv = sk + TILE_B;
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      const int j0 = t * kBwdTile + 32 * sub;
      if (j0 >= lim_hi) break;  // no query of the wave sees these
      f32x16_t s = {}, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) dp[i] = -delta;
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) s = mfma32<kBF16>(ta.a(sk, sub, ds), qreg[ds], s);
#pragma unroll
      for (int ds = 0; ds < DS; ++ds) dp = mfma32<kBF16>(ta.a(sv, sub, ds), doreg[ds], dp);
      if (j0 + 32 > lim_lo) {
        const int rel = lim - j0 - 4 * half;  // key 8 (i / 4) + i % 4 of the lane is seen iff < rel
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (8 * (i / 4) + i % 4 >= rel) s[i] = -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int i = 1; i < 16; ++i) mx = fmaxf(mx, s[i]);
      mx = max_xor32(mx) * p.scale_log2;
      if (__builtin_amdgcn_ballot_w64(mx > m + kSlack) != 0) {
        const float mn = fmaxf(m, mx);
        const float alpha = fast_exp2(m - mn);
        m = mn;
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
  const float base = kBF16 ? m : m + (float)e;
  if (half == 0 && row < qs.len) {
    const int64_t w = (int64_t)head * p.total_q + at;
    p.lse[w] = l > 0.f ? base + __builtin_amdgcn_logf(l) : INFINITY;
    p.delta[w] = delta;
  }
  __syncthreads();  // every wave is done with the tiles
  write_rows<kBF16, D>(acc, l > 0.f ? p.scale / l : 0.f, s_kv + wave * 32 * ROWB,
                       p.dq + (int64_t)qs.row * p.dq_st + head * p.dq_sh, p.dq_st, wrow, qs.len,
                       lane);
}

// ------------------------------------------------------------------- dk, dv
// Eight waves: four groups of 32 keys, twice, for the two halves of a tile's 64
// queries; the halves' sums meet in LDS at the end.  (With four waves that take
// both halves in turn the two waves of a SIMD belong to two workgroups, of which
// a causal launch leaves the one with more queries alone for most of the time.)
constexpr int kDkvThreads = 512;

// A wave's accumulators to LDS, 16 bytes a lane at a time, and added from there.
template <int DT>
__device__ inline void put_acc(const f32x16_t (&acc)[DT], char* s, int lane) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      *reinterpret_cast<f32x4_t*>(s + ((dt * 4 + j) * 64 + lane) * 16) =
          f32x4_t{acc[dt][4 * j], acc[dt][4 * j + 1], acc[dt][4 * j + 2], acc[dt][4 * j + 3]};
}
template <int DT>
__device__ inline void add_acc(f32x16_t (&acc)[DT], const char* s, int lane) {
#pragma unroll
  for (int dt = 0; dt < DT; ++dt)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t x = *reinterpret_cast<const f32x4_t*>(s + ((dt * 4 + j) * 64 + lane) * 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[dt][4 * j + i] += x[i];
    }
}

template <bool kBF16, int D>
__global__ __launch_bounds__(kDkvThreads, 2) void varlen_dkv_kernel(VarlenBwdParams p) {
  constexpr int ROWB = D * 2, TILE_B = kBwdTile * ROWB, DS = D / 16, DT = D / 32;
  __shared__ __align__(1024) char s_qd[2 * 2 * TILE_B];
  __shared__ __align__(16) float s_st[2 * 2 * kBwdTile];  // a stage's lse, delta
  __shared__ float s_top[8];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sub = wave >> 2;  // the wave's half of a tile's queries
  const int lane = threadIdx.x & 63, l32 = lane & 31, half = lane >> 5;
  // (Under a causal mask a sequence's earlier blocks are seen by more queries.)
  const int tile = (int)(blockIdx.x / (unsigned)p.num_kv_heads);
  const int kv = (int)(blockIdx.x % (unsigned)p.num_kv_heads);
  const int group = p.num_heads / p.num_kv_heads;
  const BwdBlock blk = find_block(p.cu_k, p.num_seqs, p.total_k, tile);
  if (!blk.found) {
    zero_rest<D, kDkvThreads>(p.cu_k, p.num_seqs, p.total_k, p.dk, p.dk_st, kv * p.dk_sh,
                              tile - blk.first, p.k_tiles - blk.first);
    zero_rest<D, kDkvThreads>(p.cu_k, p.num_seqs, p.total_k, p.dv, p.dv_st, kv * p.dv_sh,
                              tile - blk.first, p.k_tiles - blk.first);
    return;
  }
  const SeqRows qs = seq_rows(p.cu_q, blk.seq, p.total_q);
  const SeqRows ks = seq_rows(p.cu_k, blk.seq, p.total_k);
  const int j0 = (tile - blk.first) * kBwdRows;  // the block's first key
  const int ahead = ks.len - qs.len;
  const int t0 = p.causal ? max(j0 - ahead, 0) / kBwdTile : 0;  // the first tile of queries that see it
  const int nt = max((qs.len + kBwdTile - 1) / kBwdTile - t0, 0);
  const int steps = nt * group;

  const uint32_t lds = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_qd);
  const uint32_t lds_st = __builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)s_st);
  // The tile requested next: head of the group, tile of its queries.
  int gi = 0, ti = 0;
  auto issue = [&](int stage) {
    int at_lane = lane;  // (what follows from the lane is formed anew each step)
    asm volatile("" : "+v"(at_lane));
    const int head = kv * group + gi, base = (t0 + ti) * kBwdTile;
    const uint32_t to = lds + (uint32_t)(stage * 2 * TILE_B);
    stage_rows<D, 8>(p.q + (int64_t)qs.row * p.q_st + head * p.q_sh, p.q_st, base, qs.len, to, wave,
                     at_lane);
    stage_rows<D, 8>(p.dout + (int64_t)qs.row * p.do_st + head * p.do_sh, p.do_st, base, qs.len,
                     to + TILE_B, wave, at_lane);
    if (wave < 2) {
      const int64_t w = (int64_t)head * p.total_q + qs.row + base + at_lane;
      const float* const at = (wave == 0 ? p.lse : p.delta) + w;
      const float* const none = wave == 0 ? &kInfRow : reinterpret_cast<const float*>(&kZeroRow);
      dma4(base + at_lane < qs.len ? at : none,
           lds_st + (uint32_t)((stage * 2 + wave) * kBwdTile * 4));
    }
    if (++ti == nt) {
      ti = 0;
      ++gi;
    }
  };
  if (steps > 0) issue(0);

  const int wkey = j0 + 32 * (wave & 3), key = wkey + l32;
  const int at = ks.row + min(key, ks.len - 1);
  uint4 kreg[DS], vreg[DS];
#pragma unroll
  for (int ds = 0; ds < DS; ++ds) {
    kreg[ds] = ld16(p.k + at * p.k_st + kv * p.k_sh + half * 16 + ds * 32);
    vreg[ds] = ld16(p.v + at * p.v_st + kv * p.v_sh + half * 16 + ds * 32);
  }
  // f16: dS is scaled by the largest |dout| of the queries (see above).
  float lift = 1.f, lower = 1.f;
  if constexpr (!kBF16) {
    float top = 0.f;
    for (int g = 0; g < group; ++g)
      for (int i = threadIdx.x; i < qs.len; i += kDkvThreads)
        top = fmaxf(top, p.top[(int64_t)(kv * group + g) * p.total_q + qs.row + i]);
    top = group_max<64>(top);
    if (lane == 0) s_top[wave] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_top[w]);
    const int e = top_exponent(top);
    lift = pow2(-e - kF16Lift);
    lower = pow2(e);
  }

  TileAt<D> ta(lane);
  f32x16_t dk[DT], dv[DT];
#pragma unroll
  for (int dt = 0; dt < DT; ++dt) dk[dt] = dv[dt] = f32x16_t{};
  int tq = t0;  // the step's tile of queries
  for (int it = 0; it < steps; ++it) {
    wait_vmcnt<0>();
    __syncthreads();
    if (it + 1 < steps) issue((it + 1) & 1);
    const char* const sq = s_qd + (it & 1) * 2 * TILE_B;
    const char* const sd = sq + TILE_B;
    const float* const st = s_st + (it & 1) * 2 * kBwdTile + 32 * sub + 4 * half;
    const int i0 = tq * kBwdTile + 32 * sub;
    if (++tq == t0 + nt) tq = t0;
    // No query of these sees a key of the wave, or there are none.
    if ((p.causal && i0 + 31 + ahead < wkey) || i0 >= qs.len) continue;
    ta.rebuild();
    f32x16_t s = {}, dp;
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) s = mfma32<kBF16>(ta.a(sq, sub, ds), kreg[ds], s);
    if (p.causal && i0 + ahead < wkey + 31) {
      const int rel = key - ahead - i0 - 4 * half;  // query 8 (i / 4) + i % 4 sees it iff >= rel
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (8 * (i / 4) + i % 4 < rel) s[i] = -INFINITY;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const f32x4_t lse = *reinterpret_cast<const f32x4_t*>(st + 8 * j);
      const f32x4_t d = *reinterpret_cast<const f32x4_t*>(st + kBwdTile + 8 * j);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float off = kBF16 ? lse[i] : lse[i] - (float)kF16Lift;
        s[4 * j + i] = fast_exp2(fmaf(s[4 * j + i], p.scale_log2, -off));
        dp[4 * j + i] = -d[i];
      }
    }
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint4 pb = pack_b<kBF16>(s, hf);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) dv[dt] = mfma32<kBF16>(ta.at(sd, sub, hf, dt), pb, dv[dt]);
    }
    ta.rebuild();
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) dp = mfma32<kBF16>(ta.a(sd, sub, ds), vreg[ds], dp);
#pragma unroll
    for (int i = 0; i < 16; ++i) dp[i] *= kBF16 ? s[i] : s[i] * lift;
#pragma unroll
    for (int hf = 0; hf < 2; ++hf) {
      const uint4 db = pack_b<kBF16>(dp, hf);
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) dk[dt] = mfma32<kBF16>(ta.at(sq, sub, hf, dt), db, dk[dt]);
    }
  }
  // The halves' sums: the first half's waves write dk, the second's dv.
  char* const s_x = s_qd + (wave & 3) * (64 * D / 2 * 4);
  __syncthreads();  // every wave is done with the tiles
  if (sub == 0) put_acc<DT>(dv, s_x, lane);
  __syncthreads();
  if (sub == 1) add_acc<DT>(dv, s_x, lane);
  __syncthreads();
  if (sub == 1) put_acc<DT>(dk, s_x, lane);
  __syncthreads();
  if (sub == 0) add_acc<DT>(dk, s_x, lane);
  __syncthreads();
  char* const s_w = s_qd + wave * 32 * ROWB;
  if (sub == 0)
    write_rows<kBF16, D>(dk, p.scale * lower, s_w, p.dk + (int64_t)ks.row * p.dk_st + kv * p.dk_sh,
                         p.dk_st, wkey, ks.len, lane);
  else
    write_rows<kBF16, D>(dv, kBF16 ? 1.f : pow2(-kF16Lift), s_w,
                         p.dv + (int64_t)ks.row * p.dv_st + kv * p.dv_sh, p.dv_st, wkey, ks.len,
                         lane);
}

// Both launches for one 16-bit type and head_dim, instantiated in
// varlen_backward_<type>.hip.
template <bool kBF16, int D>
void launch_varlen_backward(const VarlenBwdParams& p, hipStream_t st);

template <bool kBF16, int D>
static void launch_varlen_backward_d(const VarlenBwdParams& p, hipStream_t st) {
  hipLaunchKernelGGL((varlen_dq_kernel<kBF16, D>), dim3((unsigned)p.q_tiles * p.num_heads),
                     dim3(kBwdThreads), 0, st, p);
  hipLaunchKernelGGL((varlen_dkv_kernel<kBF16, D>), dim3((unsigned)p.k_tiles * p.num_kv_heads),
                     dim3(kDkvThreads), 0, st, p);
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
