// Paged-KV decode attention over MXFP4 pools (mx4.h) on CDNA4 matrix cores.
//
// The mathematics, partitions and merge are those of paged_decode_mfma.h: for
// each (sequence, kv head) the G query heads of the group attend the tokens
// j < L that the mask leaves, by an online softmax in the exp2 domain.  What
// differs is that a row is 17 D / 32 bytes (68 at head_dim 128), so a CU's
// share of the HBM rate is a row every ~7 cycles and the work between the load
// and the matrix cores is what has to be kept small:
//
//   * S^T = K Q^T takes the codes as they are: v_mfma_scale_f32_16x16x128
//     multiplies e2m1 K rows (A: 16 bytes a lane, its scale byte beside them)
//     by an fp8 Q.  A query is cut once into e4m3 terms, each holding four
//     more of its significant bits (two for bf16, three for f16) with a power
//     of two of its own, so that the products lose nothing of it.  The
//     instruction aligns the products of neighbouring k before adding: sums
//     came out within 4.2e-5 of the norm of the products (rms 4e-6 over 12800
//     sums), against 2^-9 by which P is rounded below.
//   * O^T += V^T P^T takes V in 16 bits.  A lane holds D / 16 neighbouring
//     elements of eight tokens (one load a token), converts them with their
//     scales (two elements an instruction) and pairs tokens with v_perm: no
//     LDS and no transposing read.  P^T is the S^T accumulator packed in place.
//
// A workgroup is W waves; wave w takes the partition's 32-token steps w, w + W,
// ... with no barrier, its loads going straight to registers, one step or more
// ahead.  The waves merge through LDS at the end.
#pragma once

#include "mx4.h"
#include "paged_decode_mfma.h"

namespace va {

struct DecodeMx4Params : DecodeParams {
  char* ks;  // scale bytes
  char* vs;
  int64_t sc_blk, sc_slot, sc_head;  // bytes
};

typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

constexpr int kMx4Step = 32;  // tokens a wave reduces at a time: two 16-token tiles

// S^T += K Q^T: e2m1 codes of 16 tokens against e4m3 queries.
__device__ inline mf_f32x4 mx4_qk(uint4 k, int ks, const mx_i32x8& q, int qs, mf_f32x4 c) {
  const mx_i32x8 a = {(int)k.x, (int)k.y, (int)k.z, (int)k.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, q, c, 4 /* e2m1 */, 0 /* e4m3 */, 0,
                                                          ks, 0, qs);
}

// O^T += V^T P^T over 32 tokens, 16-bit.
template <typename ET>
__device__ inline mf_f32x4 mx4_pv(uint4 v, uint4 p, mf_f32x4 c) {
  return DecodeMma<ET>::qk(v, p, c);
}

// N e4m3 terms of 16 floats: term t takes what the terms before it left, times
// 16 each time, so its unit is 2^-4 of the one before.  x is consumed.
template <int N>
__device__ inline void mx4_split16(float (&x)[16], uint4 (&term)[N]) {
#pragma unroll
  for (int t = 0; t < N; ++t) {
    int w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
      w[i] = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], w[i], true);
    }
    term[t] = make_uint4(w[0], w[1], w[2], w[3]);
    if (t + 1 < N) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], false);
        const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8(w[i], true);
        x[4 * i] = (x[4 * i] - lo[0]) * 16.0f;
        x[4 * i + 1] = (x[4 * i + 1] - lo[1]) * 16.0f;
        x[4 * i + 2] = (x[4 * i + 2] - hi[0]) * 16.0f;
        x[4 * i + 3] = (x[4 * i + 3] - hi[1]) * 16.0f;
      }
    }
  }
}

template <int D>
struct Mx4DecodeShape {
  static constexpr int ROWB = D / 2;               // bytes of a row's codes
  static constexpr int NS = D / kMx4Group;         // scales of a row
  static constexpr int CH = D <= 128 ? 1 : D / 128;  // 128-element chunks of a row
  static constexpr int NV = D / 16;                // V elements of a lane and token
  using V = std::conditional_t<D == 64, uint16_t, std::conditional_t<D == 128, uint32_t, uint2>>;
  using S = std::conditional_t<D == 64, uint16_t, std::conditional_t<D == 128, uint32_t, uint2>>;
};

// What a lane (r16 = lane % 16, c4 = lane / 16) holds of a step: K codes of
// token r16 of each tile, their scale, V codes (elements NV r16 ..) of tokens
// 4 c4 .. 4 c4 + 3 of both tiles, and all scales of token 4 c4 + r16 % 4.
template <int D>
struct Mx4Step {
  using Sh = Mx4DecodeShape<D>;
  uint4 k[2][Sh::CH];
  uint32_t ks[2][Sh::CH];
  typename Sh::V v[2][4];
  typename Sh::S vs[2];
  uint32_t mask[2];
  uint32_t ok;  // bit t: tile t's block is in the pool and it holds tokens (uniform)
};

template <typename ET, int D, int G, bool kProlog, bool kMask, int W>
__global__ __launch_bounds__(W * 64, 2) void paged_decode_mx4_kernel(DecodeMx4Params p) {
  using Sh = Mx4DecodeShape<D>;
  using M = DecodeMma<ET>;
  using VT = typename Sh::V;
  using ST = typename Sh::S;
  constexpr int CH = Sh::CH, NV = Sh::NV;
  constexpr int NT = W * 64, ROW16 = D * 2;
  constexpr int TERMS = ET::kIsBF16 ? 2 : 3;        // e4m3 terms of a query
  constexpr int QM = D == 64 ? (TERMS + 1) / 2 : TERMS;  // products per chunk (two terms share one at 64)
  constexpr int LPR = D / 8, RPL = 64 / LPR, E = 8;  // the row layout of prologue.h
  constexpr int QROWS = (G + RPL - 1) / RPL;
  static_assert(W % 4 == 0, "the wave merge reads (m, l) of four waves at a time");

  __shared__ __align__(16) float s_o[W * G * D];
  __shared__ __align__(16) float s_ml[2 * G * W];
  // kProlog: each wave's processed query rows and current key row.
  __shared__ __align__(16) char s_q[kProlog ? W * (G + 1) * ROW16 : 16];

  // Grid (kv head, sequence, partition), as the other decode kernels.
  const int b = blockIdx.y, h = blockIdx.x, part = blockIdx.z;
  const int tid = threadIdx.x;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63;
  const int r16 = lane & 15, c4 = lane >> 4;
  const int rg = lane / LPR, col = lane % LPR;
  const int64_t table_row = (int64_t)b * p.t_sb;

  // ---- lengths and the partition ----
  const uint32_t* const lensw = reinterpret_cast<const uint32_t*>(p.lens);
  const uint32_t len_hi = lensw[(int64_t)(b + p.lens_cum) << p.lens_i64];
  const uint32_t len_lo = lensw[(int64_t)b << p.lens_i64];
  int L = __builtin_amdgcn_readfirstlane((int)(p.lens_cum ? len_hi - len_lo : len_lo));
  const int Lr = L;
  L = attend_len(p, L);
  if (p.num_blocks <= 0) L = 0;
  const int col_new = Lr >= 1 ? (int)fast_div((uint32_t)(Lr - 1), p.bs_div) : 0;
  const bool detached = current_row_detached(p, Lr, L, col_new);
  int64_t new_slot = -1;
  if (p.new_slots != nullptr) new_slot = load_index(p.new_slots, b, p.new_slots_i64);
  const int P = partition_tokens(p, L > 0 ? L : 1);
  const int start = part * P;
  const bool last_part = part == p.max_parts - 1;
  const int end = L <= 0 ? 0 : (last_part ? L : min(start + P, L));
  const bool writes_row = detached && part == 0;  // this workgroup writes the detached row
  if (start >= L && !writes_row && !(part == 0 && L <= 0)) return;
  int nparts = L > 0 ? (L + P - 1) / P : 1;
  if (nparts > p.max_parts) nparts = p.max_parts;  // the last partition absorbs the rest

  const int nsteps = end > start ? (end - start + kMx4Step - 1) / kMx4Step : 0;
  const int ntw = nsteps > wave ? (nsteps - wave + W - 1) / W : 0;  // steps of this wave
  const int new_tok =
      (!detached && p.new_k != nullptr && L - 1 >= start && L - 1 < end) ? L - 1 : -1;
  const int new_step = new_tok >= 0 ? (new_tok - start) / kMx4Step : -1;
  const bool owns_new = new_step >= 0 && new_step % W == wave;
  const int64_t cap = (int64_t)p.num_blocks * p.block_size;

  // ---- block ids: lane l holds tile l % 2 of the wave's step 32 i + l / 2,
  // turned into the tile's byte offsets 32 steps at a time; the ids of the
  // next 32 steps are requested then ----
  const int64_t head_off = (int64_t)h * p.s_head, head_sc = (int64_t)h * p.sc_head;
  auto tile_tok = [&](int k0) { return start + kMx4Step * (wave + W * (k0 + (lane >> 1))) + 16 * (lane & 1); };
  auto load_ids = [&](int k0) -> int {
    const int tok = tile_tok(k0);
    if (tok >= end) return -1;
    const int idx = (int)fast_div((uint32_t)tok, p.bs_div);
    if (idx >= p.table_width) return 0;
    // Both words of a 64-bit id (the same word twice of a 32-bit one).
    const int32_t* const w = reinterpret_cast<const int32_t*>(p.table) + ((table_row + idx) << p.table_i64);
    const int lo = w[0], hi = w[p.table_i64];
    return p.table_i64 && hi != 0 ? -1 : lo;
  };
  int64_t toff = 0, tsc = 0;
  uint64_t tok_ok = 0;
  auto take_ids = [&](int k0, int blk) {
    const bool ok = blk >= 0 && blk < p.num_blocks;
    const int64_t bl = ok ? blk : 0;  // tiles without a block read block 0 and are masked
    const int in = ok ? (int)fast_mod((uint32_t)tile_tok(k0), p.bs_div) : 0;
    toff = bl * p.s_blk + (int64_t)in * p.s_slot + head_off;
    tsc = bl * p.sc_blk + (int64_t)in * p.sc_slot + head_sc;
    tok_ok = __builtin_amdgcn_ballot_w64(ok);
  };
  int ids = -1;
  if (ntw > 0) {
    ids = load_ids(0);
    take_ids(0, ids);
    if (ntw > 32) ids = load_ids(32);
  }

  // ---- a step's loads ----
  const uint32_t k_lane = (uint32_t)(r16 * (int)p.s_slot + (D == 64 ? (c4 & 1) : c4) * 16);
  const uint32_t ks_lane = (uint32_t)(r16 * (int)p.sc_slot + (D == 64 ? (c4 & 1) : c4));
  const uint32_t v_lane = (uint32_t)(4 * c4 * (int)p.s_slot + r16 * (NV / 2));
  const uint32_t vs_lane = (uint32_t)((4 * c4 + (r16 & 3)) * (int)p.sc_slot);
  auto lane64 = [&](int64_t x, int l) -> int64_t {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)x, l);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), l);
    return (int64_t)(((uint64_t)hi << 32) | lo);
  };
  const uint8_t* const mrow = p.valid + (kMask ? (int64_t)b * p.valid_sb : 0);
  auto load = [&](Mx4Step<D>& s, int k) {
    if (k > 0 && (k & 31) == 0) {
      take_ids(k, ids);
      if (k + 32 < ntw) ids = load_ids(k + 32);
    }
    s.ok = (uint32_t)(tok_ok >> (2 * (k & 31))) & 3u;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int l = 2 * (k & 31) + t;
      const int64_t off = lane64(toff, l), sc = lane64(tsc, l);
      const char* const kb = p.kp + off;
      const char* const vb = p.vp + off;
      const char* const ksb = p.ks + sc;
      const char* const vsb = p.vs + sc;
#pragma unroll
      for (int c = 0; c < CH; ++c) {
        s.k[t][c] = *reinterpret_cast<const uint4*>(kb + (k_lane + 64u * c));
        s.ks[t][c] = *reinterpret_cast<const uint8_t*>(ksb + (ks_lane + 4u * c));
      }
      s.vs[t] = *reinterpret_cast<const ST*>(vsb + vs_lane);
#pragma unroll
      for (int r = 0; r < 4; ++r)
        s.v[t][r] = *reinterpret_cast<const VT*>(vb + r * p.s_slot + v_lane);
      if constexpr (kMask) {
        const int tok = start + kMx4Step * (wave + W * k) + 16 * t + 4 * c4 + (r16 & 3);
        s.mask[t] = tok < p.valid_len && tok < end ? mrow[tok] : 1u;
      }
    }
  };

  // ---- queries: 16-element pieces of row r16 in the order of the products'
  // B operand (lane (r16, c4): elements 128 c + 64 f + 16 c4 .. + 15, f = 0, 1) ----
  constexpr int PC = D == 64 ? 1 : 2;  // pieces per chunk
  uint4 qraw[CH][PC][2];
  float pro_c[E], pro_s[E];
  const bool has_new = p.new_k != nullptr && (owns_new || (writes_row && wave == 0));
  if constexpr (!kProlog) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int f = 0; f < PC; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          qraw[c][f][i] = r16 < G ? ld16(p.q + b * p.q_sb + (int64_t)(h * G + r16) * p.q_sh +
                                         (128 * c + 64 * f + 16 * c4) * 2 + 16 * i)
                                  : make_uint4(0, 0, 0, 0);
  }

  Mx4Step<D> s0, s1;
  if (ntw > 0) load(s0, 0);
  if (ntw > 1) load(s1, 1);

  if constexpr (kProlog) {
    // Rows in the row layout, then through LDS (the wave's own part of it).
    int64_t pos = load_index(p.pro.pos, b, p.pro.pos_i64);
    pos = pos < 0 ? 0 : (pos >= p.pro.max_pos ? p.pro.max_pos - 1 : pos);
    load_rotary<E, LPR>(p.pro, pos, col, D, pro_c, pro_s);
    char* const s_w = s_q + wave * (G + 1) * ROW16;
    float w[E], x[E];
    convert_weights<E>(load_weights_raw<E>(p.pro.q_w, p.pro.w_dtype, col * E), p.pro.w_dtype, w);
#pragma unroll
    for (int i = 0; i < QROWS; ++i) {
      const int g = rg + RPL * i;
      const uint4 u = g < G ? ld16(p.q + b * p.q_sb + (int64_t)(h * G + g) * p.q_sh + col * 16)
                            : make_uint4(0, 0, 0, 0);
      ET::unpack(u, x);
      qk_prologue<ET, LPR, E>(x, w, p.pro.eps, D, pro_c, pro_s);
      if (g < G) st16(s_w + g * ROW16 + col * 16, ET::pack(x));
    }
    if (has_new) {
      convert_weights<E>(load_weights_raw<E>(p.pro.k_w, p.pro.w_dtype, col * E), p.pro.w_dtype, w);
      ET::unpack(ld16(p.new_k + b * p.nk_sb + h * p.nk_sh + col * 16), x);
      qk_prologue<ET, LPR, E>(x, w, p.pro.eps, D, pro_c, pro_s);
      if (rg == 0) st16(s_w + G * ROW16 + col * 16, ET::pack(x));
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int f = 0; f < PC; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i)
          qraw[c][f][i] =
              r16 < G ? *reinterpret_cast<const uint4*>(s_w + r16 * ROW16 +
                                                        (128 * c + 64 * f + 16 * c4) * 2 + 16 * i)
                      : make_uint4(0, 0, 0, 0);
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
  if (writes_row && wave == 0) store_row();
  if (L <= 0) {
    // Nothing to attend: the output is defined as 0.
    if (part == 0) {
      for (int idx = tid; idx < G * D / E; idx += NT) {
        const int g = idx / (D / E), d = (idx % (D / E)) * E;
        st16(p.out + b * p.o_sb + (int64_t)(h * G + g) * p.o_sh + d * 2, make_uint4(0, 0, 0, 0));
      }
    }
    return;
  }
  if (start >= L) return;

  // ---- the queries' e4m3 terms: the row's largest magnitude goes to
  // [2^7, 2^8), so a term's unit is at most 2^-9 of it ----
  mx_i32x8 qf[QM][CH];
  int qs[QM];
  {
    uint32_t mag = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int f = 0; f < PC; ++f)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t m8 = mx4_absmax8(qraw[c][f][i]);
          mag = mag > m8 ? mag : m8;
        }
    const uint32_t m16 = (uint32_t)__shfl_xor((int)mag, 16, 64);
    mag = mag > m16 ? mag : m16;
    const uint32_t m32 = (uint32_t)__shfl_xor((int)mag, 32, 64);
    mag = mag > m32 ? mag : m32;
    const uint32_t bits = ET::kIsBF16
                              ? mag << 16
                              : __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)mag));
    // Scale byte of the first term; a row below 2^-100 keeps fewer bits, a
    // row with an infinity or a NaN scores NaN.
    int e = (int)(bits >> 23) - 7;
    e = e < 27 ? 27 : e;
    const float inv = __uint_as_float((uint32_t)(254 - e) << 23);
    const bool bad = bits >= 0x7f800000u;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      uint4 term[PC][TERMS];
#pragma unroll
      for (int f = 0; f < PC; ++f) {
        float x[16];
        float(&x0)[8] = *reinterpret_cast<float(*)[8]>(&x[0]);
        float(&x1)[8] = *reinterpret_cast<float(*)[8]>(&x[8]);
        ET::unpack(qraw[c][f][0], x0);
        ET::unpack(qraw[c][f][1], x1);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] *= inv;
        mx4_split16<TERMS>(x, term[f]);
      }
      auto join = [](uint4 lo, uint4 hi) {
        return mx_i32x8{(int)lo.x, (int)lo.y, (int)lo.z, (int)lo.w,
                        (int)hi.x, (int)hi.y, (int)hi.z, (int)hi.w};
      };
#pragma unroll
      for (int t = 0; t < QM; ++t) {
        if constexpr (D == 64)
          qf[t][c] = join(term[0][2 * t], 2 * t + 1 < TERMS ? term[0][2 * t + 1 < TERMS ? 2 * t + 1 : 0]
                                                            : make_uint4(0, 0, 0, 0));
        else
          qf[t][c] = join(term[0][t], term[PC - 1][t]);
      }
    }
#pragma unroll
    for (int t = 0; t < QM; ++t) {
      const int first = D == 64 ? 2 * t + (c4 >> 1) : t;
      qs[t] = bad ? 255 : e - 4 * first;
    }
  }

  float m = kNegBig, l = 0.f;
  mf_f32x4 o[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) o[i] = mf_f32x4{0.f, 0.f, 0.f, 0.f};

  auto reduce = [&](Mx4Step<D>& s, int k) {
    const int c = wave + W * k;
    const int tb = start + kMx4Step * c;
    if (c == new_step && dst_off != INT64_MIN) {
      // The current row in place of the pool's.
      const int r = new_tok - tb;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        if (r16 == r - 16 * t) {
#pragma unroll
          for (int cc = 0; cc < CH; ++cc) {
            s.k[t][cc] = kq[cc];
            s.ks[t][cc] = kqs[cc];
          }
        }
        const int j = r - 16 * t - 4 * c4;  // the lane's token, when 0 .. 3
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (j == i) s.v[t][i] = vq;
      }
    }
    // S^T: the lane's scores are tokens 4 c4 + i of both tiles, head r16.
    mf_f32x4 sc[2];
    uint32_t live[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      sc[t] = mf_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int cc = 0; cc < CH; ++cc)
#pragma unroll
        for (int q = 0; q < QM; ++q) sc[t] = mx4_qk(s.k[t][cc], s.ks[t][cc], qf[q][cc], qs[q], sc[t]);
      const int rel = (s.ok >> t) & 1u ? end - tb - 16 * t - 4 * c4 : 0;
      live[t] = rel >= 4 ? 15u : (rel <= 0 ? 0u : (1u << rel) - 1u);
      if constexpr (kMask)  // lane (i, c4) holds token 4 c4 + i's byte
        live[t] &= (uint32_t)(__builtin_amdgcn_ballot_w64(s.mask[t] != 0) >> (16 * c4));
    }
    float sv[8];
    float mx = -INFINITY;
#pragma unroll
    for (int t = 0; t < 2; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sv[4 * t + i] = (live[t] >> i) & 1u ? sc[t][i] : -INFINITY;
        mx = fmaxf(mx, sv[4 * t + i]);
      }
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

    // V's scales as floats: token i of a tile from lane i of each quad, then
    // the byte of the lane's elements.  A dead token's scale is 0, so that
    // nothing its row may hold (a NaN scale) meets its P of 0.
    float vsc[8];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      uint32_t w;
      if constexpr (D == 256)
        w = 0;
      else
        w = s.vs[t];
      auto bcast = [&](uint32_t x, int i) -> uint32_t {
        switch (i) {
          case 0: return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x00, 0xF, 0xF, false);
          case 1: return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0x55, 0xF, 0xF, false);
          case 2: return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xAA, 0xF, 0xF, false);
          default: return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, 0xFF, 0xF, 0xF, false);
        }
      };
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        uint32_t x;
        if constexpr (D == 256) {
          const uint32_t lo = bcast(s.vs[t].x, i), hi = bcast(s.vs[t].y, i);
          x = r16 >= 8 ? hi : lo;
        } else {
          x = bcast(w, i);
        }
        constexpr int LPS = kMx4Group / NV;  // lanes per scale
        const uint32_t byte = (x >> (((r16 / LPS) & 3) * 8)) & 0xffu;
        uint32_t f = byte << 23;
        if (c == new_step && dst_off != INT64_MIN && new_tok - tb - 16 * t - 4 * c4 == i)
          f = vqs << 23;
        vsc[4 * t + i] = __uint_as_float((live[t] >> i) & 1u ? f : 0u);
      }
    }
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
      for (int j = 0; j < 8; ++j) x[j] = mx4_pair<ET, B>(word(s.v[j >> 2][j & 3], i), vsc[j]);
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
  };

  for (int k = 0; k < ntw; k += 2) {
    reduce(s0, k);
    if (k + 2 < ntw) load(s0, k + 2);
    if (k + 1 < ntw) {
      reduce(s1, k + 1);
      if (k + 3 < ntw) load(s1, k + 3);
    }
  }

  // ---- merge the waves through LDS ----
  l = sum_xor16(l);
  l = sum_xor32(l);
  float* const s_m = s_ml;          // [G][W]
  float* const s_l = s_ml + G * W;  // [G][W]
  if (r16 < G) {
    // Lane (r16, c4) holds o of head r16 at d = NV (4 c4 + r) + i.
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int i = 0; i < NV; i += 4)
        *reinterpret_cast<mf_f32x4*>(s_o + (wave * G + r16) * D + NV * (4 * c4 + r) + i) =
            mf_f32x4{o[i][r], o[i + 1][r], o[i + 2][r], o[i + 3][r]};
    if (c4 == 0) {
      s_m[r16 * W + wave] = ntw > 0 ? m : kNegBig;
      s_l[r16 * W + wave] = ntw > 0 ? l : 0.f;
    }
  }
  __syncthreads();
  const int64_t pair = (int64_t)b * p.num_kv_heads + h;
  for (int qd = tid; qd < G * D / 4; qd += NT) {
    const int g = qd / (D / 4), d = (qd % (D / 4)) * 4;
    float mw[W], lw[W];
#pragma unroll
    for (int w = 0; w < W; w += 4) {
      const mf_f32x4 mv = *reinterpret_cast<const mf_f32x4*>(s_m + g * W + w);
      const mf_f32x4 lv = *reinterpret_cast<const mf_f32x4*>(s_l + g * W + w);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        mw[w + i] = mv[i];
        lw[w + i] = lv[i];
      }
    }
    float Mx = kNegBig;
#pragma unroll
    for (int w = 0; w < W; ++w) Mx = fmaxf(Mx, mw[w]);
    float Lt = 0.f;
    mf_f32x4 acc = mf_f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const float f = fast_exp2(mw[w] - Mx);
      Lt += lw[w] * f;
      acc += f * *reinterpret_cast<const mf_f32x4*>(s_o + (w * G + g) * D + d);
    }
    if (nparts == 1) {
      const float inv = Lt > 0.f ? 1.0f / Lt : (Lt == 0.f ? 0.f : Lt);  // a NaN stays one
      uint2 u;
      u.x = M::pack2(acc[0] * inv, acc[1] * inv);
      u.y = M::pack2(acc[2] * inv, acc[3] * inv);
      *reinterpret_cast<uint2*>(p.out + b * p.o_sb + (int64_t)(h * G + g) * p.o_sh + d * 2) = u;
    } else {
      const int64_t slot = (pair * p.max_parts + part) * G + g;
      *reinterpret_cast<mf_f32x4*>(p.part_o + slot * D + d) = acc;
      if (d == 0) {
        p.part_ml[slot * 2] = Mx;
        p.part_ml[slot * 2 + 1] = Lt;
      }
    }
  }
  if (owns_new) store_row();
}

// ------------------------------------------------------------- launching
template <typename ET, int D, int G, int W>
static void launch_decode_mx4_w(const DecodeMx4Params& p, dim3 grid, hipStream_t s) {
  const dim3 nt(W * 64);
  const bool mask = p.valid != nullptr && p.valid_len > 0;
  if (p.has_pro && mask)
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, true, true, W>), grid, nt, 0, s, p);
  else if (p.has_pro)
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, true, false, W>), grid, nt, 0, s, p);
  else if (mask)
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, false, true, W>), grid, nt, 0, s, p);
  else
    hipLaunchKernelGGL((paged_decode_mx4_kernel<ET, D, G, false, false, W>), grid, nt, 0, s, p);
}

template <typename ET, int D, int G>
static void launch_decode_mx4(const DecodeMx4Params& p, dim3 grid, hipStream_t s) {
  launch_decode_mx4_w<ET, D, G, 8>(p, grid, s);
  if (p.max_parts > 1)
    hipLaunchKernelGGL((paged_decode_merge_kernel<ET, D, G, 2>), dim3(grid.x, grid.y), dim3(256),
                       0, s, p);
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
