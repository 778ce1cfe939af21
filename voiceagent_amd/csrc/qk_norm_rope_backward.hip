// The gradient of the Qwen3 q/k prologue (qk_norm_rope.hip): with n = x r,
// r = 1 / sqrt(mean x^2 + eps), y = n w and z the rotation of y,
//     dy = R^T dz,  dw = sum over tokens and heads of dy n,
//     dx = r (dy w - n mean(dy w n)),
// in fp32 (the forward's roundings to the element type count as the identity).
//
// Bound by HBM: x and dz read, dx written once, 3 x 2 bytes an element in
// 16-bit types.  Rows lie on lanes as in the forward kernel (prologue.h): the
// two sums over a row are DPP reductions.  A lane adds up its own columns'
// dy n of the rows it meets in registers; a workgroup's sums meet in LDS and
// leave as one row of partials, and a second launch (3 to 4 us) adds the partials
// of all workgroups, in a fixed order: no atomics, so calls repeat bit for bit.
#include <algorithm>

#include "fastdiv.h"
#include "prologue.h"

namespace va {

struct QkBwdParams {
  const char* dz[2];  // [q, k] gradients of the outputs
  int64_t dz_st[2], dz_sh[2];  // bytes
  const char* x[2];
  int64_t x_st[2], x_sh[2];
  char* dx[2];
  int64_t dx_st[2], dx_sh[2];
  int32_t hq, hkv;
  uint32_t units;    // of work, unit_div.d a token
  FastDiv unit_div;
  float* part;    // [blocks][2][D]
  PrologueParams pp;
};

constexpr int kQbThreads = 256;
constexpr int kQbBlocks = 1024;  // rows of partials at most
// Row groups of a wave's unit of work, all of whose loads are in flight at once: of
// 16 + 8 heads of 128 in bf16 8561 tokens take 31.8 us (158 MB, 5.0 TB/s) and 420 take
// 5.6; two row groups 32.6 and 5.7, one 38.7 and 5.2 (and leaves three times the
// partial sums).  Half the workgroups, 36 us.  A unit past the last head loads its rows
// again, so what suits depends on the heads: calls of 158 MB with three, two and one
// row groups, both launches, take 37.3, 39.1 and 44.2 us at 16 + 8 heads of 128, 41.9,
// 38.5 and 45.6 at 14 + 14 of 64, 52.5, 49.9 and 62.4 at 8 + 1 of 64, 38.1, 37.0 and
// 42.7 at 8 key heads of 128 alone, 38.4, 39.0 and 42.4 at 7 + 3 of 256, and 34.0, 34.7
// and 39.4 at 16 + 8 of 128 in fp32.
constexpr int kQbChunk = 3;

template <typename ET, int D>
__global__ __launch_bounds__(kQbThreads) void qk_norm_rope_backward_kernel(QkBwdParams p) {
  constexpr int E = ET::kPerVec;
  constexpr int LPR = D / E;
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int col = lane % LPR, sub = lane / LPR;
  const int heads = p.hq + p.hkv;
  // (With no query (key) heads the other side's weights stand in; unused.)
  const WeightRaw<E> wqr = load_weights_raw<E>(p.hq > 0 ? p.pp.q_w : p.pp.k_w, p.pp.w_dtype, col * E);
  const WeightRaw<E> wkr = load_weights_raw<E>(p.hkv > 0 ? p.pp.k_w : p.pp.q_w, p.pp.w_dtype, col * E);
  float dw[2][E] = {};
  for (uint32_t u = blockIdx.x * (kQbThreads / 64) + wave; u < p.units;
       u += gridDim.x * (kQbThreads / 64)) {
    const uint32_t tok = fast_div(u, p.unit_div);
    const int h0 = (int)(u - tok * p.unit_div.d) * kQbChunk * RPW;
    int64_t pos = load_index_words(p.pp.pos, tok, p.pp.pos_i64);
    uint4 xr[kQbChunk], zr[kQbChunk];
#pragma unroll
    for (int j = 0; j < kQbChunk; ++j) {
      const int hh = min(h0 + j * RPW + sub, heads - 1);
      const int side = hh < p.hq ? 0 : 1, head = hh < p.hq ? hh : hh - p.hq;
      const char* const xs = side ? p.x[1] + tok * p.x_st[1] + head * p.x_sh[1]
                                  : p.x[0] + tok * p.x_st[0] + head * p.x_sh[0];
      const char* const zs = side ? p.dz[1] + tok * p.dz_st[1] + head * p.dz_sh[1]
                                  : p.dz[0] + tok * p.dz_st[0] + head * p.dz_sh[0];
      xr[j] = ld16_nt(xs + col * 16);
      zr[j] = ld16_nt(zs + col * 16);
    }
    pos = pos < 0 ? 0 : (pos >= p.pp.max_pos ? p.pp.max_pos - 1 : pos);
    float c[E], s[E];
    load_rotary<E, LPR>(p.pp, pos, col, D, c, s);
#pragma unroll
    for (int j = 0; j < kQbChunk; ++j) {
      if (h0 + j * RPW >= heads) break;  // whole row groups past the token's last row
      const int hh = h0 + j * RPW + sub;
      const bool isq = hh < p.hq, live = hh < heads;
      float x[E], z[E], w[E];
      ET::unpack(xr[j], x);
      ET::unpack(zr[j], z);
      WeightRaw<E> wr;
      wr.a = isq ? wqr.a : wkr.a;
      wr.b = isq ? wqr.b : wkr.b;
      convert_weights<E>(wr, p.pp.w_dtype, w);
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) ss = fmaf(x[e], x[e], ss);
      ss = group_sum<LPR>(ss);
      const float r = 1.0f / sqrtf(ss / (float)D + p.pp.eps);
      // s holds -sin in the row's first half, +sin in the second: the
      // transposed rotation takes the partner's share with its sign turned.
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float dy = fmaf(-rotary_partner<LPR>(z[e]), s[e], z[e] * c[e]);
        x[e] *= r;  // n
        const float g = live ? dy * x[e] : 0.f;
        dw[0][e] += isq ? g : 0.f;
        dw[1][e] += isq ? 0.f : g;
        z[e] = dy * w[e];
        dot = fmaf(z[e], x[e], dot);
      }
      dot = group_sum<LPR>(dot) / (float)D;
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] = r * fmaf(-x[e], dot, z[e]);
      if (live) {
        const int head = isq ? hh : hh - p.hq;
        char* const to = isq ? p.dx[0] + tok * p.dx_st[0] + head * p.dx_sh[0]
                             : p.dx[1] + tok * p.dx_st[1] + head * p.dx_sh[1];
        st16_nt(to + col * 16, ET::pack(x));
      }
    }
  }
  // The workgroup's sums: every lane's go to LDS as they are, and a thread adds up
  // those of one column.  (Summed over a wave's row groups by lane permutes first,
  // 16 columns in turn, they cost a small call 2 us.)
  constexpr int kRowsWg = kQbThreads / 64 * RPW;
  __shared__ float s_dw[kRowsWg][2][D];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int e = 0; e < E; e += 4)
      *reinterpret_cast<float4*>(&s_dw[wave * RPW + sub][side][col * E + e]) =
          make_float4(dw[side][e], dw[side][e + 1], dw[side][e + 2], dw[side][e + 3]);
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kQbThreads) {
    float v = 0.f;
#pragma unroll
    for (int n = 0; n < kRowsWg; ++n) v += (&s_dw[n][0][0])[i];
    p.part[(int64_t)blockIdx.x * 2 * D + i] = v;
  }
}

// dw of both sides: 16 columns a workgroup, 64 strands of partial rows each.
constexpr int kQbSumThreads = 1024, kQbSumCols = 16;
__global__ __launch_bounds__(kQbSumThreads) void qk_weight_sum_kernel(const float* part, int rows,
                                                                      int d, void* dqw, void* dkw,
                                                                      int w_dtype) {
  constexpr int STRANDS = kQbSumThreads / kQbSumCols;
  __shared__ float s_sum[STRANDS][kQbSumCols];
  const int c = threadIdx.x % kQbSumCols, strand = threadIdx.x / kQbSumCols;
  const int col = blockIdx.x * kQbSumCols + c;
  // All of a strand's rows (1 to 16) are requested at once; the last stands in for
  // those that are not there.
  constexpr int kMost = kQbBlocks / STRANDS;
  float x[kMost], v = 0.f;
#pragma unroll
  for (int i = 0; i < kMost; ++i)
    x[i] = rows > 0 ? part[(int64_t)min(strand + i * STRANDS, rows - 1) * 2 * d + col] : 0.f;
#pragma unroll
  for (int i = 0; i < kMost; ++i) v += strand + i * STRANDS < rows ? x[i] : 0.f;
  s_sum[strand][c] = v;
  __syncthreads();
  for (int n = STRANDS / 2; n > 0; n /= 2) {
    if (strand < n) s_sum[strand][c] += s_sum[strand + n][c];
    __syncthreads();
  }
  if (strand != 0) return;
  void* const to = col < d ? dqw : dkw;
  if (to == nullptr) return;
  const int i = col < d ? col : col - d;
  v = s_sum[0][c];
  if (w_dtype == VA_F32)
    reinterpret_cast<float*>(to)[i] = v;
  else if (w_dtype == VA_BF16)
    reinterpret_cast<uint16_t*>(to)[i] = BF16::from_float(v);
  else
    reinterpret_cast<_Float16*>(to)[i] = (_Float16)v;
}

struct QkBwdPlan {
  uint32_t per_token;  // units of a token
  int64_t units;
  int blocks;
};
static QkBwdPlan qk_bwd_plan(const va_qk_norm_rope_bwd_args* a) {
  const int e = a->dtype == VA_F32 ? 4 : 8;
  const int rows = kQbChunk * (64 / (a->head_dim / e));
  QkBwdPlan p;
  p.per_token = (uint32_t)((a->num_heads + a->num_kv_heads + rows - 1) / rows);
  p.units = (int64_t)a->num_tokens * p.per_token;
  p.blocks = (int)std::min<int64_t>(kQbBlocks, (p.units + kQbThreads / 64 - 1) / (kQbThreads / 64));
  return p;
}

template <typename ET>
static void launch_qk_bwd(int D, const QkBwdParams& p, int blocks, hipStream_t st) {
  switch (D) {
    case 64: hipLaunchKernelGGL((qk_norm_rope_backward_kernel<ET, 64>), dim3(blocks), dim3(kQbThreads), 0, st, p); break;
    case 128: hipLaunchKernelGGL((qk_norm_rope_backward_kernel<ET, 128>), dim3(blocks), dim3(kQbThreads), 0, st, p); break;
    case 256: hipLaunchKernelGGL((qk_norm_rope_backward_kernel<ET, 256>), dim3(blocks), dim3(kQbThreads), 0, st, p); break;
  }
}

static bool qk_bwd_sizes(const va_qk_norm_rope_bwd_args* a) {
  return a->num_tokens >= 0 && a->num_heads >= 0 && a->num_kv_heads >= 0 &&
         (int64_t)a->num_heads + a->num_kv_heads > 0 &&
         (int64_t)a->num_heads + a->num_kv_heads <= 65536 &&
         (a->head_dim == 64 || a->head_dim == 128 || a->head_dim == 256);
}

}  // namespace va

extern "C" size_t va_qk_norm_rope_backward_workspace_bytes(const va_qk_norm_rope_bwd_args* a) {
  if (a == nullptr || a->struct_size != sizeof(va_qk_norm_rope_bwd_args) || !va::qk_bwd_sizes(a))
    return 0;
  return (size_t)va::qk_bwd_plan(a).blocks * 2 * a->head_dim * sizeof(float);
}

extern "C" int va_qk_norm_rope_backward(const va_qk_norm_rope_bwd_args* a, void* stream) {
  using namespace va;
  const char* const fn = "va_qk_norm_rope_backward";
  VA_CHECK_ARG(a != nullptr, "%s: null args", fn);
  VA_CHECK_ARG(a->struct_size == sizeof(va_qk_norm_rope_bwd_args),
               "%s: struct_size %u != %zu (header/library mismatch)", fn, a->struct_size,
               sizeof(va_qk_norm_rope_bwd_args));
  const int eb = a->dtype == VA_F32 ? 4 : (a->dtype == VA_BF16 || a->dtype == VA_F16) ? 2 : 0;
  VA_CHECK_ARG(eb != 0, "%s: unknown dtype %d", fn, a->dtype);
  VA_CHECK_ARG(qk_bwd_sizes(a), "%s: num_tokens < 0, head_dim (64, 128 or 256) or head counts "
               "(1 to 65536)", fn);
  const bool any = a->num_tokens > 0;  // (none: the weights' sums are zeros)
  VA_CHECK_ARG(a->num_heads == 0 || ((!any || (a->dq_out && a->q && a->dq)) && a->dq_weight),
               "%s: null pointer argument (query side)", fn);
  VA_CHECK_ARG(a->num_kv_heads == 0 || ((!any || (a->dk_out && a->k && a->dk)) && a->dk_weight),
               "%s: null pointer argument (key side)", fn);
  const va_qk_prologue& pr = a->prologue;
  VA_CHECK_ARG(!any || (pr.cos_sin_cache && pr.positions && pr.max_position > 0 &&
                        pr.cos_sin_stride >= a->head_dim), "%s: rotary cache / positions", fn);
  VA_CHECK_ARG((a->num_heads == 0 || pr.q_norm_weight) && (a->num_kv_heads == 0 || pr.k_norm_weight),
               "%s: norm weights missing", fn);
  VA_CHECK_ARG(pr.weight_dtype == VA_BF16 || pr.weight_dtype == VA_F16 || pr.weight_dtype == VA_F32,
               "%s: weight_dtype", fn);
  VA_CHECK_ARG(pr.positions_dtype == VA_I32 || pr.positions_dtype == VA_I64, "%s: positions_dtype",
               fn);
  const int64_t strides[] = {a->dq_out_stride_tok, a->dq_out_stride_head, a->dk_out_stride_tok,
                             a->dk_out_stride_head, a->q_stride_tok, a->q_stride_head,
                             a->k_stride_tok, a->k_stride_head, a->dq_stride_tok,
                             a->dq_stride_head, a->dk_stride_tok, a->dk_stride_head};
  for (int64_t s : strides)
    VA_CHECK_ARG((s * eb) % 16 == 0, "%s: strides must be 16-byte multiples", fn);
  const uintptr_t ptrs[] = {(uintptr_t)a->dq_out, (uintptr_t)a->dk_out, (uintptr_t)a->q,
                            (uintptr_t)a->k, (uintptr_t)a->dq, (uintptr_t)a->dk};
  for (uintptr_t p : ptrs)
    VA_CHECK_ARG(p % 16 == 0, "%s: pointers must be 16-byte aligned", fn);
  VA_CHECK_ARG((uintptr_t)pr.q_norm_weight % 16 == 0 && (uintptr_t)pr.k_norm_weight % 16 == 0,
               "%s: norm weights must be 16-byte aligned", fn);
  const QkBwdPlan plan = qk_bwd_plan(a);
  VA_CHECK_ARG(plan.units < ((int64_t)1 << 31), "%s: too many (token, head) rows", fn);
  const size_t need = (size_t)plan.blocks * 2 * a->head_dim * sizeof(float);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need || (uintptr_t)a->workspace % 16 != 0)) {
    set_error("%s: needs a 16-byte aligned workspace of %zu bytes", fn, need);
    return VA_ERR_WORKSPACE;
  }
  QkBwdParams p;
  p.dz[0] = (const char*)a->dq_out;
  p.dz_st[0] = a->dq_out_stride_tok * eb;
  p.dz_sh[0] = a->dq_out_stride_head * eb;
  p.dz[1] = (const char*)a->dk_out;
  p.dz_st[1] = a->dk_out_stride_tok * eb;
  p.dz_sh[1] = a->dk_out_stride_head * eb;
  p.x[0] = (const char*)a->q;
  p.x_st[0] = a->q_stride_tok * eb;
  p.x_sh[0] = a->q_stride_head * eb;
  p.x[1] = (const char*)a->k;
  p.x_st[1] = a->k_stride_tok * eb;
  p.x_sh[1] = a->k_stride_head * eb;
  p.dx[0] = (char*)a->dq;
  p.dx_st[0] = a->dq_stride_tok * eb;
  p.dx_sh[0] = a->dq_stride_head * eb;
  p.dx[1] = (char*)a->dk;
  p.dx_st[1] = a->dk_stride_tok * eb;
  p.dx_sh[1] = a->dk_stride_head * eb;
  p.hq = a->num_heads;
  p.hkv = a->num_kv_heads;
  p.units = (uint32_t)plan.units;
  p.unit_div = make_fastdiv(plan.per_token);
  p.part = (float*)a->workspace;
  p.pp.q_w = pr.q_norm_weight;
  p.pp.k_w = pr.k_norm_weight;
  p.pp.w_dtype = pr.weight_dtype;
  p.pp.eps = pr.eps;
  p.pp.cs = pr.cos_sin_cache;
  p.pp.cs_stride = pr.cos_sin_stride;
  p.pp.max_pos = pr.max_position;
  p.pp.pos_i64 = pr.positions_dtype == VA_I64;
  p.pp.pos = pr.positions;
  const hipStream_t st = (hipStream_t)stream;
  if (plan.blocks > 0) {
    switch (a->dtype) {
      case VA_BF16: launch_qk_bwd<BF16>(a->head_dim, p, plan.blocks, st); break;
      case VA_F16: launch_qk_bwd<F16>(a->head_dim, p, plan.blocks, st); break;
      case VA_F32: launch_qk_bwd<F32>(a->head_dim, p, plan.blocks, st); break;
    }
  }
  hipLaunchKernelGGL(qk_weight_sum_kernel, dim3(2 * a->head_dim / kQbSumCols), dim3(kQbSumThreads),
                     0, st, p.part, plan.blocks, a->head_dim,
                     a->num_heads > 0 ? a->dq_weight : nullptr,
                     a->num_kv_heads > 0 ? a->dk_weight : nullptr, pr.weight_dtype);
  return check_launch(fn);
}
