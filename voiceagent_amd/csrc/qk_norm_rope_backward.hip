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
// leave as one row of partials, and a second launch adds the partials of all
// workgroups, in a fixed order: no atomics, so calls repeat bit for bit.
#include <algorithm>

#include "prologue.h"

namespace va {

struct QkBwdParams {
  const char* dz[2];  // [q, k] gradients of the outputs
  int64_t dz_st[2], dz_sh[2];  // bytes
  const char* x[2];
  int64_t x_st[2], x_sh[2];
  char* dx[2];
  int64_t dx_st[2], dx_sh[2];
  int32_t num_tokens, hq, hkv;
  int32_t waves_per_token, groups_per_wave;
  int64_t units;  // num_tokens * waves_per_token
  float* part;    // [blocks][2][D]
  PrologueParams pp;
};

constexpr int kQbThreads = 256;
constexpr int kQbBlocks = 1024;  // rows of partials at most
// Row groups whose loads (x and dz) a lane keeps in flight at once.
constexpr int kQbChunk = 3;
constexpr int64_t kQbTargetWaves = 4096;

template <typename ET, int D>
__global__ __launch_bounds__(kQbThreads) void qk_norm_rope_backward_kernel(QkBwdParams p) {
  constexpr int E = ET::kPerVec;
  constexpr int LPR = D / E;
  constexpr int RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int col = lane % LPR, sub = lane / LPR;
  const int heads = p.hq + p.hkv;
  float w[2][E], dw[2][E];
#pragma unroll
  for (int e = 0; e < E; ++e) {
    // (With no query (key) heads the other side's weights stand in; unused.)
    w[0][e] = load_weight(p.hq > 0 ? p.pp.q_w : p.pp.k_w, p.pp.w_dtype, col * E + e);
    w[1][e] = load_weight(p.hkv > 0 ? p.pp.k_w : p.pp.q_w, p.pp.w_dtype, col * E + e);
    dw[0][e] = dw[1][e] = 0.f;
  }
  for (int64_t u = (int64_t)blockIdx.x * (kQbThreads / 64) + wave; u < p.units;
       u += (int64_t)gridDim.x * (kQbThreads / 64)) {
    const int64_t tok = u / p.waves_per_token;
    const int r0 = (int)(u % p.waves_per_token) * p.groups_per_wave * RPW;
    const int r1 = min(r0 + p.groups_per_wave * RPW, heads);
    int64_t pos = load_index(p.pp.pos, tok, p.pp.pos_i64);
    float c[E], s[E];
    for (int h0 = r0; h0 < r1; h0 += kQbChunk * RPW) {
      uint4 xr[kQbChunk], zr[kQbChunk];
#pragma unroll
      for (int j = 0; j < kQbChunk; ++j) {
        const int hh = min(h0 + j * RPW + sub, r1 - 1);
        const int side = hh < p.hq ? 0 : 1, head = hh < p.hq ? hh : hh - p.hq;
        const char* const xs = side ? p.x[1] + tok * p.x_st[1] + head * p.x_sh[1]
                                    : p.x[0] + tok * p.x_st[0] + head * p.x_sh[0];
        const char* const zs = side ? p.dz[1] + tok * p.dz_st[1] + head * p.dz_sh[1]
                                    : p.dz[0] + tok * p.dz_st[0] + head * p.dz_sh[0];
        xr[j] = ld16_nt(xs + col * 16);
        zr[j] = ld16_nt(zs + col * 16);
      }
      if (h0 == r0) {
        pos = pos < 0 ? 0 : (pos >= p.pp.max_pos ? p.pp.max_pos - 1 : pos);
        load_rotary<E, LPR>(p.pp, pos, col, D, c, s);
      }
#pragma unroll
      for (int j = 0; j < kQbChunk; ++j) {
        if (h0 + j * RPW >= r1) break;  // whole row groups past the wave's last row
        const int hh = h0 + j * RPW + sub;
        const bool isq = hh < p.hq, live = hh < r1;
        float x[E], z[E];
        ET::unpack(xr[j], x);
        ET::unpack(zr[j], z);
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
          z[e] = dy * (isq ? w[0][e] : w[1][e]);
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
  }
  // The workgroup's sums: over a wave's row groups, then over its waves.
  __shared__ float s_dw[kQbThreads / 64][2][D];
#pragma unroll
  for (int side = 0; side < 2; ++side)
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float v = strided_sum<LPR>(dw[side][e]);
      if (sub == 0) s_dw[wave][side][col * E + e] = v;
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * D; i += kQbThreads) {
    const float* const v = &s_dw[0][0][0] + i;
    p.part[(int64_t)blockIdx.x * 2 * D + i] = (v[0] + v[2 * D]) + (v[4 * D] + v[6 * D]);
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
  float v = 0.f;
#pragma unroll 4
  for (int r = strand; r < rows; r += STRANDS) v += part[(int64_t)r * 2 * d + col];
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
  int wpt, gpw;
  int64_t units;
  int blocks;
};
static QkBwdPlan qk_bwd_plan(const va_qk_norm_rope_bwd_args* a) {
  const int e = a->dtype == VA_F32 ? 4 : 8;
  const int rpw = 64 / (a->head_dim / e);
  const int groups = (a->num_heads + a->num_kv_heads + rpw - 1) / rpw;
  QkBwdPlan p{};
  if (a->num_tokens == 0) return p;
  // Waves per token as in the forward: several while the tokens alone would not
  // fill the chip.
  p.wpt = (int)std::min<int64_t>(
      groups, std::max<int64_t>(1, (kQbTargetWaves + a->num_tokens - 1) / a->num_tokens));
  p.gpw = (groups + p.wpt - 1) / p.wpt;
  p.wpt = (groups + p.gpw - 1) / p.gpw;
  p.units = (int64_t)a->num_tokens * p.wpt;
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
  const QkBwdPlan plan = qk_bwd_plan(a);
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
  p.num_tokens = a->num_tokens;
  p.hq = a->num_heads;
  p.hkv = a->num_kv_heads;
  p.waves_per_token = plan.wpt;
  p.groups_per_wave = plan.gpw;
  p.units = plan.units;
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
