// Rotary positions in every form: of each head's first r elements, pairs
// (2 i, 2 i + 1) or (i, i + r / 2) turn by the angle whose cosine and sine
// stand at [position][i] and [position][r / 2 + i] of the table:
//     a' = a cos - b sin,  b' = b cos + a sin
// (inverse: sin negated, the transposed matrix, which is the gradient); the
// elements from r on are copied.  fp32, rounded once.
//
// Bound by HBM: every row is read and written once.  A lane holds one unit of a
// row (16 bytes of pairs, both halves of it in the half-split form, or 16 bytes
// to copy) of one token, keeps its cosines and sines in registers and takes
// that unit of kRotHeads head rows, all loads in flight at once.  Rows whose
// addresses or sizes are no 16-byte multiples go element by element.
#include <algorithm>

#include "common.h"
#include "fastdiv.h"

namespace va {

struct RotaryParams {
  const char* x[2];  // [q, k]
  int64_t x_st[2], x_sh[2];  // bytes
  char* y[2];
  int64_t y_st[2], y_sh[2];
  int32_t hq, heads;
  int32_t half;             // r / 2
  int32_t turning, units;   // units of a row that turn; with those that are copied
  uint32_t total;           // num_tokens * units
  FastDiv unit_div;
  const float* cs;
  int64_t cs_stride;
  int32_t max_pos, pos_i64;
  const void* pos;
  float sign;  // -1: inverse
};

constexpr int kRotThreads = 256;
// Head rows a lane takes.  16 + 8 heads of 128 in bf16, with 2, 4, 6 and 8: 8561 tokens
// of the whole head in halves (105 MB) 24.6, 25.2, 25.3 and 25.5 us, of half the head
// in interleaved pairs 26.6, 23.9, 24.2 and 23.7; 32 tokens 3.6, 4.3, 4.9 and 5.4.
constexpr int kRotHeads = 4;

// N elements at p as floats, and back.
template <typename ET, int N>
__device__ inline void rot_load(const char* p, float (&f)[N]) {
  if constexpr (N == ET::kPerVec) {
    ET::unpack(ld16_nt(p), f);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (ET::kBytes == 4)
        f[i] = reinterpret_cast<const float*>(p)[i];
      else if constexpr (ET::kIsBF16)
        f[i] = __uint_as_float((uint32_t)reinterpret_cast<const uint16_t*>(p)[i] << 16);
      else
        f[i] = (float)reinterpret_cast<const _Float16*>(p)[i];
    }
  }
}
template <typename ET, int N>
__device__ inline void rot_store(char* p, const float (&f)[N]) {
  if constexpr (N == ET::kPerVec) {
    st16_nt(p, ET::pack(f));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      if constexpr (ET::kBytes == 4)
        reinterpret_cast<float*>(p)[i] = f[i];
      else if constexpr (ET::kIsBF16)
        reinterpret_cast<uint16_t*>(p)[i] = BF16::from_float(f[i]);
      else
        reinterpret_cast<_Float16*>(p)[i] = (_Float16)f[i];
    }
  }
}

// kPairs: interleaved.  E: elements of an access (16 bytes, or one; interleaved
// at least two).
template <typename ET, int E, bool kPairs>
__global__ __launch_bounds__(kRotThreads) void rotary_kernel(RotaryParams p) {
  constexpr int NC = kPairs ? E / 2 : E;           // angles of a unit
  constexpr int CE = E == ET::kPerVec ? E : 1;     // elements of a copied unit
  const uint32_t w = blockIdx.x * kRotThreads + threadIdx.x;
  if (w >= p.total) return;
  const uint32_t tok = fast_div(w, p.unit_div);
  const int u = (int)(w - tok * p.unit_div.d);
  const int h0 = (int)blockIdx.y * kRotHeads;
  // Where head row h0 + j of the token begins, the last one repeated.
  auto source = [&](int j) {
    const int h = min(h0 + j, p.heads - 1);
    return h < p.hq ? p.x[0] + tok * p.x_st[0] + h * p.x_sh[0]
                    : p.x[1] + tok * p.x_st[1] + (h - p.hq) * p.x_sh[1];
  };
  auto target = [&](int j) {
    const int h = h0 + j;
    return h < p.hq ? p.y[0] + tok * p.y_st[0] + h * p.y_sh[0]
                    : p.y[1] + tok * p.y_st[1] + (h - p.hq) * p.y_sh[1];
  };
  if (u >= p.turning) {
    const int64_t at = (int64_t)(2 * p.half + (u - p.turning) * CE) * ET::kBytes;
    float a[kRotHeads][CE];
#pragma unroll
    for (int j = 0; j < kRotHeads; ++j) rot_load<ET, CE>(source(j) + at, a[j]);
#pragma unroll
    for (int j = 0; j < kRotHeads; ++j)
      if (h0 + j < p.heads) rot_store<ET, CE>(target(j) + at, a[j]);
    return;
  }
  int64_t pos = load_index_words(p.pos, tok, p.pos_i64);
  const int64_t at = (int64_t)u * E * ET::kBytes;
  const int64_t other = (int64_t)p.half * ET::kBytes;  // half-split: from a to b
  float a[kRotHeads][E], b[kRotHeads][kPairs ? 1 : E];
#pragma unroll
  for (int j = 0; j < kRotHeads; ++j) {
    rot_load<ET, E>(source(j) + at, a[j]);
    if constexpr (!kPairs) rot_load<ET, E>(source(j) + other + at, b[j]);
  }
  pos = pos < 0 ? 0 : (pos >= p.max_pos ? p.max_pos - 1 : pos);
  const float* const row = p.cs + pos * p.cs_stride + u * NC;
  float c[NC], s[NC];
#pragma unroll
  for (int i = 0; i < NC; ++i) {
    c[i] = row[i];
    s[i] = row[p.half + i] * p.sign;
  }
#pragma unroll
  for (int j = 0; j < kRotHeads; ++j) {
    if (h0 + j >= p.heads) break;
    char* const to = target(j) + at;
    if constexpr (kPairs) {
      float y[E];
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        y[2 * i] = fmaf(a[j][2 * i], c[i], -a[j][2 * i + 1] * s[i]);
        y[2 * i + 1] = fmaf(a[j][2 * i + 1], c[i], a[j][2 * i] * s[i]);
      }
      rot_store<ET, E>(to, y);
    } else {
      float y[E], z[E];
#pragma unroll
      for (int i = 0; i < E; ++i) {
        y[i] = fmaf(a[j][i], c[i], -b[j][i] * s[i]);
        z[i] = fmaf(b[j][i], c[i], a[j][i] * s[i]);
      }
      rot_store<ET, E>(to, y);
      rot_store<ET, E>(to + other, z);
    }
  }
}

template <typename ET>
static void launch_rotary(const RotaryParams& p, bool pairs, bool vec, hipStream_t st) {
  const dim3 grid((p.total + kRotThreads - 1) / kRotThreads,
                  (unsigned)((p.heads + kRotHeads - 1) / kRotHeads));
  constexpr int V = ET::kPerVec;
  if (vec && pairs) hipLaunchKernelGGL((rotary_kernel<ET, V, true>), grid, dim3(kRotThreads), 0, st, p);
  else if (vec) hipLaunchKernelGGL((rotary_kernel<ET, V, false>), grid, dim3(kRotThreads), 0, st, p);
  else if (pairs) hipLaunchKernelGGL((rotary_kernel<ET, 2, true>), grid, dim3(kRotThreads), 0, st, p);
  else hipLaunchKernelGGL((rotary_kernel<ET, 1, false>), grid, dim3(kRotThreads), 0, st, p);
}

}  // namespace va

extern "C" int va_rotary(const va_rotary_args* a, void* stream) {
  using namespace va;
  VA_CHECK_ARG(a != nullptr, "va_rotary: null args");
  VA_CHECK_ARG(a->struct_size == sizeof(va_rotary_args),
               "va_rotary: struct_size %u != %zu (header/library mismatch)", a->struct_size,
               sizeof(va_rotary_args));
  VA_CHECK_ARG(a->num_tokens >= 0, "va_rotary: num_tokens < 0");
  if (a->num_tokens == 0) return VA_OK;
  const int eb = a->dtype == VA_F32 ? 4 : (a->dtype == VA_BF16 || a->dtype == VA_F16) ? 2 : 0;
  VA_CHECK_ARG(eb != 0, "va_rotary: unknown dtype %d", a->dtype);
  VA_CHECK_ARG(a->num_heads >= 0 && a->num_kv_heads >= 0 &&
                   (int64_t)a->num_heads + a->num_kv_heads > 0 &&
                   (int64_t)a->num_heads + a->num_kv_heads <= 65535,
               "va_rotary: there must be 1 to 65535 heads");
  VA_CHECK_ARG(a->rotary_dim > 0 && a->rotary_dim % 2 == 0 && a->rotary_dim <= a->head_dim &&
                   a->head_dim <= (1 << 20),
               "va_rotary: rotary_dim %d must be even and within head_dim %d", a->rotary_dim,
               a->head_dim);
  VA_CHECK_ARG(a->num_heads == 0 || (a->q && a->q_out), "va_rotary: q / q_out missing");
  VA_CHECK_ARG(a->num_kv_heads == 0 || (a->k && a->k_out), "va_rotary: k / k_out missing");
  VA_CHECK_ARG(a->cos_sin_cache && a->positions && a->max_position > 0 &&
                   a->cos_sin_stride >= a->rotary_dim, "va_rotary: rotary cache / positions");
  VA_CHECK_ARG(a->positions_dtype == VA_I32 || a->positions_dtype == VA_I64,
               "va_rotary: positions_dtype");
  RotaryParams p;
  const void* const ptrs[] = {a->q, a->k, a->q_out, a->k_out};
  const int64_t strides[] = {a->q_stride_tok,     a->q_stride_head,     a->k_stride_tok,
                             a->k_stride_head,    a->q_out_stride_tok,  a->q_out_stride_head,
                             a->k_out_stride_tok, a->k_out_stride_head};
  const int per = 16 / eb;
  bool vec = a->head_dim % per == 0 && a->rotary_dim % (a->interleaved ? per : 2 * per) == 0;
  for (const void* q : ptrs) {
    VA_CHECK_ARG((uintptr_t)q % eb == 0, "va_rotary: pointers must be aligned to the elements");
    vec = vec && (uintptr_t)q % 16 == 0;
  }
  for (int64_t s : strides) vec = vec && (s * eb) % 16 == 0;
  p.x[0] = (const char*)a->q;
  p.x_st[0] = a->q_stride_tok * eb;
  p.x_sh[0] = a->q_stride_head * eb;
  p.x[1] = (const char*)a->k;
  p.x_st[1] = a->k_stride_tok * eb;
  p.x_sh[1] = a->k_stride_head * eb;
  p.y[0] = (char*)a->q_out;
  p.y_st[0] = a->q_out_stride_tok * eb;
  p.y_sh[0] = a->q_out_stride_head * eb;
  p.y[1] = (char*)a->k_out;
  p.y_st[1] = a->k_out_stride_tok * eb;
  p.y_sh[1] = a->k_out_stride_head * eb;
  p.hq = a->num_heads;
  p.heads = a->num_heads + a->num_kv_heads;
  p.half = a->rotary_dim / 2;
  p.turning = vec ? a->rotary_dim / (a->interleaved ? per : 2 * per) : p.half;
  // In place there is nothing to copy.
  const bool moved = (a->num_heads > 0 && a->q != a->q_out) || (a->num_kv_heads > 0 && a->k != a->k_out);
  p.units = p.turning + (moved ? (a->head_dim - a->rotary_dim) / (vec ? per : 1) : 0);
  const int64_t total = (int64_t)a->num_tokens * p.units;
  VA_CHECK_ARG(total < ((int64_t)1 << 31), "va_rotary: too many tokens");
  p.total = (uint32_t)total;
  p.unit_div = make_fastdiv((uint32_t)p.units);
  p.cs = a->cos_sin_cache;
  p.cs_stride = a->cos_sin_stride;
  p.max_pos = a->max_position;
  p.pos_i64 = a->positions_dtype == VA_I64;
  p.pos = a->positions;
  p.sign = a->inverse ? -1.f : 1.f;
  const hipStream_t st = (hipStream_t)stream;
  switch (a->dtype) {
    case VA_BF16: launch_rotary<BF16>(p, a->interleaved != 0, vec, st); break;
    case VA_F16: launch_rotary<F16>(p, a->interleaved != 0, vec, st); break;
    case VA_F32: launch_rotary<F32>(p, a->interleaved != 0, vec, st); break;
  }
  return check_launch("va_rotary");
}
