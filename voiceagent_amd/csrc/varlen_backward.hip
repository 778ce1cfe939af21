// Host side of the varlen attention's gradient: argument checks, workspace and
// dispatch (kernels in varlen_backward_kernel.h, instantiated per element type
// in varlen_backward_{bf16,f16}.hip).
#include <algorithm>

#include "varlen_backward_kernel.h"

namespace va {

// How many workgroups share the queries that see a block of keys.  Few blocks,
// each of them seen by many queries (long sequences, or several query heads to a
// kv head), leave most of the chip idle otherwise, and a block's steps (a tile of
// queries of one head) come one after the other.  Parts save a block that all
// queries see its share of them, about 1.5 us each at head_dim 128 and 1.2 at 64,
// and cost a launch and their sums' way to memory and back.  At head_dim 128, 16
// heads over 8, whole and in parts by this rule's estimate, us a gradient: one
// sequence of 512 rows 43.7 and 34.0 (4 parts), two 44.2 and 42.1 (3), four 48.4
// (whole; in 3 parts 57); one of 2000 142.7 and 108.1 (4); 4 of 600 to 2000, 32
// heads over 4 of 64, dk and dv 291 and 165 (4 parts).  More than two workgroups
// for each place on the chip, that one: 184 (6).
static int dkv_parts(const va_varlen_bwd_args* a) {
  if (a->num_seqs <= 0 || a->num_kv_heads <= 0 || a->total_q <= 0 || a->total_k <= 0) return 1;
  const int64_t blocks = ((int64_t)a->total_k / kDkvKeys + a->num_seqs) * a->num_kv_heads;
  const int64_t slots = (a->head_dim == 64 ? 3 : 2) * (int64_t)current_device_cus();
  const int64_t tiles = ((int64_t)a->total_q / a->num_seqs + kDkvTile - 1) / kDkvTile;
  const int64_t steps = tiles * (a->num_heads / a->num_kv_heads);
  const int64_t most =
      std::min<int64_t>({2 * slots / blocks, steps / (a->causal ? 4 : 2), 16});  // (two steps a part)
  const double step = a->head_dim == 64 ? 1.2 : 1.5;  // us
  const double sums = 2.0 * (2 * kDkvKeys * a->head_dim * 4) / 8e6;  // us a block and part, at 8 TB/s
  int parts = 1;
  double best = 0;
  for (int n = 2; n <= most; ++n) {
    const double saved = step * (double)steps * (n - 1) / n - (4.0 + sums * (double)blocks * n);
    if (saved > best) {
      best = saved;
      parts = n;
    }
  }
  return parts;
}

// Queries of a workgroup of the first launch: two workgroups fit a CU, and where
// blocks of 128 queries would not fill them, blocks of 64, whose keys two waves
// share, take less time: a sequence of 420 rows and 16 heads of 128 15.4 us
// against 18.5, 8 answers of 40 to 260 rows behind 700 keys 27 against 31.  Where
// they do fill them the tiles' copies, twice as many, cost more: windows of 104
// rows 34 us against 27, a sequence of 8192 428 against 401.
static int dq_rows(const va_varlen_bwd_args* a) {
  const int64_t blocks = ((int64_t)a->total_q / 128 + a->num_seqs) * a->num_heads;
  return blocks < 2 * (int64_t)current_device_cus() ? 64 : 128;
}

// The longest sequence, where one launch takes them whole (0: it does not; four tiles
// of 128 rows of 64 are what LDS holds twice, and of 128 elements only once).
static int window_rows(const va_varlen_bwd_args* a) {
  const int most = std::max(a->max_seqlen_q, a->max_seqlen_k);
  return a->head_dim == 64 && a->num_heads == a->num_kv_heads && a->max_seqlen_q > 0 &&
                 a->max_seqlen_k > 0 && most <= kWindowMost
             ? most
             : 0;
}

// Workgroups of a launch: 256 threads each, 2^32 in all.
constexpr int64_t kMostItems = (1 << 24) - 1;

// Workspace: the first launch's results for the second (lse, delta and, for f16,
// the rows' largest |dout|), and the parts' sums.
struct BwdLayout {
  int64_t k_tiles;
  int parts;
  size_t rows, sums, total;  // bytes; sums: where they begin
};
static BwdLayout backward_layout(const va_varlen_bwd_args* a) {
  BwdLayout l;
  l.rows = (size_t)a->num_heads * (size_t)a->total_q * sizeof(float);
  l.k_tiles = (int64_t)a->total_k / kDkvKeys + a->num_seqs + 1;
  l.parts = dkv_parts(a);
  l.sums = (l.rows * (a->dtype == VA_F16 ? 3 : 2) + 255) / 256 * 256;
  l.total = l.sums;
  if (l.parts > 1)
    l.total += (size_t)l.k_tiles * l.parts * a->num_kv_heads * 2 * kDkvKeys * a->head_dim * sizeof(float);
  return l;
}

}  // namespace va

extern "C" size_t va_varlen_attention_backward_workspace_bytes(const va_varlen_bwd_args* a) {
  if (a == nullptr || a->struct_size != sizeof(va_varlen_bwd_args)) return 0;
  if (a->num_heads <= 0 || a->num_kv_heads <= 0 || a->num_heads % a->num_kv_heads != 0 ||
      a->num_seqs < 0 || a->total_q <= 0 || a->total_k < 0 ||
      (a->head_dim != 64 && a->head_dim != 128))
    return 0;
  return va::window_rows(a) > 0 ? 0 : va::backward_layout(a).total;
}

extern "C" int va_varlen_attention_backward(const va_varlen_bwd_args* a, void* stream) {
  using namespace va;
  const char* const fn = "va_varlen_attention_backward";
  VA_CHECK_ARG(a != nullptr, "%s: null args", fn);
  VA_CHECK_ARG(a->struct_size == sizeof(va_varlen_bwd_args),
               "%s: struct_size %u != %zu (header/library mismatch)", fn, a->struct_size,
               sizeof(va_varlen_bwd_args));
  VA_CHECK_ARG(a->num_seqs >= 0 && a->total_q >= 0 && a->total_k >= 0,
               "%s: negative num_seqs, total_q or total_k", fn);
  if (a->total_q == 0 && a->total_k == 0) return VA_OK;
  VA_CHECK_ARG(a->dtype == VA_BF16 || a->dtype == VA_F16,
               "%s: dtype must be VA_BF16 or VA_F16 (MFMA path)", fn);
  VA_CHECK_ARG(a->head_dim == 64 || a->head_dim == 128, "%s: head_dim %d (64 or 128)", fn,
               a->head_dim);
  VA_CHECK_ARG(a->num_kv_heads > 0 && a->num_heads > 0 && a->num_heads % a->num_kv_heads == 0,
               "%s: num_heads (%d) must be a positive multiple of num_kv_heads (%d)", fn,
               a->num_heads, a->num_kv_heads);
  VA_CHECK_ARG(a->cu_seqlens_q && a->cu_seqlens_k, "%s: cu_seqlens missing", fn);
  VA_CHECK_ARG(a->total_q == 0 || (a->q && a->out && a->dout && a->dq),
               "%s: null pointer argument (query side)", fn);
  VA_CHECK_ARG(a->total_k == 0 || (a->k && a->v && a->dk && a->dv),
               "%s: null pointer argument (key side)", fn);
  const int64_t strides[] = {a->q_stride_tok,    a->q_stride_head,    a->k_stride_tok,
                             a->k_stride_head,   a->v_stride_tok,     a->v_stride_head,
                             a->out_stride_tok,  a->out_stride_head,  a->dout_stride_tok,
                             a->dout_stride_head, a->dq_stride_tok,   a->dq_stride_head,
                             a->dk_stride_tok,   a->dk_stride_head,   a->dv_stride_tok,
                             a->dv_stride_head};
  for (int64_t s : strides)
    VA_CHECK_ARG(s % 8 == 0, "%s: strides must be 16-byte multiples", fn);
  // (A tile's lane offsets are 32-bit.)
  const int64_t toks[] = {a->q_stride_tok, a->dout_stride_tok, a->k_stride_tok, a->v_stride_tok};
  for (int64_t s : toks)
    VA_CHECK_ARG(s >= 0 && s * 2 < ((int64_t)1 << 25),
                 "%s: token strides of q, k, v and dout must be non-negative and below 32 MiB", fn);
  const uintptr_t ptrs[] = {(uintptr_t)a->q,    (uintptr_t)a->k,  (uintptr_t)a->v,  (uintptr_t)a->out,
                            (uintptr_t)a->dout, (uintptr_t)a->dq, (uintptr_t)a->dk, (uintptr_t)a->dv};
  for (uintptr_t p : ptrs)
    VA_CHECK_ARG(p % 16 == 0, "%s: pointers must be 16-byte aligned", fn);
  VA_CHECK_ARG(a->scale > 0.f && a->scale < INFINITY, "%s: scale must be > 0", fn);
  // A workgroup per block of every sequence; one more, which finds none, writes
  // the zeros of rows outside the sequences.
  const int q_rows = dq_rows(a);
  const int64_t q_tiles = (int64_t)a->total_q / q_rows + a->num_seqs + 1;
  const BwdLayout lay = backward_layout(a);
  VA_CHECK_ARG(a->max_seqlen_q >= 0 && a->max_seqlen_k >= 0, "%s: negative max_seqlen", fn);
  const int window = window_rows(a);
  VA_CHECK_ARG(((int64_t)a->num_seqs + 1 + std::max(a->total_q, a->total_k) / kWindowExtra) *
                       a->num_heads <= kMostItems && q_tiles * a->num_heads <= kMostItems &&
                   lay.k_tiles * lay.parts * a->num_kv_heads <= kMostItems,
               "%s: too many (sequence, head, block) items", fn);
  const size_t need = a->total_q > 0 && window == 0 ? lay.total : 0;
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need ||
                   (uintptr_t)a->workspace % 16 != 0)) {
    set_error("%s: needs a 16-byte aligned workspace of %zu bytes", fn, need);
    return VA_ERR_WORKSPACE;
  }

  VarlenBwdParams p;
  p.q = (const char*)a->q;
  p.q_st = a->q_stride_tok * 2;
  p.q_sh = a->q_stride_head * 2;
  p.k = (const char*)a->k;
  p.k_st = a->k_stride_tok * 2;
  p.k_sh = a->k_stride_head * 2;
  p.v = (const char*)a->v;
  p.v_st = a->v_stride_tok * 2;
  p.v_sh = a->v_stride_head * 2;
  p.out = (const char*)a->out;
  p.o_st = a->out_stride_tok * 2;
  p.o_sh = a->out_stride_head * 2;
  p.dout = (const char*)a->dout;
  p.do_st = a->dout_stride_tok * 2;
  p.do_sh = a->dout_stride_head * 2;
  p.dq = (char*)a->dq;
  p.dq_st = a->dq_stride_tok * 2;
  p.dq_sh = a->dq_stride_head * 2;
  p.dk = (char*)a->dk;
  p.dk_st = a->dk_stride_tok * 2;
  p.dk_sh = a->dk_stride_head * 2;
  p.dv = (char*)a->dv;
  p.dv_st = a->dv_stride_tok * 2;
  p.dv_sh = a->dv_stride_head * 2;
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.scale = a->scale;
  p.scale_log2 = a->scale * 1.4426950408889634f;
  p.causal = a->causal;
  p.num_seqs = a->num_seqs;
  p.total_q = a->total_q;
  p.total_k = a->total_k;
  p.num_heads = a->num_heads;
  p.num_kv_heads = a->num_kv_heads;
  p.q_tiles = (int)q_tiles;
  p.q_rows = q_rows;
  p.window = window;
  p.k_tiles = (int)lay.k_tiles;
  p.parts = lay.parts;
  p.lse = (float*)a->workspace;
  p.delta = (float*)((char*)a->workspace + lay.rows);
  p.top = (float*)((char*)a->workspace + 2 * lay.rows);
  p.part = (float*)((char*)a->workspace + lay.sums);
  const hipStream_t st = (hipStream_t)stream;
  if (a->dtype == VA_BF16)
    a->head_dim == 64 ? launch_varlen_backward<true, 64>(p, st) : launch_varlen_backward<true, 128>(p, st);
  else
    a->head_dim == 64 ? launch_varlen_backward<false, 64>(p, st) : launch_varlen_backward<false, 128>(p, st);
  return check_launch(fn);
}
