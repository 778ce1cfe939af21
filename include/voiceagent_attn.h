/*
 * voiceagent_attn.h — C ABI of the MI355X (gfx950) attention core for qwen_asr_vllm.
 *
 * Every entry point takes one plain-old-data argument struct plus a HIP stream
 * handle (passed as void*, so this header needs no HIP include), launches on
 * that stream, never allocates, never synchronises the host, and returns
 * VA_OK (0) or a negative status.  The message for the last failure on the
 * calling thread is available from va_last_error().
 *
 * Tensors are described by device pointers and element (not byte) strides;
 * the innermost (head_dim) dimension is always contiguous.  Element type is
 * chosen by a va_dtype; index arrays (block tables, lengths, slot maps) by a
 * va_index_dtype.  The caller owns every buffer.
 *
 * Reference interfaces replaced (paths relative to the reference repository):
 *   va_store_kvcache      <- store_kvcache / _store_kvcache_kernel,
 *                            qwen_asr_vllm/layers/attention.py:31-67
 *   va_paged_decode       <- flash_attn_varlen_func(block_table=..., q_len 1),
 *                            qwen_asr_vllm/layers/attention.py:87-107, and
 *                            paged_attention_decode / _paged_decode_attention_kernel,
 *                            qwen_asr_vllm/agent/qwen_tts_paged_attention.py:130-287, 383-516
 *   va_varlen_attention   <- flash_attn_varlen_func(causal=True, block_table / no cache),
 *                            qwen_asr_vllm/layers/attention.py:92-107, and
 *                            flash_attn_varlen_func(causal=False),
 *                            qwen_asr_vllm/layers/attention.py:121-139
 *   va_qk_norm_rope       <- q_norm / k_norm + rotary_emb of Qwen3Attention.forward,
 *                            qwen_asr_vllm/models/qwen3.py:42-48 (RMSNorm._norm,
 *                            layers/layernorm.py:19-25; apply_rotary_emb and
 *                            RotaryEmbedding.forward, layers/rotary_embedding.py:9-32);
 *                            also fused into va_paged_decode (va_decode_args.prologue)
 */
#ifndef VOICEAGENT_ATTN_H
#define VOICEAGENT_ATTN_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define VA_ATTN_ABI_VERSION 7

/* status codes */
#define VA_OK 0
#define VA_ERR_INVALID_ARG (-1)
#define VA_ERR_UNSUPPORTED (-2)
#define VA_ERR_WORKSPACE (-3)
#define VA_ERR_LAUNCH (-4)

/* element types */
#define VA_BF16 0
#define VA_F16 1
#define VA_F32 2

/* index types */
#define VA_I32 0
#define VA_I64 1

/* KV pool element formats (va_kv_pool.kv_format) */
#define VA_KV_NATIVE 0   /* the entry point's dtype (bf16 / f16 / f32)              */
#define VA_KV_FP8_E4M3 1 /* OCP float8 e4m3 (float8_e4m3fn); element = code * scale */
#define VA_KV_MXFP4 2    /* OCP MX e2m1 codes with e8m0 scales (the *_mx4 entry points) */

/* how va_decode_args.lens is read */
#define VA_LENS_PER_SEQ 0    /* lens[b] = context length of sequence b           */
#define VA_LENS_CUMULATIVE 1 /* lens[b+1] - lens[b] (cu_seqlens_k, num_seqs + 1) */

/*
 * KV pool addressing shared by all entry points.  Token slot s of a sequence
 * whose block table row is T lives at
 *     base + T[s / block_size] * stride_block + (s % block_size) * stride_slot
 *          + kv_head * stride_head + d
 * which covers the engine's NHD pool [num_blocks, block_size, Hkv, D]
 * (qwen_asr_vllm/engine/model_runner.py:116-131) and the TTS talker's HND
 * pool [pages, Hkv, page_size, D]
 * (qwen_asr_vllm/agent/qwen_tts_outer_paged_cache.py:116-119).
 */
typedef struct va_kv_pool {
  void* k;                /* key pool                                    */
  void* v;                /* value pool (same strides as k)              */
  int64_t stride_block;   /* elements between consecutive blocks/pages   */
  int64_t stride_slot;    /* elements between slots inside one block     */
  int64_t stride_head;    /* elements between kv heads                   */
  int32_t block_size;     /* tokens per block (any positive value)       */
  int32_t num_blocks;     /* blocks in the pool; out-of-range ids are    */
                          /* treated as masked and never dereferenced    */
  /* Element format (VA_KV_*).  An FP8 pool holds OCP e4m3 codes (strides
   * count bytes); a key element's value is code * k_scale, a value
   * element's code * v_scale (one scale per pool, > 0).  Every store into
   * it quantises: code = e4m3_rne(clamp(x * (1 / scale), -448, 448)), with
   * 1 / scale and the product rounded to fp32.  FP8 pools need 16-bit
   * q / k / v and, for decode, a block size that is a multiple of 16. */
  int32_t kv_format;
  float k_scale;
  float v_scale;
} va_kv_pool;

/* ---------------------------------------------------------------- store */
typedef struct va_store_args {
  uint32_t struct_size;   /* sizeof(va_store_args)                        */
  int32_t dtype;          /* VA_BF16 / VA_F16 / VA_F32                    */
  const void* key;        /* [num_tokens, Hkv, D]                         */
  const void* value;
  int64_t key_stride_tok, key_stride_head;
  int64_t value_stride_tok, value_stride_head;
  va_kv_pool pool;
  const void* slot_mapping; /* [num_tokens]; slot < 0 or >= capacity skips */
  int32_t slot_dtype;       /* VA_I32 / VA_I64                             */
  int32_t num_tokens;
  int32_t num_kv_heads;
  int32_t head_dim;
} va_store_args;

/* Scatter key/value rows into the pool by slot_mapping (bit-exact copy).
 * Replaces store_kvcache, qwen_asr_vllm/layers/attention.py:52-67. */
int va_store_kvcache(const va_store_args* args, void* stream);

/* ------------------------------------------------------ q/k prologue */
/* Qwen3's per-head query/key prologue: RMSNorm over head_dim,
 *   n = to_dtype(x * 1/sqrt(mean(x^2) + eps)),  y = to_dtype(n * weight)
 * (layers/layernorm.py:19-25), then rotary embedding in the half-split
 * convention with the fp32 cache [max_position, head_dim] = [cos | sin],
 *   out[i]       = to_dtype(y[i] cos[i] - y[i + D/2] sin[i]),
 *   out[i + D/2] = to_dtype(y[i + D/2] cos[i] + y[i] sin[i]),    i < D/2
 * at the token's position (layers/rotary_embedding.py:9-32).  The rotation's
 * products are rounded before their sum (no fused multiply-add), as torch
 * evaluates them; the mean of squares is summed in another order than
 * torch's (with fused multiply-adds), so 1/sqrt(mean + eps) can differ from
 * torch's in its last bit. */
typedef struct va_qk_prologue {
  const void* q_norm_weight;  /* [head_dim] in weight_dtype                 */
  const void* k_norm_weight;  /* [head_dim] in weight_dtype                 */
  int32_t weight_dtype;       /* VA_BF16 / VA_F16 / VA_F32                  */
  float eps;
  const float* cos_sin_cache; /* [max_position, head_dim]: cos | sin halves */
  int64_t cos_sin_stride;     /* elements between consecutive positions     */
  int32_t max_position;       /* positions are clamped to [0, max_position) */
  int32_t positions_dtype;    /* VA_I32 / VA_I64                            */
  const void* positions;      /* decode: [num_seqs]; va_qk_norm_rope: [num_tokens] */
} va_qk_prologue;

typedef struct va_qk_norm_rope_args {
  uint32_t struct_size;   /* sizeof(va_qk_norm_rope_args)                 */
  int32_t dtype;          /* q, k and the outputs share it                */
  const void* q;          /* [num_tokens, Hq, D]                          */
  int64_t q_stride_tok, q_stride_head;
  const void* k;          /* [num_tokens, Hkv, D]                         */
  int64_t k_stride_tok, k_stride_head;
  void* q_out;            /* [num_tokens, Hq, D]; may equal q (in place)  */
  int64_t q_out_stride_tok, q_out_stride_head;
  void* k_out;            /* [num_tokens, Hkv, D]; may equal k            */
  int64_t k_out_stride_tok, k_out_stride_head;
  int32_t num_tokens, num_heads, num_kv_heads, head_dim;
  va_qk_prologue prologue; /* positions: one per token                    */
} va_qk_norm_rope_args;

/* Apply the prologue to every query and key row (prefill and any batch the
 * fused decode path does not take). */
int va_qk_norm_rope(const va_qk_norm_rope_args* args, void* stream);

/* ---------------------------------------------------- q/k prologue, backward */
/* The gradient of va_qk_norm_rope.  With r = 1/sqrt(mean(x^2) + eps), n = x r,
 * y = n weight and z the rotation of y, from dz: dy is the transposed rotation
 * of dz, dweight = sum over tokens and heads of dy n,
 *   dx = r (dy weight - n mean(dy weight n)).
 * All in fp32, rounded once at the end; the forward's roundings to the element
 * type count as the identity.  No atomics: calls repeat bit for bit.  dq and dk
 * may be dq_out and dk_out or q and k themselves.  Norm weights and rows are
 * 16-byte aligned. */
typedef struct va_qk_norm_rope_bwd_args {
  uint32_t struct_size;   /* sizeof(va_qk_norm_rope_bwd_args)             */
  int32_t dtype;          /* VA_BF16 / VA_F16 / VA_F32, all rows          */
  const void* dq_out;     /* [num_tokens, Hq, D] gradient of q_out        */
  int64_t dq_out_stride_tok, dq_out_stride_head;
  const void* dk_out;     /* [num_tokens, Hkv, D] gradient of k_out       */
  int64_t dk_out_stride_tok, dk_out_stride_head;
  const void* q;          /* the forward's inputs                         */
  int64_t q_stride_tok, q_stride_head;
  const void* k;
  int64_t k_stride_tok, k_stride_head;
  void* dq;               /* [num_tokens, Hq, D]                          */
  int64_t dq_stride_tok, dq_stride_head;
  void* dk;               /* [num_tokens, Hkv, D]                         */
  int64_t dk_stride_tok, dk_stride_head;
  void* dq_weight;        /* [D] in the prologue's weight_dtype           */
  void* dk_weight;
  int32_t num_tokens, num_heads, num_kv_heads, head_dim; /* heads of a side may be 0 */
  va_qk_prologue prologue;
  void* workspace;        /* of va_qk_norm_rope_backward_workspace_bytes  */
  size_t workspace_bytes; /* (written; needs no initialisation)           */
} va_qk_norm_rope_bwd_args;

int va_qk_norm_rope_backward(const va_qk_norm_rope_bwd_args* args, void* stream);
size_t va_qk_norm_rope_backward_workspace_bytes(const va_qk_norm_rope_bwd_args* args);

/* -------------------------------------------------------------- rotary */
/* Rotary positions alone, in every form: of each head's first rotary_dim
 * elements, pairs (2 i, 2 i + 1) (interleaved) or (i, i + rotary_dim / 2) turn,
 *   a' = a cos[i] - b sin[i],  b' = b cos[i] + a sin[i]
 * with the table's row [cos | sin] at the token's position; the others are
 * copied.  inverse negates the sines: the transposed rotation, which is its
 * gradient.  fp32, rounded once.  A scaled table (longer contexts) may carry a
 * factor in its entries. */
typedef struct va_rotary_args {
  uint32_t struct_size;   /* sizeof(va_rotary_args)                       */
  int32_t dtype;          /* VA_BF16 / VA_F16 / VA_F32                    */
  const void* q;          /* [num_tokens, Hq, D]                          */
  int64_t q_stride_tok, q_stride_head;
  const void* k;          /* [num_tokens, Hkv, D]                         */
  int64_t k_stride_tok, k_stride_head;
  void* q_out;            /* may be q itself, k_out k itself (in place)   */
  int64_t q_out_stride_tok, q_out_stride_head;
  void* k_out;
  int64_t k_out_stride_tok, k_out_stride_head;
  int32_t num_tokens, num_heads, num_kv_heads, head_dim; /* heads of a side may be 0 */
  int32_t rotary_dim, interleaved, inverse;
  const float* cos_sin_cache; /* [max_position, rotary_dim]: cos | sin halves */
  int64_t cos_sin_stride;
  int32_t max_position;   /* positions are clamped to [0, max_position)   */
  int32_t positions_dtype;
  const void* positions;  /* [num_tokens]                                 */
} va_rotary_args;

int va_rotary(const va_rotary_args* args, void* stream);

/* --------------------------------------------------------------- decode */
typedef struct va_decode_args {
  uint32_t struct_size;   /* sizeof(va_decode_args)                       */
  int32_t dtype;          /* q, pool, out and new rows share it           */
  const void* q;          /* [num_seqs, Hq, D]: one query token per seq   */
  int64_t q_stride_seq, q_stride_head;
  void* out;              /* [num_seqs, Hq, D] in dtype                   */
  int64_t out_stride_seq, out_stride_head;
  va_kv_pool pool;
  const void* block_tables; /* [num_seqs, table_width]; entries at index  */
  int32_t table_dtype;      /* >= table_width read as block 0, as the TTS  */
  int64_t table_stride_seq; /* padding does (qwen_tts_paged_attention.py:458-465) */
  int32_t table_width;
  const void* lens;       /* see VA_LENS_*                                */
  int32_t lens_dtype;
  int32_t lens_kind;
  const uint8_t* valid_mask; /* optional [num_seqs, valid_len] bool; token */
  int64_t valid_stride_seq;  /* t < len is attended iff t >= valid_len or  */
  int32_t valid_len;         /* valid_mask[b, t] != 0                      */
  /* Optional current row, written to the pool at position len-1 and used
   * for that position in the same launch (the TTS fused write,
   * qwen_tts_paged_attention.py:181-221).  [num_seqs, Hkv, D]. */
  const void* new_k;
  int64_t new_k_stride_seq, new_k_stride_head;
  const void* new_v;
  int64_t new_v_stride_seq, new_v_stride_head;
  /* Optional destination slots for the current row ([num_seqs], slot < 0
   * skips the write and the substitution).  NULL: the slot of position len-1
   * through the block table. */
  const void* new_slots;
  int32_t new_slots_dtype;
  int32_t num_seqs, num_heads, num_kv_heads, head_dim;
  int32_t max_seq_len;    /* upper bound of every len; sizes the grid     */
  int32_t split_tokens;   /* tokens per context partition, 0 = automatic, */
                          /* VA_SPLIT_EXACT: automatic, exact bound       */
  float scale;            /* softmax scale                                */
  void* workspace;        /* partial results; see va_paged_decode_workspace_bytes */
  size_t workspace_bytes; /* (no initialisation needed; launches sharing one   */
                          /*  workspace must be ordered on one stream)         */
  /* Optional Qwen3 prologue (NULL: q and new_k are used as given).  When set,
   * q (and new_k, if given) are the raw projections: q is normalised and
   * rotated at positions[b] before attention, and new_k likewise before it
   * is written and attended (its position is also positions[b]). */
  const va_qk_prologue* prologue;
  /* Optional bounds of the attended keys, as the TTS kernel's MAX_SEQ_LEN
   * (kernel_seq_len) and num_page_slots (kernel_page_count) bound them
   * (qwen_tts_paged_attention.py:223-241): tokens at or past key_limit are
   * not attended (0: no bound), and block-table columns at or past
   * table_read_width read as block 0 when attending (0: table_width).  The
   * current row is still written at len - 1, through the table's own entry
   * (qwen_tts_paged_attention.py:182-221). */
  int32_t key_limit;
  int32_t table_read_width;
} va_decode_args;

/* Bytes of workspace va_paged_decode needs for these arguments (the
 * struct's workspace fields are ignored); 0 when no sequence can span more
 * than one context partition.  With split_tokens = 0 the partition size
 * depends on the current device's compute-unit count, so query the size with
 * the same device current as the launch. */
size_t va_paged_decode_workspace_bytes(const va_decode_args* args);

/* split_tokens = VA_SPLIT_EXACT: the automatic split, told that max_seq_len
 * is the exact longest context of the batch (an eager step's maximum, as
 * qwen_asr_vllm/engine/model_runner.py:213 computes it).  Its partitions are
 * then fixed from max_seq_len at any length, and each workgroup requests its
 * first tiles before the lengths arrive; with 0 that holds only up to 4096
 * tokens, above which each workgroup sizes its partition from its own
 * length (right for a bound that is only an upper limit, such as the
 * max_model_len a captured decode graph passes).  The workspace bound is
 * the automatic split's either way. */
#define VA_SPLIT_EXACT (-1)

/* One-token GQA attention over a paged pool: split-context partitions, then
 * (only when a context spans several) a merge pass.  Replaces the decode use of
 * flash_attn_varlen_func (qwen_asr_vllm/layers/attention.py:96-107) and
 * paged_attention_decode (qwen_tts_paged_attention.py:383-516).  head_dim
 * 64 / 128 / 256 with groups of 1 / 2 / 4 / 8 run the vector kernels (16-byte
 * aligned strides and pointers); any other head_dim up to 1024 and any group
 * run a scalar kernel that needs element alignment only and never splits
 * (no prologue, no FP8 pool there). */
int va_paged_decode(const va_decode_args* args, void* stream);

/* Size of the scratch buffer of va_paged_decode_noalloc, per GPU. */
#define VA_DECODE_NOALLOC_SCRATCH_BYTES ((size_t)4 << 20)

/* va_paged_decode without a caller workspace and without any allocation: the
 * split-context partials live in a scratch buffer of
 * VA_DECODE_NOALLOC_SCRATCH_BYTES that the library holds in device memory, one
 * per GPU, for the life of the process (its address is looked up on the first
 * call on each device).  The args' workspace fields are ignored.  A split
 * needing more than the buffer (only an explicit split_tokens can; every
 * automatic split fits) fails with VA_ERR_WORKSPACE.  Calls that overlap on
 * one GPU (on two streams, say) share the buffer and race: order them.  No
 * counterpart in the reference: it is for callers that cannot allocate, such
 * as code under HIP graph capture that must not touch an allocator, tight
 * serving loops and harnesses that forbid hipMalloc. */
int va_paged_decode_noalloc(const va_decode_args* args, void* stream);

/* --------------------------------------------------------------- varlen */
typedef struct va_varlen_args {
  uint32_t struct_size;   /* sizeof(va_varlen_args)                       */
  int32_t dtype;          /* VA_BF16 / VA_F16                             */
  const void* q;          /* [total_q, Hq, D]                             */
  int64_t q_stride_tok, q_stride_head;
  const void* k;          /* [total_k or total_q, Hkv, D]; NULL with a    */
  int64_t k_stride_tok, k_stride_head; /* pool = every key from the pool  */
  const void* v;
  int64_t v_stride_tok, v_stride_head;
  void* out;              /* [total_q, Hq, D]                             */
  int64_t out_stride_tok, out_stride_head;
  const int32_t* cu_seqlens_q; /* [num_seqs + 1]                          */
  const int32_t* cu_seqlens_k; /* [num_seqs + 1]                          */
  int32_t num_seqs, total_q;
  int32_t num_heads, num_kv_heads, head_dim;
  /* max_seqlen_q sizes the launch's query blocks and must be at least every
   * q_len (as flash_attn_varlen_func requires): query rows past it are not
   * computed.  Key ranges come from cu_seqlens_k; max_seqlen_k, where it is
   * at least max_seqlen_q, only tells the launch how long contexts may be (a
   * pool's table may be wider), for its choice of items and their splitting. */
  int32_t max_seqlen_q, max_seqlen_k;
  int32_t causal;         /* 1: bottom-right aligned causal mask          */
  float scale;
  /* Optional paged pool.  Keys j < k_len - q_len of a sequence come from the
   * pool; the rest from k/v rows aligned with the queries (or from the pool
   * too when k is NULL). */
  va_kv_pool pool;
  const void* block_tables;
  int32_t table_dtype;
  int64_t table_stride_seq;
  int32_t table_width;
  /* Optional fused store: q row i's k/v row is also written to slot
   * slot_mapping[i] (slot < 0 skips), as store_kvcache would. */
  const void* slot_mapping;
  int32_t slot_dtype;
  /* Optional (no varlen launch needs a workspace; va_varlen_workspace_bytes
   * returns 0): with at least va_varlen_split_workspace_bytes, 16-byte
   * aligned, the launch may split long items' keys over several workgroups.
   * No initialisation needed; it is written, so launches sharing one must be
   * ordered on one stream (ABI 6 and earlier left the field unused).  An FP8 pool's prefix rows are converted to the 16-bit type
   * (code * scale, rounded once) inside the kernel, tile by tile, and its
   * new rows are stored quantised after the attention. */
  void* workspace;
  size_t workspace_bytes;
  /* Optional Qwen3 query prologue (NULL: q is used as given).  When set, q
   * holds the raw query projections: each query row is normalised with
   * q_norm_weight and rotated at positions[token] (one position per query
   * token, [total_q]) inside the launch, with the arithmetic of
   * va_qk_norm_rope; k and the pool must already hold normalised, rotated
   * keys (va_qk_norm_rope with num_heads = 0 does the keys alone).  Causal
   * launches with head_dim 128; k_norm_weight is not read. */
  const va_qk_prologue* prologue;
} va_varlen_args;

/* Variable-length attention over packed sequences: causal with bottom-right
 * alignment (prefill, optionally over a paged prefix, with the store and the
 * Qwen3 query prologue fused), or non-causal block-diagonal (audio encoder
 * windows). */
int va_varlen_attention(const va_varlen_args* args, void* stream);

/* Bytes of workspace va_varlen_attention needs: always 0 (kept for callers
 * written against the earlier contract). */
size_t va_varlen_workspace_bytes(const va_varlen_args* args);

/* Bytes of workspace with which va_varlen_attention may split these
 * arguments' long items over several workgroups (few items, or some with far
 * more keys than the others); 0 where splitting does not help.  Without it, or
 * with less, the launch runs unsplit.  A split launch sums in another order and
 * rounds P to 16 bits against other reference maxima, so its result equals the
 * unsplit one up to rounding, and in its last bits depends on the launch's
 * other sequences.  Depends on the current device's compute-unit count. */
size_t va_varlen_split_workspace_bytes(const va_varlen_args* args);

/* --------------------------------------------------- varlen, backward */
/* The gradient of va_varlen_attention without a pool: with P = softmax(scale
 * q k^T) over the visible keys and delta_i = sum_d dout_i out_i,
 *   dS_ij = P_ij (dout_i . v_j - delta_i),  dq_i = scale sum_j dS_ij k_j,
 *   dk_j = scale sum_i dS_ij q_i,  dv_j = sum_i P_ij dout_i,
 * dk and dv summed over the query heads of their group.  P is recomputed, in
 * fp32; P and dS are rounded to the element type before the products with
 * dout, q and k, whose sums are fp32 (f16: both scaled by powers of two first,
 * so that small gradients do not fall among f16's subnormals, nor values of v
 * near f16's largest take dS beyond it).
 * q, k, v, out and dout are as in the forward call (any group size); rows that
 * belong to no sequence get a gradient of zeros, as do queries that see no key
 * and keys that no query sees.  Lengths come from cu_seqlens, held to the rows
 * there are; the maxima only choose the launch, and a sequence longer than a
 * maximum of at most 128 may get NaN.  No atomics: calls repeat bit for bit.  The
 * gradients must not overlap the inputs or one another.  Pointers and strides
 * are 16-byte multiples; token strides of q, k, v and dout are from 0 to under
 * 32 MiB. */
typedef struct va_varlen_bwd_args {
  uint32_t struct_size;   /* sizeof(va_varlen_bwd_args)                   */
  int32_t dtype;          /* VA_BF16 / VA_F16                             */
  const void* q;          /* [total_q, Hq, D]                             */
  int64_t q_stride_tok, q_stride_head;
  const void* k;          /* [total_k, Hkv, D]                            */
  int64_t k_stride_tok, k_stride_head;
  const void* v;
  int64_t v_stride_tok, v_stride_head;
  const void* out;        /* [total_q, Hq, D], the forward's result       */
  int64_t out_stride_tok, out_stride_head;
  const void* dout;       /* [total_q, Hq, D]                             */
  int64_t dout_stride_tok, dout_stride_head;
  void* dq;               /* [total_q, Hq, D]                             */
  int64_t dq_stride_tok, dq_stride_head;
  void* dk;               /* [total_k, Hkv, D]                            */
  int64_t dk_stride_tok, dk_stride_head;
  void* dv;
  int64_t dv_stride_tok, dv_stride_head;
  const int32_t* cu_seqlens_q; /* [num_seqs + 1]                          */
  const int32_t* cu_seqlens_k; /* [num_seqs + 1]                          */
  int32_t num_seqs, total_q, total_k;
  int32_t num_heads, num_kv_heads, head_dim; /* head_dim 64 or 128        */
  int32_t max_seqlen_q, max_seqlen_k; /* at least every length; 0: unknown */
  int32_t causal;         /* 1: bottom-right aligned causal mask          */
  float scale;
  void* workspace;        /* of va_varlen_attention_backward_workspace_bytes */
  size_t workspace_bytes; /* (written; needs no initialisation)           */
} va_varlen_bwd_args;

int va_varlen_attention_backward(const va_varlen_bwd_args* args, void* stream);
size_t va_varlen_attention_backward_workspace_bytes(const va_varlen_bwd_args* args);

/* ----------------------------------------------------------- MXFP4 pools */
/*
 * A pool of kv_format VA_KV_MXFP4 holds a row of D elements as D / 2 bytes of
 * 4-bit e2m1 codes (element 2 i in the low half of byte i) and, in an array of
 * its own, D / 32 e8m0 scale bytes, one per 32 elements: a code c with scale
 * byte s stands for c * 2^(s - 127).  Its va_kv_pool gives the codes, strides
 * counting bytes; va_mx4_scales gives the scales, addressed alike.  The pool's
 * k_scale / v_scale are not read.  Rows of codes are 16-byte aligned, rows of
 * scales aligned to D / 32 bytes where that is 2, 4 or 8.  At head_dim 64 the
 * scales' block stride is a multiple of 4: attention finds a row's pair in an
 * aligned 4-byte word.
 *
 * A store quantises 16-bit rows: the scale is the smallest 2^e with
 * max |x| < 7 * 2^e over the group, with e in [-125, 125] for bf16 rows and
 * [-23, 13] for f16 (6 * 2^e and 2^e / 2 are representable in the type), the
 * codes are x / 2^e rounded to nearest, ties to even, saturating at 6.  A
 * group that holds a NaN gets scale byte 255 and codes 0, and reads as NaN.
 * A pool is read in the type it was written in, or in bf16: f16 does not hold
 * every value that bf16 rows may have stored.
 */
typedef struct va_mx4_scales {
  uint32_t struct_size; /* sizeof(va_mx4_scales)                         */
  void* k;              /* scale bytes of the key pool                   */
  void* v;              /* scale bytes of the value pool (same strides)  */
  int64_t stride_block; /* bytes between consecutive blocks              */
  int64_t stride_slot;  /* bytes between slots inside one block          */
  int64_t stride_head;  /* bytes between kv heads                        */
} va_mx4_scales;

/* va_store_kvcache into an MXFP4 pool; 16-bit key / value rows, head_dim a
 * multiple of 32. */
int va_store_kvcache_mx4(const va_store_args* args, const va_mx4_scales* scales, void* stream);

typedef struct va_load_args {
  uint32_t struct_size;   /* sizeof(va_load_args)                        */
  int32_t dtype;          /* VA_BF16 / VA_F16                            */
  void* key;              /* [num_tokens, Hkv, D], written               */
  void* value;
  int64_t key_stride_tok, key_stride_head;
  int64_t value_stride_tok, value_stride_head;
  va_kv_pool pool;
  const void* slot_mapping; /* [num_tokens]; slot < 0 or >= capacity reads as zeros */
  int32_t slot_dtype;       /* VA_I32 / VA_I64                            */
  int32_t num_tokens;
  int32_t num_kv_heads;
  int32_t head_dim;
} va_load_args;

/* The rows stored at slot_mapping, as 16-bit values (exact in the type they
 * were stored from): the inverse of va_store_kvcache_mx4.  The pool has a block
 * at least. */
int va_load_kvcache_mx4(const va_load_args* args, const va_mx4_scales* scales, void* stream);

/* va_paged_decode over an MXFP4 pool: bf16 / f16 q, head_dim 64 / 128 / 256,
 * group 1 / 2 / 4 / 8, a block size that is a multiple of 16, scale > 0.  The
 * current row is stored quantised and attended as stored. */
int va_paged_decode_mx4(const va_decode_args* args, const va_mx4_scales* scales, void* stream);

/* Bytes of workspace va_paged_decode_mx4 needs for these arguments; see
 * va_paged_decode_workspace_bytes. */
size_t va_paged_decode_mx4_workspace_bytes(const va_decode_args* args);

/* va_varlen_attention over an MXFP4 pool: head_dim 64 / 128, no query
 * prologue.  Prefix rows are converted inside the kernel; new rows are attended
 * as given and stored quantised in the same launch.  The workspace is
 * va_varlen_split_workspace_bytes'. */
int va_varlen_attention_mx4(const va_varlen_args* args, const va_mx4_scales* scales,
                            void* stream);

/* -------------------------------------------------------- step metadata */
/*
 * The metadata of one step over num_seqs requests, from their lengths on the
 * device: request i's new tokens are positions [num_computed[i], lens[i]), its
 * block table is row rows[i] (NULL: row i) of request_tables, and the outputs
 * are those that the engine's host builders make
 * (qwen_asr_vllm/engine/model_runner.py:183-233 and graph_runner.py:150-191).
 * lens[i] is taken as 0 when negative and num_computed[i] held to
 * [0, lens[i]].
 *
 * Rows num_seqs .. padded_seqs - 1 are padding as a captured decode graph has
 * it: one token at position 0 with slot -1, table row 0, key length 1.  A
 * request whose rows[i] is outside the table has slots and entries -1, and so
 * has a token whose column is past the table's width or whose block id is
 * negative.  Tokens past max_tokens are not written; entries of positions and
 * slot_mapping behind the last token are 0 and -1.  Sums stop at 2^31 - 1.
 *
 * totals counts every token, max_tokens or not.  With cut the cumulative
 * lengths are those of the tokens written: a request's queries end where
 * max_tokens does, its keys with them, so attention over max_tokens rows stays
 * inside them whatever the lengths say.  Without it they are the full sums,
 * which attention may be given only where totals[0] <= max_tokens.  Blocks are
 * taken for all of lens either way.
 *
 * With free_count, request i holds the blocks of its computed tokens (columns
 * below ceil(num_computed[i] / block_size)), and the blocks of its new columns
 * are taken from the free list's end: the k-th block taken, in request order
 * and ascending columns, is free_blocks[free_count - 1 - k].  They are written
 * to the request's row of request_tables (rows[i] must then be distinct);
 * columns past its width are not taken, and a request without a row in the
 * table takes none.  When the list runs out, the columns left get -1, and so
 * the slots.  free_count is not written, nor may it lie in totals: totals says
 * what is left, and a launch with the same inputs gives the same outputs.  A
 * step that lacked blocks, or had more tokens than max_tokens, is to be made
 * again from the free_count and the num_computed it began with: columns below
 * num_computed are held whatever the table says, so those that got -1 would
 * stay without a block.  The output arrays may not overlap the input ones.
 */
typedef struct va_batch_args {
  uint32_t struct_size; /* sizeof(va_batch_args)                          */
  int32_t index_dtype;  /* of lens and num_computed: VA_I32 / VA_I64      */
  const void* lens;     /* [num_seqs] context lengths after the step      */
  const void* num_computed; /* [num_seqs] tokens computed before it       */
  int32_t* request_tables;  /* [num_requests, request_width]; read, and   */
  int64_t request_stride;   /* written where blocks are taken             */
  int32_t num_requests, request_width;
  const int32_t* rows;      /* optional [num_seqs]                        */
  int32_t num_seqs, padded_seqs; /* num_seqs <= padded_seqs <= 65535      */
  int32_t block_size;
  int32_t max_tokens;       /* entries of positions and slot_mapping      */
  int64_t* positions;       /* [max_tokens]                               */
  int32_t* slot_mapping;    /* [max_tokens]                               */
  int32_t* cu_seqlens_q;    /* [padded_seqs + 1]                          */
  int32_t* cu_seqlens_k;    /* [padded_seqs + 1]                          */
  int32_t* block_tables;    /* optional [padded_seqs, table_width]; -1    */
  int64_t table_stride;     /* behind a request's last block              */
  int32_t table_width;
  int32_t* totals;          /* [5]: tokens, longest query, longest        */
                            /* context, free blocks left, blocks missing  */
  const int32_t* free_blocks; /* optional, with free_count                */
  const int32_t* free_count;  /* [1] entries of free_blocks in use        */
  int32_t free_capacity;      /* entries of free_blocks                   */
  int32_t cut;                /* cumulative lengths stop at max_tokens    */
} va_batch_args;

int va_batch_metadata(const va_batch_args* args, void* stream);

/* ----------------------------------------------------------------- misc */
const char* va_last_error(void);
int va_abi_version(void);

#ifdef __cplusplus
}
#endif

#endif /* VOICEAGENT_ATTN_H */
