// MXFP4 KV pools: the store of new K/V rows (quantise and scatter by
// slot_mapping, the counterpart of store_kvcache.hip) and the load of stored
// rows (gather by slot and dequantise).
//
// Both move every byte once and are bound by HBM: a row of D elements is 2 D
// bytes on the 16-bit side and 17 D / 32 on the pool's.  The K and V rows of
// all tokens are cut into words of 8 elements (16 bytes and 4), flattened over
// 256-lane workgroups so that consecutive lanes touch consecutive words on
// both sides; a group's 4 words are 4 neighbouring lanes, whose largest
// magnitude meets in two DPP steps.  A lane issues the loads of kWords words,
// 256 words apart, before its first store, with no branch among them: the slots'
// type and the width of slot numbers are template arguments.  8561 rows of 8 heads
// of 128 are stored in 12.5 us and loaded in 9.9 (15.6 and 10.4 with branches on
// them, where the compiler waits for each word's loads in turn); scales written a
// word for four groups instead of a byte each did not help the store (12.8).
#include <type_traits>

#include "fastdiv.h"
#include "mx4.h"

namespace va {

struct Mx4CacheParams {
  char* key;  // the 16-bit rows: read by the store, written by the load
  char* value;
  int64_t key_stride_tok, key_stride_head;      // bytes
  int64_t value_stride_tok, value_stride_head;  // bytes
  char* k_pool;
  char* v_pool;
  int64_t stride_block, stride_slot, stride_head;  // bytes of codes
  uint8_t* k_scales;
  uint8_t* v_scales;
  int64_t sc_block, sc_slot, sc_head;  // bytes
  int64_t capacity;                    // num_blocks * block_size
  int32_t block_size;
  const void* slots;
  int32_t slot_i64;
  uint32_t total_words;  // num_tokens * 2 * words_per_row, below 2^31
  int32_t words_per_row;
  FastDiv tok_div;   // 2 * words_per_row: words per token
  FastDiv head_div;  // head_dim / 8: words per head
  FastDiv bs_div;
  int32_t slot_small;  // capacity <= 2^31: slots divide by bs_div
};

constexpr int kMx4Threads = 256;

// Where word w of the flattened (token, K | V, head, word) space lies.
struct Mx4Word {
  char* row;  // the word's 16 bytes of the 16-bit rows
  uint32_t tok, head, word;
  bool is_v;
};
__device__ inline Mx4Word mx4_word(const Mx4CacheParams& p, uint32_t w) {
  Mx4Word r;
  const uint32_t wpr = (uint32_t)p.words_per_row;
  r.tok = fast_div(w, p.tok_div);
  const uint32_t part = w - r.tok * p.tok_div.d;
  r.is_v = part >= wpr;
  const uint32_t rem = r.is_v ? part - wpr : part;
  r.head = fast_div(rem, p.head_div);
  r.word = rem - r.head * p.head_div.d;
  r.row = (r.is_v ? p.value + (int64_t)r.tok * p.value_stride_tok +
                        (int64_t)r.head * p.value_stride_head
                  : p.key + (int64_t)r.tok * p.key_stride_tok + (int64_t)r.head * p.key_stride_head) +
          r.word * 16;
  return r;
}

// Byte offsets of the word's codes and of its group's scale in the pool; false
// for a slot outside it (-1 is padding), with offsets inside it all the same
// (slot 0's).  kBig: slots past 2^31.
template <bool kBig>
__device__ inline bool mx4_place(const Mx4CacheParams& p, const Mx4Word& r, int64_t slot,
                                 int64_t& codes, int64_t& scale) {
  const bool ok = slot >= 0 && slot < p.capacity;
  slot = ok ? slot : 0;
  const int64_t blk = kBig ? slot / p.block_size : (int64_t)fast_div((uint32_t)slot, p.bs_div);
  const int64_t off = slot - blk * p.block_size;
  codes = blk * p.stride_block + off * p.stride_slot + (int64_t)r.head * p.stride_head + r.word * 4;
  scale = blk * p.sc_block + off * p.sc_slot + (int64_t)r.head * p.sc_head + (r.word >> 2);
  return ok;
}

template <bool kI64>
__device__ inline int64_t mx4_slot(const Mx4CacheParams& p, uint32_t tok) {
  return load_index(p.slots, tok, kI64);
}

template <typename ET, int kWords, bool kI64, bool kBig>
__global__ __launch_bounds__(kMx4Threads) void store_mx4_kernel(Mx4CacheParams p) {
  const uint32_t total = p.total_words;
  for (uint32_t base = blockIdx.x * (kMx4Threads * kWords) + threadIdx.x; base - threadIdx.x < total;
       base += gridDim.x * (kMx4Threads * kWords)) {
    uint4 data[kWords];
    int64_t slot[kWords];
    Mx4Word at[kWords];
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      // Words past the end reload the last word and store nothing; a group is
      // wholly inside or wholly past it (4 words divide the total).
      const uint32_t w = base + u * kMx4Threads;
      at[u] = mx4_word(p, w < total ? w : total - 1);
    }
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      data[u] = ld16_nt(at[u].row);
      slot[u] = mx4_slot<kI64>(p, at[u].tok);
    }
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const uint32_t scale = mx4_scale<ET>(quad_max(mx4_absmax8(data[u])));
      const uint32_t codes = mx4_codes8<ET>(data[u], scale);
      int64_t co, so;
      if (mx4_place<kBig>(p, at[u], slot[u], co, so) && base + u * kMx4Threads < total) {
        *reinterpret_cast<uint32_t*>((at[u].is_v ? p.v_pool : p.k_pool) + co) = codes;
        if ((at[u].word & 3) == 0) (at[u].is_v ? p.v_scales : p.k_scales)[so] = (uint8_t)scale;
      }
    }
  }
}

template <typename ET, int kWords, bool kI64, bool kBig>
__global__ __launch_bounds__(kMx4Threads) void load_mx4_kernel(Mx4CacheParams p) {
  const uint32_t total = p.total_words;
  for (uint32_t base = blockIdx.x * (kMx4Threads * kWords) + threadIdx.x; base < total;
       base += gridDim.x * (kMx4Threads * kWords)) {
    uint32_t codes[kWords], scale[kWords];
    int64_t slot[kWords];
    Mx4Word at[kWords];
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      const uint32_t w = base + u * kMx4Threads;
      at[u] = mx4_word(p, w < total ? w : total - 1);
      slot[u] = mx4_slot<kI64>(p, at[u].tok);
    }
    int64_t co[kWords], so[kWords];
    bool ok[kWords];
#pragma unroll
    for (int u = 0; u < kWords; ++u) ok[u] = mx4_place<kBig>(p, at[u], slot[u], co[u], so[u]);
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      codes[u] = *reinterpret_cast<const uint32_t*>((at[u].is_v ? p.v_pool : p.k_pool) + co[u]);
      scale[u] = (at[u].is_v ? p.v_scales : p.k_scales)[so[u]];
    }
#pragma unroll
    for (int u = 0; u < kWords; ++u) {
      // A slot outside the pool reads as zeros.
      const uint4 v = mx4_values8<ET>(ok[u] ? codes[u] : 0u, ok[u] ? scale[u] : 0u);
      if (base + u * kMx4Threads < total) st16_nt(at[u].row, v);
    }
  }
}

int check_mx4(const char* fn, const va_kv_pool& pool, const va_mx4_scales* sc, int head_dim) {
  VA_CHECK_ARG(sc != nullptr && sc->struct_size == sizeof(va_mx4_scales),
               "%s: scales struct_size %u != %zu (header/library mismatch)", fn,
               sc != nullptr ? sc->struct_size : 0u, sizeof(va_mx4_scales));
  VA_CHECK_ARG(pool.kv_format == VA_KV_MXFP4, "%s: kv_format %d is not VA_KV_MXFP4", fn,
               pool.kv_format);
  VA_CHECK_ARG(sc->k && sc->v, "%s: null scale pointer", fn);
  VA_CHECK_ARG(head_dim > 0 && head_dim % kMx4Group == 0,
               "%s: head_dim %d is not a multiple of 32", fn, head_dim);
  const int64_t pstrides[] = {pool.stride_block, pool.stride_slot, pool.stride_head};
  for (int64_t s : pstrides)
    VA_CHECK_ARG(s % 16 == 0, "%s: pool strides must be 16-byte multiples", fn);
  VA_CHECK_ARG((uintptr_t)pool.k % 16 == 0 && (uintptr_t)pool.v % 16 == 0,
               "%s: pool pointers must be 16-byte aligned", fn);
  // A row's scales are read as one word of 2, 4 or 8 bytes (head_dim 64, 128,
  // 256); other head_dims only as bytes.
  const int64_t word = head_dim / kMx4Group;
  const int64_t align = word == 2 || word == 4 || word == 8 ? word : 1;
  const int64_t sstrides[] = {sc->stride_block, sc->stride_slot, sc->stride_head};
  for (int64_t s : sstrides)
    VA_CHECK_ARG(s % align == 0, "%s: scale strides must be multiples of head_dim / 32 bytes", fn);
  // (The attention finds head_dim 64's pairs of scales in words of 4 bytes, which
  // blocks must not shift.)
  VA_CHECK_ARG(word != 2 || sc->stride_block % 4 == 0,
               "%s: the scales' block stride must be a multiple of 4 bytes", fn);
  VA_CHECK_ARG((uintptr_t)sc->k % align == 0 && (uintptr_t)sc->v % align == 0,
               "%s: scale pointers must be aligned to head_dim / 32 bytes", fn);
  return VA_OK;
}

// What the two entry points share: the checks and the launches, `chunk` tokens
// at a time.
template <bool kStore>
static int mx4_cache(const char* fn, int dtype, char* key, char* value, const int64_t (&strides)[4],
                     const va_kv_pool& pool, const va_mx4_scales* sc, const void* slots,
                     int slot_dtype, int num_tokens, int num_kv_heads, int head_dim, void* stream) {
  VA_CHECK_ARG(dtype == VA_BF16 || dtype == VA_F16, "%s: dtype must be VA_BF16 or VA_F16", fn);
  VA_CHECK_ARG(num_tokens >= 0, "%s: num_tokens < 0", fn);
  if (num_tokens == 0) return VA_OK;
  VA_CHECK_ARG(key && value && pool.k && pool.v && slots, "%s: null pointer argument", fn);
  VA_CHECK_ARG(num_kv_heads > 0, "%s: num_kv_heads", fn);
  VA_CHECK_ARG(pool.block_size > 0 && pool.num_blocks >= 0, "%s: bad pool geometry", fn);
  VA_CHECK_ARG(kStore || pool.num_blocks > 0, "%s: an empty pool has no rows", fn);
  VA_CHECK_ARG(slot_dtype == VA_I32 || slot_dtype == VA_I64,
               "%s: slot_dtype must be VA_I32 or VA_I64", fn);
  if (const int rc = check_mx4(fn, pool, sc, head_dim)) return rc;
  for (int64_t s : strides)
    VA_CHECK_ARG((s * 2) % 16 == 0, "%s: strides must be 16-byte multiples", fn);
  VA_CHECK_ARG((uintptr_t)key % 16 == 0 && (uintptr_t)value % 16 == 0,
               "%s: pointers must be 16-byte aligned", fn);
  const int64_t words_per_tok = 2 * (int64_t)num_kv_heads * (head_dim / 8);
  VA_CHECK_ARG(words_per_tok < ((int64_t)1 << 31), "%s: rows too wide", fn);

  Mx4CacheParams p;
  p.key_stride_tok = strides[0] * 2;
  p.key_stride_head = strides[1] * 2;
  p.value_stride_tok = strides[2] * 2;
  p.value_stride_head = strides[3] * 2;
  p.k_pool = (char*)pool.k;
  p.v_pool = (char*)pool.v;
  p.stride_block = pool.stride_block;
  p.stride_slot = pool.stride_slot;
  p.stride_head = pool.stride_head;
  p.k_scales = (uint8_t*)sc->k;
  p.v_scales = (uint8_t*)sc->v;
  p.sc_block = sc->stride_block;
  p.sc_slot = sc->stride_slot;
  p.sc_head = sc->stride_head;
  p.capacity = (int64_t)pool.num_blocks * pool.block_size;
  p.block_size = pool.block_size;
  p.slot_i64 = slot_dtype == VA_I64;
  p.words_per_row = (int32_t)(words_per_tok / 2);
  p.tok_div = make_fastdiv((uint32_t)words_per_tok);
  p.head_div = make_fastdiv((uint32_t)(head_dim / 8));
  p.bs_div = make_fastdiv((uint32_t)pool.block_size);
  p.slot_small = p.capacity <= ((int64_t)1 << 31);

  const int64_t chunk = (((int64_t)1 << 31) - 1) / words_per_tok;
  const hipStream_t s = (hipStream_t)stream;
  for (int64_t t0 = 0; t0 < num_tokens; t0 += chunk) {
    const int64_t n = num_tokens - t0 < chunk ? num_tokens - t0 : chunk;
    p.key = key + t0 * p.key_stride_tok;
    p.value = value + t0 * p.value_stride_tok;
    p.slots = (const char*)slots + t0 * (p.slot_i64 ? 8 : 4);
    p.total_words = (uint32_t)(n * words_per_tok);
    // Four words per lane once that still gives every CU a workgroup.
    const bool wide = p.total_words >= (uint32_t)current_device_cus() * kMx4Threads * 4u;
    const int64_t per_wg = (int64_t)kMx4Threads * (wide ? 4 : 1);
    int64_t grid = (p.total_words + per_wg - 1) / per_wg;
    if (grid > 65536) grid = 65536;
    const dim3 g((unsigned)grid), b(kMx4Threads);
    auto launch = [&](auto et, auto words, auto i64, auto big) {
      using ET = decltype(et);
      constexpr int kW = decltype(words)::value;
      constexpr bool kI = decltype(i64)::value, kB = decltype(big)::value;
      if constexpr (kStore)
        hipLaunchKernelGGL((store_mx4_kernel<ET, kW, kI, kB>), g, b, 0, s, p);
      else
        hipLaunchKernelGGL((load_mx4_kernel<ET, kW, kI, kB>), g, b, 0, s, p);
    };
    auto by_slots = [&](auto et, auto words) {
      if (!p.slot_i64) launch(et, words, std::false_type{}, std::false_type{});  // all below 2^31
      else if (p.slot_small) launch(et, words, std::true_type{}, std::false_type{});
      else launch(et, words, std::true_type{}, std::true_type{});
    };
    auto by_words = [&](auto et) {
      if (wide) by_slots(et, std::integral_constant<int, 4>{});
      else by_slots(et, std::integral_constant<int, 1>{});
    };
    if (dtype == VA_BF16) by_words(BF16{});
    else by_words(F16{});
  }
  return check_launch(fn);
}

}  // namespace va

extern "C" int va_store_kvcache_mx4(const va_store_args* a, const va_mx4_scales* sc, void* stream) {
  using namespace va;
  VA_CHECK_ARG(a != nullptr, "va_store_kvcache_mx4: null args");
  VA_CHECK_ARG(a->struct_size == sizeof(va_store_args),
               "va_store_kvcache_mx4: struct_size %u != %zu (header/library mismatch)",
               a->struct_size, sizeof(va_store_args));
  const int64_t strides[4] = {a->key_stride_tok, a->key_stride_head, a->value_stride_tok,
                              a->value_stride_head};
  return mx4_cache<true>("va_store_kvcache_mx4", a->dtype, (char*)a->key, (char*)a->value, strides,
                         a->pool, sc, a->slot_mapping, a->slot_dtype, a->num_tokens,
                         a->num_kv_heads, a->head_dim, stream);
}

extern "C" int va_load_kvcache_mx4(const va_load_args* a, const va_mx4_scales* sc, void* stream) {
  using namespace va;
  VA_CHECK_ARG(a != nullptr, "va_load_kvcache_mx4: null args");
  VA_CHECK_ARG(a->struct_size == sizeof(va_load_args),
               "va_load_kvcache_mx4: struct_size %u != %zu (header/library mismatch)",
               a->struct_size, sizeof(va_load_args));
  const int64_t strides[4] = {a->key_stride_tok, a->key_stride_head, a->value_stride_tok,
                              a->value_stride_head};
  return mx4_cache<false>("va_load_kvcache_mx4", a->dtype, (char*)a->key, (char*)a->value, strides,
                          a->pool, sc, a->slot_mapping, a->slot_dtype, a->num_tokens,
                          a->num_kv_heads, a->head_dim, stream);
}
