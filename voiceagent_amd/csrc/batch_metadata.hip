// Step metadata from request lengths (va_batch_metadata): positions, slots,
// cumulative lengths and block tables, and the new tokens' blocks off a free
// list.
//
// Every output element follows from its request's lengths and three sums over
// the requests before it (query tokens, computed tokens, blocks taken), so one
// launch does it all: a workgroup serves R consecutive requests, first sums
// the requests before them (16 bytes each, from L2), scans its own, and then
// writes their tokens and table rows, both striped over the grid's second
// dimension.  No workgroup reads what another writes: the blocks of new
// columns come from the free list on both sides (the token's and the table's),
// and the list's count is an input whose new value is an output of its own.
#include <algorithm>

#include "common.h"
#include "fastdiv.h"

namespace va {

constexpr int kBatchThreads = 256;
constexpr int kBatchMaxR = 256;

struct BatchParams {
  const void* lens;
  const void* done;
  int32_t i64;
  int32_t* req;
  int64_t req_stride;
  int32_t num_req, req_width;
  const int32_t* rows;
  int32_t num_seqs, padded, per_wg;
  int32_t block_size, max_tokens;
  FastDiv bs_div;
  int64_t* positions;
  int32_t* slots;
  int32_t* cu_q;
  int32_t* cu_k;
  int32_t* tables;
  int64_t t_stride;
  int32_t t_width;
  int32_t* totals;
  const int32_t* free_blocks;
  const int32_t* free_count;
  int32_t free_capacity;
  int32_t cu_limit;  // cumulative query lengths stop here
};

// A request's computed and context lengths, the table columns it holds and
// needs (padding rows: none), and its row of the request table (-1: outside it,
// -2: padding).  Without a row there is nowhere to write a block: such a request
// takes none.
struct Request {
  int done, len, held, cols, row;
};
__device__ inline Request load_request(const BatchParams& p, int i) {
  Request r;
  if (i >= p.num_seqs) {
    r.done = 0;
    r.len = 1;
    r.held = r.cols = 0;
    r.row = -2;
    return r;
  }
  auto clamp = [](int64_t x, int64_t hi) { return (int)(x < 0 ? 0 : (x > hi ? hi : x)); };
  const int64_t most = INT32_MAX - p.block_size;
  r.len = clamp(load_index(p.lens, i, p.i64), most);
  r.done = clamp(load_index(p.done, i, p.i64), r.len);
  auto columns = [&](int n) {
    const int c = (int)fast_div((uint32_t)(n + p.block_size - 1), p.bs_div);
    return c < p.req_width ? c : p.req_width;
  };
  r.cols = columns(r.len);
  const int row = p.rows != nullptr ? p.rows[i] : i;
  r.row = row >= 0 && row < p.num_req ? row : -1;
  r.held = p.free_count != nullptr && r.row >= 0 ? columns(r.done) : r.cols;
  return r;
}

// Sums of lengths stop at 2^31 - 1, so that no lengths, however wrong, give an
// index that wraps (the sum of non-negative terms stays associative).
__device__ inline int sat_add(int a, int b) { return __builtin_elementwise_add_sat(a, b); }

// Sum (or maximum) of x over the workgroup, in every lane.
template <bool kMax>
__device__ inline int block_all(int x, int* s) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int y = __shfl_xor(x, o, 64);
    x = kMax ? max(x, y) : sat_add(x, y);
  }
  __syncthreads();  // s may still be read from its last use
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = x;
  __syncthreads();
  int r = s[0];
#pragma unroll
  for (int w = 1; w < kBatchThreads / 64; ++w) r = kMax ? max(r, s[w]) : sat_add(r, s[w]);
  return r;
}

__global__ __launch_bounds__(kBatchThreads) void batch_metadata_kernel(BatchParams p) {
  __shared__ int s_red[kBatchThreads / 64];
  __shared__ int s_q[kBatchMaxR + 1], s_take[kBatchMaxR + 1];  // first token / taken block
  __shared__ int s_done[kBatchMaxR], s_held[kBatchMaxR], s_cols[kBatchMaxR], s_row[kBatchMaxR];
  const int tid = threadIdx.x;
  const int r0 = blockIdx.x * p.per_wg;
  const int nr = min(p.per_wg, p.padded - r0);  // requests of this workgroup (0 of an empty batch)
  const bool last = blockIdx.x == gridDim.x - 1;
  const int stripe = blockIdx.y, stripes = gridDim.y;
  const int count = p.free_count != nullptr ? max(0, min(*p.free_count, p.free_capacity)) : 0;

  // The requests before this workgroup's.
  int q0 = 0, done0 = 0, take0 = 0, mq = 0, mk = 0;
  for (int i = tid; i < r0; i += kBatchThreads) {
    const Request r = load_request(p, i);
    q0 = sat_add(q0, r.len - r.done);
    done0 = sat_add(done0, r.done);
    take0 = sat_add(take0, r.cols - r.held);
    mq = max(mq, r.len - r.done);
    mk = max(mk, r.len);
  }
  // Its own, one a lane.
  Request mine = {0, 0, 0, 0, -1};
  if (tid < nr) mine = load_request(p, r0 + tid);
  q0 = block_all<false>(q0, s_red);
  done0 = block_all<false>(done0, s_red);
  take0 = block_all<false>(take0, s_red);
  // Inclusive scans over lanes, then over waves.
  int q = mine.len - mine.done, done = mine.done, take = mine.cols - mine.held;
  const int lane = tid & 63, wave = tid >> 6;
  __shared__ int s_scan[3][kBatchThreads / 64];
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int a = __shfl_up(q, o, 64), b = __shfl_up(done, o, 64), c = __shfl_up(take, o, 64);
    if (lane >= o) {
      q = sat_add(q, a);
      done = sat_add(done, b);
      take = sat_add(take, c);
    }
  }
  if (lane == 63) {
    s_scan[0][wave] = q;
    s_scan[1][wave] = done;
    s_scan[2][wave] = take;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    q = sat_add(q, s_scan[0][w]);
    done = sat_add(done, s_scan[1][w]);
    take = sat_add(take, s_scan[2][w]);
  }
  if (tid == 0) s_q[0] = s_take[0] = 0;
  if (tid < nr) {
    s_q[tid + 1] = q;
    s_take[tid + 1] = take;
    s_done[tid] = mine.done;
    s_held[tid] = mine.held;
    s_cols[tid] = mine.cols;
    s_row[tid] = mine.row;
    if (stripe == 0) {
      // Context tokens are computed ones and those of the queries that there
      // is room for (sums of non-negative terms, saturated at the end alike).
      const int cq = min(sat_add(q0, q), p.cu_limit);
      p.cu_q[r0 + tid + 1] = cq;
      p.cu_k[r0 + tid + 1] = sat_add(sat_add(done0, done), cq);
    }
  }
  if (blockIdx.x == 0 && stripe == 0 && tid == 0) p.cu_q[0] = p.cu_k[0] = 0;
  __syncthreads();
  const int total = s_q[nr];
  if (last && stripe == 0) {
    mq = block_all<true>(max(mq, mine.len - mine.done), s_red);
    mk = block_all<true>(max(mk, mine.len), s_red);
    if (tid == 0) {
      const int taken = sat_add(take0, s_take[nr]);
      p.totals[0] = sat_add(q0, total);
      p.totals[1] = mq;
      p.totals[2] = mk;
      p.totals[3] = max(0, count - taken);
      p.totals[4] = p.free_count != nullptr ? max(0, taken - count) : 0;
    }
  }

  // The block id of column c of the workgroup's request r.
  auto block_at = [&](int r, int c) -> int {
    if (s_row[r] < 0 || c >= s_cols[r]) return -1;
    if (c < s_held[r]) return p.req[(int64_t)s_row[r] * p.req_stride + c];
    const int64_t at = count - 1 - ((int64_t)take0 + s_take[r] + c - s_held[r]);
    return at >= 0 ? p.free_blocks[at] : -1;
  };

  // Tokens.
  const int room = p.max_tokens > q0 ? min(total, p.max_tokens - q0) : 0;
  for (int64_t i = stripe * kBatchThreads + tid; i < room; i += stripes * kBatchThreads) {
    const int t = (int)i;
    int lo = 0, hi = nr;  // the last request whose first token is at most t
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (s_q[mid] <= t) lo = mid;
      else hi = mid;
    }
    int pos = 0, slot = -1;
    if (s_row[lo] != -2) {
      pos = s_done[lo] + t - s_q[lo];
      const int c = (int)fast_div((uint32_t)pos, p.bs_div);
      const int blk = block_at(lo, c);
      const int64_t s = (int64_t)blk * p.block_size + (pos - c * p.block_size);
      if (blk >= 0 && s <= INT32_MAX) slot = (int)s;
    }
    p.positions[q0 + t] = pos;
    p.slots[q0 + t] = slot;
  }
  // Behind the last token.
  if (last)
    for (int64_t t = (int64_t)q0 + total + stripe * kBatchThreads + tid; t < p.max_tokens;
         t += stripes * kBatchThreads) {
      p.positions[t] = 0;
      p.slots[t] = -1;
    }
  // Table rows, a wave each.
  for (int r = wave; r < nr; r += kBatchThreads / 64) {
    const int width = max(p.tables != nullptr ? p.t_width : 0, s_cols[r]);
    for (int c = stripe * 64 + lane; c < width; c += stripes * 64) {
      const int blk = s_row[r] == -2 ? 0 : block_at(r, c);
      if (p.tables != nullptr && c < p.t_width) p.tables[(int64_t)(r0 + r) * p.t_stride + c] = blk;
      if (s_row[r] >= 0 && c >= s_held[r] && c < s_cols[r])
        p.req[(int64_t)s_row[r] * p.req_stride + c] = blk;
    }
  }
}

}  // namespace va

extern "C" int va_batch_metadata(const va_batch_args* a, void* stream) {
  using namespace va;
  VA_CHECK_ARG(a != nullptr, "va_batch_metadata: null args");
  VA_CHECK_ARG(a->struct_size == sizeof(va_batch_args),
               "va_batch_metadata: struct_size %u != %zu (header/library mismatch)",
               a->struct_size, sizeof(va_batch_args));
  VA_CHECK_ARG(a->index_dtype == VA_I32 || a->index_dtype == VA_I64,
               "va_batch_metadata: index_dtype");
  VA_CHECK_ARG(a->num_seqs >= 0 && a->padded_seqs >= a->num_seqs,
               "va_batch_metadata: padded_seqs (%d) must be at least num_seqs (%d), 0 or more",
               a->padded_seqs, a->num_seqs);
  VA_CHECK_ARG(a->padded_seqs <= 65535, "va_batch_metadata: padded_seqs > 65535");
  VA_CHECK_ARG(a->block_size > 0, "va_batch_metadata: block_size");
  VA_CHECK_ARG(a->max_tokens >= 0 && a->num_requests >= 0 && a->request_width >= 0 &&
                   a->table_width >= 0 && a->free_capacity >= 0,
               "va_batch_metadata: sizes must be non-negative");
  VA_CHECK_ARG(a->num_seqs == 0 || (a->lens && a->num_computed),
               "va_batch_metadata: null lengths");
  VA_CHECK_ARG(a->request_tables || a->num_requests == 0 || a->request_width == 0,
               "va_batch_metadata: null request_tables");
  VA_CHECK_ARG(a->num_requests < 2 || a->request_stride >= a->request_width,
               "va_batch_metadata: request_tables rows overlap");
  VA_CHECK_ARG(a->max_tokens == 0 || (a->positions && a->slot_mapping),
               "va_batch_metadata: null positions / slot_mapping");
  VA_CHECK_ARG(a->cu_seqlens_q && a->cu_seqlens_k && a->totals,
               "va_batch_metadata: null output");
  VA_CHECK_ARG(a->block_tables == nullptr || a->padded_seqs < 2 ||
                   a->table_stride >= a->table_width,
               "va_batch_metadata: block_tables rows overlap");
  VA_CHECK_ARG(a->free_count ? a->free_blocks != nullptr || a->free_capacity == 0
                             : a->free_blocks == nullptr,
               "va_batch_metadata: free_blocks and free_count must be given together");
  VA_CHECK_ARG(!a->free_count || (uintptr_t)a->free_count + 4 <= (uintptr_t)a->totals ||
                   (uintptr_t)a->free_count >= (uintptr_t)(a->totals + 5),
               "va_batch_metadata: free_count must not lie in totals (which the launch writes)");

  BatchParams p;
  p.lens = a->lens;
  p.done = a->num_computed;
  p.i64 = a->index_dtype == VA_I64;
  p.req = a->request_tables;
  p.req_stride = a->request_stride;
  p.num_req = a->request_width > 0 ? a->num_requests : 0;
  p.req_width = a->num_requests > 0 ? a->request_width : 0;
  p.rows = a->rows;
  p.num_seqs = a->num_seqs;
  p.padded = a->padded_seqs;
  p.block_size = a->block_size;
  p.max_tokens = a->max_tokens;
  p.cu_limit = a->cut ? a->max_tokens : INT32_MAX;
  p.bs_div = make_fastdiv((uint32_t)a->block_size);
  p.positions = a->positions;
  p.slots = a->slot_mapping;
  p.cu_q = a->cu_seqlens_q;
  p.cu_k = a->cu_seqlens_k;
  p.tables = a->block_tables;
  p.t_stride = a->table_stride;
  p.t_width = a->table_width;
  p.totals = a->totals;
  p.free_blocks = a->free_blocks;
  p.free_count = a->free_count;
  p.free_capacity = a->free_capacity;

  // Four requests a workgroup (a wave's table row each), more where that would
  // take over 512 workgroups, each of which sums all requests before its own;
  // stripes so that a lane writes about four tokens, or columns.
  const int rows = std::max(1, a->padded_seqs);
  p.per_wg = std::min(kBatchMaxR, std::max(4, (rows + 511) / 512));
  const int gx = (rows + p.per_wg - 1) / p.per_wg;
  const int64_t tokens = (a->max_tokens + (int64_t)gx * kBatchThreads * 4 - 1) /
                         ((int64_t)gx * kBatchThreads * 4);
  const int64_t cols = ((int64_t)(a->block_tables ? a->table_width : 0) + 64 * 8 - 1) / (64 * 8);
  const int gy = (int)std::min<int64_t>(64, std::max<int64_t>(1, std::max(tokens, cols)));
  hipLaunchKernelGGL(batch_metadata_kernel, dim3(gx, gy), dim3(kBatchThreads), 0,
                     (hipStream_t)stream, p);
  return check_launch("va_batch_metadata");
}
