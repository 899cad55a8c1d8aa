// sf_paged.h -- which tokens and pages a call on the paged cache works on.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

#include "sf_q4.h"
#include "sf_q4_internal.h"

namespace sf {

constexpr int kMaxBatch = 4096;

// Greatest b in [0, n) with f(b) <= v, for a non-decreasing f with f(0) <= v; the warp probes 32 places at a time.
template <typename F>
__device__ __forceinline__ int warp_last_le(int n, long long v, F&& f) {
  int lo = 0, hi = n;
  const int lane = threadIdx.x & 31;
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32, b = lo + step * (lane + 1);
    const unsigned m = __ballot_sync(0xffffffffu, b < hi && f(b) <= v);
    lo += step * __popc(m);
    hi = min(hi, lo + step);
  }
  return lo;
}

// First new row of sequence b (b = batch: the end), and whether sequence b's rows lie in the call's T rows.
__device__ __forceinline__ int first_row(const sf_paged_cache& c, int T, int b) {
  return c.starts ? c.starts[b] : b * (T / c.batch);
}

__device__ __forceinline__ bool len_ok(const sf_paged_cache& c, int len) {
  return len >= 0 && len <= (long long)c.pages_per_seq * c.page_size;
}

struct TokenAt {
  bool ok;
  int b, pos;
};
// Sequence and position of row `tok` (negative for a padding row and for a row of no sequence, before the first one's or
// behind the last one's); called by whole warps.
__device__ __forceinline__ TokenAt token_at(const sf_paged_cache& c, int T, int tok) {
  const int b = c.starts ? warp_last_le(c.batch, tok, [&](int i) { return (long long)c.starts[i]; })
                         : tok / (T / c.batch);
  const int r0 = first_row(c, T, b), r1 = first_row(c, T, b + 1);
  const bool rows_ok = r0 >= 0 && r0 <= r1 && r1 <= T;
  if (rows_ok && ((b == 0 && tok < r0) || (b == c.batch - 1 && tok >= r1))) return {true, b, -1};
  const int len = c.seq_lens[b];
  return {rows_ok && r0 <= tok && tok < r1 && len_ok(c, len), b, len - r1 + tok};
}

// Work units of an append: one for each page that a sequence's new rows may touch.  Sequence b's units start at
// starts[b] / page_size + 2 b, which leaves room for the pages that n rows touch, at most (n - 2) / page_size + 2.
struct SeqSpan {
  bool ok;
  int b;                // sequence
  int row;              // the call's row of position 0, were it one of them
  int page, lo, hi;     // page of the sequence, and the new positions [lo, hi) that it takes
};
__host__ __device__ __forceinline__ int units_per_seq(int n, int page_size) { return (n + page_size - 2) / page_size + 1; }

inline int max_units(const sf_paged_cache& c, int T) {
  return c.starts ? T / c.page_size + 2 * c.batch : c.batch * units_per_seq(T / c.batch, c.page_size);
}

__device__ __forceinline__ SeqSpan unit_span(const sf_paged_cache& c, int T, int unit) {
  SeqSpan s{};
  int j;
  if (c.starts) {
    const auto at = [&](int i) { return (long long)c.starts[i] / c.page_size + 2ll * i; };
    s.b = warp_last_le(c.batch, unit, at);
    j = (int)(unit - at(s.b));
  } else {
    const int per = units_per_seq(T / c.batch, c.page_size);
    s.b = unit / per;
    j = unit % per;
  }
  const int r0 = first_row(c, T, s.b), r1 = first_row(c, T, s.b + 1), len = c.seq_lens[s.b];
  s.ok = r0 >= 0 && r0 <= r1 && r1 <= T && len_ok(c, len);
  if (!s.ok) return s;
  s.row = r1 - len;
  const int first = max(0, len - (r1 - r0));
  s.page = first / c.page_size + j;
  const long long p0 = (long long)s.page * c.page_size;   // may pass 31 bits for a unit that holds nothing
  s.lo = (int)min((long long)len, max((long long)first, p0));
  s.hi = (int)min((long long)len, p0 + c.page_size);
  return s;
}

inline int check_paged(const sf_paged_cache* c, int T) {
  if (!c) return fail(SF_ERR_NULL, "null pointer argument");
  if (T < 0 || c->batch < 1 || c->n_kv_heads < 1 || c->num_pages < 1 || c->pages_per_seq < 1)
    return fail(SF_ERR_SHAPE, "need T >= 0 and batch, n_kv_heads, num_pages, pages_per_seq >= 1");
  if (c->batch > kMaxBatch) return fail(SF_ERR_UNSUPPORTED, "batch %d is above %d", c->batch, kMaxBatch);
  if (!c->starts && T % c->batch) return fail(SF_ERR_SHAPE, "without starts, T must be a multiple of batch");
  if (c->page_size < 16 || c->page_size > 256 || (c->page_size & (c->page_size - 1)))
    return fail(SF_ERR_UNSUPPORTED, "page_size %d not built (16, 32, 64, 128, 256)", c->page_size);
  if (!(c->head_dim == 64 || c->head_dim == 96 || c->head_dim == 128 || c->head_dim == 256))
    return fail(SF_ERR_UNSUPPORTED, "head_dim %d not built (64, 96, 128, 256)", c->head_dim);
  // the kernels look up to 3 tiles of 128 keys beyond a sequence's last one, in 32 bits
  if ((long long)c->pages_per_seq * c->page_size > 0x7fffffffll - 1023)
    return fail(SF_ERR_SHAPE, "a sequence may hold at most 2^31 - 1024 tokens");
  if (T == 0) return SF_OK;
  if (!c->k_codes || !c->k_scales || !c->v_codes || !c->v_scales || !c->block_table || !c->seq_lens)
    return fail(SF_ERR_NULL, "null pointer argument");
  if ((reinterpret_cast<uintptr_t>(c->k_codes) | reinterpret_cast<uintptr_t>(c->v_codes)) & 15)
    return fail(SF_ERR_ALIGN, "k_codes and v_codes must be 16-byte aligned");
  return SF_OK;
}

}  // namespace sf
