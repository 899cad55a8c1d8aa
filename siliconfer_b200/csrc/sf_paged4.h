// sf_paged4.h -- the 4-bit cache: geometry, and the order of a vector's codes.
//
// Element e of a head of D elements lies in quarter c = e / (D/4) at place r = e % (D/4); its code is bits 4c .. 4c + 3
// of the vector's 16-bit word r and stands for (code - 8) * scale[c].  So a 32-bit word holds the same two places of
// all quarters: one mask gives a pair of codes of one quarter, which is a pair of fp16 numbers as it stands (a code n
// in a number's lowest bits is n * 2^-24), for the keys' products as for the values'; and a rotary pair of a head, or
// of its first half, lies in one word.
#pragma once
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "sf_paged.h"
#include "sf_q4.h"

namespace sf {

// The tokens and pages of a 4-bit cache, for the functions that the e4m3 cache uses; its scales are not floats, and
// nothing reads them through this.
inline sf_paged_cache geometry(const sf_paged4_cache& c) {
  sf_paged_cache g{};
  g.k_codes = c.k_codes;
  g.k_scales = reinterpret_cast<float*>(c.k_scales);
  g.v_codes = c.v_codes;
  g.v_scales = reinterpret_cast<float*>(c.v_scales);
  g.block_table = c.block_table;
  g.seq_lens = c.seq_lens;
  g.starts = c.starts;
  g.num_pages = c.num_pages;
  g.n_kv_heads = c.n_kv_heads;
  g.page_size = c.page_size;
  g.head_dim = c.head_dim;
  g.batch = c.batch;
  g.pages_per_seq = c.pages_per_seq;
  return g;
}

inline int check_paged4(const sf_paged4_cache* c, int T, sf_paged_cache& g) {
  if (!c) return fail(SF_ERR_NULL, "null pointer argument");
  g = geometry(*c);
  if (int rc = check_paged(&g, T)) return rc;
  if (T > 0 && ((reinterpret_cast<uintptr_t>(c->k_scales) | reinterpret_cast<uintptr_t>(c->v_scales)) & 15))
    return fail(SF_ERR_ALIGN, "k_scales and v_scales must be 16-byte aligned");
  return SF_OK;
}

}  // namespace sf
