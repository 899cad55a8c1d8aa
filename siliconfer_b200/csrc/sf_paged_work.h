// sf_paged_work.h -- how a call's attention over a paged cache is cut into shares and joined again; for the kernels over
// the e4m3 cache and over the 4-bit one.
//
// A call's work is a list of units of 128 keys, for each (sequence, kv head, tile of RT query rows) in turn; the list is
// cut into contiguous shares, one per CTA.  A CTA that holds all of a tile's units writes the result; the others leave
// their parts in the workspace, which a second kernel merges.
#pragma once
#include <climits>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_paged.h"
#include "sf_q4_internal.h"

namespace sf {
namespace {

constexpr int UNIT = 128;            // keys of a unit
constexpr int kMaxRows = 8;          // query rows of a tile: 8, or 1 where no sequence has more
constexpr size_t kBlockSmem = 232448;   // 227 KB: dynamic and static arrays of a block
constexpr float kNone = -1e30f;      // the reference of a part without a key
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  sf_paged_cache c;
  const void* q;
  long long qts, qhs;
  void* out;
  float* lse;
  float* part;          // [CTA][2][rows x D unnormalised sums, then rows x (m, l)], up to kMaxRows
  int* desc;            // [CTA][8]: the tile that this CTA began and others ended
  int H, T, G, q_dtype, out_dtype, window, lg_page, resident;
  float scale;
};

struct SeqInfo {
  long long first;      // units of the sequences before
  int len, n;
};

__device__ __forceinline__ float load_q(const AttnArgs& a, long long i) {
  if (a.q_dtype == SF_F32) return static_cast<const float*>(a.q)[i];
  if (a.q_dtype == SF_F16) return __half2float(static_cast<const __half*>(a.q)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[i]);
}
__device__ __forceinline__ void store_out(const AttnArgs& a, size_t o, float v) {
  if (a.out_dtype == SF_F32) static_cast<float*>(a.out)[o] = v;
  else if (a.out_dtype == SF_F16) static_cast<__half*>(a.out)[o] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float lg2(float x) {
  float y;
  asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float warp_max(float x) {
  float y;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(y) : "f"(x));
  return y;
}
// First key that a row sees which sees none from `end` on.  Rows before their sequence have an `end` below zero, which
// must not be taken from a window near 2^31.
__device__ __forceinline__ int first_seen(const AttnArgs& a, int end) {
  return a.window > 0 ? max(0, max(0, end) - a.window) : 0;
}
// First key that the sequence's units cover, a multiple of UNIT.
__device__ __forceinline__ int keys_from(const AttnArgs& a, int len, int n) {
  return first_seen(a, len - n + 1) & ~(UNIT - 1);
}

// A list is long at this many units for each resident CTA: at 80 (64 x 4096 keys, 32 kv heads) the small CTAs gain 0.13
// of the time, at 18 (16 x 8192, 8 kv heads) their own beginnings cost 0.24 of it.
constexpr int kLong = 40;
// CTAs' shares of `total` units: `first` equal ones of the first `most` units, `small` ones of the rest.
struct Shares {
  long long total, most, first, small;
  __device__ __forceinline__ Shares(long long total_, int resident, int grid) : total(total_) {
    const bool two = grid >= 2 * resident && total >= (long long)kLong * resident;
    first = min((long long)min(grid, resident), total);
    small = two ? resident : 0;
    most = two ? total * 4 / 5 : total;
  }
  __device__ __forceinline__ long long ctas() const { return first + small; }
  __device__ __forceinline__ long long begin(long long cta) const {
    return cta <= first ? (first ? most * cta / first : 0) : most + (total - most) * (cta - first) / small;
  }
  // the CTA that holds a unit
  __device__ __forceinline__ long long holder(long long u) const {
    return u < most ? ((u + 1) * first - 1) / most : first + ((u - most + 1) * small - 1) / (total - most);
  }
};

// The part of a tile of query rows that begins at unit u and is this CTA's.
struct Part {
  int b, kvh, row0, last_row, r_first, pos0;
  int ta, tb;                 // keys [ta, tb), ta a multiple of UNIT
  int tile_lo, all_lo, all_hi;   // first key that some row sees; keys that every row sees
  long long u1, seg0, seg1;   // end of the part; units of the whole tile
};
template <int RT>
__device__ __forceinline__ Part part_at(const AttnArgs& a, const SeqInfo* info, long long u, long long u_end, int& b) {
  while (b + 1 < a.c.batch && info[b + 1].first <= u) ++b;
  const SeqInfo s = info[b];
  Part p;
  p.b = b;
  const int tiles = (int)(((long long)s.n * a.G + RT - 1) / RT);
  const int from = keys_from(a, s.len, s.n), per = max(1, (s.len - from + UNIT - 1) / UNIT);
  const long long rel = u - s.first, seg = rel / per;
  const int j0 = (int)(rel - seg * per);
  p.kvh = (int)(seg / tiles);
  p.row0 = (int)(seg % tiles) * RT;
  p.seg0 = s.first + seg * per;
  p.seg1 = p.seg0 + per;
  p.u1 = p.seg1 < u_end ? p.seg1 : u_end;
  p.r_first = first_row(a.c, a.T, b);
  p.pos0 = s.len - s.n;
  p.last_row = min(p.row0 + RT, s.n * a.G) - 1;
  const int tile_hi = p.pos0 + p.last_row / a.G + 1;
  p.all_hi = p.pos0 + p.row0 / a.G + 1;
  p.tile_lo = first_seen(a, p.all_hi);
  p.all_lo = first_seen(a, tile_hi);
  // tiles of keys without one that some row sees are left out
  p.ta = max(from + j0 * UNIT, p.tile_lo & ~(UNIT - 1));
  p.tb = (int)min((long long)tile_hi, from + (long long)(j0 + (p.u1 - u)) * UNIT);
  return p;
}

// Result of the call's rows that no sequence holds, [0, from) and [to, T), each written by one CTA.
__device__ __forceinline__ void clear_rows(const AttnArgs& a, int from, int to) {
  const size_t width = (size_t)a.H * a.c.head_dim;
  for (int i = blockIdx.x; i < from + (a.T - to); i += gridDim.x) {
    const size_t row = i < from ? i : to + (i - from);
    for (size_t e = threadIdx.x; e < width; e += blockDim.x) store_out(a, row * width + e, 0.f);
    if (a.lse)
      for (int h = threadIdx.x; h < a.H; h += blockDim.x) a.lse[row * a.H + h] = -INFINITY;
  }
}

// One block for each (CTA that began a divided tile, row of it): the parts by the same rule, in order.
template <int D, int RT>
__global__ void __launch_bounds__(D) paged_attention_merge_kernel(const AttnArgs a) {
  griddep_wait();
  const int* dsc = a.desc + 8 * blockIdx.x;
  const int parts = dsc[0], row = blockIdx.y, q_row = dsc[3] + row;
  if (parts == 0 || q_row > dsc[4]) return;
  const auto part = [&](int i) {
    return a.part + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kMaxRows * (D + 2);
  };
  float M = kNone;
  for (int i = 0; i < parts; ++i) M = fmaxf(M, part(i)[RT * D + 2 * row]);
  float A = 0.f, Ls = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* p = part(i);
    const float c = ex2(p[RT * D + 2 * row] - M);
    A += p[row * D + threadIdx.x] * c;
    Ls += p[RT * D + 2 * row + 1] * c;
  }
  const size_t th = (size_t)(dsc[1] + q_row / a.G) * a.H + dsc[2] * a.G + q_row % a.G;
  store_out(a, th * D + threadIdx.x, Ls == 0.f ? 0.f : A / Ls);
  if (threadIdx.x == 0 && a.lse) a.lse[th] = Ls == 0.f ? -INFINITY : M * kLn2 + logf(Ls);
}

}  // namespace
}  // namespace sf
