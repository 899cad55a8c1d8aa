// sf_rotary.cu -- rotary positions, and keys and values written into the pages of an e4m3 cache.
//
//   pair (a, b) of a head at position p:  (a cos - b sin, a sin + b cos), cos and sin from a table's row p
//   page and kv head:  scale = 2^e, the least e with max|value| <= 448 * 2^e;  code = e4m3(value / scale)
//
// A power of two makes value / scale and the rewriting of a page's older codes for a larger scale exact (but where a
// code becomes subnormal), and costs a floating-point code no precision.
#include <atomic>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_q4_internal.h"
#include "sf_paged.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_rotary)
extern std::atomic<long long> g_launches;

namespace {

struct Turn {
  const float* table;   // [max_pos, rot]: cosines, then sines; NULL: nothing is turned (rot = 0)
  int max_pos, rot, interleaved;
};

struct Rows {
  const void* p;
  long long ts, hs;     // token and head strides
};

// One head's D elements are cut into items: a turned one (8 pairs, or with VEC = false one pair) or a copied one
// (8 elements, or one).  VEC needs every stride and offset it meets to be a multiple of 8 elements.
template <bool VEC>
__device__ __forceinline__ int turned_items(const Turn& t) {
  return VEC ? (t.interleaved ? t.rot / 8 : t.rot / 16) : t.rot / 2;
}
template <bool VEC>
__device__ __forceinline__ int head_items(const Turn& t, int D) {
  return turned_items<VEC>(t) + (D - t.rot) / (VEC ? 8 : 1);
}

template <bool VEC>
struct Piece {
  static constexpr int W = VEC ? 8 : 1;
  int da, db;           // first element of a; of b, or -1 when there is none
  float a[W], b[W];
};

template <typename TX, bool VEC>
__device__ __forceinline__ void load_w(const TX* p, float (&v)[Piece<VEC>::W]) {
  if constexpr (VEC) load8(p, v);
  else v[0] = to_f32(*p);
}

// `trow` is the table's row of the token's position.
template <typename TX, bool VEC>
__device__ __forceinline__ void turn_item(const TX* x, int item, const Turn& t, const float* trow, bool pos_ok,
                                          Piece<VEC>& p) {
  constexpr int W = Piece<VEC>::W;
  const int nt = turned_items<VEC>(t), half = t.rot / 2;
  p.db = -1;
  if (item >= nt) {
    p.da = t.rot + (item - nt) * W;
    load_w<TX, VEC>(x + p.da, p.a);
    return;
  }
  const float nan = __int_as_float(0x7fffffff);
  if (VEC && t.interleaved) {
    p.da = 8 * item;
    load_w<TX, VEC>(x + p.da, p.a);
#pragma unroll
    for (int i = 0; i < W / 2; ++i) {
      const float c = pos_ok ? trow[4 * item + i] : nan, s = pos_ok ? trow[half + 4 * item + i] : nan;
      const float a = p.a[2 * i], b = p.a[2 * i + 1];
      p.a[2 * i] = a * c - b * s;
      p.a[2 * i + 1] = a * s + b * c;
    }
    return;
  }
  p.da = t.interleaved ? 2 * item : W * item;
  p.db = t.interleaved ? 2 * item + 1 : half + W * item;
  load_w<TX, VEC>(x + p.da, p.a);
  load_w<TX, VEC>(x + p.db, p.b);
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float c = pos_ok ? trow[W * item + i] : nan, s = pos_ok ? trow[half + W * item + i] : nan;
    const float a = p.a[i], b = p.b[i];
    p.a[i] = a * c - b * s;
    p.b[i] = a * s + b * c;
  }
}

template <typename TX, bool VEC>
__device__ __forceinline__ void store_w(TX* p, const float (&v)[Piece<VEC>::W]) {
  if constexpr (VEC) store8(p, v);
  else *p = from_f32<TX>(v[0]);
}

template <typename TX, bool VEC>
__device__ __forceinline__ void turn_token(const TX* x, long long xhs, TX* out, long long ohs, int H, int D,
                                           const Turn& t, long long pos) {
  const bool ok = t.rot == 0 || (pos >= 0 && pos < t.max_pos);
  if (!ok && threadIdx.x == 0) atomicOr(&g_dev_error, kErrIndex);
  const float* trow = t.table + (ok ? pos * t.rot : 0);
  const int per = head_items<VEC>(t, D);
  for (int i = threadIdx.x; i < H * per; i += blockDim.x) {
    const int h = i / per;
    Piece<VEC> p;
    turn_item<TX, VEC>(x + h * xhs, i % per, t, trow, ok, p);
    store_w<TX, VEC>(out + h * ohs + p.da, p.a);
    if (p.db >= 0) store_w<TX, VEC>(out + h * ohs + p.db, p.b);
  }
}

template <typename TX, bool VEC>
__global__ void __launch_bounds__(256) rotary_kernel(const Rows x, void* out, long long ots, long long ohs,
                                                     const void* positions, int pos64, const Turn t, int H, int D) {
  const size_t tok = blockIdx.x;
  const long long pos = pos64 ? static_cast<const long long*>(positions)[tok] : static_cast<const int*>(positions)[tok];
  turn_token<TX, VEC>(static_cast<const TX*>(x.p) + tok * x.ts, x.hs, static_cast<TX*>(out) + tok * ots, ohs, H, D, t,
                      pos);
}

struct AppendArgs {
  sf_paged_cache c;
  Rows k, v, q;
  void* q_out;
  Turn turn;
  int H, T, units;      // units: an upper bound of the pages that the call touches
};

// One warp writes one (page, kv head, keys or values): first the largest magnitude of its new rows, then the codes.
template <typename TX, bool VEC>
__device__ void append_unit(const AppendArgs& a, int unit, int h, int which) {
  const int lane = threadIdx.x & 31, D = a.c.head_dim, BS = a.c.page_size;
  const SeqSpan s = unit_span(a.c, a.T, unit);
  if (!s.ok) {
    if (lane == 0) atomicOr(&g_dev_error, kErrIndex);
    return;
  }
  if (s.lo >= s.hi) return;
  const int page = s.page < a.c.pages_per_seq ? a.c.block_table[(size_t)s.b * a.c.pages_per_seq + s.page] : -1;
  if (page < 0 || page >= a.c.num_pages) {
    if (lane == 0) atomicOr(&g_dev_error, kErrIndex);
    return;
  }
  const Rows& src = which ? a.v : a.k;
  Turn t = a.turn;
  if (which) t.rot = 0;
  uint8_t* codes = (which ? a.c.v_codes : a.c.k_codes) + ((size_t)page * a.c.n_kv_heads + h) * BS * D;
  float* scale_at = (which ? a.c.v_scales : a.c.k_scales) + (size_t)page * a.c.n_kv_heads + h;
  const TX* x0 = static_cast<const TX*>(src.p) + (size_t)(s.row + s.lo) * src.ts + h * src.hs;
  const int slot0 = s.lo - s.page * BS, rows = s.hi - s.lo, per = head_items<VEC>(t, D);
  const bool turned = t.rot > 0;
  auto each = [&](auto&& fn) {
    for (int i = lane; i < rows * per; i += 32) {
      const int r = i / per, pos = s.lo + r;
      const bool ok = !turned || pos < t.max_pos;
      Piece<VEC> p;
      turn_item<TX, VEC>(x0 + r * src.ts, i % per, t, t.table + (turned && ok ? (size_t)pos * t.rot : 0), ok, p);
      fn(r, p);
    }
  };
  if (turned && s.hi > t.max_pos && lane == 0) atomicOr(&g_dev_error, kErrIndex);
  uint32_t top = 0;   // bits of the largest finite magnitude
  auto see = [&](float v) {
    const uint32_t u = __float_as_uint(v) & 0x7fffffffu;
    if (u < 0x7f800000u) top = max(top, u);
  };
  each([&](int, const Piece<VEC>& p) {
#pragma unroll
    for (int i = 0; i < Piece<VEC>::W; ++i) {
      see(p.a[i]);
      if (p.db >= 0) see(p.b[i]);
    }
  });
  top = __reduce_max_sync(0xffffffffu, top);
  int e = (int)(top >> 23) - 127 - ((top & 0x7fffffu) <= 0x600000u ? 8 : 7);   // 448 = 1.75 * 2^8
  if (e < -64) e = -64;
  float scale = __int_as_float((e + 127) << 23);
  if (slot0 > 0) {
    const float old = *scale_at;
    if (old >= scale) {
      scale = old;
    } else {
      const float ratio = old / scale;
      for (int i = lane; i < slot0 * D / 16; i += 32) {
        uint4 u = reinterpret_cast<uint4*>(codes)[i];
        uint8_t* c = reinterpret_cast<uint8_t*>(&u);
#pragma unroll
        for (int j = 0; j < 16; ++j) c[j] = to_e4m3(from_e4m3(c[j]) * ratio);
        reinterpret_cast<uint4*>(codes)[i] = u;
      }
    }
  }
  const float inv = 1.f / scale;
  auto put = [&](int r, int d, const float (&v)[Piece<VEC>::W]) {
    uint8_t* o = codes + (size_t)(slot0 + r) * D + d;
    if constexpr (VEC) {
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) w[i] = v[i] * inv;
      *reinterpret_cast<uint2*>(o) = to_e4m3x8(w);
    } else {
      *o = to_e4m3(v[0] * inv);
    }
  };
  each([&](int r, const Piece<VEC>& p) {
    put(r, p.da, p.a);
    if (p.db >= 0) put(r, p.db, p.b);
  });
  __syncwarp();
  if (lane == 0) *scale_at = scale;
}

// The first blocks turn one query token each; each warp of the others writes one (page, kv head, keys or values).
template <typename TX, bool VEC>
__global__ void __launch_bounds__(256) paged_append_kernel(const AppendArgs a, int q_blocks) {
  if ((int)blockIdx.x < q_blocks) {
    const int tok = blockIdx.x;
    const TokenAt at = token_at(a.c, a.T, tok);
    if (!at.ok && threadIdx.x == 0) atomicOr(&g_dev_error, kErrIndex);
    turn_token<TX, VEC>(static_cast<const TX*>(a.q.p) + tok * a.q.ts, a.q.hs,
                        static_cast<TX*>(a.q_out) + (size_t)tok * a.H * a.c.head_dim, a.c.head_dim, a.H, a.c.head_dim,
                        a.turn, at.ok ? max(at.pos, 0) : -1);
    return;
  }
  const long long w = (long long)(blockIdx.x - q_blocks) * 8 + (threadIdx.x >> 5);
  const long long heads = w >> 1;
  if (heads >= (long long)a.units * a.c.n_kv_heads) return;
  append_unit<TX, VEC>(a, (int)(heads / a.c.n_kv_heads), (int)(heads % a.c.n_kv_heads), (int)(w & 1));
}

bool rows_vec(const void* p, long long ts, long long hs, int dtype) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ts % 8 == 0 && hs % 8 == 0;
}
bool turn_vec(int rot, int interleaved, int D) {
  return D % 8 == 0 && rot % (interleaved ? 8 : 16) == 0;
}

int check_turn(const float* table, int max_pos, int rot, int D) {
  if (rot < 0 || rot % 2 || rot > D) return fail(SF_ERR_SHAPE, "rot must be even and at most head_dim");
  if (rot > 0 && (!table || max_pos < 1)) return fail(SF_ERR_SHAPE, "the rotary table is missing or empty");
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

int sf_rotary(const void* x, int dtype, long long xts, long long xhs, void* out, long long ots, long long ohs,
              const void* positions, int pos64, const float* table, int max_pos, int rot, int interleaved, int T, int H,
              int D, void* stream) {
  if (T < 0 || H < 0 || D < 1) return fail(SF_ERR_SHAPE, "need T, H >= 0 and head_dim >= 1");
  if (dtype < 0 || dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (int rc = check_turn(table, max_pos, rot, D)) return rc;
  if (T == 0 || H == 0) return SF_OK;
  if (!x || !out || !positions) return fail(SF_ERR_NULL, "null pointer argument");
  const Turn t{table, max_pos, rot, interleaved};
  const bool vec = turn_vec(rot, interleaved, D) && rows_vec(x, xts, xhs, dtype) && rows_vec(out, ots, ohs, dtype);
  const Rows rows{x, xts, xhs};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto* fn = vec ? rotary_kernel<TX, true> : rotary_kernel<TX, false>;
    fn<<<(unsigned)T, 256, 0, st>>>(rows, out, ots, ohs, positions, pos64, t, H, D);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return cuda_fail(e, "rotary_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

int sf_paged_append(const sf_paged_cache* cache, const void* k, long long kts, long long khs, const void* v,
                    long long vts, long long vhs, const void* q, long long qts, long long qhs, void* q_out, int dtype,
                    int H, int T, const float* table, int max_pos, int rot, int interleaved, void* stream) {
  if (int rc = check_paged(cache, T)) return rc;
  if (dtype < 0 || dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (T == 0) return SF_OK;
  if (!k || !v || (q && !q_out)) return fail(SF_ERR_NULL, "null pointer argument");
  if (q && H < 1) return fail(SF_ERR_SHAPE, "need H >= 1 query heads");
  const int D = cache->head_dim;
  if (table) {
    if (int rc = check_turn(table, max_pos, rot, D)) return rc;
  } else {
    rot = 0;
  }
  AppendArgs a{};
  a.c = *cache;
  a.k = Rows{k, kts, khs};
  a.v = Rows{v, vts, vhs};
  a.q = Rows{q, qts, qhs};
  a.q_out = q_out;
  a.turn = Turn{table, max_pos, rot, interleaved};
  a.H = H;
  a.T = T;
  a.units = max_units(*cache, T);
  const bool vec = turn_vec(rot, interleaved, D) && rows_vec(k, kts, khs, dtype) && rows_vec(v, vts, vhs, dtype) &&
                   (!q || (rows_vec(q, qts, qhs, dtype) && rows_vec(q_out, D, D, dtype)));
  const int q_blocks = q ? T : 0;
  const long long warps = 2ll * a.units * cache->n_kv_heads;
  const long long blocks = q_blocks + (warps + 7) / 8;
  if (blocks > 0x7fffffffll) return fail(SF_ERR_UNSUPPORTED, "too many tokens in one call");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto* fn = vec ? paged_append_kernel<TX, true> : paged_append_kernel<TX, false>;
    fn<<<(unsigned)blocks, 256, 0, st>>>(a, q_blocks);
    return cudaGetLastError();
  });
  if (e != cudaSuccess) return cuda_fail(e, "paged_append_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

}  // extern "C"
