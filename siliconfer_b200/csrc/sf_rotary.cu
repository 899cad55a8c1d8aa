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

// One head's D elements are cut into items of 16 elements (VEC: two runs of 8) or 2: the pairs of a turned item, or
// what is copied beyond them.  VEC needs every stride and offset it meets to be a multiple of 8 elements.
template <bool VEC>
__device__ __forceinline__ int turned_items(const Turn& t) {
  return t.rot / (VEC ? 16 : 2);
}
template <bool VEC>
__device__ __forceinline__ int head_items(const Turn& t, int D) {
  return turned_items<VEC>(t) + (D - t.rot + (VEC ? 15 : 1)) / (VEC ? 16 : 2);
}

template <bool VEC>
struct Piece {
  static constexpr int W = VEC ? 8 : 1;
  int da, db;           // first element of a; of b, or -1 where the head ends before it
  float a[W], b[W];
};

template <typename TX, bool VEC>
__device__ __forceinline__ void load_w(const TX* p, float (&v)[Piece<VEC>::W]) {
  if constexpr (VEC) load8(p, v);
  else v[0] = to_f32(*p);
}

// Cosines and sines of an item's pairs, from the table's row of the token's position (NaN without one).
template <bool VEC>
struct Angles {
  static constexpr int W = Piece<VEC>::W;
  float c[W], s[W];
};
template <bool VEC>
__device__ __forceinline__ void load_angles(const Turn& t, int item, const float* trow, bool ok, Angles<VEC>& a) {
  constexpr int W = Piece<VEC>::W;
  if (item >= turned_items<VEC>(t)) return;
  if (!ok) {
#pragma unroll
    for (int i = 0; i < W; ++i) a.c[i] = a.s[i] = __int_as_float(0x7fffffff);
    return;
  }
  const int half = t.rot / 2;
  if constexpr (VEC) {
#pragma unroll
    for (int i = 0; i < 8; i += 4) {
      *reinterpret_cast<float4*>(a.c + i) = __ldg(reinterpret_cast<const float4*>(trow + 8 * item + i));
      *reinterpret_cast<float4*>(a.s + i) = __ldg(reinterpret_cast<const float4*>(trow + half + 8 * item + i));
    }
  } else {
    a.c[0] = __ldg(trow + item);
    a.s[0] = __ldg(trow + half + item);
  }
}

template <typename TX, bool VEC>
__device__ __forceinline__ void load_item(const TX* x, int item, const Turn& t, int D, Piece<VEC>& p) {
  constexpr int W = Piece<VEC>::W;
  const int nt = turned_items<VEC>(t);
  if (item < nt && !t.interleaved) {
    p.da = W * item;
    p.db = t.rot / 2 + W * item;
  } else {
    p.da = item < nt ? 2 * W * item : t.rot + (item - nt) * 2 * W;
    p.db = p.da + W < D ? p.da + W : -1;
  }
  load_w<TX, VEC>(x + p.da, p.a);
  if (p.db >= 0) load_w<TX, VEC>(x + p.db, p.b);
}
template <bool VEC>
__device__ __forceinline__ void turn_item(Piece<VEC>& p, int item, const Turn& t, const Angles<VEC>& w) {
  if (item >= turned_items<VEC>(t)) return;
  if (VEC && t.interleaved) {   // pairs side by side: four in a, four in b
#pragma unroll
    for (int i = 0; i < Piece<VEC>::W / 2; ++i) {
      const float a = p.a[2 * i], b = p.a[2 * i + 1], c = p.b[2 * i], d = p.b[2 * i + 1];
      constexpr int H = Piece<VEC>::W / 2;
      p.a[2 * i] = a * w.c[i] - b * w.s[i];
      p.a[2 * i + 1] = a * w.s[i] + b * w.c[i];
      p.b[2 * i] = c * w.c[H + i] - d * w.s[H + i];
      p.b[2 * i + 1] = c * w.s[H + i] + d * w.c[H + i];
    }
  } else {
#pragma unroll
    for (int i = 0; i < Piece<VEC>::W; ++i) {
      const float a = p.a[i], b = p.b[i];
      p.a[i] = a * w.c[i] - b * w.s[i];
      p.b[i] = a * w.s[i] + b * w.c[i];
    }
  }
}

template <typename TX, bool VEC>
__device__ __forceinline__ void store_w(TX* p, const float (&v)[Piece<VEC>::W]) {
  if constexpr (VEC) store8(p, v);
  else *p = from_f32<TX>(v[0]);
}

template <typename TX, bool VEC, typename Position>
__device__ __forceinline__ void turn_token(const TX* x, long long xhs, TX* out, long long ohs, int H, int D,
                                           const Turn& t, Position&& position) {
  // A thread takes one item of every (blockDim / per)-th head, two heads at a time: their elements are asked for first,
  // the angles, which hang on the position, once.
  const int per = head_items<VEC>(t, D), lanes = per < (int)blockDim.x ? (int)blockDim.x / per * per : (int)blockDim.x;
  const int heads = per < (int)blockDim.x ? lanes / per : 1, h0 = per < (int)blockDim.x ? (int)threadIdx.x / per : 0;
  for (int item = threadIdx.x % per; item < per; item += blockDim.x) {
    Angles<VEC> w;
    bool ok = true, first = true;
    for (int h = h0; h < H || first; h += 2 * heads) {
      Piece<VEC> p[2];
      const bool in0 = h < H && (int)threadIdx.x < lanes, in1 = h + heads < H && (int)threadIdx.x < lanes;
      if (in0) load_item<TX, VEC>(x + h * xhs, item, t, D, p[0]);
      if (in1) load_item<TX, VEC>(x + (h + heads) * xhs, item, t, D, p[1]);
      if (first) {
        const long long pos = position();   // by whole warps
        ok = t.rot == 0 || (pos >= 0 && pos < t.max_pos);
        if (!ok && threadIdx.x == 0) atomicOr(&g_dev_error, kErrIndex);
        load_angles<VEC>(t, item, t.table + (ok ? pos * t.rot : 0), ok, w);
        first = false;
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if (!(i ? in1 : in0)) continue;
        turn_item<VEC>(p[i], item, t, w);
        TX* o = out + (h + i * heads) * ohs;
        store_w<TX, VEC>(o + p[i].da, p[i].a);
        if (p[i].db >= 0) store_w<TX, VEC>(o + p[i].db, p[i].b);
      }
    }
  }
}

template <typename TX, bool VEC>
__global__ void __launch_bounds__(256) rotary_kernel(const Rows x, void* out, long long ots, long long ohs,
                                                     const void* positions, int pos64, const Turn t, int H, int D) {
  griddep_launch_dependents();
  griddep_wait();
  const size_t tok = blockIdx.x;
  turn_token<TX, VEC>(static_cast<const TX*>(x.p) + tok * x.ts, x.hs, static_cast<TX*>(out) + tok * ots, ohs, H, D, t, [&] {
    return pos64 ? static_cast<const long long*>(positions)[tok] : (long long)static_cast<const int*>(positions)[tok];
  });
}

struct AppendArgs {
  sf_paged_cache c;
  Rows k, v, q;
  void* q_out;
  Turn turn;
  int H, T, units;      // units: an upper bound of the pages that the call touches
};

// WARPS warps write one (page, kv head, keys or values): the largest magnitude of its new rows, then the codes.  A
// thread keeps what it loaded where it has at most KEEP items, else it loads them again.
template <typename TX, bool VEC, int WARPS>
__device__ void append_unit(const AppendArgs& a, int unit, int h, int which, uint32_t* red) {
  constexpr int KEEP = 2, THREADS = 32 * WARPS;
  const int tid = threadIdx.x % THREADS, lane = threadIdx.x & 31, D = a.c.head_dim, BS = a.c.page_size;
  const SeqSpan s = unit_span(a.c, a.T, unit);
  if (!s.ok) {
    if (tid == 0) atomicOr(&g_dev_error, kErrIndex);
    return;
  }
  if (s.lo >= s.hi) return;
  const int page = s.page < a.c.pages_per_seq ? a.c.block_table[(size_t)s.b * a.c.pages_per_seq + s.page] : -1;
  if (page < 0 || page >= a.c.num_pages) {
    if (tid == 0) atomicOr(&g_dev_error, kErrIndex);
    return;
  }
  const Rows& src = which ? a.v : a.k;
  Turn t = a.turn;
  if (which) t.rot = 0;
  uint8_t* codes = (which ? a.c.v_codes : a.c.k_codes) + ((size_t)page * a.c.n_kv_heads + h) * BS * D;
  float* scale_at = (which ? a.c.v_scales : a.c.k_scales) + (size_t)page * a.c.n_kv_heads + h;
  const TX* x0 = static_cast<const TX*>(src.p) + (size_t)(s.row + s.lo) * src.ts + h * src.hs;
  const int slot0 = s.lo - s.page * BS, per = head_items<VEC>(t, D), items = (s.hi - s.lo) * per;
  const bool turned = t.rot > 0;
  const float old = slot0 > 0 ? *scale_at : 0.f;
  const auto load = [&](int i, Piece<VEC>& p) {
    const int r = i / per, item = i % per, pos = s.lo + r;
    const bool ok = !turned || pos < t.max_pos;
    Angles<VEC> w;
    load_angles<VEC>(t, item, t.table + (turned && ok ? (size_t)pos * t.rot : 0), ok, w);
    load_item<TX, VEC>(x0 + r * src.ts, item, t, D, p);
    turn_item<VEC>(p, item, t, w);
  };
  if (turned && s.hi > t.max_pos && tid == 0) atomicOr(&g_dev_error, kErrIndex);
  uint32_t top = 0;   // bits of the largest finite magnitude
  const auto see = [&](const Piece<VEC>& p) {
#pragma unroll
    for (int i = 0; i < Piece<VEC>::W; ++i) {
      const uint32_t u = __float_as_uint(p.a[i]) & 0x7fffffffu, v = p.db >= 0 ? __float_as_uint(p.b[i]) & 0x7fffffffu : 0u;
      if (u < 0x7f800000u) top = max(top, u);
      if (v < 0x7f800000u) top = max(top, v);
    }
  };
  Piece<VEC> kept[KEEP];
  const bool keep = items <= KEEP * THREADS;
  if (keep) {
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (tid + c * THREADS < items) load(tid + c * THREADS, kept[c]);
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (tid + c * THREADS < items) see(kept[c]);
  } else {
#pragma unroll 2
    for (int i = tid; i < items; i += THREADS) {
      Piece<VEC> p;
      load(i, p);
      see(p);
    }
  }
  top = __reduce_max_sync(0xffffffffu, top);
  if constexpr (WARPS > 1) {
    if (lane == 0) red[threadIdx.x >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = max(top, red[w]);
  }
  int e = (int)(top >> 23) - 127 - ((top & 0x7fffffu) <= 0x600000u ? 8 : 7);   // 448 = 1.75 * 2^8
  if (e < -64) e = -64;
  float scale = __int_as_float((e + 127) << 23);
  if (old >= scale) {
    scale = old;
  } else if (slot0 > 0) {
    const float ratio = old / scale;
    for (int i = tid; i < slot0 * D / 16; i += THREADS) {
      uint4 u = reinterpret_cast<uint4*>(codes)[i];
      uint8_t* c = reinterpret_cast<uint8_t*>(&u);
#pragma unroll
      for (int j = 0; j < 16; ++j) c[j] = to_e4m3(from_e4m3(c[j]) * ratio);
      reinterpret_cast<uint4*>(codes)[i] = u;
    }
  }
  const float inv = 1.f / scale;
  const auto put = [&](int r, int d, const float (&v)[Piece<VEC>::W]) {
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
  const auto store = [&](int i, const Piece<VEC>& p) {
    put(i / per, p.da, p.a);
    if (p.db >= 0) put(i / per, p.db, p.b);
  };
  if (keep) {
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (tid + c * THREADS < items) store(tid + c * THREADS, kept[c]);
  } else {
#pragma unroll 2
    for (int i = tid; i < items; i += THREADS) {
      Piece<VEC> p;
      load(i, p);
      store(i, p);
    }
  }
  if (tid == 0) *scale_at = scale;   // every thread has read the old one: before the block's barrier, or in this warp
}

// The first blocks turn one query token each; of the others, 8 / WARPS units a block.
template <typename TX, bool VEC, int WARPS>
__global__ void __launch_bounds__(256, 3) paged_append_kernel(const AppendArgs a, int q_blocks) {
  __shared__ uint32_t red[8];
  griddep_launch_dependents();
  griddep_wait();
  if ((int)blockIdx.x < q_blocks) {
    const int tok = blockIdx.x;
    turn_token<TX, VEC>(static_cast<const TX*>(a.q.p) + tok * a.q.ts, a.q.hs,
                        static_cast<TX*>(a.q_out) + (size_t)tok * a.H * a.c.head_dim, a.c.head_dim, a.H, a.c.head_dim,
                        a.turn, [&] {
      const TokenAt at = token_at(a.c, a.T, tok);
      return at.ok ? (long long)max(at.pos, 0) : -1ll;
    });
    return;
  }
  const long long w = (long long)(blockIdx.x - q_blocks) * (8 / WARPS) + threadIdx.x / (32 * WARPS);
  const long long heads = w >> 1;
  if (heads >= (long long)a.units * a.c.n_kv_heads) return;
  append_unit<TX, VEC, WARPS>(a, (int)(heads / a.c.n_kv_heads), (int)(heads % a.c.n_kv_heads), (int)(w & 1), red);
}

bool rows_vec(const void* p, long long ts, long long hs) {
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && ts % 8 == 0 && hs % 8 == 0;
}
bool turn_vec(const float* table, int rot, int D) {
  return D % 8 == 0 && rot % 16 == 0 && reinterpret_cast<uintptr_t>(table) % 16 == 0;
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
  const bool vec = turn_vec(table, rot, D) && rows_vec(x, xts, xhs) && rows_vec(out, ots, ohs);
  const Rows rows{x, xts, xhs};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto* fn = vec ? rotary_kernel<TX, true> : rotary_kernel<TX, false>;
    return launch_kernel(fn, T, 256, 0, st, true, rows, out, ots, ohs, positions, pos64, t, H, D);
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
  const bool vec = turn_vec(table, rot, D) && rows_vec(k, kts, khs) && rows_vec(v, vts, vhs) &&
                   (!q || (rows_vec(q, qts, qhs) && rows_vec(q_out, D, D)));
  const int q_blocks = q ? T : 0;
  // a warp for the few rows of a decode step, a block for a page of a prompt
  const bool wide = T / cache->batch > 4;
  const long long work = 2ll * a.units * cache->n_kv_heads;
  const long long blocks = q_blocks + (wide ? work : (work + 7) / 8);
  if (blocks > 0x7fffffffll) return fail(SF_ERR_UNSUPPORTED, "too many tokens in one call");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto* fn = wide ? (vec ? paged_append_kernel<TX, true, 8> : paged_append_kernel<TX, false, 8>)
                    : (vec ? paged_append_kernel<TX, true, 1> : paged_append_kernel<TX, false, 1>);
    return launch_kernel(fn, (int)blocks, 256, 0, st, true, a, q_blocks);
  });
  if (e != cudaSuccess) return cuda_fail(e, "paged_append_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

}  // extern "C"
