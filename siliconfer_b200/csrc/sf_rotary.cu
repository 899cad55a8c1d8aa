// sf_rotary.cu -- rotary positions, and keys and values written into the pages of an e4m3 cache.
//
//   pair (a, b) of a head at position p:  (a cos - b sin, a sin + b cos), cos and sin from a table's row p
//   page and kv head:  scale = 2^e, the least e with max|value| <= 448 * 2^e;  code = e4m3(value / scale)
//
// A power of two makes value / scale and the rewriting of a page's older codes for a larger scale exact (but where a
// code becomes subnormal), and costs a floating-point code no precision.
//
// Every element is read and written once, and a page's rows wait in registers for the page's largest value.  A decode
// step (8 tokens, 32 heads) takes 3.8 us, most of it the launch.  4096 tokens with 64 query and 8 kv heads of 128 take
// 43.7 us, 3.7 TB/s: queries pass at the memory's rate, the pages' part is held by its instructions (a maximum, a turn,
// a conversion for each element), so it runs first.  With a division for every item instead of a fixed item for a
// thread, that call took 49 us.
#include <atomic>
#include <cstdint>
#include <type_traits>

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

// One head's D elements are cut into items of 8 elements (VEC: two runs of 4) or 2: the pairs of a turned item, or what
// is copied beyond them.  VEC needs every stride and offset it meets to be a multiple of 4 elements.  Runs of 8 need
// twice the registers for as many bytes under way, which spilled.
template <bool VEC>
__host__ __device__ __forceinline__ int turned_items(const Turn& t) {
  return t.rot / (VEC ? 8 : 2);
}
template <bool VEC>
__host__ __device__ __forceinline__ int head_items(const Turn& t, int D) {
  return turned_items<VEC>(t) + (D - t.rot + (VEC ? 7 : 1)) / (VEC ? 8 : 2);
}

template <bool VEC>
struct Piece {
  static constexpr int W = VEC ? 4 : 1;
  float a[W], b[W];
};

// An item as it was loaded: half the registers of its fp32 form for the 16-bit types, so more can be under way.
template <typename TX, bool VEC>
struct Raw {
  using Word = std::conditional_t<VEC, std::conditional_t<sizeof(TX) == 2, uint2, float4>, TX>;
  Word a, b;
};
struct Place {
  int da, db;           // first element of a; of b, or -1 where the head ends before it
};
template <bool VEC>
__device__ __forceinline__ Place place_of(int item, const Turn& t, int D) {
  constexpr int W = Piece<VEC>::W;
  const int nt = turned_items<VEC>(t);
  if (item < nt && !t.interleaved) return {W * item, t.rot / 2 + W * item};
  const int da = item < nt ? 2 * W * item : t.rot + (item - nt) * 2 * W;
  return {da, da + W < D ? da + W : -1};
}
template <typename TX, bool VEC>
__device__ __forceinline__ void load_item(const TX* x, const Place& at, Raw<TX, VEC>& r) {
  using Word = typename Raw<TX, VEC>::Word;
  r.a = *reinterpret_cast<const Word*>(x + at.da);
  if (at.db >= 0) r.b = *reinterpret_cast<const Word*>(x + at.db);
}
__device__ __forceinline__ void widen1(float4 u, float (&v)[4], const float*) { v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w; }
__device__ __forceinline__ void widen1(uint2 u, float (&v)[4], const __nv_bfloat16*) {
  v[0] = __uint_as_float(u.x << 16), v[1] = __uint_as_float(u.x & 0xffff0000u);
  v[2] = __uint_as_float(u.y << 16), v[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void widen1(uint2 u, float (&v)[4], const __half*) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u.x)), g = __half22float2(*reinterpret_cast<const __half2*>(&u.y));
  v[0] = f.x, v[1] = f.y, v[2] = g.x, v[3] = g.y;
}
template <typename TX>
__device__ __forceinline__ void widen1(TX u, float (&v)[1], const TX*) { v[0] = to_f32(u); }
template <typename TX, bool VEC>
__device__ __forceinline__ void widen(const Raw<TX, VEC>& r, Piece<VEC>& p) {
  widen1(r.a, p.a, static_cast<const TX*>(nullptr));
  widen1(r.b, p.b, static_cast<const TX*>(nullptr));
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
    const float4 c = __ldg(reinterpret_cast<const float4*>(trow + 4 * item));
    const float4 s = __ldg(reinterpret_cast<const float4*>(trow + half + 4 * item));
    a.c[0] = c.x, a.c[1] = c.y, a.c[2] = c.z, a.c[3] = c.w;
    a.s[0] = s.x, a.s[1] = s.y, a.s[2] = s.z, a.s[3] = s.w;
  } else {
    a.c[0] = __ldg(trow + item);
    a.s[0] = __ldg(trow + half + item);
  }
}

// A sum that is to be rounded again, to a code of 4 bits (a power of two from it): where fp32 leaves it within 16 last
// places of a tie between two codes, it is the sum in fp64, where both products are exact, cut to fp32 with its last bit
// set if anything was cut, which lies on the same side of the tie.  Of 25 million turned keys 34 codes were one step off
// without this, and the largest of them decide a page's error.  (Below 2^-6 of a code the ties lie elsewhere; those
// codes' steps are 2^-9.)
__device__ __forceinline__ float before_code(float y, float a, float c, float b, float s) {
  if (((__float_as_uint(y) + 0x80010u) & 0xfffffu) > 32u) return y;
  const double v = fma((double)a, (double)c, (double)b * (double)s);
  const float r = __double2float_rz(v);
  return (double)r == v ? r : __uint_as_float(__float_as_uint(r) | 1u);
}
// (a, b) <- (a c - b s, a s + b c)
template <bool CODE>
__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
  float ya = __fmaf_rn(a, c, -__fmul_rn(b, s)), yb = __fmaf_rn(b, c, __fmul_rn(a, s));
  if constexpr (CODE) {
    ya = before_code(ya, a, c, -b, s);
    yb = before_code(yb, b, c, a, s);
  }
  a = ya;
  b = yb;
}
template <bool VEC, bool CODE>
__device__ __forceinline__ void turn_item(Piece<VEC>& p, int item, const Turn& t, const Angles<VEC>& w) {
  if (item >= turned_items<VEC>(t)) return;
  if (VEC && t.interleaved) {   // pairs side by side: two in a, two in b
    constexpr int H = Piece<VEC>::W / 2;
#pragma unroll
    for (int i = 0; i < H; ++i) {
      turn<CODE>(p.a[2 * i], p.a[2 * i + 1], w.c[i], w.s[i]);
      turn<CODE>(p.b[2 * i], p.b[2 * i + 1], w.c[H + i], w.s[H + i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < Piece<VEC>::W; ++i) turn<CODE>(p.a[i], p.b[i], w.c[i], w.s[i]);
  }
}

__device__ __forceinline__ void store_w(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store_w(__half* p, const float (&v)[4]) {
  const __half2 a = __floats2half2_rn(v[0], v[1]), b = __floats2half2_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
__device__ __forceinline__ void store_w(__nv_bfloat16* p, const float (&v)[4]) {
  const __nv_bfloat162 a = __floats2bfloat162_rn(v[0], v[1]), b = __floats2bfloat162_rn(v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
}
template <typename TX>
__device__ __forceinline__ void store_w(TX* p, const float (&v)[1]) { *p = from_f32<TX>(v[0]); }

// Items under way in a thread.
template <typename TX>
constexpr int kAtOnce = sizeof(TX) == 2 ? 4 : 2;

// Threads that turn one token: enough for kAtOnce items each, and where the tokens are too few to fill the GPU, a block.
template <typename TX>
int token_threads(int T, int H, int per) {
  int n = 256;
  while (n > 32 && (long long)H * per * 2 <= (long long)n * kAtOnce<TX> && (long long)T * n > 1024ll * device_info().sms) n /= 2;
  return n;
}

template <typename TX, bool VEC, typename Position>
__device__ __forceinline__ void turn_token(int tid, int threads, const TX* x, long long xhs, TX* out, long long ohs, int H,
                                           int D, const Turn& t, Position&& position) {
  // A thread takes one item of every (threads / per)-th head, some heads at a time: their elements are asked for first,
  // the angles, which hang on the position, once.  The position is found in the first pass of both loops, the only one
  // that every lane of a warp makes.
  constexpr int M = kAtOnce<TX>;
  const int per = head_items<VEC>(t, D), heads = per < threads ? threads / per : 1, lanes = per < threads ? heads * per : threads;
  const int h0 = per < threads ? tid / per : 0;
  long long pos = 0;
  bool known = false, ok = true;
  for (int item = per < threads ? tid - h0 * per : tid; item < per; item += threads) {
    const Place at = place_of<VEC>(item, t, D);
    Angles<VEC> w;
    bool first = true;
    for (int h = h0; h < H || first; h += M * heads) {
      Raw<TX, VEC> raw[M];
#pragma unroll
      for (int i = 0; i < M; ++i)
        if (h + i * heads < H && tid < lanes) load_item<TX, VEC>(x + (h + i * heads) * xhs, at, raw[i]);
      if (!known) {
        known = true;
        pos = position();   // by whole warps
        ok = t.rot == 0 || (pos >= 0 && pos < t.max_pos);
        if (!ok && tid == 0) atomicOr(&g_dev_error, kErrIndex);
      }
      if (first) {
        load_angles<VEC>(t, item, t.table + (ok ? pos * t.rot : 0), ok, w);
        first = false;
      }
#pragma unroll
      for (int i = 0; i < M; ++i) {
        if (h + i * heads >= H || tid >= lanes) continue;
        Piece<VEC> p;
        widen<TX, VEC>(raw[i], p);
        turn_item<VEC, false>(p, item, t, w);
        TX* o = out + (h + i * heads) * ohs;
        store_w(o + at.da, p.a);
        if (at.db >= 0) store_w(o + at.db, p.b);
      }
    }
  }
}

template <typename TX, bool VEC>
__global__ void __launch_bounds__(256, 4) rotary_kernel(const Rows x, void* out, long long ots, long long ohs,
                                                        const void* positions, int pos64, const Turn t, int T, int H, int D,
                                                        int threads) {
  griddep_launch_dependents();
  griddep_wait();
  const int each = 256 / threads, tok = blockIdx.x * each + threadIdx.x / threads;
  if (tok >= T) return;
  turn_token<TX, VEC>(threadIdx.x % threads, threads, static_cast<const TX*>(x.p) + (size_t)tok * x.ts, x.hs,
                      static_cast<TX*>(out) + (size_t)tok * ots, ohs, H, D, t, [&] {
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
// thread keeps its items where they are at most KEEP, else it loads and turns them again.
template <typename TX, bool VEC, int WARPS>
__device__ void append_unit(const AppendArgs& a, int unit, int h, int which, uint32_t* red) {
  constexpr int KEEP = WARPS > 1 ? 4 : 2, THREADS = 32 * WARPS;
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
  const int slot0 = s.lo - s.page * BS, rows = s.hi - s.lo, per = head_items<VEC>(t, D);
  const bool turned = t.rot > 0;
  const float old = slot0 > 0 ? *scale_at : 0.f;
  // a thread's item is the same in every row it takes (where a row has more items than there are threads, it takes
  // several of every row)
  const int step = per < THREADS ? THREADS / per : 1, lanes = per < THREADS ? step * per : THREADS;
  const int r0 = per < THREADS ? tid / per : 0, item0 = per < THREADS ? tid - r0 * per : tid;
  const int end = tid < lanes ? rows : 0;
  const auto load = [&](int r, const Place& at, Raw<TX, VEC>& raw) { load_item<TX, VEC>(x0 + r * src.ts, at, raw); };
  const auto turned_piece = [&](int r, int item, const Raw<TX, VEC>& raw, Piece<VEC>& p) {
    const int pos = s.lo + r;
    const bool ok = !turned || pos < t.max_pos;
    Angles<VEC> w;
    load_angles<VEC>(t, item, t.table + (turned && ok ? (size_t)pos * t.rot : 0), ok, w);
    widen<TX, VEC>(raw, p);
    turn_item<VEC, true>(p, item, t, w);
  };
  if (turned && s.hi > t.max_pos && tid == 0) atomicOr(&g_dev_error, kErrIndex);
  // The largest magnitude (the maximum passes NaN over); with FINITE, of the finite ones.
  float top = 0.f;
  const auto see = [&](const Place& at, const Piece<VEC>& p, bool finite) {
    constexpr int W = Piece<VEC>::W;
    const float inf = __int_as_float(0x7f800000);
#pragma unroll
    for (int e = 0; e < W; ++e) {
      const float u = fabsf(p.a[e]), v = at.db >= 0 ? fabsf(p.b[e]) : 0.f;
      top = finite ? fmaxf(top, fmaxf(u < inf ? u : 0.f, v < inf ? v : 0.f)) : fmaxf(top, fmaxf(u, v));
    }
  };
  // Calls fn(place, item, row, turned elements) for all of this thread's.
  const auto each = [&](auto&& fn) {
    for (int item = item0; item < per; item += THREADS) {
      const Place at = place_of<VEC>(item, t, D);
#pragma unroll 1
      for (int r = r0; r < end; r += step) {
        Raw<TX, VEC> raw;
        Piece<VEC> p;
        load(r, at, raw);
        turned_piece(r, item, raw, p);
        fn(at, r, p);
      }
    }
  };
  const bool keep = per <= THREADS && rows <= KEEP * step;
  const Place at0 = place_of<VEC>(item0, t, D);
  Piece<VEC> kept[KEEP];
  if (keep) {
    Raw<TX, VEC> raw[KEEP];
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (r0 + c * step < end) load(r0 + c * step, at0, raw[c]);
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (r0 + c * step < end) {
        turned_piece(r0 + c * step, item0, raw[c], kept[c]);
        see(at0, kept[c], false);
      }
  } else {
    each([&](const Place& at, int, const Piece<VEC>& p) { see(at, p, false); });
  }
  const auto join = [&] {
    uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
    if constexpr (WARPS > 1) {
      if (lane == 0) red[threadIdx.x >> 5] = bits;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < WARPS; ++w) bits = max(bits, red[w]);
    }
    return bits;
  };
  uint32_t bits = join();
  if (bits == 0x7f800000u) {   // an infinity, which saturates; the scale is the finite ones'
    if constexpr (WARPS > 1) __syncthreads();
    top = 0.f;
    each([&](const Place& at, int, const Piece<VEC>& p) { see(at, p, true); });
    bits = join();
  }
  int e = (int)(bits >> 23) - 127 - ((bits & 0x7fffffu) <= 0x600000u ? 8 : 7);   // 448 = 1.75 * 2^8
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
      *reinterpret_cast<uint32_t*>(o) = to_e4m3x2(v[0] * inv, v[1] * inv) | to_e4m3x2(v[2] * inv, v[3] * inv) << 16;
    } else {
      *o = to_e4m3(v[0] * inv);
    }
  };
  const auto store = [&](const Place& at, int r, const Piece<VEC>& p) {
    put(r, at.da, p.a);
    if (at.db >= 0) put(r, at.db, p.b);
  };
  if (keep) {
#pragma unroll
    for (int c = 0; c < KEEP; ++c)
      if (r0 + c * step < end) store(at0, r0 + c * step, kept[c]);
  } else {
    each(store);
  }
  if (tid == 0) *scale_at = scale;   // every thread has read the old one: before the block's barrier, or in this warp
}

// The first blocks write 8 / WARPS units each, which take longer; the others turn 256 / q_threads query tokens.
template <typename TX, bool VEC, int WARPS>
__global__ void __launch_bounds__(256, WARPS > 1 ? 4 : 3) paged_append_kernel(const AppendArgs a, int kv_blocks, int q_threads) {
  __shared__ uint32_t red[8];
  griddep_launch_dependents();
  griddep_wait();
  if ((int)blockIdx.x >= kv_blocks) {
    const int each = 256 / q_threads, tok = ((int)blockIdx.x - kv_blocks) * each + threadIdx.x / q_threads;
    if (tok >= a.T) return;
    turn_token<TX, VEC>(threadIdx.x % q_threads, q_threads, static_cast<const TX*>(a.q.p) + (size_t)tok * a.q.ts, a.q.hs,
                        static_cast<TX*>(a.q_out) + (size_t)tok * a.H * a.c.head_dim, a.c.head_dim, a.H, a.c.head_dim,
                        a.turn, [&] {
      const TokenAt at = token_at(a.c, a.T, tok);
      return at.ok ? (long long)max(at.pos, 0) : -1ll;
    });
    return;
  }
  const long long w = (long long)blockIdx.x * (8 / WARPS) + threadIdx.x / (32 * WARPS);
  const long long heads = w >> 1;
  if (heads >= (long long)a.units * a.c.n_kv_heads) return;
  append_unit<TX, VEC, WARPS>(a, (int)(heads / a.c.n_kv_heads), (int)(heads % a.c.n_kv_heads), (int)(w & 1), red);
}

bool rows_vec(const void* p, int dtype, long long ts, long long hs) {
  return reinterpret_cast<uintptr_t>(p) % (dtype == SF_F32 ? 16 : 8) == 0 && ts % 4 == 0 && hs % 4 == 0;
}
bool turn_vec(const float* table, int rot, int D) {
  return D % 8 == 0 && rot % 8 == 0 && reinterpret_cast<uintptr_t>(table) % 16 == 0;
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
  const bool vec = turn_vec(table, rot, D) && rows_vec(x, dtype, xts, xhs) && rows_vec(out, dtype, ots, ohs);
  const Rows rows{x, xts, xhs};
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto* fn = vec ? rotary_kernel<TX, true> : rotary_kernel<TX, false>;
    const int threads = token_threads<TX>(T, H, vec ? head_items<true>(t, D) : head_items<false>(t, D));
    return launch_kernel(fn, (T + 256 / threads - 1) / (256 / threads), 256, 0, st, true, rows, out, ots, ohs, positions,
                         pos64, t, T, H, D, threads);
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
  const bool vec = turn_vec(table, rot, D) && rows_vec(k, dtype, kts, khs) && rows_vec(v, dtype, vts, vhs) &&
                   (!q || (rows_vec(q, dtype, qts, qhs) && rows_vec(q_out, dtype, D, D)));
  // a warp for the few rows of a decode step, a block for a page of a prompt
  const bool wide = T / cache->batch > 4;
  const long long work = 2ll * a.units * cache->n_kv_heads, kv_blocks = wide ? work : (work + 7) / 8;
  if (kv_blocks + T > 0x7fffffffll) return fail(SF_ERR_UNSUPPORTED, "too many tokens in one call");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    auto* fn = wide ? (vec ? paged_append_kernel<TX, true, 8> : paged_append_kernel<TX, false, 8>)
                    : (vec ? paged_append_kernel<TX, true, 1> : paged_append_kernel<TX, false, 1>);
    const int threads = token_threads<TX>(T, H, vec ? head_items<true>(a.turn, D) : head_items<false>(a.turn, D));
    const int q_blocks = q ? (T + 256 / threads - 1) / (256 / threads) : 0;
    return launch_kernel(fn, (int)kv_blocks + q_blocks, 256, 0, st, true, a, (int)kv_blocks, threads);
  });
  if (e != cudaSuccess) return cuda_fail(e, "paged_append_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

}  // extern "C"
