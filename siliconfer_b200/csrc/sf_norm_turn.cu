// sf_norm_turn.cu -- norms and rotary positions of query and key heads, and keys and values into a 4-bit cache.
//
//   y = x / sqrt(mean(x^2) + eps) * weight        of a head's D elements
//   pair (a, b), pair number j:  (a cos - b sin, a sin + b cos), cos and sin from row positions[axes[j]] of a table
//   quarter c of a vector:  scale = bf16(max|y| / 7.5), at least 2^-126;  code = clamp(rint(y / scale), -8, 7) + 8
//
// A block takes one token and some of its heads: the angles, which hang on one or several positions, are brought to shared
// memory once.  A group of lanes takes a vector at a time, the next one's elements under way; a lane the same W places of
// all four quarters: these hold both elements of its rotary pairs, and the codes of a place are one 16-bit word.
//
// Measured in a graph: 4096 tokens, 64 query and 8 kv heads of 128, three axes, norms: turned 32 us (4.8 TB/s of the copy
// rate's 6.5), appended 40 us (3.9 TB/s); one token 2.6 us, 8 tokens of 32 heads appended 4.0.  No unit is full: a turn uses
// 66 % of the issue slots and 39 % of DRAM's time with 6.8 warps a scheduler, which wait for shared memory and shuffles (0.32
// of a warp's time between two instructions), for fixed latencies (0.17) and for each other's turn (0.16); an append 66 % and
// 33 %, fp64 units 6 %, conversions 19 %.  A warp takes up to 10 passes in turn (3: 39 us, 6: 33); keys are normed, turned
// and cut in fp64, which the 64-bit units do beside the rest, so that a code is the exact value's.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdint>
#include <initializer_list>
#include <type_traits>

#include "sf_e4m3.h"
#include "sf_paged4.h"
#include "sf_q4_internal.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_norm_turn)
extern std::atomic<long long> g_launches;

namespace {

constexpr int kRounds = 10, kThreads = 256, kMaxDim = 512, kMaxAxes = 8;

struct Vectors {
  const void* p;
  long long ts;         // token stride
  int hs;               // head stride
};
struct Out {
  void* p;
  long long ts;
  int hs;
};
enum Pairs { kNoPairs, kHalves, kHalvesOfHalf, kNeighbours, kAnyPairs };

struct HeadArgs {
  Vectors q, k, v;
  Out qo, ko;
  const void *wq, *wk;  // norm weights or NULL
  int w_dtype, norm;
  float eps, inv_d;     // 1 / D
  double inv_d64, eps64;
  const float* table;   // [max_pos, rot]: cosines, then sines
  int max_pos, rot, interleaved, pairs;
  const void* positions;   // [T, axes_n] or NULL: a token's place in its sequence
  int pos64, axes_n;
  const uint8_t* axes;  // [rot / 2] or NULL: all pairs belong to axis 0
  int H, Hkv, T, D;
  sf_paged_cache c;     // the cache's; without one, which rows are tokens where seq_lens is given
  __nv_bfloat16 *ks, *vs;
};

// W consecutive elements as they are loaded.
template <typename TX, int W>
struct Raw {
  static constexpr int BYTES = W * (int)sizeof(TX);
  using Word = std::conditional_t<BYTES == 16, uint4, std::conditional_t<BYTES == 8, uint2, std::conditional_t<BYTES == 4, uint32_t, uint16_t>>>;
  union {
    Word w;
    TX e[W];
  };
  __device__ __forceinline__ Raw() {}
};
template <typename TX, int W, bool VEC>
__device__ __forceinline__ void load_raw(const TX* x, Raw<TX, W>& r) {
  if constexpr (VEC) {
    r.w = *reinterpret_cast<const typename Raw<TX, W>::Word*>(x);
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) r.e[i] = x[i];
  }
}

// A vector's elements: y[c][i] is element c * D/4 + r0 + i.
// F: float, or double for keys on their way to codes.
template <typename F>
__device__ __forceinline__ void turn_pair(F& a, F& b, F c, F s) {
  const F ya = fma(a, c, -(b * s)), yb = fma(b, c, a * s);
  a = ya;
  b = yb;
}
// two pairs at once
__device__ __forceinline__ void turn_pairs(float& a0, float& a1, float& b0, float& b1, float c0, float c1, float s0, float s1) {
  const uint64_t a = pack2(a0, a1), b = pack2(b0, b1), c = pack2(c0, c1), s = pack2(s0, s1), n = pack2(-s0, -s1);
  unpack2(fma2(a, c, mul2(b, n)), a0, a1);
  unpack2(fma2(b, c, mul2(a, s)), b0, b1);
}

template <int W>
__device__ __forceinline__ void load_floats(const float* p, float (&v)[W]) {
  if constexpr (W == 4) {
    const float4 u = *reinterpret_cast<const float4*>(p);
    v[0] = u.x, v[1] = u.y, v[2] = u.z, v[3] = u.w;
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = p[i];
  }
}
// cs, sn: pair j's cosine and sine; buf: a place in shared memory for the vector, used where a pair's two elements lie
// in different lanes.  Called by whole warps; lanes with there = false turn nothing.
template <typename F, int W>
__device__ __forceinline__ void turn_vector(F (&y)[4][W], bool there, int r0, const HeadArgs& a, const float* cs,
                                            const float* sn, F* buf) {
  const int Q = a.D / 4, half = a.rot / 2;
  if (a.pairs == kAnyPairs) {
    __syncwarp();
    if (there) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) buf[c * Q + r0 + i] = y[c][i];
    }
    __syncwarp();
    if (!there) return;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const int e = c * Q + r0 + i;
        if (e >= a.rot) continue;
        const bool second = a.interleaved ? e & 1 : e >= half;
        const int j = a.interleaved ? e / 2 : second ? e - half : e;
        const int other = a.interleaved ? e ^ 1 : second ? e - half : e + half;
        y[c][i] = fma(y[c][i], (F)cs[j], buf[other] * (F)(second ? sn[j] : -sn[j]));
      }
    return;
  }
  if (!there) return;
  // W pairs (x[i], z[i])
  const auto run = [&](F (&x)[W], F (&z)[W], int j) {
    float c[W], s[W];
    load_floats<W>(cs + j, c);
    load_floats<W>(sn + j, s);
    if constexpr (W > 1 && sizeof(F) == 4) {
#pragma unroll
      for (int i = 0; i < W; i += 2) turn_pairs(x[i], x[i + 1], z[i], z[i + 1], c[i], c[i + 1], s[i], s[i + 1]);
    } else {
#pragma unroll
      for (int i = 0; i < W; ++i) turn_pair<F>(x[i], z[i], c[i], s[i]);
    }
  };
  if (a.pairs == kHalves) {
    run(y[0], y[2], r0);
    run(y[1], y[3], Q + r0);
  } else if (a.pairs == kHalvesOfHalf) {
    run(y[0], y[1], r0);
  } else if (a.pairs == kNeighbours) {
    if constexpr (W > 1) {
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < W; i += 2) {
          const int e = c * Q + r0 + i;
          if (e < a.rot) turn_pair<F>(y[c][i], y[c][i + 1], cs[e / 2], sn[e / 2]);
        }
    }
  }
}

// y / s to the nearest whole number (ties to even), limited to -8 .. 7; inv = 1 / s.  The quotient is corrected by what it
// leaves of y, which rounds it like a division: a tie is one exactly where y is (n + 1/2) s.
__device__ __forceinline__ int code_of(float y, float s, float inv) {
  const float t = y * inv, q = fmaf(fmaf(-t, s, y), inv, t);
  return min(max(__float_as_int(q + 12582912.f) - 0x4b400000, -8), 7);
}
__device__ __forceinline__ int code_of(double y, double s, double inv) {
  const double t = y * inv, q = fma(fma(-t, s, y), inv, t);
  return min(max(__double2loint(q + 6755399441055744.0), -8), 7);
}
// max|y| / 7.5 in fp32
__device__ __forceinline__ float scale_of(double top) { return (float)(top * (1.0 / 7.5)); }
// Largest magnitude of each quarter over a vector's lanes, as bits (an infinity or a NaN is above every number).
template <int GP, int W>
__device__ __forceinline__ uint32_t quarter_tops(const float (&y)[4][W], uint32_t (&top)[4]) {
  uint32_t most = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    top[c] = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) top[c] = max(top[c], __float_as_uint(y[c][i]) & 0x7fffffffu);
#pragma unroll
    for (int o = GP / 2; o; o >>= 1) top[c] = max(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
    most = max(most, top[c]);
  }
  return most;
}
__device__ __forceinline__ uint32_t scale_bits(float s, bool finite) {
  return finite ? __bfloat16_as_ushort(__float2bfloat16_rn(fmaxf(s, 0x1p-126f))) : 0x7fc0u;
}

// A lane's words and, from a vector's first lane, its scales.
__device__ __forceinline__ void store_codes(const HeadArgs& a, long long slot, int kind, int h, int r0,
                                            bool finite, const uint32_t (&words)[4], const uint32_t (&sb)[4]) {
  const long long vec = slot + (long long)h * a.c.page_size;   // slot: (page * n_kv_heads) * page_size + slot
  uint8_t* codes = (kind == 1 ? a.c.k_codes : a.c.v_codes) + vec * (a.D / 2) + 2 * r0;
  *reinterpret_cast<uint2*>(codes) = finite ? make_uint2(words[0] | words[1] << 16, words[2] | words[3] << 16)
                                            : make_uint2(0x88888888u, 0x88888888u);
  if (r0 == 0)
    *reinterpret_cast<uint2*>((kind == 1 ? a.ks : a.vs) + vec * 4) = make_uint2(sb[0] | sb[1] << 16, sb[2] | sb[3] << 16);
}

struct TokenPlace {
  bool put;        // the row is a sequence's token, and its page is there
  int pos;         // -1: none; -2: a padding row
  long long slot;  // (page * n_kv_heads) * page_size + slot
};

template <typename TX, int W, int GP, bool VEC, bool CACHE>
__global__ void __launch_bounds__(kThreads, CACHE && sizeof(TX) == 4 ? 3 : 4) norm_turn_kernel(const __grid_constant__ HeadArgs a) {
  static_assert(!CACHE || W == 4, "a lane's words are stored as 8 bytes");
  constexpr int AT = 32 / GP;   // vectors of a warp at a time
  extern __shared__ __align__(16) double exchange[];
  __shared__ __align__(16) float cs[kMaxDim / 2], sn[kMaxDim / 2], weights[2][kMaxDim];
  __shared__ TokenPlace place;
  griddep_launch_dependents();
  griddep_wait();
  const int D = a.D, Q = D / 4, tid = threadIdx.x, lane = tid & 31, r0 = lane % GP * W, tok = blockIdx.x;
  // A pass is a kind of vectors (1 keys, 2 values, 0 queries, in that order) and AT of its heads; this warp's are first,
  // first + step, ...
  const int k_passes = (a.Hkv + AT - 1) / AT, kv_passes = k_passes * (CACHE ? 2 : 1), passes = kv_passes + (a.H + AT - 1) / AT;
  const int step = (int)(blockDim.x / 32 * gridDim.y),
            first = __shfl_sync(0xffffffffu, (int)(blockIdx.y * (blockDim.x / 32) + tid / 32), 0);
  const auto kind_of = [&](int p) { return p < k_passes ? 1 : CACHE && p < kv_passes ? 2 : 0; };
  const auto head_of = [&](int p, int kind) {
    return (p - (kind == 1 ? 0 : kind == 2 ? k_passes : kv_passes)) * AT + lane / GP;
  };
  const auto there_of = [&](int h, int kind) { return r0 < Q && h < (kind == 0 ? a.H : a.Hkv); };
  Raw<TX, W> next[4];
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int i = 0; i < W; ++i) next[c].e[i] = TX(0.f);   // lanes beyond a vector's end add nothing to its sums
  const TX *qx = static_cast<const TX*>(a.q.p) + (long long)tok * a.q.ts + r0, *kx = static_cast<const TX*>(a.k.p) + (long long)tok * a.k.ts + r0,
           *vx = static_cast<const TX*>(a.v.p) + (long long)tok * a.v.ts + r0;
  const auto load = [&](int p) {
    if (p >= passes) return;
    const int kind = kind_of(p), h = head_of(p, kind);
    if (!there_of(h, kind)) return;
    const TX* x = kind == 0 ? qx + (long long)h * a.q.hs : kind == 1 ? kx + (long long)h * a.k.hs : vx + (long long)h * a.v.hs;
#pragma unroll
    for (int c = 0; c < 4; ++c) load_raw<TX, W, VEC>(x + c * Q, next[c]);
  };
  load(first);

  // ---- the token's place and angles ----
  const bool rows_known = CACHE || a.c.seq_lens;
  if (rows_known) {
    if (tid < 32) {
      const TokenAt at = token_at(a.c, a.T, tok);
      if (tid == 0) {
        TokenPlace p{false, -1, 0};
        if (!at.ok) {
          atomicOr(&g_dev_error, kErrIndex);
        } else if (at.pos < 0) {
          p.pos = -2;
        } else if (CACHE) {
          p.pos = at.pos;
          const int page = a.c.block_table[(size_t)at.b * a.c.pages_per_seq + at.pos / a.c.page_size];
          p.put = page >= 0 && page < a.c.num_pages;
          if (p.put) p.slot = (long long)page * a.c.n_kv_heads * a.c.page_size + at.pos % a.c.page_size;
          else atomicOr(&g_dev_error, kErrIndex);
        }
        place = p;
      }
    }
    __syncthreads();
  }
  const int half = a.rot / 2;
  for (int j = tid; j < half; j += blockDim.x) {
    long long p;
    if (rows_known && place.pos == -2) {
      p = 0;   // a padding row's positions are nobody's
    } else if (a.positions) {
      const int axis = a.axes ? a.axes[j] : 0;
      const long long at = (long long)tok * a.axes_n + axis;
      p = axis >= a.axes_n ? -1
          : a.pos64        ? static_cast<const long long*>(a.positions)[at]
                           : (long long)static_cast<const int*>(a.positions)[at];
    } else {
      p = place.pos;
    }
    const bool ok = p >= 0 && p < a.max_pos;
    if (!ok) atomicOr(&g_dev_error, kErrIndex);
    const float nan = __int_as_float(0x7fffffff);
    cs[j] = ok ? __ldg(a.table + p * a.rot + j) : nan;
    sn[j] = ok ? __ldg(a.table + p * a.rot + half + j) : nan;
  }
  if (a.norm) {
    for (int i = tid; i < 2 * Q; i += blockDim.x) {   // four weights each
      const int which = i >= Q, e = 4 * (which ? i - Q : i);
      const void* w = which ? a.wk : a.wq;
      float v[4] = {1.f, 1.f, 1.f, 1.f};
      if (w && a.w_dtype == SF_F32) {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = static_cast<const float*>(w)[e + j];
      } else if (w) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const unsigned short x = static_cast<const unsigned short*>(w)[e + j];
          v[j] = a.w_dtype == SF_BF16 ? __uint_as_float((uint32_t)x << 16) : __half2float(__ushort_as_half(x));
        }
      }
      *reinterpret_cast<float4*>(&weights[which][e]) = make_float4(v[0], v[1], v[2], v[3]);
    }
  }
  __syncthreads();
  const bool put = CACHE && place.put;
  const long long slot = CACHE ? place.slot : 0;
  TX *qo = static_cast<TX*>(a.qo.p) + (long long)tok * a.qo.ts + r0, *ko = static_cast<TX*>(a.ko.p) + (long long)tok * a.ko.ts + r0;
  // this vector's place in its warp's part of the exchange, room for 128 W doubles
  double* buf64 = exchange + (tid / 32) * (128 * W) + lane / GP * D;
  float* buf32 = reinterpret_cast<float*>(exchange + (tid / 32) * (128 * W)) + lane / GP * D;

#pragma unroll 1
  for (int p = first; p < passes; p += step) {
    const int kind = kind_of(p), h = head_of(p, kind);
    const bool there = there_of(h, kind);
    Raw<TX, W> raw[4];
#pragma unroll
    for (int c = 0; c < 4; ++c) raw[c] = next[c];
    load(p + step);
    // whole warps go through it, since sums and maxima are shuffled
    if constexpr (CACHE) {
      if (kind == 1) {
        // ---- keys, in fp64, to their codes ----
        double z[4][W];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < W; ++i) z[c][i] = (double)to_f32(raw[c].e[i]);
        if (a.norm) {
          double ss = 0;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) ss = fma(z[c][i], z[c][i], ss);
#pragma unroll
          for (int o = GP / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
          const double r = rsqrt(ss * a.inv_d64 + a.eps64);
          if (there) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              float w[W];
              load_floats<W>(weights[1] + c * Q + r0, w);
#pragma unroll
              for (int i = 0; i < W; ++i) z[c][i] = z[c][i] * r * (double)w[i];
            }
          }
        }
        turn_vector<double, W>(z, there, r0, a, cs, sn, buf64);
        uint32_t top[4], words[4] = {0x8888u, 0x8888u, 0x8888u, 0x8888u}, sb[4];
        float y[4][W];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < W; ++i) y[c][i] = (float)z[c][i];
        bool finite = quarter_tops<GP, W>(y, top) < 0x7f800000u;
        uint32_t up = 0;   // what its scales' bits are short of
        if (__any_sync(0xffffffffu, !finite)) {   // a number past fp32's range, which a turn makes, is one: a 16th of it is cut
          up = finite ? 0u : 4u << 7;
          const double down = finite ? 1.0 : 0x1p-4;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < W; ++i) y[c][i] = (float)(z[c][i] *= down);
          finite = quarter_tops<GP, W>(y, top) < 0x7f800000u;
          if (!finite) up = 0;
        }
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float s = scale_of(__uint_as_float(top[c]));
          // within 4 last places of a tie of two scales: from the largest magnitude in fp64
          const bool near = ((__float_as_uint(s) - 0x7ffcu) & 0xffffu) <= 8u;
          if (__any_sync(0xffffffffu, near)) {
            double big = 0;
#pragma unroll
            for (int i = 0; i < W; ++i) big = fmax(big, fabs(z[c][i]));
#pragma unroll
            for (int o = GP / 2; o; o >>= 1) big = fmax(big, __shfl_xor_sync(0xffffffffu, big, o));
            if (near) s = scale_of(big);
          }
          sb[c] = scale_bits(s, finite);
          s = __uint_as_float(sb[c] << 16);
          const double s64 = s, near_inv = __frcp_rn(s), inv = near_inv * fma(-s64, near_inv, 2.0);
#pragma unroll
          for (int i = 0; i < W; ++i) words[i] += code_of(z[c][i], s64, inv) * (1 << 4 * c);
          if (sb[c] != 0x0080u) sb[c] += up;   // but the least scale, of zeros
        }
        if (there && put) store_codes(a, slot, 1, h, r0, finite, words, sb);
        continue;
      }
      if (kind == 2) {
        // ---- values, exact as they are, to their codes ----
        float y[4][W];
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < W; ++i) y[c][i] = to_f32(raw[c].e[i]);
        uint32_t top[4], words[4] = {0x8888u, 0x8888u, 0x8888u, 0x8888u}, sb[4];
        const bool finite = quarter_tops<GP, W>(y, top) < 0x7f800000u;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          sb[c] = scale_bits(scale_of(__uint_as_float(top[c])), finite);
          const float s = __uint_as_float(sb[c] << 16), inv = __frcp_rn(s);
#pragma unroll
          for (int i = 0; i < W; ++i) words[i] += code_of(y[c][i], s, inv) * (1 << 4 * c);
        }
        if (there && put) store_codes(a, slot, 2, h, r0, finite, words, sb);
        continue;
      }
    }
    // ---- queries, or keys that stay ones, to their own type ----
    float y[4][W];
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int i = 0; i < W; ++i) y[c][i] = to_f32(raw[c].e[i]);
    if (a.norm) {
      float ss = 0;
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < W; ++i) ss = fmaf(y[c][i], y[c][i], ss);
#pragma unroll
      for (int o = GP / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      const float r = rsqrtf(fmaf(ss, a.inv_d, a.eps));
      if (there) {
        const float* w = weights[kind] + r0;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          float u[W];
          load_floats<W>(w + c * Q, u);
          if constexpr (W > 1) {
#pragma unroll
            for (int i = 0; i < W; i += 2)
              unpack2(mul2(pack2(y[c][i], y[c][i + 1]), mul2(pack2(r, r), pack2(u[i], u[i + 1]))), y[c][i], y[c][i + 1]);
          } else {
            y[c][0] *= r * u[0];
          }
        }
      }
    }
    turn_vector<float, W>(y, there, r0, a, cs, sn, buf32);
    if (there) {
      TX* o = kind == 0 ? qo + (long long)h * a.qo.hs : ko + (long long)h * a.ko.hs;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        Raw<TX, W> w;
#pragma unroll
        for (int i = 0; i < W; ++i) w.e[i] = from_f32<TX>(y[c][i]);
        if constexpr (VEC) {
          *reinterpret_cast<typename Raw<TX, W>::Word*>(o + c * Q) = w.w;
        } else {
#pragma unroll
          for (int i = 0; i < W; ++i) o[c * Q + i] = w.e[i];
        }
      }
    }
  }
}

bool aligned_rows(const void* p, int dtype, long long ts, long long hs, int W) {
  const int size = dtype == SF_F32 ? 4 : 2;
  return reinterpret_cast<uintptr_t>(p) % (size * W) == 0 && ts % W == 0 && hs % W == 0;
}

bool strides_ok(std::initializer_list<long long> head_strides) {
  for (const long long x : head_strides)
    if (x < 0 || x > 0x7fffffffll) return false;
  return true;
}

int check_args(const HeadArgs& a, int dtype) {
  if (dtype < 0 || dtype > 2 || a.w_dtype < 0 || a.w_dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (a.rot < 0 || a.rot % 2 || a.rot > a.D) return fail(SF_ERR_SHAPE, "rot must be even and at most head_dim");
  if (a.rot > 0 && (!a.table || a.max_pos < 1)) return fail(SF_ERR_SHAPE, "the rotary table is missing or empty");
  if (a.positions && (a.axes_n < 1 || a.axes_n > kMaxAxes || (a.axes_n > 1 && !a.axes)))
    return fail(SF_ERR_SHAPE, "need 1 to %d axes, and with more than one the axis of each pair", kMaxAxes);
  return SF_OK;
}

// A positive eps stays one in fp32, or a vector of zeros would be 0 times infinity.
float eps_f32(double eps) { return eps > 0. ? std::max((float)eps, FLT_MIN) : (float)eps; }

// Warps of a block and blocks of a token: a warp takes its vectors at once where the tokens are few, else up to kRounds times in turn.
template <typename TX, int W, bool CACHE>
cudaError_t launch(HeadArgs& a, bool vec, cudaStream_t st) {
  const int lanes = a.D / 4 / W;
  a.inv_d64 = 1.0 / a.D;
  a.inv_d = (float)a.inv_d64;
  const auto go = [&](auto gp) -> cudaError_t {
    constexpr int GP = decltype(gp)::value, AT = 32 / GP;
    const int passes = (a.Hkv + AT - 1) / AT * (CACHE ? 2 : 1) + (a.H + AT - 1) / AT;
    const long long fill = 32ll * device_info().sms;   // warps
    const int rounds = (int)std::min<long long>(kRounds, std::max<long long>(1, (long long)a.T * passes / fill));
    const int warps = (passes + rounds - 1) / rounds, parts = (warps + kThreads / 32 - 1) / (kThreads / 32);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.T, (unsigned)parts);
    cfg.blockDim = dim3((unsigned)((warps + parts - 1) / parts * 32));
    cfg.dynamicSmemBytes = a.pairs == kAnyPairs ? (size_t)cfg.blockDim.x / 32 * 128 * W * sizeof(double) : 0;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    auto* fn = vec ? norm_turn_kernel<TX, W, GP, true, CACHE> : norm_turn_kernel<TX, W, GP, false, CACHE>;
    return cudaLaunchKernelEx(&cfg, fn, a);
  };
  if constexpr (W == 4) {
    if (lanes <= 4) return go(std::integral_constant<int, 4>());
    if (lanes <= 8) return go(std::integral_constant<int, 8>());
    if (CACHE || lanes <= 16) return go(std::integral_constant<int, 16>());
  }
  if constexpr (W == 2) {
    if (lanes <= 16) return go(std::integral_constant<int, 16>());
  }
  if constexpr (CACHE) return cudaErrorInvalidValue;   // a head of the cache has at most 256 elements
  else return go(std::integral_constant<int, 32>());
}

// Which of a head's elements make its pairs, as the lanes hold them (W places of every quarter).
int pairs_of(const HeadArgs& a, int W) {
  if (a.rot == 0) return kNoPairs;
  if (a.interleaved) return W > 1 ? kNeighbours : kAnyPairs;
  return a.rot == a.D ? kHalves : 2 * a.rot == a.D ? kHalvesOfHalf : kAnyPairs;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

int sf_qk_norm_rotary_rows(const void* q, long long qts, long long qhs, void* q_out, long long qots, long long qohs, int H,
                           const void* k, long long kts, long long khs, void* k_out, long long kots, long long kohs, int Hkv,
                           int dtype, const void* q_weight, const void* k_weight, int w_dtype, double eps,
                           const void* positions, int pos64, int axes_n, const uint8_t* axes, const float* table, int max_pos,
                           int rot, int interleaved, int T, int D, const int* seq_lens, const int* starts, int batch,
                           void* stream) {
  if (T < 0 || H < 0 || Hkv < 0) return fail(SF_ERR_SHAPE, "need T, H, Hkv >= 0");
  if (D < 4 || D % 4 || D > (D % 16 == 0 ? 512 : D % 8 == 0 ? 256 : 128))
    return fail(SF_ERR_UNSUPPORTED, "head_dim %d not built (multiples of 16 up to 512, of 8 up to 256, of 4 up to 128)", D);
  if (H <= 1) qhs = qohs = 0;   // no second head: never used
  if (Hkv <= 1) khs = kohs = 0;
  HeadArgs a{};
  a.q = Vectors{q, qts, (int)qhs};
  a.k = Vectors{k, kts, (int)khs};
  a.qo = Out{q_out, qots, (int)qohs};
  a.ko = Out{k_out, kots, (int)kohs};
  a.wq = q_weight; a.wk = k_weight; a.w_dtype = w_dtype;
  a.norm = eps >= 0.;
  a.eps64 = eps;
  a.eps = eps_f32(eps);
  a.table = table; a.max_pos = max_pos; a.rot = rot; a.interleaved = interleaved;
  a.positions = positions; a.pos64 = pos64; a.axes_n = axes_n; a.axes = axes;
  a.H = H; a.Hkv = Hkv; a.T = T; a.D = D;
  if (int rc = check_args(a, dtype)) return rc;
  if (seq_lens) {
    if (batch < 1) return fail(SF_ERR_SHAPE, "need batch >= 1");
    if (!starts && T % batch) return fail(SF_ERR_SHAPE, "without starts, T must be a multiple of batch");
    a.c.seq_lens = seq_lens;
    a.c.starts = starts;
    a.c.batch = batch;
    a.c.page_size = 1;
    a.c.pages_per_seq = 0x7fffffff;   // a sequence of any length: it has no pages here
  } else if (starts) {
    return fail(SF_ERR_NULL, "starts without seq_lens");
  }
  if (T == 0 || H + Hkv == 0) return SF_OK;
  if ((H && (!q || !q_out)) || (Hkv && (!k || !k_out)) || (rot && !positions)) return fail(SF_ERR_NULL, "null pointer argument");
  if (!strides_ok({qhs, qohs, khs, kohs})) return fail(SF_ERR_UNSUPPORTED, "a head stride above 2^31 - 1 elements");
  if ((long long)H + Hkv > 0xffff) return fail(SF_ERR_UNSUPPORTED, "more than 65535 heads");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    const auto go = [&](auto w) {
      constexpr int W = decltype(w)::value;
      a.pairs = pairs_of(a, W);
      const bool vec = (!H || (aligned_rows(q, dtype, qts, qhs, W) && aligned_rows(q_out, dtype, qots, qohs, W))) &&
                       (!Hkv || (aligned_rows(k, dtype, kts, khs, W) && aligned_rows(k_out, dtype, kots, kohs, W)));
      return launch<TX, W, false>(a, vec, st);
    };
    return D % 16 == 0  ? go(std::integral_constant<int, 4>())
           : D % 8 == 0 ? go(std::integral_constant<int, 2>())
                        : go(std::integral_constant<int, 1>());
  });
  if (e != cudaSuccess) return cuda_fail(e, "norm_turn_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

int sf_qk_norm_rotary(const void* q, long long qts, long long qhs, void* q_out, long long qots, long long qohs, int H,
                      const void* k, long long kts, long long khs, void* k_out, long long kots, long long kohs, int Hkv,
                      int dtype, const void* q_weight, const void* k_weight, int w_dtype, double eps,
                      const void* positions, int pos64, int axes_n, const uint8_t* axes, const float* table, int max_pos,
                      int rot, int interleaved, int T, int D, void* stream) {
  return sf_qk_norm_rotary_rows(q, qts, qhs, q_out, qots, qohs, H, k, kts, khs, k_out, kots, kohs, Hkv, dtype, q_weight,
                                k_weight, w_dtype, eps, positions, pos64, axes_n, axes, table, max_pos, rot, interleaved, T, D,
                                nullptr, nullptr, 0, stream);
}

int sf_paged4_append(const sf_paged4_cache* cache, const void* k, long long kts, long long khs, const void* v,
                     long long vts, long long vhs, const void* q, long long qts, long long qhs, void* q_out, int dtype,
                     int H, int T, const void* q_weight, const void* k_weight, int w_dtype, double eps,
                     const void* positions, int pos64, int axes_n, const uint8_t* axes, const float* table, int max_pos,
                     int rot, int interleaved, void* stream) {
  HeadArgs a{};
  if (int rc = check_paged4(cache, T, a.c)) return rc;
  const int D = cache->head_dim;
  if (H <= 1) qhs = 0;   // no second head: never used
  if (cache->n_kv_heads == 1) khs = vhs = 0;
  a.q = Vectors{q, qts, (int)qhs};
  a.k = Vectors{k, kts, (int)khs};
  a.v = Vectors{v, vts, (int)vhs};
  a.qo = Out{q_out, (long long)H * D, D};
  a.wq = q_weight; a.wk = k_weight; a.w_dtype = w_dtype;
  a.norm = eps >= 0.;
  a.eps64 = eps;
  a.eps = eps_f32(eps);
  a.table = table; a.max_pos = max_pos; a.rot = table ? rot : 0; a.interleaved = interleaved;
  a.positions = positions; a.pos64 = pos64; a.axes_n = axes_n; a.axes = axes;
  a.H = q ? H : 0; a.Hkv = cache->n_kv_heads; a.T = T; a.D = D;
  a.ks = static_cast<__nv_bfloat16*>(cache->k_scales);
  a.vs = static_cast<__nv_bfloat16*>(cache->v_scales);
  if (int rc = check_args(a, dtype)) return rc;
  if (T == 0) return SF_OK;
  if (!k || !v || (q && !q_out)) return fail(SF_ERR_NULL, "null pointer argument");
  if (q && H < 1) return fail(SF_ERR_SHAPE, "need H >= 1 query heads");
  if (!strides_ok({khs, vhs, qhs})) return fail(SF_ERR_UNSUPPORTED, "a head stride above 2^31 - 1 elements");
  if ((long long)a.H + 2ll * a.Hkv > 0xffff) return fail(SF_ERR_UNSUPPORTED, "more than 65535 heads");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const cudaError_t e = with_type(dtype, [&](auto* p) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(p)>>;
    a.pairs = pairs_of(a, 4);
    const bool vec = aligned_rows(k, dtype, kts, khs, 4) && aligned_rows(v, dtype, vts, vhs, 4) &&
                     (!q || (aligned_rows(q, dtype, qts, qhs, 4) && aligned_rows(q_out, dtype, D, D, 4)));
    return launch<TX, 4, true>(a, vec, st);
  });
  if (e != cudaSuccess) return cuda_fail(e, "norm_turn_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

}  // extern "C"
