// sf_paged_attention.cu -- attention over the pages of an e4m3 cache.
//
//   p_j = softmax_j(scale * q . k_j),  out = sum_j p_j v_j,  k_j = code * scale of its page and head
//
// The softmax keeps a running maximum m and sum l: keys in order, out and l are multiplied by e^(m - m') when the
// maximum grows to m'.  Parts of a row's keys merge by the same rule.
//
// A call's work is a list of units of 4 * WB keys, for each (sequence, kv head, tile of query rows) in turn; a row is
// one (new token, query head of the kv head's group), so that a group reads its keys once.  Every CTA takes an equal,
// contiguous share of that list, whatever the sequences' lengths: it finds its place from a prefix sum over the
// batch.  A CTA that holds all of a tile's units writes the result; the others leave their parts in the workspace,
// which a second kernel merges.
//
// Per warp, WB keys at a time, on mma.sync m16n8k16 (fp16 in, fp32 sums):
//  * S = Q K^T, rows of the tile by keys.  K's codes become fp16 exactly; its fragments are 32-bit words of a key's
//    row, for which the 16 columns of an MMA are taken in the order 4t .. 4t+3 per lane t, in Q and in K alike.
//  * O += P V with P's accumulators as the next MMA's operand.  A lane's words of four keys, byte-transposed, are its
//    fragments for four 8-column tiles: column g of tile j is column 4g + j of each 32.
//  * Tiles of at most 8 rows put a row's high part in MMA row g and its low part in row g + 8: queries and weights
//    keep 22 bits for the price of the padding that 16 rows would be.  Tiles of 16 rows (16-bit queries, which fp16
//    holds exactly after a power-of-two scaling of each row) round weights to 11 bits.
//  * V's scales fold into P relative to the largest one met (exact: powers of two), times 2^10 to keep small weights
//    clear of fp16's subnormals.
#include <atomic>
#include <cmath>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_q4_internal.h"
#include "sf_paged.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_paged)
extern std::atomic<long long> g_launches;

namespace {

constexpr int kWarps = 4;
constexpr int kMaxCtasPerSm = 3;
constexpr float kPScale = 1024.f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct AttnArgs {
  sf_paged_cache c;
  const void* q;
  long long qts, qhs;
  void* out;
  float* lse;
  float* part;          // [CTA][2][16][D + 2]: unnormalised sums, then m and l
  int* desc;            // [CTA][8]: the tile that this CTA began and others ended
  int H, T, G, q_dtype, out_dtype, window, lg_page;
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
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// four e4m3 codes -> two fp16 pairs, exactly
__device__ __forceinline__ void e4m3x4_to_h2x2(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
      : "=r"(lo), "=r"(hi)
      : "r"(w));
}
__device__ __forceinline__ uint32_t h2u(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ void split_h2(float x0, float x1, uint32_t& hi, uint32_t& lo) {
  const __half2 h = __floats2half2_rn(x0, x1);
  const float2 f = __half22float2(h);
  hi = h2u(h);
  lo = h2u(__floats2half2_rn(x0 - f.x, x1 - f.y));
}
__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
  uint32_t d;
  asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
  return d;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}

// Shared memory: per warp STAGES x (WB key rows, then WB value rows), a row D + 16 bytes apart so that the fragment
// reads of 8 key rows, and of 4 value rows by 32 bytes, fall into different banks; then the batch's SeqInfo.  The
// stages hold the warps' sums when a CTA's part of a tile ends.
template <int D>
struct Lay {
  static constexpr int WB = D <= 128 ? 32 : 16;
  static constexpr int STAGES = 2;
  static constexpr int RP = D + 16;
  static constexpr int KV = WB * RP;
  static constexpr int WARP = STAGES * 2 * KV;
  static constexpr int UNIT = kWarps * WB;
  static constexpr size_t smem(int batch) { return (size_t)kWarps * WARP + (size_t)batch * sizeof(SeqInfo); }
};

// Keys that the sequence's units cover: from lo (a multiple of 16) to len.
__device__ __forceinline__ int keys_from(const AttnArgs& a, int len, int n) {
  return a.window > 0 ? max(0, len - n + 1 - a.window) & ~15 : 0;
}

template <int D, bool HL>
__global__ void __launch_bounds__(32 * kWarps, D <= 128 ? kMaxCtasPerSm : 2) paged_attention_kernel(const AttnArgs a) {
  using L = Lay<D>;
  constexpr int WB = L::WB, RT = HL ? 8 : 16, RPL = HL ? 1 : 2;   // rows of a tile, rows of a lane
  constexpr int KS = D / 16, NT = WB / 8, DB = D / 32, CH = D / 16;
  constexpr int GPB = WB / 16, NB = 32 / GPB;                      // 16-key granules of a block, blocks of 32 granules
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float wm[kWarps][16], wl[kWarps][16], wv[kWarps];
  __shared__ long long wsum[kWarps];
  SeqInfo* info = reinterpret_cast<SeqInfo*>(smem + kWarps * L::WARP);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  griddep_launch_dependents();

  // ---- the batch's units, and this CTA's share ----
  const int B = a.c.batch, Hkv = a.c.n_kv_heads, page_size = a.c.page_size;
  long long total = 0;
  for (int base = 0; base < B; base += 32 * kWarps) {
    const int b = base + threadIdx.x;
    long long u = 0;
    int len = 0, n = 0;
    if (b < B) {
      const int r0 = first_row(a.c, a.T, b), r1 = first_row(a.c, a.T, b + 1);
      len = a.c.seq_lens[b];
      n = r1 - r0;
      if (r0 < 0 || n < 0 || r1 > a.T) {
        n = 0;
        atomicOr(&g_dev_error, kErrIndex);
      }
      if (!len_ok(a.c, len)) {
        len = 0;
        atomicOr(&g_dev_error, kErrIndex);
      }
      const int tiles = (int)(((long long)n * a.G + RT - 1) / RT);
      u = (long long)tiles * Hkv * max(1, (len - keys_from(a, len, n) + L::UNIT - 1) / L::UNIT);
    }
    long long incl = u;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long x = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += x;
    }
    if (lane == 31) wsum[warp] = incl;
    __syncthreads();
    long long before = total;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += wsum[w];
      total += wsum[w];
    }
    if (b < B) info[b] = SeqInfo{before + incl - u, len, n};
    __syncthreads();
  }
  const long long C = min((long long)gridDim.x, total), cta = blockIdx.x;   // CTAs with a share: at least a unit each
  if (threadIdx.x == 0) a.desc[8 * cta] = 0;
  if (cta >= C) return;
  long long u = total * cta / C;
  const long long u_end = total * (cta + 1) / C;
  int b = 0;
  for (int lo = 0, hi = B; hi - lo > 1;) {
    const int mid = (lo + hi) >> 1;
    if (info[mid].first <= u) lo = mid;
    else hi = mid;
    b = lo;
  }

  const uint32_t wbase = smem_u32(smem + warp * L::WARP);
  for (; u < u_end;) {
    // ---- the tile that holds unit u, and the part [u, u1) of its units that is this CTA's ----
    while (b + 1 < B && info[b + 1].first <= u) ++b;
    const SeqInfo s = info[b];
    const int tiles = (int)(((long long)s.n * a.G + RT - 1) / RT);
    const int from = keys_from(a, s.len, s.n);
    const int per = max(1, (s.len - from + L::UNIT - 1) / L::UNIT);
    const long long rel = u - s.first, seg = rel / per;
    const int j0 = (int)(rel % per), kvh = (int)(seg / tiles), row0 = (int)(seg % tiles) * RT;
    const long long seg0 = s.first + seg * per, seg1 = seg0 + per;
    const long long u1 = seg1 < u_end ? seg1 : u_end;
    const int r_first = first_row(a.c, a.T, b);
    const int pos0 = s.len - s.n;                                // position of the sequence's first new row
    const int last_row = min(row0 + RT, s.n * a.G) - 1;
    const int tile_hi = pos0 + last_row / a.G + 1;               // keys that some row sees: [tile_lo, tile_hi)
    const int tile_lo = a.window > 0 ? max(0, pos0 + row0 / a.G + 1 - a.window) : 0;
    const int all_hi = pos0 + row0 / a.G + 1;                    // keys that every row sees: [all_lo, all_hi)
    const int all_lo = a.window > 0 ? max(0, tile_hi - a.window) : 0;
    // the unit grid starts at `from`; blocks without a key that some row sees are left out
    int ta = from + j0 * L::UNIT;
    const int tb = (int)min((long long)tile_hi, from + (long long)(j0 + (u1 - u)) * L::UNIT);
    if (ta < (tile_lo & ~15)) ta = tile_lo & ~15;

    // ---- query fragments ----
    uint32_t qf[KS][4];
    float f[RPL];
    int rhi[RPL], rlo[RPL];
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      const int row = row0 + g + 8 * i;
      const bool in = row <= last_row;
      const int tok = row / a.G, pos = pos0 + tok;
      rhi[i] = in ? pos + 1 : 0;
      rlo[i] = in && a.window > 0 ? max(0, pos + 1 - a.window) : 0;
      const long long qo = (long long)(r_first + tok) * a.qts + (long long)(kvh * a.G + row % a.G) * a.qhs;
      uint32_t top = 0;
      for (int k = 0; k < KS && in; ++k)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(load_q(a, qo + 16 * k + 4 * t + e)) & 0x7fffffffu);
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      // the row over 2^ex, which puts its largest value in [1, 2); zero, subnormal and non-finite rows as they are
      int ex = (int)(top >> 23) - 127;
      if (ex == -127 || ex == 128) ex = 0;
      if (ex > 126) ex = 126;                                    // 2^-ex has to be a normal number
      const float down = __int_as_float((127 - ex) << 23);
      f[i] = __int_as_float((127 + ex) << 23) * (a.scale * kLog2e);
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (in) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = load_q(a, qo + 16 * k + 4 * t + e) * down;
        }
        if constexpr (HL) {
          split_h2(v[0], v[1], qf[k][0], qf[k][1]);
          split_h2(v[2], v[3], qf[k][2], qf[k][3]);
        } else {
          qf[k][i] = h2u(__floats2half2_rn(v[0], v[1]));
          qf[k][2 + i] = h2u(__floats2half2_rn(v[2], v[3]));
        }
      }
    }

    // ---- this warp's blocks: keys ta + WB (warp + 4 i) .. ----
    // Lane l of a set holds page and scales of the set's granule l: block l / GPB, its keys 16 (l % GPB) ..
    struct Set {
      int page;
      float ks, vs;
    };
    const auto load_set = [&](int set) {
      Set x{-1, 0.f, 0.f};
      const long long tok = ta + (long long)WB * (warp + kWarps * (NB * set + lane / GPB)) + 16 * (lane % GPB);
      if (tok < tb) {
        const int page = a.c.block_table[(size_t)b * a.c.pages_per_seq + (tok >> a.lg_page)];
        if (page >= 0 && page < a.c.num_pages) {
          x.page = page;
          x.ks = a.c.k_scales[(size_t)page * Hkv + kvh];
          x.vs = a.c.v_scales[(size_t)page * Hkv + kvh];
        } else {
          atomicOr(&g_dev_error, kErrIndex);
        }
      }
      return x;
    };
    Set cur = load_set(0), nxt = load_set(1);
    const auto issue = [&](int i, const Set& x) {
      const int base = ta + WB * (warp + kWarps * i);
      int pg[GPB];
#pragma unroll
      for (int e = 0; e < GPB; ++e) pg[e] = __shfl_sync(0xffffffffu, x.page, (i % NB) * GPB + e);
      if (base < tb) {
        const uint32_t st = wbase + (uint32_t)(i % L::STAGES) * (2 * L::KV);
#pragma unroll
        for (int k = 0; k < WB * CH / 32; ++k) {
          const int c = lane + 32 * k, r = c / CH, dp = (c % CH) * 16, key = base + r;
          const int page = GPB == 1 ? pg[0] : (r < 16 ? pg[0] : pg[GPB - 1]);
          // rows of no key are zeros: what lies past a sequence's end may be NaN, and 0 * NaN is not 0
          const bool v = key < tb && key >= tile_lo && page >= 0;
          const size_t at = (((size_t)(v ? page : 0) * Hkv + kvh) * page_size + (v ? key & (page_size - 1) : 0)) * D + dp;
          cp_async16(st + r * L::RP + dp, a.c.k_codes + at, v);
          cp_async16(st + L::KV + r * L::RP + dp, a.c.v_codes + at, v);
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };

    float m[RPL], l[RPL], o[4 * DB][4], vref = 0x1p-100f;
#pragma unroll
    for (int i = 0; i < RPL; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 4 * DB; ++i) o[i][0] = o[i][1] = o[i][2] = o[i][3] = 0.f;

    issue(0, cur);
    for (int i = 0;; ++i) {
      const int base = ta + WB * (warp + kWarps * i);
      if (base >= tb) break;
      issue(i + 1, (i + 1) % NB ? cur : nxt);
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncwarp();
      const uint32_t st = wbase + (uint32_t)(i % L::STAGES) * (2 * L::KV);
      float ks[GPB], vs[GPB];
      bool whole = base + WB <= tb && base >= all_lo && base + WB <= all_hi;
#pragma unroll
      for (int e = 0; e < GPB; ++e) {
        const int src = (i % NB) * GPB + e;
        ks[e] = __shfl_sync(0xffffffffu, cur.ks, src);
        vs[e] = __shfl_sync(0xffffffffu, cur.vs, src);
        if (__shfl_sync(0xffffffffu, cur.page, src) < 0) whole = false;
      }
      // ---- scores ----
      float x[NT][2 * RPL];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        float acc[4] = {0.f, 0.f, 0.f, 0.f};
        const uint32_t kr = st + (8 * j + g) * L::RP + 4 * t;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t b0, b1;
          e4m3x4_to_h2x2(lds32(kr + 16 * k), b0, b1);
          mma16816(acc, qf[k], b0, b1);
        }
        const float sk = ks[j / 2];
        if constexpr (HL) {
          x[j][0] = (acc[0] + acc[2]) * (f[0] * sk);
          x[j][1] = (acc[1] + acc[3]) * (f[0] * sk);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) x[j][e] = acc[e] * (f[e / 2] * sk);
        }
      }
      if (!whole) {
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          const bool there = __shfl_sync(0xffffffffu, cur.page, (i % NB) * GPB + j / 2) >= 0;
#pragma unroll
          for (int e = 0; e < 2 * RPL; ++e) {
            const int key = base + 8 * j + 2 * t + (e & 1), r = e / 2;
            if (!there || key < rlo[r] || key >= rhi[r] || key >= tb) x[j][e] = -INFINITY;
          }
        }
      }
      // ---- running softmax ----
      float ref[RPL], corr[RPL];
      float vmax = vs[0];
#pragma unroll
      for (int e = 1; e < GPB; ++e) vmax = fmaxf(vmax, vs[e]);
      const float vnew = fmaxf(vref, vmax), vinv = 1.f / vnew, vdown = vref * vinv;
      vref = vnew;
#pragma unroll
      for (int r = 0; r < RPL; ++r) {
        float bm = -INFINITY;
#pragma unroll
        for (int j = 0; j < NT; ++j) bm = fmaxf(bm, fmaxf(x[j][2 * r], x[j][2 * r + 1]));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 1));
        bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, 2));
        const float mn = fmaxf(m[r], bm);
        ref[r] = mn == -INFINITY ? 0.f : mn;
        corr[r] = ex2(m[r] - ref[r]);
        m[r] = mn;
        l[r] *= corr[r];
        corr[r] *= vdown;
      }
      bool same = corr[0] == 1.f;
      if (RPL == 2) same = same && corr[RPL - 1] == 1.f;
      if (!__all_sync(0xffffffffu, same)) {
#pragma unroll
        for (int i2 = 0; i2 < 4 * DB; ++i2) {
          o[i2][0] *= corr[0];
          o[i2][1] *= corr[0];
          o[i2][2] *= corr[RPL - 1];
          o[i2][3] *= corr[RPL - 1];
        }
      }
      uint32_t pf[NT / 2][4];
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        const float fold = vs[j / 2] * (kPScale * vinv);
        float p[2 * RPL];
#pragma unroll
        for (int e = 0; e < 2 * RPL; ++e) {
          p[e] = ex2(x[j][e] - ref[e / 2]);
          l[e / 2] += p[e];
          p[e] *= fold;
        }
        if constexpr (HL) {
          split_h2(p[0], p[1], pf[j / 2][2 * (j & 1)], pf[j / 2][2 * (j & 1) + 1]);
        } else {
          pf[j / 2][2 * (j & 1)] = h2u(__floats2half2_rn(p[0], p[1]));
          pf[j / 2][2 * (j & 1) + 1] = h2u(__floats2half2_rn(p[2 * RPL - 2], p[2 * RPL - 1]));
        }
      }
      // ---- values ----
      // Where rows see different keys, a NaN among the values must reach only the rows that see its key, and 0 * NaN
      // is not 0: such a block's NaN codes are put into those rows' sums by hand, and become zeros.
      if (!(base >= all_lo && min(base + WB, tb) <= all_hi)) {
        const uint32_t sv = st + L::KV;
        uint32_t found = 0;
        for (int c = lane; c < WB * D / 4; c += 32) {
          const uint32_t w = lds32(sv + (c / (D / 4)) * L::RP + (c % (D / 4)) * 4);
          found |= ((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
        }
        if (__any_sync(0xffffffffu, found != 0)) {
          for (int r = 0; r < WB; ++r) {
#pragma unroll
            for (int e = 0; e < RPL; ++e) {
              const int key = base + r;
              if (key < rlo[e] || key >= rhi[e] || key >= tb) continue;
#pragma unroll
              for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                  const uint32_t w = lds32(sv + r * L::RP + 32 * db + 8 * t + 4 * h);
#pragma unroll
                  for (int j = 0; j < 4; ++j)
                    if (((w >> (8 * j)) & 0x7fu) == 0x7fu) o[4 * db + j][2 * e + h] = __int_as_float(0x7fffffff);
                }
            }
          }
          __syncwarp();
          for (int c = lane; c < WB * D / 4; c += 32) {
            const uint32_t at = sv + (c / (D / 4)) * L::RP + (c % (D / 4)) * 4;
            uint32_t w = lds32(at);
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (((w >> (8 * j)) & 0x7fu) == 0x7fu) w &= ~(0xffu << (8 * j));
            asm volatile("st.shared.u32 [%0], %1;" ::"r"(at), "r"(w) : "memory");
          }
          __syncwarp();
        }
      }
      const uint32_t vr = st + L::KV + 2 * t * L::RP + 4 * g;
#pragma unroll
      for (int kk = 0; kk < NT / 2; ++kk) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const uint32_t at = vr + 16 * kk * L::RP + 32 * db;
          const uint32_t w0 = lds32(at), w1 = lds32(at + L::RP), w2 = lds32(at + 8 * L::RP), w3 = lds32(at + 9 * L::RP);
          uint32_t b0[4], b1[4];
          e4m3x4_to_h2x2(prmt(w0, w1, 0x5140), b0[0], b0[1]);
          e4m3x4_to_h2x2(prmt(w0, w1, 0x7362), b0[2], b0[3]);
          e4m3x4_to_h2x2(prmt(w2, w3, 0x5140), b1[0], b1[1]);
          e4m3x4_to_h2x2(prmt(w2, w3, 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int j = 0; j < 4; ++j) mma16816(o[4 * db + j], pf[kk], b0[j], b1[j]);
        }
      }
      __syncwarp();   // the stage may be filled again
      if ((i + 1) % NB == 0) {
        cur = nxt;
        nxt = load_set((i + 1) / NB + 1);
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");

    // ---- the four warps' parts ----
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
      l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    }
    __syncthreads();   // every warp is done with its stages
    float* sums = reinterpret_cast<float*>(smem);   // [warp][row][D]
    const float unit = vref * (1.f / kPScale);
#pragma unroll
    for (int r = 0; r < RPL; ++r) {
      if (t == 0) {
        wm[warp][g + 8 * r] = m[r];
        wl[warp][g + 8 * r] = l[r];
      }
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float4 v;
          float* p = &v.x;
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = HL ? o[4 * db + j][h] + o[4 * db + j][2 + h] : o[4 * db + j][2 * r + h];
          *reinterpret_cast<float4*>(sums + ((size_t)warp * RT + g + 8 * r) * D + 32 * db + 8 * t + 4 * h) = v;
        }
    }
    if (lane == 0) wv[warp] = unit;
    __syncthreads();
    const bool begins = u == seg0, ends = u1 == seg1;
    float* part = a.part + ((size_t)cta * 2 + (begins ? 1 : 0)) * 16 * (D + 2);
    for (int i = threadIdx.x; i < RT * D; i += 32 * kWarps) {
      const int row = i / D, d = i % D;
      if (row0 + row > last_row) break;
      float M = -INFINITY;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) M = fmaxf(M, wm[w][row]);
      float A = 0.f, Ls = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        const float c = M == -INFINITY ? 0.f : ex2(wm[w][row] - M);
        A += sums[(w * RT + row) * D + d] * (c * wv[w]);
        Ls += wl[w][row] * c;
      }
      if (begins && ends) {
        const int q_row = row0 + row, head = kvh * a.G + q_row % a.G;
        const size_t th = (size_t)(r_first + q_row / a.G) * a.H + head;
        store_out(a, th * D + d, Ls == 0.f ? 0.f : A / Ls);
        if (d == 0 && a.lse) a.lse[th] = Ls == 0.f ? -INFINITY : M * kLn2 + logf(Ls);
      } else {
        part[row * D + d] = A;
        if (d == 0) {
          part[16 * D + 2 * row] = M;
          part[16 * D + 2 * row + 1] = Ls;
        }
      }
    }
    if (begins && !ends && threadIdx.x == 0) {
      // CTAs of the tile's parts: this one to the one that holds its last unit
      const long long last = (seg1 * C - 1) / total;
      int* dsc = a.desc + 8 * cta;
      dsc[0] = (int)(last - cta + 1);
      dsc[1] = r_first;
      dsc[2] = kvh;
      dsc[3] = row0;
      dsc[4] = last_row;
    }
    __syncthreads();   // sums is stages again
    u = u1;
  }
}

// One block for each (CTA that began a divided tile, row of it): the parts by the same rule, in order.
template <int D>
__global__ void __launch_bounds__(D) paged_attention_merge_kernel(const AttnArgs a) {
  griddep_launch_dependents();
  griddep_wait();
  const int* dsc = a.desc + 8 * blockIdx.x;
  const int parts = dsc[0], row = blockIdx.y, q_row = dsc[3] + row;
  if (parts == 0 || q_row > dsc[4]) return;
  const auto part = [&](int i) {
    return a.part + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * 16 * (D + 2);
  };
  float M = -INFINITY;
  for (int i = 0; i < parts; ++i) M = fmaxf(M, part(i)[16 * D + 2 * row]);
  float A = 0.f, Ls = 0.f;
#pragma unroll 4
  for (int i = 0; i < parts; ++i) {
    const float* p = part(i);
    const float c = M == -INFINITY ? 0.f : ex2(p[16 * D + 2 * row] - M);
    A += p[row * D + threadIdx.x] * c;
    Ls += p[16 * D + 2 * row + 1] * c;
  }
  const size_t th = (size_t)(dsc[1] + q_row / a.G) * a.H + dsc[2] * a.G + q_row % a.G;
  store_out(a, th * D + threadIdx.x, Ls == 0.f ? 0.f : A / Ls);
  if (threadIdx.x == 0 && a.lse) a.lse[th] = Ls == 0.f ? -INFINITY : M * kLn2 + logf(Ls);
}

template <int D, bool HL>
cudaError_t launch(const AttnArgs& a, cudaStream_t st) {
  using L = Lay<D>;
  static_assert(kWarps * L::WARP >= kWarps * 16 * D * 4 || HL, "the sums must fit the stages");
  auto* fn = paged_attention_kernel<D, HL>;
  const size_t smem = L::smem(a.c.batch);
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
  if (e != cudaSuccess) return e;
  int per_sm = (int)(228 * 1024 / (smem + 2048));
  const int most = D <= 128 ? kMaxCtasPerSm : 2;
  per_sm = per_sm > most ? most : per_sm < 1 ? 1 : per_sm;
  // no more CTAs than units there may be
  const long long cap = ((long long)a.c.pages_per_seq * a.c.page_size + L::UNIT - 1) / L::UNIT;
  const long long tiles = (long long)a.T * a.G / (HL ? 8 : 16) + a.c.batch;
  const double units = (double)cap * (double)tiles * a.c.n_kv_heads;
  int grid = device_info().sms * per_sm;
  if (units < grid) grid = (int)units;
  e = launch_kernel(fn, grid, 32 * kWarps, smem, st, false, a);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, HL ? 8 : 16);
  cfg.blockDim = dim3(D);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, paged_attention_merge_kernel<D>, a);
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

size_t sf_paged_attention_workspace_bytes(int head_dim) {
  if (head_dim <= 0) return 0;
  const size_t ctas = (size_t)device_info().sms * kMaxCtasPerSm;
  return ctas * (2 * 16 * ((size_t)head_dim + 2) * 4 + 32);
}

int sf_paged_attention(const sf_paged_cache* cache, const void* q, int q_dtype, long long qts, long long qhs, void* out,
                       int out_dtype, float* lse, int H, int T, float scale, int window, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (int rc = check_paged(cache, T)) return rc;
  if (q_dtype < 0 || q_dtype > 2 || out_dtype < 0 || out_dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (H < 1 || H % cache->n_kv_heads) return fail(SF_ERR_SHAPE, "H must be a positive multiple of n_kv_heads");
  if (T == 0) return SF_OK;
  if (!q || !out || !workspace) return fail(SF_ERR_NULL, "null pointer argument");
  const int D = cache->head_dim;
  const size_t need = sf_paged_attention_workspace_bytes(D);
  if (workspace_bytes < need) return fail(SF_ERR_SHAPE, "workspace too small: need %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(SF_ERR_ALIGN, "workspace must be 16-byte aligned");
  AttnArgs a{};
  a.c = *cache; a.q = q; a.qts = qts; a.qhs = qhs; a.out = out; a.lse = lse;
  a.desc = static_cast<int*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (size_t)device_info().sms * kMaxCtasPerSm * 32);
  a.H = H; a.T = T; a.G = H / cache->n_kv_heads; a.q_dtype = q_dtype; a.out_dtype = out_dtype; a.window = window;
  a.lg_page = __builtin_ctz((unsigned)cache->page_size);
  a.scale = scale;
  if ((long long)T * a.G > 0x7fffffffll) return fail(SF_ERR_UNSUPPORTED, "too many query rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // 8 rows in two parts when a sequence has no more rows, or for fp32 queries, which one fp16 part cannot hold
  const bool hl = q_dtype == SF_F32 || (!cache->starts && (long long)(T / cache->batch) * a.G <= 8) || (T == 1 && a.G <= 8);
  const auto go = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    return hl ? launch<DD, true>(a, st) : launch<DD, false>(a, st);
  };
  const cudaError_t e = D == 64    ? go(std::integral_constant<int, 64>())
                        : D == 96  ? go(std::integral_constant<int, 96>())
                        : D == 128 ? go(std::integral_constant<int, 128>())
                                   : go(std::integral_constant<int, 256>());
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention_kernel launch");
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return SF_OK;
}

}  // extern "C"
