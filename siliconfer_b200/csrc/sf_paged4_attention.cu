// sf_paged4_attention.cu -- attention over the pages of a 4-bit cache.
//
//   p_j = softmax_j(scale * q . k_j),  out = sum_j p_j v_j,  element = (code - 8) * scale of its vector's quarter
//
// The softmax keeps a running reference m and sum l of e^(score - m): keys in order, out and l are multiplied by
// e^(m - m') when the reference moves to m'.  Parts of a row's keys, a warp's, a CTA's, merge by the same rule.  m is a
// largest score plus the logarithm of its value vector's largest scale; it moves only when a key would exceed it by a
// factor of 2, so that a weight times a scale is bounded and most keys need no reduction over the lanes.  Scales below 2^-60
// count as 2^-60 there, or l would pass fp32's range: their weights, which stay in fp16, lose digits.
//
// One row of a kv head's group is one (new token, query head); a tile has 8 rows, so that a group reads its keys once.
// Both products are mma.sync m16n8k16 in fp16 with the codes as the larger operand and the 8 rows as columns:
//  * S^T[key, row] = K Q^T: 16 keys are the MMA's rows; each quarter of the head has sums of its own, which are added
//    times the key's scale in fp32.  A pair of codes becomes the numbers n - 8 at one mask and one sum.  (As they stand, n
//    in a number's lowest bits, less 8 times the sum of the queries, they save the sum, 2 % of the time, but the tensor cores
//    align such subnormals without their leading zeros: 2^-17 of the largest product is lost, 1e-3 of a log-sum where a few
//    elements of a query stand out.)  A query row is brought to at most 2^14 by a power of two; fp16 then holds a bf16 or fp16
//    row as it is, and two parts an fp32 row.
//  * out^T[d, row] += V^T P^T: a quarter's weights are the softmax's times the key's scale of that quarter, codes the numbers
//    n - 8.  Weights are fp16 numbers, 2^-12 of each at most, where queries and outputs have 16 bits: less than the output's
//    own rounding for bf16, as much for fp16, where two parts take 0.1 more of the time.  With fp32 among the types: two
//    parts, 22 bits.
//
// A warp takes its keys by itself: 32 at a time by bulk copies into a ring of its own, which brings a page's rows as they
// lie, and no warp waits for another before the end of a part.  Measured in a graph, 64 query and 8 kv heads of 128, 16 x 8192
// keys 54 us (2.8 TB/s), one sequence of 131072 with 32 query heads 58; 32 heads of their own, 64 sequences of up to 4096
// keys 222 (3.0 TB/s).  What bounds it: three warps a scheduler, each one chain of load, mask, product, exponential and
// product, some 440 instructions for 16 keys.  At 16 x 8192 issue slots are 58 % and integer units 49 % in use, DRAM 35 %; of
// the time from one instruction of a warp to the next 0.25 is fixed latency, 0.21 its turn, 0.16 loads, 0.15 the others' turn.
// On the way, 16 x 8192 and 64 x 4096 keys in us, keys' codes as subnormals: copies by each lane, 16 keys at a time, 128
// registers and 4 CTAs an SM 71 and 289; by bulk 65 and 261; queries in shared memory 60 and 235; 32 keys at a time, 168
// registers and 3 CTAs 53 and 241, and with fp16 weights in one part for fp16 queries 217; at 128 registers 60 and 207.
//
// Long runs of 16-bit queries with 16-bit outputs go to the kernel of sf_paged4_prompt.h.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_paged4.h"
#include "sf_paged_work.h"
#include "sf_q4_internal.h"
#include "sf_tcgen05.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_paged4)
extern std::atomic<long long> g_launches;

namespace {

constexpr int kWarps = 4, kThreads = 32 * kWarps, kBlock = 16, kStep = 32;   // keys of an MMA, and of a warp's copy
constexpr unsigned kErrCopy = 1u << 17;
constexpr int kCtas = 3;             // of an SM, head_dim up to 128
constexpr float kTopLog = 13.f;      // log2 of a weight times its scale, at most one above it

struct Attn4Args : AttnArgs {
  const __nv_bfloat16 *ks, *vs;      // [pages, n_kv_heads, page_size, 4]
};

__device__ __forceinline__ void mma16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma16_first(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ void mma8(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t b0) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5}, {%6}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(b0));
}
// an 8 x 8 matrix of 16-bit elements, transposed over the warp
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ uint32_t half2_bits(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 half2_floats(uint32_t b) { return __half22float2(*reinterpret_cast<const __half2*>(&b)); }
__device__ __forceinline__ uint32_t add_half2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("add.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
// quarter C's pair of codes of a word, less 8, times 1 or 16: the lowest bits of 1024 + n or 1024 + 16 n; magic is 0x64006400, in a register
template <int C>
__device__ __forceinline__ uint32_t centred(uint32_t w, uint32_t magic) {
  uint32_t x;
  asm("lop3.b32 %0, %1, %2, %3, 0xea;" : "=r"(x) : "r"(C >= 2 ? w >> 8 : w), "n"(C % 2 ? 0x00f000f0u : 0x000f000fu), "r"(magic));
  return add_half2(x, C % 2 ? 0xe480e480u : 0xe408e408u);
}
// four bf16 scales
__device__ __forceinline__ void scales_of(uint2 u, float (&s)[4]) {
  s[0] = __uint_as_float(u.x << 16), s[1] = __uint_as_float(u.x & 0xffff0000u);
  s[2] = __uint_as_float(u.y << 16), s[3] = __uint_as_float(u.y & 0xffff0000u);
}
// the largest of four scales that are not negative, NaN above all numbers
__device__ __forceinline__ float top_scale(uint2 u) {
  const uint32_t m = __vmaxu2(u.x, u.y);
  return __uint_as_float(max(m << 16, m & 0xffff0000u));
}
__device__ __forceinline__ float at_most(float x, float most) { return x > most ? most : x; }   // a NaN stays one
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* p, uint32_t (&w)[N]) {
  if constexpr (N % 4 == 0) {
#pragma unroll
    for (int c = 0; c < N; c += 4) {
      const uint4 u = *reinterpret_cast<const uint4*>(p + 4 * c);
      w[c] = u.x, w[c + 1] = u.y, w[c + 2] = u.z, w[c + 3] = u.w;
    }
  } else if constexpr (N % 2 == 0) {
#pragma unroll
    for (int c = 0; c < N; c += 2) {
      const uint2 u = *reinterpret_cast<const uint2*>(p + 4 * c);
      w[c] = u.x, w[c + 1] = u.y;
    }
  } else {
#pragma unroll
    for (int c = 0; c < N; ++c) w[c] = *reinterpret_cast<const uint32_t*>(p + 4 * c);
  }
}

// A warp's copy is kStep keys as they lie in their pages: rows of D / 2 bytes of codes, and of 8 bytes of scales.  A lane
// (g = lane / 4, t = lane % 4) reads KW words of two keys from word t * KW on, and the VW words of four values that lane
// group g turns into rows of V^T.  An MMA's row m is the copy's row m ^ (m / 2 % 2): at D = 128 the rows that a phase of
// loads touches lie in both halves of the banks then, for the keys' loads and for the values'.
template <int D>
struct Lay4 {
  static constexpr int Q = D / 4, WORDS = D / 8, ROW = D / 2, KW = WORDS / 4, VW = (WORDS + 7) / 8;
  static constexpr int STAGES = D == 64 ? 3 : 2;
  static constexpr uint32_t K0 = 0, V0 = kStep * ROW, KS0 = 2 * V0, VS0 = KS0 + kStep * 8, STAGE = VS0 + kStep * 8;
  static constexpr uint32_t RING = kWarps * STAGES * STAGE, JOIN = kWarps * 8 * (D + 4) * 4;
  static constexpr uint32_t INFO = RING > JOIN ? RING : JOIN;
  static constexpr size_t smem(int batch) { return INFO + (size_t)batch * sizeof(SeqInfo); }
  // the word that lane group g holds in set s
  __device__ static __forceinline__ int word(int s, int g) { return D == 96 ? 8 * s + g : g * VW + s; }
};

template <int D, int QP, int PP>
__global__ void __launch_bounds__(kThreads, D <= 128 ? kCtas : 2) paged4_attention_kernel(const __grid_constant__ Attn4Args a, int q_pairs) {
  using L = Lay4<D>;
  constexpr int RT = 8, KW = L::KW, VW = L::VW, Q = L::Q, ST = L::STAGES;
  extern __shared__ __align__(128) uint8_t mem[];
  __shared__ long long wsum[kWarps];
  __shared__ float wm[kWarps][RT], wl[kWarps][RT];
  __shared__ __align__(8) uint64_t bars[kWarps][ST];
  __shared__ int abort_word;
  __shared__ __align__(16) uint32_t q_sm[4][QP][32 * KW];   // queries: lane's words of quarter c, part
  __shared__ uint32_t row_top[kWarps][RT];
  volatile int* abort_flag = &abort_word;
  SeqInfo* info = reinterpret_cast<SeqInfo*>(mem + L::INFO);
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3, warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0);
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w)
      for (int i = 0; i < ST; ++i) bar_init(smem_u32(&bars[w][i]), 1);
    abort_word = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  griddep_wait();

  // ---- the batch's units, and this CTA's share ----
  const int B = a.c.batch, Hkv = a.c.n_kv_heads, page_size = a.c.page_size;
  const int rows0 = first_row(a.c, a.T, 0), rows1 = first_row(a.c, a.T, B);
  long long total = 0;
  int bad = 0;
  for (int at = 0; at < B; at += kThreads) {
    const int b = at + threadIdx.x;
    long long u = 0;
    int len = 0, n = 0, off = 0;
    if (b < B) {
      const int r0 = first_row(a.c, a.T, b), r1 = first_row(a.c, a.T, b + 1);
      len = a.c.seq_lens[b];
      n = r1 - r0;
      if (r0 < 0 || n < 0 || r1 > a.T) {
        n = 0;
        off = 1;
        atomicOr(&g_dev_error, kErrIndex);
      }
      if (!len_ok(a.c, len)) {
        len = 0;
        atomicOr(&g_dev_error, kErrIndex);
      }
      const int tiles = (int)(((long long)n * a.G + RT - 1) / RT);
      u = (long long)tiles * Hkv * max(1, (len - keys_from(a, len, n) + UNIT - 1) / UNIT);
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
    bad |= __syncthreads_or(off);
  }
  if (bad) total = 0;
  clear_rows(a, bad ? 0 : rows0, bad ? 0 : rows1);
  const long long cta = blockIdx.x;
  const Shares shares(total, a.resident, (int)gridDim.x);
  if (threadIdx.x == 0) a.desc[8 * cta] = 0;
  long long u = 0, u_end = 0;
  int b = 0;
  if (cta < shares.ctas()) {
    u = shares.begin(cta);
    u_end = shares.begin(cta + 1);
    for (int lo = 0, hi = B; hi - lo > 1;) {
      const int mid = (lo + hi) >> 1;
      if (info[mid].first <= u) lo = mid;
      else hi = mid;
      b = lo;
    }
  }

  // This lane's copy: keys' codes, values' codes, keys' scales or values' scales (lane % 4) of box lane / 4 of a step.
  const int box = min(page_size, kStep), boxes = kStep / box, my_box = lane >> 2;
  const uint32_t row_bytes = t < 2 ? L::ROW : 8, page_bytes = (uint32_t)(Hkv * page_size) * row_bytes;
  const uint8_t* const src = t == 0   ? a.c.k_codes
                             : t == 1 ? a.c.v_codes
                                      : reinterpret_cast<const uint8_t*>(t == 2 ? a.ks : a.vs);
  const uint32_t ring = smem_u32(mem) + warp * ST * L::STAGE, bar0 = smem_u32(&bars[warp][0]),
                 dst = ring + (t == 0 ? L::K0 : t == 1 ? L::V0 : t == 2 ? L::KS0 : L::VS0) + my_box * box * row_bytes;
  const uint32_t k_row = (g ^ (g >> 1 & 1)) * L::ROW + t * KW * 4, s_row = (g ^ (g >> 1 & 1)) * 8;
  uint32_t slot = 0, phase = 0;   // of this warp's next step
  uint32_t magic;
  asm volatile("mov.b32 %0, 0x64006400;" : "=r"(magic));
  bool ok = true;

  while (u < u_end) {
    const Part p = part_at<RT>(a, info, u, u_end, b);
    // ---- copies: this warp takes the steps at p.ta + kStep * (warp + kWarps * i) ----
    const int* pages = a.c.block_table + (size_t)p.b * a.c.pages_per_seq;
    const uint32_t head = (uint32_t)(p.kvh * page_size);
    int copy_key = p.ta + kStep * warp + my_box * box;   // first key of this lane's box of the next copy
    // Page of the box at `key`, -1 where there is none; a page that ends before the first key in sight may have been given up.
    const auto page_of = [&](int key) {
      int page = -1;
      if (my_box < boxes && key < p.tb && key + box > p.tile_lo) {
        page = __ldg(pages + (key >> a.lg_page));
        if ((unsigned)page >= (unsigned)a.c.num_pages) {
          if (t == 0) atomicOr(&g_dev_error, kErrIndex);
          page = -1;
        }
      }
      return page;
    };
    int page = page_of(copy_key);
    uint32_t there = 0;   // bits 2 s and 2 s + 1: the halves of the step in slot s that have a page
    const auto copy = [&](uint32_t s) {
      if (copy_key - my_box * box >= p.tb) return;
      const int now = page, key = copy_key;
      copy_key += kStep * kWarps;
      page = page_of(copy_key);
      const unsigned have = __ballot_sync(0xffffffffu, now >= 0);
      there = (there & ~(3u << (2 * s))) | (boxes == 1 ? (have & 1) * 3 : (have & 1) | (have >> 3 & 2)) << (2 * s);
      if (lane == 0) bar_expect_tx(bar0 + 8 * s, __popc(have) / 4 * box * (uint32_t)(D + 16));
      __syncwarp();
      if (now >= 0) {
        const uint8_t* from = src + (unsigned long long)(unsigned)now * page_bytes + (head + (key & (page_size - 1))) * row_bytes;
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst + s * L::STAGE),
                     "l"(from), "r"(box * row_bytes), "r"(bar0 + 8 * s)
                     : "memory");
      }
    };
    if (ok) {
      uint32_t s = slot;
#pragma unroll
      for (int i = 0; i < ST; ++i) {
        copy(s);
        s = s + 1 == ST ? 0 : s + 1;
      }
    }

    // ---- queries: warp c cuts quarter c of the 8 rows into the second operand's registers, for all warps ----
    static_assert(kWarps == 4, "a quarter for each warp");
    float f[2];
    {
      const int row = p.row0 + g;
      const bool real = row <= p.last_row;
      const long long qo = (long long)(p.r_first + row / a.G) * a.qts + (long long)(p.kvh * a.G + row % a.G) * a.qhs + warp * Q + 2 * t * KW;
      float v[2 * KW];
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 2 * KW; e += 2) {
        if (!real) {
          v[e] = v[e + 1] = 0.f;
        } else if (q_pairs && a.q_dtype == SF_BF16) {
          const uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const __nv_bfloat16*>(a.q) + qo + e);
          v[e] = __uint_as_float(w << 16);
          v[e + 1] = __uint_as_float(w & 0xffff0000u);
        } else if (q_pairs && a.q_dtype == SF_F16) {
          const float2 w = half2_floats(*reinterpret_cast<const uint32_t*>(static_cast<const __half*>(a.q) + qo + e));
          v[e] = w.x;
          v[e + 1] = w.y;
        } else {
          v[e] = load_q(a, qo + e);
          v[e + 1] = load_q(a, qo + e + 1);
        }
        top = max(top, max(__float_as_uint(v[e]) & 0x7fffffffu, __float_as_uint(v[e + 1]) & 0x7fffffffu));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      if (t == 0) row_top[warp][g] = top;
      __syncthreads();
      const auto top_of = [&](int r) { return max(max(row_top[0][r], row_top[1][r]), max(row_top[2][r], row_top[3][r])); };
      // the row's largest value to [2^13, 2^14) by a power of two
      const auto exponent = [](uint32_t x) { return min(max((int)(x >> 23) - 140, -126), 113); };
      const float down = __int_as_float((127 - exponent(top_of(g))) << 23) * (warp % 2 ? 0.0625f : 1.f);   // odd quarters' codes lie four bits higher
#pragma unroll
      for (int i = 0; i < KW; ++i) {
        float x = v[2 * i] * down, y = v[2 * i + 1] * down;
#pragma unroll
        for (int part = 0; part < QP; ++part) {
          const uint32_t w = half2_bits(x, y);
          const float2 h = half2_floats(w);
          q_sm[warp][part][lane * KW + i] = w;
          x -= h.x;
          y -= h.y;
        }
      }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        // an infinity or a NaN: the row is NaN
        const uint32_t x = top_of(2 * t + e);
        f[e] = x >= 0x7f800000u ? __int_as_float(0x7fffffff)
                                : __int_as_float((127 + exponent(x)) << 23) * (a.scale * kLog2e);
      }
      __syncthreads();
    }

    float nm[2] = {0.f, 0.f};   // minus the reference of columns 2t and 2t + 1
    float l[2] = {0.f, 0.f};    // their sums
    bool fresh = true;          // the warp has rows without a reference
    bool none[2] = {true, true};   // no key yet
    float o[VW][4][4];          // sums: rows 2 * word (+ 1) of quarter c, columns 2t, 2t + 1
#pragma unroll
    for (int s = 0; s < VW; ++s)
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[s][c][e] = 0.f;

    // NB times 16 keys from k0 on; edge: not every row sees all of them
    const auto block = [&](auto edge, auto nb, const uint8_t* codes_at, const uint8_t* scales_at, int k0) {
      constexpr bool EDGE = decltype(edge)::value;
      constexpr int NB = decltype(nb)::value;
      // ---- scores ----
      float y[NB][4];   // keys g, g, g + 8, g + 8 (in the copy's order) of each 16; columns 2t, 2t + 1
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        uint32_t w[2][KW];
#pragma unroll
        for (int r = 0; r < 2; ++r) load_words<KW>(codes_at + L::K0 + k_row + (n * kBlock + r * 8) * L::ROW, w[r]);
        float ks[2][4];
#pragma unroll
        for (int r = 0; r < 2; ++r) scales_of(*reinterpret_cast<const uint2*>(scales_at + L::KS0 + s_row + (n * kBlock + r * 8) * 8), ks[r]);
        const auto quarter = [&](auto cc) {
          constexpr int C = decltype(cc)::value;
          float s[4];
          uint32_t q[QP][KW];
#pragma unroll
          for (int part = 0; part < QP; ++part) load_words<KW>(reinterpret_cast<const uint8_t*>(&q_sm[C][part][lane * KW]), q[part]);
          const auto codes = [&](uint32_t x) { return centred<C>(x, magic); };
#pragma unroll
          for (int j = 0; j + 1 < KW; j += 2) {
            const uint32_t a0 = codes(w[0][j]), a1 = codes(w[1][j]), a2 = codes(w[0][j + 1]), a3 = codes(w[1][j + 1]);
#pragma unroll
            for (int part = 0; part < QP; ++part) {
              if (j + part == 0) mma16_first(s, a0, a1, a2, a3, q[part][j], q[part][j + 1]);
              else mma16(s, a0, a1, a2, a3, q[part][j], q[part][j + 1]);
            }
          }
          if constexpr (KW % 2) {
#pragma unroll
            for (int part = 0; part < QP; ++part) mma8(s, codes(w[0][KW - 1]), codes(w[1][KW - 1]), q[part][KW - 1]);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) y[n][e] = C == 0 ? s[e] * ks[e >> 1][C] : fmaf(s[e], ks[e >> 1][C], y[n][e]);
        };
        quarter(std::integral_constant<int, 0>());
        quarter(std::integral_constant<int, 1>());
        quarter(std::integral_constant<int, 2>());
        quarter(std::integral_constant<int, 3>());
      }
      uint2 vs[NB][2];
      float lv[NB][2], over = -INFINITY;
      bool hidden[NB][4] = {};
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          y[n][e] = fmaf(y[n][e], f[e & 1], nm[e & 1]);
          if constexpr (EDGE) {
            const int key = k0 + n * kBlock + (g ^ (g >> 1 & 1)) + 8 * (e >> 1), pos = p.pos0 + (p.row0 + 2 * t + (e & 1)) / a.G;
            hidden[n][e] = key >= p.tb || key > pos || (a.window > 0 && key <= pos - a.window);
            if (hidden[n][e]) y[n][e] = -INFINITY;
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          vs[n][r] = *reinterpret_cast<const uint2*>(scales_at + L::VS0 + s_row + (n * kBlock + r * 8) * 8);
          lv[n][r] = fmaxf(lg2(top_scale(vs[n][r])), -60.f);
          over = fmaxf(over, fmaxf(y[n][2 * r], y[n][2 * r + 1]) + lv[n][r]);
        }
      }
      // ---- the reference, if a key exceeds it by more than a factor of 2 ----
      if (__any_sync(0xffffffffu, over > kTopLog + 1.f) || fresh) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          float top = -INFINITY;
#pragma unroll
          for (int n = 0; n < NB; ++n) top = fmaxf(top, fmaxf(y[n][e] + lv[n][0], y[n][e + 2] + lv[n][1]));
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          if (none[e] && top == -INFINITY) continue;   // the row has seen no key
          // below what the roundings of a large score may add, so that the largest key's weight is no less than 2^kTopLog
          const float to = fmaf(fabsf(nm[e]) + fabsf(top), -0x1p-22f, top - kTopLog);
          const float up = none[e] || !(to <= 0.f) ? to : 0.f, c = none[e] ? 1.f : ex2(-up);   // an infinite score: NaN
          none[e] = false;
          nm[e] -= up;
#pragma unroll
          for (int n = 0; n < NB; ++n) {   // so that it may be more than a weight has room for: it is limited
            y[n][e] = at_most(y[n][e] - up, kTopLog + 2.f - lv[n][0]);
            y[n][e + 2] = at_most(y[n][e + 2] - up, kTopLog + 2.f - lv[n][1]);
          }
          l[e] *= c;
#pragma unroll
          for (int s = 0; s < VW; ++s)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              o[s][q][e] *= c;
              o[s][q][e + 2] *= c;
            }
        }
        fresh = __any_sync(0xffffffffu, none[0] || none[1]);
      }
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        // ---- weights, times each quarter's scale, as the second operand ----
        float pw[4], sv[2][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) pw[e] = ex2(y[n][e]);
        l[0] += pw[0] + pw[2];
        l[1] += pw[1] + pw[3];
        uint32_t pf[4][PP][2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          scales_of(vs[n][r], sv[r]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            float x = pw[2 * r] * sv[r][c], z = pw[2 * r + 1] * sv[r][c];
            if constexpr (EDGE) {   // 0 times a NaN scale is not 0
              if (hidden[n][2 * r]) x = 0.f;
              if (hidden[n][2 * r + 1]) z = 0.f;
            }
#pragma unroll
            for (int part = 0; part < PP; ++part) {
              const uint32_t h = half2_bits(x, z);
              pf[c][part][r] = transpose8(h);
              if (part + 1 < PP) {
                const float2 w = half2_floats(h);
                x -= w.x;
                z -= w.y;
              }
            }
          }
        }
        // ---- sums: row m of the scores, and so of the weights, is the copy's row m ^ (m / 2 % 2) ----
        uint32_t w[4][VW];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint8_t* row = codes_at + L::V0 + (n * kBlock + ((2 * t + (e & 1)) ^ (t & 1)) + (e >> 1) * 8) * L::ROW;
          if constexpr (D == 96) {
            w[e][0] = *reinterpret_cast<const uint32_t*>(row + 4 * g);
            w[e][1] = g < 4 ? *reinterpret_cast<const uint32_t*>(row + 32 + 4 * g) : 0u;
          } else {
            load_words<VW>(row + 4 * VW * g, w[e]);
          }
        }
#pragma unroll
        for (int s = 0; s < VW; ++s) {
          // both tokens' half-words of a place side by side
          const uint32_t lo0 = __byte_perm(w[0][s], w[1][s], 0x5410), hi0 = __byte_perm(w[0][s], w[1][s], 0x7632),
                         lo1 = __byte_perm(w[2][s], w[3][s], 0x5410), hi1 = __byte_perm(w[2][s], w[3][s], 0x7632);
          const auto quarter = [&](auto cc) {
            constexpr int C = decltype(cc)::value;
            const uint32_t a0 = centred<C>(lo0, magic), a1 = centred<C>(hi0, magic), a2 = centred<C>(lo1, magic),
                           a3 = centred<C>(hi1, magic);
#pragma unroll
            for (int part = 0; part < PP; ++part) mma16(o[s][C], a0, a1, a2, a3, pf[C][part][0], pf[C][part][1]);
          };
          quarter(std::integral_constant<int, 0>());
          quarter(std::integral_constant<int, 1>());
          quarter(std::integral_constant<int, 2>());
          quarter(std::integral_constant<int, 3>());
        }
      }
    };

    const int whole_lo = p.all_lo, whole_hi = min(p.all_hi, p.tb);
#pragma unroll 1
    for (int k0 = p.ta + kStep * warp; k0 < p.tb; k0 += kStep * kWarps) {
      ok = ok && __all_sync(0xffffffffu, bar_wait(bar0 + 8 * slot, phase, kErrCopy, abort_flag));
      if (!ok) break;
      const uint32_t have = there >> (2 * slot) & 3;
      const uint8_t* st = mem + (warp * ST + slot) * L::STAGE;
      if (k0 >= whole_lo && k0 + kStep <= whole_hi && have == 3) {
        block(std::false_type(), std::integral_constant<int, 2>(), st, st, k0);
      } else {
#pragma unroll 1
        for (int half = 0; half < 2; ++half)
          if ((have >> half & 1) && k0 + kBlock * half < p.tb)
            block(std::true_type(), std::integral_constant<int, 1>(), st + half * (kBlock * L::ROW), st + half * (kBlock * 8), k0 + kBlock * half);
      }
      __syncwarp();   // the step's rows have been read
      copy(slot);
      if (++slot == ST) slot = 0, phase ^= 1;
    }

    // ---- the warps' parts ----
#pragma unroll
    for (int e = 0; e < 2; ++e) {
#pragma unroll
      for (int x = 4; x < 32; x <<= 1) l[e] += __shfl_xor_sync(0xffffffffu, l[e], x);
      if (g == 0) {
        wm[warp][2 * t + e] = none[e] ? kNone : -nm[e];
        wl[warp][2 * t + e] = l[e];
      }
    }
    __syncthreads();   // the rings are free, too
    float* join = reinterpret_cast<float*>(mem);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int col = 2 * t + e;
      const float M = fmaxf(fmaxf(wm[0][col], wm[1][col]), fmaxf(wm[2][col], wm[3][col]));
      const float c = ex2(wm[warp][col] - M);
      float* to = join + (warp * RT + col) * (D + 4);
#pragma unroll
      for (int s = 0; s < VW; ++s) {
        const int word = L::word(s, g);
        if (word >= L::WORDS) continue;
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float2*>(to + q * Q + 2 * word) =
              make_float2(o[s][q][e] * c * (q % 2 ? 0.0625f : 1.f), o[s][q][e + 2] * c * (q % 2 ? 0.0625f : 1.f));
      }
    }
    __syncthreads();
    const bool begins = u == p.seg0, ends = p.u1 == p.seg1;
    float* part = a.part + ((size_t)cta * 2 + (begins ? 1 : 0)) * kMaxRows * (D + 2);
    for (int x = threadIdx.x; x < RT * D; x += kThreads) {
      const int r = x / D, d = x % D, row = p.row0 + r;
      if (row > p.last_row) break;
      const float M = fmaxf(fmaxf(wm[0][r], wm[1][r]), fmaxf(wm[2][r], wm[3][r]));
      float A = 0.f, Ls = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        A += join[(w * RT + r) * (D + 4) + d];
        Ls += wl[w][r] * ex2(wm[w][r] - M);
      }
      const size_t th = (size_t)(p.r_first + row / a.G) * a.H + p.kvh * a.G + row % a.G;
      if (begins && ends) store_out(a, th * D + d, Ls == 0.f ? 0.f : A / Ls);
      else part[r * D + d] = A;
      if (d == 0) {
        if (!(begins && ends)) {
          part[RT * D + 2 * r] = M;
          part[RT * D + 2 * r + 1] = Ls;
        } else if (a.lse) {
          a.lse[th] = Ls == 0.f ? -INFINITY : M * kLn2 + logf(Ls);
        }
      }
    }
    if (begins && !ends && threadIdx.x == 0) {
      // CTAs of the tile's parts: this one to the one that holds its last unit
      int* dsc = a.desc + 8 * cta;
      dsc[0] = (int)(shares.holder(p.seg1 - 1) - cta + 1);
      dsc[1] = p.r_first;
      dsc[2] = p.kvh;
      dsc[3] = p.row0;
      dsc[4] = p.last_row;
    }
    // the join's place is the next part's rings, which copies write
    fence_async_smem();
    __syncthreads();
    u = p.u1;
  }
  // after an expired wait the copies under way are not counted any more: give them time
  if (!ok) {
    const long long t0 = clock64();
    while (clock64() - t0 < kWaitCycles / 64) {
    }
  }
  griddep_launch_dependents();   // not before: the merge's blocks would wait in the place of the next call's
}

// One block for each (CTA that began a divided tile, row of it): GROUPS groups of threads take the parts in turn, D columns
// each, and are added in order.  A tile of 55 parts (131072 keys) takes 6 us less in 4 groups than in one.
template <int D, int GROUPS>
__global__ void __launch_bounds__(GROUPS * D) paged4_merge_kernel(const AttnArgs a) {
  constexpr int RT = 8;
  __shared__ float sum[GROUPS][D], lsum[GROUPS];
  griddep_wait();
  const int* dsc = a.desc + 8 * blockIdx.x;
  const int parts = dsc[0], row = blockIdx.y, q_row = dsc[3] + row, grp = threadIdx.x / D, d = threadIdx.x % D;
  if (parts == 0 || q_row > dsc[4]) return;
  const auto part = [&](int i) {
    return a.part + ((size_t)(blockIdx.x + i) * 2 + (i == 0 ? 1 : 0)) * kMaxRows * (D + 2);
  };
  float M = kNone;
  for (int i = 0; i < parts; ++i) M = fmaxf(M, part(i)[RT * D + 2 * row]);
  float A = 0.f, Ls = 0.f;
#pragma unroll 4
  for (int i = grp; i < parts; i += GROUPS) {
    const float* p = part(i);
    const float c = ex2(p[RT * D + 2 * row] - M);
    A += p[row * D + d] * c;
    Ls += p[RT * D + 2 * row + 1] * c;
  }
  sum[grp][d] = A;
  if (d == 0) lsum[grp] = Ls;
  __syncthreads();
  if (grp > 0) return;
#pragma unroll
  for (int i = 1; i < GROUPS; ++i) {
    A += sum[i][d];
    Ls += lsum[i];
  }
  const size_t th = (size_t)(dsc[1] + q_row / a.G) * a.H + dsc[2] * a.G + q_row % a.G;
  store_out(a, th * D + d, Ls == 0.f ? 0.f : A / Ls);
  if (d == 0 && a.lse) a.lse[th] = Ls == 0.f ? -INFINITY : M * kLn2 + logf(Ls);
}

template <int D, int QP, int PP>
int launch4(Attn4Args a, cudaStream_t st) {
  using L = Lay4<D>;
  const sf_paged_cache& c = a.c;
  auto* fn = paged4_attention_kernel<D, QP, PP>;
  const size_t smem = L::smem(c.batch);
  // the limit is the process's: the same for calls of every batch, or another thread's could lower it before this launch
  static_assert(L::smem(kMaxBatch) + 4 * QP * 128 * L::KW + 2048 <= kBlockSmem, "shared memory plan");
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem(kMaxBatch));
  if (e != cudaSuccess) return cuda_fail(e, "paged4_attention_kernel shared memory");
  int per_sm = (int)(228 * 1024 / (smem + 4 * QP * 128 * L::KW + 2048));
  const int most = D <= 128 ? kCtas : 2;
  if (per_sm > most) per_sm = most;
  if (per_sm < 1) per_sm = 1;
  // no more CTAs than units there may be
  const double cap = ((double)c.pages_per_seq * c.page_size + UNIT - 1) / UNIT;
  const double units = cap * ((double)a.T * a.G / 8 + c.batch) * c.n_kv_heads;
  a.resident = device_info().sms * per_sm;
  int grid = 2 * a.resident;
  if (units < (double)kLong * a.resident) grid = units < a.resident ? (int)units : a.resident;
  const size_t size = a.q_dtype == SF_F32 ? 4 : 2;
  const int pairs = reinterpret_cast<uintptr_t>(a.q) % (2 * size) == 0 && a.qts % 2 == 0 && a.qhs % 2 == 0;
  e = launch_kernel(fn, grid, kThreads, smem, st, true, a, pairs);
  if (e != cudaSuccess) return cuda_fail(e, "paged4_attention_kernel launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, 8);
  // many parts of each tile where the tiles are few
  const double tiles = ((double)a.T * a.G / 8 + c.batch) * c.n_kv_heads;
  const bool many = tiles * 8 <= a.resident;
  constexpr int GROUPS = 512 / D;
  cfg.blockDim = dim3(many ? GROUPS * D : D);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, many ? paged4_merge_kernel<D, GROUPS> : paged4_merge_kernel<D, 1>, static_cast<const AttnArgs&>(a));
  if (e != cudaSuccess) return cuda_fail(e, "paged4_merge_kernel launch");
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return SF_OK;
}

constexpr int kMaxCtasPerSm = kCtas;

#include "sf_paged4_prompt.h"

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

size_t sf_paged4_attention_workspace_bytes(int head_dim) {
  if (head_dim <= 0) return 0;
  const size_t ctas = (size_t)device_info().sms * kMaxCtasPerSm * 2;
  return ctas * (2 * kMaxRows * ((size_t)head_dim + 2) * 4 + 32);
}

int sf_paged4_attention(const sf_paged4_cache* cache, const void* q, int q_dtype, long long qts, long long qhs, void* out,
                        int out_dtype, float* lse, int H, int T, float scale, int window, void* workspace,
                        size_t workspace_bytes, void* stream) {
  Attn4Args a{};
  if (int rc = check_paged4(cache, T, a.c)) return rc;
  if (q_dtype < 0 || q_dtype > 2 || out_dtype < 0 || out_dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (H < 1 || H % cache->n_kv_heads) return fail(SF_ERR_SHAPE, "H must be a positive multiple of n_kv_heads");
  if (T == 0) return SF_OK;
  if (!q || !out || !workspace) return fail(SF_ERR_NULL, "null pointer argument");
  const int D = cache->head_dim;
  const size_t need = sf_paged4_attention_workspace_bytes(D);
  if (workspace_bytes < need) return fail(SF_ERR_SHAPE, "workspace too small: need %zu bytes", need);
  if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(SF_ERR_ALIGN, "workspace must be 16-byte aligned");
  a.q = q; a.qts = qts; a.qhs = qhs; a.out = out; a.lse = lse;
  a.ks = static_cast<const __nv_bfloat16*>(cache->k_scales);
  a.vs = static_cast<const __nv_bfloat16*>(cache->v_scales);
  a.desc = static_cast<int*>(workspace);
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (size_t)device_info().sms * kMaxCtasPerSm * 2 * 32);
  a.H = H; a.T = T; a.G = H / cache->n_kv_heads; a.q_dtype = q_dtype; a.out_dtype = out_dtype;
  a.window = window < (long long)cache->pages_per_seq * cache->page_size ? window : 0;   // a wider one hides nothing
  a.lg_page = __builtin_ctz((unsigned)cache->page_size);
  a.scale = scale;
  if ((long long)T * a.G > 0x7fffffffll) return fail(SF_ERR_UNSUPPORTED, "too many query rows");
  if ((long long)cache->n_kv_heads * cache->page_size * D > 0x7fffffffll)
    return fail(SF_ERR_UNSUPPORTED, "a page of all kv heads has more than 2^31 - 1 elements");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool fine = q_dtype == SF_F32 || out_dtype == SF_F32;
  // Tiles of 256 rows: an SM takes some 2.8 us for 128 keys of a tile, however many of its rows are in use, and 14 us before
  // and after.  Tiles of 8 rows: all SMs together take 0.5 ns for 128 keys of a row, and 20 us before and after.  So the rows
  // of a round of tiles decide; of the lengths the host knows only the block table's.
  // Measured, 64 query and 8 kv heads, tiles of 256 and of 8 rows, in us.  Head_dim 128: 18 sequences of 8 tokens, 256 keys
  // 20 and 38, 2048 keys 69 and 117, 32768 keys 902 and 1228; 8 such, 2048 keys 58 and 58, 32768 keys 738 and 562; one of 32
  // tokens 21 and 18, 59 and 35, 706 and 293; one of 256, 2048 keys 61 and 183.  Head_dim 64: 8 sequences of 8 tokens, 2048
  // keys 49 and 45, 32768 keys 646 and 431; 16 such, 256 keys 16 and 25, 2048 keys 52 and 77.
  const long long items = ((long long)T * a.G / kPromptRows + cache->batch) * cache->n_kv_heads;
  const int sms = device_info().sms;
  const long long keys = std::min((long long)cache->pages_per_seq * cache->page_size,
                                  a.window > 0 ? (long long)a.window + kPromptRows : LLONG_MAX);
  const long long tiles = std::max(((long long)T * a.G + kPromptRows - 1) / kPromptRows, (long long)cache->batch) * cache->n_kv_heads,
                  rounds = (tiles + sms - 1) / sms, key_tiles = (keys + UNIT - 1) / UNIT;
  const bool many = (double)T * H * (key_tiles + 7) >= 5800.0 * rounds * (key_tiles + 2);
  const bool prompt = !fine && (D == 64 || D == 128) && many && cache->batch <= kPromptBatch && items <= 0x7fffffffll &&
                      reinterpret_cast<uintptr_t>(out) % 16 == 0;
  if (prompt) {
    const bool q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && qts % 8 == 0 && qhs % 8 == 0;
    return D == 64 ? launch_prompt4<64>(a, items, q_vec, st) : launch_prompt4<128>(a, items, q_vec, st);
  }
  const auto go = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    if (q_dtype == SF_F32) return launch4<DD, 2, 2>(a, st);
    return fine ? launch4<DD, 1, 2>(a, st) : launch4<DD, 1, 1>(a, st);
  };
  return D == 64    ? go(std::integral_constant<int, 64>())
         : D == 96  ? go(std::integral_constant<int, 96>())
         : D == 128 ? go(std::integral_constant<int, 128>())
                    : go(std::integral_constant<int, 256>());
}

}  // extern "C"
