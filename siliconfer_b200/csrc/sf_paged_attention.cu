// sf_paged_attention.cu -- attention over the pages of an e4m3 cache on the sm_100a tcgen05 tensor cores.
//
//   p_j = softmax_j(scale * q . k_j),  out = sum_j p_j v_j,  k_j = code * scale of its page and head
//
// The softmax keeps a running reference m and sum l of e^(score - m): keys in order, out and l are multiplied by
// e^(m - m') when the reference moves to m'.  Parts of a row's keys merge by the same rule.  m is a largest score plus
// the logarithm of its page's V scale; it moves only when a key would exceed it by a factor of 2, so that a weight
// times its scale is at most 2 and most tiles of keys need no reduction over the threads.
//
// A call's work is a list of units of 128 keys, for each (sequence, kv head, tile of RT query rows) in turn; a row is
// one (new token, query head of the kv head's group), so that a group reads its keys once.  The list is cut into
// contiguous shares, one per CTA, whatever the sequences' lengths: a CTA finds its place from a prefix sum over the
// batch.  The SMs do not get memory at the same pace (with equal shares they were busy between 0.66 and 0.92 of the
// kernel's time), so the CTAs that are resident at first share 4/5 of a long list, and as many small CTAs that follow
// where an SM is through share the rest.  A CTA that holds all of a tile's units writes the result; the others leave
// their parts in the workspace, which a second kernel merges.
//
// Both products run on the codes as they lie in the cache (kind::f8f6f4), and no code is ever converted:
//  * S^T[key, column] = K Q^T: 128 keys are the MMA's rows.  A query row is scaled by a power of two to at most 256 and
//    cut into e4m3 parts of 4 bits each, 2^4 apart; each part is a column, so its sums are exact on their own and are
//    added, scaled, in fp32.  2 parts hold a bf16 row, 3 an fp16 row, 6 an fp32 row (24 bits; elements far below the
//    row's largest lose what lies under 2^-17, 2^-21 or 2^-33 of it).
//  * out^T[d, column] = V^T P^T: the head's columns are the MMA's rows, V is its transposed operand.  Weights are cut
//    into as many parts as queries: 8, 12 or 24 bits, and no coarser than 2^-21 of the reference for bf16.
// The finer of the queries' and the output's types decides the parts: an fp32 output of bf16 queries has six.  With two, a
// weight is within 2^-8 of itself, which moves a bf16 output by 3e-4 to 9e-4 of its norm; its own rounding does by 1.7e-3.
// A third part costs a decode step of grouped heads up to 12 % (64 sequences of 2000 tokens, 64/8 heads: 73 us, 65 with
// two), tiles of a prompt 44 % (8 x 256 tokens: 1008 and 700 us); six parts take 16 x 8192 tokens 66 us, two 61.
// Both scores and partial sums go to fresh TMEM buffers, two each; a thread is one key for the scores and one column d
// for the sums, which it keeps in registers in fp32.
//
// Long runs of bf16 queries with 16-bit outputs go to the kernel of sf_paged_prompt.h.
//
// Measured in a graph.  Bound by the cache's bytes: 64 sequences of up to 4096 tokens, 32 heads, 204 us, 5.7 TB/s (one call
// after another 205 to 211).  16 sequences of 8192 tokens, 64 query and 8 kv heads of 128, 61 us, 4.4 TB/s: DRAM 54 % and
// issue slots 26 % in use, waits for loads first among the stalls.  Bound by latency: one sequence of 1000 tokens, 12 us,
// of which the merge is 4.
//
// Warps 0-3: softmax and sums.  Warp 4: TMA copies of pages.  Warp 5: MMAs.  Every wait is bounded: on expiry the
// kernel records it in the device error word and raises a flag on which the other roles stop waiting.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_q4_internal.h"
#include "sf_paged.h"
#include "sf_paged_work.h"
#include "sf_tcgen05.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_paged)
extern std::atomic<long long> g_launches;

namespace {

constexpr int kSoftWarps = 4, kProdWarp = 4, kMmaWarp = 5, kThreads = 192;
constexpr int kMaxCtasPerSm = 4;
constexpr float kPScale = 128.f;     // of a weight: at most 256, within e4m3
constexpr unsigned kErrProd = 1u << 17, kErrMma = 1u << 18, kErrSoft = 1u << 19, kErrDrain = 1u << 22;

// Arrives at barrier 1 of the THREADS softmax threads, and says whether any thread's p is true.
template <int THREADS = 128>
__device__ __forceinline__ bool any_of(bool p) {
  int any;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, 1, %2, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
      : "=r"(any)
      : "r"((int)p), "r"(THREADS)
      : "memory");
  return any;
}
// d = a * b + c and d = a + b over rows, two to an instruction
template <int R, typename A, typename B, typename C>
__device__ __forceinline__ void fma_rows(float (&d)[R], A&& a, B&& b, C&& c) {
  if constexpr (R % 2 == 0) {
#pragma unroll
    for (int r = 0; r < R; r += 2) {
      unpack2(fma2(pack2(a(r), a(r + 1)), pack2(b(r), b(r + 1)), pack2(c(r), c(r + 1))), d[r], d[r + 1]);
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) d[r] = fmaf(a(r), b(r), c(r));
  }
}
template <int R, typename A, typename B>
__device__ __forceinline__ void mul_rows(float (&d)[R], A&& a, B&& b) {
  if constexpr (R % 2 == 0) {
#pragma unroll
    for (int r = 0; r < R; r += 2) {
      unpack2(mul2(pack2(a(r), a(r + 1)), pack2(b(r), b(r + 1))), d[r], d[r + 1]);
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) d[r] = a(r) * b(r);
  }
}
template <int R, typename A, typename B>
__device__ __forceinline__ void add_rows(float (&d)[R], A&& a, B&& b) {
  if constexpr (R % 2 == 0) {
#pragma unroll
    for (int r = 0; r < R; r += 2) {
      unpack2(add2(pack2(a(r), a(r + 1)), pack2(b(r), b(r + 1))), d[r], d[r + 1]);
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) d[r] = a(r) + b(r);
  }
}
// four values of at most 448, to e4m3 codes, leaving what they lack, times 16
__device__ __forceinline__ uint32_t take_e4m3(float (&v)[4]) {
  const uint32_t c0 = to_e4m3x2(v[0], v[1]), c1 = to_e4m3x2(v[2], v[3]);
  const __half2_raw h0 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c0, __NV_E4M3),
                    h1 = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)c1, __NV_E4M3);
  const float2 a = __half22float2(__half2(h0)), b = __half22float2(__half2(h1));
  v[0] = (v[0] - a.x) * 16.f;
  v[1] = (v[1] - a.y) * 16.f;
  v[2] = (v[2] - b.x) * 16.f;
  v[3] = (v[3] - b.y) * 16.f;
  return c0 | (c1 << 16);
}

// A tile's rows lie in shared memory as TMA brings them: sub-tiles of INNER bytes a row in the swizzle of that width.
//  K (rows = keys) is a K-major operand: a step of 32 columns is 32 bytes further in the sub-tile, or, where INNER is
//  32, the next sub-tile.  V (rows = keys) is an MN-major operand: a step of 32 keys is 32 rows further, the MMA's
//  128 rows are 128 / INNER sub-tiles, and those beyond the head's columns are whatever lies there, in TMEM lanes
//  that nothing looks at.
//  Q^T: [column][d] in cores of 8 columns x 16 bytes, without swizzle.  P^T: [key][16 columns], likewise.
template <int D, int PARTS, int RT>
struct Lay {
  static constexpr int INNER = D % 128 == 0 ? 128 : D == 64 ? 64 : 32;
  static constexpr int SUBS = D / INNER;                  // sub-tiles of a tile
  static constexpr uint32_t SUB = UNIT * INNER;
  static constexpr uint32_t TILE = UNIT * D;              // bytes of a K or V tile
  static constexpr int STAGES = D == 64 ? 3 : 2;
  static constexpr int MT = (D + 127) / 128;              // MMAs over d
  static constexpr int N = (RT * PARTS + 15) / 16 * 16;   // columns
  static constexpr uint32_t TMEM_USED = 2 * N + 2 * MT * N;
  static constexpr uint32_t TMEM_COLS = TMEM_USED <= 64 ? 64 : TMEM_USED <= 128 ? 128 : TMEM_USED <= 256 ? 256 : 512;
  static constexpr uint32_t K0 = 0, V0 = STAGES * TILE, Q0 = 2 * STAGES * TILE, P0 = Q0 + N * D;
  static constexpr uint32_t P = N * UNIT;                 // bytes of a P buffer
  // V's operand may reach 128 rows of SUB bytes beyond the last tile's start: inside the block's memory
  static constexpr uint32_t REACH = V0 + (STAGES - 1) * TILE + (128 / INNER > SUBS ? 128 / INNER : SUBS) * SUB;
  static constexpr uint32_t CTL = P0 + 2 * P > REACH ? P0 + 2 * P : REACH;
  static constexpr uint32_t INFO = CTL + 2048;
  static constexpr uint64_t SWZ = INNER == 128 ? kSw128 : INNER == 64 ? kSw64 : kSw32;
  static constexpr size_t smem(int batch) { return 1024 + INFO + (size_t)batch * sizeof(SeqInfo); }
  static_assert(TMEM_USED <= 512, "TMEM plan");
};

template <int D, int PARTS, int RT>
__global__ void __launch_bounds__(kThreads, D == 64 ? 4 : D <= 128 ? 3 : 1)
    paged_attention_kernel(const __grid_constant__ CUtensorMap mapK, const __grid_constant__ CUtensorMap mapV,
                           const AttnArgs a) {
  using L = Lay<D, PARTS, RT>;
  constexpr int N = L::N, MT = L::MT, ST = L::STAGES;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  __shared__ __align__(16) float red[RT][4];              // one number per row and softmax warp
  __shared__ float row_f[RT];
  __shared__ long long wsum[kThreads / 32];
  const uint32_t raw = smem_u32(smem_raw), base = (raw + 1023u) & ~1023u;
  uint8_t* mem = smem_raw + (base - raw);
  SeqInfo* info = reinterpret_cast<SeqInfo*>(mem + L::INFO);
  const uint32_t ctl = base + L::CTL;
  const uint32_t kfull = ctl, kempty = ctl + 32, vfull = ctl + 64, vempty = ctl + 96, sfull = ctl + 128, pfull = ctl + 144,
                 ofull = ctl + 160, qfull = ctl + 176, drain = ctl + 184;
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(mem + L::CTL + 256);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(mem + L::CTL + 264);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      bar_init(kfull + 8 * s, 1);
      bar_init(kempty + 8 * s, 1);
      bar_init(vfull + 8 * s, 1);
      bar_init(vempty + 8 * s, 1);
    }
    for (int i = 0; i < 2; ++i) {
      bar_init(sfull + 8 * i, 1);
      bar_init(pfull + 8 * i, kSoftWarps);
      bar_init(ofull + 8 * i, 1);
    }
    bar_init(qfull, kSoftWarps);
    bar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kProdWarp && lane == 0) {
    prefetch_map(&mapK);
    prefetch_map(&mapV);
  }
  if (warp == kMmaWarp) tmem_alloc(smem_u32((const void*)tmem_slot), L::TMEM_COLS);
  griddep_wait();   // the set-up above runs beside the end of the kernel before; memory is touched from here on

  // ---- the batch's units, and this CTA's share ----
  const int B = a.c.batch, Hkv = a.c.n_kv_heads, page_size = a.c.page_size;
  // with starts that are none (below 0, falling, past T) no row is a sequence's
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
    for (int w = 0; w < kThreads / 32; ++w) {
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
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot, tmem_s = tmem, tmem_o = tmem + 2 * N;

  if (warp == kProdWarp) {
    // ---------------- page copies ----------------
    const int box = min(page_size, UNIT), boxes = UNIT / box;
    uint32_t it = 0;
    bool ok = true;
    while (u < u_end && ok) {
      const Part p = part_at<RT>(a, info, u, u_end, b);
      const int* pages = a.c.block_table + (size_t)p.b * a.c.pages_per_seq;
      const auto page_of = [&](int key) {
        return lane < boxes && key < p.tb ? __ldg(pages + (key >> a.lg_page)) : -1;
      };
      int key = p.ta + lane * box, next = page_of(key);
      for (int k0 = p.ta; k0 < p.tb; k0 += UNIT, ++it, key += UNIT) {
        const int page = next;
        next = page_of(key + UNIT);
        const bool load = page >= 0 && page < a.c.num_pages;
        const int y = load ? (page * Hkv + p.kvh) * page_size + (key & (page_size - 1)) : 0;
        const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, load)) * (uint32_t)(box * D);
        const uint32_t s = it % ST, ph = (it / ST) & 1;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          const uint32_t full = (v ? vfull : kfull) + 8 * s, empty = (v ? vempty : kempty) + 8 * s;
          ok = ok && bar_wait(empty, ph ^ 1, kErrProd, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane == 0) bar_expect_tx(full, bytes);
          __syncwarp();
          const uint32_t dst = base + (v ? L::V0 : L::K0) + s * L::TILE + (uint32_t)(lane * box * L::INNER);
          if (load) {
#pragma unroll
            for (int i = 0; i < L::SUBS; ++i) tma_load(dst + i * L::SUB, v ? &mapV : &mapK, i * L::INNER, y, full);
          }
        }
        if (!ok) break;
      }
      u = p.u1;
    }
    // every issued copy has landed before the block ends
    const uint32_t pending = it < (uint32_t)ST ? it : (uint32_t)ST;
    if (lane == 0 && ok)
      for (uint32_t j = it - pending; j < it; ++j) {
        bar_drain(kfull + 8 * (j % ST), (j / ST) & 1, kErrDrain);
        bar_drain(vfull + 8 * (j % ST), (j / ST) & 1, kErrDrain);
      }
    // after an expired wait the copies under way are not counted any more: give them time
    if (!ok) {
      const long long t0 = clock64();
      while (clock64() - t0 < kWaitCycles / 64) {
      }
    }
    __syncwarp();
  } else if (warp == kMmaWarp) {
    // ---------------- MMAs: the scores of a tile, then the sums of the one before ----------------
    constexpr uint32_t idesc_s = idesc_e4m3(128, N), idesc_o = idesc_e4m3(128, N, true, true);
    constexpr uint32_t hk = desc_high(8 * L::INNER, L::SWZ), hq = desc_high(D / 16 * 128, kSwNone),
                       hv = desc_high(8 * L::INNER, L::SWZ), hp = desc_high(UNIT * 16, kSwNone);
    const uint32_t dk = desc_low(base + L::K0, 16), dq = desc_low(base + L::Q0, 128), dv = desc_low(base + L::V0, L::SUB),
                   dp = desc_low(base + L::P0, 128);
    uint32_t it = 0, seg = 0;
    bool ok = true;
    const auto scores = [&](uint32_t j) {
      const uint32_t s = j % ST;
      if (!__all_sync(0xffffffffu, bar_wait(kfull + 8 * s, (j / ST) & 1, kErrMma, abort_flag))) return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t k0 = dk + s * (L::TILE >> 4), d = tmem_s + (j & 1) * N;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) {
          constexpr int PER = L::INNER / 32;   // steps of a sub-tile
          const uint32_t at = k / PER * L::SUB + k % PER * 32;
          mma_f8(d, desc_of(k0 + (at >> 4), hk), desc_of(dq + k * 16, hq), idesc_s, k != 0);
        }
        mma_commit(sfull + 8 * (j & 1));
        mma_commit(kempty + 8 * s);
      }
      __syncwarp();
      return true;
    };
    const auto sums = [&](uint32_t j) {
      const uint32_t s = j % ST;
      if (!__all_sync(0xffffffffu, bar_wait(vfull + 8 * s, (j / ST) & 1, kErrMma, abort_flag) &&
                                       bar_wait(pfull + 8 * (j & 1), (j >> 1) & 1, kErrMma, abort_flag)))
        return false;
      tc_fence_after();
      if (elect_one()) {
        const uint32_t v0 = dv + s * (L::TILE >> 4), p0 = dp + (j & 1) * (L::P >> 4), d = tmem_o + (j & 1) * MT * N;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
          for (int k = 0; k < UNIT / 32; ++k)
            mma_f8(d + m * N, desc_of(v0 + ((m * L::SUB + k * 32 * L::INNER) >> 4), hv), desc_of(p0 + k * 32, hp), idesc_o,
                   k != 0);
        mma_commit(ofull + 8 * (j & 1));
        mma_commit(vempty + 8 * s);
      }
      __syncwarp();
      return true;
    };
    while (u < u_end && ok) {
      const Part p = part_at<RT>(a, info, u, u_end, b);
      const int tiles = p.tb > p.ta ? (p.tb - p.ta + UNIT - 1) / UNIT : 0;
      if (tiles > 0) {
        ok = __all_sync(0xffffffffu, bar_wait(qfull, seg & 1, kErrMma, abort_flag));
        ++seg;
        if (ok) ok = scores(it);
        for (int i = 0; i < tiles && ok; ++i) {
          if (i + 1 < tiles) ok = scores(it + i + 1);
          if (ok) ok = sums(it + i);
        }
        it += tiles;
      }
      u = p.u1;
    }
    // every issued MMA has completed before TMEM is freed
    if (elect_one()) mma_commit(drain);
    __syncwarp();
    bar_drain(drain, 0, kErrDrain);
  } else {
    // ---------------- softmax and sums: a thread is key tid of a tile, and column tid of the head ----------------
    // After an expired wait these warps go on through their loops (every wait then returns at once), so that none of
    // them waits for another in the block's barrier.
    const int tid = threadIdx.x;
    const uint32_t my_lanes = (uint32_t)(32 * warp) << 16;
    uint32_t it = 0, seg = 0;
    const auto part_scale = [](int part) { return __int_as_float((127 - 4 * part) << 23); };   // 2^(-4 part)
    while (u < u_end) {
      const Part p = part_at<RT>(a, info, u, u_end, b);
      const int tiles = p.tb > p.ta ? (p.tb - p.ta + UNIT - 1) / UNIT : 0;
      float nm[RT], l[RT], o[MT][RT];   // minus the reference; this thread's share of l; the sums of column tid
      uint32_t fresh = (1u << RT) - 1;  // rows that have no reference yet; the same in every thread
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        nm[r] = 0.f;
        l[r] = 0.f;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) o[mt][r] = 0.f;
      }
      if (tiles > 0) {
        // ---- query parts: 16 threads a row, D / 16 columns each ----
        {
          constexpr int E = D / 16;
          const int r = tid >> 4, row = p.row0 + r, d0 = (tid & 15) * E;
          float v[E];
          uint32_t top = 0;
          const long long qo = (long long)(p.r_first + row / a.G) * a.qts + (long long)(p.kvh * a.G + row % a.G) * a.qhs + d0;
#pragma unroll
          for (int e = 0; e < E; ++e) {
            v[e] = r < RT && row <= p.last_row ? load_q(a, qo + e) : 0.f;
            top = max(top, __float_as_uint(v[e]) & 0x7fffffffu);
          }
#pragma unroll
          for (int o2 = 8; o2; o2 >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o2));
          // the row's largest value to [128, 256) by a power of two
          const int ex = min(max((int)(top >> 23) - 134, -126), 126);
          const float down = __int_as_float((127 - ex) << 23);
          if (r < RT && (tid & 15) == 0) {
            // an infinity would saturate: its row is NaN
            row_f[r] = top >= 0x7f800000u ? __int_as_float(0x7fffffff)
                                          : __int_as_float((127 + ex) << 23) * (a.scale * kLog2e);
          }
          if (r < RT) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
              const int d = d0 + e;
              float x = v[e] * down;
#pragma unroll
              for (int i = 0; i < PARTS; ++i) {
                const uint8_t c = to_e4m3(x);
                x = (x - from_e4m3(c)) * 16.f;
                const int col = i * RT + r;
                mem[L::Q0 + (col / 8) * (D * 8) + (d / 16) * 128 + (col % 8) * 16 + d % 16] = c;
              }
            }
          }
          fence_async_smem();
          named_barrier_sync(1, 32 * kSoftWarps);   // row_f, too
          if (lane == 0) bar_arrive(qfull);
        }
        float f[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) f[r] = row_f[r];

        // page and scales of this thread's key, one and two tiles ahead
        const int* pages = a.c.block_table + (size_t)p.b * a.c.pages_per_seq;
        const auto page_of = [&](int key) {
          if (key >= p.tb || key < p.tile_lo) return -1;
          const int page = __ldg(pages + (key >> a.lg_page));
          if (page >= 0 && page < a.c.num_pages) return page;
          atomicOr(&g_dev_error, kErrIndex);
          return -1;
        };
        const auto scales_of = [&](int page, float& ks, float& vs) {
          const size_t at = (size_t)max(page, 0) * Hkv + p.kvh;
          ks = page >= 0 ? __ldg(a.c.k_scales + at) : 0.f;
          vs = page >= 0 ? __ldg(a.c.v_scales + at) : 0.f;
        };
        int page = page_of(p.ta + tid), page1 = page_of(p.ta + UNIT + tid);
        float ks, vs;
        scales_of(page, ks, vs);

        const auto add_sums = [&](uint32_t j) {
          bar_wait(ofull + 8 * (j & 1), (j >> 1) & 1, kErrSoft, abort_flag);
          tc_fence_after();
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int n = 0; n < N; n += 16) {
              uint32_t w[16];
              tmem_ld(tmem_o + my_lanes + ((j & 1) * MT + mt) * N + n, w);
              tmem_wait(w);
#pragma unroll
              for (int q = 0; q < 16 / RT; ++q)
                if (n / RT + q < PARTS)
                  fma_rows(o[mt], [&](int r) { return __uint_as_float(w[(RT * q + r) % 16]); },
                           [&](int) { return part_scale(n / RT + q); }, [&](int r) { return o[mt][r]; });
            }
        };

        for (int i = 0; i < tiles; ++i) {
          const uint32_t j = it + i;
          const int k0 = p.ta + UNIT * i, key = k0 + tid;
          const bool there = page >= 0;
          const float ks_i = ks, vs_i = vs;
          page = page1;
          scales_of(page, ks, vs);
          page1 = page_of(key + 2 * UNIT);
          // ---- scores, less the reference ----
          float y[RT], fk[RT];
          mul_rows(fk, [&](int r) { return f[r]; }, [&](int) { return ks_i; });
          bar_wait(sfull + 8 * (j & 1), (j >> 1) & 1, kErrSoft, abort_flag);
          tc_fence_after();
#pragma unroll
          for (int n = 0; n < N; n += 16) {
            uint32_t w[16];
            tmem_ld(tmem_s + my_lanes + (j & 1) * N + n, w);
            tmem_wait(w);
#pragma unroll
            for (int q = 0; q < 16 / RT; ++q) {
              const int part = n / RT + q;
              if (part == 0) {
#pragma unroll
                for (int r = 0; r < RT; ++r) y[r] = __uint_as_float(w[r % 16]);
              } else if (part < PARTS) {
                fma_rows(y, [&](int r) { return __uint_as_float(w[(RT * q + r) % 16]); },
                         [&](int) { return part_scale(part); }, [&](int r) { return y[r]; });
              }
            }
          }
          fma_rows(y, [&](int r) { return y[r]; }, [&](int r) { return fk[r]; }, [&](int r) { return nm[r]; });
          const bool alike = k0 >= p.all_lo && min(k0 + UNIT, p.tb) <= p.all_hi;   // rows see the same of these keys
          if (__builtin_expect(!there, 0)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) y[r] = -INFINITY;
          }
          if (__builtin_expect(!alike, 0)) {
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const int pos = p.pos0 + (p.row0 + r) / a.G;
              if (key > pos || (a.window > 0 && key <= pos - a.window)) y[r] = -INFINITY;
            }
          }
          // ---- the reference, if a key exceeds it by more than a factor of 2 ----
          const float lv = fmaxf(lg2(vs_i), -60.f);
          float over = y[0];
#pragma unroll
          for (int r = 1; r < RT; ++r) over = fmaxf(over, y[r]);
          bool added = i == 0;
          if (any_of(over + lv > 1.f) || fresh) {
            if (!added) add_sums(j - 1);
            added = true;
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const float top = warp_max(y[r] + lv);
              if (lane == 0) red[r][warp] = top;
            }
            named_barrier_sync(1, 32 * kSoftWarps);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              const float4 w = *reinterpret_cast<const float4*>(red[r]);
              const float top = fmaxf(fmaxf(w.x, w.y), fmaxf(w.z, w.w));
              const bool first = fresh & (1u << r);      // l and o are zero then
              if (first && top == -INFINITY) continue;   // the row has seen no key
              const float up = first ? top : fmaxf(top, 0.f), c = first ? 1.f : ex2(-up);
              fresh &= ~(1u << r);
              nm[r] -= up;
              y[r] -= up;
              l[r] *= c;
#pragma unroll
              for (int mt = 0; mt < MT; ++mt) o[mt][r] *= c;
            }
            named_barrier_sync(1, 32 * kSoftWarps);   // red may be written again
          }
          // ---- weights to shared memory ----
          float pw[RT];
#pragma unroll
          for (int r = 0; r < RT; ++r) pw[r] = ex2(y[r]);
          add_rows(l, [&](int r) { return l[r]; }, [&](int r) { return pw[r]; });
          const float fold = vs_i * kPScale;
          mul_rows(pw, [&](int r) { return pw[r]; }, [&](int) { return fold; });
          uint8_t* pb = mem + L::P0 + (j & 1) * L::P;
          if constexpr (RT >= 4) {
            uint32_t w[N / RT][RT / 4];
#pragma unroll
            for (int r = 0; r < RT; r += 4) {
              float v[4] = {pw[r], pw[r + 1], pw[r + 2], pw[r + 3]};
#pragma unroll
              for (int q = 0; q < N / RT; ++q) {
                if (q < PARTS - 1) w[q][r / 4] = take_e4m3(v);
                else if (q < PARTS) w[q][r / 4] = to_e4m3x2(v[0], v[1]) | (to_e4m3x2(v[2], v[3]) << 16);
                else w[q][r / 4] = 0;
              }
            }
            const uint32_t* all = &w[0][0];
#pragma unroll
            for (int n = 0; n < N / 16; ++n)
              *reinterpret_cast<uint4*>(pb + n * UNIT * 16 + tid * 16) = make_uint4(all[4 * n], all[4 * n + 1], all[4 * n + 2], all[4 * n + 3]);
          } else {
            // one row: its parts are the first columns, the others zeros
            uint32_t w[4] = {0, 0, 0, 0};
#pragma unroll
            for (int q = 0; q < PARTS; ++q) {
              const uint32_t c = to_e4m3(pw[0]);
              pw[0] = (pw[0] - from_e4m3((uint8_t)c)) * 16.f;
              w[q / 4] |= c << (8 * (q % 4));
            }
            *reinterpret_cast<uint4*>(pb + tid * 16) = make_uint4(w[0], w[1], w[2], w[3]);
          }
          // ---- values that must not reach a sum, where 0 * NaN is not 0 ----
          uint8_t* vt = mem + L::V0 + (j % ST) * L::TILE;
          if (__builtin_expect(!__all_sync(0xffffffffu, there), 0)) {
            // rows of no key of the sequence: whatever their page holds becomes 0
            bar_wait(vfull + 8 * (j % ST), (j / ST) & 1, kErrSoft, abort_flag);
            if (!there) {
#pragma unroll
              for (int s = 0; s < L::SUBS; ++s)
#pragma unroll
                for (int e = 0; e < L::INNER; e += 16)
                  *reinterpret_cast<uint4*>(vt + s * L::SUB + tid * L::INNER + e) = make_uint4(0, 0, 0, 0);
            }
          }
          if (__builtin_expect(!alike, 0)) {
            // a NaN code reaches only the rows that see its key: it is put into their sums by hand, and becomes 0
            bar_wait(vfull + 8 * (j % ST), (j / ST) & 1, kErrSoft, abort_flag);
            named_barrier_sync(1, 32 * kSoftWarps);   // the zeros above
            uint32_t found = 0;
            for (uint32_t at = tid * 4; at < L::TILE; at += 512) {
              const uint32_t y = *reinterpret_cast<const uint32_t*>(vt + at);
              found |= ((y & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u;
            }
            const bool any = any_of(found != 0);
            if (any) {
              for (int kk = 0; kk < UNIT && k0 + kk < p.tb; ++kk)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                  const int d = 128 * mt + tid;
                  if (d >= D) continue;
                  const uint32_t at = d / L::INNER * L::SUB + kk * L::INNER + d % L::INNER;
                  // TMA's swizzle: 16-byte pieces of a row exchanged by the row's place in 8 rows (16 or 32 bits apart)
                  const uint32_t sw = at ^ (L::INNER == 128 ? (at >> 3) & 0x70 : L::INNER == 64 ? (at >> 3) & 0x30 : (at >> 3) & 0x10);
                  if ((vt[sw] & 0x7fu) != 0x7fu) continue;
#pragma unroll
                  for (int r = 0; r < RT; ++r) {
                    const int pos = p.pos0 + (p.row0 + r) / a.G;
                    if (k0 + kk <= pos && (a.window <= 0 || k0 + kk > pos - a.window)) o[mt][r] = __int_as_float(0x7fffffff);
                  }
                }
              named_barrier_sync(1, 32 * kSoftWarps);
              for (uint32_t at = tid; at < L::TILE; at += 128)
                if ((vt[at] & 0x7fu) == 0x7fu) vt[at] = 0;
            }
          }
          fence_async_smem();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) bar_arrive(pfull + 8 * (j & 1));
          if (!added) add_sums(j - 1);
        }
        add_sums(it + tiles - 1);
        it += tiles;
        ++seg;
      }
      // ---- the part's result ----
#pragma unroll
      for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int o2 = 16; o2; o2 >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o2);
        if (lane == 0) red[r][warp] = l[r];
      }
      named_barrier_sync(1, 32 * kSoftWarps);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float4 w = *reinterpret_cast<const float4*>(red[r]);
        l[r] = (w.x + w.y) + (w.z + w.w);
      }
      named_barrier_sync(1, 32 * kSoftWarps);   // red may be written again
      const bool begins = u == p.seg0, ends = p.u1 == p.seg1;
      float* part = a.part + ((size_t)cta * 2 + (begins ? 1 : 0)) * kMaxRows * (D + 2);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const int row = p.row0 + r;
        if (row > p.last_row) break;
        const size_t th = (size_t)(p.r_first + row / a.G) * a.H + p.kvh * a.G + row % a.G;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          const int d = 128 * mt + tid;
          const float A = o[mt][r] * (1.f / kPScale);
          if (d < D) {
            if (begins && ends) store_out(a, th * D + d, l[r] == 0.f ? 0.f : A / l[r]);
            else part[r * D + d] = A;
          }
        }
        if (tid == 0) {
          if (!(begins && ends)) {
            part[RT * D + 2 * r] = fresh & (1u << r) ? kNone : -nm[r];
            part[RT * D + 2 * r + 1] = l[r];
          } else if (a.lse) {
            a.lse[th] = l[r] == 0.f ? -INFINITY : -nm[r] * kLn2 + logf(l[r]);
          }
        }
      }
      if (begins && !ends && tid == 0) {
        // CTAs of the tile's parts: this one to the one that holds its last unit
        int* dsc = a.desc + 8 * cta;
        dsc[0] = (int)(shares.holder(p.seg1 - 1) - cta + 1);
        dsc[1] = p.r_first;
        dsc[2] = p.kvh;
        dsc[3] = p.row0;
        dsc[4] = p.last_row;
      }
      u = p.u1;
    }
  }
  griddep_launch_dependents();   // not before: the merge's blocks would wait in the place of the next call's
  tc_fence_before();
  __syncthreads();
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, L::TMEM_COLS);
  }
}

#include "sf_paged_prompt.h"

template <int D, int PARTS, int RT>
int launch(AttnArgs a, cudaStream_t st) {
  using L = Lay<D, PARTS, RT>;
  const sf_paged_cache& c = a.c;
  const uint64_t rows = (uint64_t)c.num_pages * c.n_kv_heads * c.page_size;
  if (rows > 0x7fffffffull) return fail(SF_ERR_UNSUPPORTED, "the cache has more than 2^31 - 1 rows");
  const CUtensorMapSwizzle swz = L::INNER == 128  ? CU_TENSOR_MAP_SWIZZLE_128B
                                 : L::INNER == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                                  : CU_TENSOR_MAP_SWIZZLE_32B;
  const uint32_t box = c.page_size < UNIT ? c.page_size : UNIT;
  CUtensorMap mk, mv;
  if (!make_tensor_map(&mk, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.k_codes, D, rows, D, L::INNER, box, swz) ||
      !make_tensor_map(&mv, CU_TENSOR_MAP_DATA_TYPE_UINT8, c.v_codes, D, rows, D, L::INNER, box, swz))
    return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled failed for the cache");
  auto* fn = paged_attention_kernel<D, PARTS, RT>;
  const size_t smem = L::smem(c.batch);
  // the limit is the process's: the same for calls of every batch, or another thread's could lower it before this launch
  static_assert(L::smem(kMaxBatch) + 1024 <= kBlockSmem, "shared memory plan");
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)L::smem(kMaxBatch));
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention_kernel shared memory");
  // what shared memory, TMEM and registers let an SM hold
  int per_sm = (int)(228 * 1024 / (smem + 2048));
  const int most = D == 64 ? 4 : D <= 128 ? 3 : 1;
  if (per_sm > most) per_sm = most;
  if (per_sm > 512 / (int)L::TMEM_COLS) per_sm = 512 / (int)L::TMEM_COLS;
  if (per_sm < 1) per_sm = 1;
  // no more CTAs than units there may be
  const double cap = ((double)c.pages_per_seq * c.page_size + UNIT - 1) / UNIT;
  const double units = cap * ((double)a.T * a.G / RT + c.batch) * c.n_kv_heads;
  a.resident = device_info().sms * per_sm;
  int grid = 2 * a.resident;
  if (units < (double)kLong * a.resident) grid = units < a.resident ? (int)units : a.resident;
  e = launch_kernel(fn, grid, kThreads, smem, st, true, mk, mv, a);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention_kernel launch");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid, RT);
  cfg.blockDim = dim3(D);
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, paged_attention_merge_kernel<D, RT>, a);
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention_merge_kernel launch");
  g_launches.fetch_add(2, std::memory_order_relaxed);
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

size_t sf_paged_attention_workspace_bytes(int head_dim) {
  if (head_dim <= 0) return 0;
  const size_t ctas = (size_t)device_info().sms * kMaxCtasPerSm * 2;
  return ctas * (2 * kMaxRows * ((size_t)head_dim + 2) * 4 + 32);
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
  a.part = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + (size_t)device_info().sms * kMaxCtasPerSm * 2 * 32);
  a.H = H; a.T = T; a.G = H / cache->n_kv_heads; a.q_dtype = q_dtype; a.out_dtype = out_dtype;
  a.window = window < (long long)cache->pages_per_seq * cache->page_size ? window : 0;   // a wider one hides nothing
  a.lg_page = __builtin_ctz((unsigned)cache->page_size);
  a.scale = scale;
  if ((long long)T * a.G > 0x7fffffffll) return fail(SF_ERR_UNSUPPORTED, "too many query rows");
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  // Tiles of 256 rows: an SM takes 3 us for 128 keys of a tile, however many of its rows are in use, and some 6 us before
  // and after.  Tiles of 8 rows: all SMs together take 0.5 ns for 128 keys of a row, and 4 ns more a row (7 at head_dim 64).
  // So the rows of a round of tiles decide, fewer where the sequences are short; of the lengths the host knows only the
  // block table's.
  // Measured, head_dim 128, tiles of 256 and of 8 rows, in us: 18 sequences of 64 rows, 256 keys 15 and 15, 2048 keys 54
  // and 30, 32768 keys 727 and 155; 64 tiles of 64 rows 17 and 25, 56 and 54, 734 and 556; 128 such 18 and 37, 58 and 90,
  // 739 and 1187; 256 rows of 64 heads 21 and 69, 63 and 175, 758 and 1174.  Head_dim 64: 64 tiles of 64 rows 14 and 27, 50
  // and 59, 671 and 401.
  // One long sequence among many short ones is not seen here: 32 sequences of 64 rows and 8 kv heads, one of 16384 keys and
  // 31 of 300, take 383 so and 134 otherwise.
  const long long items = ((long long)T * a.G / kPromptRows + cache->batch) * cache->n_kv_heads;
  const int sms = device_info().sms;
  const long long keys = std::min((long long)cache->pages_per_seq * cache->page_size,
                                  a.window > 0 ? (long long)a.window + kPromptRows : LLONG_MAX);
  const long long tiles = std::max(((long long)T * a.G + kPromptRows - 1) / kPromptRows, (long long)cache->batch) * cache->n_kv_heads,
                  rounds = (tiles + sms - 1) / sms, key_tiles = (keys + UNIT - 1) / UNIT;
  const bool many = (double)T * H * (key_tiles + (D == 64 ? 14 : 7)) >= 5800.0 * rounds * (key_tiles + 2);
  const int type = std::min(q_dtype, out_dtype);   // the finer one
  const bool prompt = q_dtype == SF_BF16 && out_dtype != SF_F32 && (D == 64 || D == 128) && many && items <= 0x7fffffffll &&
                      reinterpret_cast<uintptr_t>(out) % 16 == 0;
  if (prompt) {
    const bool q_vec = reinterpret_cast<uintptr_t>(q) % 16 == 0 && qts % 8 == 0 && qhs % 8 == 0;
    return D == 64 ? launch_prompt<64>(a, items, q_vec, st) : launch_prompt<128>(a, items, q_vec, st);
  }
  const auto go = [&](auto d) {
    constexpr int DD = decltype(d)::value;
    if ((long long)T * a.G <= cache->batch)
      return type == SF_BF16 ? launch<DD, 2, 1>(a, st) : type == SF_F16 ? launch<DD, 3, 1>(a, st) : launch<DD, 6, 1>(a, st);
    return type == SF_BF16 ? launch<DD, 2, 8>(a, st) : type == SF_F16 ? launch<DD, 3, 8>(a, st) : launch<DD, 6, 8>(a, st);
  };
  return D == 64    ? go(std::integral_constant<int, 64>())
         : D == 96  ? go(std::integral_constant<int, 96>())
         : D == 128 ? go(std::integral_constant<int, 128>())
                    : go(std::integral_constant<int, 256>());
}

}  // extern "C"
