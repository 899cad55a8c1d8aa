// sf_fp8_linear.cu -- Y = X W^T over e4m3 rows (one scale per row and 128 columns) and e4m3 weights (one scale per
// 128 x 128 block) on the sm_100a tcgen05 tensor cores.
//
//   Y[t,n] = sum_kb xs[t,kb] * ws[n/128,kb] * sum_{k in block kb} X[t,k] * W[n,k]  (+ bias[n])
//
// Tokens are the rows of the MMA (M = 128: one TMEM lane each), weight rows its columns, so that a k-block's scale
// is one number per thread: xs of its lane's token times ws of its 128 columns.  Each k-block of 128 is one set of
// four tcgen05.mma.kind::f8f6f4 into a fresh TMEM buffer; eight warps read it back and add it, scaled, to sums that
// stay in registers in fp32 for the whole of K, while the next k-block's MMAs fill the other buffer.
//
// Two shapes of the same pipeline (TMA -> shared memory -> MMA -> TMEM -> registers):
//  * split: one 128 x 128 tile per CTA, K cut between the S CTAs of a cluster.  Their sums meet in shared memory over
//    the cluster (each CTA adds the S parts of its share of the columns, in rank order), so that few tokens still
//    spread the weight read over the SMs, in one launch and with the same result every time.  With few tokens only
//    the rows that exist are loaded; what the MMA reads above them ends in TMEM lanes that nothing looks at.
//  * persistent: 128 x 256 tiles in turn on one CTA per SM, stored through shared memory by TMA.
//
// Measured (tokens x K x N) in a graph; called one after another 3 to 15 us more.  Weight-bound: 16 x 8192 x 28672 46.7 us,
// 5.1 TB/s.  Bound by latency, the first copies and the cluster's exchange: 1 x 4096 x 4096 8.6 us, 77 x 896 x 4864 10 us.
// 2048 x 4096 x 11008 120 us, 1540 TFLOP/s: the tensor pipe works 38 % of the time, issue slots 34 %; the summing warps wait
// for TMEM (long scoreboard) and for their own chain, with two accumulator buffers to hide it.
#include <atomic>
#include <cstdint>
#include <cstring>

#include "sf_e4m3.h"
#include "sf_q4_internal.h"
#include "sf_tcgen05.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_fp8)
extern std::atomic<long long> g_launches;

namespace {

constexpr int kBK = 128;                // k per stage: one 128-byte swizzle row, and one block of scales
constexpr int kSumWarps = 8, kProdWarp = 8, kMmaWarp = 9;
constexpr int kSmemLimit = 232448;      // 227 KB opt-in per block
constexpr unsigned kErrProd = 1u << 13, kErrMma = 1u << 14, kErrSum = 1u << 15, kErrDrain = 1u << 16;

struct Fp8Params {
  const float* xs;
  const float* ws;
  const float* bias;
  void* Y;
  int T, N, KB, y_dtype;
  int mtiles, ntiles;
  int rows;        // rows of X that a stage holds (16, 32, 64 or 128)
  int stages;
  int split;       // CTAs of a cluster along K
  int tma_store;
};

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void st_cluster(uint32_t saddr, uint32_t rank, float v) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(saddr), "r"(rank));
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(a), "f"(v) : "memory");
}

__device__ __forceinline__ void store_y(void* Y, size_t o, float v, int dt) {
  if (dt == SF_F32) static_cast<float*>(Y)[o] = v;
  else if (dt == SF_F16) static_cast<__half*>(Y)[o] = __float2half_rn(v);
  else static_cast<__nv_bfloat16*>(Y)[o] = __float2bfloat16_rn(v);
}
__device__ __forceinline__ uint32_t pack16(float lo, float hi, int dt) {
  uint32_t d;
  if (dt == SF_BF16) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  else asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Shared memory: `stages` x (X rows, then W tile), then for the persistent kernel one 4 KB store buffer per warp,
// then the barriers.  An MMA reads 128 rows wherever X starts: with fewer loaded, the rest are bytes of the same
// stage's W tile.  The split kernel reuses the stages for the sums that the cluster exchanges.
template <bool SPLIT>
struct Plan {
  static constexpr int BN = SPLIT ? 128 : 256;
  static constexpr int NBUF = 2;
  static constexpr uint32_t TMEM_COLS = NBUF * BN;
  static constexpr int CW = BN / 2;                      // columns of a summing warp
  static constexpr int CH = SPLIT ? 16 : 32;             // columns it reads at a time
  static constexpr int NR = SPLIT ? 1 : 2;               // reads in flight
  static constexpr int LA = SPLIT ? 2 : 4;               // k-blocks whose scales are loaded ahead
  // The persistent kernel has a third warpgroup so that setmaxnreg can move registers from it to the summing warps,
  // which keep 128 sums each: launched with 384 x 168 = 64512, then 256 x 232 + 128 x 40 = 64512.
  static constexpr int THREADS = SPLIT ? 320 : 384;
  static constexpr uint32_t W = BN * kBK;
  static constexpr uint32_t CTL = 512;
  static constexpr uint32_t TAIL = SPLIT ? 0 : kSumWarps * 4096;
  static constexpr int MAX_STAGES = 12;
  static constexpr uint32_t stage(int rows) { return W + (uint32_t)rows * kBK; }
  static constexpr size_t bytes(int rows, int stages) { return 1024 + (size_t)stages * stage(rows) + TAIL + CTL; }
};

template <bool SPLIT>
__global__ void __launch_bounds__(Plan<SPLIT>::THREADS, SPLIT ? 2 : 1)
    fp8_linear_kernel(const __grid_constant__ CUtensorMap mapX, const __grid_constant__ CUtensorMap mapW,
                      const __grid_constant__ CUtensorMap mapY, const Fp8Params p) {
  using L = Plan<SPLIT>;
  constexpr int BN = L::BN, NBUF = L::NBUF, CW = L::CW, CH = L::CH;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  const uint32_t xbytes = (uint32_t)p.rows * kBK, stage_bytes = L::W + xbytes;
  const uint32_t tail = base + (uint32_t)p.stages * stage_bytes;
  const uint32_t ctl = tail + L::TAIL;
  const uint32_t full0 = ctl, empty0 = ctl + 8 * L::MAX_STAGES, accf0 = ctl + 16 * L::MAX_STAGES, acce0 = accf0 + 16,
                 drain = acce0 + 16;
  uint8_t* ctl_gen = smem_raw + (ctl - raw);
  volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(ctl_gen + 400);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(ctl_gen + 408);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int S = p.stages;
  griddep_launch_dependents();
  // lane quarters that hold tokens: their two warps each release an accumulator buffer
  const int quarters = SPLIT ? (p.rows + 31) / 32 : 4;
  if (threadIdx.x == 0) {
    for (int s = 0; s < S; ++s) {
      bar_init(full0 + 8 * s, 1);
      bar_init(empty0 + 8 * s, 1);
    }
    for (int b = 0; b < NBUF; ++b) {
      bar_init(accf0 + 8 * b, 1);
      bar_init(acce0 + 8 * b, 2 * quarters);
    }
    bar_init(drain, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == kProdWarp && lane == 0) {
    prefetch_map(&mapX);
    prefetch_map(&mapW);
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32((const void*)tmem_slot), L::TMEM_COLS);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  griddep_wait();   // the set-up above runs beside the end of the kernel before; memory is touched from here on

  const int ntiles = p.mtiles * p.ntiles;
  const int rank = SPLIT ? (int)(blockIdx.x % p.split) : 0;
  const int kb0 = SPLIT ? (int)((long long)p.KB * rank / p.split) : 0;
  const int kb1 = SPLIT ? (int)((long long)p.KB * (rank + 1) / p.split) : p.KB;
  const int tile0 = SPLIT ? (int)(blockIdx.x / p.split) : (int)blockIdx.x;
  const int tile_step = SPLIT ? ntiles : (int)gridDim.x;   // the split kernel has one tile

  // Ends a role: all MMAs and copies of the block are done (of the cluster, before its sums are exchanged).
  const auto meet = [&] {
    tc_fence_before();
    __syncthreads();
    if (SPLIT && p.split > 1) cluster_sync();
  };
  const uint32_t pitch = 4u * (32 * quarters + 1);   // of the exchanged sums, below
  const int cols = SPLIT ? BN / p.split : BN, lg_cols = 31 - __clz(cols);

  if (warp >= kProdWarp) {
    // one instruction for the warpgroup
    if (!SPLIT) asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    if (warp == kProdWarp) {
      // ---------------- TMA producer ----------------
      if (lane == 0) {
        uint32_t it = 0;
        bool ok = true;
        for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
          const int m0 = (tile % p.mtiles) * 128, n0 = (tile / p.mtiles) * BN;
          for (int kb = kb0; kb < kb1; ++kb, ++it) {
            const uint32_t s = it % S, ph = (it / S) & 1;
            if (!bar_wait(empty0 + 8 * s, ph ^ 1, kErrProd, abort_flag)) { ok = false; break; }
            const uint32_t st = base + s * stage_bytes;
            bar_expect_tx(full0 + 8 * s, stage_bytes);
            tma_load(st, &mapX, kb * kBK, m0, full0 + 8 * s);
            tma_load(st + xbytes, &mapW, kb * kBK, n0, full0 + 8 * s);
          }
        }
        // every issued copy has landed before the block goes on
        const uint32_t pending = it < (uint32_t)S ? it : (uint32_t)S;
        for (uint32_t j = it - pending; j < it; ++j) bar_drain(full0 + 8 * (j % S), (j / S) & 1, kErrDrain);
      }
      __syncwarp();
      meet();
    } else if (warp == kMmaWarp) {
      // ---------------- MMA issuer ----------------
      constexpr uint32_t idesc = idesc_e4m3(128, BN), high = desc_high(1024, kSw128);
      const uint32_t low = desc_low(base, 16), step = stage_bytes >> 4;
      uint32_t s = 0, ph = 0, b = 0, use = 0;
      bool ok = true;
      for (int tile = tile0; tile < ntiles && ok; tile += tile_step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = bar_wait(acce0 + 8 * b, use ^ 1, kErrMma, abort_flag) && bar_wait(full0 + 8 * s, ph, kErrMma, abort_flag);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t x = low + s * step, w = x + (xbytes >> 4);
#pragma unroll
            for (int kk = 0; kk < kBK / 32; ++kk)
              mma_f8(tmem + b * BN, desc_of(x + 2 * kk, high), desc_of(w + 2 * kk, high), idesc, kk != 0);
            mma_commit(accf0 + 8 * b);
            mma_commit(empty0 + 8 * s);
          }
          __syncwarp();
          if (++s == (uint32_t)S) {
            s = 0;
            ph ^= 1;
          }
          if (++b == NBUF) {
            b = 0;
            use ^= 1;
          }
        }
      }
      // every issued MMA has completed before TMEM is freed
      if (elect_one()) mma_commit(drain);
      __syncwarp();
      bar_drain(drain, 0, kErrDrain);
      __syncwarp();
      meet();
    } else {
      meet();
    }
  } else {
    // ---------------- scaled sums ----------------
    // Warp w: tokens 32 (w % 4) .. of the tile, columns CW (w / 4) .. (inside one 128-column block of ws).
    if (!SPLIT) asm volatile("setmaxnreg.inc.sync.aligned.u32 232;");
    const int q = warp & 3, c0 = (warp >> 2) * CW;
    const uint32_t lane_base = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)c0;
    uint32_t it = 0;
    uint64_t acc[CW / 2];
    if (q < quarters) {
      for (int tile = tile0; tile < ntiles; tile += tile_step) {
        const int m0 = (tile % p.mtiles) * 128, n0 = (tile / p.mtiles) * BN;
        const int t = m0 + 32 * q + lane, nb = (n0 + c0) / 128;
        const bool in = t < p.T && nb * 128 < p.N;
        const float* xrow = p.xs + (size_t)(in ? t : 0) * p.KB;
        const float* wrow = p.ws + (size_t)(in ? nb : 0) * p.KB;
#pragma unroll
        for (int i = 0; i < CW / 2; ++i) acc[i] = 0;
        // the scales of the next LA k-blocks are loaded while these are used: the rows of a full tile are too many
        // for what shared memory leaves of L1
        constexpr int LA = L::LA;
        float s4[LA], x4[LA], w4[LA];
        const auto fetch = [&](int kb) {
#pragma unroll
          for (int i = 0; i < LA; ++i) {
            const int k = min(kb + i, kb1 - 1);
            x4[i] = __ldg(xrow + k);
            w4[i] = __ldg(wrow + k);
          }
        };
        fetch(kb0);
        bool ok = true;
        for (int kb = kb0; kb < kb1 && ok; kb += LA) {
#pragma unroll
          for (int i = 0; i < LA; ++i) s4[i] = x4[i] * w4[i];
          fetch(kb + LA);
#pragma unroll
          for (int i = 0; i < LA; ++i) {
            if (kb + i >= kb1) break;
            const uint32_t b = it % NBUF, use = it / NBUF;
            ++it;
            const uint64_t s2 = pack2(s4[i], s4[i]);
            if (!bar_wait(accf0 + 8 * b, use & 1, kErrSum, abort_flag)) { ok = false; break; }
            tc_fence_after();
            uint32_t r[L::NR][CH];
            tmem_ld(lane_base + b * BN, r[0]);
#pragma unroll
            for (int c = 0; c < CW / CH; ++c) {
              tmem_wait(r[c % L::NR]);
              if (L::NR == 2 && c + 1 < CW / CH) tmem_ld(lane_base + b * BN + CH * (c + 1), r[(c + 1) % L::NR]);
              if (c + 1 == CW / CH) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive(acce0 + 8 * b);
              }
#pragma unroll
              for (int e = 0; e < CH / 2; ++e)
                acc[CH / 2 * c + e] = fma2(pack2(__uint_as_float(r[c % L::NR][2 * e]),
                                                 __uint_as_float(r[c % L::NR][2 * e + 1])), s2, acc[CH / 2 * c + e]);
              if (L::NR == 1 && c + 1 < CW / CH) tmem_ld(lane_base + b * BN + CH * (c + 1), r[0]);
            }
          }
        }
        if (!ok) break;
        if constexpr (SPLIT) {
          // stored below, when the cluster's stages are free
        } else if (p.tma_store) {
          // 128 bytes of each of the warp's 32 tokens at a time, in the 128-byte swizzle, stored by TMA, which
          // leaves out rows past T and columns past N
          const uint32_t buf = tail + (uint32_t)warp * 4096;
          const int per = p.y_dtype == SF_F32 ? 32 : 64;
#pragma unroll
          for (int g = 0; g < L::CW / 32; ++g) {
            if (per == 64 && (g & 1)) continue;
            if (n0 + c0 + 32 * g >= p.N) break;
            if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              uint32_t w[4];
              if (per == 32) {
                float v[4];
                unpack2(acc[16 * g + 2 * j], v[0], v[1]);
                unpack2(acc[16 * g + 2 * j + 1], v[2], v[3]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const int n = n0 + c0 + 32 * g + 4 * j + e;
                  if (p.bias && n < p.N) v[e] += __ldg(p.bias + n);
                  w[e] = __float_as_uint(v[e]);
                }
              } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  float2 f;
                  unpack2(acc[(16 * g + 4 * j + e) % (L::CW / 2)], f.x, f.y);
                  const int n = n0 + c0 + 32 * g + 8 * j + 2 * e;
                  if (p.bias && n < p.N) f.x += __ldg(p.bias + n);
                  if (p.bias && n + 1 < p.N) f.y += __ldg(p.bias + n + 1);
                  w[e] = pack16(f.x, f.y, p.y_dtype);
                }
              }
              asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(buf + lane * 128 + ((j ^ (lane & 7)) << 4)),
                           "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                           : "memory");
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0 && m0 + 32 * q < p.T) tma_store(&mapY, n0 + c0 + 32 * g, m0 + 32 * q, buf);
          }
        } else if (t < p.T) {
#pragma unroll
          for (int i = 0; i < L::CW / 2; ++i) {
            float2 f;
            unpack2(acc[i], f.x, f.y);
            const int n = n0 + c0 + 2 * i;
            if (n < p.N) store_y(p.Y, (size_t)t * p.N + n, f.x + (p.bias ? __ldg(p.bias + n) : 0.f), p.y_dtype);
            if (n + 1 < p.N) store_y(p.Y, (size_t)t * p.N + n + 1, f.y + (p.bias ? __ldg(p.bias + n + 1) : 0.f), p.y_dtype);
          }
        }
      }
      if (!SPLIT && p.tma_store && lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    }
    __syncwarp();
    meet();
    if (SPLIT && q < quarters && 32 * q + lane < p.rows) {
      // To the CTA of the cluster that adds this column: [rank][column][token], one float further than the tokens
      // apart, so that neither the lanes here (tokens) nor those of the addition (columns) meet in a bank.
      const uint32_t at = base + (uint32_t)(32 * q + lane) * 4;
#pragma unroll
      for (int i = 0; i < CW; ++i) {
        const int c = c0 + i;
        float2 f;
        unpack2(acc[i / 2], f.x, f.y);
        const uint32_t o = at + (uint32_t)(rank * cols + (c & (cols - 1))) * pitch;
        if (p.split > 1) st_cluster(o, (uint32_t)(c >> lg_cols), i & 1 ? f.y : f.x);
        else asm volatile("st.shared.f32 [%0], %1;" ::"r"(o), "f"(i & 1 ? f.y : f.x) : "memory");
      }
    }
  }

  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_free(tmem, L::TMEM_COLS);
  }
  if constexpr (SPLIT) {
    // ---------------- the cluster's sums, in rank order ----------------
    __syncwarp();
    if (p.split > 1) cluster_sync();
    else __syncthreads();
    const int m0 = (tile0 % p.mtiles) * 128, n0 = (tile0 / p.mtiles) * BN + rank * cols;
    const int rows = min(p.rows, p.T - m0);
    const float* sums = reinterpret_cast<const float*>(smem_raw + (base - raw));
    const int step = cols * (int)(pitch / 4);
    for (int i = threadIdx.x; i < cols * rows; i += L::THREADS) {
      const int c = i & (cols - 1), t = i >> lg_cols, n = n0 + c;
      if (n >= p.N) continue;
      const float* at = sums + c * (int)(pitch / 4) + t;
      float v = 0.f;
#pragma unroll
      for (int r = 0; r < 8; ++r)
        if (r < p.split) v += at[r * step];
      store_y(p.Y, (size_t)(m0 + t) * p.N + n, v + (p.bias ? __ldg(p.bias + n) : 0.f), p.y_dtype);
    }
  }
}

bool make_map(CUtensorMap* m, CUtensorMapDataType dt, const void* base, uint64_t inner, uint64_t rows, uint64_t pitch,
              uint32_t box_inner, uint32_t box_rows) {
  return make_tensor_map(m, dt, base, inner, rows, pitch, box_inner, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

template <bool SPLIT>
cudaError_t launch(const CUtensorMap& mx, const CUtensorMap& mw, const CUtensorMap& my, const Fp8Params& p, int grid,
                   cudaStream_t st) {
  auto* fn = fp8_linear_kernel<SPLIT>;
  const size_t smem = Plan<SPLIT>::bytes(p.rows, p.stages);
  // the limit is the process's: the same for calls of every size, or another thread's could lower it before this launch
  cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(Plan<SPLIT>::THREADS);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)p.split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = p.split > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, fn, mx, mw, my, p);
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" int sf_fp8_linear(const uint8_t* X, long long ldx, const float* xs, const uint8_t* W, long long ldw,
                             const float* ws, const float* bias, void* Y, int y_dtype, int T, int N, int K,
                             void* stream) {
  if (T < 0 || N < 0 || K < 1) return fail(SF_ERR_SHAPE, "need T >= 0, N >= 0 and K >= 1");
  if (y_dtype < 0 || y_dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (T == 0 || N == 0) return SF_OK;
  if (!X || !xs || !W || !ws || !Y) return fail(SF_ERR_NULL, "null pointer argument");
  if (ldx < K || ldw < K) return fail(SF_ERR_SHAPE, "a row stride is below K");
  if (((reinterpret_cast<uintptr_t>(X) | reinterpret_cast<uintptr_t>(W)) & 15) || ldx % 16 || ldw % 16)
    return fail(SF_ERR_ALIGN, "X and W must start at multiples of 16 bytes and have row strides that are multiples of 16");
  DeviceInfo& di = device_info();
  Fp8Params p{};
  p.xs = xs; p.ws = ws; p.bias = bias; p.Y = Y;
  p.T = T; p.N = N; p.KB = (K + kBK - 1) / kBK; p.y_dtype = y_dtype;
  p.mtiles = (T + 127) / 128;
  p.rows = T <= 16 ? 16 : T <= 32 ? 32 : T <= 64 ? 64 : 128;
  // 128 x 256 tiles on every SM when there are enough of them, else 128 x 128 tiles with K cut until the SMs are busy
  const bool split = (long long)p.mtiles * ((N + 255) / 256) < di.sms;
  const int BN = split ? 128 : 256;
  p.ntiles = (N + BN - 1) / BN;
  if ((long long)p.mtiles * p.ntiles > (1 << 28)) return fail(SF_ERR_UNSUPPORTED, "too many tiles");
  const int tiles = p.mtiles * p.ntiles;
  p.split = 1;
  if (split)
    while (p.split < 8 && tiles * p.split * 2 <= 2 * di.sms && p.KB >= 2 * 2 * p.split) p.split *= 2;
  CUtensorMap mx, mw, my;
  memset(&my, 0, sizeof(my));
  if (!make_map(&mx, CU_TENSOR_MAP_DATA_TYPE_UINT8, X, (uint64_t)K, (uint64_t)T, (uint64_t)ldx, kBK, (uint32_t)p.rows) ||
      !make_map(&mw, CU_TENSOR_MAP_DATA_TYPE_UINT8, W, (uint64_t)K, (uint64_t)N, (uint64_t)ldw, kBK, (uint32_t)BN))
    return fail(SF_ERR_CUDA, "cuTensorMapEncodeTiled failed (T=%d N=%d K=%d)", T, N, K);
  cudaError_t e;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (split) {
    using L = Plan<true>;
    // two CTAs fit an SM; the cluster's sums (128 columns of up to 129 floats) fit the stages
    const int most = (int)((kSmemLimit / 2 - 1024 - 1024 - L::CTL) / L::stage(p.rows));
    p.stages = most > L::MAX_STAGES ? L::MAX_STAGES : most;
    e = launch<true>(mx, mw, my, p, tiles * p.split, st);
  } else {
    using L = Plan<false>;
    p.stages = 4;
    const int es = y_dtype == SF_F32 ? 4 : 2;
    p.tma_store = reinterpret_cast<uintptr_t>(Y) % 16 == 0 && (size_t)N * es % 16 == 0 &&
                  make_map(&my, y_dtype == SF_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                : y_dtype == SF_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                     : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                           Y, (uint64_t)N, (uint64_t)T, (uint64_t)N * es, 128 / es, 32);
    static_assert(L::bytes(128, 4) <= (size_t)kSmemLimit, "shared memory plan");
    e = launch<false>(mx, mw, my, p, tiles < di.sms ? tiles : di.sms, st);
  }
  if (e != cudaSuccess) return cuda_fail(e, "fp8_linear_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}
