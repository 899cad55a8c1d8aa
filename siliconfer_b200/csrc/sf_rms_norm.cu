// sf_rms_norm.cu -- root-mean-square norm with the residual's addition, and e4m3 codes with one scale for each row
// and 128 columns.
//
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight
//   scale = max|y| / 448 over 128 columns,  code = e4m3(y / scale)   (both quotients rounded once, to fp32)
//
// h stays in registers in fp32 between the sum and the output, so x and the residual are read once and the sum is
// rounded only where it is stored.
//
// 4096 x 8192 bf16 with the residual and e4m3 output, 236 MB, takes 52 us = 4.6 TB/s (issue slots 62 % and DRAM 45 % in use,
// waits for loads first among the stalls), 8192 x 4096 49 us; one row of 4096 2.4 us, a launch; quantizing 8192 x 4096
// 31 us.  Codes by one product with the reciprocal, which may be a step off near a tie, took 48, 46 and 2.2 us.  Rows whose
// length is no multiple of 8 take loads of one element (4096 x 4097: 70 us).
#include <atomic>
#include <cfloat>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_q4_internal.h"

namespace sf {
extern std::atomic<long long> g_launches;

namespace {

struct NormArgs {
  const void* x;
  const void* r;
  void* h;
  const void* w;
  void* y;
  float* scales;
  long long ldx, ldr, ldy;
  int T, K, w_dtype, y_dtype, norm;
  float eps;
};

// The 8 weights of columns k .. k + 7.
template <bool VEC>
__device__ __forceinline__ void load_weights(const NormArgs& a, int k, float (&w)[8]) {
  const auto from = [&](auto* p) {
    if constexpr (VEC) {
      load8(p + k, w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) w[e] = k + e < a.K ? to_f32(p[k + e]) : 0.f;
    }
  };
  if (!a.w) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
  } else if (a.w_dtype == SF_F32) {
    from(static_cast<const float*>(a.w));
  } else if (a.w_dtype == SF_F16) {
    from(static_cast<const __half*>(a.w));
  } else {
    from(static_cast<const __nv_bfloat16*>(a.w));
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_cols(const T* p, int k, int K, float (&v)[8]) {
  if constexpr (VEC) {
    if (k < K) {
      load8(p + k, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = k + e < K ? to_f32(p[k + e]) : 0.f;
  }
}
template <typename T, bool VEC>
__device__ __forceinline__ void store_cols(T* p, int k, int K, const float (&v)[8]) {
  if constexpr (VEC) {
    store8(p + k, v);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k + e < K) p[k + e] = from_f32<T>(v[e]);
  }
}

__device__ __forceinline__ float max_nan(float a, float b) {
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}

// A code is e4m3(y / scale), the quotient rounded to fp32 first: where y and the group's largest are in a simple ratio the
// quotient of their exact values is a tie between two codes, which this rounding restores (of 67 million codes of a norm
// 787 then differ from the exact values', 1150 by the unrounded quotient).  y times the reciprocal is off by at most 2^-22
// of itself (2^-23 of the reciprocal, 2^-24 of each product), so the products with a reciprocal 2^-21 smaller and larger
// have the quotient between them, and 8 columns are divided only where these round to different codes.
__device__ __forceinline__ uint2 quotient_codes(const float (&y)[8], float scale) {
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(scale));
  const float near = inv * (1 - 0x1p-21f), far = inv * (1 + 0x1p-21f);
  float lo[8], hi[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    unpack2(mul2(pack2(y[e], y[e + 1]), pack2(near, near)), lo[e], lo[e + 1]);
    unpack2(mul2(pack2(y[e], y[e + 1]), pack2(far, far)), hi[e], hi[e + 1]);
  }
  const uint2 code = to_e4m3x8(lo), other = to_e4m3x8(hi);
  if (code.x == other.x && code.y == other.y) return code;
  float q[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) q[e] = __fdiv_rn(y[e], scale);
  return to_e4m3x8(q);
}

// y of 8 columns to memory, in its type or as codes.  16 neighbouring lanes hold one 128-column group; every lane of
// the warp calls this, with k >= K where it has no columns.
template <bool VEC>
__device__ __forceinline__ void put_columns(const NormArgs& a, size_t row, int k, const float (&y)[8]) {
  if (a.y_dtype == SF_E4M3) {
    // infinities and NaN win, and spoil only their own group
    float amax = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max_nan(amax, fabsf(y[e]));
#pragma unroll
    for (int o = 8; o; o >>= 1) amax = max_nan(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    if (k >= a.K) return;
    float scale = amax == 0.f ? 1.f : amax / kE4m3Max;
    if (scale < FLT_MIN) scale = FLT_MIN;
    if ((threadIdx.x & 15) == 0) a.scales[row * ((a.K + 127) / 128) + k / 128] = scale;
    const uint2 codes = quotient_codes(y, scale);
    uint8_t* out = static_cast<uint8_t*>(a.y) + row * a.ldy + k;
    if (VEC) {
      *reinterpret_cast<uint2*>(out) = codes;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (k + e < a.K) out[e] = (uint8_t)((e < 4 ? codes.x : codes.y) >> 8 * (e % 4));
    }
    return;
  }
  if (k >= a.K) return;
  if (a.y_dtype == SF_F32) store_cols<float, VEC>(static_cast<float*>(a.y) + row * a.ldy, k, a.K, y);
  else if (a.y_dtype == SF_F16) store_cols<__half, VEC>(static_cast<__half*>(a.y) + row * a.ldy, k, a.K, y);
  else store_cols<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(a.y) + row * a.ldy, k, a.K, y);
}

// blockDim.x threads a row (whole warps), blockDim.y rows a block (several only where one warp takes a row).  A thread
// keeps CH x 8 columns of h, blockDim.x x 8 apart; with CH = 0 it reads them again for the output instead (rows of more
// than 32768).  VEC: every row starts at 16 bytes and K is a multiple of 8.
// NT: the most threads; rows of 2 chunks a
// thread keep to 40 registers so that 3 blocks of 512 fit an SM (that case 52 us; with 50 registers and 2 blocks 61).
template <typename TX, int CH, bool VEC, int NT>
__global__ void __launch_bounds__(NT, CH == 2 && NT == 512 ? 3 : 1) rms_norm_kernel(const NormArgs a) {
  __shared__ float part[32];
  griddep_wait();
  const size_t row = (size_t)blockIdx.x * blockDim.y + threadIdx.y;
  if (row >= (size_t)a.T) return;   // whole warps
  const int step = blockDim.x * 8, k0 = threadIdx.x * 8;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TX* r = a.r ? static_cast<const TX*>(a.r) + row * a.ldr : nullptr;
  TX* h_out = static_cast<TX*>(a.h) + (a.h ? row * a.K : 0);
  const auto load_h = [&](int k, float (&h)[8]) {
    load_cols<TX, VEC>(x, k, a.K, h);
    if (r) {
      float v[8];
      load_cols<TX, VEC>(r, k, a.K, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) h[e] += v[e];
    }
  };
  constexpr int KEEP = CH > 0 ? CH : 1;
  // Few rows: the weights come with the row, not after its sum (1 x 4096, fp32 weights: 0.2 us less).  With many
  // rows other blocks fill that wait, and the registers cost more (8192 x 4096 with 2 chunks: 52 us so, 45 otherwise).
  constexpr bool EARLY = CH == 1;
  float h[KEEP][8], w_kept[EARLY ? CH : 1][8], ss = 0.f;
  if constexpr (CH > 0) {
    // every load of the thread before the first use
#pragma unroll
    for (int c = 0; c < CH; ++c) load_cols<TX, VEC>(x, k0 + c * step, a.K, h[c]);
    if constexpr (EARLY) {
#pragma unroll
      for (int c = 0; c < CH; ++c)
        if (a.norm && k0 + c * step < a.K) load_weights<VEC>(a, k0 + c * step, w_kept[c]);
    }
    if (r) {
      float v[CH][8];
#pragma unroll
      for (int c = 0; c < CH; ++c) load_cols<TX, VEC>(r, k0 + c * step, a.K, v[c]);
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          unpack2(add2(pack2(h[c][e], h[c][e + 1]), pack2(v[c][e], v[c][e + 1])), h[c][e], h[c][e + 1]);
    }
    griddep_launch_dependents();
    uint64_t sq = 0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int e = 0; e < 8; e += 2) sq = fma2(pack2(h[c][e], h[c][e + 1]), pack2(h[c][e], h[c][e + 1]), sq);
    float lo, hi;
    unpack2(sq, lo, hi);
    ss = lo + hi;
  } else {
    for (int k = k0; k < a.K; k += step) {
      load_h(k, h[0]);
#pragma unroll
      for (int e = 0; e < 8; ++e) ss = fmaf(h[0][e], h[0][e], ss);
    }
  }
  float rstd = 1.f;
  if (a.norm) {
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (blockDim.x > 32) {
      if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
      __syncthreads();
      ss = (threadIdx.x & 31) < blockDim.x / 32 ? part[threadIdx.x & 31] : 0.f;
#pragma unroll
      for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    }
    rstd = 1.f / sqrtf(ss / (float)a.K + a.eps);
  }
  const auto finish = [&](int c, int k, float (&v)[8]) {
    if (k < a.K && a.h) store_cols<TX, VEC>(h_out, k, a.K, v);
    if (a.norm && k < a.K) {
      float w[8];
      if constexpr (EARLY) {
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = w_kept[c][e];
      } else {
        load_weights<VEC>(a, k, w);
      }
#pragma unroll
      for (int e = 0; e < 8; e += 2)
        unpack2(mul2(mul2(pack2(v[e], v[e + 1]), pack2(rstd, rstd)), pack2(w[e], w[e + 1])), v[e], v[e + 1]);
    }
    put_columns<VEC>(a, row, k, v);
  };
  if constexpr (CH > 0) {
#pragma unroll
    for (int c = 0; c < CH; ++c)
      if (c == 0 || c * step < a.K) finish(c, k0 + c * step, h[c]);
  } else {
    for (int base = 0; base < a.K; base += step) {
      load_h(k0 + base, h[0]);
      finish(0, k0 + base, h[0]);
    }
  }
}

int run_norm(const NormArgs& a, int x_dtype, cudaStream_t st) {
  if (a.T == 0) return SF_OK;
  const size_t xe = x_dtype == SF_F32 ? 4 : 2, ye = a.y_dtype == SF_E4M3 ? 1 : a.y_dtype == SF_F32 ? 4 : 2;
  const auto at16 = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
  const bool vec = a.K % 8 == 0 && at16(a.x) && at16(a.r) && at16(a.h) && at16(a.w) && at16(a.y) &&
                   a.ldx * xe % 16 == 0 && a.ldr * xe % 16 == 0 && (size_t)a.K * xe % 16 == 0 && a.ldy * ye % (a.y_dtype == SF_E4M3 ? 8 : 16) == 0;
  // Few rows: as many threads as the row has chunks, for the shortest chain of loads.  Many rows: 2 chunks a thread
  // (4096 x 8192, codes by one product: 48 us; 1 chunk 60, 4 chunks 52, 8 chunks 69), more where the row is too long for 512 threads.
  const int chunks = (a.K + 7) / 8;
  const bool few = a.T <= 2 * device_info().sms;
  const int ch = few && chunks <= 1024 ? 1 : chunks <= 1024 || (few && chunks <= 2048) ? 2 : chunks <= 2048 ? 4 : chunks <= 4096 ? 8 : 0;
  const int nt = ch == 0 ? 1024 : ((chunks + ch - 1) / ch + 31) / 32 * 32;
  const int rows = nt == 32 ? 4 : 1;
  const cudaError_t e = with_type(x_dtype, [&](auto* t) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    auto* fn = ch == 1   ? (vec ? rms_norm_kernel<TX, 1, true, 1024> : rms_norm_kernel<TX, 1, false, 1024>)
               : ch == 2 ? (nt <= 512 ? (vec ? rms_norm_kernel<TX, 2, true, 512> : rms_norm_kernel<TX, 2, false, 512>)
                                      : (vec ? rms_norm_kernel<TX, 2, true, 1024> : rms_norm_kernel<TX, 2, false, 1024>))
               : ch == 4 ? (vec ? rms_norm_kernel<TX, 4, true, 512> : rms_norm_kernel<TX, 4, false, 512>)
               : ch == 8 ? (vec ? rms_norm_kernel<TX, 8, true, 512> : rms_norm_kernel<TX, 8, false, 512>)
                         : (vec ? rms_norm_kernel<TX, 0, true, 1024> : rms_norm_kernel<TX, 0, false, 1024>);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(((long long)a.T + rows - 1) / rows));
    cfg.blockDim = dim3((unsigned)nt, (unsigned)rows);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, fn, a);
  });
  if (e != cudaSuccess) return cuda_fail(e, "rms_norm_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

int sf_rms_norm(const void* x, int x_dtype, long long ldx, const void* residual, long long ldr, void* h_out,
                const void* weight, int w_dtype, float eps, void* y, int y_dtype, long long ldy, float* scales, int T,
                int K, void* stream) {
  if (T < 0 || K < 1) return fail(SF_ERR_SHAPE, "need T >= 0 and K >= 1");
  if (x_dtype < 0 || x_dtype > 2 || y_dtype < 0 || y_dtype > 3 || (weight && (w_dtype < 0 || w_dtype > 2)))
    return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (T > 0 && (!x || !y || (y_dtype == SF_E4M3 && !scales))) return fail(SF_ERR_NULL, "null pointer argument");
  if (T > 0 && !residual != !h_out) return fail(SF_ERR_NULL, "residual and h_out go together");
  if (ldx < K || ldy < K || (residual && ldr < K)) return fail(SF_ERR_SHAPE, "a row stride is below K");
  NormArgs a{};
  a.x = x; a.r = residual; a.h = h_out; a.w = weight; a.y = y; a.scales = scales;
  a.ldx = ldx; a.ldr = ldr; a.ldy = ldy;
  a.T = T; a.K = K; a.w_dtype = w_dtype; a.y_dtype = y_dtype; a.norm = 1; a.eps = eps;
  return run_norm(a, x_dtype, static_cast<cudaStream_t>(stream));
}

int sf_quantize_e4m3(const void* x, int x_dtype, long long ldx, uint8_t* codes, long long ldy, float* scales, int T,
                     int K, void* stream) {
  if (T < 0 || K < 1) return fail(SF_ERR_SHAPE, "need T >= 0 and K >= 1");
  if (x_dtype < 0 || x_dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (T > 0 && (!x || !codes || !scales)) return fail(SF_ERR_NULL, "null pointer argument");
  if (ldx < K || ldy < K) return fail(SF_ERR_SHAPE, "a row stride is below K");
  NormArgs a{};
  a.x = x; a.y = codes; a.scales = scales; a.ldx = ldx; a.ldy = ldy;
  a.T = T; a.K = K; a.y_dtype = SF_E4M3; a.norm = 0;
  return run_norm(a, x_dtype, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
