// sf_rms_norm.cu -- root-mean-square norm with the residual's addition, and e4m3 codes with one scale for each row
// and 128 columns.
//
//   h = x + residual,  y = h / sqrt(mean(h^2) + eps) * weight
//   scale = max|y| / 448 over 128 columns,  code = e4m3(y / scale)
//
// h stays in registers in fp32 between the sum and the output, so x and the residual are read once and the sum is
// rounded only where it is stored.
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

__device__ __forceinline__ float load_w(const NormArgs& a, int k) {
  if (!a.w) return 1.f;
  if (a.w_dtype == SF_F32) return static_cast<const float*>(a.w)[k];
  if (a.w_dtype == SF_F16) return __half2float(static_cast<const __half*>(a.w)[k]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.w)[k]);
}

// One block per row; a thread takes 8 columns at a time, so that 16 neighbouring lanes hold one 128-column group.
template <typename TX>
__global__ void __launch_bounds__(256) rms_norm_kernel(const NormArgs a) {
  __shared__ float part[8];
  const size_t row = blockIdx.x;
  const TX* x = static_cast<const TX*>(a.x) + row * a.ldx;
  const TX* r = a.r ? static_cast<const TX*>(a.r) + row * a.ldr : nullptr;
  float rstd = 1.f;
  if (a.norm) {
    float ss = 0.f;
    for (int k = threadIdx.x; k < a.K; k += 256) {
      const float h = to_f32(x[k]) + (r ? to_f32(r[k]) : 0.f);
      ss = fmaf(h, h, ss);
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = ss;
    __syncthreads();
    ss = 0.f;
    for (int i = 0; i < 8; ++i) ss += part[i];
    rstd = 1.f / sqrtf(ss / (float)a.K + a.eps);
  }
  const int G = (a.K + 127) / 128;
  for (int base = 0; base < a.K; base += 256 * 8) {
    const int k0 = base + 8 * threadIdx.x;
    float y[8];
    uint32_t amax = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int k = k0 + e;
      float h = 0.f;
      if (k < a.K) h = to_f32(x[k]) + (r ? to_f32(r[k]) : 0.f);
      if (k < a.K && a.h) static_cast<TX*>(a.h)[row * a.K + k] = from_f32<TX>(h);
      y[e] = k < a.K && a.norm ? h * rstd * load_w(a, k) : h;
      amax = max(amax, __float_as_uint(y[e]) & 0x7fffffffu);
    }
    if (a.y_dtype != SF_E4M3) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        if (k0 + e >= a.K) continue;
        const size_t o = row * a.ldy + k0 + e;
        if (a.y_dtype == SF_F32) static_cast<float*>(a.y)[o] = y[e];
        else if (a.y_dtype == SF_F16) static_cast<__half*>(a.y)[o] = __float2half_rn(y[e]);
        else static_cast<__nv_bfloat16*>(a.y)[o] = __float2bfloat16_rn(y[e]);
      }
      continue;
    }
    // the largest magnitude as an integer: infinities and NaN win, and spoil only their own group
#pragma unroll
    for (int o = 8; o; o >>= 1) amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, o));
    float scale = amax ? __uint_as_float(amax) / kE4m3Max : 1.f;
    if (scale < FLT_MIN) scale = FLT_MIN;
    if ((threadIdx.x & 15) == 0 && k0 < a.K) a.scales[row * G + k0 / 128] = scale;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (k0 + e < a.K) static_cast<uint8_t*>(a.y)[row * a.ldy + k0 + e] = to_e4m3(y[e] / scale);
  }
}

int run_norm(const NormArgs& a, int x_dtype, cudaStream_t st) {
  if (a.T == 0) return SF_OK;
  const cudaError_t e = with_type(x_dtype, [&](auto* t) {
    using TX = std::remove_const_t<std::remove_pointer_t<decltype(t)>>;
    rms_norm_kernel<TX><<<(unsigned)a.T, 256, 0, st>>>(a);
    return cudaGetLastError();
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
