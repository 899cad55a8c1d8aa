// sf_fp8_linear.cu -- Y = X W^T over e4m3 rows (one scale per row and 128 columns) and e4m3 weights (one scale per
// 128 x 128 block), accumulated in fp32.
#include <atomic>
#include <cstdint>

#include "sf_e4m3.h"
#include "sf_q4_internal.h"

namespace sf {
SF_DEFINE_ERROR_READER(take_dev_error_fp8)
extern std::atomic<long long> g_launches;

namespace {

struct Fp8Args {
  const uint8_t* X;
  const uint8_t* W;
  const float* xs;
  const float* ws;
  const float* bias;
  void* Y;
  long long ldx, ldw;
  int T, N, K, y_dtype;
};

// 64 tokens x 64 rows per block, 4 x 4 outputs per thread; tiles of 32 k are decoded into shared memory.
__global__ void __launch_bounds__(256) fp8_linear_kernel(const Fp8Args a) {
  __shared__ float xt[32][65], wt[32][65];
  const int t0 = blockIdx.y * 64, n0 = blockIdx.x * 64, KB = (a.K + 127) / 128;
  const int ty = threadIdx.x / 16, tx = threadIdx.x % 16;
  float acc[4][4] = {};
  for (int k0 = 0; k0 < a.K; k0 += 32) {
    for (int i = threadIdx.x; i < 64 * 32; i += 256) {
      const int r = i / 32, k = k0 + i % 32, t = t0 + r, n = n0 + r;
      xt[i % 32][r] = t < a.T && k < a.K ? from_e4m3(a.X[t * a.ldx + k]) * a.xs[(size_t)t * KB + k / 128] : 0.f;
      wt[i % 32][r] = n < a.N && k < a.K ? from_e4m3(a.W[n * a.ldw + k]) * a.ws[(size_t)(n / 128) * KB + k / 128] : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 32; ++k)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xt[k][ty + 16 * i], wt[k][tx + 16 * j], acc[i][j]);
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int t = t0 + ty + 16 * i, n = n0 + tx + 16 * j;
      if (t >= a.T || n >= a.N) continue;
      const float y = acc[i][j] + (a.bias ? a.bias[n] : 0.f);
      const size_t o = (size_t)t * a.N + n;
      if (a.y_dtype == SF_F32) static_cast<float*>(a.Y)[o] = y;
      else if (a.y_dtype == SF_F16) static_cast<__half*>(a.Y)[o] = __float2half_rn(y);
      else static_cast<__nv_bfloat16*>(a.Y)[o] = __float2bfloat16_rn(y);
    }
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
  const Fp8Args a{X, W, xs, ws, bias, Y, ldx, ldw, T, N, K, y_dtype};
  const dim3 grid((unsigned)((N + 63) / 64), (unsigned)((T + 63) / 64));
  fp8_linear_kernel<<<grid, 256, 0, static_cast<cudaStream_t>(stream)>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "fp8_linear_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}
