// sf_paged_attention.cu -- attention over the pages of an e4m3 cache.
//
//   p_j = softmax_j(scale * q . k_j),  out = sum_j p_j v_j,  k_j = code * scale of its page and head
//
// The softmax keeps a running maximum m and sum l: keys in order, out and l are multiplied by e^(m - m') when the
// maximum grows to m'.
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

struct AttnArgs {
  sf_paged_cache c;
  const void* q;
  long long qts, qhs;
  void* out;
  float* lse;
  int H, T, q_dtype, out_dtype, window;
  float scale;
};

__device__ __forceinline__ float load_q(const AttnArgs& a, long long i) {
  if (a.q_dtype == SF_F32) return static_cast<const float*>(a.q)[i];
  if (a.q_dtype == SF_F16) return __half2float(static_cast<const __half*>(a.q)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(a.q)[i]);
}

// One warp per (token, query head): 32 keys at a time, a key to a lane for the scores, then D / 32 columns to a lane.
template <int D>
__global__ void __launch_bounds__(128) paged_attention_kernel(const AttnArgs a) {
  __shared__ float qs[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long w = (long long)blockIdx.x * 4 + warp;
  if (w >= (long long)a.T * a.H) return;
  const int tok = (int)(w / a.H), h = (int)(w % a.H), kvh = h / (a.H / a.c.n_kv_heads);
  for (int d = lane; d < D; d += 32) qs[warp][d] = load_q(a, tok * a.qts + h * a.qhs + d);
  __syncwarp();
  const TokenAt at = token_at(a.c, a.T, tok);
  if (!at.ok && lane == 0) atomicOr(&g_dev_error, kErrIndex);
  const int hi = at.ok ? max(at.pos + 1, 0) : 0, lo = a.window > 0 ? max(0, hi - a.window) : 0;
  float m = -INFINITY, l = 0.f, acc[D / 32] = {};
  for (int base = lo; base < hi; base += 32) {
    const int j = base + lane;
    int page = -1;
    if (j < hi) {
      page = a.c.block_table[(size_t)at.b * a.c.pages_per_seq + j / a.c.page_size];
      if (page < 0 || page >= a.c.num_pages) {
        atomicOr(&g_dev_error, kErrIndex);
        page = -1;
      }
    }
    const size_t ph = (size_t)max(page, 0) * a.c.n_kv_heads + kvh;
    const size_t row = (ph * a.c.page_size + j % a.c.page_size) * D;
    float s = -INFINITY;
    if (page >= 0) {
      s = 0.f;
      for (int d = 0; d < D; ++d) s = fmaf(qs[warp][d], from_e4m3(a.c.k_codes[row + d]), s);
      s *= a.c.k_scales[ph] * a.scale;
    }
    float bm = s;
#pragma unroll
    for (int o = 16; o; o >>= 1) bm = fmaxf(bm, __shfl_xor_sync(0xffffffffu, bm, o));
    const float mn = fmaxf(m, bm), ref = mn == -INFINITY ? 0.f : mn;
    const float corr = expf(m - ref), p = expf(s - ref);
    const float vs = page >= 0 ? a.c.v_scales[ph] : 0.f;
    float sum = p;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    l = l * corr + sum;
    m = mn;
#pragma unroll
    for (int e = 0; e < D / 32; ++e) acc[e] *= corr;
    for (int i = 0; i < 32 && base + i < hi; ++i) {
      const float pi = __shfl_sync(0xffffffffu, p * vs, i);
      const size_t ri = __shfl_sync(0xffffffffu, row, i);
      if (__shfl_sync(0xffffffffu, page, i) < 0) continue;
#pragma unroll
      for (int e = 0; e < D / 32; ++e) acc[e] = fmaf(pi, from_e4m3(a.c.v_codes[ri + lane + 32 * e]), acc[e]);
    }
  }
#pragma unroll
  for (int e = 0; e < D / 32; ++e) {
    const float y = l == 0.f ? 0.f : acc[e] / l;
    const size_t o = (size_t)w * D + lane + 32 * e;
    if (a.out_dtype == SF_F32) static_cast<float*>(a.out)[o] = y;
    else if (a.out_dtype == SF_F16) static_cast<__half*>(a.out)[o] = __float2half_rn(y);
    else static_cast<__nv_bfloat16*>(a.out)[o] = __float2bfloat16_rn(y);
  }
  if (a.lse && lane == 0) a.lse[w] = l == 0.f ? -INFINITY : m + logf(l);
}

}  // namespace
}  // namespace sf

using namespace sf;

extern "C" {

size_t sf_paged_attention_workspace_bytes(int head_dim) { return head_dim > 0 ? 16 : 0; }

int sf_paged_attention(const sf_paged_cache* cache, const void* q, int q_dtype, long long qts, long long qhs, void* out,
                       int out_dtype, float* lse, int H, int T, float scale, int window, void* workspace,
                       size_t workspace_bytes, void* stream) {
  if (int rc = check_paged(cache, T)) return rc;
  if (q_dtype < 0 || q_dtype > 2 || out_dtype < 0 || out_dtype > 2) return fail(SF_ERR_DTYPE, "unknown dtype code");
  if (H < 1 || H % cache->n_kv_heads) return fail(SF_ERR_SHAPE, "H must be a positive multiple of n_kv_heads");
  if (T == 0) return SF_OK;
  if (!q || !out || !workspace) return fail(SF_ERR_NULL, "null pointer argument");
  if (workspace_bytes < sf_paged_attention_workspace_bytes(cache->head_dim))
    return fail(SF_ERR_SHAPE, "workspace too small: need %zu bytes", sf_paged_attention_workspace_bytes(cache->head_dim));
  AttnArgs a{};
  a.c = *cache; a.q = q; a.qts = qts; a.qhs = qhs; a.out = out; a.lse = lse;
  a.H = H; a.T = T; a.q_dtype = q_dtype; a.out_dtype = out_dtype; a.window = window; a.scale = scale;
  const unsigned grid = (unsigned)(((long long)T * H + 3) / 4);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  switch (cache->head_dim) {
    case 64: paged_attention_kernel<64><<<grid, 128, 0, st>>>(a); break;
    case 96: paged_attention_kernel<96><<<grid, 128, 0, st>>>(a); break;
    case 128: paged_attention_kernel<128><<<grid, 128, 0, st>>>(a); break;
    default: paged_attention_kernel<256><<<grid, 128, 0, st>>>(a); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_fail(e, "paged_attention_kernel launch");
  g_launches.fetch_add(1, std::memory_order_relaxed);
  return SF_OK;
}

}  // extern "C"
