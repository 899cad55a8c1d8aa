// sf_torch_ext.cpp -- the thin PyTorch binding of the C ABI (include/sf_q4.h).
//
// Q4Linear.__call__ (siliconfer/model/q4_linear.py:49-68) reaches its kernel
// through the reference's pybind module (siliconfer/kernels/neon/
// bindings.cpp:97-150), which checks shapes, allocates the output and throws
// std::runtime_error on a mismatch.  This module is the same layer for torch
// tensors on the GPU: it checks devices, shapes and dtypes, allocates Y with
// torch, runs the library's entry point on torch's current CUDA stream and
// turns a status code into RuntimeError with the library's message.  No
// computation happens here.
#include <torch/extension.h>
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <climits>
#include <cmath>
#include <stdexcept>
#include <string>
#include <vector>

#include "sf_q4.h"

namespace {

int dtype_code(const at::ScalarType t) {
  switch (t) {
    case at::kFloat: return SF_F32;
    case at::kHalf: return SF_F16;
    case at::kBFloat16: return SF_BF16;
    default: throw std::runtime_error("unsupported activation dtype (fp32, fp16 or bf16)");
  }
}

void check(int rc) {
  if (rc != SF_OK) throw std::runtime_error(std::string(sf_last_error()));
}

const void* ptr_or_null(const c10::optional<at::Tensor>& t) {
  return t.has_value() && t->defined() ? t->data_ptr() : nullptr;
}

void check_weights(const at::Tensor& W, const at::Tensor& S, const c10::optional<at::Tensor>& Z,
                   const c10::optional<at::Tensor>& bias, const at::Tensor& X) {
  TORCH_CHECK(W.is_cuda() && S.is_cuda() && X.is_cuda(), "W, scales and X must be CUDA tensors");
  TORCH_CHECK(W.dim() == 2 && S.dim() == 2 && X.dim() == 2, "W, scales and X must be 2-D");
  TORCH_CHECK(W.scalar_type() == at::kByte && S.scalar_type() == at::kFloat, "W must be uint8, scales fp32");
  TORCH_CHECK(W.is_contiguous() && S.is_contiguous() && X.is_contiguous(), "tensors must be contiguous");
  TORCH_CHECK(W.get_device() == X.get_device() && S.get_device() == X.get_device(), "tensors on one device");
  if (Z.has_value() && Z->defined())
    TORCH_CHECK(Z->is_cuda() && Z->scalar_type() == at::kFloat && Z->is_contiguous() && Z->sizes() == S.sizes(),
                "zeros must be a contiguous fp32 CUDA tensor shaped like scales");
  if (bias.has_value() && bias->defined())
    TORCH_CHECK(bias->is_cuda() && bias->scalar_type() == at::kFloat && bias->is_contiguous(),
                "bias must be a contiguous fp32 CUDA tensor");
}

// Y[T, N] = X[T, K] @ dequant(W)^T (+ bias): sf_q4_linear (4 bits) or sf_q2_linear (2 bits).
at::Tensor linear(const at::Tensor& W, const at::Tensor& S, const c10::optional<at::Tensor>& Z,
                  const c10::optional<at::Tensor>& bias, const at::Tensor& X, int64_t group_size,
                  at::ScalarType out_dtype, int64_t bits, bool pdl) {
  check_weights(W, S, Z, bias, X);
  TORCH_CHECK(bits == 4 || bits == 2, "bits must be 4 or 2");
  const c10::cuda::CUDAGuard guard(X.device());
  const int64_t T = X.size(0), K = X.size(1), N = W.size(0);
  TORCH_CHECK(W.size(1) * (8 / bits) == K, "X/W in_features mismatch");
  at::Tensor Y = at::empty({T, N}, X.options().dtype(out_dtype));
  void* st = at::cuda::getCurrentCUDAStream(X.get_device()).stream();
  const auto* w = static_cast<const uint8_t*>(W.data_ptr());
  const auto* s = static_cast<const float*>(S.data_ptr());
  const auto* z = static_cast<const float*>(ptr_or_null(Z));
  const auto* b = static_cast<const float*>(ptr_or_null(bias));
  if (bits == 2)
    check(sf_q2_linear(w, s, z, b, X.data_ptr(), dtype_code(X.scalar_type()), Y.data_ptr(), dtype_code(out_dtype),
                       (int)N, (int)K, (int)T, (int)group_size, st));
  else
    check(sf_q4_linear(w, s, z, b, X.data_ptr(), dtype_code(X.scalar_type()), Y.data_ptr(), dtype_code(out_dtype),
                       (int)N, (int)K, (int)T, (int)group_size, pdl ? SF_FLAG_PDL : 0, st));
  return Y;
}

// silu(gate) * up over interleaved gate/up rows (sf_q4_linear_swiglu); W has 2N rows.
at::Tensor linear_swiglu(const at::Tensor& W, const at::Tensor& S, const c10::optional<at::Tensor>& Z,
                         const c10::optional<at::Tensor>& bias, const at::Tensor& X, int64_t group_size,
                         at::ScalarType out_dtype) {
  check_weights(W, S, Z, bias, X);
  const c10::cuda::CUDAGuard guard(X.device());
  const int64_t T = X.size(0), K = X.size(1), N = W.size(0) / 2;
  TORCH_CHECK(W.size(1) * 2 == K, "X/W in_features mismatch");
  at::Tensor Y = at::empty({T, N}, X.options().dtype(out_dtype));
  check(sf_q4_linear_swiglu(static_cast<const uint8_t*>(W.data_ptr()), static_cast<const float*>(S.data_ptr()),
                            static_cast<const float*>(ptr_or_null(Z)), static_cast<const float*>(ptr_or_null(bias)),
                            X.data_ptr(), dtype_code(X.scalar_type()), Y.data_ptr(), dtype_code(out_dtype), (int)N,
                            (int)K, (int)T, (int)group_size, at::cuda::getCurrentCUDAStream(X.get_device()).stream()));
  return Y;
}

// ---- 8-bit decoder operators ------------------------------------------------

using OptTensor = c10::optional<at::Tensor>;

bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

void* stream_of(const at::Tensor& t) { return at::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

void on_device(const at::Tensor& t, const at::Tensor& ref, const char* name) {
  TORCH_CHECK(t.is_cuda(), name, " must be a CUDA tensor");
  TORCH_CHECK(t.get_device() == ref.get_device(), name, " must be on the same device as the other tensors");
}

bool is_codes(const at::Tensor& t) {
  return t.scalar_type() == at::kFloat8_e4m3fn || t.scalar_type() == at::kByte;
}

// [..., K] as rows of K contiguous elements with one row stride (a copy where the layout does not allow it).
struct RowView {
  at::Tensor t;
  int64_t rows, K, ld;
};
RowView rows_of(const at::Tensor& x, const char* name) {
  TORCH_CHECK(x.dim() >= 1 && x.size(-1) >= 1, name, " must have at least one column");
  const int64_t K = x.size(-1);
  at::Tensor y = x.dim() == 2 ? x : x.reshape({x.numel() / K, K});
  if ((K > 1 && y.stride(1) != 1) || (y.size(0) > 1 && y.stride(0) < K)) y = y.contiguous();
  TORCH_CHECK(y.size(0) <= INT_MAX && K <= INT_MAX, name, " is too large");
  return {y, y.size(0), K, y.size(0) > 1 ? y.stride(0) : K};
}
// `t` [rows, n] in the shape [..., n] of x's leading dimensions.
at::Tensor like_rows(const at::Tensor& t, const at::Tensor& x) {
  if (x.dim() == 2) return t;
  auto sizes = x.sizes().vec();
  sizes.back() = t.size(1);
  return t.view(sizes);
}
// Uninitialised tensors on ref's device.
at::Tensor empty_on(at::IntArrayRef sizes, at::ScalarType dtype, const at::Tensor& ref) {
  return at::detail::empty_cuda(sizes, dtype, ref.device(), c10::nullopt);
}
// Code rows that start at multiples of 16 bytes.
at::Tensor empty_codes(int64_t T, int64_t K, const at::Tensor& ref) {
  return at::detail::empty_strided_cuda({T, K}, {(K + 15) / 16 * 16, 1}, at::kFloat8_e4m3fn, ref.device());
}

std::tuple<at::Tensor, OptTensor, OptTensor> rms_norm(const at::Tensor& x, const OptTensor& weight, double eps,
                                                      const OptTensor& residual, c10::optional<at::ScalarType> out_dtype,
                                                      bool e4m3) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  const RowView v = rows_of(x, "x");
  RowView r{};
  if (given(residual)) {
    on_device(*residual, x, "residual");
    TORCH_CHECK(residual->sizes() == x.sizes() && residual->scalar_type() == x.scalar_type(),
                "residual must have x's shape and dtype");
    r = rows_of(*residual, "residual");
  }
  at::Tensor w;
  if (given(weight)) {
    on_device(*weight, x, "weight");
    TORCH_CHECK(weight->dim() == 1 && weight->size(0) == v.K, "weight must be [K]");
    w = weight->contiguous();
  }
  const int xdt = dtype_code(x.scalar_type()), wdt = w.defined() ? dtype_code(w.scalar_type()) : SF_F32;
  OptTensor h, scales;
  if (r.t.defined()) h = empty_on({v.rows, v.K}, x.scalar_type(), x);
  at::Tensor y;
  int ydt = SF_E4M3;
  if (e4m3) {
    y = empty_codes(v.rows, v.K, x);
    scales = empty_on({v.rows, (v.K + 127) / 128}, at::kFloat, x);
  } else {
    const at::ScalarType yt = out_dtype.value_or(x.scalar_type());
    ydt = dtype_code(yt);
    y = empty_on({v.rows, v.K}, yt, x);
  }
  check(sf_rms_norm(v.t.data_ptr(), xdt, v.ld, r.t.defined() ? r.t.data_ptr() : nullptr, r.ld,
                    h ? h->data_ptr() : nullptr, w.defined() ? w.data_ptr() : nullptr, wdt, (float)eps, y.data_ptr(), ydt,
                    e4m3 ? (v.K + 15) / 16 * 16 : v.K, e4m3 ? scales->data_ptr<float>() : nullptr, (int)v.rows, (int)v.K,
                    stream_of(x)));
  if (h) h = like_rows(*h, x);
  if (scales) scales = like_rows(*scales, x);
  return {like_rows(y, x), scales, h};
}

std::tuple<at::Tensor, at::Tensor> quantize_e4m3(const at::Tensor& x) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  const c10::cuda::CUDAGuard guard(x.device());
  const RowView v = rows_of(x, "x");
  at::Tensor y = empty_codes(v.rows, v.K, x);
  at::Tensor scales = empty_on({v.rows, (v.K + 127) / 128}, at::kFloat, x);
  check(sf_quantize_e4m3(v.t.data_ptr(), dtype_code(x.scalar_type()), v.ld, static_cast<uint8_t*>(y.data_ptr()),
                         (v.K + 15) / 16 * 16, scales.data_ptr<float>(), (int)v.rows, (int)v.K, stream_of(x)));
  return {like_rows(y, x), like_rows(scales, x)};
}

at::Tensor fp8_linear(const at::Tensor& X, const at::Tensor& xs, const at::Tensor& W, const at::Tensor& ws,
                      const OptTensor& bias, at::ScalarType out_dtype) {
  TORCH_CHECK(X.is_cuda(), "x must be a CUDA tensor");
  on_device(xs, X, "x_scales");
  on_device(W, X, "w");
  on_device(ws, X, "w_scales");
  TORCH_CHECK(is_codes(X) && is_codes(W), "x and w must hold e4m3 codes (float8_e4m3fn or uint8)");
  TORCH_CHECK(xs.scalar_type() == at::kFloat && ws.scalar_type() == at::kFloat, "the scales must be fp32");
  const c10::cuda::CUDAGuard guard(X.device());
  const RowView x = rows_of(X, "x");
  TORCH_CHECK(W.dim() == 2 && W.size(1) == x.K, "w must be [N, K] with x's K");
  const int64_t N = W.size(0), KB = (x.K + 127) / 128;
  TORCH_CHECK(N <= INT_MAX, "w is too large");
  TORCH_CHECK(W.stride(1) == 1 || x.K == 1, "w's rows must be contiguous");
  TORCH_CHECK(xs.dim() >= 1 && xs.size(-1) == KB && xs.numel() == x.rows * KB,
              "x_scales must be [..., ceil(K / 128)] for x's rows");
  TORCH_CHECK(ws.dim() == 2 && ws.size(0) == (N + 127) / 128 && ws.size(1) == KB,
              "w_scales must be [ceil(N / 128), ceil(K / 128)]");
  const at::Tensor xsc = xs.contiguous(), wsc = ws.contiguous();
  at::Tensor b;
  if (given(bias)) {
    on_device(*bias, X, "bias");
    TORCH_CHECK(bias->scalar_type() == at::kFloat && bias->dim() == 1 && bias->size(0) == N, "bias must be fp32 [N]");
    b = bias->contiguous();
  }
  at::Tensor Y = empty_on({x.rows, N}, out_dtype, X);
  // a single row's stride has no meaning: the kernel is told one that its loads accept
  const int64_t ldx = x.rows > 1 ? x.ld : (x.K + 15) / 16 * 16, ldw = N > 1 ? W.stride(0) : (x.K + 15) / 16 * 16;
  check(sf_fp8_linear(static_cast<const uint8_t*>(x.t.data_ptr()), ldx, xsc.data_ptr<float>(),
                      static_cast<const uint8_t*>(W.data_ptr()), ldw, wsc.data_ptr<float>(),
                      b.defined() ? b.data_ptr<float>() : nullptr, Y.data_ptr(), dtype_code(out_dtype), (int)x.rows,
                      (int)N, (int)x.K, stream_of(X)));
  return like_rows(Y, X);
}

void check_table(const at::Tensor& table, const at::Tensor& ref, int64_t D) {
  on_device(table, ref, "table");
  TORCH_CHECK(table.scalar_type() == at::kFloat && table.dim() == 2 && table.is_contiguous(),
              "table must be a contiguous fp32 [max_pos, rot]");
  TORCH_CHECK(table.size(1) <= D && table.size(1) % 2 == 0, "rot must be even and at most head_dim");
  TORCH_CHECK(table.size(0) >= 1 && table.size(0) <= INT_MAX, "table must have between 1 and 2^31 - 1 positions");
}

at::Tensor rotary(const at::Tensor& x, const at::Tensor& positions, const at::Tensor& table, bool interleaved,
                  const OptTensor& out) {
  TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
  TORCH_CHECK(x.dim() == 3 && x.size(2) >= 1, "x must be [T, heads, head_dim]");
  const int64_t T = x.size(0), H = x.size(1), D = x.size(2);
  on_device(positions, x, "positions");
  TORCH_CHECK(positions.dim() == 1 && positions.size(0) == T, "positions must be [T]");
  TORCH_CHECK(positions.scalar_type() == at::kInt || positions.scalar_type() == at::kLong,
              "positions must be int32 or int64");
  check_table(table, x, D);
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y;
  if (given(out)) {
    y = *out;
    on_device(y, x, "out");
    TORCH_CHECK(y.sizes() == x.sizes() && y.scalar_type() == x.scalar_type(), "out must have x's shape and dtype");
    TORCH_CHECK(y.stride(2) == 1 || D == 1, "out's heads must be contiguous");
  }
  const at::Tensor xi = x.stride(2) == 1 || D == 1 ? x : x.contiguous();
  if (!y.defined()) y = empty_on({T, H, D}, x.scalar_type(), x);
  TORCH_CHECK(y.data_ptr() != xi.data_ptr() || y.strides() == xi.strides(),
              "out may be x itself, but no other view of x's memory");
  const at::Tensor pos = positions.contiguous();
  check(sf_rotary(xi.data_ptr(), dtype_code(x.scalar_type()), xi.stride(0), xi.stride(1), y.data_ptr(), y.stride(0),
                  y.stride(1), pos.data_ptr(), pos.scalar_type() == at::kLong, table.data_ptr<float>(),
                  (int)table.size(0), (int)table.size(1), interleaved, (int)T, (int)H, (int)D, stream_of(x)));
  return y;
}

// The cache's tensors as the C struct; `keep` holds copies alive that had to be made.
sf_paged_cache paged_cache(const at::Tensor& kc, const at::Tensor& ks, const at::Tensor& vc, const at::Tensor& vs,
                           const at::Tensor& bt, const at::Tensor& lens, const OptTensor& starts, const at::Tensor& ref,
                           std::vector<at::Tensor>& keep) {
  on_device(kc, ref, "k_codes");
  on_device(vc, ref, "v_codes");
  on_device(ks, ref, "k_scales");
  on_device(vs, ref, "v_scales");
  on_device(bt, ref, "block_table");
  on_device(lens, ref, "seq_lens");
  TORCH_CHECK(is_codes(kc) && is_codes(vc) && kc.dim() == 4 && kc.sizes() == vc.sizes() && kc.is_contiguous() &&
                  vc.is_contiguous(),
              "k_codes and v_codes must be contiguous e4m3 [pages, n_kv_heads, page_size, head_dim]");
  TORCH_CHECK(ks.scalar_type() == at::kFloat && vs.scalar_type() == at::kFloat && ks.is_contiguous() &&
                  vs.is_contiguous() && ks.dim() == 2 && ks.size(0) == kc.size(0) && ks.size(1) == kc.size(1) &&
                  vs.sizes() == ks.sizes(),
              "k_scales and v_scales must be contiguous fp32 [pages, n_kv_heads]");
  TORCH_CHECK(bt.scalar_type() == at::kInt && bt.dim() == 2, "block_table must be int32 [batch, pages_per_seq]");
  TORCH_CHECK(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == bt.size(0),
              "seq_lens must be int32 [batch]");
  for (int i = 0; i < 4; ++i) TORCH_CHECK(kc.size(i) <= INT_MAX, "the cache is too large");
  TORCH_CHECK(bt.size(1) <= INT_MAX && bt.size(0) <= INT_MAX, "block_table is too large");
  keep.push_back(bt.contiguous());
  keep.push_back(lens.contiguous());
  sf_paged_cache c{};
  c.k_codes = static_cast<uint8_t*>(kc.data_ptr());
  c.k_scales = ks.data_ptr<float>();
  c.v_codes = static_cast<uint8_t*>(vc.data_ptr());
  c.v_scales = vs.data_ptr<float>();
  c.block_table = keep[0].data_ptr<int>();
  c.seq_lens = keep[1].data_ptr<int>();
  if (given(starts)) {
    on_device(*starts, ref, "starts");
    TORCH_CHECK(starts->scalar_type() == at::kInt && starts->dim() == 1 && starts->size(0) == bt.size(0) + 1,
                "starts must be int32 [batch + 1]");
    keep.push_back(starts->contiguous());
    c.starts = keep[2].data_ptr<int>();
  }
  c.num_pages = (int)kc.size(0);
  c.n_kv_heads = (int)kc.size(1);
  c.page_size = (int)kc.size(2);
  c.head_dim = (int)kc.size(3);
  c.batch = (int)bt.size(0);
  c.pages_per_seq = (int)bt.size(1);
  return c;
}

at::Tensor head_rows(const at::Tensor& x) { return x.stride(2) == 1 ? x : x.contiguous(); }

OptTensor paged_append(const at::Tensor& k, const at::Tensor& v, const at::Tensor& kc, const at::Tensor& ks,
                       const at::Tensor& vc, const at::Tensor& vs, const at::Tensor& bt, const at::Tensor& lens,
                       const OptTensor& starts, const OptTensor& q, const OptTensor& table, bool interleaved) {
  TORCH_CHECK(k.is_cuda(), "k must be a CUDA tensor");
  on_device(v, k, "v");
  std::vector<at::Tensor> keep;
  const sf_paged_cache c = paged_cache(kc, ks, vc, vs, bt, lens, starts, k, keep);
  TORCH_CHECK(k.dim() == 3 && k.size(1) == c.n_kv_heads && k.size(2) == c.head_dim && v.sizes() == k.sizes() &&
                  v.scalar_type() == k.scalar_type(),
              "k and v must be [T, n_kv_heads, head_dim] of one dtype");
  TORCH_CHECK(k.size(0) <= INT_MAX, "k is too large");
  const c10::cuda::CUDAGuard guard(k.device());
  const at::Tensor ki = head_rows(k), vi = head_rows(v);
  at::Tensor qi, qo;
  if (given(q)) {
    on_device(*q, k, "q");
    TORCH_CHECK(given(table), "q is only turned: it needs a rotary table");
    TORCH_CHECK(q->dim() == 3 && q->size(0) == k.size(0) && q->size(2) == c.head_dim &&
                    q->scalar_type() == k.scalar_type(),
                "q must be [T, heads, head_dim] of k's dtype");
    qi = head_rows(*q);
    qo = empty_on(q->sizes(), q->scalar_type(), k);
  }
  if (given(table)) check_table(*table, k, c.head_dim);
  check(sf_paged_append(&c, ki.data_ptr(), ki.stride(0), ki.stride(1), vi.data_ptr(), vi.stride(0), vi.stride(1),
                        qi.defined() ? qi.data_ptr() : nullptr, qi.defined() ? qi.stride(0) : 0,
                        qi.defined() ? qi.stride(1) : 0, qo.defined() ? qo.data_ptr() : nullptr,
                        dtype_code(k.scalar_type()), qi.defined() ? (int)qi.size(1) : 0, (int)k.size(0),
                        given(table) ? table->data_ptr<float>() : nullptr, given(table) ? (int)table->size(0) : 0,
                        given(table) ? (int)table->size(1) : 0, interleaved, stream_of(k)));
  return qo.defined() ? OptTensor(qo) : OptTensor();
}

std::tuple<at::Tensor, OptTensor> paged_attention(const at::Tensor& q, const at::Tensor& kc, const at::Tensor& ks,
                                                  const at::Tensor& vc, const at::Tensor& vs, const at::Tensor& bt,
                                                  const at::Tensor& lens, const OptTensor& starts,
                                                  c10::optional<double> scale, int64_t window,
                                                  c10::optional<at::ScalarType> out_dtype, bool return_lse) {
  TORCH_CHECK(q.is_cuda(), "q must be a CUDA tensor");
  std::vector<at::Tensor> keep;
  const sf_paged_cache c = paged_cache(kc, ks, vc, vs, bt, lens, starts, q, keep);
  TORCH_CHECK(q.dim() == 3 && q.size(2) == c.head_dim, "q must be [T, heads, head_dim]");
  TORCH_CHECK(q.size(0) <= INT_MAX && q.size(1) <= INT_MAX, "q is too large");
  TORCH_CHECK(window <= INT_MAX, "window is too large");
  const c10::cuda::CUDAGuard guard(q.device());
  const at::Tensor qi = head_rows(q);
  const at::ScalarType ot = out_dtype.value_or(q.scalar_type());
  at::Tensor out = empty_on(q.sizes(), ot, q);
  OptTensor lse;
  if (return_lse) lse = empty_on({q.size(0), q.size(1)}, at::kFloat, q);
  const size_t bytes = sf_paged_attention_workspace_bytes(c.head_dim);
  at::Tensor ws = empty_on({(int64_t)bytes}, at::kByte, q);
  const double s = scale.has_value() ? *scale : 1.0 / std::sqrt((double)c.head_dim);
  check(sf_paged_attention(&c, qi.data_ptr(), dtype_code(q.scalar_type()), qi.stride(0), qi.stride(1), out.data_ptr(),
                           dtype_code(ot), return_lse ? lse->data_ptr<float>() : nullptr, (int)q.size(1), (int)q.size(0),
                           (float)s, window > 0 ? (int)window : 0, ws.data_ptr(), bytes, stream_of(q)));
  return {out, lse};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "torch binding of libsf_q4 (include/sf_q4.h)";
  m.def("linear", &linear, "Y = X @ dequant(W)^T (+ bias) on the GPU", py::arg("W"), py::arg("scales"),
        py::arg("zeros"), py::arg("bias"), py::arg("X"), py::arg("group_size"), py::arg("out_dtype"),
        py::arg("bits") = 4, py::arg("pdl") = false);
  m.def("linear_swiglu", &linear_swiglu, "silu(gate) * up over interleaved gate/up rows", py::arg("W"),
        py::arg("scales"), py::arg("zeros"), py::arg("bias"), py::arg("X"), py::arg("group_size"),
        py::arg("out_dtype"));
  m.def("rms_norm", &rms_norm, "RMS norm with the residual's addition -> (y, scales or None, h or None)");
  m.def("quantize_e4m3", &quantize_e4m3, "e4m3 codes and scales of each row's 128-column groups");
  m.def("fp8_linear", &fp8_linear, "product of e4m3 rows with an e4m3 weight in 128 x 128 blocks");
  m.def("rotary", &rotary, "rotary positions");
  m.def("paged_append", &paged_append, "rotary positions, and keys and values into the pages of an e4m3 cache");
  m.def("paged_attention", &paged_attention, "attention over the pages of an e4m3 cache -> (out, lse or None)");
}
