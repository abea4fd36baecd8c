// torch_ops8.cpp -- the bodies of the pi05_w8a8 PyTorch ops (8-bit serving) on
// top of the C ABI of libw4a4_sm100.so.  Schemas and fakes are defined from
// Python, in w8a8/extension.py; as in torch_ops.cpp the bodies are registered
// under CompositeExplicitAutograd, so CPU tensors reach the checks below.

#include <torch/library.h>

#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/AutogradState.h>
#include <c10/util/Exception.h>

#include <cstdint>
#include <optional>
#include <tuple>
#include <vector>

#include "w4a4_sm100.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t kBlock = 16;  // cache tokens that share a scale

void check_status(int status) {
  if (status == W4A4_OK) return;
  char buf[1024];
  w4a4_last_error(buf, sizeof(buf));
  TORCH_CHECK(false, buf, " (status ", status, ")");
}

int32_t dtype_code(at::ScalarType t, bool fp32_too, const char* what) {
  if (t == at::kHalf) return W4A4_F16;
  if (t == at::kBFloat16) return W4A4_BF16;
  if (t == at::kFloat && fp32_too) return W4A4_F32;
  TORCH_CHECK(false, what, " must be float16", fp32_too ? ", bfloat16 or float32" : " or bfloat16", ", got ", t);
}

void check_cuda(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), "pi05_w8a8 expects CUDA tensors: ", what, " is on ", t.device());
}

void check_device(const Tensor& t, const Tensor& x, const char* what) {
  TORCH_CHECK(t.device() == x.device(), what, " is on ", t.device(), " but the input is on ", x.device());
}

// The results have no gradient: an input that wants one, or that carries a
// forward-mode tangent, would silently lose it.
void check_no_gradient(const Tensor& t, const char* what) {
  TORCH_CHECK(!t.requires_grad() || !at::GradMode::is_enabled(),
              "the pi05_w8a8 ops have no gradient, but ", what, " requires one: call them under torch.no_grad()");
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined() || !c10::AutogradState::get_tls_state().get_fw_grad_mode(),
              "the pi05_w8a8 ops have no gradient, but ", what, " carries a forward-mode tangent: give them its primal");
}

int32_t as_i32(int64_t v, const char* what) {
  TORCH_CHECK(v <= INT32_MAX, what, " is too large: ", v);
  return static_cast<int32_t>(v);
}

cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }

// A contiguous tensor on x's device, without the dispatcher's way to the same function.
Tensor empty_on(const Tensor& x, at::IntArrayRef size, at::ScalarType type) {
  return at::detail::empty_cuda(size, type, x.device(), std::nullopt);
}

// x [..., h] as rows [m, h] with unit inner stride: x itself where its strides allow it (no view is made of it), else
// a copy.
struct Rows {
  Tensor t;
  int64_t m, ld;
  const void* data() const { return t.const_data_ptr(); }
};
Rows rows_of(const Tensor& x) {
  const auto size = x.sizes(), stride = x.strides();
  const int64_t h = size.back(), m = x.numel() / h;
  int64_t ld = h, next = -1;  // ld: the stride of the innermost dimension with more than one entry
  bool fits = stride.back() == 1 || h == 1;
  for (int64_t d = x.dim() - 2; d >= 0 && fits; --d) {
    if (size[d] == 1) continue;
    if (next < 0) ld = next = stride[d];
    fits = stride[d] == next && ld >= h;
    next *= size[d];
  }
  if (fits) return {x, m, ld};
  return {x.contiguous(), m, h};
}

// int8 of x's shape whose rows begin at multiples of 128 bytes, the product's
// steps (a step of an unaligned row takes two lines of L2), or of 16 bytes
// where a row is no longer than that.
Tensor empty_codes(const Tensor& x, int64_t m, int64_t* ld) {
  const int64_t h = x.size(-1);
  *ld = h <= 128 ? (h + 15) / 16 * 16 : (h + 127) / 128 * 128;
  if (*ld == h) return empty_on(x, x.sizes(), at::kChar);
  std::vector<int64_t> stride(x.dim(), 1);
  int64_t step = *ld;
  for (int64_t i = x.dim() - 2; i >= 0; --i) {
    stride[i] = step;
    step *= x.size(i);
  }
  return empty_on(x, {m * *ld}, at::kChar).as_strided(x.sizes(), stride);
}

void check_rows(const Tensor& x, const char* what) {
  check_cuda(x, what);
  TORCH_CHECK(x.dim() > 0 && x.size(-1) > 0, what, " needs a non-empty last dimension");
}

// A parameter of a row operator: [h], or [b, h] for an input [b, ..., h].
struct Param {
  Tensor t;
  const void* ptr = nullptr;
  int64_t stride = 0;  // elements from one observation's row to the next (0: shared)
};
Param param(const OptTensor& p, const Tensor& x, at::ScalarType type, const char* what) {
  Param r;
  if (!p.has_value()) return r;
  const int64_t h = x.size(-1);
  check_device(*p, x, what);
  check_no_gradient(*p, what);
  TORCH_CHECK(p->scalar_type() == type, what, " must be ", type, ", got ", p->scalar_type());
  const bool per_obs = p->dim() == 2;
  TORCH_CHECK((p->dim() == 1 || (per_obs && x.dim() >= 2 && p->size(0) == x.size(0))) && p->size(-1) == h, what,
              " must be [", h, "] or [batch, ", h, "] for an input [batch, ..., ", h, "], got ", p->sizes());
  r.t = p->stride(-1) == 1 || h == 1 ? *p : p->contiguous();
  r.ptr = r.t.const_data_ptr();
  r.stride = per_obs ? r.t.stride(0) : 0;
  return r;
}

std::tuple<Tensor, Tensor, Tensor> rms_norm_quant(const Tensor& x, const Tensor& gain, double eps,
                                                  const OptTensor& delta, const OptTensor& gate,
                                                  const OptTensor& shift) {
  check_rows(x, "x");
  check_no_gradient(x, "x");
  if (delta.has_value()) check_no_gradient(*delta, "delta");
  const int32_t dt = dtype_code(x.scalar_type(), true, "x");
  if (delta.has_value()) {
    check_device(*delta, x, "delta");
    TORCH_CHECK(delta->sizes() == x.sizes() && delta->scalar_type() == x.scalar_type(),
                "delta must have x's shape and dtype, got ", delta->sizes(), " ", delta->scalar_type());
  }
  TORCH_CHECK(delta.has_value() || !gate.has_value(), "a gate needs a delta");
  const Param g = param(gate, x, x.scalar_type(), "gate");
  const Param w = param(gain, x, at::kFloat, "gain");
  const Param s = param(shift, x, at::kFloat, "shift");
  c10::cuda::CUDAGuard guard(x.device());
  const Rows xr = rows_of(x);
  const Rows dr = delta.has_value() ? rows_of(*delta) : Rows{Tensor(), 0, 0};
  int64_t ldc;
  Tensor codes = empty_codes(x, xr.m, &ldc);
  Tensor scale = empty_on(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  Tensor total = empty_on(x, delta.has_value() ? x.sizes() : at::IntArrayRef({0}), x.scalar_type());
  if (xr.m == 0) return {codes, scale, total};
  const int64_t per_batch = x.dim() >= 2 ? xr.m / x.size(0) : 1;
  check_status(w4a4_rms_norm_quant8(
      xr.data(), xr.ld, delta.has_value() ? dr.data() : nullptr, dr.ld, g.ptr, g.stride,
      static_cast<const float*>(w.ptr), w.stride, static_cast<const float*>(s.ptr), s.stride, static_cast<float>(eps),
      dt, xr.m, as_i32(per_batch, "rows per observation"), as_i32(x.size(-1), "the row length"),
      delta.has_value() ? total.data_ptr() : nullptr, codes.data_ptr<int8_t>(), ldc, scale.data_ptr<float>(),
      stream_of(x)));
  return {codes, scale, total};
}

std::tuple<Tensor, Tensor> quantize(const Tensor& x, const OptTensor& up) {
  check_rows(x, "x");
  check_no_gradient(x, "x");
  if (up.has_value()) check_no_gradient(*up, "up");
  const int32_t dt = dtype_code(x.scalar_type(), true, "x");
  if (up.has_value()) {
    check_device(*up, x, "up");
    TORCH_CHECK(up->sizes() == x.sizes() && up->scalar_type() == x.scalar_type(),
                "up must have x's shape and dtype, got ", up->sizes(), " ", up->scalar_type());
  }
  c10::cuda::CUDAGuard guard(x.device());
  const Rows xr = rows_of(x);
  const Rows ur = up.has_value() ? rows_of(*up) : Rows{Tensor(), 0, 0};
  int64_t ldc;
  Tensor codes = empty_codes(x, xr.m, &ldc);
  Tensor scale = empty_on(x, x.sizes().slice(0, x.dim() - 1), at::kFloat);
  if (xr.m == 0) return {codes, scale};
  check_status(w4a4_quant8(xr.data(), xr.ld, up.has_value() ? ur.data() : nullptr, ur.ld, dt, xr.m,
                           as_i32(x.size(-1), "the row length"), codes.data_ptr<int8_t>(), ldc,
                           scale.data_ptr<float>(), stream_of(x)));
  return {codes, scale};
}

// Codes [..., k] and their row scales.
Rows check_codes(const Tensor& codes, const Tensor& scale, const char* what, const char* scale_what) {
  check_rows(codes, what);
  TORCH_CHECK(codes.scalar_type() == at::kChar, what, " must be int8, got ", codes.scalar_type());
  check_device(scale, codes, scale_what);
  const int64_t m = codes.numel() / codes.size(-1);
  TORCH_CHECK(scale.scalar_type() == at::kFloat && scale.numel() == m && scale.is_contiguous(), scale_what,
              " must be contiguous float32 with one value per row (", m, "), got ", scale.sizes(), " ",
              scale.scalar_type());
  check_no_gradient(scale, scale_what);
  return rows_of(codes);
}

Tensor dequantize(const Tensor& codes, const Tensor& scale, at::ScalarType dtype) {
  const int32_t dt = dtype_code(dtype, true, "dtype");
  const Rows r = check_codes(codes, scale, "codes", "scale");
  c10::cuda::CUDAGuard guard(codes.device());
  Tensor out = empty_on(codes, codes.sizes(), dtype);
  check_status(w4a4_dequant8(static_cast<const int8_t*>(r.data()), r.ld, scale.const_data_ptr<float>(), dt, r.m,
                             as_i32(codes.size(-1), "the row length"), out.data_ptr(), stream_of(codes)));
  return out;
}

// Rows that the product can read with TMA: 16-byte steps and base.
Rows tma_rows(Rows r, const char* what) {
  const int64_t k = r.t.size(-1);
  if (r.ld % 16 == 0 && reinterpret_cast<uintptr_t>(r.data()) % 16 == 0) return r;
  if (r.m == 1 && reinterpret_cast<uintptr_t>(r.data()) % 16 == 0) {
    r.ld = (k + 15) / 16 * 16;  // one row: the stride is never used
    return r;
  }
  TORCH_WARN_ONCE("pi05_w8a8.linear: rows of ", what,
                  " do not begin at multiples of 16 bytes; copying them on every call. quantize, rms_norm_quant and "
                  "pack_weight lay them out.");
  const int64_t ld = (k + 127) / 128 * 128;
  Tensor t = empty_on(r.t, {r.m, ld}, at::kChar).narrow(1, 0, k);
  t.copy_(r.t.reshape({r.m, k}));
  return {t, r.m, ld};
}

// A vector from a multiple of 16 bytes (copied if it is a view that is not).
Tensor aligned16(const Tensor& t) {
  return reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 ? t : t.clone();
}

Tensor linear(const Tensor& codes, const Tensor& scale, const Tensor& weight, const Tensor& weight_scale,
              const OptTensor& bias, at::ScalarType dtype) {
  const int32_t dt = dtype_code(dtype, true, "dtype");
  Rows a = check_codes(codes, scale, "codes", "scale");
  TORCH_CHECK(weight.dim() == 2 && weight.size(-1) == codes.size(-1), "weight must be [N, ", codes.size(-1), "], got ",
              weight.sizes());
  check_device(weight, codes, "weight");
  const int64_t n = weight.size(0), k = weight.size(1);
  TORCH_CHECK(n > 0, "weight must have at least one row");
  c10::cuda::CUDAGuard guard(codes.device());
  Rows w = check_codes(weight, weight_scale, "weight", "weight_scale");
  if (bias.has_value()) {
    check_device(*bias, codes, "bias");
    TORCH_CHECK(bias->scalar_type() == dtype && bias->dim() == 1 && bias->size(0) == n && bias->is_contiguous(),
                "bias must be contiguous ", dtype, " [", n, "], got ", bias->sizes(), " ", bias->scalar_type());
    check_no_gradient(*bias, "bias");
  }
  std::vector<int64_t> shape(codes.sizes().begin(), codes.sizes().end());
  shape.back() = n;
  Tensor y = empty_on(codes, shape, dtype);
  if (a.m == 0) return y;
  a = tma_rows(a, "codes");
  w = tma_rows(w, "weight");
  const Tensor sw = aligned16(weight_scale), b = bias.has_value() ? aligned16(*bias) : Tensor();
  check_status(w4a4_gemm8(static_cast<const int8_t*>(a.data()), a.ld, scale.const_data_ptr<float>(),
                          static_cast<const int8_t*>(w.data()), w.ld, sw.const_data_ptr<float>(),
                          bias.has_value() ? b.const_data_ptr() : nullptr, dt, a.m, as_i32(n, "N"), as_i32(k, "K"),
                          y.data_ptr(), stream_of(codes)));
  return y;
}

// The cache's tensors; its strides of batch, token and head.
struct Cache {
  int64_t stride[3];
  int64_t batch, capacity, heads, width;
};
Cache check_cache(const Tensor& k, const Tensor& v, const Tensor& ks, const Tensor& vs) {
  check_cuda(k, "the cache");
  TORCH_CHECK(k.dim() == 4 && k.scalar_type() == at::kChar, "cache keys must be int8 [batch, capacity, heads, width], got ",
              k.sizes(), " ", k.scalar_type());
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == at::kChar && v.strides() == k.strides(),
              "cache values must be laid out like the keys");
  check_device(v, k, "cache values");
  Cache c{{k.stride(0), k.stride(1), k.stride(2)}, k.size(0), k.size(1), k.size(2), k.size(3)};
  TORCH_CHECK(c.heads > 0 && c.width > 0 && k.stride(3) == 1, "cache rows must be contiguous");
  for (int i = 0; i < 3; ++i)
    if (k.size(i) <= 1) c.stride[i] = c.width;  // never used
  TORCH_CHECK(c.capacity % kBlock == 0, "the cache's capacity must be a multiple of ", kBlock, ", got ", c.capacity);
  for (const Tensor* s : {&ks, &vs}) {
    check_device(*s, k, "cache scales");
    TORCH_CHECK(s->scalar_type() == at::kFloat && s->is_contiguous() && s->dim() == 3 && s->size(0) == c.batch &&
                    s->size(1) == c.heads && s->size(2) == c.capacity / kBlock,
                "cache scales must be contiguous float32 [batch, heads, capacity / ", kBlock, "], got ", s->sizes(), " ",
                s->scalar_type());
    check_no_gradient(*s, "a cache scale");
  }
  return c;
}

const int32_t* check_lengths(const Tensor& t, const Tensor& k, const char* what) {
  check_device(t, k, what);
  TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == k.size(0) && t.is_contiguous(), what,
              " must be contiguous int32 [", k.size(0), "], got ", t.sizes(), " ", t.scalar_type());
  return t.const_data_ptr<int32_t>();
}

// A [batch, tokens, heads, width] tensor with contiguous rows (copied if not).
Tensor with_rows(const Tensor& t, int64_t align) {
  bool good = t.stride(3) == 1 || t.size(3) == 1;
  if (good && align > 1)
    for (int i = 0; i < 3; ++i) good = good && t.stride(i) % align == 0;
  if (good && align > 1) good = reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0;
  if (good) return t;
  return t.clone(at::MemoryFormat::Contiguous);
}

Tensor kv_append(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale, const Tensor& v_scale,
                 const Tensor& k, const Tensor& v, const Tensor& start, const OptTensor& valid) {
  const Cache c = check_cache(k_cache, v_cache, k_scale, v_scale);
  const int32_t dt = dtype_code(k.scalar_type(), false, "new keys");
  TORCH_CHECK(k.dim() == 4 && k.size(0) == c.batch && k.size(2) == c.heads && k.size(3) == c.width,
              "new keys must be [", c.batch, ", tokens, ", c.heads, ", ", c.width, "], got ", k.sizes());
  TORCH_CHECK(v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(), "new values must have the keys' shape and dtype");
  check_device(k, k_cache, "new keys");
  check_device(v, k_cache, "new values");
  check_no_gradient(k, "the new keys");
  check_no_gradient(v, "the new values");
  const int32_t* start_ptr = check_lengths(start, k_cache, "start");
  const int64_t tokens = k.size(1);
  Tensor mask;
  if (valid.has_value()) {
    check_device(*valid, k_cache, "valid");
    TORCH_CHECK((valid->scalar_type() == at::kBool || valid->scalar_type() == at::kByte) && valid->dim() == 2 &&
                    valid->size(0) == c.batch && valid->size(1) == tokens,
                "valid must be bool or uint8 [", c.batch, ", ", tokens, "], got ", valid->sizes(), " ",
                valid->scalar_type());
  }
  c10::cuda::CUDAGuard guard(k_cache.device());
  if (valid.has_value()) mask = valid->stride(1) == 1 || tokens <= 1 ? *valid : valid->contiguous();
  const Tensor kr = with_rows(k, 1), vr = with_rows(v, 1);
  Tensor lengths = empty_on(start, {c.batch}, at::kInt);
  if (c.batch == 0) return lengths;
  const int64_t ks[3] = {kr.stride(0), kr.stride(1), kr.stride(2)}, vs[3] = {vr.stride(0), vr.stride(1), vr.stride(2)};
  check_status(w4a4_kv8_append(
      static_cast<int8_t*>(k_cache.data_ptr()), static_cast<int8_t*>(v_cache.data_ptr()), k_scale.data_ptr<float>(),
      v_scale.data_ptr<float>(), c.stride, as_i32(c.capacity, "the capacity"), kr.const_data_ptr(), ks,
      vr.const_data_ptr(), vs, dt, valid.has_value() ? static_cast<const uint8_t*>(mask.const_data_ptr()) : nullptr,
      valid.has_value() ? mask.stride(0) : 0, start_ptr, lengths.data_ptr<int32_t>(), as_i32(c.batch, "the batch"),
      as_i32(tokens, "the token count"), as_i32(c.heads, "the head count"), as_i32(c.width, "the head width"),
      stream_of(k_cache)));
  return lengths;
}

std::tuple<Tensor, Tensor> kv_values(const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                                     const Tensor& v_scale, const Tensor& lengths, at::ScalarType dtype) {
  const Cache c = check_cache(k_cache, v_cache, k_scale, v_scale);
  const int32_t dt = dtype_code(dtype, true, "dtype");
  const int32_t* len = check_lengths(lengths, k_cache, "lengths");
  c10::cuda::CUDAGuard guard(k_cache.device());
  Tensor k = empty_on(k_cache, k_cache.sizes(), dtype);
  Tensor v = empty_on(k_cache, k_cache.sizes(), dtype);
  if (c.batch == 0) return {k, v};
  check_status(w4a4_kv8_values(k_cache.const_data_ptr<int8_t>(), v_cache.const_data_ptr<int8_t>(),
                               k_scale.const_data_ptr<float>(), v_scale.const_data_ptr<float>(), c.stride,
                               as_i32(c.capacity, "the capacity"), len, dt, as_i32(c.batch, "the batch"),
                               as_i32(c.heads, "the head count"), as_i32(c.width, "the head width"), k.data_ptr(),
                               v.data_ptr(), stream_of(k_cache)));
  return {k, v};
}

Tensor kv_attention(const Tensor& q, const Tensor& k_cache, const Tensor& v_cache, const Tensor& k_scale,
                    const Tensor& v_scale, const Tensor& lengths, bool causal, double scale) {
  const Cache c = check_cache(k_cache, v_cache, k_scale, v_scale);
  check_device(q, k_cache, "q");
  check_no_gradient(q, "q");
  const int32_t dt = dtype_code(q.scalar_type(), false, "q");
  TORCH_CHECK(q.dim() == 4 && q.size(0) == c.batch && q.size(3) == c.width && q.size(2) > 0 && q.size(2) % c.heads == 0,
              "q must be [", c.batch, ", tokens, a multiple of ", c.heads, " heads, ", c.width, "], got ", q.sizes());
  const int32_t* len = check_lengths(lengths, k_cache, "lengths");
  c10::cuda::CUDAGuard guard(k_cache.device());
  const Tensor qr = with_rows(q, 8);
  Tensor out = empty_on(q, q.sizes(), q.scalar_type());
  if (q.numel() == 0) return out;
  const int64_t qs[3] = {qr.stride(0), qr.stride(1), qr.stride(2)};
  int64_t bytes = 0;
  check_status(w4a4_attention8_workspace(as_i32(c.batch, "the batch"), as_i32(q.size(1), "the token count"),
                                         as_i32(q.size(2), "the query head count"), as_i32(c.heads, "the head count"),
                                         as_i32(c.width, "the head width"), as_i32(c.capacity, "the capacity"), &bytes));
  Tensor workspace;
  if (bytes > 0) workspace = empty_on(q, {bytes}, at::kByte);
  check_status(w4a4_attention8(qr.const_data_ptr(), qs, k_cache.const_data_ptr<int8_t>(),
                               v_cache.const_data_ptr<int8_t>(), k_scale.const_data_ptr<float>(),
                               v_scale.const_data_ptr<float>(), c.stride, as_i32(c.capacity, "the capacity"), len, dt,
                               as_i32(c.batch, "the batch"), as_i32(q.size(1), "the token count"),
                               as_i32(q.size(2), "the query head count"), as_i32(c.heads, "the head count"),
                               as_i32(c.width, "the head width"), causal ? 1 : 0, static_cast<float>(scale),
                               out.data_ptr(), bytes > 0 ? workspace.data_ptr() : nullptr, bytes, stream_of(q)));
  return out;
}

}  // namespace

TORCH_LIBRARY_IMPL(pi05_w8a8, CompositeExplicitAutograd, m) {
  m.impl("rms_norm_quant", &rms_norm_quant);
  m.impl("quantize", &quantize);
  m.impl("dequantize", &dequantize);
  m.impl("linear", &linear);
  m.impl("kv_append", &kv_append);
  m.impl("kv_values", &kv_values);
  m.impl("kv_attention", &kv_attention);
}

// No op has a gradient (check_no_gradient): calls go past the autograd keys to the bodies.
namespace {
void past_autograd(torch::Library& m) {
  for (const char* op : {"rms_norm_quant", "quantize", "dequantize", "linear", "kv_append", "kv_values", "kv_attention"})
    m.impl(op, torch::CppFunction::makeFallthrough());
}
}  // namespace
TORCH_LIBRARY_IMPL(pi05_w8a8, AutogradCUDA, m) { past_autograd(m); }
TORCH_LIBRARY_IMPL(pi05_w8a8, AutogradCPU, m) { past_autograd(m); }
