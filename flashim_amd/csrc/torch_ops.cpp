// The C entry points as torch operators of the namespace flashim_amd: each allocates its outputs with torch's caching
// allocator, makes one C call on the current stream of its input's device and raises on a nonzero status. Registered in
// C++, an eager call takes torch's C++ dispatcher only (a Python custom op costs about 10 us a call on the host, more
// than a small layer's kernel); the fakes stay in library.py. Arguments arrive normalized by the Python impls (dtypes,
// contiguity, devices); 1-byte float formats cross as they are or as their uint8 views (the bodies read bytes), and come
// back as uint8.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/forward_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/library.h>

#include <array>
#include <limits>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/flashim_amd.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

constexpr int64_t BLOCK = 32;

hipStream_t stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.device().index()).stream(); }

template <typename T>
T* ptr(const Tensor& t) { return static_cast<T*>(t.data_ptr()); }
template <typename T>
T* ptr(const OptTensor& t) { return t ? static_cast<T*>(t->data_ptr()) : nullptr; }

int dtype_code(const Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return 0;
    case at::kBFloat16: return 1;
    case at::kHalf: return 2;
    default: TORCH_CHECK_TYPE(false, "unsupported dtype ", t.scalar_type());
  }
}

int bias_code(const Tensor& t) { return t.scalar_type() == at::kBFloat16 ? 1 : 0; }
int bias_code(const OptTensor& t) { return t && t->scalar_type() == at::kBFloat16 ? 1 : 0; }

// Status 99 as the package's own exception, raised here so that compiled graphs, which call the operators themselves, see
// its type too.
[[noreturn]] void raise_unsupported(const std::string& message) {
  pybind11::gil_scoped_acquire gil;
  PyErr_SetString(pybind11::module_::import("flashim_amd._lib").attr("UnsupportedShape").ptr(), message.c_str());
  throw pybind11::error_already_set();
}

template <typename... What>
void check(int code, const What&... what) {
  if (code == FIM_OK) return;
  if (code == FIM_ERR_UNSUPPORTED) raise_unsupported(c10::str(what..., ": no HIP kernel for this shape/layout (code 99)"));
  TORCH_CHECK(false, what..., " launch failed (code ", code, ")");
}

// size() and stride() of the leading dimensions would read an input of more dimensions as one of fewer
void check_dims(const Tensor& t, int64_t dims, const char* what) {
  TORCH_CHECK_VALUE(t.dim() == dims, what, ": expected ", dims, " dimensions, got shape ", t.sizes());
}

Tensor empty(at::IntArrayRef sizes, const Tensor& like, at::ScalarType dtype) {
  return at::empty(sizes, like.options().dtype(dtype).requires_grad(false).memory_format(std::nullopt));
}

// [..., C] as [B, H, W, C] sizes and strides, copying only where leading dimensions do not merge.
struct View4 {
  Tensor t;
  std::array<int64_t, 4> n{1, 1, 1, 1}, s{0, 0, 0, 0};
  explicit View4(const Tensor& x) : t(x) {
    if (t.dim() > 4) t = t.reshape({-1, t.size(-3), t.size(-2), t.size(-1)});
    const int64_t d = t.dim(), pad = 4 - d;
    for (int64_t i = 0; i < d; ++i) {
      n[pad + i] = t.size(i);
      s[pad + i] = t.stride(i);
    }
    for (int64_t i = pad - 1; i >= 0; --i) s[i] = i == 3 ? 1 : n[i + 1] * s[i + 1];  // as unsqueeze does
  }
};

#define FIM_VIEW4(v) v.n[0], v.n[1], v.n[2], v.n[3], v.s[0], v.s[1], v.s[2], v.s[3]

std::vector<int64_t> padded_sizes(const Tensor& value, int64_t padded) {
  auto sizes = value.sizes().vec();
  if (!sizes.empty()) sizes.pop_back();
  sizes.push_back(padded);
  return sizes;
}

Tensor quantize_mxfp8(const Tensor& value, const Tensor& exponent, int64_t padded) {
  const c10::DeviceGuard guard(value.device());
  Tensor out = empty(padded_sizes(value, padded), value, at::kByte);
  const View4 v(value);
  check(fim_quantize_mxfp8(v.t.data_ptr(), dtype_code(value), FIM_VIEW4(v), ptr<const int8_t>(exponent),
                           ptr<uint8_t>(out), padded, stream_of(value)),
        "quantize_mxfp8 ", value.sizes());
  return out;
}

Tensor gelu_quantize_mxfp8(const Tensor& value, const Tensor& exponent, int64_t padded, const OptTensor& input_bias,
                           bool tanh) {
  const c10::DeviceGuard guard(value.device());
  Tensor out = empty(padded_sizes(value, padded), value, at::kByte);
  const View4 v(value);
  check(fim_gelu_quantize_mxfp8(v.t.data_ptr(), dtype_code(value), FIM_VIEW4(v), tanh, ptr<const float>(input_bias),
                                ptr<const int8_t>(exponent), ptr<uint8_t>(out), padded, stream_of(value)),
        "gelu_quantize_mxfp8 ", value.sizes());
  return out;
}

Tensor quantize_int8(const Tensor& value, const Tensor& scale, const OptTensor& channel_scale) {
  const c10::DeviceGuard guard(value.device());
  Tensor out = empty(value.sizes(), value, at::kChar);
  const View4 v(value);
  check(fim_quantize_int8(v.t.data_ptr(), dtype_code(value), FIM_VIEW4(v), ptr<const float>(scale),
                          ptr<const float>(channel_scale), ptr<int8_t>(out), stream_of(value)),
        "quantize_int8 ", value.sizes());
  return out;
}

Tensor gelu_quantize_int8(const Tensor& value, const Tensor& scale, bool tanh) {
  const c10::DeviceGuard guard(value.device());
  Tensor out = empty(value.sizes(), value, at::kChar);
  const View4 v(value);
  check(fim_gelu_quantize_int8(v.t.data_ptr(), dtype_code(value), FIM_VIEW4(v), tanh, ptr<const float>(scale),
                               ptr<int8_t>(out), stream_of(value)),
        "gelu_quantize_int8 ", value.sizes());
  return out;
}

// Swizzled scales: whole 128-row x 4-block tiles; the bytes past the matrix are zero.
Tensor swizzled_scales(int64_t rows, int64_t groups, const Tensor& like) {
  Tensor t = empty({(rows + 127) / 128 * 128 * ((groups + 3) / 4 * 4)}, like, at::kByte);
  if (rows % 128 || groups % 4) t.zero_();
  return t;
}

std::tuple<Tensor, Tensor> quantize_mxfp8_dynamic(const Tensor& value_in, bool swizzled) {
  check_dims(value_in, 2, "quantize_mxfp8_dynamic");
  const c10::DeviceGuard guard(value_in.device());
  Tensor value = value_in;
  if (reinterpret_cast<uintptr_t>(value.data_ptr()) % 16)  // the kernel reads 16-byte rows
    value = value.clone(at::MemoryFormat::Contiguous);
  const int64_t rows = value.size(0), cols = value.size(1), groups = cols / BLOCK;
  Tensor out = empty({rows, cols}, value, at::kByte);
  Tensor scales = swizzled ? swizzled_scales(rows, groups, value) : empty({rows, groups}, value, at::kChar);
  check(fim_quantize_mxfp8_dynamic(value.data_ptr(), dtype_code(value), rows, cols, value.stride(0), ptr<uint8_t>(out),
                                   swizzled ? nullptr : ptr<int8_t>(scales), swizzled ? ptr<uint8_t>(scales) : nullptr,
                                   stream_of(value)),
        "quantize_mxfp8_dynamic ", rows, "x", cols);
  return {out, scales};
}

std::tuple<Tensor, Tensor> quantize_int8_rows(const Tensor& value, bool reciprocal) {
  check_dims(value, 2, "quantize_int8_rows");
  const c10::DeviceGuard guard(value.device());
  const int64_t rows = value.size(0), k = value.size(1);
  Tensor q = empty({rows, k}, value, at::kChar), scale = empty({rows}, value, at::kFloat);
  check(fim_quantize_int8_rows(value.data_ptr(), dtype_code(value), rows, k, value.stride(0), reciprocal, ptr<int8_t>(q),
                               ptr<float>(scale), stream_of(value)),
        "quantize_int8_rows ", rows, "x", k);
  return {q, scale};
}

Tensor calibrate_block32(const Tensor& matrix) {
  check_dims(matrix, 2, "calibrate_block32");
  const c10::DeviceGuard guard(matrix.device());
  const int64_t rows = matrix.size(0), channels = matrix.size(1), groups = (channels + BLOCK - 1) / BLOCK;
  Tensor workspace = empty({groups}, matrix, at::kInt), exponent = empty({groups}, matrix, at::kChar);
  check(fim_calibrate_block32(matrix.data_ptr(), dtype_code(matrix), rows, channels, matrix.stride(0),
                              ptr<uint32_t>(workspace), ptr<int8_t>(exponent), stream_of(matrix)),
        "calibrate_block32");
  return exponent;
}

struct Residual {
  const void* data = nullptr;
  int code = 0;
  int64_t channels = 0;
  std::array<int64_t, 4> strides{};
  const int64_t* stride_ptr = nullptr;
  explicit Residual(const OptTensor& r) {
    if (!r) return;
    data = r->data_ptr();
    code = dtype_code(*r);
    channels = r->size(-1);
    for (int64_t i = 0; i < r->dim() && i < 4; ++i) strides[i] = r->stride(i);
    stride_ptr = strides.data();
  }
};

// kh .. dw of a convolution call as the C ABI takes them, and its output size
struct Geometry {
  int kh, kw, sh, sw, ph, pw, dh, dw;
  int64_t out(int64_t n, int k, int s, int p, int d) const {  // Python's floor division
    const int64_t a = n + 2 * p - static_cast<int64_t>(d) * (k - 1) - 1;
    return (a >= 0 ? a / s : -((-a + s - 1) / s)) + 1;
  }
  int64_t ho(int64_t h) const { return out(h, kh, sh, ph, dh); }
  int64_t wo(int64_t w) const { return out(w, kw, sw, pw, dw); }
};

#define FIM_GEO_PARAMS int64_t kh, int64_t kw, int64_t sh, int64_t sw, int64_t ph, int64_t pw, int64_t dh, int64_t dw
#define FIM_GEO Geometry { (int)kh, (int)kw, (int)sh, (int)sw, (int)ph, (int)pw, (int)dh, (int)dw }
#define FIM_GEO_ARGS(g) g.kh, g.kw, g.sh, g.sw, g.ph, g.pw, g.dh, g.dw

Tensor int8_conv2d(const Tensor& x, const Tensor& weight, const Tensor& a_scale, const Tensor& w_scale,
                   const OptTensor& bias, FIM_GEO_PARAMS, bool relu, bool gelu, const OptTensor& residual,
                   const OptTensor& out_scale) {
  check_dims(x, 4, "int8_conv2d");
  TORCH_CHECK_INDEX(!residual || residual->dim() <= 4, "int8_conv2d: residual of shape ", residual->sizes());
  const c10::DeviceGuard guard(x.device());
  const Geometry g = FIM_GEO;
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), cin = x.size(3), cout = weight.size(0);
  TORCH_CHECK(sh > 0 && sw > 0, "int8_conv2d: strides must be positive");
  Tensor out = empty({b, g.ho(h), g.wo(w), cout}, x, out_scale ? at::kChar : at::kBFloat16);
  const Residual r(residual);
  check(fim_int8_conv2d(ptr<const int8_t>(x), b, h, w, cin, ptr<const int8_t>(weight), cout, ptr<const float>(a_scale),
                        ptr<const float>(w_scale), ptr<const void>(bias), bias_code(bias), FIM_GEO_ARGS(g), relu, gelu,
                        r.data, r.code, r.channels, r.stride_ptr, ptr<const float>(out_scale), out.data_ptr(),
                        stream_of(x)),
        "int8_conv2d ", x.sizes(), " -> ", cout, " k", kh, "x", kw);
  return out;
}

std::tuple<Tensor, Tensor> int8_conv2d_maxpool(const Tensor& x, const Tensor& weight, const Tensor& a_scale,
                                               const Tensor& w_scale, const OptTensor& bias, FIM_GEO_PARAMS, bool relu,
                                               const Tensor& out_scale) {
  check_dims(x, 4, "int8_conv2d_maxpool");
  const c10::DeviceGuard guard(x.device());
  const Geometry g = FIM_GEO;
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), cin = x.size(3), cout = weight.size(0);
  TORCH_CHECK(sh > 0 && sw > 0, "int8_conv2d_maxpool: strides must be positive");
  const int64_t ho = g.ho(h), wo = g.wo(w);
  Tensor out = empty({b, ho, wo, cout}, x, at::kBFloat16), pooled = empty({b, ho / 2, wo / 2, cout}, x, at::kChar);
  check(fim_int8_conv2d_maxpool(ptr<const int8_t>(x), b, h, w, cin, ptr<const int8_t>(weight), cout,
                                ptr<const float>(a_scale), ptr<const float>(w_scale), ptr<const void>(bias),
                                bias_code(bias), FIM_GEO_ARGS(g), relu, ptr<const float>(out_scale), out.data_ptr(),
                                ptr<int8_t>(pooled), stream_of(x)),
        "int8_conv2d_maxpool ", x.sizes(), " -> ", cout, " k", kh, "x", kw);
  return {out, pooled};
}

Tensor mxfp8_conv2d(const Tensor& x, const Tensor& channel_exponent, const Tensor& weight, const Tensor& weight_exponent,
                    const OptTensor& bias, FIM_GEO_PARAMS, bool relu, bool gelu, const OptTensor& residual,
                    const OptTensor& out_exponent) {
  check_dims(x, 4, "mxfp8_conv2d");
  TORCH_CHECK_INDEX(!residual || residual->dim() <= 4, "mxfp8_conv2d: residual of shape ", residual->sizes());
  const c10::DeviceGuard guard(x.device());
  const Geometry g = FIM_GEO;
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), cin = x.size(3), cout = weight.size(0);
  TORCH_CHECK(sh > 0 && sw > 0, "mxfp8_conv2d: strides must be positive");
  Tensor out = empty({b, g.ho(h), g.wo(w), cout}, x, out_exponent ? at::kByte : at::kBFloat16);
  const Residual r(residual);
  check(fim_mxfp8_conv2d(ptr<const uint8_t>(x), b, h, w, cin, ptr<const int8_t>(channel_exponent),
                         ptr<const uint8_t>(weight), cout, ptr<const int8_t>(weight_exponent), ptr<const void>(bias),
                         bias_code(bias), FIM_GEO_ARGS(g), relu, gelu, r.data, r.code, r.channels, r.stride_ptr,
                         ptr<const int8_t>(out_exponent), out.data_ptr(), stream_of(x)),
        "mxfp8_conv2d ", x.sizes(), " -> ", cout, " k", kh, "x", kw);
  return out;
}

Tensor int8_linear(const Tensor& a, const Tensor& weight, const Tensor& a_scale, const Tensor& w_scale,
                   const OptTensor& bias, bool relu, bool gelu, const OptTensor& residual) {
  check_dims(a, 2, "int8_linear");
  const c10::DeviceGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = weight.size(0);
  const bool per_row = a_scale.numel() != 1;
  Tensor out = empty({m, n}, a, at::kBFloat16);
  const Residual r(residual);
  check(fim_int8_linear(ptr<const int8_t>(a), m, k, ptr<const int8_t>(weight), n,
                        per_row ? nullptr : ptr<const float>(a_scale), per_row ? ptr<const float>(a_scale) : nullptr,
                        ptr<const float>(w_scale), ptr<const void>(bias), bias_code(bias), relu, gelu, r.data, r.code,
                        r.channels, r.strides[0], nullptr, out.data_ptr(), stream_of(a)),
        "int8_linear ", m, "x", k, " -> ", n);
  return out;
}

void int8_linear_quantize_(const Tensor& a, const Tensor& weight, const Tensor& a_scale, const Tensor& w_scale,
                           const OptTensor& bias, const Tensor& out_scale, const Tensor& out) {
  check_dims(a, 2, "int8_linear_quantize_");
  const c10::DeviceGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = weight.size(0);
  const bool per_row = a_scale.numel() != 1;
  check(fim_int8_linear_quantize(ptr<const int8_t>(a), m, k, ptr<const int8_t>(weight), n,
                                 per_row ? nullptr : ptr<const float>(a_scale),
                                 per_row ? ptr<const float>(a_scale) : nullptr, ptr<const float>(w_scale),
                                 ptr<const void>(bias), bias_code(bias), ptr<const float>(out_scale), ptr<int8_t>(out),
                                 out.stride(0), stream_of(a)),
        "int8_linear_quantize ", m, "x", k, " -> ", n);
}

Tensor mxfp8_scaled_mm(const Tensor& a, const Tensor& a_scale_swizzled, const Tensor& weight,
                       const Tensor& weight_exponent, const OptTensor& bias, bool weight_scale_e8m0) {
  check_dims(a, 2, "mxfp8_scaled_mm");
  const c10::DeviceGuard guard(a.device());
  const int64_t m = a.size(0), k = a.size(1), n = weight.size(0);
  Tensor out = empty({m, n}, a, at::kBFloat16);
  check(fim_mxfp8_scaled_mm(ptr<const uint8_t>(a), m, k, ptr<const uint8_t>(a_scale_swizzled),
                            ptr<const uint8_t>(weight), n, ptr<const int8_t>(weight_exponent), weight_scale_e8m0,
                            ptr<const void>(bias), bias_code(bias), out.data_ptr(), stream_of(a)),
        "mxfp8_scaled_mm ", m, "x", k, " -> ", n);
  return out;
}

Tensor im2col_gather(const Tensor& x, FIM_GEO_PARAMS) {
  check_dims(x, 4, "im2col_gather");
  const c10::DeviceGuard guard(x.device());
  const Geometry g = FIM_GEO;
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), c = x.size(3);
  TORCH_CHECK(sh > 0 && sw > 0, "im2col_gather: strides must be positive");
  Tensor out = empty({b * g.ho(h) * g.wo(w), kh * kw * c}, x, at::kByte);
  check(fim_im2col_gather(ptr<const uint8_t>(x), b, h, w, c, FIM_GEO_ARGS(g), ptr<uint8_t>(out), stream_of(x)),
        "im2col_gather");
  return out;
}

Tensor refiner_mlp(int64_t kind, int64_t semantics, const Tensor& x, const Tensor& x_scale, const Tensor& w1,
                   const Tensor& w1_scale, const OptTensor& b1, const Tensor& h_scale, const Tensor& w2,
                   const Tensor& w2_scale, const OptTensor& b2, const OptTensor& residual) {
  check_dims(x, 2, "refiner_mlp");
  const c10::DeviceGuard guard(x.device());
  const int64_t rows = x.size(0), c = x.size(1), h = w1.size(0);
  Tensor out = empty({rows, w2.size(0)}, x, at::kBFloat16);
  check(fim_refiner_mlp((int)kind, (int)semantics, ptr<const uint8_t>(x), rows, c, h, x_scale.data_ptr(),
                        ptr<const uint8_t>(w1), w1_scale.data_ptr(), ptr<const void>(b1), bias_code(b1),
                        h_scale.data_ptr(), ptr<const uint8_t>(w2), w2_scale.data_ptr(), ptr<const void>(b2),
                        bias_code(b2), ptr<const uint16_t>(residual), ptr<uint16_t>(out), stream_of(x)),
        "refiner_mlp ", rows, "x", c);
  return out;
}

constexpr int DW_MX_DYNAMIC = 0, DW_INT8 = 1, DW_BF16 = 2, DW_MX_STATIC = 3;

Tensor depthwise5x5(const Tensor& x, const Tensor& weight, const Tensor& bias, int64_t act, int64_t mode,
                    const OptTensor& scale, const OptTensor& exponent) {
  check_dims(x, 4, "depthwise5x5");
  const c10::DeviceGuard guard(x.device());
  TORCH_CHECK(mode == DW_INT8 || mode == DW_BF16 || mode == DW_MX_STATIC, "depthwise5x5: no output mode ", mode);
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), c = x.size(3);
  Tensor out = empty({b * h * w, c}, x, mode == DW_INT8 ? at::kChar : mode == DW_BF16 ? at::kBFloat16 : at::kByte);
  check(fim_depthwise5x5(ptr<const uint16_t>(x), b, h, w, c, ptr<const uint16_t>(weight), bias.data_ptr(),
                         bias_code(bias), (int)act, (int)mode, ptr<const float>(scale), ptr<const int8_t>(exponent),
                         out.data_ptr(), nullptr, nullptr, stream_of(x)),
        "depthwise5x5 ", x.sizes());
  return out;
}

std::tuple<Tensor, Tensor> depthwise5x5_mx_dynamic(const Tensor& x, const Tensor& weight, const Tensor& bias) {
  check_dims(x, 4, "depthwise5x5_mx_dynamic");
  const c10::DeviceGuard guard(x.device());
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), c = x.size(3), rows = b * h * w;
  Tensor out = empty({rows, c}, x, at::kByte), swz = swizzled_scales(rows, c / BLOCK, x);
  check(fim_depthwise5x5(ptr<const uint16_t>(x), b, h, w, c, ptr<const uint16_t>(weight), bias.data_ptr(),
                         bias_code(bias), 0, DW_MX_DYNAMIC, nullptr, nullptr, out.data_ptr(), nullptr,
                         ptr<uint8_t>(swz), stream_of(x)),
        "depthwise5x5 ", x.sizes());
  return {out, swz};
}

Tensor depthwise5x5_relu_pointwise_mxfp8(const Tensor& x, const Tensor& dw_weight, const Tensor& dw_bias,
                                         const Tensor& pw_weight, const Tensor& pw_e8m0, const OptTensor& pw_bias) {
  check_dims(x, 4, "depthwise5x5_relu_pointwise_mxfp8");
  const c10::DeviceGuard guard(x.device());
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), c = x.size(3), n = pw_weight.size(0);
  Tensor out = empty({b, h, w, n}, x, at::kBFloat16);
  check(fim_depthwise5x5_relu_pointwise_mxfp8(ptr<const uint16_t>(x), b, h, w, c, ptr<const uint16_t>(dw_weight),
                                              dw_bias.data_ptr(), bias_code(dw_bias), ptr<const uint8_t>(pw_weight), n,
                                              ptr<const uint8_t>(pw_e8m0), ptr<const void>(pw_bias), bias_code(pw_bias),
                                              ptr<uint16_t>(out), stream_of(x)),
        "depthwise5x5_relu_pointwise_mxfp8 ", x.sizes());
  return out;
}

Tensor depthwise5x5_relu_pointwise_int8(const Tensor& x, const Tensor& dw_weight, const Tensor& dw_bias,
                                        const Tensor& scale, const Tensor& pw_weight, const Tensor& pw_wscale,
                                        const OptTensor& pw_bias) {
  check_dims(x, 4, "depthwise5x5_relu_pointwise_int8");
  const c10::DeviceGuard guard(x.device());
  const int64_t b = x.size(0), h = x.size(1), w = x.size(2), c = x.size(3), n = pw_weight.size(0);
  Tensor out = empty({b, h, w, n}, x, at::kBFloat16);
  check(fim_depthwise5x5_relu_pointwise_int8(ptr<const uint16_t>(x), b, h, w, c, ptr<const uint16_t>(dw_weight),
                                             dw_bias.data_ptr(), bias_code(dw_bias), ptr<const float>(scale),
                                             ptr<const int8_t>(pw_weight), n, ptr<const float>(pw_wscale),
                                             ptr<const void>(pw_bias), bias_code(pw_bias), ptr<uint16_t>(out),
                                             stream_of(x)),
        "depthwise5x5_relu_pointwise_int8 ", x.sizes());
  return out;
}

Tensor conv3x3_small_cin_quantize_int8(const Tensor& x, const Tensor& packed, const Tensor& bias, const Tensor& scale) {
  check_dims(x, 4, "conv2d_small_cin_quantize_int8");
  const c10::DeviceGuard guard(x.device());
  const int64_t b = x.size(0), cin = x.size(1), h = x.size(2), w = x.size(3), cout = packed.size(0);
  Tensor out = empty({b, h, w, cout}, x, at::kChar);
  check(fim_conv3x3_small_cin_quantize_int8(ptr<const uint16_t>(x), b, cin, h, w, ptr<const uint16_t>(packed), cout,
                                            bias.data_ptr(), bias_code(bias), ptr<const float>(scale),
                                            ptr<int8_t>(out), stream_of(x)),
        "conv2d_small_cin_quantize_int8 ", x.sizes(), " -> ", cout);
  return out;
}

Tensor bias_relu_quantize_int8(const Tensor& raw, const Tensor& bias, const Tensor& scale) {
  check_dims(raw, 4, "bias_relu_quantize_int8");
  const c10::DeviceGuard guard(raw.device());
  const int64_t b = raw.size(0), c = raw.size(1), h = raw.size(2), w = raw.size(3);
  Tensor out = empty({b, h, w, c}, raw, at::kChar);
  check(fim_bias_relu_quantize_int8(ptr<const uint16_t>(raw), b, c, h, w, bias.data_ptr(), bias_code(bias),
                                    ptr<const float>(scale), ptr<int8_t>(out), stream_of(raw)),
        "bias_relu_quantize_int8 ", raw.sizes());
  return out;
}

Tensor pointwise_bf16(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
  check_dims(x, 2, "pointwise_bf16");
  const c10::DeviceGuard guard(x.device());
  const int64_t m = x.size(0), k = x.size(1), n = weight.size(0);
  Tensor out = empty({m, n}, x, at::kBFloat16);
  check(fim_pointwise_bf16(ptr<const uint16_t>(x), m, k, ptr<const uint16_t>(weight), n, ptr<const void>(bias),
                           bias_code(bias), ptr<uint16_t>(out), stream_of(x)),
        "pointwise_bf16 ", m, "x", k, "x", n);
  return out;
}

// -- training-step operators -------------------------------------------------------------------------------------------

int float_code(const OptTensor& t) { return t ? dtype_code(*t) : 0; }

// x as [B, P, C] with unit channel stride: its own memory where its strides allow that view, else a copy's
struct ImageRows {
  Tensor hold;
  int64_t b, p = 1, c, sb, sp;
  ImageRows(const Tensor& x, const char* what) : hold(x) {
    TORCH_CHECK_VALUE(x.dim() >= 2, what, ": expected [B, ..., C], got shape ", x.sizes());
    b = x.size(0);
    c = x.size(-1);
    bool view = x.stride(-1) == 1 || c == 1;
    sp = c;
    for (int64_t i = x.dim() - 2; i > 0; --i) {
      if (x.size(i) != 1) {
        if (p == 1) sp = x.stride(i);
        else view = view && x.stride(i) == sp * p;
      }
      p *= x.size(i);
    }
    sb = x.stride(0);
    if (view) return;
    hold = x.contiguous();
    sp = c;
    sb = c * p;
  }
};

// x as [rows, C] with unit column stride
Tensor matrix_rows(const Tensor& x, const char* what) {
  TORCH_CHECK_VALUE(x.dim() >= 1, what, ": expected [..., C], got a scalar");
  const int64_t c = x.size(-1);
  if (x.dim() == 2 && (x.stride(1) == 1 || c == 1)) return x;
  int64_t m = 1;
  for (int64_t i = 0; i < x.dim() - 1; ++i) m *= x.size(i);
  Tensor t = x.reshape({m, c});
  return t.stride(1) == 1 || c == 1 ? t : t.contiguous();
}

OptTensor dense(const OptTensor& t) { return t && !t->is_contiguous() ? OptTensor(t->contiguous()) : t; }

void check_same(const Tensor& t, at::ScalarType dtype, const Tensor& like, const char* what) {
  TORCH_CHECK_TYPE(t.scalar_type() == dtype, what, ": expected ", dtype, ", got ", t.scalar_type());
  TORCH_CHECK_VALUE(t.device() == like.device(), what, ": on ", t.device(), ", expected ", like.device());
}

void check_vector(const OptTensor& t, int64_t n, const Tensor& like, const char* what) {
  if (!t) return;
  TORCH_CHECK_VALUE(t->dim() == 1 && t->size(0) == n, what, ": expected ", n, " values, got shape ", t->sizes());
  TORCH_CHECK_VALUE(t->device() == like.device(), what, ": on ", t->device(), ", expected ", like.device());
}

Tensor norm_workspace(const ImageRows& v, int64_t groups, int backward) {
  int64_t floats = 0;
  check(fim_group_norm_workspace(v.b, v.p, v.c, groups, backward, &floats), "group_norm_act ", v.hold.sizes(), " in ",
        groups, " groups");
  return empty({floats}, v.hold, at::kFloat);
}

std::tuple<Tensor, Tensor> group_norm_act(const Tensor& x, int64_t groups, const OptTensor& weight, const OptTensor& bias,
                                          double eps, int64_t act) {
  const c10::DeviceGuard guard(x.device());
  const ImageRows v(x, "group_norm_act");
  const int64_t b = v.b, p = v.p, c = v.c;
  TORCH_CHECK_VALUE(groups > 0 && c > 0 && c % groups == 0, "group_norm_act: ", c, " channels in ", groups, " groups");
  check_vector(weight, c, x, "group_norm_act: weight");
  check_vector(bias, c, x, "group_norm_act: bias");
  const OptTensor w = dense(weight), bi = dense(bias);
  Tensor out = empty(x.sizes(), x, x.scalar_type()), stats = empty({b, groups, 2}, x, at::kFloat);
  const Tensor ws = norm_workspace(v, groups, 0);
  check(fim_group_norm(v.hold.data_ptr(), dtype_code(x), b, p, c, v.sb, v.sp, groups, ptr<const void>(w),
                       float_code(w), ptr<const void>(bi), float_code(bi), (float)eps, (int)act, out.data_ptr(),
                       ptr<float>(stats), ptr<float>(ws), stream_of(x)),
        "group_norm_act ", x.sizes(), " in ", groups, " groups");
  return {out, stats};
}

// d_weight and d_bias are empty where there is no weight or bias
std::tuple<Tensor, Tensor, Tensor> group_norm_act_backward(const Tensor& d_out, const Tensor& x, const Tensor& stats,
                                                           int64_t groups, const OptTensor& weight, const OptTensor& bias,
                                                           int64_t act) {
  const c10::DeviceGuard guard(x.device());
  TORCH_CHECK_VALUE(d_out.sizes() == x.sizes(), "group_norm_act: gradient of shape ", d_out.sizes(), " for ", x.sizes());
  check_same(d_out, x.scalar_type(), x, "group_norm_act: gradient");
  const ImageRows v(x, "group_norm_act"), d(d_out, "group_norm_act");
  const int64_t b = v.b, p = v.p, c = v.c;
  check_same(stats, at::kFloat, x, "group_norm_act: stats");
  TORCH_CHECK_VALUE(stats.is_contiguous() && stats.numel() == 2 * b * groups, "group_norm_act: stats of shape ",
                    stats.sizes());
  check_vector(weight, c, x, "group_norm_act: weight");
  check_vector(bias, c, x, "group_norm_act: bias");
  const OptTensor w = dense(weight), bi = dense(bias);
  Tensor dx = empty(x.sizes(), x, x.scalar_type());
  Tensor dw = empty({weight ? c : 0}, x, weight ? weight->scalar_type() : at::kFloat);
  Tensor db = empty({bias ? c : 0}, x, bias ? bias->scalar_type() : at::kFloat);
  if (x.numel() == 0) {
    dw.zero_();
    db.zero_();
    return {dx, dw, db};
  }
  const Tensor ws = norm_workspace(v, groups, 1);
  check(fim_group_norm_backward(v.hold.data_ptr(), d.hold.data_ptr(), dtype_code(x), b, p, c, v.sb, v.sp, d.sb, d.sp,
                                groups, ptr<const void>(w), float_code(w), ptr<const void>(bi),
                                float_code(bi), (int)act, ptr<const float>(stats), dx.data_ptr(),
                                weight ? dw.data_ptr() : nullptr, bias ? db.data_ptr() : nullptr, ptr<float>(ws),
                                stream_of(x)),
        "group_norm_act backward ", x.sizes(), " in ", groups, " groups");
  return {dx, dw, db};
}

// The operands of a gated product, checked and as the C ABI reads them
struct Gated {
  Tensor x, wg, wu;
  OptTensor bg, bu;
  int64_t m, k, h;
  int bias_dtype;
  Gated(const Tensor& x_in, const Tensor& w_gate, const Tensor& w_up, const OptTensor& b_gate, const OptTensor& b_up) {
    x = matrix_rows(x_in, "gated_linear");
    m = x.size(0);
    k = x.size(1);
    check_dims(w_gate, 2, "gated_linear: w_gate");
    h = w_gate.size(0);
    TORCH_CHECK_VALUE(w_gate.size(1) == k && w_up.sizes() == w_gate.sizes(), "gated_linear: weights ", w_gate.sizes(),
                      " and ", w_up.sizes(), " for ", k, " channels");
    check_same(w_gate, x.scalar_type(), x, "gated_linear: w_gate");
    check_same(w_up, x.scalar_type(), x, "gated_linear: w_up");
    check_vector(b_gate, h, x, "gated_linear: b_gate");
    check_vector(b_up, h, x, "gated_linear: b_up");
    const auto& any = b_gate ? b_gate : b_up;
    TORCH_CHECK_TYPE(!any || any->scalar_type() == at::kFloat || any->scalar_type() == x.scalar_type(),
                     "gated_linear: biases of ", any->scalar_type(), " beside ", x.scalar_type());
    TORCH_CHECK_TYPE(!b_gate || !b_up || b_gate->scalar_type() == b_up->scalar_type(),
                     "gated_linear: biases of two types");
    wg = matrix_rows(w_gate, "gated_linear");
    wu = matrix_rows(w_up, "gated_linear");
    bg = dense(b_gate);
    bu = dense(b_up);
    bias_dtype = float_code(any);
  }
};

Tensor gated_workspace(const Gated& g, int backward) {
  int64_t bytes = 0;
  check(fim_gated_linear_workspace(g.x.data_ptr(), g.m, g.k, g.x.stride(0), g.wg.data_ptr(), g.wg.stride(0),
                                   g.wu.data_ptr(), g.wu.stride(0), g.h, backward, &bytes),
        "gated_linear ", g.m, "x", g.k, " -> ", g.h);
  return bytes > 0 ? empty({bytes}, g.x, at::kByte) : Tensor();
}

std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
  auto sizes = x.sizes().vec();
  sizes.back() = last;
  return sizes;
}

Tensor gated_linear(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const OptTensor& b_gate,
                    const OptTensor& b_up, int64_t act) {
  const c10::DeviceGuard guard(x.device());
  const Gated g(x, w_gate, w_up, b_gate, b_up);
  Tensor out = empty(with_last(x, g.h), x, x.scalar_type());
  const Tensor ws = gated_workspace(g, 0);  // undefined: none is needed
  check(fim_gated_linear(g.x.data_ptr(), dtype_code(x), g.m, g.k, g.x.stride(0), g.wg.data_ptr(), g.wg.stride(0),
                         g.wu.data_ptr(), g.wu.stride(0), g.h, ptr<const void>(g.bg), ptr<const void>(g.bu),
                         g.bias_dtype, (int)act, out.data_ptr(), ws.defined() ? ws.data_ptr() : nullptr,
                         ws.defined() ? ws.numel() : 0, stream_of(x)),
        "gated_linear ", g.m, "x", g.k, " -> ", g.h);
  return out;
}

// Gradients that are not wanted come back empty.
std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> gated_linear_backward(
    const Tensor& d_out, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const OptTensor& b_gate,
    const OptTensor& b_up, int64_t act, bool want_x, bool want_weights, bool want_biases) {
  const c10::DeviceGuard guard(x.device());
  const Gated g(x, w_gate, w_up, b_gate, b_up);
  TORCH_CHECK_VALUE(d_out.sizes() == at::IntArrayRef(with_last(x, g.h)), "gated_linear: gradient of shape ",
                    d_out.sizes(), " for ", x.sizes(), " -> ", g.h);
  check_same(d_out, x.scalar_type(), x, "gated_linear: gradient");
  Tensor d = matrix_rows(d_out, "gated_linear");
  if (d.stride(0) >= (1 << 22)) d = d.contiguous();  // (the kernels' limit)
  auto weight_grad = [&](bool want) { return want ? empty({g.h, g.k}, x, x.scalar_type()) : empty({0}, x, x.scalar_type()); };
  auto bias_grad = [&](const OptTensor& b) {
    return empty({want_biases && b ? g.h : 0}, x, b ? b->scalar_type() : at::kFloat);
  };
  Tensor dx = want_x ? empty(x.sizes(), x, x.scalar_type()) : empty({0}, x, x.scalar_type());
  Tensor dwg = weight_grad(want_weights), dwu = weight_grad(want_weights), dbg = bias_grad(b_gate), dbu = bias_grad(b_up);
  if (g.m == 0) {
    for (Tensor* t : {&dwg, &dwu, &dbg, &dbu}) t->zero_();
    return {dx, dwg, dwu, dbg, dbu};
  }
  auto out = [](const Tensor& t) { return t.numel() ? t.data_ptr() : nullptr; };
  const Tensor ws = gated_workspace(g, 1);
  check(fim_gated_linear_backward(g.x.data_ptr(), dtype_code(x), g.m, g.k, g.x.stride(0), g.wg.data_ptr(),
                                  g.wg.stride(0), g.wu.data_ptr(), g.wu.stride(0), g.h, ptr<const void>(g.bg),
                                  ptr<const void>(g.bu), g.bias_dtype, (int)act, d.data_ptr(), d.stride(0), out(dx),
                                  out(dwg), out(dwu), out(dbg), out(dbu), ws.data_ptr(), ws.numel(), stream_of(x)),
        "gated_linear backward ", g.m, "x", g.k, " -> ", g.h);
  return {dx, dwg, dwu, dbg, dbu};
}

// Refusals that the ops' predicates leave to these operators: in Python, looking at hundreds of tensors costs more than the
// kernels take
void check_grad(const Tensor& t, const Tensor& first) {
  const auto type = t.scalar_type();
  TORCH_CHECK_NOT_IMPLEMENTED(t.device() == first.device() && t.is_cuda(),
                              "no HIP impl applies: gradients on ", first.device(), " and ", t.device());
  TORCH_CHECK_NOT_IMPLEMENTED(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf,
                              "no HIP impl applies: a gradient of ", type);
}

// The gradients of a list as the C ABI takes them: dense, each in the order of its memory
struct GradList {
  std::vector<Tensor> hold;
  std::vector<const void*> ptrs;
  std::vector<int> dtypes;
  std::vector<int64_t> numel;
  explicit GradList(at::TensorList grads) {
    hold.reserve(grads.size());
    ptrs.reserve(grads.size());
    dtypes.reserve(grads.size());
    numel.reserve(grads.size());
    for (const Tensor& t : grads) {
      check_grad(t, grads[0]);
      hold.push_back(t.is_non_overlapping_and_dense() ? t : t.contiguous());
      ptrs.push_back(hold.back().data_ptr());
      dtypes.push_back(dtype_code(t));
      numel.push_back(t.numel());
    }
  }
  int64_t count() const { return (int64_t)hold.size(); }
};

int norm_code(double norm_type) {
  TORCH_CHECK_VALUE(norm_type == 2.0 || norm_type == std::numeric_limits<double>::infinity(),
                    "the norm is 2 or infinity, got ", norm_type);
  return norm_type == 2.0 ? 2 : 0;
}

Tensor grad_workspace(const GradList& g) {
  int64_t doubles = 0;
  check(fim_grad_norm_workspace(g.count(), g.numel.data(), &doubles), "grad_norm");
  return empty({doubles}, g.hold[0], at::kDouble);
}

Tensor grad_norm(at::TensorList grads, double norm_type) {
  TORCH_CHECK_VALUE(!grads.empty(), "grad_norm: no gradients");
  const c10::DeviceGuard guard(grads[0].device());
  const GradList g(grads);
  Tensor total = empty({}, grads[0], at::kFloat);
  const Tensor ws = grad_workspace(g);
  check(fim_grad_norm(g.count(), g.ptrs.data(), g.dtypes.data(), g.numel.data(), norm_code(norm_type), ptr<float>(total),
                      ptr<double>(ws), stream_of(grads[0])),
        "grad_norm");
  return total;
}

Tensor clip_grad_norm_out(at::TensorList grads, at::TensorList out, double max_norm, double norm_type) {
  TORCH_CHECK_VALUE(!grads.empty(), "clip_grad_norm_: no gradients");
  TORCH_CHECK_VALUE(grads.size() == out.size(), "clip_grad_norm_: ", out.size(), " outputs for ", grads.size(),
                    " gradients");
  const c10::DeviceGuard guard(grads[0].device());
  const GradList g(grads);
  std::vector<Tensor> to;  // written by the kernel: `out` itself where its memory lies as the gradient's
  std::vector<void*> ptrs;
  std::vector<int> dtypes;
  to.reserve(out.size());
  ptrs.reserve(out.size());
  dtypes.reserve(out.size());
  for (size_t i = 0; i < out.size(); ++i) {
    const Tensor& t = out[i];
    check_grad(t, grads[0]);
    TORCH_CHECK_NOT_IMPLEMENTED(t.sizes() == grads[i].sizes(), "no HIP impl applies: an output of shape ", t.sizes(),
                                " for a gradient of shape ", grads[i].sizes());
    const Tensor& from = g.hold[i];
    const bool same = t.is_non_overlapping_and_dense() && t.strides() == from.strides();
    to.push_back(same ? t : at::empty_strided(from.sizes(), from.strides(), t.options().requires_grad(false)));
    ptrs.push_back(to.back().data_ptr());
    dtypes.push_back(dtype_code(t));
  }
  Tensor total = empty({}, grads[0], at::kFloat);
  const Tensor ws = grad_workspace(g);
  check(fim_clip_grad_norm(g.count(), g.ptrs.data(), g.dtypes.data(), ptrs.data(), dtypes.data(), g.numel.data(),
                           (float)max_norm, norm_code(norm_type), ptr<float>(total), ptr<double>(ws),
                           stream_of(grads[0])),
        "clip_grad_norm_");
  for (size_t i = 0; i < out.size(); ++i)
    if (!to[i].is_same(out[i])) out[i].copy_(to[i]);
  return total;
}

Tensor clip_grad_norm_(at::TensorList grads, double max_norm, double norm_type) {
  return clip_grad_norm_out(grads, grads, max_norm, norm_type);
}

}  // namespace

#define FIM_GEO_SCHEMA "SymInt kh, SymInt kw, SymInt sh, SymInt sw, SymInt ph, SymInt pw, SymInt dh, SymInt dw"

// name, schema, function: one row per operator
#define FIM_OPS(X)                                                                                                     \
  X(quantize_mxfp8, "(Tensor value, Tensor exponent, SymInt padded) -> Tensor")                                        \
  X(gelu_quantize_mxfp8,                                                                                               \
    "(Tensor value, Tensor exponent, SymInt padded, Tensor? input_bias, bool tanh=False) -> Tensor")                   \
  X(quantize_int8, "(Tensor value, Tensor scale, Tensor? channel_scale) -> Tensor")                                    \
  X(gelu_quantize_int8, "(Tensor value, Tensor scale, bool tanh=False) -> Tensor")                                     \
  X(quantize_mxfp8_dynamic, "(Tensor value, bool swizzled) -> (Tensor, Tensor)")                                       \
  X(quantize_int8_rows, "(Tensor value, bool reciprocal) -> (Tensor, Tensor)")                                         \
  X(calibrate_block32, "(Tensor matrix) -> Tensor")                                                                    \
  X(int8_conv2d, "(Tensor x, Tensor weight, Tensor a_scale, Tensor w_scale, Tensor? bias, " FIM_GEO_SCHEMA             \
                 ", bool relu, bool gelu, Tensor? residual, Tensor? out_scale) -> Tensor")                             \
  X(int8_conv2d_maxpool, "(Tensor x, Tensor weight, Tensor a_scale, Tensor w_scale, Tensor? bias, " FIM_GEO_SCHEMA     \
                         ", bool relu, Tensor out_scale) -> (Tensor, Tensor)")                                         \
  X(mxfp8_conv2d, "(Tensor x, Tensor channel_exponent, Tensor weight, Tensor weight_exponent, Tensor? bias, "          \
                  FIM_GEO_SCHEMA ", bool relu, bool gelu, Tensor? residual, Tensor? out_exponent) -> Tensor")          \
  X(int8_linear, "(Tensor a, Tensor weight, Tensor a_scale, Tensor w_scale, Tensor? bias, bool relu, bool gelu, "      \
                 "Tensor? residual) -> Tensor")                                                                        \
  X(int8_linear_quantize_, "(Tensor a, Tensor weight, Tensor a_scale, Tensor w_scale, Tensor? bias, "                  \
                           "Tensor out_scale, Tensor(a!) out) -> ()")                                                  \
  X(mxfp8_scaled_mm, "(Tensor a, Tensor a_scale_swizzled, Tensor weight, Tensor weight_exponent, Tensor? bias, "       \
                     "bool weight_scale_e8m0=False) -> Tensor")                                                        \
  X(im2col_gather, "(Tensor x, " FIM_GEO_SCHEMA ") -> Tensor")                                                         \
  X(refiner_mlp, "(SymInt kind, SymInt semantics, Tensor x, Tensor x_scale, Tensor w1, Tensor w1_scale, Tensor? b1, "  \
                 "Tensor h_scale, Tensor w2, Tensor w2_scale, Tensor? b2, Tensor? residual) -> Tensor")                \
  X(depthwise5x5, "(Tensor x, Tensor weight, Tensor bias, SymInt act, SymInt mode, Tensor? scale, Tensor? exponent) "  \
                  "-> Tensor")                                                                                         \
  X(depthwise5x5_mx_dynamic, "(Tensor x, Tensor weight, Tensor bias) -> (Tensor, Tensor)")                             \
  X(depthwise5x5_relu_pointwise_mxfp8, "(Tensor x, Tensor dw_weight, Tensor dw_bias, Tensor pw_weight, "               \
                                       "Tensor pw_e8m0, Tensor? pw_bias) -> Tensor")                                   \
  X(depthwise5x5_relu_pointwise_int8, "(Tensor x, Tensor dw_weight, Tensor dw_bias, Tensor scale, Tensor pw_weight, "  \
                                      "Tensor pw_wscale, Tensor? pw_bias) -> Tensor")                                  \
  X(conv3x3_small_cin_quantize_int8, "(Tensor x, Tensor packed, Tensor bias, Tensor scale) -> Tensor")                 \
  X(bias_relu_quantize_int8, "(Tensor raw, Tensor bias, Tensor scale) -> Tensor")                                      \
  X(pointwise_bf16, "(Tensor x, Tensor weight, Tensor? bias) -> Tensor")                                               \
  X(group_norm_act_backward, "(Tensor d_out, Tensor x, Tensor stats, int groups, Tensor? weight, Tensor? bias, "       \
                             "int act) -> (Tensor, Tensor, Tensor)")                                                   \
  X(gated_linear_backward, "(Tensor d_out, Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, "       \
                           "int act, bool want_x, bool want_weights, bool want_biases) "                               \
                           "-> (Tensor, Tensor, Tensor, Tensor, Tensor)")                                              \
  X(grad_norm, "(Tensor[] grads, float norm_type) -> Tensor")

// those with an autograd kernel of their own (below)
#define FIM_AUTOGRAD_OPS(X)                                                                                            \
  X(clip_grad_norm_, "(Tensor(a!)[] grads, float max_norm, float norm_type) -> Tensor")                                \
  X(clip_grad_norm_out, "(Tensor[] grads, Tensor(a!)[] out, float max_norm, float norm_type) -> Tensor")               \
  X(group_norm_act, "(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, int act) -> (Tensor, Tensor)")    \
  X(gated_linear, "(Tensor x, Tensor w_gate, Tensor w_up, Tensor? b_gate, Tensor? b_up, int act) -> Tensor")

TORCH_LIBRARY(flashim_amd, m) {
#define X(name, schema) m.def(#name schema, {at::Tag::pt2_compliant_tag});
  FIM_OPS(X)
  FIM_AUTOGRAD_OPS(X)
#undef X
}

TORCH_LIBRARY_IMPL(flashim_amd, CUDA, m) {
#define X(name, schema) m.impl(#name, TORCH_FN(name));
  FIM_OPS(X)
  FIM_AUTOGRAD_OPS(X)
#undef X
}

namespace {

// No derivative formulas. Reverse mode: the outputs of inputs that require a gradient carry a node that raises. Forward
// mode alone: the tangents of dual inputs stop here and the outputs have none (torch's own fallback for operators without
// formulas refuses every dual input).
void no_derivative(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const std::string& name = op.schema().name();
  torch::autograd::variable_list inputs;  // that require a gradient
  if (at::GradMode::is_enabled()) {
    bool dual = false;
    auto look = [&](const Tensor& t) {
      if (t.requires_grad()) inputs.push_back(t);
      dual = dual || torch::autograd::isFwGradDefined(t);
    };
    for (const c10::IValue& arg : torch::jit::last(*stack, op.schema().arguments().size())) {
      if (arg.isTensor()) look(arg.toTensor());
      if (arg.isTensorList())
        for (const Tensor& t : arg.toTensorVector()) look(t);
    }
    TORCH_CHECK_NOT_IMPLEMENTED(inputs.empty() || !dual, name,
                                ": no forward-mode derivative, and an input requires a gradient");
  }
  {
    at::AutoDispatchBelowAutograd guard;
    op.redispatchBoxed(keys & c10::after_autograd_keyset, stack);
  }
  if (inputs.empty()) return;
  std::shared_ptr<torch::autograd::Node> node(new torch::autograd::NotImplemented(name), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(inputs));
  for (const c10::IValue& out : torch::jit::last(*stack, op.schema().returns().size()))
    if (out.isTensor() && torch::autograd::isDifferentiableType(out.toTensor().scalar_type()))
      torch::autograd::set_history(out.toTensor(), node);
}

// The version counters of the arguments that are written, by which autograd finds a saved tensor that was overwritten
// since (torch's own fallback counts for returned tensors only).
void count_writes(const c10::OperatorHandle& op, c10::DispatchKeySet keys, torch::jit::Stack* stack) {
  const auto& args = op.schema().arguments();
  std::vector<Tensor> written;
  for (size_t i = 0; i < args.size(); ++i) {
    if (args[i].alias_info() == nullptr || !args[i].alias_info()->isWrite()) continue;
    const c10::IValue& arg = torch::jit::peek(*stack, i, args.size());
    if (arg.isTensor()) written.push_back(arg.toTensor());
    if (arg.isTensorList())
      for (const Tensor& t : arg.toTensorVector()) written.push_back(t);
  }
  {
    at::AutoDispatchBelowADInplaceOrView guard;
    op.redispatchBoxed(keys & c10::after_ADInplaceOrView_keyset, stack);
  }
  for (const Tensor& t : written)
    if (!t.is_inference()) torch::autograd::increment_version(t);
}

// Clipping below autograd, the versions of what it wrote counted: as no_derivative and count_writes do for any operator, but
// without boxing hundreds of tensors. A tangent is refused whatever the mode: the tensor's values would change and its tangent
// stay, or an output keep the tangent of what it held.
void refuse_derivatives(at::TensorList tensors) {
  const bool grads = at::GradMode::is_enabled();
  // (no level, no tangents: one look a call, not one a tensor)
  const bool tangents = torch::autograd::ForwardADLevel::try_get_by_idx(0) != nullptr;
  if (!grads && !tangents) return;
  for (const Tensor& t : tensors) {
    TORCH_CHECK_NOT_IMPLEMENTED(!grads || !t.requires_grad(), "clip_grad_norm_: no derivative, and a tensor requires a gradient");
    TORCH_CHECK_NOT_IMPLEMENTED(!tangents || !torch::autograd::isFwGradDefined(t),
                                "clip_grad_norm_: no derivative, and a tensor has a tangent");
  }
}

void count_writes_to(at::TensorList tensors) {
  for (const Tensor& t : tensors)
    if (!t.is_inference()) torch::autograd::increment_version(t);
}

// Derivatives: each a torch operator of its own, so that compiled graphs hold it (and a second derivative raises).
OptTensor as_optional(const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); }
Tensor as_tensor(const OptTensor& t) { return t ? *t : Tensor(); }

template <typename Signature>
c10::TypedOperatorHandle<Signature> typed_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}

Tensor clip_grad_norm_out_autograd(at::TensorList grads, at::TensorList out, double max_norm, double norm_type) {
  refuse_derivatives(grads);
  refuse_derivatives(out);
  static const auto op = typed_op<decltype(clip_grad_norm_out)>("flashim_amd::clip_grad_norm_out");
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor total = op.call(grads, out, max_norm, norm_type);
  count_writes_to(out);
  return total;
}

Tensor clip_grad_norm_autograd_(at::TensorList grads, double max_norm, double norm_type) {
  refuse_derivatives(grads);
  static const auto op = typed_op<decltype(clip_grad_norm_)>("flashim_amd::clip_grad_norm_");
  at::AutoDispatchBelowADInplaceOrView guard;
  Tensor total = op.call(grads, max_norm, norm_type);
  count_writes_to(grads);
  return total;
}

// The backward operators are linear in the incoming gradient, but stop its tangents
void refuse_tangent(const Tensor& grad, const char* name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!torch::autograd::isFwGradDefined(grad), name, ": no forward-mode derivative of the backward pass");
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x, int64_t groups,
                                                const OptTensor& weight, const OptTensor& bias, double eps, int64_t act) {
    at::AutoDispatchBelowAutograd guard;
    static const auto op = typed_op<decltype(group_norm_act)>("flashim_amd::group_norm_act");
    auto [out, stats] = op.call(x, groups, weight, bias, eps, act);
    ctx->save_for_backward({x, as_tensor(weight), as_tensor(bias), stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    ctx->mark_non_differentiable({stats});
    return {out, stats};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    refuse_tangent(grads[0], "group_norm_act");
    const auto saved = ctx->get_saved_variables();
    std::optional<at::AutoDispatchBelowAutograd> below;  // (nothing is recorded: past the refusal of second derivatives)
    if (!at::GradMode::is_enabled()) below.emplace();
    static const auto op = typed_op<decltype(group_norm_act_backward)>("flashim_amd::group_norm_act_backward");
    auto [dx, dw, db] = op.call(grads[0], saved[0], saved[3], ctx->saved_data["groups"].toInt(), as_optional(saved[1]),
                                as_optional(saved[2]), ctx->saved_data["act"].toInt());
    return {dx, Tensor(), saved[1].defined() ? dw : Tensor(), saved[2].defined() ? db : Tensor(), Tensor(), Tensor()};
  }
};

// Whether an operator has anything to record, or a tangent to refuse (no_grad ends the recording, not forward mode): a node
// costs 2 us of host time
template <typename... Tensors>
bool records(const Tensors&... tensors) {
  const bool grads = at::GradMode::is_enabled();
  const auto one = [grads](const OptTensor& t) {
    return t && t->defined() && ((grads && t->requires_grad()) || torch::autograd::isFwGradDefined(*t));
  };
  return (one(tensors) || ...);
}

std::tuple<Tensor, Tensor> group_norm_act_autograd(const Tensor& x, int64_t groups, const OptTensor& weight,
                                                   const OptTensor& bias, double eps, int64_t act) {
  if (!records(x, weight, bias)) {
    at::AutoDispatchBelowAutograd guard;
    static const auto op = typed_op<decltype(group_norm_act)>("flashim_amd::group_norm_act");
    return op.call(x, groups, weight, bias, eps, act);
  }
  auto out = GroupNormAct::apply(x, groups, weight, bias, eps, act);
  return {out[0], out[1]};
}

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up,
                        const OptTensor& b_gate, const OptTensor& b_up, int64_t act) {
    at::AutoDispatchBelowAutograd guard;
    static const auto op = typed_op<decltype(gated_linear)>("flashim_amd::gated_linear");
    ctx->save_for_backward({x, w_gate, w_up, as_tensor(b_gate), as_tensor(b_up)});
    ctx->saved_data["act"] = act;
    return op.call(x, w_gate, w_up, b_gate, b_up, act);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    if (!grads[0].defined()) return {Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    refuse_tangent(grads[0], "gated_linear");
    const auto saved = ctx->get_saved_variables();
    std::optional<at::AutoDispatchBelowAutograd> below;  // (nothing is recorded: past the refusal of second derivatives)
    if (!at::GradMode::is_enabled()) below.emplace();
    const bool want_x = ctx->needs_input_grad(0);
    const bool want_w = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const bool bias[2] = {saved[3].defined(), saved[4].defined()};
    bool want_b = false;  // (the edges count the tensors that are there)
    for (int i = 3; i < 3 + bias[0] + bias[1]; ++i) want_b = want_b || ctx->needs_input_grad(i);
    static const auto op = typed_op<decltype(gated_linear_backward)>("flashim_amd::gated_linear_backward");
    auto [dx, dwg, dwu, dbg, dbu] = op.call(grads[0], saved[0], saved[1], saved[2], as_optional(saved[3]),
                                            as_optional(saved[4]), ctx->saved_data["act"].toInt(), want_x, want_w, want_b);
    return {want_x ? dx : Tensor(),  want_w ? dwg : Tensor(),           want_w ? dwu : Tensor(),
            want_b && bias[0] ? dbg : Tensor(), want_b && bias[1] ? dbu : Tensor(), Tensor()};
  }
};

Tensor gated_linear_autograd(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const OptTensor& b_gate,
                             const OptTensor& b_up, int64_t act) {
  if (!records(x, w_gate, w_up, b_gate, b_up)) {
    at::AutoDispatchBelowAutograd guard;
    static const auto op = typed_op<decltype(gated_linear)>("flashim_amd::gated_linear");
    return op.call(x, w_gate, w_up, b_gate, b_up, act);
  }
  return GatedLinear::apply(x, w_gate, w_up, b_gate, b_up, act);
}

}  // namespace

TORCH_LIBRARY_IMPL(flashim_amd, Autograd, m) {
#define X(name, schema) m.impl(#name, torch::CppFunction::makeFromBoxedFunction<&no_derivative>());
  FIM_OPS(X)
#undef X
  m.impl("group_norm_act", TORCH_FN(group_norm_act_autograd));
  m.impl("gated_linear", TORCH_FN(gated_linear_autograd));
  m.impl("clip_grad_norm_", TORCH_FN(clip_grad_norm_autograd_));
  m.impl("clip_grad_norm_out", TORCH_FN(clip_grad_norm_out_autograd));
}

TORCH_LIBRARY_IMPL(flashim_amd, ADInplaceOrView, m) {
  for (const char* name : {"int8_linear_quantize_", "clip_grad_norm_", "clip_grad_norm_out"})
    m.impl(name, torch::CppFunction::makeFromBoxedFunction<&count_writes>());
}

// clip_grad_norm_ (out None) and clip_grad_norm_out of Python lists or tuples, through the same dispatcher: torch's binding
// of operators converts a list of tensors three times over, 0.12 us a tensor, which for hundreds of gradients is more than
// the kernels take. None where an element is not a plain tensor (a subclass has its own say in operators): the caller then
// goes through torch.ops. Called with the GIL held.
extern "C" PyObject* flashim_amd_clip_lists(PyObject* grads, PyObject* out, double max_norm, double norm_type) {
  HANDLE_TH_ERRORS
  const auto unpack = [](PyObject* list, std::vector<Tensor>& to) {
    if (!PyList_Check(list) && !PyTuple_Check(list)) return false;
    const Py_ssize_t n = PySequence_Fast_GET_SIZE(list);
    to.reserve(n);
    for (Py_ssize_t i = 0; i < n; ++i) {
      PyObject* item = PySequence_Fast_GET_ITEM(list, i);
      if (!THPVariable_CheckExact(item)) return false;
      to.push_back(THPVariable_Unpack(item));
    }
    return true;
  };
  std::vector<Tensor> from, to;
  if (!unpack(grads, from) || (out != Py_None && !unpack(out, to))) Py_RETURN_NONE;
  static const auto in_place = typed_op<decltype(clip_grad_norm_)>("flashim_amd::clip_grad_norm_");
  static const auto into = typed_op<decltype(clip_grad_norm_out)>("flashim_amd::clip_grad_norm_out");
  Tensor total;
  {
    pybind11::gil_scoped_release release;
    total = out == Py_None ? in_place.call(from, max_norm, norm_type) : into.call(from, to, max_norm, norm_type);
  }
  return THPVariable_Wrap(total);
  END_HANDLE_TH_ERRORS
}
