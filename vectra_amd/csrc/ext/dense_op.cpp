// torch.library registration of the dense operators around a block's attention:
//   linear           act(x W^T + b) + residual
//   gated_linear     act(x G^T + b_g) * (x U^T + b_u)
//   linear_backward  the gradients of either
//   quantize_rows, dequantize_rows   the 8-bit form of rows
//
//   CUDA key (HIP tensors on ROCm)  -> libvectra_dense.so (include/vectra_dense.h),
//                                      on the caller's current HIP stream, with
//                                      scratch memory from torch's allocator
//   CPU key                         -> the same formulas in fp32 tensors
//   Autograd key                    -> the layers: saves the input (or its 8-bit
//                                      form), calls linear_backward; the others:
//                                      no derivative, refused
//   Autocast keys                   -> the layers in autocast's type, as
//                                      torch's own linear layers are
//   fake/meta                       -> registered from Python
// There is no CPU fallback for device tensors: if the HIP library cannot be
// loaded this extension does not load either.

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <algorithm>
#include <array>
#include <cmath>
#include <optional>
#include <string_view>
#include <vector>

#include "op_common.h"
#include "vectra_dense.h"

namespace {

using namespace vectra_ops;

constexpr int64_t kBlock = 32;  // elements of a row that share a power of two

bool eight_bit(std::string_view checkpoint, const char* op) {
  TORCH_CHECK_VALUE(checkpoint == "none" || checkpoint == "e4m3", op, ": checkpoint must be 'none' or 'e4m3'; got '",
                    std::string(checkpoint), "'");
  return checkpoint == "e4m3";
}

void check_residual_shape(const Tensor& x, const Tensor& weight, const Tensor& residual, const char* op) {
  bool same = residual.dim() == x.dim() && residual.size(-1) == weight.size(0);
  for (int64_t d = 0; same && d + 1 < x.dim(); ++d) same = residual.size(d) == x.size(d);
  TORCH_CHECK(same, op, ": residual must have the output's shape; got ", residual.sizes());
}

void check_layer(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual, bool gated,
                 const char* op) {
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2, op, ": x must be [..., width_in] and weight [width, width_in]; got ",
              x.sizes(), " and ", weight.sizes());
  TORCH_CHECK(x.size(-1) == weight.size(1), op, ": x's last dimension ", x.size(-1), " is not weight's ",
              weight.size(1));
  TORCH_CHECK(!gated || weight.size(0) % 2 == 0, op,
              ": weight must hold the gate's rows and as many rows of the up projection; got ", weight.sizes());
  TORCH_CHECK(dense_dtype(x.scalar_type()) >= 0, op, ": x must be float32, float16 or bfloat16; got ", x.scalar_type());
  TORCH_CHECK(weight.scalar_type() == x.scalar_type(), op, ": x and weight must share a dtype; got ", x.scalar_type(),
              " and ", weight.scalar_type());
  TORCH_CHECK(weight.device() == x.device(), op, ": weight must be on ", x.device(), "; got ", weight.device());
  if (has(bias)) {
    TORCH_CHECK(bias->dim() == 1 && bias->size(0) == weight.size(0), op, ": bias must be [", weight.size(0), "]; got ",
                bias->sizes());
    TORCH_CHECK(bias->scalar_type() == x.scalar_type() || bias->scalar_type() == at::kFloat, op,
                ": bias must have x's dtype or float32; got ", bias->scalar_type());
    TORCH_CHECK(bias->device() == x.device(), op, ": bias must be on ", x.device(), "; got ", bias->device());
  }
  if (has(residual)) {
    check_residual_shape(x, weight, *residual, op);
    TORCH_CHECK(residual->scalar_type() == x.scalar_type(), op, ": residual must have x's dtype; got ",
                residual->scalar_type());
    TORCH_CHECK(residual->device() == x.device(), op, ": residual must be on ", x.device(), "; got ",
                residual->device());
  }
}

// Scales [..., ceil(width / 32)] beside codes [..., width].
bool scales_fit(const Tensor& codes, const Tensor& scales) {
  return codes.dim() >= 1 && scales.sizes() == at::IntArrayRef(with_last(codes, (codes.size(-1) + kBlock - 1) / kBlock));
}

void check_status(int status, const char* op) {
  TORCH_CHECK(status == VECTRA_DENSE_OK, op, ": ", vectra_dense_status_string(status));
}

vectra_dense_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<vectra_dense_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

// ---------------------------------------------------------------- device

Tensor forward_hip(const Tensor& x, const Tensor& weight, const OptTensor& bias_in, const OptTensor& residual,
                   int32_t activation, bool gated, const char* op) {
  c10::DeviceGuard guard(x.device());
  const int64_t n = gated ? weight.size(0) / 2 : weight.size(0);
  Tensor out = at::empty(with_last(x, n), x.options());
  const Rows xr = as_rows(x), wr = as_rows(weight);
  const Tensor bias = has(bias_in) ? bias_in->contiguous() : Tensor();
  Rows rr;
  if (has(residual)) rr = as_rows(*residual);
  vectra_dense_args a{};
  a.struct_size = sizeof(a);
  a.x = xr.t.data_ptr();
  a.weight = wr.t.data_ptr();
  a.bias = bias.defined() ? bias.data_ptr() : nullptr;
  a.residual = rr.t.defined() ? rr.t.data_ptr() : nullptr;
  a.out = out.data_ptr();
  a.dtype = dense_dtype(x.scalar_type());
  a.bias_dtype = bias.defined() ? dense_dtype(bias.scalar_type()) : a.dtype;
  a.activation = activation;
  a.gated = gated;
  a.rows = rows_of(x);
  a.width_in = x.size(-1);
  a.width_out = n;
  a.x_stride = xr.stride;
  a.weight_stride = wr.stride;
  a.residual_stride = rr.stride;
  a.out_stride = std::max<int64_t>(n, 1);
  const int64_t need = vectra_dense_forward_workspace_bytes(&a);
  if (need < 0) check_status(static_cast<int>(-need), op);
  Tensor workspace;
  if (need > 0) workspace = at::empty({need}, x.options().dtype(at::kByte));
  check_status(vectra_dense_forward(&a, need > 0 ? workspace.data_ptr() : nullptr, need, stream_of(x)), op);
  return out;
}

Tensor linear_hip(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                  c10::string_view activation, c10::string_view checkpoint) {
  constexpr const char* op = "vectra::linear";
  check_layer(x, weight, bias, residual, false, op);
  eight_bit(checkpoint, op);
  return forward_hip(x, weight, bias, residual, activation_of(activation, op), false, op);
}

Tensor gated_linear_hip(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation,
                        c10::string_view checkpoint) {
  constexpr const char* op = "vectra::gated_linear";
  check_layer(x, weight, bias, std::nullopt, true, op);
  eight_bit(checkpoint, op);
  return forward_hip(x, weight, bias, std::nullopt, activation_of(activation, op), true, op);
}

void check_backward(const Tensor& grad, const Tensor& x, const OptTensor& scales, const Tensor& weight,
                    const OptTensor& bias, bool gated, at::ArrayRef<bool> wanted) {
  constexpr const char* op = "vectra::linear_backward";
  TORCH_CHECK(wanted.size() == 3, op, ": wanted must name three gradients (x, weight, bias)");
  if (has(scales)) {
    TORCH_CHECK(x.scalar_type() == at::kFloat8_e4m3fn && scales->scalar_type() == at::kFloat8_e8m0fnu, op,
                ": an input given with scales must be float8_e4m3fn codes and float8_e8m0fnu scales; got ",
                x.scalar_type(), " and ", scales->scalar_type());
    TORCH_CHECK(scales_fit(x, *scales), op, ": scales must be [..., ceil(width_in / 32)]; got ", scales->sizes(),
                " for codes ", x.sizes());
    TORCH_CHECK(scales->device() == x.device(), op, ": scales must be on ", x.device());
    check_layer(grad.new_empty({0, x.size(-1)}, x.options().dtype(weight.scalar_type())), weight, bias, std::nullopt,
                gated, op);
  } else {
    check_layer(x, weight, bias, std::nullopt, gated, op);
  }
  const int64_t n = gated ? weight.size(0) / 2 : weight.size(0);
  bool same = grad.dim() == x.dim() && grad.size(-1) == n;
  for (int64_t d = 0; same && d + 1 < x.dim(); ++d) same = grad.size(d) == x.size(d);
  TORCH_CHECK(same, op, ": grad must have the output's shape; got ", grad.sizes());
  TORCH_CHECK(grad.scalar_type() == weight.scalar_type() && grad.device() == x.device(), op,
              ": grad must have weight's dtype and device; got ", grad.scalar_type(), " on ", grad.device());
}

std::vector<Tensor> linear_backward_hip(const Tensor& grad, const Tensor& x, const OptTensor& scales,
                                        const Tensor& weight, const OptTensor& bias_in, c10::string_view activation,
                                        bool gated, std::array<bool, 3> wanted) {
  constexpr const char* op = "vectra::linear_backward";
  check_backward(grad, x, scales, weight, bias_in, gated, wanted);
  const int32_t act = activation_of(activation, op);
  c10::DeviceGuard guard(x.device());
  const Rows gr = as_rows(grad), wr = as_rows(weight);
  Rows xr, sr;
  const Tensor bias = has(bias_in) ? bias_in->contiguous() : Tensor();
  std::vector<Tensor> out;
  Tensor dx, dw, db;
  vectra_dense_grad_args a{};
  a.struct_size = sizeof(a);
  if (has(scales)) {
    xr = as_rows(x.view(at::kByte));
    sr = as_rows(scales->view(at::kByte));
    a.codes = xr.t.data_ptr();
    a.scales = sr.t.data_ptr();
    a.codes_stride = xr.stride;
    a.scales_stride = sr.stride;
  } else if (gated || act != VECTRA_DENSE_NONE || wanted[1]) {  // (else x's values are not read)
    xr = as_rows(x);
    a.x = xr.t.data_ptr();
    a.x_stride = xr.stride;
  }
  if (wanted[0]) out.push_back(dx = at::empty(x.sizes(), weight.options()));
  if (wanted[1]) out.push_back(dw = at::empty(weight.sizes(), weight.options()));
  if (wanted[2]) out.push_back(db = at::empty({weight.size(0)}, bias.defined() ? bias.options() : weight.options()));
  a.weight = wr.t.data_ptr();
  a.bias = bias.defined() ? bias.data_ptr() : nullptr;
  a.grad = gr.t.data_ptr();
  a.dx = dx.defined() ? dx.data_ptr() : nullptr;
  a.dweight = dw.defined() ? dw.data_ptr() : nullptr;
  a.dbias = db.defined() ? db.data_ptr() : nullptr;
  a.dtype = dense_dtype(weight.scalar_type());
  a.bias_dtype = bias.defined() ? dense_dtype(bias.scalar_type()) : a.dtype;
  a.activation = act;
  a.gated = gated;
  a.rows = rows_of(x);
  a.width_in = x.size(-1);
  a.width_out = gated ? weight.size(0) / 2 : weight.size(0);
  a.weight_stride = wr.stride;
  a.grad_stride = gr.stride;
  a.dx_stride = a.dweight_stride = std::max<int64_t>(a.width_in, 1);
  const int64_t need = vectra_dense_backward_workspace_bytes(&a);
  if (need < 0) check_status(static_cast<int>(-need), op);
  Tensor workspace;
  if (need > 0) workspace = at::empty({need}, weight.options().dtype(at::kByte));
  check_status(vectra_dense_backward(&a, need > 0 ? workspace.data_ptr() : nullptr, need, stream_of(x)), op);
  return out;
}

void check_rows(const Tensor& x) {
  TORCH_CHECK(x.dim() >= 1, "vectra::quantize_rows: x must be [..., width]; got a scalar");
  TORCH_CHECK(dense_dtype(x.scalar_type()) >= 0, "vectra::quantize_rows: x must be float32, float16 or bfloat16; got ",
              x.scalar_type());
}

std::tuple<Tensor, Tensor> quantize_rows_hip(const Tensor& x) {
  check_rows(x);
  c10::DeviceGuard guard(x.device());
  const int64_t width = x.size(-1), blocks = (width + kBlock - 1) / kBlock;
  const Rows xr = as_rows(x);
  Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scales = at::empty(with_last(x, blocks), x.options().dtype(at::kFloat8_e8m0fnu));
  check_status(vectra_rows_quantize(xr.t.data_ptr(), dense_dtype(x.scalar_type()), rows_of(x), width, xr.stride,
                                    codes.data_ptr(), std::max<int64_t>(width, 1), scales.data_ptr(),
                                    std::max<int64_t>(blocks, 1), stream_of(x)),
               "vectra::quantize_rows");
  return {codes, scales};
}

void check_codes(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  constexpr const char* op = "vectra::dequantize_rows";
  TORCH_CHECK(codes.scalar_type() == at::kFloat8_e4m3fn && scales.scalar_type() == at::kFloat8_e8m0fnu, op,
              ": codes must be float8_e4m3fn and scales float8_e8m0fnu; got ", codes.scalar_type(), " and ",
              scales.scalar_type());
  TORCH_CHECK(scales_fit(codes, scales), op, ": scales must be [..., ceil(width / 32)]; got ", scales.sizes(),
              " for codes ", codes.sizes());
  TORCH_CHECK(scales.device() == codes.device(), op, ": scales must be on ", codes.device());
  TORCH_CHECK(dense_dtype(dtype) >= 0, op, ": dtype must be float32, float16 or bfloat16; got ", dtype);
}

Tensor dequantize_rows_hip(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  check_codes(codes, scales, dtype);
  c10::DeviceGuard guard(codes.device());
  const Rows cr = as_rows(codes.view(at::kByte)), sr = as_rows(scales.view(at::kByte));
  Tensor out = at::empty(codes.sizes(), codes.options().dtype(dtype));
  const int64_t width = codes.size(-1);
  check_status(vectra_rows_dequantize(cr.t.data_ptr(), cr.stride, sr.t.data_ptr(), sr.stride, dense_dtype(dtype),
                                      rows_of(codes), width, out.data_ptr(), std::max<int64_t>(width, 1),
                                      stream_of(codes)),
               "vectra::dequantize_rows");
  return out;
}

// ------------------------------------------------------------------- host
//
// The operators off the GPU: the same formulas on fp32 tensors.

Tensor project_cpu(const Tensor& x, const Tensor& weight, const OptTensor& bias) {
  Tensor z = at::matmul(x.to(at::kFloat), weight.to(at::kFloat).t());
  return has(bias) ? z + bias->to(at::kFloat) : z;
}

Tensor linear_cpu(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                  c10::string_view activation, c10::string_view checkpoint) {
  constexpr const char* op = "vectra::linear";
  check_layer(x, weight, bias, residual, false, op);
  eight_bit(checkpoint, op);
  const int32_t act = activation_of(activation, op);
  Tensor y = project_cpu(x, weight, bias);
  if (act != VECTRA_DENSE_NONE) y = activation_cpu(y, act).first;
  if (has(residual)) y = y + residual->to(at::kFloat);
  return y.to(x.scalar_type()).contiguous();
}

Tensor gated_linear_cpu(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation,
                        c10::string_view checkpoint) {
  constexpr const char* op = "vectra::gated_linear";
  check_layer(x, weight, bias, std::nullopt, true, op);
  eight_bit(checkpoint, op);
  const auto z = project_cpu(x, weight, bias).chunk(2, -1);
  return (activation_cpu(z[0], activation_of(activation, op)).first * z[1]).to(x.scalar_type()).contiguous();
}

std::tuple<Tensor, Tensor> quantize_rows_cpu(const Tensor& x) {
  check_rows(x);
  const int64_t width = x.size(-1), rows = rows_of(x), blocks = (width + kBlock - 1) / kBlock;
  const bool half = x.scalar_type() == at::kHalf;
  const int32_t lowest = half ? -15 : -117, highest = half ? 8 : 120;
  const Tensor xf = x.to(at::kFloat).reshape({rows, width}).contiguous();
  Tensor values = at::empty({rows, width}, xf.options());
  Tensor scales = at::empty({rows, blocks}, x.options().dtype(at::kByte));
  const float* p = xf.const_data_ptr<float>();
  float* v = values.mutable_data_ptr<float>();
  uint8_t* s = scales.mutable_data_ptr<uint8_t>();
  for (int64_t r = 0; r < rows; ++r) {
    for (int64_t b = 0; b < blocks; ++b) {
      const int64_t first = r * width + b * kBlock, last = std::min(first + kBlock, (r + 1) * width);
      float largest = 0.f;
      for (int64_t i = first; i < last; ++i)
        if (std::isfinite(p[i])) largest = std::max(largest, std::fabs(p[i]));
      int e = lowest;
      if (largest > 0.f) {
        int x2 = 0;
        const float m = std::frexp(largest, &x2);  // largest = m 2^x2, m in [1/2, 1); 448 = 0.875 * 2^9
        e = std::max(lowest, x2 - 9 + (m > 0.875f ? 1 : 0));
      }
      for (int64_t i = first; i < last; ++i) {
        float y = std::isfinite(p[i]) ? std::ldexp(p[i], -e) : std::nanf("");
        if (e == highest && std::fabs(y) >= 248.f) y = std::copysign(240.f, y);
        v[i] = y;
      }
      s[r * blocks + b] = static_cast<uint8_t>(e + 127);
    }
  }
  return {values.to(at::kFloat8_e4m3fn).reshape(x.sizes()), scales.view(at::kFloat8_e8m0fnu).reshape(with_last(x, blocks))};
}

Tensor dequantize_rows_cpu(const Tensor& codes, const Tensor& scales, at::ScalarType dtype) {
  check_codes(codes, scales, dtype);
  const Tensor s = scales.contiguous().view(at::kByte).to(at::kInt) - 127;
  const Tensor wide = s.repeat_interleave(kBlock, -1).narrow(-1, 0, codes.size(-1));
  const Tensor value = at::ldexp(codes.to(at::kDouble), wide);
  return at::where(wide == 128, at::full_like(value, std::nan("")), value).to(dtype);
}

std::vector<Tensor> linear_backward_cpu(const Tensor& grad, const Tensor& x_in, const OptTensor& scales,
                                        const Tensor& weight, const OptTensor& bias, c10::string_view activation,
                                        bool gated, std::array<bool, 3> wanted) {
  check_backward(grad, x_in, scales, weight, bias, gated, wanted);
  const int32_t act = activation_of(activation, "vectra::linear_backward");
  const int64_t k = x_in.size(-1), rows = rows_of(x_in), n = grad.size(-1);
  const Tensor x = (has(scales) ? dequantize_rows_cpu(x_in, *scales, weight.scalar_type()) : x_in)
                       .to(at::kFloat).reshape({rows, k});
  const Tensor g = grad.to(at::kFloat).reshape({rows, n});
  Tensor dz = g;
  if (gated) {
    const auto z = project_cpu(x, weight, bias).chunk(2, -1);
    const auto [value, slope] = activation_cpu(z[0], act);
    dz = at::cat({g * z[1] * slope, g * value}, 1);
  } else if (act != VECTRA_DENSE_NONE) {
    dz = g * activation_cpu(project_cpu(x, weight, bias), act).second;
  }
  std::vector<Tensor> out;
  if (wanted[0]) out.push_back(at::matmul(dz, weight.to(at::kFloat)).to(weight.scalar_type()).reshape(x_in.sizes()));
  if (wanted[1]) out.push_back(at::matmul(dz.t(), x).to(weight.scalar_type()).contiguous());
  if (wanted[2]) out.push_back(dz.sum(0).to(has(bias) ? bias->scalar_type() : weight.scalar_type()));
  return out;
}

// --------------------------------------------------------------- gradients

Tensor call_linear(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                   c10::string_view activation, c10::string_view checkpoint) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vectra::linear", "")
                       .typed<Tensor(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, c10::string_view,
                                     c10::string_view)>();
  return op.call(x, weight, bias, residual, activation, checkpoint);
}

Tensor call_gated(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation,
                  c10::string_view checkpoint) {
  static auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra::gated_linear", "")
          .typed<Tensor(const Tensor&, const Tensor&, const OptTensor&, c10::string_view, c10::string_view)>();
  return op.call(x, weight, bias, activation, checkpoint);
}

std::tuple<Tensor, Tensor> call_quantize(const Tensor& x) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vectra::quantize_rows", "")
                       .typed<std::tuple<Tensor, Tensor>(const Tensor&)>();
  return op.call(x);
}

std::vector<Tensor> call_backward(const Tensor& grad, const Tensor& x, const OptTensor& scales, const Tensor& weight,
                                  const OptTensor& bias, c10::string_view activation, bool gated,
                                  std::array<bool, 3> wanted) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vectra::linear_backward", "")
                       .typed<std::vector<Tensor>(const Tensor&, const Tensor&, const OptTensor&, const Tensor&,
                                                  const OptTensor&, c10::string_view, bool, std::array<bool, 3>)>();
  return op.call(grad, x, scales, weight, bias, activation, gated, wanted);
}

// One function for both operators.  Saved: the weight, the bias, and the input
// (or its 8-bit form) where a gradient needs it; no pre-activation is kept.
class Layer : public torch::autograd::Function<Layer> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& weight,
                        const OptTensor& bias, const OptTensor& residual, const std::string& activation,
                        const std::string& checkpoint, bool gated) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor y = gated ? call_gated(x, weight, bias, activation, checkpoint)
                           : call_linear(x, weight, bias, residual, activation, checkpoint);
    const bool slope = gated || activation != "none";
    const bool want_x = x.requires_grad(), want_w = weight.requires_grad();
    const bool want_b = has(bias) && bias->requires_grad();
    ctx->saved_data["activation"] = activation;
    ctx->saved_data["gated"] = gated;
    ctx->saved_data["wanted"] = (want_x ? 1 : 0) | (want_w ? 2 : 0) | (want_b ? 4 : 0);
    ctx->saved_data["residual"] = has(residual) && residual->requires_grad();
    ctx->saved_data["sizes"] = x.sizes().vec();
    if (!want_x && !want_w && !want_b) return y;
    Tensor kept, scales;
    if (want_w || slope) {
      if (checkpoint == "e4m3") {
        std::tie(kept, scales) = call_quantize(x);
      } else {
        kept = x;
      }
    }
    ctx->save_for_backward({kept, scales, weight, has(bias) ? *bias : Tensor()});
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(),
                "vectra::linear: gradients of gradients are not supported (create_graph=True)");
    torch::autograd::variable_list out(7);
    const Tensor& grad = grads[0];
    if (!grad.defined()) return out;
    if (ctx->saved_data["residual"].toBool()) out[3] = grad;  // the residual's
    const int64_t wanted = ctx->saved_data["wanted"].toInt();
    if (wanted == 0) return out;
    const auto saved = ctx->get_saved_variables();
    const OptTensor scales = saved[1].defined() ? OptTensor(saved[1]) : std::nullopt;
    const OptTensor bias = saved[3].defined() ? OptTensor(saved[3]) : std::nullopt;
    Tensor kept = saved[0];
    if (!kept.defined()) {  // neither a slope nor the weight's gradient: the input's values are not read
      kept = at::empty({1}, saved[2].options()).expand(ctx->saved_data["sizes"].toIntVector());
    }
    const auto g = call_backward(grad, kept, scales, saved[2], bias, ctx->saved_data["activation"].toStringRef(),
                                 ctx->saved_data["gated"].toBool(),
                                 {(wanted & 1) != 0, (wanted & 2) != 0, (wanted & 4) != 0});
    size_t at = 0;
    for (int i = 0; i < 3; ++i)
      if (wanted >> i & 1) out[i] = g[at++];
    return out;
  }
};

// The layers have no forward-mode derivative: below autograd a tangent would be
// dropped without a word.
void refuse_tangents(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                     const char* op) {
  const auto dual = [](const Tensor& t) { return t._fw_grad(/*level=*/0).defined(); };
  TORCH_CHECK_NOT_IMPLEMENTED(!dual(x) && !dual(weight) && !(has(bias) && dual(*bias)) &&
                                  !(has(residual) && dual(*residual)),
                              op, ": forward-mode derivatives are not supported (an argument carries a tangent)");
}

bool any_requires_grad(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual) {
  return at::GradMode::is_enabled() && (x.requires_grad() || weight.requires_grad() ||
                                        (has(bias) && bias->requires_grad()) ||
                                        (has(residual) && residual->requires_grad()));
}

Tensor linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                       c10::string_view activation, c10::string_view checkpoint) {
  refuse_tangents(x, weight, bias, residual, "vectra::linear");
  if (!any_requires_grad(x, weight, bias, residual)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_linear(x, weight, bias, residual, activation, checkpoint);
  }
  return Layer::apply(x, weight, bias, residual, std::string(activation), std::string(checkpoint), false);
}

Tensor gated_linear_autograd(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation,
                             c10::string_view checkpoint) {
  refuse_tangents(x, weight, bias, std::nullopt, "vectra::gated_linear");
  if (!any_requires_grad(x, weight, bias, std::nullopt)) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_gated(x, weight, bias, activation, checkpoint);
  }
  return Layer::apply(x, weight, bias, std::nullopt, std::string(activation), std::string(checkpoint), true);
}

// ---------------------------------------------------------------- autocast
//
// x and weight in autocast's type.  A bias of fp32 stays as it is: it joins the
// product's fp32 sums.  So does a residual of another type, the fp32 stream that
// blocks under autocast add their 16-bit branches to: it is added to the layer's
// output by torch's own rules, and the result has the wider type.

Tensor cast_to(at::ScalarType type, const Tensor& t, c10::DeviceType device) {
  return at::autocast::cached_cast(type, t, device);
}

OptTensor cast_bias(at::ScalarType type, const OptTensor& bias, c10::DeviceType device) {
  return has(bias) && bias->scalar_type() != at::kFloat ? OptTensor(cast_to(type, *bias, device)) : bias;
}

template <c10::DeviceType kDevice, c10::DispatchKey kKey>
Tensor linear_autocast(const Tensor& x, const Tensor& weight, const OptTensor& bias, const OptTensor& residual,
                       c10::string_view activation, c10::string_view checkpoint) {
  c10::impl::ExcludeDispatchKeyGuard no_autocast(kKey);
  const at::ScalarType type = at::autocast::get_autocast_dtype(kDevice);
  const Tensor xc = cast_to(type, x, kDevice), wc = cast_to(type, weight, kDevice);
  const OptTensor bc = cast_bias(type, bias, kDevice);
  if (!has(residual) || residual->scalar_type() == xc.scalar_type())
    return call_linear(xc, wc, bc, residual, activation, checkpoint);
  const Tensor y = call_linear(xc, wc, bc, std::nullopt, activation, checkpoint);
  check_residual_shape(x, weight, *residual, "vectra::linear");
  return at::add(*residual, y);
}

template <c10::DeviceType kDevice, c10::DispatchKey kKey>
Tensor gated_linear_autocast(const Tensor& x, const Tensor& weight, const OptTensor& bias, c10::string_view activation,
                             c10::string_view checkpoint) {
  c10::impl::ExcludeDispatchKeyGuard no_autocast(kKey);
  const at::ScalarType type = at::autocast::get_autocast_dtype(kDevice);
  return call_gated(cast_to(type, x, kDevice), cast_to(type, weight, kDevice), cast_bias(type, bias, kDevice), activation,
                    checkpoint);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(vectra, m) {
  m.def(
      "linear(Tensor x, Tensor weight, Tensor? bias=None, Tensor? residual=None, str activation='none', "
      "str checkpoint='none') -> Tensor");
  m.def(
      "gated_linear(Tensor x, Tensor weight, Tensor? bias=None, str activation='silu', str checkpoint='none') "
      "-> Tensor");
  m.def(
      "linear_backward(Tensor grad, Tensor x, Tensor? scales, Tensor weight, Tensor? bias, str activation, bool gated, "
      "bool[3] wanted) -> Tensor[]");
  m.def("quantize_rows(Tensor x) -> (Tensor, Tensor)");
  m.def("dequantize_rows(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
}

TORCH_LIBRARY_IMPL(vectra, CUDA, m) {
  m.impl("linear", linear_hip);
  m.impl("gated_linear", gated_linear_hip);
  m.impl("linear_backward", linear_backward_hip);
  m.impl("quantize_rows", quantize_rows_hip);
  m.impl("dequantize_rows", dequantize_rows_hip);
}

TORCH_LIBRARY_IMPL(vectra, CPU, m) {
  m.impl("linear", linear_cpu);
  m.impl("gated_linear", gated_linear_cpu);
  m.impl("linear_backward", linear_backward_cpu);
  m.impl("quantize_rows", quantize_rows_cpu);
  m.impl("dequantize_rows", dequantize_rows_cpu);
}

TORCH_LIBRARY_IMPL(vectra, Autograd, m) {
  m.impl("linear", linear_autograd);
  m.impl("gated_linear", gated_linear_autograd);
  // No derivatives: a backward pass that reaches one of these raises, and so
  // does a tangent.
  m.impl("linear_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("quantize_rows", torch::autograd::autogradNotImplementedFallback());
  m.impl("dequantize_rows", torch::autograd::autogradNotImplementedFallback());
}

// (Autocast is the key of GPU tensors.)
TORCH_LIBRARY_IMPL(vectra, Autocast, m) {
  m.impl("linear", TORCH_FN((linear_autocast<at::kCUDA, c10::DispatchKey::Autocast>)));
  m.impl("gated_linear", TORCH_FN((gated_linear_autocast<at::kCUDA, c10::DispatchKey::Autocast>)));
}

TORCH_LIBRARY_IMPL(vectra, AutocastCPU, m) {
  m.impl("linear", TORCH_FN((linear_autocast<at::kCPU, c10::DispatchKey::AutocastCPU>)));
  m.impl("gated_linear", TORCH_FN((gated_linear_autocast<at::kCPU, c10::DispatchKey::AutocastCPU>)));
}
