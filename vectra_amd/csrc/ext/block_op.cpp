// torch.library registration of the operators between a block's dense products:
//   dropout                 kept elements scaled, the others zero, by a counter-based generator
//   dropout_pass            what one pass of a program draws from, counted on
//   residual_norm           a branch onto the residual stream, and the stream's norm
//   residual_norm_8bit      the same with the norm in 8-bit rows
//   residual_norm_backward  residual_norm's gradients
//   quantize_blocks         a matrix in 8 bits: rows of 128, or tiles of 128 x 128, that
//                           share a power of two
//   linear_8bit             act(x^ W^T + b) + residual on such codes
//   gated_linear_8bit       act(x^ G^T + b_g) * (x^ U^T + b_u)
//
//   CUDA key (HIP tensors on ROCm)  -> libvectra_block.so (include/vectra_block.h),
//                                      on the caller's current HIP stream, with
//                                      scratch memory from torch's allocator
//   CPU key                         -> the same formulas in fp32 tensors
//   Autograd key                    -> dropout: itself on the gradient; residual_norm:
//                                      calls residual_norm_backward; the others: no
//                                      derivative, refused
//   fake/meta                       -> registered from Python
// There is no CPU fallback for device tensors: if the HIP library cannot be
// loaded this extension does not load either.

#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/library.h>

#include <array>
#include <cmath>
#include <cstring>
#include <tuple>

#include "op_common.h"
#include "vectra_block.h"

namespace {

using namespace vectra_ops;

void check_status(int status, const char* op) {
  TORCH_CHECK(status == VECTRA_BLOCK_OK, op, ": ", vectra_block_status_string(status));
}

vectra_block_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<vectra_block_stream_t>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

bool is_float(at::ScalarType t) { return dense_dtype(t) >= 0; }

// ----------------------------------------------------------------- dropout

// The probability as 65536ths, after checks of what the generator reads.
int32_t check_dropout(const Tensor& x, double p, const OptTensor& rng, int64_t stream, const char* op) {
  const double threshold = std::nearbyint(65536.0 * p);
  TORCH_CHECK_VALUE(p >= 0.0 && p < 1.0 && threshold < 65536.0, op, ": p must be at least 0 and at most 1 - 2^-16; got ", p);
  TORCH_CHECK_VALUE(stream >= 0 && stream < (int64_t{1} << 32), op, ": stream must be at least 0 and less than 2^32; got ",
                    stream);
  TORCH_CHECK(p == 0.0 || has(rng), op, ": dropout needs rng, the seed and the offset");
  if (has(rng)) {
    TORCH_CHECK(rng->scalar_type() == at::kLong && rng->dim() == 1 && rng->size(0) == 2, op,
                ": rng must be two int64, the seed and the offset; got ", rng->scalar_type(), " ", rng->sizes());
    TORCH_CHECK(rng->device() == x.device(), op, ": rng must be on ", x.device(), "; got ", rng->device());
  }
  return static_cast<int32_t>(threshold);
}

void check_dropped(const Tensor& x) {
  TORCH_CHECK(is_float(x.scalar_type()), "vectra::dropout: x must be float32, float16 or bfloat16; got ", x.scalar_type());
}

Tensor dropout_hip(const Tensor& x_in, double p, const Tensor& rng_in, int64_t stream) {
  constexpr const char* op = "vectra::dropout";
  check_dropped(x_in);
  const int32_t threshold = check_dropout(x_in, p, rng_in, stream, op);
  c10::DeviceGuard guard(x_in.device());
  const Tensor x = x_in.dim() ? x_in : x_in.reshape({1});
  Tensor y = at::empty(x_in.sizes(), x_in.options());
  const Rows xr = as_rows(x);
  const Tensor rng = rng_in.contiguous();
  check_status(vectra_dropout(xr.t.data_ptr(), dense_dtype(x.scalar_type()), rows_of(x), x.size(-1), xr.stride,
                              y.data_ptr(), std::max<int64_t>(x.size(-1), 1), threshold, rng.const_data_ptr<int64_t>(),
                              static_cast<uint32_t>(stream), stream_of(x)),
               op);
  return y;
}

// The elements' factors, 0 or 65536 / (65536 - t), as fp32 [rows, width].
Tensor factors_cpu(int64_t rows, int64_t width, int32_t threshold, const Tensor& rng_in, int64_t stream) {
  Tensor out = at::empty({rows, width}, at::TensorOptions().dtype(at::kFloat));
  float* const f = out.mutable_data_ptr<float>();
  const Tensor rng = rng_in.contiguous();
  const uint64_t seed = static_cast<uint64_t>(rng.const_data_ptr<int64_t>()[0]);
  const uint32_t offset = static_cast<uint32_t>(rng.const_data_ptr<int64_t>()[1]);
  const float scale = static_cast<float>(65536.0 / (65536 - threshold));
  const int64_t groups = (width + 7) / 8;
  for (int64_t r = 0; r < rows; ++r) {
    for (int64_t g = 0; g < groups; ++g) {
      const uint64_t at = static_cast<uint64_t>(r * groups + g);
      uint32_t c[4] = {static_cast<uint32_t>(at), static_cast<uint32_t>(at >> 32), static_cast<uint32_t>(stream), offset};
      uint32_t k0 = static_cast<uint32_t>(seed), k1 = static_cast<uint32_t>(seed >> 32);
      for (int round = 0; round < 10; ++round) {
        const uint64_t p = uint64_t{0xD2511F53u} * c[0], q = uint64_t{0xCD9E8D57u} * c[2];
        const uint32_t next[4] = {static_cast<uint32_t>(q >> 32) ^ c[1] ^ k0, static_cast<uint32_t>(q),
                                  static_cast<uint32_t>(p >> 32) ^ c[3] ^ k1, static_cast<uint32_t>(p)};
        std::memcpy(c, next, sizeof(c));
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
      }
      for (int64_t e = 0; e < std::min<int64_t>(8, width - g * 8); ++e) {
        const uint32_t bits = e % 2 ? c[e / 2] >> 16 : c[e / 2] & 0xffffu;
        f[r * width + g * 8 + e] = bits >= static_cast<uint32_t>(threshold) ? scale : 0.f;
      }
    }
  }
  return out;
}

// The generator's state as it is, and counted on in place.  One operator, because of
// compilers: of a clone and an addition in place they see through the first and
// leave the backward pass the tensor that the second has changed.
// A forward pass within a backward one is one run again (activation checkpointing):
// it has to draw what it drew before, which the state no longer tells.
Tensor dropout_pass(Tensor& state) {
  TORCH_CHECK(torch::autograd::get_current_graph_task_id() == -1,
              "vectra::dropout_pass: called within a backward pass. A forward pass that is run again there, as activation "
              "checkpointing does, has to drop the same elements: take its draws before the checkpointed function and pass "
              "them to it as an argument");
  TORCH_CHECK(state.scalar_type() == at::kLong && state.dim() == 1 && state.size(0) == 2,
              "vectra::dropout_pass: state must be two int64, the seed and the offset; got ", state.scalar_type(), " ",
              state.sizes());
  c10::DeviceGuard guard(state.device());
  Tensor rng = state.clone(at::MemoryFormat::Contiguous);
  state.select(0, 1).add_(1);
  return rng;
}

// x * factors, 0 where dropped whatever x holds.
Tensor drop_cpu(const Tensor& x, const Tensor& factors) {
  return at::where(factors.eq(0), at::zeros_like(x), x * factors);
}

Tensor dropout_cpu(const Tensor& x_in, double p, const Tensor& rng, int64_t stream) {
  constexpr const char* op = "vectra::dropout";
  check_dropped(x_in);
  const int32_t threshold = check_dropout(x_in, p, rng, stream, op);
  const Tensor x = x_in.dim() ? x_in : x_in.reshape({1});
  const int64_t rows = rows_of(x), width = x.size(-1);
  const Tensor flat = x.reshape({rows, width}).to(at::kFloat);
  return drop_cpu(flat, factors_cpu(rows, width, threshold, rng, stream)).to(x.scalar_type()).reshape(x_in.sizes()).contiguous();
}

// -------------------------------------------------------------------- norms

int32_t norm_of(std::string_view name, bool none, const char* what, const char* op) {
  if (name == "rms") return VECTRA_BLOCK_RMS;
  if (name == "layer") return VECTRA_BLOCK_LAYER;
  if (none && name == "none") return VECTRA_BLOCK_NO_NORM;
  TORCH_CHECK_VALUE(false, op, ": ", what, " must be ", none ? "'none', " : "", "'rms' or 'layer'; got '",
                    std::string(name), "'");
}

// A per-column vector of x's type or fp32.
void check_vector(const OptTensor& v, int64_t width, at::ScalarType dtype, const at::Device& device, const char* what,
                  const char* op) {
  if (!has(v)) return;
  TORCH_CHECK(v->dim() == 1 && v->size(0) == width, op, ": ", what, " must be [", width, "]; got ", v->sizes());
  TORCH_CHECK(v->scalar_type() == dtype || v->scalar_type() == at::kFloat, op, ": ", what,
              " must have x's dtype or float32; got ", v->scalar_type());
  TORCH_CHECK(v->device() == device, op, ": ", what, " must be on ", device, "; got ", v->device());
}

// How many consecutive rows of x share a row of the gate: its shape is [width], or
// x's own with the dimensions from some one on, but for the last, of size 1.
int64_t gate_rows_of(const OptTensor& gate, at::IntArrayRef sizes, const char* op) {
  int64_t rows = 1;
  for (size_t d = 0; d + 1 < sizes.size(); ++d) rows *= sizes[d];
  if (!has(gate) || gate->dim() == 1) return std::max<int64_t>(rows, 1);
  bool same = gate->dim() == static_cast<int64_t>(sizes.size()), ones = false;
  int64_t gates = 1;
  for (size_t d = 0; same && d + 1 < sizes.size(); ++d) {
    const int64_t size = gate->size(static_cast<int64_t>(d));
    if (ones || size != sizes[d]) ones = same = size == 1;
    gates *= size;
  }
  TORCH_CHECK(same, op, ": gate must be [width], or of x's shape with size 1 from some dimension on; got ", gate->sizes(),
              " for ", sizes);
  return gates ? std::max<int64_t>(rows / gates, 1) : 1;
}

// What the forward and the backward call share.
struct NormOptions {
  int32_t norm, post, threshold;
  uint32_t stream;
  float eps, residual_scale;
  int64_t gate_rows;
};

NormOptions check_norm(at::IntArrayRef sizes, at::ScalarType dtype, const Tensor& some, const OptTensor& weight,
                       const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                       const OptTensor& post_bias, std::string_view norm, std::string_view post, double eps,
                       double residual_scale, double p, const OptTensor& rng, int64_t stream, const char* op) {
  NormOptions o{};
  o.norm = norm_of(norm, false, "norm", op);
  o.post = norm_of(post, true, "post", op);
  const int64_t width = sizes.back();
  check_vector(weight, width, dtype, some.device(), "weight", op);
  check_vector(bias, width, dtype, some.device(), "bias", op);
  check_vector(post_weight, width, dtype, some.device(), "post_weight", op);
  check_vector(post_bias, width, dtype, some.device(), "post_bias", op);
  TORCH_CHECK(o.post != VECTRA_BLOCK_NO_NORM || (!has(post_weight) && !has(post_bias)), op,
              ": post_weight and post_bias need a post norm");
  if (has(gate)) {
    TORCH_CHECK(gate->dim() >= 1 && gate->size(-1) == width, op, ": gate's last dimension must be ", width, "; got ",
                gate->sizes());
    TORCH_CHECK(gate->scalar_type() == dtype || gate->scalar_type() == at::kFloat, op,
                ": gate must have x's dtype or float32; got ", gate->scalar_type());
    TORCH_CHECK(gate->device() == some.device(), op, ": gate must be on ", some.device(), "; got ", gate->device());
  }
  o.gate_rows = gate_rows_of(gate, sizes, op);
  TORCH_CHECK_VALUE(eps >= 0.0 && std::isfinite(static_cast<float>(eps)), op, ": eps must be at least 0 and finite; got ", eps);
  o.eps = static_cast<float>(eps);
  o.residual_scale = static_cast<float>(residual_scale);
  o.threshold = check_dropout(some, p, rng, stream, op);
  o.stream = static_cast<uint32_t>(stream);
  return o;
}

void check_branch(const Tensor& x, const Tensor& residual, const char* op) {
  TORCH_CHECK(x.dim() >= 1 && x.sizes() == residual.sizes(), op, ": x and residual must be [..., width], of one shape; got ",
              x.sizes(), " and ", residual.sizes());
  TORCH_CHECK(is_float(x.scalar_type()), op, ": x must be float32, float16 or bfloat16; got ", x.scalar_type());
  TORCH_CHECK(residual.scalar_type() == x.scalar_type() || residual.scalar_type() == at::kFloat, op,
              ": residual must have x's dtype or float32; got ", residual.scalar_type());
  TORCH_CHECK(residual.device() == x.device(), op, ": residual must be on ", x.device(), "; got ", residual.device());
}

// A gate as the rows the C ABI reads.
Rows gate_rows(const Tensor& gate) { return as_rows(gate.dim() == 1 ? gate.unsqueeze(0) : gate); }

int32_t dtype_of(const OptTensor& t) { return has(t) ? dense_dtype(t->scalar_type()) : 0; }

// Contiguous vectors, kept alive for the call, as pointers.
struct Vectors {
  std::array<Tensor, 5> kept;
  const void* add(size_t i, const OptTensor& t) {
    if (!has(t)) return nullptr;
    kept[i] = t->contiguous();
    return kept[i].data_ptr();
  }
};

// n: an output tensor, or undefined with codes and scales.
void norm_forward_hip(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& bias,
                      const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                      const NormOptions& o, const OptTensor& rng_in, Tensor& h, Tensor& n, Tensor& codes, Tensor& scales,
                      const char* op) {
  const int64_t width = x.size(-1);
  const Rows xr = as_rows(x), rr = as_rows(residual);
  Rows gr;
  if (has(gate)) gr = gate_rows(*gate);
  Tensor rng;
  if (o.threshold) rng = rng_in->contiguous();
  Vectors v;
  vectra_norm_args a{};
  a.struct_size = sizeof(a);
  a.x = xr.t.data_ptr();
  a.residual = rr.t.data_ptr();
  a.weight = v.add(0, weight);
  a.bias = v.add(1, bias);
  a.gate = gr.t.defined() ? gr.t.data_ptr() : nullptr;
  a.post_weight = v.add(2, post_weight);
  a.post_bias = v.add(3, post_bias);
  a.rng = rng.defined() ? rng.const_data_ptr<int64_t>() : nullptr;
  a.h = h.data_ptr();
  a.n = n.defined() ? n.data_ptr() : nullptr;
  a.codes = codes.defined() ? codes.data_ptr() : nullptr;
  a.scales = scales.defined() ? scales.data_ptr() : nullptr;
  a.dtype = dense_dtype(x.scalar_type());
  a.stream_dtype = dense_dtype(residual.scalar_type());
  a.weight_dtype = dtype_of(weight);
  a.bias_dtype = dtype_of(bias);
  a.gate_dtype = dtype_of(gate);
  a.post_weight_dtype = dtype_of(post_weight);
  a.post_bias_dtype = dtype_of(post_bias);
  a.norm = o.norm;
  a.post = o.post;
  a.threshold = o.threshold;
  a.stream_id = o.stream;
  a.eps = o.eps;
  a.residual_scale = o.residual_scale;
  a.rows = rows_of(x);
  a.width = width;
  a.gate_rows = o.gate_rows;
  a.x_stride = xr.stride;
  a.residual_stride = rr.stride;
  a.gate_stride = gr.stride;
  a.h_stride = a.n_stride = std::max<int64_t>(width, 1);
  check_status(vectra_norm_forward(&a, stream_of(x)), op);
}

std::tuple<Tensor, Tensor> residual_norm_hip(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                             const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                                             const OptTensor& post_bias, c10::string_view norm, c10::string_view post,
                                             double eps, double residual_scale, double p, const OptTensor& rng,
                                             int64_t stream) {
  constexpr const char* op = "vectra::residual_norm";
  check_branch(x, residual, op);
  const NormOptions o = check_norm(x.sizes(), x.scalar_type(), x, weight, bias, gate, post_weight, post_bias, norm, post,
                                   eps, residual_scale, p, rng, stream, op);
  c10::DeviceGuard guard(x.device());
  Tensor h = at::empty(x.sizes(), residual.options()), n = at::empty(x.sizes(), x.options()), none;
  norm_forward_hip(x, residual, weight, bias, gate, post_weight, post_bias, o, rng, h, n, none, none, op);
  return {h, n};
}

std::vector<int64_t> codes_sizes(const Tensor& x) { return with_last(x, (x.size(-1) + 127) / 128 * 128); }
std::vector<int64_t> scales_sizes(const Tensor& x) { return with_last(x, (x.size(-1) + 511) / 512 * 4); }

std::tuple<Tensor, Tensor, Tensor> residual_norm_8bit_hip(const Tensor& x, const Tensor& residual,
                                                          const OptTensor& weight, const OptTensor& bias,
                                                          const OptTensor& gate, const OptTensor& post_weight,
                                                          const OptTensor& post_bias, c10::string_view norm,
                                                          c10::string_view post, double eps, double residual_scale,
                                                          double p, const OptTensor& rng, int64_t stream) {
  constexpr const char* op = "vectra::residual_norm_8bit";
  check_branch(x, residual, op);
  const NormOptions o = check_norm(x.sizes(), x.scalar_type(), x, weight, bias, gate, post_weight, post_bias, norm, post,
                                   eps, residual_scale, p, rng, stream, op);
  c10::DeviceGuard guard(x.device());
  Tensor h = at::empty(x.sizes(), residual.options()), none;
  Tensor codes = at::empty(codes_sizes(x), x.options().dtype(at::kFloat8_e4m3fn));
  Tensor scales = at::empty(scales_sizes(x), x.options().dtype(at::kFloat8_e8m0fnu));
  norm_forward_hip(x, residual, weight, bias, gate, post_weight, post_bias, o, rng, h, none, codes, scales, op);
  return {h, codes, scales};
}

// Whether the gradients read x and the residual, or h (of a stream of this type).
bool reads_branch(at::ScalarType stream_dtype, const OptTensor& gate, std::string_view post) {
  return has(gate) || post != "none" || stream_dtype != at::kFloat;
}
bool reads_branch(const OptTensor& h, const OptTensor& residual, const OptTensor& gate, std::string_view post) {
  return reads_branch(has(residual) ? residual->scalar_type() : has(h) ? h->scalar_type() : at::kFloat, gate, post);
}

// The gradients' operands.
NormOptions check_norm_backward(const OptTensor& grad_h, const OptTensor& grad_n, const OptTensor& h, const OptTensor& x,
                                const OptTensor& residual, const OptTensor& weight, const OptTensor& bias,
                                const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                                std::string_view norm, std::string_view post, double eps, double residual_scale, double p,
                                const OptTensor& rng, int64_t stream, at::ScalarType dtype, at::ArrayRef<bool> wanted) {
  constexpr const char* op = "vectra::residual_norm_backward";
  TORCH_CHECK(wanted.size() == 7, op, ": wanted must name seven gradients (x, residual, weight, bias, gate, post_weight, post_bias)");
  const bool branch = reads_branch(h, residual, gate, post);
  TORCH_CHECK(branch ? has(x) && has(residual) : has(h), op, ": needs ",
              branch ? "x and residual with a gate, a post norm or a stream of 16 bits" : "h, the forward pass's result");
  const Tensor& stream_side = branch ? *residual : *h;
  TORCH_CHECK(is_float(dtype), op, ": dtype, x's, must be float32, float16 or bfloat16; got ", dtype);
  TORCH_CHECK(stream_side.dim() >= 1, op, ": h or residual must be [..., width]; got a scalar");
  if (branch) {
    check_branch(*x, *residual, op);
    TORCH_CHECK(x->scalar_type() == dtype, op, ": x must have dtype ", dtype, "; got ", x->scalar_type());
  }
  const at::ScalarType stream_dtype = stream_side.scalar_type();
  TORCH_CHECK(stream_dtype == dtype || stream_dtype == at::kFloat, op, ": the residual stream must have x's dtype or float32; got ",
              stream_dtype);
  const auto check_grad = [&](const OptTensor& g, at::ScalarType want, const char* what) {
    if (!has(g)) return;
    TORCH_CHECK(g->sizes() == stream_side.sizes(), op, ": ", what, " must be ", stream_side.sizes(), "; got ", g->sizes());
    TORCH_CHECK(g->scalar_type() == want && g->device() == stream_side.device(), op, ": ", what, " must be ", want, " on ",
                stream_side.device(), "; got ", g->scalar_type(), " on ", g->device());
  };
  check_grad(grad_h, stream_dtype, "grad_h");
  check_grad(grad_n, dtype, "grad_n");
  const bool missing = (wanted[4] && !has(gate)) || ((wanted[5] || wanted[6]) && post == "none") ||
                       (wanted[2] && !has(weight)) || (wanted[3] && !has(bias)) || (wanted[5] && !has(post_weight)) ||
                       (wanted[6] && !has(post_bias));
  TORCH_CHECK(!missing, op, ": wanted names the gradient of an argument that is not given");
  return check_norm(stream_side.sizes(), dtype, stream_side, weight, bias, gate, post_weight, post_bias, norm, post, eps,
                    residual_scale, p, rng, stream, op);
}

std::vector<Tensor> residual_norm_backward_hip(const OptTensor& grad_h, const OptTensor& grad_n, const OptTensor& h,
                                               const OptTensor& x, const OptTensor& residual, const OptTensor& weight,
                                               const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                                               const OptTensor& post_bias, c10::string_view norm, c10::string_view post,
                                               double eps, double residual_scale, double p, const OptTensor& rng_in,
                                               int64_t stream, at::ScalarType dtype, std::array<bool, 7> wanted) {
  constexpr const char* op = "vectra::residual_norm_backward";
  const NormOptions o = check_norm_backward(grad_h, grad_n, h, x, residual, weight, bias, gate, post_weight, post_bias, norm,
                                            post, eps, residual_scale, p, rng_in, stream, dtype, wanted);
  const bool branch = reads_branch(h, residual, gate, post);
  const Tensor& side = branch ? *residual : *h;
  c10::DeviceGuard guard(side.device());
  const int64_t width = side.size(-1), rows = rows_of(side);
  Rows gh, gn, hr, xr, rr, gr;
  if (has(grad_h)) gh = as_rows(*grad_h);
  if (has(grad_n)) gn = as_rows(*grad_n);
  if (branch) {
    xr = as_rows(*x);
    rr = as_rows(*residual);
  } else {
    hr = as_rows(*h);
  }
  if (has(gate)) gr = gate_rows(*gate);
  Tensor rng;
  if (o.threshold) rng = rng_in->contiguous();
  Vectors v;
  const auto at_or_null = [](const Rows& r) -> const void* { return r.t.defined() ? r.t.data_ptr() : nullptr; };
  vectra_norm_grad_args a{};
  a.struct_size = sizeof(a);
  a.grad_h = at_or_null(gh);
  a.grad_n = at_or_null(gn);
  a.x = at_or_null(xr);
  a.residual = at_or_null(rr);
  a.h = at_or_null(hr);
  a.weight = v.add(0, weight);
  a.gate = at_or_null(gr);
  a.post_weight = v.add(1, post_weight);
  a.post_bias = v.add(2, post_bias);
  a.rng = rng.defined() ? rng.const_data_ptr<int64_t>() : nullptr;
  std::vector<Tensor> out;
  const auto make = [&](int i, at::IntArrayRef sizes, const at::TensorOptions& options) -> void* {
    if (!wanted[i]) return nullptr;
    out.push_back(rows ? at::empty(sizes, options) : at::zeros(sizes, options));
    return out.back().data_ptr();
  };
  a.dx = make(0, side.sizes(), side.options().dtype(dtype));
  a.dresidual = make(1, side.sizes(), side.options());
  if (wanted[2]) a.dweight = make(2, weight->sizes(), weight->options());
  if (wanted[3]) a.dbias = make(3, bias->sizes(), bias->options());
  if (wanted[4]) a.dgate = make(4, gate->sizes(), gate->options());
  if (wanted[5]) a.dpost_weight = make(5, post_weight->sizes(), post_weight->options());
  if (wanted[6]) a.dpost_bias = make(6, post_bias->sizes(), post_bias->options());
  if (rows == 0) return out;  // zeros
  a.dtype = dense_dtype(dtype);
  a.stream_dtype = dense_dtype(side.scalar_type());
  a.weight_dtype = dtype_of(weight);
  a.bias_dtype = dtype_of(bias);
  a.gate_dtype = dtype_of(gate);
  a.post_weight_dtype = dtype_of(post_weight);
  a.post_bias_dtype = dtype_of(post_bias);
  a.norm = o.norm;
  a.post = o.post;
  a.threshold = o.threshold;
  a.stream_id = o.stream;
  a.eps = o.eps;
  a.residual_scale = o.residual_scale;
  a.rows = rows;
  a.width = width;
  a.gate_rows = o.gate_rows;
  a.grad_h_stride = gh.stride;
  a.grad_n_stride = gn.stride;
  a.x_stride = xr.stride;
  a.residual_stride = rr.stride;
  a.h_stride = hr.stride;
  a.gate_stride = gr.stride;
  a.dx_stride = a.dresidual_stride = a.dgate_stride = std::max<int64_t>(width, 1);
  const int64_t need = vectra_norm_backward_workspace_bytes(&a);
  if (need < 0) check_status(static_cast<int>(-need), op);
  Tensor workspace;
  if (need > 0) workspace = at::empty({need}, side.options().dtype(at::kByte));
  check_status(vectra_norm_backward(&a, need > 0 ? workspace.data_ptr() : nullptr, need, stream_of(side)), op);
  return out;
}

// ------------------------------------------------------------------- host
//
// The operators off the GPU: the same formulas on fp32 tensors.

Tensor wide(const Tensor& t) { return t.to(at::kFloat); }

// (x - mean) / deviation and 1 / deviation.
std::pair<Tensor, Tensor> normalised_cpu(const Tensor& x, int32_t kind, float eps) {
  const Tensor c = kind == VECTRA_BLOCK_LAYER ? x - x.mean(-1, true) : x;
  const Tensor r = at::rsqrt((c * c).mean(-1, true) + eps);
  return {c * r, r};
}

Tensor affine_cpu(Tensor x, const OptTensor& weight, const OptTensor& bias) {
  if (has(weight)) x = x * wide(*weight);
  if (has(bias)) x = x + wide(*bias);
  return x;
}

Tensor transpose_cpu(const Tensor& g, const Tensor& hat, const Tensor& r, int32_t kind) {
  Tensor d = g - hat * (g * hat).mean(-1, true);
  if (kind == VECTRA_BLOCK_LAYER) d = d - g.mean(-1, true);
  return d * r;
}

// The branch before its gate, and what its gradient needs.
struct BranchCpu {
  Tensor v, hat, r, factors, gate;
};

BranchCpu branch_cpu(const Tensor& x, const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                     const NormOptions& o, const OptTensor& rng) {
  const int64_t width = x.size(-1), rows = rows_of(x);
  BranchCpu b;
  b.v = wide(x).reshape({rows, width});
  if (o.post != VECTRA_BLOCK_NO_NORM) {
    std::tie(b.hat, b.r) = normalised_cpu(b.v, o.post, o.eps);
    b.v = affine_cpu(b.hat, post_weight, post_bias);
  }
  if (o.threshold) {
    b.factors = factors_cpu(rows, width, o.threshold, *rng, o.stream);
    b.v = drop_cpu(b.v, b.factors);
  }
  if (has(gate)) b.gate = wide(*gate).expand(x.sizes()).reshape({rows, width});
  return b;
}

// h and n, unrounded, as [rows, width].
std::pair<Tensor, Tensor> norm_forward_cpu(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                           const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                                           const OptTensor& post_bias, const NormOptions& o, const OptTensor& rng) {
  const BranchCpu b = branch_cpu(x, gate, post_weight, post_bias, o, rng);
  const Tensor h = wide(residual).reshape(b.v.sizes()) * o.residual_scale + (b.gate.defined() ? b.v * b.gate : b.v);
  return {h, affine_cpu(normalised_cpu(h, o.norm, o.eps).first, weight, bias)};
}

std::tuple<Tensor, Tensor> residual_norm_cpu(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                             const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                                             const OptTensor& post_bias, c10::string_view norm, c10::string_view post,
                                             double eps, double residual_scale, double p, const OptTensor& rng,
                                             int64_t stream) {
  constexpr const char* op = "vectra::residual_norm";
  check_branch(x, residual, op);
  const NormOptions o = check_norm(x.sizes(), x.scalar_type(), x, weight, bias, gate, post_weight, post_bias, norm, post,
                                   eps, residual_scale, p, rng, stream, op);
  const auto [h, n] = norm_forward_cpu(x, residual, weight, bias, gate, post_weight, post_bias, o, rng);
  return {h.reshape(x.sizes()).to(residual.scalar_type()).clone(at::MemoryFormat::Contiguous),
          n.reshape(x.sizes()).to(x.scalar_type()).clone(at::MemoryFormat::Contiguous)};
}

// Codes and scales of fp32 [rows, width]; blocks of `high` rows of 128.
std::tuple<Tensor, Tensor> quantize_cpu(const Tensor& x_in, int64_t high) {
  const Tensor x = x_in.contiguous();
  const int64_t rows = x.size(0), width = x.size(1), depth = (width + 127) / 128 * 128, across = (width + 511) / 512 * 4;
  Tensor values = at::zeros({rows, depth}, x.options());
  Tensor scales = at::zeros({(rows + high - 1) / high, across}, x.options().dtype(at::kByte));
  const float* const from = x.const_data_ptr<float>();
  float* const to = values.mutable_data_ptr<float>();
  uint8_t* const s = scales.mutable_data_ptr<uint8_t>();
  for (int64_t r0 = 0; r0 < rows; r0 += high) {
    for (int64_t c0 = 0; c0 < width; c0 += 128) {
      const int64_t r1 = std::min(r0 + high, rows), c1 = std::min<int64_t>(c0 + 128, width);
      float largest = 0.f;
      for (int64_t r = r0; r < r1; ++r)
        for (int64_t c = c0; c < c1; ++c)
          if (std::isfinite(from[r * width + c])) largest = std::max(largest, std::fabs(from[r * width + c]));
      int e = -117;
      if (largest > 0.f) {
        int x2 = 0;
        const float m = std::frexp(largest, &x2);  // largest = m 2^x2, m in [1/2, 1); 448 = 0.875 * 2^9
        e = std::max(e, x2 - 9 + (m > 0.875f ? 1 : 0));
      }
      for (int64_t r = r0; r < r1; ++r)
        for (int64_t c = c0; c < c1; ++c) {
          const float v = from[r * width + c];
          float y = std::isfinite(v) ? std::ldexp(v, -e) : std::nanf("");
          if (e == 120 && std::fabs(y) >= 248.f) y = std::copysign(240.f, y);
          to[r * depth + c] = y;
        }
      s[r0 / high * across + c0 / 128] = static_cast<uint8_t>(e + 127);
    }
  }
  return {values.to(at::kFloat8_e4m3fn), scales.view(at::kFloat8_e8m0fnu)};
}

std::tuple<Tensor, Tensor, Tensor> residual_norm_8bit_cpu(const Tensor& x, const Tensor& residual,
                                                          const OptTensor& weight, const OptTensor& bias,
                                                          const OptTensor& gate, const OptTensor& post_weight,
                                                          const OptTensor& post_bias, c10::string_view norm,
                                                          c10::string_view post, double eps, double residual_scale,
                                                          double p, const OptTensor& rng, int64_t stream) {
  constexpr const char* op = "vectra::residual_norm_8bit";
  check_branch(x, residual, op);
  const NormOptions o = check_norm(x.sizes(), x.scalar_type(), x, weight, bias, gate, post_weight, post_bias, norm, post,
                                   eps, residual_scale, p, rng, stream, op);
  const auto [h, n] = norm_forward_cpu(x, residual, weight, bias, gate, post_weight, post_bias, o, rng);
  const auto [codes, scales] = quantize_cpu(n, 1);
  return {h.reshape(x.sizes()).to(residual.scalar_type()).clone(at::MemoryFormat::Contiguous), codes.reshape(codes_sizes(x)),
          scales.reshape(scales_sizes(x))};
}

std::vector<Tensor> residual_norm_backward_cpu(const OptTensor& grad_h, const OptTensor& grad_n, const OptTensor& h_in,
                                               const OptTensor& x, const OptTensor& residual, const OptTensor& weight,
                                               const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                                               const OptTensor& post_bias, c10::string_view norm, c10::string_view post,
                                               double eps, double residual_scale, double p, const OptTensor& rng,
                                               int64_t stream, at::ScalarType dtype, std::array<bool, 7> wanted) {
  const NormOptions o = check_norm_backward(grad_h, grad_n, h_in, x, residual, weight, bias, gate, post_weight, post_bias,
                                            norm, post, eps, residual_scale, p, rng, stream, dtype, wanted);
  const bool with_branch = reads_branch(h_in, residual, gate, post);
  const Tensor& side = with_branch ? *residual : *h_in;
  const int64_t width = side.size(-1), rows = rows_of(side);
  BranchCpu b;
  Tensor h;
  if (with_branch) {
    b = branch_cpu(*x, gate, post_weight, post_bias, o, rng);
    h = wide(*residual).reshape({rows, width}) * o.residual_scale + (b.gate.defined() ? b.v * b.gate : b.v);
  } else {
    h = wide(*h_in).reshape({rows, width});
    if (o.threshold) b.factors = factors_cpu(rows, width, o.threshold, *rng, o.stream);
  }
  const auto flat = [&](const OptTensor& g) { return has(g) ? wide(*g).reshape({rows, width}) : at::zeros_like(h); };
  const auto [hat, r] = normalised_cpu(h, o.norm, o.eps);
  const Tensor gn = flat(grad_n);
  Tensor gt = flat(grad_h);
  if (has(grad_n)) gt = gt + transpose_cpu(has(weight) ? gn * wide(*weight) : gn, hat, r, o.norm);
  Tensor gu = b.gate.defined() ? gt * b.gate : gt;
  if (b.factors.defined()) gu = drop_cpu(gu, b.factors);
  std::array<Tensor, 7> d;
  if (wanted[1]) d[1] = (gt * o.residual_scale).to(side.scalar_type());
  if (wanted[2]) d[2] = (gn * hat).sum(0).to(weight->scalar_type());
  if (wanted[3]) d[3] = gn.sum(0).to(bias->scalar_type());
  if (wanted[4]) d[4] = (gt * b.v).reshape(side.sizes()).sum_to_size(gate->sizes()).to(gate->scalar_type());
  if (wanted[5]) d[5] = (gu * b.hat).sum(0).to(post_weight->scalar_type());
  if (wanted[6]) d[6] = gu.sum(0).to(post_bias->scalar_type());
  if (wanted[0]) {
    if (b.hat.defined()) gu = transpose_cpu(has(post_weight) ? gu * wide(*post_weight) : gu, b.hat, b.r, o.post);
    d[0] = gu.to(dtype);
  }
  std::vector<Tensor> out;
  for (int i = 0; i < 7; ++i)
    if (wanted[i]) out.push_back((i < 2 ? d[i].reshape(side.sizes()) : d[i]).clone(at::MemoryFormat::Contiguous));
  return out;
}

// ------------------------------------------------------------- products in 8 bits

std::tuple<Tensor, Tensor> check_quantised(const Tensor& x, bool tiles) {
  constexpr const char* op = "vectra::quantize_blocks";
  TORCH_CHECK(x.dim() >= 1 && (!tiles || x.dim() == 2), op, ": x must be ", tiles ? "a matrix for tiles" : "[..., width]",
              "; got ", x.sizes());
  TORCH_CHECK(is_float(x.scalar_type()), op, ": x must be float32, float16 or bfloat16; got ", x.scalar_type());
  std::vector<int64_t> sizes = scales_sizes(x);
  if (tiles) sizes[0] = (sizes[0] + 127) / 128;
  return {at::empty(codes_sizes(x), x.options().dtype(at::kFloat8_e4m3fn)),
          at::empty(sizes, x.options().dtype(at::kFloat8_e8m0fnu))};
}

std::tuple<Tensor, Tensor> quantize_blocks_hip(const Tensor& x, bool tiles) {
  c10::DeviceGuard guard(x.device());
  auto [codes, scales] = check_quantised(x, tiles);
  const Rows xr = as_rows(x);
  check_status(vectra_blocks_quantize(xr.t.data_ptr(), dense_dtype(x.scalar_type()), rows_of(x), x.size(-1), xr.stride, tiles,
                                      codes.data_ptr(), scales.data_ptr(), stream_of(x)),
               "vectra::quantize_blocks");
  return {codes, scales};
}

std::tuple<Tensor, Tensor> quantize_blocks_cpu(const Tensor& x, bool tiles) {
  auto [codes, scales] = check_quantised(x, tiles);
  const auto [c, s] = quantize_cpu(wide(x).reshape({rows_of(x), x.size(-1)}), tiles ? 128 : 1);
  return {c.reshape(codes.sizes()), s.reshape(scales.sizes())};
}

// A layer's arguments: the result's type and the contraction's width.
struct Layer8 {
  at::ScalarType dtype;
  int64_t width, n_w;
};

Layer8 check_layer8(const Tensor& x, const Tensor& weight, const Tensor& weight_scales, const OptTensor& bias,
                    const OptTensor& residual, const OptTensor& scales, std::optional<at::ScalarType> dtype,
                    std::optional<int64_t> width, bool gated, const char* op) {
  TORCH_CHECK(x.dim() >= 1 && weight.dim() == 2 && weight_scales.dim() == 2, op,
              ": x must be [..., width], weight and weight_scales matrices; got ", x.sizes(), ", ", weight.sizes(), " and ",
              weight_scales.sizes());
  TORCH_CHECK(weight.scalar_type() == at::kFloat8_e4m3fn && weight_scales.scalar_type() == at::kFloat8_e8m0fnu, op,
              ": weight must be float8_e4m3fn codes with float8_e8m0fnu scales; got ", weight.scalar_type(), " and ",
              weight_scales.scalar_type());
  Layer8 l{x.scalar_type(), x.size(-1), weight.size(0)};
  if (has(scales)) {
    TORCH_CHECK(x.scalar_type() == at::kFloat8_e4m3fn && scales->scalar_type() == at::kFloat8_e8m0fnu, op,
                ": an input given with scales must be float8_e4m3fn codes and float8_e8m0fnu scales; got ", x.scalar_type(),
                " and ", scales->scalar_type());
    TORCH_CHECK(l.width % 128 == 0 && scales->sizes() == at::IntArrayRef(scales_sizes(x)), op,
                ": codes must be whole blocks of 128 and scales [..., 4 ceil(width / 512)]; got ", x.sizes(), " and ",
                scales->sizes());
    TORCH_CHECK(dtype.has_value(), op, ": an input in 8 bits needs dtype, the result's");
    TORCH_CHECK(is_float(*dtype), op, ": dtype must be float32, float16 or bfloat16; got ", *dtype);
    TORCH_CHECK(scales->device() == x.device(), op, ": scales must be on ", x.device(), "; got ", scales->device());
    l.dtype = *dtype;
  } else {
    TORCH_CHECK(is_float(l.dtype), op, ": x must be float32, float16 or bfloat16, or codes with their scales; got ", l.dtype);
    TORCH_CHECK(!dtype.has_value() || *dtype == l.dtype, op, ": dtype must be x's, ", l.dtype, "; got ", *dtype);
  }
  TORCH_CHECK(weight.size(1) == (l.width + 127) / 128 * 128 && weight_scales.size(0) == (l.n_w + 127) / 128 &&
                  weight_scales.size(1) == (l.width + 511) / 512 * 4,
              op, ": weight must be [width_out, width] in tiles of 128 x 128, as quantize_blocks makes it; got ",
              weight.sizes(), " with scales ", weight_scales.sizes(), " for x ", x.sizes());
  // (Codes and scales tell the weight's width only rounded up to a block.)
  TORCH_CHECK(!width.has_value() || (has(scales) ? (*width >= 0 && (*width + 127) / 128 * 128 == l.width) : *width == l.width), op,
              ": x must be ", width.value_or(0), " wide, as the weight is; got ", x.sizes(), has(scales) ? " of codes" : "");
  TORCH_CHECK(!gated || l.n_w % 2 == 0, op, ": weight must hold the gate's rows and as many rows of the up projection; got ",
              weight.sizes());
  TORCH_CHECK(weight.device() == x.device() && weight_scales.device() == x.device(), op, ": weight and weight_scales must be on ",
              x.device(), "; got ", weight.device(), " and ", weight_scales.device());
  if (has(bias)) check_vector(bias, l.n_w, l.dtype, x.device(), "bias", op);
  if (has(residual)) {
    TORCH_CHECK(residual->sizes() == at::IntArrayRef(with_last(x, l.n_w)), op, ": residual must have the output's shape; got ",
                residual->sizes());
    TORCH_CHECK(residual->scalar_type() == l.dtype && residual->device() == x.device(), op, ": residual must be ", l.dtype, " on ",
                x.device(), "; got ", residual->scalar_type(), " on ", residual->device());
  }
  return l;
}

// Bytes that lie one row after the other, from a multiple of 16 bytes on.
Tensor packed(const Tensor& t) {
  const Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.const_data_ptr()) % 16 ? c.clone() : c;
}

Tensor layer8_hip(const Tensor& x, const Tensor& weight_in, const Tensor& weight_scales_in, const OptTensor& bias_in,
                  const OptTensor& residual, c10::string_view activation, const OptTensor& scales_in,
                  std::optional<at::ScalarType> dtype, std::optional<int64_t> width, bool gated, const char* op) {
  const Layer8 l = check_layer8(x, weight_in, weight_scales_in, bias_in, residual, scales_in, dtype, width, gated, op);
  const int32_t act = activation_of(activation, op);
  c10::DeviceGuard guard(x.device());
  const int64_t n = gated ? l.n_w / 2 : l.n_w;
  Tensor out = at::empty(with_last(x, n), x.options().dtype(l.dtype));
  const Tensor weight = packed(weight_in), weight_scales = packed(weight_scales_in);
  const Tensor bias = has(bias_in) ? bias_in->contiguous() : Tensor();
  Rows xr, rr;
  Tensor codes, scales;
  vectra_linear8_args a{};
  a.struct_size = sizeof(a);
  if (has(scales_in)) {
    codes = packed(x);
    scales = packed(*scales_in);
    a.codes = codes.data_ptr();
    a.scales = scales.data_ptr();
  } else {
    xr = as_rows(x);
    a.x = xr.t.data_ptr();
  }
  if (has(residual)) rr = as_rows(*residual);
  a.weight = weight.data_ptr();
  a.weight_scales = weight_scales.data_ptr();
  a.bias = bias.defined() ? bias.data_ptr() : nullptr;
  a.residual = rr.t.defined() ? rr.t.data_ptr() : nullptr;
  a.out = out.data_ptr();
  a.dtype = dense_dtype(l.dtype);
  a.bias_dtype = bias.defined() ? dense_dtype(bias.scalar_type()) : a.dtype;
  a.activation = act;
  a.gated = gated;
  a.rows = rows_of(x);
  a.width = l.width;
  a.width_out = n;
  a.x_stride = xr.stride;
  a.residual_stride = rr.stride;
  a.out_stride = std::max<int64_t>(n, 1);
  const int64_t need = vectra_linear8_workspace_bytes(&a);
  if (need < 0) check_status(static_cast<int>(-need), op);
  Tensor workspace;
  if (need > 0) workspace = at::empty({need}, x.options().dtype(at::kByte));
  check_status(vectra_linear8_forward(&a, need > 0 ? workspace.data_ptr() : nullptr, need, stream_of(x)), op);
  return out;
}

// What codes and scales stand for, in fp32 [rows, depth].
Tensor values_cpu(const Tensor& codes_in, const Tensor& scales_in, int64_t high) {
  const Tensor codes = codes_in.reshape({-1, codes_in.size(-1)});
  const Tensor e = scales_in.contiguous().view(at::kByte).reshape({-1, scales_in.size(-1)}).to(at::kInt) - 127;
  const Tensor each = e.narrow(1, 0, codes.size(1) / 128).repeat_interleave(high, 0).narrow(0, 0, codes.size(0)).repeat_interleave(128, 1);
  const Tensor value = at::ldexp(codes.to(at::kDouble), each);
  return at::where(each == 128, at::full_like(value, std::nan("")), value).to(at::kFloat);
}

Tensor layer8_cpu(const Tensor& x, const Tensor& weight, const Tensor& weight_scales, const OptTensor& bias,
                  const OptTensor& residual, c10::string_view activation, const OptTensor& scales,
                  std::optional<at::ScalarType> dtype, std::optional<int64_t> width, bool gated, const char* op) {
  const Layer8 l = check_layer8(x, weight, weight_scales, bias, residual, scales, dtype, width, gated, op);
  const int32_t act = activation_of(activation, op);
  const int64_t rows = rows_of(x), n = gated ? l.n_w / 2 : l.n_w;
  if (rows == 0 || n == 0) return at::empty(with_last(x, n), x.options().dtype(l.dtype));
  Tensor z;
  if (l.width == 0) {
    z = at::zeros({rows, l.n_w}, x.options().dtype(at::kFloat));
  } else {
    const auto [c, s] = has(scales) ? std::tuple<Tensor, Tensor>(x, *scales) : quantize_cpu(wide(x).reshape({rows, l.width}), 1);
    z = at::matmul(values_cpu(c, s, 1), values_cpu(weight, weight_scales, 128).t());
  }
  if (has(bias)) z = z + wide(*bias);
  Tensor y;
  if (gated) {
    const auto halves = z.chunk(2, -1);
    y = activation_cpu(halves[0], act).first * halves[1];
  } else {
    y = act == VECTRA_DENSE_NONE ? z : activation_cpu(z, act).first;
  }
  if (has(residual)) y = y + wide(*residual).reshape({rows, n});
  return y.to(l.dtype).reshape(with_last(x, n)).contiguous();
}

template <Tensor (*kLayer)(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, c10::string_view,
                           const OptTensor&, std::optional<at::ScalarType>, std::optional<int64_t>, bool, const char*)>
Tensor linear_8bit(const Tensor& x, const Tensor& weight, const Tensor& weight_scales, const OptTensor& bias,
                   const OptTensor& residual, c10::string_view activation, const OptTensor& scales,
                   std::optional<at::ScalarType> dtype, std::optional<int64_t> width) {
  return kLayer(x, weight, weight_scales, bias, residual, activation, scales, dtype, width, false, "vectra::linear_8bit");
}

template <Tensor (*kLayer)(const Tensor&, const Tensor&, const Tensor&, const OptTensor&, const OptTensor&, c10::string_view,
                           const OptTensor&, std::optional<at::ScalarType>, std::optional<int64_t>, bool, const char*)>
Tensor gated_linear_8bit(const Tensor& x, const Tensor& weight, const Tensor& weight_scales, const OptTensor& bias,
                         c10::string_view activation, const OptTensor& scales, std::optional<at::ScalarType> dtype,
                         std::optional<int64_t> width) {
  return kLayer(x, weight, weight_scales, bias, std::nullopt, activation, scales, dtype, width, true,
                "vectra::gated_linear_8bit");
}

// --------------------------------------------------------------- gradients

Tensor call_dropout(const Tensor& x, double p, const Tensor& rng, int64_t stream) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vectra::dropout", "")
                       .typed<Tensor(const Tensor&, double, const Tensor&, int64_t)>();
  return op.call(x, p, rng, stream);
}

std::tuple<Tensor, Tensor> call_norm(const Tensor& x, const Tensor& residual, const OptTensor& weight, const OptTensor& bias,
                                     const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                                     c10::string_view norm, c10::string_view post, double eps, double residual_scale,
                                     double p, const OptTensor& rng, int64_t stream) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("vectra::residual_norm", "")
                       .typed<std::tuple<Tensor, Tensor>(const Tensor&, const Tensor&, const OptTensor&, const OptTensor&,
                                                         const OptTensor&, const OptTensor&, const OptTensor&,
                                                         c10::string_view, c10::string_view, double, double, double,
                                                         const OptTensor&, int64_t)>();
  return op.call(x, residual, weight, bias, gate, post_weight, post_bias, norm, post, eps, residual_scale, p, rng, stream);
}

std::vector<Tensor> call_norm_backward(const OptTensor& grad_h, const OptTensor& grad_n, const OptTensor& h,
                                       const OptTensor& x, const OptTensor& residual, const OptTensor& weight,
                                       const OptTensor& bias, const OptTensor& gate, const OptTensor& post_weight,
                                       const OptTensor& post_bias, c10::string_view norm, c10::string_view post, double eps,
                                       double residual_scale, double p, const OptTensor& rng, int64_t stream,
                                       at::ScalarType dtype, std::array<bool, 7> wanted) {
  static auto op =
      c10::Dispatcher::singleton()
          .findSchemaOrThrow("vectra::residual_norm_backward", "")
          .typed<std::vector<Tensor>(const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                                     const OptTensor&, const OptTensor&, const OptTensor&, const OptTensor&,
                                     const OptTensor&, c10::string_view, c10::string_view, double, double, double,
                                     const OptTensor&, int64_t, at::ScalarType, std::array<bool, 7>)>();
  return op.call(grad_h, grad_n, h, x, residual, weight, bias, gate, post_weight, post_bias, norm, post, eps,
                 residual_scale, p, rng, stream, dtype, wanted);
}

bool wants(const OptTensor& t) { return has(t) && t->requires_grad(); }

void refuse_second(const char* op) {
  TORCH_CHECK(!at::GradMode::is_enabled(), op, ": gradients of gradients are not supported (create_graph=True)");
}

// Below autograd a tangent would be dropped without a word.
bool dual(const OptTensor& t) { return has(t) && t->_fw_grad(/*level=*/0).defined(); }

void refuse_tangent(bool any, const char* op) {
  TORCH_CHECK_NOT_IMPLEMENTED(!any, op, ": forward-mode derivatives are not supported (an argument carries a tangent)");
}

// The gradient is the operator itself on it: nothing is kept but rng.
class Dropout : public torch::autograd::Function<Dropout> {
 public:
  static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, double p, const Tensor& rng, int64_t stream) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor y = call_dropout(x, p, rng, stream);
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    ctx->save_for_backward({rng});
    return y;
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    torch::autograd::variable_list out(4);
    if (!grads[0].defined()) return out;
    // (Through autograd again: linear in x, so gradients of gradients are its too.)
    out[0] = call_dropout(grads[0], ctx->saved_data["p"].toDouble(), ctx->get_saved_variables()[0],
                          ctx->saved_data["stream"].toInt());
    return out;
  }
};

Tensor dropout_autograd(const Tensor& x, double p, const Tensor& rng, int64_t stream) {
  refuse_tangent(dual(x), "vectra::dropout");
  if (!at::GradMode::is_enabled() || !x.requires_grad()) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_dropout(x, p, rng, stream);
  }
  return Dropout::apply(x, p, rng, stream);
}

// Saved: x and the residual, or an fp32 h that tells all that matters.
class ResidualNorm : public torch::autograd::Function<ResidualNorm> {
 public:
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const Tensor& x,
                                                const Tensor& residual, const OptTensor& weight, const OptTensor& bias,
                                                const OptTensor& gate, const OptTensor& post_weight,
                                                const OptTensor& post_bias, const std::string& norm, const std::string& post,
                                                double eps, double residual_scale, double p, const OptTensor& rng,
                                                int64_t stream) {
    at::AutoDispatchBelowADInplaceOrView below;
    const auto [h, n] = call_norm(x, residual, weight, bias, gate, post_weight, post_bias, norm, post, eps, residual_scale, p,
                                  rng, stream);
    const OptTensor leaves[7] = {x, residual, weight, bias, gate, post_weight, post_bias};
    int64_t wanted = 0;
    for (int i = 0; i < 7; ++i) wanted |= static_cast<int64_t>(wants(leaves[i])) << i;
    ctx->saved_data["wanted"] = wanted;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["post"] = post;
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["residual_scale"] = residual_scale;
    ctx->saved_data["p"] = p;
    ctx->saved_data["stream"] = stream;
    ctx->saved_data["dtype"] = static_cast<int64_t>(x.scalar_type());
    const bool branch = reads_branch(residual.scalar_type(), gate, post);
    const auto kept = [](const OptTensor& t) { return has(t) ? *t : Tensor(); };
    ctx->save_for_backward({branch ? Tensor() : h, branch ? x : Tensor(), branch ? residual : Tensor(), kept(weight),
                            kept(bias), kept(gate), kept(post_weight), kept(post_bias), p > 0 ? kept(rng) : Tensor()});
    ctx->set_materialize_grads(false);
    return {h, n};
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    refuse_second("vectra::residual_norm");
    torch::autograd::variable_list out(14);
    if (!grads[0].defined() && !grads[1].defined()) return out;
    const int64_t mask = ctx->saved_data["wanted"].toInt();
    std::array<bool, 7> wanted{};
    for (int i = 0; i < 7; ++i) wanted[i] = mask >> i & 1;
    const auto saved = ctx->get_saved_variables();
    const auto given = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    const auto g = call_norm_backward(given(grads[0]), given(grads[1]), given(saved[0]), given(saved[1]), given(saved[2]),
                                      given(saved[3]), given(saved[4]), given(saved[5]), given(saved[6]), given(saved[7]),
                                      ctx->saved_data["norm"].toStringRef(), ctx->saved_data["post"].toStringRef(),
                                      ctx->saved_data["eps"].toDouble(), ctx->saved_data["residual_scale"].toDouble(),
                                      ctx->saved_data["p"].toDouble(), given(saved[8]), ctx->saved_data["stream"].toInt(),
                                      static_cast<at::ScalarType>(ctx->saved_data["dtype"].toInt()), wanted);
    size_t at = 0;
    for (int i = 0; i < 7; ++i)
      if (wanted[i]) out[i] = g[at++];
    return out;
  }
};

std::tuple<Tensor, Tensor> residual_norm_autograd(const Tensor& x, const Tensor& residual, const OptTensor& weight,
                                                  const OptTensor& bias, const OptTensor& gate,
                                                  const OptTensor& post_weight, const OptTensor& post_bias,
                                                  c10::string_view norm, c10::string_view post, double eps,
                                                  double residual_scale, double p, const OptTensor& rng, int64_t stream) {
  refuse_tangent(dual(x) || dual(residual) || dual(weight) || dual(bias) || dual(gate) || dual(post_weight) || dual(post_bias),
                 "vectra::residual_norm");
  if (!at::GradMode::is_enabled() || !(wants(x) || wants(residual) || wants(weight) || wants(bias) || wants(gate) ||
                                       wants(post_weight) || wants(post_bias))) {
    at::AutoDispatchBelowADInplaceOrView below;
    return call_norm(x, residual, weight, bias, gate, post_weight, post_bias, norm, post, eps, residual_scale, p, rng, stream);
  }
  const auto out = ResidualNorm::apply(x, residual, weight, bias, gate, post_weight, post_bias, std::string(norm),
                                       std::string(post), eps, residual_scale, p, rng, stream);
  return {out[0], out[1]};
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(vectra, m) {
  m.def("dropout(Tensor x, float p, Tensor rng, int stream=0) -> Tensor");
  m.def("dropout_pass(Tensor(a!) state) -> Tensor");
  m.def(
      "residual_norm(Tensor x, Tensor residual, Tensor? weight=None, Tensor? bias=None, Tensor? gate=None, "
      "Tensor? post_weight=None, Tensor? post_bias=None, *, str norm='rms', str post='none', float eps=1e-6, "
      "float residual_scale=1.0, float p=0.0, Tensor? rng=None, int stream=0) -> (Tensor, Tensor)");
  m.def(
      "residual_norm_8bit(Tensor x, Tensor residual, Tensor? weight=None, Tensor? bias=None, Tensor? gate=None, "
      "Tensor? post_weight=None, Tensor? post_bias=None, *, str norm='rms', str post='none', float eps=1e-6, "
      "float residual_scale=1.0, float p=0.0, Tensor? rng=None, int stream=0) -> (Tensor, Tensor, Tensor)");
  m.def(
      "residual_norm_backward(Tensor? grad_h, Tensor? grad_n, Tensor? h, Tensor? x, Tensor? residual, Tensor? weight, "
      "Tensor? bias, Tensor? gate, Tensor? post_weight, Tensor? post_bias, str norm, str post, float eps, "
      "float residual_scale, float p, Tensor? rng, int stream, ScalarType dtype, bool[7] wanted) -> Tensor[]");
  m.def("quantize_blocks(Tensor x, bool tiles=False) -> (Tensor, Tensor)");
  m.def(
      "linear_8bit(Tensor x, Tensor weight, Tensor weight_scales, Tensor? bias=None, Tensor? residual=None, "
      "str activation='none', *, Tensor? scales=None, ScalarType? dtype=None, int? width=None) -> Tensor");
  m.def(
      "gated_linear_8bit(Tensor x, Tensor weight, Tensor weight_scales, Tensor? bias=None, str activation='silu', *, "
      "Tensor? scales=None, ScalarType? dtype=None, int? width=None) -> Tensor");
}

TORCH_LIBRARY_IMPL(vectra, CUDA, m) {
  m.impl("dropout", dropout_hip);
  m.impl("dropout_pass", dropout_pass);
  m.impl("residual_norm", residual_norm_hip);
  m.impl("residual_norm_8bit", residual_norm_8bit_hip);
  m.impl("residual_norm_backward", residual_norm_backward_hip);
  m.impl("quantize_blocks", quantize_blocks_hip);
  m.impl("linear_8bit", linear_8bit<layer8_hip>);
  m.impl("gated_linear_8bit", gated_linear_8bit<layer8_hip>);
}

TORCH_LIBRARY_IMPL(vectra, CPU, m) {
  m.impl("dropout", dropout_cpu);
  m.impl("dropout_pass", dropout_pass);
  m.impl("residual_norm", residual_norm_cpu);
  m.impl("residual_norm_8bit", residual_norm_8bit_cpu);
  m.impl("residual_norm_backward", residual_norm_backward_cpu);
  m.impl("quantize_blocks", quantize_blocks_cpu);
  m.impl("linear_8bit", linear_8bit<layer8_cpu>);
  m.impl("gated_linear_8bit", gated_linear_8bit<layer8_cpu>);
}

TORCH_LIBRARY_IMPL(vectra, Autograd, m) {
  m.impl("dropout", dropout_autograd);
  m.impl("residual_norm", residual_norm_autograd);
  // No derivatives: a backward pass that reaches one of these raises, and so
  // does a tangent.
  m.impl("residual_norm_8bit", torch::autograd::autogradNotImplementedFallback());
  m.impl("residual_norm_backward", torch::autograd::autogradNotImplementedFallback());
  m.impl("quantize_blocks", torch::autograd::autogradNotImplementedFallback());
  m.impl("linear_8bit", torch::autograd::autogradNotImplementedFallback());
  m.impl("gated_linear_8bit", torch::autograd::autogradNotImplementedFallback());
}
