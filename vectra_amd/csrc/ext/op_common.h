// What the operators' torch registrations share: tensors as the C ABIs take them,
// activations by name and on the CPU.
#pragma once

#include <ATen/ATen.h>
#include <c10/hip/HIPStream.h>

#include <algorithm>
#include <cmath>
#include <optional>
#include <string>
#include <string_view>
#include <utility>
#include <vector>

#include "vectra_dense.h"

namespace vectra_ops {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

inline bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

inline int32_t dense_dtype(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return VECTRA_DENSE_F32;
    case at::kHalf: return VECTRA_DENSE_F16;
    case at::kBFloat16: return VECTRA_DENSE_BF16;
    default: return -1;
  }
}

inline int32_t activation_of(std::string_view name, const char* op) {
  if (name == "none") return VECTRA_DENSE_NONE;
  if (name == "relu") return VECTRA_DENSE_RELU;
  if (name == "gelu") return VECTRA_DENSE_GELU;
  if (name == "gelu_tanh") return VECTRA_DENSE_GELU_TANH;
  if (name == "silu") return VECTRA_DENSE_SILU;
  TORCH_CHECK_VALUE(false, op, ": activation must be 'none', 'relu', 'gelu', 'gelu_tanh' or 'silu'; got '",
                    std::string(name), "'");
}

inline std::vector<int64_t> with_last(const Tensor& x, int64_t last) {
  std::vector<int64_t> sizes(x.sizes().begin(), x.sizes().end());
  sizes.back() = last;
  return sizes;
}

inline int64_t rows_of(const Tensor& x) {
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
  return rows;
}

// A matrix the C ABI can read: rows with unit element stride, one row stride
// of at least a row, 256 rows within 2^31 bytes.  A view that has none (a
// transposed or an expanded one, or one of rows very far apart) is copied.
struct Rows {
  Tensor t;
  int64_t stride = 0;
};

inline Rows as_rows(const Tensor& x) {
  const int64_t width = x.size(-1);
  const int64_t rows = rows_of(x);
  Rows r;
  if (x.dim() == 2) {
    r.t = x;
  } else {
    r.t = x.reshape({rows, width});
  }
  const bool near = rows <= 1 || (r.t.stride(0) >= width && r.t.stride(0) < (int64_t{1} << 23) / x.element_size());
  if ((width > 1 && r.t.stride(1) != 1) || !near) r.t = r.t.contiguous();
  r.stride = rows > 1 ? r.t.stride(0) : std::max<int64_t>(width, 1);
  return r;
}

// act(z) and act'(z).
inline std::pair<Tensor, Tensor> activation_cpu(const Tensor& z, int32_t act) {
  switch (act) {
    case VECTRA_DENSE_RELU: return {z.clamp_min(0), z.gt(0).to(z.scalar_type())};
    case VECTRA_DENSE_GELU: {
      const Tensor cdf = at::erfc(z * -std::sqrt(0.5)) * 0.5;
      return {z * cdf, cdf + z * at::exp(z * z * -0.5) * (1.0 / std::sqrt(2.0 * M_PI))};
    }
    case VECTRA_DENSE_GELU_TANH: {
      const double c = std::sqrt(2.0 / M_PI), k = 0.044715;
      const Tensor y = (z + z * z * z * k) * (2 * c), s = at::sigmoid(y);
      // (z^2 held finite, as on the GPU.)
      return {z * s, s + z * s * at::sigmoid(-y) * ((z * z).clamp_max(1e30) * (3 * k) + 1) * (2 * c)};
    }
    case VECTRA_DENSE_SILU: {
      const Tensor s = at::sigmoid(z);
      return {z * s, s + z * s * at::sigmoid(-z)};
    }
    default: return {z, at::ones_like(z)};
  }
}

}  // namespace vectra_ops
