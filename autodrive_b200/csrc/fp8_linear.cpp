// Linear layer with both operands in 8 bits, for training:
//
//   y  = Q(x) Q(w)^T + b      Q: e4m3 with scales for blocks of 128
//   dx = Q(dy) Q(w)           rounding counts as the identity
//   dw = dy^T x               16-bit operands, fp32 sums
//   db = sum of dy's rows     in fp32
//
// The weight gradient's operands are x and dy as they are where both are bf16
// or both fp16. Otherwise they are rounded to bf16: the tensor cores take 16
// bits at full rate, and what the rounding adds, 2^-8 of each term at most, is
// a sixteenth of what the layer's own e4m3 rounding of x and dy does to y and dx.
//
// One call runs the quantisers and the product, and one backward its
// kernels, so that no Python runs between the launches.
#include <torch/extension.h>
#include <c10/core/DeviceGuard.h>

#include <algorithm>

#include "fp8.h"
#include "lm_host.h"

namespace py = pybind11;

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// `x` as an operand of the weight gradient, bf16 or fp16: rows that start 16
// bytes apart on an aligned base (a copy only where they do not).
torch::Tensor operand(const torch::Tensor& x, torch::ScalarType type) {
  const int64_t rows = x.size(0), k = x.size(1);
  if (x.scalar_type() == type && (rows <= 1 || x.stride(0) % 8 == 0) && (k <= 1 || x.stride(1) == 1) &&
      reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && rows != 1)
    return x;
  auto y = torch::empty({rows, (k + 7) / 8 * 8}, x.options().dtype(type)).narrow(1, 0, k);
  y.copy_(x);
  return y;
}

// Counts a backward's launches towards the read-backs of the status word, and
// raises what one has found (ops/tc_linear.py), as a forward does.
void poll_status(const c10::Device& device) {
  const py::gil_scoped_acquire gil;
  py::module_::import("autodrive_b200.ops.tc_linear").attr("_Status").attr("after_launch")(py::cast(device));
}

struct Fp8LinearFn : torch::autograd::Function<Fp8LinearFn> {
  static torch::Tensor forward(AutogradContext* ctx, const torch::Tensor& x, const torch::Tensor& weight,
                               const c10::optional<torch::Tensor>& bias_, int64_t out_dtype, bool grad,
                               const torch::Tensor& status) {
    at::AutoDispatchBelowADInplaceOrView below;
    const c10::DeviceGuard guard(x.device());
    const torch::Tensor bias = bias_ ? *bias_ : torch::Tensor();
    const auto x2 = fp8::as_matrix(x);
    const bool need_x = grad && x.requires_grad(), need_w = grad && weight.requires_grad();
    const auto xq = fp8::quantize_rows(x2);
    // the input gradient reads the weight down its columns: its transposed copy is written by the same pass
    const auto wq = fp8::quantize_blocks(fp8::as_matrix(weight), need_x);
    torch::Tensor b;
    if (bias.defined()) b = bias.to(torch::kFloat32).contiguous();
    const auto y = fp8::matmul(xq.first, xq.second, wq[0], wq[1], b, static_cast<torch::ScalarType>(out_dtype), status,
                               fp8::kWaitNs);
    torch::Tensor keep;   // what the weight gradient reads: the caller's x where it can be read as it is
    if (need_w && x2.scalar_type() == torch::kFloat32) keep = x2.to(torch::kBFloat16);
    else if (need_w) keep = x2.is_alias_of(x) ? x : x2;
    ctx->save_for_backward({keep, need_x ? wq[2] : torch::Tensor(), need_x ? wq[3] : torch::Tensor()});
    ctx->saved_data["status"] = status;   // every call's, cleared by others: not a variable of this graph
    ctx->saved_data["x_sizes"] = x.sizes().vec();
    ctx->saved_data["n"] = weight.size(0);
    ctx->saved_data["x_type"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["w_type"] = static_cast<int64_t>(weight.scalar_type());
    ctx->saved_data["b_type"] = bias.defined() ? static_cast<int64_t>(bias.scalar_type()) : -1;
    auto sizes = x.sizes().vec();
    sizes.back() = weight.size(0);
    return y.view(sizes);
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    TORCH_CHECK(!at::GradMode::is_enabled(), "fp8_linear has no second derivative (create_graph)");
    const auto saved = ctx->get_saved_variables();
    const auto x_sizes = ctx->saved_data["x_sizes"].toIntVector();
    const int64_t n = ctx->saved_data["n"].toInt(), k = x_sizes.back();
    const c10::DeviceGuard guard(grads[0].device());
    const auto g = fp8::as_matrix(grads[0]);
    const auto status = ctx->saved_data["status"].toTensor();
    variable_list out(6);
    if (ctx->needs_input_grad(0)) {
      const auto gq = fp8::quantize_rows(g);
      out[0] = fp8::matmul(gq.first, gq.second, saved[1], saved[2], {},
                           static_cast<torch::ScalarType>(ctx->saved_data["x_type"].toInt()), status, fp8::kWaitNs)
                   .view(x_sizes);
    }
    if (ctx->needs_input_grad(1)) {
      const auto rows = fp8::as_matrix(saved[0]);
      const auto type = g.scalar_type() == torch::kHalf && rows.scalar_type() == torch::kHalf ? torch::kHalf : torch::kBFloat16;
      out[1] = fp8::weight_gradient(operand(g, type), operand(rows, type),
                                    static_cast<torch::ScalarType>(ctx->saved_data["w_type"].toInt()), status);
    }
    const int64_t b_type = ctx->saved_data["b_type"].toInt();
    if (b_type >= 0 && ctx->needs_input_grad(2))
      out[2] = fp8::column_sums(g, static_cast<torch::ScalarType>(b_type));
    if (ctx->needs_input_grad(0) || ctx->needs_input_grad(1)) poll_status(g.device());
    return out;
  }
};

torch::Tensor fp8_linear(torch::Tensor x, torch::Tensor weight, c10::optional<torch::Tensor> bias, py::object dtype,
                         torch::Tensor status) {
  LM_CHECK_VALUE(x.is_cuda() && fp8::known_type(x.scalar_type()) && x.dim() >= 1 &&
                        fp8::known_type(weight.scalar_type()) && weight.dim() == 2,
                    "fp8_linear takes fp32, bf16 or fp16 rows [..., K] and a weight [N, K]");
  LM_CHECK_VALUE(x.size(-1) == weight.size(1) &&
                        (!bias || (bias->dim() == 1 && bias->size(0) == weight.size(0) &&
                                   fp8::known_type(bias->scalar_type()))),
                    "fp8_linear: x ", x.sizes(), ", weight ", weight.sizes(), " and bias do not fit");
  LM_CHECK_VALUE(weight.device() == x.device() && status.device() == x.device() &&
                        (!bias || bias->device() == x.device()),
                    "fp8_linear needs all of its tensors on one device");
  TORCH_CHECK(status.scalar_type() == torch::kInt32, "fp8_linear: status must be int32");
  LM_CHECK_NO_TANGENT("fp8_linear", x, weight, bias);
  return Fp8LinearFn::apply(x, weight, bias,
                            static_cast<int64_t>(torch::python::detail::py_object_to_dtype(dtype)),
                            at::GradMode::is_enabled(), status);
}

}  // namespace

void register_fp8_linear_ops(py::module& m) {
  m.def("fp8_linear", &fp8_linear, "linear layer with both operands quantised to e4m3, with autograd", py::arg("x"),
        py::arg("weight"), py::arg("bias"), py::arg("out_dtype"), py::arg("status"));
}
