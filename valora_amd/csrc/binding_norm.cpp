// Torch binding of the norms around a layer's blocks (include/mlora.h).
#include <ATen/core/grad_mode.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <utility>

#include "binding_common.h"

namespace {

using Maybe = c10::optional<at::Tensor>;

py::tuple block_norm(const at::Tensor &x, const Maybe &weight, const Maybe &bias, const Maybe &block, const Maybe &block_weight, const Maybe &block_bias,
                     const Maybe &gate, double residual_scale, double block_scale, double eps, bool layer, double offset, const Maybe &residual_out,
                     const Maybe &out) {
  // (a result without a history would drop the gradient without a word)
  const auto no_gradient = [](const at::Tensor &t, const char *name) {
    if (t.requires_grad()) raise(std::string("block_norm has no backward pass: ") + name + " requires a gradient (call it under torch.no_grad())");
  };
  if (at::GradMode::is_enabled()) {
    no_gradient(x, "x");
    const std::pair<const Maybe &, const char *> others[] = {{weight, "weight"}, {bias, "bias"}, {block, "block"}, {block_weight, "block_weight"},
                                                             {block_bias, "block_bias"}, {gate, "gate"}, {residual_out, "residual_out"}, {out, "out"}};
    for (const auto &[t, name] : others)
      if (t.has_value()) no_gradient(*t, name);
  }
  if (!x.is_cuda()) raise("x must be a CUDA tensor");
  const c10::Device dev = x.device();
  const mlora_dtype code = dtype_code(x);
  if ((int)code < 0) raise("No suitable kernel. block_norm dtype=" + dtype_name(x));
  if (x.dim() != 2) raise("x must be [tokens, width]");
  mlora_norm n{};
  n.T = x.size(0);
  n.H = x.size(1);
  const auto on_device = [&](const at::Tensor &t, const char *name) {
    if (!t.is_cuda()) raise(std::string(name) + " must be a CUDA tensor");
    if (t.device() != dev) raise(std::string(name) + " is on " + t.device().str() + ", expected " + dev.str());
  };
  const auto rows = [&](const at::Tensor &t, const char *name, int64_t &stride) {
    on_device(t, name);
    if (t.scalar_type() != x.scalar_type()) raise(std::string("No suitable kernel. ") + name + " dtype=" + dtype_name(t));
    if (t.dim() != 2 || t.size(0) != n.T || t.size(1) != n.H) raise(std::string(name) + " must have x's shape");
    if (n.H > 1 && t.numel() > 0 && t.stride(1) != 1) raise(std::string(name) + ": elements of a row must be contiguous");
    stride = n.T > 1 ? t.stride(0) : n.H;
    return t.data_ptr();
  };
  const auto vector = [&](const Maybe &t, const char *name, int flag) -> const void * {
    if (!t.has_value()) return nullptr;
    on_device(*t, name);
    if (t->scalar_type() == at::kFloat) n.f32 |= flag;
    else if (t->scalar_type() != x.scalar_type()) raise(std::string("No suitable kernel. ") + name + " dtype=" + dtype_name(*t));
    if (t->dim() != 1 || t->size(0) != n.H || !t->is_contiguous()) raise(std::string(name) + " must be a contiguous vector of x's width");
    return t->data_ptr();
  };
  n.x = rows(x, "x", n.x_stride);
  n.weight = vector(weight, "weight", MLORA_NORM_F32_WEIGHT);
  n.bias = vector(bias, "bias", MLORA_NORM_F32_BIAS);
  n.block_weight = vector(block_weight, "block_weight", MLORA_NORM_F32_BLOCK_WEIGHT);
  n.block_bias = vector(block_bias, "block_bias", MLORA_NORM_F32_BLOCK_BIAS);
  if (!block.has_value() && (block_weight.has_value() || gate.has_value() || residual_out.has_value() || residual_scale != 1.0 || block_scale != 1.0))
    raise("block_norm: block's operands without block");
  if (!block.has_value() && !weight.has_value()) raise("block_norm: neither a block to add nor a weight to normalise with");
  if (block_bias.has_value() && !block_weight.has_value()) raise("block_norm: block_bias without block_weight");
  if (bias.has_value() && !weight.has_value()) raise("block_norm: bias without weight");
  if (out.has_value() && !weight.has_value()) raise("block_norm: out without weight");
  py::object r = py::none(), h = py::none();
  at::Tensor r_new, h_new;
  if (block.has_value()) {
    n.block = rows(*block, "block", n.block_stride);
    if (gate.has_value()) {
      const at::Tensor &g = *gate;
      on_device(g, "gate");
      if (g.scalar_type() == at::kFloat) n.f32 |= MLORA_NORM_F32_GATE;
      else if (g.scalar_type() != x.scalar_type()) raise("No suitable kernel. gate dtype=" + dtype_name(g));
      // one a channel, one a token, one an element
      if (g.dim() == 1 && g.size(0) == n.H) {
        n.gate_column_stride = g.stride(0);
      } else if (g.dim() == 2 && g.size(0) == n.T && (g.size(1) == n.H || g.size(1) == 1)) {
        n.gate_row_stride = n.T > 1 ? g.stride(0) : 0;
        n.gate_column_stride = g.size(1) == 1 ? 0 : g.stride(1);
      } else {
        raise("gate must be [width], [tokens, 1] or [tokens, width]");
      }
      if (n.H == 1) n.gate_column_stride = 0;
      if (n.gate_column_stride != 0 && n.gate_column_stride != 1) raise("gate: elements of a row must be contiguous");
      n.gate = g.data_ptr();
    }
    r_new = residual_out.has_value() ? *residual_out : at::empty_like(x, x.options(), at::MemoryFormat::Contiguous);
    n.residual_out = rows(r_new, "residual_out", n.residual_stride);
    r = py::cast(r_new);
  } else {
    r = py::cast(x);
  }
  if (weight.has_value()) {
    h_new = out.has_value() ? *out : at::empty_like(x, x.options(), at::MemoryFormat::Contiguous);
    n.out = rows(h_new, "out", n.out_stride);
    h = py::cast(h_new);
  }
  n.residual_scale = (float)residual_scale;
  n.block_scale = (float)block_scale;
  n.eps = (float)eps;
  n.offset = (float)offset;
  n.layer = layer;
  if (n.H > 0 || n.T > 0) {
    const c10::DeviceGuard on(dev);
    const hipStream_t st = c10::hip::getCurrentHIPStream(dev.index()).stream();
    check_unlocked([&] { return mlora_block_norm(st, &n, code); });
  }
  return py::make_tuple(r, h);
}

}  // namespace

void bind_norm(py::module_ &m) { m.def("block_norm", &block_norm); }
