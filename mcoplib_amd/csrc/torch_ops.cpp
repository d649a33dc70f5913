// torch_ops.cpp -- the operator surfaces of the fused norm/quant path as a C++ torch extension
// (module mcoplib_amd._torch_ops) over the C ABI of libmcop_norm.so (include/mcop_norm.h).
//
// Two surfaces, as the reference builds them in C++:
//   - mcoplib.op (pybind, op/pybind.cpp:42-44, 51, 54, 55): rms_norm_dynamic_per_token_quant
//     (fused_rms_norm_dq), rms_norm_dynamic_per_token_quant_custom, scale_dynamic_quant,
//     fused_add_rms_norm_dynamic_per_token_quant_padding_output, rms_norm, head_rms_norm;
//   - torch.ops._C (TORCH_LIBRARY, op/vllm/torch_bindings.cpp:155-164, 216-229, 359-364,
//     374-379): rms_norm, fused_add_rms_norm, rms_norm_dynamic_per_token_quant,
//     rms_norm_per_block_quant, dynamic_scaled_int8_quant, dynamic_per_token_scaled_fp8_quant,
//     registered by register_vllm_ops() for the CUDA (HIP) key, plus a no-op Meta kernel;
//     and, of the same kind without a counterpart in the reference, the 4-bit operators
//     (mxfp4_quant, mxfp4_dequant, rms_norm_mxfp4_quant, mxfp4_scaled_mm) and the quantized
//     key/value cache (kv_cache_write_quant, kv_cache_read_dequant, kv_cache_attention) with its
//     pages (kv_cache_copy_pages, kv_cache_fork, kv_cache_extend, kv_cache_free, kv_cache_compact).
// Every function checks its arguments as the reference does (TORCH_CHECK with the reference's
// condition text) and, beyond the reference, that every tensor is on the device and that element
// counts match (the kernels trust them); then it makes the input's device current and enqueues
// one kernel on torch's current stream of that device.  Nothing synchronizes.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/hip/HIPContext.h>
#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <torch/library.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "../../include/mcop_norm.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;

mcop_dtype code_of(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return MCOP_BF16;
    case at::kHalf: return MCOP_F16;
    case at::kFloat: return MCOP_F32;
    case at::kChar: return MCOP_I8;
    case at::kFloat8_e4m3fn: return MCOP_FP8_E4M3FN;
    default: TORCH_CHECK(false, "libmcop_norm: unsupported dtype ", t);
  }
}

void* stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}

void check_rc(int rc) {
  if (rc != MCOP_OK) TORCH_CHECK(false, mcop_last_error());
}

bool is_float_type(at::ScalarType t) {
  return t == at::kFloat || t == at::kHalf || t == at::kBFloat16;
}

// The error AT_DISPATCH_* raises for a dtype outside its list.
void dispatch_check(at::ScalarType t, const char* name) {
  TORCH_CHECK(is_float_type(t), '"', name, "\" not implemented for '", c10::toString(t), "'");
}

void on_device(const char* name, std::initializer_list<const Tensor*> ts) {
  const Tensor* first = nullptr;
  for (const Tensor* t : ts) {
    if (t == nullptr || !t->defined()) continue;
    TORCH_CHECK(t->is_cuda(), name, ": all tensors must be on a CUDA (HIP) device, got ",
                t->device());
    if (first == nullptr) {
      first = t;
    } else {
      TORCH_CHECK(t->device() == first->device(), name, ": tensors on different devices (",
                  first->device(), " and ", t->device(), ")");
    }
  }
}

const Tensor* opt(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }

void numel_check(const char* name, const char* what, const Tensor& t, int64_t n) {
  TORCH_CHECK(t.numel() == n, name, ": ", what, " has ", t.numel(), " elements, expected ", n);
}

void contiguous_check(const char* name, const char* what, const Tensor& t) {
  TORCH_CHECK(t.is_contiguous(), name, ": ", what, " must be contiguous");
}

// (num_tokens, hidden_size) of a [..., hidden_size] tensor (numel / size(-1), as the reference)
std::pair<int64_t, int64_t> rows_of(const Tensor& t) {
  TORCH_CHECK(t.dim() > 0, "expected a tensor with at least one dimension");
  const int64_t h = t.size(-1);
  TORCH_CHECK(h > 0, "hidden_size (the last dimension) must be positive");
  return {t.numel() / h, h};
}

// Element stride between the rows of t, for tensors whose rows are uniformly strided.  Dimensions of
// size one may have any stride and say nothing of the others'.
int64_t row_stride(const char* name, const Tensor& t, int64_t T, int64_t H) {
  if (T <= 1) return H;
  int64_t stride = 0, rows = 0;  // of the dimensions so far, the last first
  for (int64_t d = t.dim() - 2; d >= 0; --d) {
    if (t.size(d) == 1) continue;
    TORCH_CHECK(rows == 0 || t.stride(d) == stride * rows, name, ": rows must be uniformly strided");
    if (rows == 0) stride = t.stride(d);
    rows = (rows == 0 ? 1 : rows) * t.size(d);
  }
  return stride;
}

const float* ub_ptr(const char* name, const OptTensor& scale_ub) {
  if (!scale_ub.has_value()) return nullptr;
  TORCH_CHECK(scale_ub->scalar_type() == at::kFloat && scale_ub->numel() >= 1, name,
              ": scale_ub must be a float32 tensor with one element");
  return scale_ub->data_ptr<float>();
}

using DeviceGuard = c10::hip::OptionalHIPGuardMasqueradingAsCUDA;

// ------------------------------------------------------------------------ mcoplib.op surface

// Shared launcher of the (residual add +) RMSNorm + per-token quant kernel, vLLM's arithmetic or
// mcoplib's own (`custom`).
void norm_quant(const char* name, Tensor& out, const Tensor& input, const Tensor& weight,
                Tensor& scales, double eps, const OptTensor& scale_ub, const OptTensor& residual,
                bool custom) {
  on_device(name, {&out, &input, &weight, &scales, opt(scale_ub), opt(residual)});
  const auto [T, H] = rows_of(input);
  numel_check(name, "out", out, T * H);
  numel_check(name, "weight", weight, H);
  numel_check(name, "scales", scales, T);
  contiguous_check(name, "weight", weight);
  contiguous_check(name, "scales", scales);
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), name,
              ": weight must have the input dtype ", input.scalar_type());
  if (residual.has_value()) {
    TORCH_CHECK(residual->scalar_type() == input.scalar_type(), name,
                ": residual must have the input dtype ", input.scalar_type());
    contiguous_check(name, "residual", *residual);
    numel_check(name, "residual", *residual, T * H);
  }
  const float* ub = ub_ptr(name, scale_ub);
  void* rp = residual.has_value() ? residual->data_ptr() : nullptr;
  const DeviceGuard guard(input.device());
  if (custom) {
    check_rc(mcop_rms_norm_dynamic_per_token_quant_custom(
        static_cast<int8_t*>(out.data_ptr()), scales.data_ptr<float>(), input.data_ptr(),
        weight.data_ptr(), ub, rp, T, H, code_of(input.scalar_type()), (float)eps,
        stream_of(input)));
  } else {
    check_rc(mcop_rms_norm_dynamic_per_token_quant(
        out.data_ptr(), code_of(out.scalar_type()), scales.data_ptr<float>(), input.data_ptr(),
        weight.data_ptr(), ub, rp, T, H, code_of(input.scalar_type()), (float)eps,
        stream_of(input)));
  }
}

// op/fused_rms_norm_dq.cu:646-667 (pybind op/pybind.cpp:42)
void op_smooth_quant(Tensor& out, const Tensor& input, const Tensor& weight,
                     const Tensor& smooth_scale, Tensor& scales, double var_epsilon,
                     Tensor& after_res, Tensor& after_norm, const OptTensor& residual,
                     bool standard_norm) {
  const char* name = "rms_norm_dynamic_per_token_quant";
  TORCH_CHECK(out.scalar_type() == at::kChar || out.scalar_type() == at::kFloat8_e4m3fn,
              "Expected out.dtype() == torch::kInt8 || out.dtype() == torch::kFloat8_e4m3fn to "
              "be true, but got false.");
  TORCH_CHECK(out.is_contiguous() && input.is_contiguous(),
              "Expected out.is_contiguous() && input.is_contiguous() to be true, but got false.");
  TORCH_CHECK(scales.scalar_type() == at::kFloat,
              "Expected scales.dtype() == torch::kFloat32 to be true, but got false.");
  dispatch_check(input.scalar_type(), "rms_norm_dynamic_per_token_quant_dispatch");
  on_device(name, {&out, &input, &weight, &smooth_scale, &scales, &after_res, &after_norm,
                   opt(residual)});
  const auto [T, H] = rows_of(input);
  numel_check(name, "out", out, T * H);
  numel_check(name, "weight", weight, H);
  numel_check(name, "smooth_scale", smooth_scale, H);
  numel_check(name, "scales", scales, T);
  contiguous_check(name, "weight", weight);
  contiguous_check(name, "smooth_scale", smooth_scale);
  contiguous_check(name, "scales", scales);
  for (const auto& [what, t] : {std::pair<const char*, const Tensor*>{"after_res", &after_res},
                                {"after_norm", &after_norm}}) {
    contiguous_check(name, what, *t);
    numel_check(name, what, *t, T * H);
    TORCH_CHECK(t->scalar_type() == input.scalar_type(), name, ": ", what,
                " must have the input dtype ", input.scalar_type());
  }
  if (residual.has_value()) {
    TORCH_CHECK(residual->scalar_type() == input.scalar_type(), name,
                ": residual must have the input dtype ", input.scalar_type());
    contiguous_check(name, "residual", *residual);
    numel_check(name, "residual", *residual, T * H);
  }
  for (const auto& [what, t] : {std::pair<const char*, const Tensor*>{"weight", &weight},
                                {"smooth_scale", &smooth_scale}}) {
    TORCH_CHECK(t->scalar_type() == input.scalar_type() || t->scalar_type() == at::kFloat, name,
                ": ", what, " must be ", input.scalar_type(), " or float32, got ",
                t->scalar_type());
  }
  const DeviceGuard guard(input.device());
  check_rc(mcop_rms_norm_smooth_quant(
      out.data_ptr(), code_of(out.scalar_type()), scales.data_ptr<float>(), input.data_ptr(),
      weight.data_ptr(), code_of(weight.scalar_type()), smooth_scale.data_ptr(),
      code_of(smooth_scale.scalar_type()), after_res.data_ptr(), after_norm.data_ptr(),
      residual.has_value() ? residual->data_ptr() : nullptr, T, H,
      code_of(input.scalar_type()), (float)var_epsilon,
      standard_norm ? (uint32_t)MCOP_SQ_STANDARD_NORM : 0u, stream_of(input)));
}

// op/rms_norm_dynamic_per_token_quant.cu:266-285 (pybind op/pybind.cpp:55)
void op_custom(Tensor& out, const Tensor& input, const Tensor& weight, Tensor& scales,
               double var_epsilon, const OptTensor& scale_ub, const OptTensor& residual) {
  TORCH_CHECK(out.scalar_type() == at::kChar,
              "Expected out.dtype() == torch::kInt8 to be true, but got false.");
  TORCH_CHECK(out.is_contiguous() && input.is_contiguous(),
              "Expected out.is_contiguous() && input.is_contiguous() to be true, but got false.");
  TORCH_CHECK(scales.scalar_type() == at::kFloat,
              "Expected scales.dtype() == torch::kFloat32 to be true, but got false.");
  dispatch_check(input.scalar_type(), " rms_norm_dynamic_per_token_quant_dispatch_");
  norm_quant("rms_norm_dynamic_per_token_quant_custom", out, input, weight, scales, var_epsilon,
             scale_ub, residual, true);
}

// op/scale_dynamic_quant.cu:127-153 (pybind op/pybind.cpp:51): returns new (codes, scales [T])
std::tuple<Tensor, Tensor> op_scale_dynamic_quant(const Tensor& hidden_states,
                                                  const Tensor& smooth_scales,
                                                  py::object dst_dtype) {
  const char* name = "scale_dynamic_quant";
  TORCH_CHECK(hidden_states.is_cuda(), "Expected hidden_states.is_cuda() to be true, but got "
                                       "false.");
  TORCH_CHECK(smooth_scales.is_cuda(), "Expected smooth_scales.is_cuda() to be true, but got "
                                       "false.");
  const at::ScalarType dt = dst_dtype.is_none()
                                ? at::kChar
                                : torch::python::detail::py_object_to_dtype(dst_dtype);
  const auto [T, H] = rows_of(hidden_states);
  Tensor output = at::empty_like(hidden_states, hidden_states.options().dtype(dt));
  Tensor scales = at::empty({T}, smooth_scales.options());
  TORCH_CHECK(hidden_states.scalar_type() == at::kBFloat16 && dt == at::kChar,
              "Only support bfloat16");
  on_device(name, {&hidden_states, &smooth_scales});
  contiguous_check(name, "hidden_states", hidden_states);
  contiguous_check(name, "smooth_scales", smooth_scales);
  numel_check(name, "smooth_scales", smooth_scales, H);
  TORCH_CHECK(smooth_scales.scalar_type() == at::kFloat, name,
              ": smooth_scales must be float32");
  const DeviceGuard guard(hidden_states.device());
  check_rc(mcop_scale_dynamic_quant(static_cast<int8_t*>(output.data_ptr()),
                                    scales.data_ptr<float>(), hidden_states.data_ptr(),
                                    smooth_scales.data_ptr<float>(), T, H,
                                    stream_of(hidden_states)));
  return {output, scales};
}

// op/fused_add_layernorm_per_token_quant_padding_output.cu:397-416 (pybind op/pybind.cpp:54)
void op_padded(Tensor& output, Tensor& output_rms, Tensor& output_quant_int8, Tensor& out_scales,
               const Tensor& input, Tensor& residual, const Tensor& weight, int64_t pad_size,
               double epsilon) {
  const char* name = "fused_add_rms_norm_dynamic_per_token_quant_padding_output";
  TORCH_CHECK(output.scalar_type() == at::kChar,
              "Expected output.dtype() == torch::kInt8 to be true, but got false.");
  TORCH_CHECK(input.scalar_type() == at::kBFloat16,
              "Expected input.dtype() == at::ScalarType::BFloat16 to be true, but got false.");
  TORCH_CHECK(output.is_contiguous() && input.is_contiguous(),
              "Expected output.is_contiguous() && input.is_contiguous() to be true, but got "
              "false.");
  on_device(name, {&output, &output_rms, &output_quant_int8, &out_scales, &input, &residual,
                   &weight});
  const auto [T, H] = rows_of(input);
  TORCH_CHECK(2 * pad_size >= H + 4, name, ": a padded row of 2*pad_size = ", 2 * pad_size,
              " bytes cannot hold ", H, " codes and a 4-byte scale");
  numel_check(name, "output", output, T * 2 * pad_size);
  const std::tuple<const char*, const Tensor*, at::ScalarType> outs[] = {
      {"output_rms", &output_rms, at::kBFloat16},
      {"output_quant_int8", &output_quant_int8, at::kChar},
      {"residual", &residual, at::kBFloat16},
      {"weight", &weight, at::kBFloat16},
      {"out_scales", &out_scales, at::kFloat}};
  for (const auto& [what, t, want] : outs) {
    TORCH_CHECK(t->scalar_type() == want, name, ": ", what, " must be ", want, ", got ",
                t->scalar_type());
    contiguous_check(name, what, *t);
  }
  numel_check(name, "output_rms", output_rms, T * H);
  numel_check(name, "output_quant_int8", output_quant_int8, T * H);
  numel_check(name, "residual", residual, T * H);
  numel_check(name, "weight", weight, H);
  numel_check(name, "out_scales", out_scales, T);
  const DeviceGuard guard(input.device());
  check_rc(mcop_fused_add_rms_norm_dynamic_per_token_quant_padding_output(
      static_cast<int8_t*>(output.data_ptr()), output_rms.data_ptr(),
      static_cast<int8_t*>(output_quant_int8.data_ptr()), out_scales.data_ptr<float>(),
      input.data_ptr(), residual.data_ptr(), weight.data_ptr(), T, H, pad_size, (float)epsilon,
      stream_of(input)));
}

// The allocating forms behind mcoplib.custom_ops (mcoplib/custom_ops.py:7-45), whose outputs are
// new tensors: allocated here, a decode-sized call (1 x 5120) takes 5.8 us of the host, 7.1 with them
// allocated one by one in Python.
at::TensorOptions with_dtype(const Tensor& t, py::handle dtype) {
  return dtype.is_none() ? t.options()
                         : t.options().dtype(torch::python::detail::py_object_to_dtype(
                               py::reinterpret_borrow<py::object>(dtype)));
}

std::tuple<Tensor, Tensor> custom_new(const Tensor& input, const Tensor& weight, double epsilon,
                                      py::object quant_dtype, const OptTensor& scale_ub,
                                      const OptTensor& residual) {
  const at::TensorOptions opts = with_dtype(input, quant_dtype);
  Tensor out, scales;
  {
    const py::gil_scoped_release allocating;  // it may wait for the device
    out = at::empty_like(input, opts);
    scales = at::empty({rows_of(input).first, 1}, input.options().dtype(at::kFloat));
  }
  op_custom(out, input, weight, scales, epsilon, scale_ub, residual);
  return {out, scales};
}

std::tuple<Tensor, Tensor, Tensor, Tensor, Tensor> padded_new(const Tensor& input,
                                                              Tensor& residual,
                                                              const Tensor& weight,
                                                              int64_t pad_size, double epsilon) {
  const int64_t T = rows_of(input).first;
  std::vector<int64_t> shape = input.sizes().vec();
  shape.back() = pad_size;
  Tensor output, rms, q, scales;
  {
    const py::gil_scoped_release allocating;
    output = at::empty(shape, input.options().dtype(at::kBFloat16));
    rms = at::empty_like(input);
    q = at::empty_like(input, input.options().dtype(at::kChar));
    scales = at::empty({T, 1}, input.options().dtype(at::kFloat));
  }
  Tensor bytes = output.view(at::kChar);
  op_padded(bytes, rms, q, scales, input, residual, weight, pad_size, epsilon);
  return {output, residual, rms, q, scales};
}

// op/fused_rms_norm_dq.cu:980-998 (pybind op/pybind.cpp:44)
void op_rms_norm(Tensor& out, const Tensor& input, const Tensor& weight, double var_epsilon,
                 const OptTensor& after_res, const OptTensor& residual, bool rms_div) {
  const char* name = "rms_norm";
  TORCH_CHECK(out.is_contiguous() && input.is_contiguous(),
              "Expected out.is_contiguous() && input.is_contiguous() to be true, but got false.");
  TORCH_CHECK(weight.is_contiguous(), "Expected weight.is_contiguous() to be true, but got "
                                      "false.");
  dispatch_check(input.scalar_type(), "rms_norm_per_token_dispatch");
  on_device(name, {&out, &input, &weight, opt(after_res), opt(residual)});
  const auto [T, H] = rows_of(input);
  TORCH_CHECK(out.scalar_type() == input.scalar_type(), name,
              ": out must have the input dtype ", input.scalar_type());
  TORCH_CHECK(weight.scalar_type() == input.scalar_type() || weight.scalar_type() == at::kFloat,
              name, ": weight must be ", input.scalar_type(), " or float32, got ",
              weight.scalar_type());
  numel_check(name, "out", out, T * H);
  numel_check(name, "weight", weight, H);
  if (residual.has_value()) {
    TORCH_CHECK(after_res.has_value(), name, ": a residual needs an after_res output");
    for (const auto& [what, t] : {std::pair<const char*, const Tensor*>{"residual", &*residual},
                                  {"after_res", &*after_res}}) {
      TORCH_CHECK(t->scalar_type() == input.scalar_type(), name, ": ", what,
                  " must have the input dtype ", input.scalar_type());
      contiguous_check(name, what, *t);
      numel_check(name, what, *t, T * H);
    }
  }
  const DeviceGuard guard(input.device());
  check_rc(mcop_rms_norm(out.data_ptr(), input.data_ptr(), weight.data_ptr(),
                         code_of(weight.scalar_type()),
                         residual.has_value() ? after_res->data_ptr() : nullptr,
                         residual.has_value() ? residual->data_ptr() : nullptr, T, H,
                         code_of(input.scalar_type()), (float)var_epsilon, rms_div ? 1 : 0,
                         stream_of(input)));
}

// op/fused_rms_norm_dq.cu:804-812 (pybind op/pybind.cpp:43)
void op_head_rms_norm(Tensor& out, const Tensor& hidden_states, const Tensor& weight,
                      double var_epsilon, int64_t head_offset, int64_t head_norm) {
  const char* name = "head_rms_norm";
  TORCH_CHECK(out.is_contiguous() && weight.is_contiguous() && hidden_states.is_contiguous(),
              "Expected out.is_contiguous() && weight.is_contiguous() && "
              "hidden_states.is_contiguous() to be true, but got false.");
  dispatch_check(hidden_states.scalar_type(), "head_rms_norm_dispatch");
  on_device(name, {&out, &hidden_states, &weight});
  TORCH_CHECK(hidden_states.dim() == 3, name,
              ": hidden_states must be [num_tokens, num_heads, head_size]");
  const int64_t T = hidden_states.size(0), NH = hidden_states.size(1),
                D = hidden_states.size(2);
  TORCH_CHECK(out.sizes() == hidden_states.sizes() &&
                  out.scalar_type() == hidden_states.scalar_type(),
              name, ": out must match hidden_states in shape and dtype");
  TORCH_CHECK(weight.scalar_type() == at::kBFloat16 || weight.scalar_type() == at::kFloat, name,
              ": weight must be bfloat16 or float32, got ", weight.scalar_type());
  TORCH_CHECK(head_offset >= 0 && head_norm >= 0 && head_offset + head_norm <= NH, name,
              ": heads [", head_offset, ", ", head_offset + head_norm,
              ") are not inside the ", NH, " heads");
  TORCH_CHECK(weight.numel() >= (head_offset + head_norm) * D, name, ": weight holds ",
              weight.numel(), " elements, needs ", (head_offset + head_norm) * D);
  const DeviceGuard guard(hidden_states.device());
  check_rc(mcop_head_rms_norm(out.data_ptr(), hidden_states.data_ptr(), weight.data_ptr(),
                              code_of(weight.scalar_type()), T, NH, D, head_offset, head_norm,
                              code_of(hidden_states.scalar_type()), (float)var_epsilon,
                              stream_of(hidden_states)));
}

// ------------------------------------------------------------------------- torch.ops._C surface

// op/vllm/layernorm_kernels.cu:186-231
void c_rms_norm(Tensor& result, const Tensor& input_arg, const Tensor& weight, double epsilon) {
  const char* name = "rms_norm";
  TORCH_CHECK(result.is_contiguous(), "Expected out.is_contiguous() to be true, but got false.");
  const Tensor input = input_arg.stride(-1) == 1 ? input_arg : input_arg.contiguous();
  TORCH_CHECK(weight.is_contiguous(), "Expected weight.is_contiguous() to be true, but got "
                                      "false.");
  dispatch_check(input.scalar_type(), "rms_norm_kernel");
  const int64_t nd = input.dim();
  TORCH_CHECK(nd == 2 || nd == 3 || nd == 4, "Expects rank 2, 3 or 4 tensors but got ", nd);
  TORCH_CHECK(weight.scalar_type() == input.scalar_type() &&
                  result.scalar_type() == input.scalar_type(),
              name, ": result, input and weight must share one dtype");
  on_device(name, {&result, &input, &weight});
  const auto [T, H] = rows_of(input);
  numel_check(name, "result", result, T * H);
  numel_check(name, "weight", weight, H);
  const DeviceGuard guard(input.device());
  check_rc(mcop_vllm_rms_norm(result.data_ptr(), input.data_ptr(), weight.data_ptr(), T, H,
                              (int)nd, input.stride(-2), nd >= 3 ? input.stride(-3) : 0,
                              nd >= 4 ? input.stride(-4) : 0, nd >= 3 ? input.size(-2) : 0,
                              nd >= 4 ? input.size(-3) : 0, code_of(input.scalar_type()),
                              (float)epsilon, stream_of(input)));
}

// op/vllm/layernorm_kernels.cu:243-292
void c_fused_add_rms_norm(Tensor& input, Tensor& residual, const Tensor& weight, double epsilon) {
  const char* name = "fused_add_rms_norm";
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(),
              "Expected weight.scalar_type() == input.scalar_type() to be true, but got false.");
  TORCH_CHECK(input.scalar_type() == residual.scalar_type(),
              "Expected input.scalar_type() == residual.scalar_type() to be true, but got false.");
  TORCH_CHECK(residual.is_contiguous(), "Expected residual.is_contiguous() to be true, but got "
                                        "false.");
  TORCH_CHECK(weight.is_contiguous(), "Expected weight.is_contiguous() to be true, but got "
                                      "false.");
  dispatch_check(input.scalar_type(), "fused_add_rms_norm_kernel");
  on_device(name, {&input, &residual, &weight});
  const auto [T, H] = rows_of(input);
  numel_check(name, "residual", residual, T * H);
  numel_check(name, "weight", weight, H);
  // rows of `input` are addressed as row * stride, its stride(-2) (the reference's input_stride) unless
  // that dimension has one row
  TORCH_CHECK(T <= 1 || input.stride(-1) == 1, name,
              ": input must be contiguous in its last dimension");
  const int64_t stride = row_stride(name, input, T, H);
  const DeviceGuard guard(input.device());
  check_rc(mcop_fused_add_rms_norm(input.data_ptr(), stride, residual.data_ptr(),
                                   weight.data_ptr(), T, H, code_of(input.scalar_type()),
                                   (float)epsilon, stream_of(input)));
}

void quant_out_checks(const Tensor& result, const Tensor& input, const Tensor& weight,
                      const Tensor& scale, const OptTensor& scale_ub, const OptTensor& residual) {
  TORCH_CHECK(result.scalar_type() == at::kFloat8_e4m3fn || result.scalar_type() == at::kChar,
              "Expected out.dtype() == kFp8Type || out.dtype() == torch::kInt8 to be true, but "
              "got false.");
  TORCH_CHECK(result.is_contiguous() && input.is_contiguous(),
              "Expected out.is_contiguous() && input.is_contiguous() to be true, but got false.");
  if (scale_ub.has_value()) {
    TORCH_CHECK(result.scalar_type() == at::kFloat8_e4m3fn,
                "Expected out.dtype() == kFp8Type to be true, but got false.");
  }
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(),
              "Expected weight.dtype() == input.dtype() to be true, but got false.");
  TORCH_CHECK(scale.scalar_type() == at::kFloat,
              "Expected scales.dtype() == torch::kFloat32 to be true, but got false.");
  if (residual.has_value()) {
    TORCH_CHECK(residual->scalar_type() == input.scalar_type(),
                "Expected residual->scalar_type() == input.scalar_type() to be true, but got "
                "false.");
  }
}

// op/vllm/quantization/fused_kernels/fused_layernorm_dynamic_per_token_quant.cu:163-192
void c_norm_quant(Tensor& result, const Tensor& input, const Tensor& weight, Tensor& scale,
                  double epsilon, const OptTensor& scale_ub, const OptTensor& residual) {
  quant_out_checks(result, input, weight, scale, scale_ub, residual);
  dispatch_check(input.scalar_type(), "rms_norm_dynamic_per_token_quant_dispatch");
  norm_quant("rms_norm_dynamic_per_token_quant", result, input, weight, scale, epsilon, scale_ub,
             residual, false);
}

// op/vllm/quantization/fused_kernels/fused_layernorm_dynamic_per_token_quant.cu:238-270
void c_per_block_quant(Tensor& result, const Tensor& input, const Tensor& weight, Tensor& scale,
                       double epsilon, const OptTensor& scale_ub, const OptTensor& residual,
                       int64_t group_size, bool is_scale_transposed) {
  const char* name = "rms_norm_per_block_quant";
  quant_out_checks(result, input, weight, scale, scale_ub, residual);
  TORCH_CHECK(group_size == 64 || group_size == 128, "Unsupported group size: ", group_size);
  dispatch_check(input.scalar_type(), "rms_norm_per_block_quant_fp_dispatch");
  on_device(name, {&result, &input, &weight, &scale, opt(scale_ub), opt(residual)});
  const auto [T, H] = rows_of(input);
  TORCH_CHECK(H % group_size == 0, name, ": hidden_size ", H,
              " is not a multiple of group_size ", group_size);
  numel_check(name, "result", result, T * H);
  numel_check(name, "weight", weight, H);
  numel_check(name, "scale", scale, T * (H / group_size));
  contiguous_check(name, "weight", weight);
  contiguous_check(name, "scale", scale);
  if (residual.has_value()) {
    contiguous_check(name, "residual", *residual);
    numel_check(name, "residual", *residual, T * H);
  }
  const float* ub = ub_ptr(name, scale_ub);
  const DeviceGuard guard(input.device());
  check_rc(mcop_rms_norm_per_block_quant(
      result.data_ptr(), code_of(result.scalar_type()), scale.data_ptr<float>(),
      input.data_ptr(), weight.data_ptr(), ub,
      residual.has_value() ? residual->data_ptr() : nullptr, T, H, code_of(input.scalar_type()),
      (float)epsilon, group_size, is_scale_transposed ? 1 : 0, stream_of(input)));
}

// op/vllm/quantization/compressed_tensors/int8_quant_kernels.cu:459-527
void c_int8_quant(Tensor& result, const Tensor& input, Tensor& scale, const OptTensor& azp) {
  const char* name = "dynamic_scaled_int8_quant";
  TORCH_CHECK(input.is_contiguous(), "Expected input.is_contiguous() to be true, but got false.");
  TORCH_CHECK(result.is_contiguous(), "Expected out.is_contiguous() to be true, but got false.");
  TORCH_CHECK(scale.is_contiguous(), "Expected scales.is_contiguous() to be true, but got "
                                     "false.");
  TORCH_CHECK(!azp.has_value() || azp->is_contiguous(),
              "Expected !azp || azp->is_contiguous() to be true, but got false.");
  dispatch_check(input.scalar_type(), "dynamic_scaled_int8_quant_kernel");
  TORCH_CHECK(result.scalar_type() == at::kChar, "expected scalar type Char but found ",
              result.scalar_type());
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "expected scalar type Float but found ",
              scale.scalar_type());
  if (azp.has_value()) {
    TORCH_CHECK(azp->scalar_type() == at::kInt, "expected scalar type Int but found ",
                azp->scalar_type());
  }
  on_device(name, {&result, &input, &scale, opt(azp)});
  const auto [T, H] = rows_of(input);
  numel_check(name, "result", result, T * H);
  numel_check(name, "scale", scale, T);
  if (azp.has_value()) numel_check(name, "azp", *azp, T);
  const DeviceGuard guard(input.device());
  check_rc(mcop_dynamic_scaled_int8_quant(
      static_cast<int8_t*>(result.data_ptr()), scale.data_ptr<float>(),
      azp.has_value() ? azp->data_ptr<int32_t>() : nullptr, input.data_ptr(), T, H,
      code_of(input.scalar_type()), stream_of(input)));
}

// op/vllm/quantization/fp8/common.cu:375-411
void c_fp8_quant(Tensor& result, const Tensor& input, Tensor& scale, const OptTensor& scale_ub) {
  const char* name = "dynamic_per_token_scaled_fp8_quant";
  TORCH_CHECK(input.stride(-1) == 1, "last dimension of input must be contiguous");
  TORCH_CHECK(result.stride(-1) == 1, "last dimension of output must be contiguous");
  dispatch_check(input.scalar_type(), "dynamic_per_token_scaled_fp8_quant_kernel_scalar_type");
  TORCH_CHECK(result.scalar_type() == at::kFloat8_e4m3fn,
              "\"dynamic_per_token_scaled_fp8_quant_kernel_fp8_type\" not implemented for '",
              c10::toString(result.scalar_type()), "'");
  TORCH_CHECK(scale.scalar_type() == at::kFloat, "expected scalar type Float but found ",
              scale.scalar_type());
  on_device(name, {&result, &input, &scale, opt(scale_ub)});
  const auto [T, H] = rows_of(input);
  TORCH_CHECK(result.sizes() == input.sizes(), name, ": result shape ", result.sizes(),
              " != input shape ", input.sizes());
  numel_check(name, "scale", scale, T);
  contiguous_check(name, "scale", scale);
  const float* ub = ub_ptr(name, scale_ub);
  const int64_t in_stride = row_stride(name, input, T, H);
  const int64_t out_stride = row_stride(name, result, T, H);
  const DeviceGuard guard(input.device());
  check_rc(mcop_dynamic_per_token_scaled_fp8_quant(
      static_cast<uint8_t*>(result.data_ptr()), scale.data_ptr<float>(), input.data_ptr(), ub, T,
      H, in_stride, out_stride, code_of(input.scalar_type()), stream_of(input)));
}

// ------------------------------------------------- 4-bit operators, quantized key/value cache
// (no counterpart in the reference; shapes and dtypes are checked before devices)

constexpr int64_t kMxBlock = 32;

bool is_codes4(at::ScalarType t) { return t == at::kByte || t == at::kFloat4_e2m1fn_x2; }
bool is_scale8(at::ScalarType t) { return t == at::kByte || t == at::kFloat8_e8m0fnu; }

// Codes and scales of rows of H values: [..., H / 2] and [..., H / 32], contiguous.
void mx_check(const char* name, const char* what, const Tensor& codes, const Tensor& scale,
              int64_t T, int64_t H) {
  TORCH_CHECK(H % kMxBlock == 0, name, ": the last dimension, ", H,
              " values, is not a multiple of the block of 32");
  TORCH_CHECK(is_codes4(codes.scalar_type()), name, ": ", what,
              " must be uint8 or float4_e2m1fn_x2, got ", codes.scalar_type());
  TORCH_CHECK(is_scale8(scale.scalar_type()), name, ": the scale of ", what,
              " must be uint8 or float8_e8m0fnu, got ", scale.scalar_type());
  TORCH_CHECK(codes.dim() > 0 && codes.size(-1) == H / 2 && codes.numel() == T * (H / 2), name,
              ": ", what, " has shape ", codes.sizes(), ", expected ", T, " rows of ", H / 2);
  TORCH_CHECK(scale.dim() > 0 && scale.size(-1) == H / kMxBlock &&
                  scale.numel() == T * (H / kMxBlock),
              name, ": the scale of ", what, " has shape ", scale.sizes(), ", expected ", T,
              " rows of ", H / kMxBlock);
  contiguous_check(name, what, codes);
  TORCH_CHECK(scale.is_contiguous(), name, ": the scale of ", what, " must be contiguous");
}

uint8_t* bytes_of(const Tensor& t) { return static_cast<uint8_t*>(t.data_ptr()); }

void c_mxfp4_quant(Tensor& result, const Tensor& input, Tensor& scale) {
  const char* name = "mxfp4_quant";
  dispatch_check(input.scalar_type(), name);
  const auto [T, H] = rows_of(input);
  TORCH_CHECK(input.stride(-1) == 1, name, ": last dimension of input must be contiguous");
  const int64_t stride = row_stride(name, input, T, H);
  mx_check(name, "result", result, scale, T, H);
  on_device(name, {&result, &input, &scale});
  const DeviceGuard guard(input.device());
  check_rc(mcop_mxfp4_quant(bytes_of(result), bytes_of(scale), input.data_ptr(), T, H, stride,
                            code_of(input.scalar_type()), stream_of(input)));
}

void c_mxfp4_dequant(Tensor& result, const Tensor& input, const Tensor& scale) {
  const char* name = "mxfp4_dequant";
  dispatch_check(result.scalar_type(), name);
  const auto [T, H] = rows_of(result);
  contiguous_check(name, "result", result);
  mx_check(name, "input", input, scale, T, H);
  on_device(name, {&result, &input, &scale});
  const DeviceGuard guard(input.device());
  check_rc(mcop_mxfp4_dequant(result.data_ptr(), code_of(result.scalar_type()), bytes_of(input),
                              bytes_of(scale), T, H, stream_of(input)));
}

void c_rms_norm_mxfp4_quant(Tensor& result, const Tensor& input, const Tensor& weight,
                            Tensor& scale, double epsilon, const OptTensor& residual,
                            const OptTensor& after_res) {
  const char* name = "rms_norm_mxfp4_quant";
  dispatch_check(input.scalar_type(), name);
  const auto [T, H] = rows_of(input);
  contiguous_check(name, "input", input);
  contiguous_check(name, "weight", weight);
  numel_check(name, "weight", weight, H);
  TORCH_CHECK(weight.scalar_type() == input.scalar_type(), name,
              ": weight must have the input dtype ", input.scalar_type());
  TORCH_CHECK(residual.has_value() == after_res.has_value(), name,
              ": residual and after_res go together");
  if (residual.has_value()) {
    for (const auto& [what, t] : {std::pair<const char*, const Tensor*>{"residual", &*residual},
                                  {"after_res", &*after_res}}) {
      TORCH_CHECK(t->scalar_type() == input.scalar_type(), name, ": ", what,
                  " must have the input dtype ", input.scalar_type());
      contiguous_check(name, what, *t);
      numel_check(name, what, *t, T * H);
    }
  }
  mx_check(name, "result", result, scale, T, H);
  on_device(name, {&result, &input, &weight, &scale, opt(residual), opt(after_res)});
  const DeviceGuard guard(input.device());
  check_rc(mcop_rms_norm_mxfp4_quant(
      bytes_of(result), bytes_of(scale), input.data_ptr(), weight.data_ptr(),
      residual.has_value() ? residual->data_ptr() : nullptr,
      after_res.has_value() ? after_res->data_ptr() : nullptr, T, H,
      code_of(input.scalar_type()), (float)epsilon, stream_of(input)));
}

void c_mxfp4_scaled_mm(Tensor& result, const Tensor& a, const Tensor& a_scale, const Tensor& b,
                       const Tensor& b_scale, const OptTensor& bias) {
  const char* name = "mxfp4_scaled_mm";
  dispatch_check(result.scalar_type(), name);
  const auto [M, half] = rows_of(a);
  const int64_t K = half * 2;
  mx_check(name, "a", a, a_scale, M, K);
  TORCH_CHECK(b.dim() == 2, name, ": b must be [N, K / 2], got ", b.sizes());
  const int64_t N = b.size(0);
  mx_check(name, "b", b, b_scale, N, K);
  TORCH_CHECK(result.dim() > 0 && result.size(-1) == N && result.numel() == M * N, name,
              ": result has shape ", result.sizes(), ", expected ", M, " rows of ", N);
  contiguous_check(name, "result", result);
  if (bias.has_value()) {
    TORCH_CHECK(bias->scalar_type() == result.scalar_type(), name,
                ": bias must have the result dtype ", result.scalar_type());
    numel_check(name, "bias", *bias, N);
    contiguous_check(name, "bias", *bias);
  }
  on_device(name, {&result, &a, &a_scale, &b, &b_scale, opt(bias)});
  const DeviceGuard guard(a.device());
  check_rc(mcop_mxfp4_scaled_mm(result.data_ptr(), code_of(result.scalar_type()), bytes_of(a),
                                bytes_of(a_scale), bytes_of(b), bytes_of(b_scale),
                                bias.has_value() ? bias->data_ptr() : nullptr, M, N, K,
                                stream_of(a)));
}

mcop_dtype cache_code(const char* name, at::ScalarType t) {
  if (t == at::kChar) return MCOP_I8;
  if (t == at::kFloat8_e4m3fn) return MCOP_FP8_E4M3FN;
  TORCH_CHECK(is_codes4(t), name, ": the cache must be int8, float8_e4m3fn or (4-bit codes) uint8 "
              "or float4_e2m1fn_x2, got ", t);
  return MCOP_MXFP4;
}

// One side of the cache and the plain tensor [tokens, heads, head_size] beside it, whose heads are `group`
// times the cache's.
mcop_kv_side kv_side(const char* name, const char* what, const Tensor& plain, const Tensor& cache,
                     const Tensor& scale, mcop_dtype format, const Tensor& key_cache,
                     int64_t group = 1) {
  TORCH_CHECK(plain.dim() == 3, name, ": ", what, " must be [tokens, heads, head_size], got ",
              plain.sizes());
  TORCH_CHECK(cache.dim() == 4, name, ": the cache of ", what,
              " must be [pages, page_size, heads, head_size], got ", cache.sizes());
  const int64_t D = plain.size(2);
  const bool four = format == MCOP_MXFP4;
  TORCH_CHECK(!four || D % kMxBlock == 0, name, ": head_size ", D, " of ", what,
              " is not a multiple of the block of 32");
  TORCH_CHECK(cache.size(3) == (four ? D / 2 : D) && cache.size(2) * group == plain.size(1), name,
              ": the cache of ", what, " has shape ", cache.sizes(), " beside ", plain.sizes());
  TORCH_CHECK(cache.size(0) == key_cache.size(0) && cache.size(1) == key_cache.size(1) &&
                  cache.size(2) == key_cache.size(2),
              name, ": the caches' shapes differ: ", key_cache.sizes(), " and ", cache.sizes());
  TORCH_CHECK(scale.dim() == (four ? 4 : 3) && scale.size(0) == cache.size(0) &&
                  scale.size(1) == cache.size(1) && scale.size(2) == cache.size(2) &&
                  (!four || scale.size(3) == D / kMxBlock),
              name, ": the scale of ", what, " has shape ", scale.sizes(), " beside a cache of ",
              cache.sizes());
  TORCH_CHECK(four ? is_scale8(scale.scalar_type()) : scale.scalar_type() == at::kFloat, name,
              ": the scale of ", what, " must be ",
              four ? "uint8 or float8_e8m0fnu" : "float32", ", got ", scale.scalar_type());
  TORCH_CHECK((plain.stride(2) == 1 || D == 1) && (cache.stride(3) == 1 || cache.size(3) == 1) &&
                  (!four || scale.stride(3) == 1 || scale.size(3) == 1),
              name, ": last dimension of ", what, ", its cache and its scale must be contiguous");
  return mcop_kv_side{plain.data_ptr(), plain.stride(0),  plain.stride(1),
                      cache.data_ptr(), cache.stride(0),  cache.stride(1), cache.stride(2),
                      scale.data_ptr(), scale.stride(0),  scale.stride(1), scale.stride(2),
                      D};
}

void no_overlap(const char* name, std::initializer_list<const Tensor*> outputs) {
  for (const Tensor* t : outputs) {
    TORCH_CHECK(at::has_internal_overlap(*t) != at::MemOverlap::Yes, name,
                ": a tensor that is written has elements that share memory");
  }
}

void kv_check(const char* name, const Tensor& key, const Tensor& value, const Tensor& key_cache,
              const Tensor& value_cache) {
  dispatch_check(key.scalar_type(), name);
  TORCH_CHECK(value.scalar_type() == key.scalar_type(), name, ": value must have key's dtype ",
              key.scalar_type());
  TORCH_CHECK(value_cache.scalar_type() == key_cache.scalar_type(), name,
              ": the caches must share a dtype, got ", key_cache.scalar_type(), " and ",
              value_cache.scalar_type());
  TORCH_CHECK(key.dim() == 3 && value.dim() == 3 && key.size(0) == value.size(0) &&
                  key.size(1) == value.size(1) && key.size(1) > 0 && key_cache.dim() == 4,
              name, ": key ", key.sizes(), " and value ", value.sizes(),
              " must be [tokens, heads, head_size] of the same tokens and heads");
}

template <class T>
const T* index_ptr(const char* name, const char* what, const Tensor& t, at::ScalarType type) {
  TORCH_CHECK(t.scalar_type() == type, name, ": ", what, " must be ", c10::toString(type),
              ", got ", t.scalar_type());
  return static_cast<const T*>(t.data_ptr());
}

const int32_t* table_ptr(const char* name, const Tensor& block_table) {
  const auto* table = index_ptr<int32_t>(name, "block_table", block_table, at::kInt);
  TORCH_CHECK(block_table.dim() == 2 && (block_table.size(1) <= 1 || block_table.stride(1) == 1),
              name, ": block_table must be [sequences, pages] with contiguous rows");
  return table;
}

// A contiguous vector of int32, of n elements (n < 0: any number).
int32_t* ints_ptr(const char* name, const char* what, const Tensor& t, int64_t n) {
  auto* p = const_cast<int32_t*>(index_ptr<int32_t>(name, what, t, at::kInt));
  TORCH_CHECK(t.dim() == 1 && t.is_contiguous() && (n < 0 || t.size(0) == n), name, ": ", what,
              " must be contiguous with ", n < 0 ? std::string("one dimension") :
              std::to_string(n) + " elements", ", got ", t.sizes());
  return p;
}

void c_kv_cache_write_quant(const Tensor& key, const Tensor& value, Tensor& key_cache,
                            Tensor& value_cache, Tensor& key_scale, Tensor& value_scale,
                            const Tensor& slot_mapping) {
  const char* name = "kv_cache_write_quant";
  kv_check(name, key, value, key_cache, value_cache);
  const mcop_dtype format = cache_code(name, key_cache.scalar_type());
  const auto* slots = index_ptr<int64_t>(name, "slot_mapping", slot_mapping, at::kLong);
  TORCH_CHECK(slot_mapping.dim() == 1 && slot_mapping.is_contiguous() &&
                  slot_mapping.size(0) <= key.size(0),
              name, ": slot_mapping must be contiguous with at most one slot a token, got ",
              slot_mapping.sizes(), " for ", key.size(0), " tokens");
  const mcop_kv_side k = kv_side(name, "key", key, key_cache, key_scale, format, key_cache);
  const mcop_kv_side v = kv_side(name, "value", value, value_cache, value_scale, format,
                                 key_cache);
  no_overlap(name, {&key_cache, &value_cache, &key_scale, &value_scale});
  on_device(name, {&key, &value, &key_cache, &value_cache, &key_scale, &value_scale,
                   &slot_mapping});
  const DeviceGuard guard(key.device());
  check_rc(mcop_kv_cache_write_quant(&k, &v, format, key_cache.size(0), key_cache.size(1),
                                     key.size(1), slots, slot_mapping.size(0),
                                     code_of(key.scalar_type()), stream_of(key)));
}

void c_kv_cache_read_dequant(Tensor& key, Tensor& value, const Tensor& key_cache,
                             const Tensor& value_cache, const Tensor& key_scale,
                             const Tensor& value_scale, const Tensor& block_table,
                             const Tensor& cu_seqlens, const OptTensor& seq_starts) {
  const char* name = "kv_cache_read_dequant";
  kv_check(name, key, value, key_cache, value_cache);
  const mcop_dtype format = cache_code(name, key_cache.scalar_type());
  const auto* table = table_ptr(name, block_table);
  const auto* cu = index_ptr<int32_t>(name, "cu_seqlens", cu_seqlens, at::kInt);
  const int64_t B = block_table.size(0);
  TORCH_CHECK(cu_seqlens.dim() == 1 && cu_seqlens.is_contiguous() && cu_seqlens.size(0) == B + 1,
              name, ": cu_seqlens must be contiguous with ", B + 1, " elements, got ",
              cu_seqlens.sizes());
  const int32_t* starts = nullptr;
  if (seq_starts.has_value()) {
    starts = index_ptr<int32_t>(name, "seq_starts", *seq_starts, at::kInt);
    TORCH_CHECK(seq_starts->dim() == 1 && seq_starts->is_contiguous() && seq_starts->size(0) == B,
                name, ": seq_starts must be contiguous with ", B, " elements, got ",
                seq_starts->sizes());
  }
  const mcop_kv_side k = kv_side(name, "key", key, key_cache, key_scale, format, key_cache);
  const mcop_kv_side v = kv_side(name, "value", value, value_cache, value_scale, format,
                                 key_cache);
  no_overlap(name, {&key, &value});
  on_device(name, {&key, &value, &key_cache, &value_cache, &key_scale, &value_scale, &block_table,
                   &cu_seqlens, opt(seq_starts)});
  const DeviceGuard guard(key.device());
  check_rc(mcop_kv_cache_read_dequant(&k, &v, format, key_cache.size(0), key_cache.size(1),
                                      key.size(1), table, B > 1 ? block_table.stride(0) : 0,
                                      block_table.size(1), cu, starts, B, key.size(0),
                                      code_of(key.scalar_type()), stream_of(key)));
}

void c_kv_cache_attention(Tensor& result, const Tensor& query, const Tensor& key_cache,
                          const Tensor& value_cache, const Tensor& key_scale,
                          const Tensor& value_scale, const Tensor& block_table,
                          const Tensor& seq_lens, double scale, int64_t window,
                          const OptTensor& lse) {
  const char* name = "kv_cache_attention";
  dispatch_check(query.scalar_type(), name);
  TORCH_CHECK(result.scalar_type() == query.scalar_type(), name, ": result must have query's dtype ",
              query.scalar_type());
  TORCH_CHECK(value_cache.scalar_type() == key_cache.scalar_type(), name,
              ": the caches must share a dtype, got ", key_cache.scalar_type(), " and ",
              value_cache.scalar_type());
  TORCH_CHECK(query.dim() == 3 && result.dim() == 3 && query.size(0) == result.size(0) &&
                  query.size(1) == result.size(1) && key_cache.dim() == 4,
              name, ": query ", query.sizes(), " and result ", result.sizes(),
              " must be [sequences, heads, head_size] of the same sequences and heads");
  const int64_t B = query.size(0), heads = key_cache.size(2), queries = query.size(1);
  TORCH_CHECK(heads > 0 && queries > 0 && queries % heads == 0, name, ": ", queries,
              " query heads are not a multiple of ", heads, " key heads");
  const mcop_dtype format = cache_code(name, key_cache.scalar_type());
  const auto* table = table_ptr(name, block_table);
  TORCH_CHECK(block_table.size(0) == B, name, ": block_table has ", block_table.size(0),
              " rows for ", B, " sequences");
  const auto* lens = ints_ptr(name, "seq_lens", seq_lens, B);
  TORCH_CHECK(window >= 0, name, ": window must not be negative, got ", window);
  if (lse.has_value()) {
    TORCH_CHECK(lse->scalar_type() == at::kFloat && lse->dim() == 2 && lse->size(0) == B &&
                    lse->size(1) == queries && lse->is_contiguous(),
                name, ": lse must be contiguous float32 [", B, ", ", queries, "], got ",
                lse->scalar_type(), " ", lse->sizes());
  }
  const mcop_kv_side k = kv_side(name, "key", query, key_cache, key_scale, format, key_cache,
                                 queries / heads);
  const mcop_kv_side v = kv_side(name, "value", result, value_cache, value_scale, format, key_cache,
                                 queries / heads);
  no_overlap(name, {&result});
  on_device(name, {&result, &query, &key_cache, &value_cache, &key_scale, &value_scale, &block_table,
                   &seq_lens, opt(lse)});
  if (B == 0) return;
  const DeviceGuard guard(query.device());
  const int64_t bytes = mcop_kv_cache_attention_workspace(heads, queries, v.head_size);
  if (bytes < 0) check_rc((int)bytes);
  // from torch's allocator: the memory stays this stream's (and a captured graph's own) until reused
  const Tensor workspace = at::empty({bytes}, query.options().dtype(at::kByte));
  check_rc(mcop_kv_cache_attention(&k, &v, format, key_cache.size(0), key_cache.size(1), heads,
                                   queries, table, B > 1 ? block_table.stride(0) : 0,
                                   block_table.size(1), lens, B, (float)scale, window,
                                   code_of(query.scalar_type()),
                                   lse.has_value() ? lse->data_ptr<float>() : nullptr,
                                   workspace.data_ptr(), bytes, stream_of(query)));
}

// The pages of a cache.

// Bytes of a page of t (all but its first dimension), which lie together in some order.
int64_t page_bytes(const char* name, const Tensor& t) {
  std::vector<std::pair<int64_t, int64_t>> dims;  // strides, sizes
  for (int64_t d = 1; d < t.dim(); ++d) {
    if (t.size(d) != 1) dims.emplace_back(t.stride(d), t.size(d));
  }
  std::sort(dims.begin(), dims.end());
  int64_t dense = 1;
  for (const auto& [stride, size] : dims) {
    TORCH_CHECK(stride == dense, name, ": a page's elements must lie together, got sizes ", t.sizes(),
                " and strides ", t.strides());
    dense *= size;
  }
  TORCH_CHECK(t.size(0) <= 1 || t.stride(0) >= dense, name, ": pages must not overlap, got sizes ",
              t.sizes(), " and strides ", t.strides());
  return dense * t.element_size();
}

void c_kv_cache_copy_pages(at::TensorList caches, const Tensor& src, const Tensor& dst) {
  const char* name = "kv_cache_copy_pages";
  const auto* from = ints_ptr(name, "src", src, -1);
  const auto* to = ints_ptr(name, "dst", dst, src.size(0));
  if (caches.empty()) return;
  std::vector<mcop_kv_pages> list;
  int64_t pages = 0;
  for (const Tensor& t : caches) {
    TORCH_CHECK(t.dim() > 0 && t.size(0) == caches[0].size(0), name,
                ": caches must be [pages, ...] of the same pages, got ", t.sizes(), " beside ",
                caches[0].sizes());
    on_device(name, {&src, &dst, &t});
    pages = t.size(0);
    if (t.numel() == 0) continue;
    const int64_t bytes = page_bytes(name, t);
    list.push_back(mcop_kv_pages{t.data_ptr(), bytes,
                                 pages > 1 ? t.stride(0) * (int64_t)t.element_size() : bytes});
  }
  const DeviceGuard guard(src.device());
  check_rc(mcop_kv_cache_copy_pages(list.data(), (int64_t)list.size(), pages, from, to, src.size(0),
                                    stream_of(src)));
}

// The tables, checked; seq_lens may be absent.
mcop_kv_pool pool_of(const char* name, const Tensor& block_table, const OptTensor& seq_lens,
                     const Tensor& ref_counts, int64_t page_size) {
  auto* table = const_cast<int32_t*>(table_ptr(name, block_table));
  auto* lens = seq_lens.has_value() ? ints_ptr(name, "seq_lens", *seq_lens, block_table.size(0)) : nullptr;
  auto* counts = ints_ptr(name, "ref_counts", ref_counts, -1);
  TORCH_CHECK(page_size > 0, name, ": page_size must be positive, got ", page_size);
  no_overlap(name, {&block_table});
  return mcop_kv_pool{table, block_table.size(0) > 1 ? block_table.stride(0) : 0, block_table.size(0),
                      block_table.size(1), lens, counts, ref_counts.size(0), page_size};
}

Tensor pages_workspace(const Tensor& like, int64_t requests, int64_t pages) {
  const int64_t bytes = mcop_kv_cache_pages_workspace(requests, pages);
  if (bytes < 0) check_rc((int)bytes);
  return at::empty({bytes}, like.options().dtype(at::kByte));
}

void c_kv_cache_fork(Tensor& block_table, Tensor& seq_lens, Tensor& ref_counts, const Tensor& parents,
                     const Tensor& children, Tensor& src, Tensor& dst, int64_t page_size) {
  const char* name = "kv_cache_fork";
  const mcop_kv_pool pool = pool_of(name, block_table, seq_lens, ref_counts, page_size);
  const auto* from = ints_ptr(name, "parents", parents, -1);
  const int64_t n = parents.size(0);
  const auto* to = ints_ptr(name, "children", children, n);
  auto* s = ints_ptr(name, "src", src, n);
  auto* d = ints_ptr(name, "dst", dst, n);
  on_device(name, {&block_table, &seq_lens, &ref_counts, &parents, &children, &src, &dst});
  if (n == 0) return;
  const DeviceGuard guard(block_table.device());
  const Tensor ws = pages_workspace(block_table, n, pool.num_pages);
  check_rc(mcop_kv_cache_fork(&pool, from, to, n, s, d, ws.data_ptr(), ws.numel(),
                              stream_of(block_table)));
}

void c_kv_cache_extend(Tensor& block_table, Tensor& seq_lens, Tensor& ref_counts,
                       const Tensor& sequences, const Tensor& cu_tokens, Tensor& slots, Tensor& starts,
                       int64_t page_size) {
  const char* name = "kv_cache_extend";
  const mcop_kv_pool pool = pool_of(name, block_table, seq_lens, ref_counts, page_size);
  const auto* who = ints_ptr(name, "sequences", sequences, -1);
  const int64_t n = sequences.size(0);
  const auto* cu = ints_ptr(name, "cu_tokens", cu_tokens, n + 1);
  auto* first = ints_ptr(name, "starts", starts, n);
  TORCH_CHECK(slots.scalar_type() == at::kLong && slots.dim() == 1 && slots.is_contiguous(), name,
              ": slots must be a contiguous vector of Long, got ", slots.scalar_type(), " ",
              slots.sizes());
  on_device(name, {&block_table, &seq_lens, &ref_counts, &sequences, &cu_tokens, &slots, &starts});
  const DeviceGuard guard(block_table.device());
  const Tensor ws = pages_workspace(block_table, n, pool.num_pages);
  check_rc(mcop_kv_cache_extend(&pool, who, cu, n, slots.data_ptr<int64_t>(), slots.size(0), first,
                                ws.data_ptr(), ws.numel(), stream_of(block_table)));
}

void c_kv_cache_free(Tensor& block_table, Tensor& seq_lens, Tensor& ref_counts,
                     const Tensor& sequences, int64_t page_size) {
  const char* name = "kv_cache_free";
  const mcop_kv_pool pool = pool_of(name, block_table, seq_lens, ref_counts, page_size);
  const auto* who = ints_ptr(name, "sequences", sequences, -1);
  on_device(name, {&block_table, &seq_lens, &ref_counts, &sequences});
  const DeviceGuard guard(block_table.device());
  check_rc(mcop_kv_cache_free(&pool, who, sequences.size(0), stream_of(block_table)));
}

void c_kv_cache_compact(Tensor& block_table, Tensor& ref_counts, Tensor& src, Tensor& dst,
                        Tensor& used) {
  const char* name = "kv_cache_compact";
  const mcop_kv_pool pool = pool_of(name, block_table, std::nullopt, ref_counts, 1);
  auto* s = ints_ptr(name, "src", src, pool.num_pages / 2);
  auto* d = ints_ptr(name, "dst", dst, pool.num_pages / 2);
  auto* u = ints_ptr(name, "used", used, 1);
  on_device(name, {&block_table, &ref_counts, &src, &dst, &used});
  const DeviceGuard guard(block_table.device());
  const Tensor ws = pages_workspace(block_table, 0, pool.num_pages);
  check_rc(mcop_kv_cache_compact(&pool, s, d, u, ws.data_ptr(), ws.numel(), stream_of(block_table)));
}

// The allocating forms (custom_ops).

std::vector<int64_t> with_last(const Tensor& t, int64_t last) {
  std::vector<int64_t> shape = t.sizes().vec();
  shape.back() = last;
  return shape;
}

// New codes and scales for rows like input's (which the operators check).
std::pair<Tensor, Tensor> mx_new(const Tensor& input) {
  const int64_t H = rows_of(input).second;
  const auto opts = input.options().dtype(at::kByte);
  const py::gil_scoped_release allocating;  // it may wait for the device
  return {at::empty(with_last(input, H / 2), opts), at::empty(with_last(input, H / kMxBlock), opts)};
}

std::tuple<Tensor, Tensor> mxfp4_quant_new(const Tensor& input) {
  auto [codes, scale] = mx_new(input);
  c_mxfp4_quant(codes, input, scale);
  return {codes, scale};
}

Tensor mxfp4_dequant_new(const Tensor& codes, const Tensor& scale, py::object out_dtype) {
  const at::ScalarType dt = torch::python::detail::py_object_to_dtype(out_dtype);
  const int64_t half = rows_of(codes).second;
  Tensor out;
  {
    const py::gil_scoped_release allocating;
    out = at::empty(with_last(codes, half * 2), codes.options().dtype(dt));
  }
  c_mxfp4_dequant(out, codes, scale);
  return out;
}

std::tuple<Tensor, Tensor, OptTensor> rms_norm_mxfp4_quant_new(const Tensor& input,
                                                               const Tensor& weight,
                                                               double epsilon,
                                                               const OptTensor& residual) {
  auto [codes, scale] = mx_new(input);
  OptTensor after;
  if (residual.has_value()) {
    const py::gil_scoped_release allocating;
    after = at::empty(residual->sizes(), residual->options());
  }
  c_rms_norm_mxfp4_quant(codes, input, weight, scale, epsilon, residual, after);
  return {codes, scale, after};
}

Tensor mxfp4_scaled_mm_new(const Tensor& a, const Tensor& a_scale, const Tensor& b,
                           const Tensor& b_scale, py::object out_dtype, const OptTensor& bias) {
  const at::ScalarType dt = torch::python::detail::py_object_to_dtype(out_dtype);
  TORCH_CHECK(a.dim() > 0 && b.dim() == 2, "mxfp4_scaled_mm: b must be [N, K / 2], got ",
              b.sizes());
  Tensor out;
  {
    const py::gil_scoped_release allocating;
    out = at::empty(with_last(a, b.size(0)), a.options().dtype(dt));
  }
  c_mxfp4_scaled_mm(out, a, a_scale, b, b_scale, bias);
  return out;
}

std::tuple<Tensor, Tensor> kv_cache_read_new(const Tensor& key_cache, const Tensor& value_cache,
                                             const Tensor& key_scale, const Tensor& value_scale,
                                             const Tensor& block_table, const Tensor& cu_seqlens,
                                             int64_t num_tokens, py::object out_dtype,
                                             const OptTensor& seq_starts) {
  const char* name = "kv_cache_read_dequant";
  const at::ScalarType dt = torch::python::detail::py_object_to_dtype(out_dtype);
  TORCH_CHECK(key_cache.dim() == 4 && value_cache.dim() == 4 && num_tokens >= 0, name,
              ": caches must be [pages, page_size, heads, head_size], num_tokens not negative");
  const int64_t wide = is_codes4(key_cache.scalar_type()) ? 2 : 1;
  const auto opts = key_cache.options().dtype(dt);
  Tensor key, value;
  {
    const py::gil_scoped_release allocating;
    key = at::empty({num_tokens, key_cache.size(2), key_cache.size(3) * wide}, opts);
    value = at::empty({num_tokens, value_cache.size(2), value_cache.size(3) * wide}, opts);
  }
  c_kv_cache_read_dequant(key, value, key_cache, value_cache, key_scale, value_scale, block_table,
                          cu_seqlens, seq_starts);
  return {key, value};
}

std::tuple<Tensor, OptTensor> kv_cache_attention_new(
    const Tensor& query, const Tensor& key_cache, const Tensor& value_cache, const Tensor& key_scale,
    const Tensor& value_scale, const Tensor& block_table, const Tensor& seq_lens,
    std::optional<double> scale, int64_t window, bool return_lse) {
  const char* name = "kv_cache_attention";
  TORCH_CHECK(query.dim() == 3 && value_cache.dim() == 4, name,
              ": query must be [sequences, heads, head_size], got ", query.sizes(),
              ", caches [pages, page_size, heads, head_size]");
  const int64_t wide = is_codes4(value_cache.scalar_type()) ? 2 : 1;
  Tensor out;
  OptTensor lse;
  {
    const py::gil_scoped_release allocating;
    out = at::empty({query.size(0), query.size(1), value_cache.size(3) * wide}, query.options());
    if (return_lse) {
      lse = at::empty({query.size(0), query.size(1)}, query.options().dtype(at::kFloat));
    }
    c_kv_cache_attention(out, query, key_cache, value_cache, key_scale, value_scale, block_table,
                         seq_lens,
                         scale.value_or(1.0 / std::sqrt((double)std::max<int64_t>(1, query.size(2)))),
                         window, lse);
  }
  return {out, lse};
}

std::tuple<Tensor, Tensor> kv_cache_fork_new(Tensor& block_table, Tensor& seq_lens,
                                             Tensor& ref_counts, const Tensor& parents,
                                             const Tensor& children, int64_t page_size) {
  const py::gil_scoped_release allocating;
  Tensor src = at::empty({parents.numel()}, parents.options().dtype(at::kInt));
  Tensor dst = at::empty_like(src);
  c_kv_cache_fork(block_table, seq_lens, ref_counts, parents, children, src, dst, page_size);
  return {src, dst};
}

std::tuple<Tensor, Tensor> kv_cache_extend_new(Tensor& block_table, Tensor& seq_lens,
                                               Tensor& ref_counts, const Tensor& sequences,
                                               const Tensor& cu_tokens, int64_t num_tokens,
                                               int64_t page_size) {
  TORCH_CHECK(num_tokens >= 0, "kv_cache_extend: num_tokens must not be negative, got ", num_tokens);
  const py::gil_scoped_release allocating;
  Tensor slots = at::empty({num_tokens}, sequences.options().dtype(at::kLong));
  Tensor starts = at::empty({sequences.numel()}, sequences.options().dtype(at::kInt));
  c_kv_cache_extend(block_table, seq_lens, ref_counts, sequences, cu_tokens, slots, starts, page_size);
  return {slots, starts};
}

std::tuple<Tensor, Tensor, Tensor> kv_cache_compact_new(Tensor& block_table, Tensor& ref_counts) {
  const py::gil_scoped_release allocating;
  const auto opts = ref_counts.options().dtype(at::kInt);
  Tensor src = at::empty({ref_counts.numel() / 2}, opts), dst = at::empty_like(src);
  Tensor used = at::empty({1}, opts);
  c_kv_cache_compact(block_table, ref_counts, src, dst, used);
  return {src, dst, used};
}

// Meta kernel of the mutating _C ops (no outputs to describe): drop the arguments.
void meta_noop(const c10::OperatorHandle& op, torch::jit::Stack* stack) {
  torch::jit::drop(*stack, op.schema().arguments().size());
}

struct VllmOp {
  const char* name;
  const char* schema;
};
constexpr VllmOp kVllmOps[] = {
    {"rms_norm", "rms_norm(Tensor! result, Tensor input, Tensor weight, float epsilon) -> ()"},
    {"fused_add_rms_norm",
     "fused_add_rms_norm(Tensor! input, Tensor! residual, Tensor weight, float epsilon) -> ()"},
    {"rms_norm_dynamic_per_token_quant",
     "rms_norm_dynamic_per_token_quant(Tensor! result, Tensor input, Tensor weight, "
     "Tensor! scale, float epsilon, Tensor? scale_ub, Tensor!? residual) -> ()"},
    {"rms_norm_per_block_quant",
     "rms_norm_per_block_quant(Tensor! result, Tensor input, Tensor weight, Tensor! scale, "
     "float epsilon, Tensor? scale_ub, Tensor!? residual, int group_size, "
     "bool is_scale_transposed) -> ()"},
    {"dynamic_scaled_int8_quant",
     "dynamic_scaled_int8_quant(Tensor! result, Tensor input, Tensor! scale, Tensor!? azp) -> ()"},
    {"dynamic_per_token_scaled_fp8_quant",
     "dynamic_per_token_scaled_fp8_quant(Tensor! result, Tensor input, Tensor! scale, "
     "Tensor? scale_ub) -> ()"},
    {"mxfp4_quant", "mxfp4_quant(Tensor! result, Tensor input, Tensor! scale) -> ()"},
    {"mxfp4_dequant", "mxfp4_dequant(Tensor! result, Tensor input, Tensor scale) -> ()"},
    {"rms_norm_mxfp4_quant",
     "rms_norm_mxfp4_quant(Tensor! result, Tensor input, Tensor weight, Tensor! scale, "
     "float epsilon, Tensor? residual, Tensor!? after_res) -> ()"},
    {"mxfp4_scaled_mm",
     "mxfp4_scaled_mm(Tensor! result, Tensor a, Tensor a_scale, Tensor b, Tensor b_scale, "
     "Tensor? bias) -> ()"},
    {"kv_cache_write_quant",
     "kv_cache_write_quant(Tensor key, Tensor value, Tensor! key_cache, Tensor! value_cache, "
     "Tensor! key_scale, Tensor! value_scale, Tensor slot_mapping) -> ()"},
    {"kv_cache_read_dequant",
     "kv_cache_read_dequant(Tensor! key, Tensor! value, Tensor key_cache, Tensor value_cache, "
     "Tensor key_scale, Tensor value_scale, Tensor block_table, Tensor cu_seqlens, "
     "Tensor? seq_starts) -> ()"},
    {"kv_cache_attention",
     "kv_cache_attention(Tensor! result, Tensor query, Tensor key_cache, Tensor value_cache, "
     "Tensor key_scale, Tensor value_scale, Tensor block_table, Tensor seq_lens, float scale, "
     "int window, Tensor!? lse) -> ()"},
    {"kv_cache_copy_pages", "kv_cache_copy_pages(Tensor(a!)[] caches, Tensor src, Tensor dst) -> ()"},
    {"kv_cache_fork",
     "kv_cache_fork(Tensor! block_table, Tensor! seq_lens, Tensor! ref_counts, Tensor parents, "
     "Tensor children, Tensor! src, Tensor! dst, int page_size) -> ()"},
    {"kv_cache_extend",
     "kv_cache_extend(Tensor! block_table, Tensor! seq_lens, Tensor! ref_counts, Tensor sequences, "
     "Tensor cu_tokens, Tensor! slots, Tensor! starts, int page_size) -> ()"},
    {"kv_cache_free",
     "kv_cache_free(Tensor! block_table, Tensor! seq_lens, Tensor! ref_counts, Tensor sequences, "
     "int page_size) -> ()"},
    {"kv_cache_compact",
     "kv_cache_compact(Tensor! block_table, Tensor! ref_counts, Tensor! src, Tensor! dst, "
     "Tensor! used) -> ()"},
};

// Registers the _C schemas (each only if no other library, e.g. vLLM's own _C, defined it) with
// CUDA implementations here and a Meta kernel for the schemas defined here.  Idempotent.
void register_vllm_ops() {
  static bool done = false;
  if (done) return;
  static std::unique_ptr<torch::Library> defs, cuda, meta;
  defs = std::make_unique<torch::Library>(torch::Library::FRAGMENT, "_C", std::nullopt, __FILE__,
                                          __LINE__);
  meta = std::make_unique<torch::Library>(torch::Library::IMPL, "_C", c10::DispatchKey::Meta,
                                          __FILE__, __LINE__);
  for (const VllmOp& o : kVllmOps) {
    const std::string full = std::string("_C::") + o.name;
    if (!c10::Dispatcher::singleton().findSchema({full, ""}).has_value()) {
      defs->def(o.schema);
      meta->impl(o.name, torch::CppFunction::makeFromBoxedFunction<&meta_noop>());
    }
  }
  cuda = std::make_unique<torch::Library>(torch::Library::IMPL, "_C", c10::DispatchKey::CUDA,
                                          __FILE__, __LINE__);
  cuda->impl("rms_norm", TORCH_FN(c_rms_norm));
  cuda->impl("fused_add_rms_norm", TORCH_FN(c_fused_add_rms_norm));
  cuda->impl("rms_norm_dynamic_per_token_quant", TORCH_FN(c_norm_quant));
  cuda->impl("rms_norm_per_block_quant", TORCH_FN(c_per_block_quant));
  cuda->impl("dynamic_scaled_int8_quant", TORCH_FN(c_int8_quant));
  cuda->impl("dynamic_per_token_scaled_fp8_quant", TORCH_FN(c_fp8_quant));
  cuda->impl("mxfp4_quant", TORCH_FN(c_mxfp4_quant));
  cuda->impl("mxfp4_dequant", TORCH_FN(c_mxfp4_dequant));
  cuda->impl("rms_norm_mxfp4_quant", TORCH_FN(c_rms_norm_mxfp4_quant));
  cuda->impl("mxfp4_scaled_mm", TORCH_FN(c_mxfp4_scaled_mm));
  cuda->impl("kv_cache_write_quant", TORCH_FN(c_kv_cache_write_quant));
  cuda->impl("kv_cache_read_dequant", TORCH_FN(c_kv_cache_read_dequant));
  cuda->impl("kv_cache_attention", TORCH_FN(c_kv_cache_attention));
  cuda->impl("kv_cache_copy_pages", TORCH_FN(c_kv_cache_copy_pages));
  cuda->impl("kv_cache_fork", TORCH_FN(c_kv_cache_fork));
  cuda->impl("kv_cache_extend", TORCH_FN(c_kv_cache_extend));
  cuda->impl("kv_cache_free", TORCH_FN(c_kv_cache_free));
  cuda->impl("kv_cache_compact", TORCH_FN(c_kv_cache_compact));
  done = true;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "mcoplib.op and torch.ops._C surfaces of the fused RMSNorm + quantization path "
            "over libmcop_norm.so (gfx950)";
  // mcoplib.op
  m.def("rms_norm_dynamic_per_token_quant", &op_smooth_quant,
        "SmoothQuant (residual add +) RMSNorm + dynamic per-token quantization "
        "(fused_rms_norm_dq; reference op/fused_rms_norm_dq.cu:646-667).\n\n"
        "after_res <- input (+ residual); after_norm <- after_res / rsqrt(mean(after_res^2) + "
        "eps) * weight (the reference's literal form; standard_norm=True multiplies by the "
        "rsqrt instead); out <- per-token quantization of after_norm * smooth_scale; scales[t] "
        "<- absmax/127 (int8) or absmax/448 (fp8-e4m3fn, an extension: the reference accepts "
        "int8 only).  residual is read, not updated; weight and smooth_scale are each the "
        "input dtype or fp32.",
        py::arg("out"), py::arg("input"), py::arg("weight"), py::arg("smooth_scale"),
        py::arg("scales"), py::arg("var_epsilon"), py::arg("after_res"), py::arg("after_norm"),
        py::arg("residual") = py::none(), py::arg("standard_norm") = false);
  m.def("rms_norm_dynamic_per_token_quant_custom", &op_custom,
        "(Residual add +) RMSNorm + dynamic per-token int8 quantization with mcoplib's own "
        "arithmetic (reference op/rms_norm_dynamic_per_token_quant.cu:266-285): scale floor "
        "1.5e-6 and codes in [-127, 127]; at H == 7168 the reference's fp32 chain (codes from "
        "(x [+ r]) * w * rsqrt(...) without bf16 rounding, scale_ub unused).  residual is "
        "updated in place to input + residual; out and scales ([T] or [T, 1] fp32) are "
        "written.",
        py::arg("out"), py::arg("input"), py::arg("weight"), py::arg("scales"),
        py::arg("var_epsilon"), py::arg("scale_ub") = py::none(),
        py::arg("residual") = py::none());
  m.def("custom_new", &custom_new,
        "rms_norm_dynamic_per_token_quant_custom into new tensors: (codes, scales [T, 1]).",
        py::arg("input"), py::arg("weight"), py::arg("epsilon"), py::arg("quant_dtype"),
        py::arg("scale_ub") = py::none(), py::arg("residual") = py::none());
  m.def("padded_new", &padded_new,
        "fused_add_rms_norm_dynamic_per_token_quant_padding_output into new tensors: (output, "
        "residual, output_rms, output_quant_int8, scales [T, 1]).",
        py::arg("input"), py::arg("residual"), py::arg("weight"), py::arg("pad_size"),
        py::arg("epsilon"));
  m.def("scale_dynamic_quant", &op_scale_dynamic_quant,
        "Smooth-scale multiply + dynamic per-token int8 quantization (reference "
        "op/scale_dynamic_quant.cu:127-153).  Returns new (codes shaped like hidden_states, "
        "scales [T] fp32).",
        py::arg("hidden_states"), py::arg("smooth_scales"), py::arg("dst_dtype") = py::none());
  m.def("fused_add_rms_norm_dynamic_per_token_quant_padding_output", &op_padded,
        "Residual add + RMSNorm + per-token int8 quantization with a padded per-row output "
        "(reference op/fused_add_layernorm_per_token_quant_padding_output.cu:397-416).\n\n"
        "output (int8, 2*pad_size bytes per row) receives each row's codes at bytes [0, H) and "
        "its fp32 scale at bytes [H, H+4); output_rms (bf16) the normalized row, "
        "output_quant_int8 the codes again, out_scales the scales; residual becomes input + "
        "residual.  H == 7168 uses the reference's fp32 chain (its \"opt\" kernel), other H its "
        "bf16-rounded chain; every output is written for every H.",
        py::arg("output"), py::arg("output_rms"), py::arg("output_quant_int8"),
        py::arg("out_scales"), py::arg("input"), py::arg("residual"), py::arg("weight"),
        py::arg("pad_size"), py::arg("epsilon"));
  m.def("rms_norm", &op_rms_norm,
        "(Residual add +) RMSNorm (reference op/fused_rms_norm_dq.cu:980-998): out <- (input [+ "
        "residual]) / rsqrt(mean(.^2) + eps) * weight when rms_div (the reference's "
        "convention), or * rsqrt(...) * weight otherwise; with a residual, after_res <- input "
        "+ residual (the residual itself is not updated).  weight is the input dtype or fp32.",
        py::arg("out"), py::arg("input"), py::arg("weight"), py::arg("var_epsilon"),
        py::arg("after_res") = py::none(), py::arg("residual") = py::none(),
        py::arg("rms_div") = true);
  m.def("head_rms_norm", &op_head_rms_norm,
        "Per-head RMSNorm of heads [head_offset, head_offset + head_norm) of hidden_states "
        "[num_tokens, num_heads, head_size] with per-head weights [num_heads, head_size] (bf16 "
        "or fp32); out (same shape) is written for those heads only (reference "
        "op/fused_rms_norm_dq.cu:804-812), as x / rsqrt(mean(x^2) + eps) * weight.",
        py::arg("out"), py::arg("hidden_states"), py::arg("weight"), py::arg("var_epsilon"),
        py::arg("head_offset"), py::arg("head_norm"));
  // torch.ops._C
  m.def("register_vllm_ops", &register_vllm_ops,
        "Register the torch.ops._C schemas and their CUDA (HIP) implementations (idempotent).");
  m.def("c_rms_norm", &c_rms_norm, py::arg("result"), py::arg("input"), py::arg("weight"),
        py::arg("epsilon"));
  m.def("c_fused_add_rms_norm", &c_fused_add_rms_norm, py::arg("input"), py::arg("residual"),
        py::arg("weight"), py::arg("epsilon"));
  m.def("c_rms_norm_dynamic_per_token_quant", &c_norm_quant, py::arg("result"),
        py::arg("input"), py::arg("weight"), py::arg("scale"), py::arg("epsilon"),
        py::arg("scale_ub") = py::none(), py::arg("residual") = py::none());
  m.def("c_rms_norm_per_block_quant", &c_per_block_quant, py::arg("result"), py::arg("input"),
        py::arg("weight"), py::arg("scale"), py::arg("epsilon"), py::arg("scale_ub"),
        py::arg("residual"), py::arg("group_size"), py::arg("is_scale_transposed"));
  m.def("c_dynamic_scaled_int8_quant", &c_int8_quant, py::arg("result"), py::arg("input"),
        py::arg("scale"), py::arg("azp") = py::none());
  m.def("c_dynamic_per_token_scaled_fp8_quant", &c_fp8_quant, py::arg("result"),
        py::arg("input"), py::arg("scale"), py::arg("scale_ub") = py::none());
  m.def("c_mxfp4_quant", &c_mxfp4_quant,
        "Rows of input (bf16, fp16, fp32; last dimension contiguous, a multiple of 32) as 4-bit "
        "codes: result [..., H / 2] (uint8 or float4_e2m1fn_x2, element 2i in the low half of byte "
        "i), scale [..., H / 32] (uint8 or float8_e8m0fnu).",
        py::arg("result"), py::arg("input"), py::arg("scale"));
  m.def("c_mxfp4_dequant", &c_mxfp4_dequant,
        "The values of codes and scales of mxfp4_quant, rounded once to result's dtype.",
        py::arg("result"), py::arg("input"), py::arg("scale"));
  m.def("c_rms_norm_mxfp4_quant", &c_rms_norm_mxfp4_quant,
        "(Residual add +) RMSNorm + mxfp4_quant of the normalized rows; after_res <- input + "
        "residual (it may be the residual or the input itself; the two are given together).",
        py::arg("result"), py::arg("input"), py::arg("weight"), py::arg("scale"),
        py::arg("epsilon"), py::arg("residual") = py::none(), py::arg("after_res") = py::none());
  m.def("c_mxfp4_scaled_mm", &c_mxfp4_scaled_mm,
        "result [..., N] (bf16, fp16, fp32) <- a [..., K / 2] times the transpose of b [N, K / 2], "
        "both codes with scales [..., K / 32], plus bias [N]; summed in fp32, rounded once.",
        py::arg("result"), py::arg("a"), py::arg("a_scale"), py::arg("b"), py::arg("b_scale"),
        py::arg("bias") = py::none());
  m.def("c_kv_cache_write_quant", &c_kv_cache_write_quant,
        "Quantizes key and value [tokens, heads, head_size] into the slots of a paged cache "
        "[pages, page_size, heads, head_size] (int8 or float8_e4m3fn with fp32 scales [pages, "
        "page_size, heads]; or 4-bit codes, uint8 [..., head_size / 2], with scales [..., "
        "head_size / 32]). slot_mapping (int64) may cover fewer tokens; a negative slot, or one "
        "past the cache, is not written. Slots that are written must differ, and the caches and "
        "scales must not overlap.",
        py::arg("key"), py::arg("value"), py::arg("key_cache"), py::arg("value_cache"),
        py::arg("key_scale"), py::arg("value_scale"), py::arg("slot_mapping"));
  m.def("c_kv_cache_read_dequant", &c_kv_cache_read_dequant,
        "Gathers sequences of such a cache into key and value [tokens, heads, head_size]: rows "
        "cu_seqlens[s] to cu_seqlens[s + 1] are positions from seq_starts[s] (or 0) on of sequence "
        "s, whose pages block_table[s] lists. Rows past the last sequence are left as they were; "
        "positions without a page read as NaN.",
        py::arg("key"), py::arg("value"), py::arg("key_cache"), py::arg("value_cache"),
        py::arg("key_scale"), py::arg("value_scale"), py::arg("block_table"),
        py::arg("cu_seqlens"), py::arg("seq_starts") = py::none());
  m.def("c_kv_cache_attention", &c_kv_cache_attention,
        "Attention of one new token a sequence over such a cache: result [sequences, query heads, "
        "value head_size] <- softmax(scale * query k) v over positions max(0, n - window) (window 0: "
        "from 0) to n - 1 of each, n = seq_lens, whose pages block_table lists. query heads are a "
        "multiple of the cache's. lse [sequences, query heads] (fp32) <- the log of each row's sum. A "
        "sequence of no positions gives 0 and -inf, one with a position without a page NaN.",
        py::arg("result"), py::arg("query"), py::arg("key_cache"), py::arg("value_cache"),
        py::arg("key_scale"), py::arg("value_scale"), py::arg("block_table"), py::arg("seq_lens"),
        py::arg("scale"), py::arg("window") = 0, py::arg("lse") = py::none(),
        py::call_guard<py::gil_scoped_release>());  // it allocates its workspace
  m.def("c_kv_cache_copy_pages",
        [](const std::vector<Tensor>& caches, const Tensor& src, const Tensor& dst) {
          c_kv_cache_copy_pages(caches, src, dst);
        },
        "Copies page src[i] to page dst[i] in every tensor [pages, ...] of caches (codes and scales of "
        "every layer); pairs with a negative index, or one past the pages, are left out. Pages that are "
        "written must differ from each other and from those that are read.",
        py::arg("caches"), py::arg("src"), py::arg("dst"));
  m.def("c_kv_cache_fork", &c_kv_cache_fork,
        "Sequence (row of block_table) children[i] becomes a copy of parents[i]: full pages are shared, a "
        "part-filled last page is replaced by the lowest free one; src, dst <- that page of the parent "
        "and of the child, for kv_cache_copy_pages, -1 where there is none.",
        py::arg("block_table"), py::arg("seq_lens"), py::arg("ref_counts"), py::arg("parents"),
        py::arg("children"), py::arg("src"), py::arg("dst"), py::arg("page_size"),
        py::call_guard<py::gil_scoped_release>());  // it allocates its workspace
  m.def("c_kv_cache_extend", &c_kv_cache_extend,
        "sequences[i] grows by cu_tokens[i + 1] - cu_tokens[i] tokens and takes the lowest free pages for "
        "them; slots <- the new tokens' slots, starts <- their first positions, -1 where the pages do "
        "not suffice.",
        py::arg("block_table"), py::arg("seq_lens"), py::arg("ref_counts"), py::arg("sequences"),
        py::arg("cu_tokens"), py::arg("slots"), py::arg("starts"), py::arg("page_size"),
        py::call_guard<py::gil_scoped_release>());
  m.def("c_kv_cache_free", &c_kv_cache_free,
        "Gives back the pages of sequences: counted once less, the rows -1, the lengths 0.",
        py::arg("block_table"), py::arg("seq_lens"), py::arg("ref_counts"), py::arg("sequences"),
        py::arg("page_size"));
  m.def("c_kv_cache_compact", &c_kv_cache_compact,
        "Moves the pages in use together: used <- their number U; src, dst [pages / 2] <- the moves from "
        "U and above to the free pages below, for kv_cache_copy_pages, -1 behind the last; block_table "
        "and ref_counts follow.",
        py::arg("block_table"), py::arg("ref_counts"), py::arg("src"), py::arg("dst"), py::arg("used"),
        py::call_guard<py::gil_scoped_release>());
  // custom_ops: the same into new tensors
  m.def("mxfp4_quant_new", &mxfp4_quant_new, py::arg("input"));
  m.def("mxfp4_dequant_new", &mxfp4_dequant_new, py::arg("codes"), py::arg("scale"),
        py::arg("out_dtype"));
  m.def("rms_norm_mxfp4_quant_new", &rms_norm_mxfp4_quant_new, py::arg("input"),
        py::arg("weight"), py::arg("epsilon"), py::arg("residual") = py::none());
  m.def("mxfp4_scaled_mm_new", &mxfp4_scaled_mm_new, py::arg("a"), py::arg("a_scale"),
        py::arg("b"), py::arg("b_scale"), py::arg("out_dtype"), py::arg("bias") = py::none());
  m.def("kv_cache_read_new", &kv_cache_read_new, py::arg("key_cache"), py::arg("value_cache"),
        py::arg("key_scale"), py::arg("value_scale"), py::arg("block_table"),
        py::arg("cu_seqlens"), py::arg("num_tokens"), py::arg("out_dtype"),
        py::arg("seq_starts") = py::none());
  m.def("kv_cache_attention_new", &kv_cache_attention_new, py::arg("query"), py::arg("key_cache"),
        py::arg("value_cache"), py::arg("key_scale"), py::arg("value_scale"), py::arg("block_table"),
        py::arg("seq_lens"), py::arg("scale") = py::none(), py::arg("window") = 0,
        py::arg("return_lse") = false);
  m.def("kv_cache_fork_new", &kv_cache_fork_new, py::arg("block_table"), py::arg("seq_lens"),
        py::arg("ref_counts"), py::arg("parents"), py::arg("children"), py::arg("page_size"));
  m.def("kv_cache_extend_new", &kv_cache_extend_new, py::arg("block_table"), py::arg("seq_lens"),
        py::arg("ref_counts"), py::arg("sequences"), py::arg("cu_tokens"), py::arg("num_tokens"),
        py::arg("page_size"));
  m.def("kv_cache_compact_new", &kv_cache_compact_new, py::arg("block_table"), py::arg("ref_counts"));
}
