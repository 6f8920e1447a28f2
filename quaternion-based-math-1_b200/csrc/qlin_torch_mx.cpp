// The package's calls on 4-bit quaternion weights and gradient clipping in
// C++ (part of the torch extension): the checks of the Python interface with
// its error classes (shape problems -> ValueError, the rest -> RuntimeError),
// output allocation, workspace from the caching allocator, one library call
// on the current stream of the tensors' device.
#include <torch/extension.h>

#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/AutogradState.h>
#include <c10/core/InferenceMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>
#include <cmath>
#include <limits>
#include <string>
#include <vector>

#include "qlin_b200.h"

namespace {

using OptTensor = c10::optional<at::Tensor>;

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return QLIN_F32;
    case at::kBFloat16: return QLIN_BF16;
    case at::kHalf: return QLIN_F16;
    default:
      TORCH_CHECK(false, "unsupported dtype ", t,
                  "; the B200 quaternion kernels take float32, bfloat16 or float16");
  }
  return -1;
}

void shape_error(const std::string& msg) { throw pybind11::value_error(msg); }

void check_status(int st, const char* what) {
  if (st == QLIN_ERR_SHAPE) shape_error(std::string(what) + ": " + qlin_status_string(st));
  TORCH_CHECK(st == QLIN_OK, what, ": ", qlin_status_string(st), " (status ", st, ")");
}

void check_cuda(const at::Tensor& t, const at::Tensor& like, bool same_type) {
  TORCH_CHECK(t.is_cuda(),
              "the B200 quaternion linear kernels require CUDA tensors (there is no CPU path); got a tensor on ",
              t.device());
  TORCH_CHECK(t.device() == like.device(), "all tensors must be on one device, got ", like.device(), " and ",
              t.device());
  TORCH_CHECK(!same_type || t.scalar_type() == like.scalar_type(), "all tensors must share one dtype, got ",
              like.scalar_type(), " and ", t.scalar_type());
}

cudaStream_t stream_of(const at::Tensor& t) {
  return at::cuda::getCurrentCUDAStream(t.device().index()).stream();
}

at::Tensor bytes_on(const at::Tensor& like, size_t n) {
  return at::empty({static_cast<int64_t>(n)}, at::TensorOptions().dtype(at::kByte).device(like.device()));
}

void check_buffer(const at::Tensor& mx, int64_t out_groups, int64_t in_groups, const at::Tensor& like) {
  size_t need = 0;
  check_status(qlin_mx_weights_size(in_groups, out_groups, &need), "4-bit weights");
  if (mx.scalar_type() != at::kByte || mx.dim() != 1 || mx.size(0) != static_cast<int64_t>(need) ||
      !mx.is_contiguous())
    shape_error("4-bit weights of a [" + std::to_string(out_groups) + ", " + std::to_string(in_groups) +
                "] layer are " + std::to_string(need) + " contiguous uint8 values");
  check_cuda(mx, like, false);
}

// Rows of K elements with a row stride of at least K, copied where the tensor has none.
at::Tensor rows_of(const at::Tensor& x, int64_t K) {
  at::Tensor r = x.reshape({-1, K});
  if (r.size(0) > 0 && (r.stride(1) != 1 || (r.size(0) > 1 && r.stride(0) < K))) r = r.contiguous();
  return r;
}
int64_t row_stride(const at::Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

const void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

struct Adapter {
  at::Tensor a, b;
  int rank = 0;
};

Adapter adapter_of(const OptTensor& a, const OptTensor& b, int64_t K, int64_t N, const at::Tensor& like) {
  Adapter out;
  const bool has_a = a.has_value() && a->defined(), has_b = b.has_value() && b->defined();
  if (has_a != has_b) shape_error("LoRA needs both A and B");
  if (!has_a) return out;
  if (a->dim() != 2 || a->size(1) != K || b->dim() != 2 || b->size(0) != N || b->size(1) != a->size(0))
    shape_error("LoRA shapes must be A [r, " + std::to_string(K) + "] and B [" + std::to_string(N) + ", r]");
  check_cuda(*a, like, true);
  check_cuda(*b, like, true);
  if (a->size(0) > std::numeric_limits<int>::max()) shape_error("LoRA rank out of range");
  out.rank = static_cast<int>(a->size(0));
  if (out.rank > 0) {
    out.a = a->contiguous();
    out.b = b->contiguous();
  }
  return out;
}

at::Tensor mx_quantize(const at::Tensor& wr, const at::Tensor& wi, const at::Tensor& wj, const at::Tensor& wk) {
  for (const at::Tensor* w : {&wr, &wi, &wj, &wk})
    if (w->dim() != 2) shape_error("weight components must be 2D [out_groups, in_groups]");
  if (wr.sizes() != wi.sizes() || wr.sizes() != wj.sizes() || wr.sizes() != wk.sizes())
    shape_error("all four weight components must share the same shape");
  for (const at::Tensor* w : {&wr, &wi, &wj, &wk}) check_cuda(*w, wr, true);
  const int code = dtype_code(wr.scalar_type());
  const int64_t n = wr.size(0), k = wr.size(1);
  size_t need = 0;
  check_status(qlin_mx_weights_size(k, n, &need), "4-bit weights");
  c10::cuda::CUDAGuard guard(wr.device());
  at::Tensor w[4] = {wr, wi, wj, wk};
  int64_t ld = n > 1 ? wr.stride(0) : k;
  bool direct = ld >= k;
  for (auto& t : w) direct = direct && (k == 1 || t.stride(1) == 1) && (n == 1 || t.stride(0) == ld);
  if (!direct) {
    for (auto& t : w) t = t.contiguous();
    ld = k;
  }
  at::Tensor mx = bytes_on(wr, need);
  check_status(qlin_mx_quantize(code, w[0].data_ptr(), w[1].data_ptr(), w[2].data_ptr(), w[3].data_ptr(), ld, k, n,
                                mx.data_ptr(), stream_of(wr)),
               "qlin_mx_quantize");
  return mx;
}

std::vector<at::Tensor> mx_dequantize(const at::Tensor& mx, int64_t out_groups, int64_t in_groups,
                                      at::ScalarType type) {
  check_buffer(mx, out_groups, in_groups, mx);
  const int code = dtype_code(type);
  c10::cuda::CUDAGuard guard(mx.device());
  std::vector<at::Tensor> w;
  for (int p = 0; p < 4; ++p) w.push_back(at::empty({out_groups, in_groups}, mx.options().dtype(type)));
  check_status(qlin_mx_dequantize(code, mx.data_ptr(), in_groups, out_groups, w[0].data_ptr(), w[1].data_ptr(),
                                  w[2].data_ptr(), w[3].data_ptr(), in_groups, stream_of(mx)),
               "qlin_mx_dequantize");
  return w;
}

at::Tensor mx_forward(const at::Tensor& x, const at::Tensor& mx, int64_t out_groups, int64_t in_groups,
                      const OptTensor& bias_opt, const OptTensor& lora_a, const OptTensor& lora_b,
                      double lora_scale) {
  const int64_t K = 4 * in_groups, N = 4 * out_groups;
  if (x.dim() == 0 || x.size(-1) % 4 != 0)
    shape_error("in_features must be divisible by 4 (quaternion packing), got " +
                std::to_string(x.dim() ? x.size(-1) : 0));
  if (x.size(-1) != K)
    shape_error("weight in_groups (" + std::to_string(in_groups) + ") must match input in_groups (" +
                std::to_string(x.size(-1) / 4) + ")");
  at::Tensor bias;
  if (bias_opt.has_value() && bias_opt->defined()) {
    if (bias_opt->dim() != 1 || bias_opt->size(0) != N) shape_error("bias must be [" + std::to_string(N) + "]");
    bias = *bias_opt;
  }
  check_cuda(x, x, true);
  const int code = dtype_code(x.scalar_type());
  check_buffer(mx, out_groups, in_groups, x);
  const Adapter ad = adapter_of(lora_a, lora_b, K, N, x);
  if (bias.defined()) {
    check_cuda(bias, x, true);
    bias = bias.contiguous();
  }
  c10::cuda::CUDAGuard guard(x.device());
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::empty(shape, x.options());
  if (y.numel() == 0) return y;
  const at::Tensor x2 = rows_of(x, K);
  const int64_t M = x2.size(0);
  size_t need = 0;
  check_status(qlin_mx_workspace_size(code, M, in_groups, out_groups, ad.rank, &need), "qlin_mx_workspace_size");
  const at::Tensor ws = need ? bytes_on(x, need) : at::Tensor();
  check_status(qlin_mx_forward(code, x2.data_ptr(), row_stride(x2), mx.data_ptr(), ptr(bias), ptr(ad.a), ptr(ad.b),
                               ad.rank, static_cast<float>(lora_scale), y.data_ptr(), N, M, in_groups, out_groups,
                               const_cast<void*>(ptr(ws)), need, stream_of(x)),
               "qlin_mx_forward");
  return y;
}

// (dx, da, db, dbias), undefined where not wanted.
std::vector<at::Tensor> mx_backward(const at::Tensor& gy, const at::Tensor& x, const at::Tensor& mx,
                                    int64_t out_groups, int64_t in_groups, const OptTensor& lora_a,
                                    const OptTensor& lora_b, double lora_scale, bool want_dx, bool want_da,
                                    bool want_db, bool want_dbias) {
  const int64_t K = 4 * in_groups, N = 4 * out_groups;
  check_cuda(gy, gy, true);
  check_cuda(x, gy, true);
  const int code = dtype_code(gy.scalar_type());
  check_buffer(mx, out_groups, in_groups, gy);
  const Adapter ad = adapter_of(lora_a, lora_b, K, N, gy);
  c10::cuda::CUDAGuard guard(gy.device());
  const auto like = gy.options();
  at::Tensor dx, da, db, dbias;
  if (want_dx) dx = at::empty(x.sizes(), like);
  if (want_da && lora_a.has_value()) da = at::empty({ad.rank, K}, like);
  if (want_db && lora_b.has_value()) db = at::empty({N, ad.rank}, like);
  if (want_dbias) dbias = at::empty({N}, like);
  const at::Tensor g2 = rows_of(gy, N), x2 = rows_of(x, K);
  const int64_t M = g2.size(0);
  size_t need = 0;
  check_status(qlin_mx_backward_workspace_size(code, M, in_groups, out_groups, ad.rank, &need),
               "qlin_mx_backward_workspace_size");
  const at::Tensor ws = need ? bytes_on(gy, need) : at::Tensor();
  auto out = [&](const at::Tensor& t) { return ad.rank > 0 ? const_cast<void*>(ptr(t)) : nullptr; };
  check_status(qlin_mx_backward(code, g2.data_ptr(), row_stride(g2), x2.data_ptr(), row_stride(x2), mx.data_ptr(),
                                ptr(ad.a), ptr(ad.b), ad.rank, static_cast<float>(lora_scale),
                                const_cast<void*>(ptr(dx)), K, out(da), out(db), const_cast<void*>(ptr(dbias)), M,
                                in_groups, out_groups, const_cast<void*>(ptr(ws)), need, stream_of(gy)),
               "qlin_mx_backward");
  return {dx, da, db, dbias};
}

// The layer under autograd, in C++ (a Python function's calls from the backward
// thread cost about 40 us a step).
class MxLinear : public torch::autograd::Function<MxLinear> {
 public:
  static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& x, const OptTensor& bias,
                            const OptTensor& a, const OptTensor& b, const at::Tensor& mx, int64_t out_groups,
                            int64_t in_groups, double scale) {
    at::AutoDispatchBelowADInplaceOrView below;
    ctx->save_for_backward({x, a.value_or(at::Tensor()), b.value_or(at::Tensor()), mx});
    ctx->saved_data["n"] = out_groups;
    ctx->saved_data["k"] = in_groups;
    ctx->saved_data["s"] = scale;
    ctx->saved_data["bias"] = bias.has_value() && bias->defined();
    return mx_forward(x, mx, out_groups, in_groups, bias, a, b, scale);
  }

  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    auto opt = [](const at::Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
    torch::autograd::variable_list out(8);
    if (!grads[0].defined()) return out;
    // the graph's edges are those of the tensors that were given: x, bias, A, B
    size_t edge = 0;
    auto wanted = [&](bool given) { return given && ctx->needs_input_grad(edge++); };
    const bool dx = wanted(true), dbias = wanted(ctx->saved_data["bias"].toBool());
    const bool da = wanted(saved[1].defined()), db = wanted(saved[2].defined());
    std::vector<at::Tensor> g;
    {
      at::NoGradGuard no_grad;
      g = mx_backward(grads[0], saved[0], saved[3], ctx->saved_data["n"].toInt(), ctx->saved_data["k"].toInt(),
                      opt(saved[1]), opt(saved[2]), ctx->saved_data["s"].toDouble(), dx, da, db, dbias);
    }
    const int from[4] = {0, 3, 1, 2};  // x, bias, a, b of (dx, da, db, dbias)
    for (int k = 0; k < 4; ++k) out[k] = g[from[k]];
    if (at::GradMode::is_enabled()) {
      // the gradients have none of their own: an error where one is asked for
      torch::autograd::variable_list there;
      for (auto& t : out)
        if (t.defined()) there.push_back(t.detach().requires_grad_(true));
      auto error = std::make_shared<torch::autograd::DelayedError>(
          "mx_quaternion_linear cannot be differentiated twice", static_cast<int64_t>(there.size()));
      there = (*error)(std::move(there));
      size_t at = 0;
      for (auto& t : out)
        if (t.defined()) t = there[at++];
    }
    return out;
  }
};

// mx_forward, differentiable in x, bias, A and B (backwards; a tangent is refused, the
// kernels would drop it).
at::Tensor mx_linear(const at::Tensor& x, const at::Tensor& mx, int64_t out_groups, int64_t in_groups,
                     const OptTensor& bias, const OptTensor& a, const OptTensor& b, double scale) {
  if (c10::AutogradState::get_tls_state().get_fw_grad_mode()) {
    auto dual = [](const OptTensor& t) { return t.has_value() && t->defined() && t->_fw_grad(0).defined(); };
    TORCH_CHECK(!x._fw_grad(0).defined() && !dual(bias) && !dual(a) && !dual(b),
                "mx_quaternion_linear has no forward-mode derivatives");
  }
  if (at::GradMode::is_enabled()) {
    auto wants = [](const OptTensor& t) { return t.has_value() && t->defined() && t->requires_grad(); };
    if (x.requires_grad() || wants(bias) || wants(a) || wants(b))
      return MxLinear::apply(x, bias, a, b, mx, out_groups, in_groups, scale);
  }
  return mx_forward(x, mx, out_groups, in_groups, bias, a, b, scale);
}

// Clips the gradients of the parameters in place, each gradient once; returns their
// global norm.  error_if_nonfinite: only a finite one, which the host waits for.
at::Tensor clip_grad_norm(const pybind11::iterable& parameters, double max_norm, bool error_if_nonfinite) {
  TORCH_CHECK_VALUE(max_norm >= 0.0, "max_norm must be at least 0, got ", max_norm);
  std::vector<at::Tensor> grads;
  std::vector<void*> seen;
  for (const auto& h : parameters) {
    TORCH_CHECK_TYPE(THPVariable_Check(h.ptr()), "parameters must be tensors, got ",
                     std::string(pybind11::str(pybind11::type::of(h))));
    const at::Tensor g = THPVariable_Unpack(h.ptr()).grad();
    if (!g.defined()) continue;
    grads.push_back(g);
    seen.push_back(g.unsafeGetTensorImpl());
  }
  // a gradient that comes up twice counts once
  std::sort(seen.begin(), seen.end());
  if (std::adjacent_find(seen.begin(), seen.end()) != seen.end()) {
    std::vector<at::Tensor> once;
    for (const at::Tensor& g : grads)
      if (std::none_of(once.begin(), once.end(), [&](const at::Tensor& o) { return o.is_same(g); })) once.push_back(g);
    grads.swap(once);
  }
  if (grads.empty()) return at::zeros({}, at::kFloat);
  std::vector<at::Tensor> dense;
  std::vector<void*> data;
  std::vector<int64_t> sizes;
  std::vector<int> types;
  for (const at::Tensor& g : grads) {
    TORCH_CHECK(g.layout() == at::kStrided, "sparse gradients are not supported");
    check_cuda(g, grads[0], false);
    types.push_back(dtype_code(g.scalar_type()));
    // nothing is written before every gradient is known to be writable
    if (!g.is_contiguous()) at::assert_no_internal_overlap(g);
    TORCH_CHECK(!g.is_inference() || c10::InferenceMode::is_enabled(),
                "a gradient made in inference mode cannot be clipped outside it");
  }
  c10::cuda::CUDAGuard guard(grads[0].device());
  at::NoGradGuard no_grad;
  for (const at::Tensor& g : grads) {
    // one with gaps in memory goes through a dense copy
    dense.push_back(g.is_contiguous() || g.is_non_overlapping_and_dense() ? g : g.contiguous());
    data.push_back(dense.back().data_ptr());
    sizes.push_back(g.numel());
  }
  const int count = static_cast<int>(grads.size());
  size_t need = 0;
  check_status(qlin_grad_clip_workspace_size(count, &need), "qlin_grad_clip_workspace_size");
  const at::Tensor ws = bytes_on(grads[0], need);
  at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
  auto run = [&](double limit) {
    check_status(qlin_grad_clip(count, data.data(), sizes.data(), types.data(), static_cast<float>(limit),
                                norm.data_ptr<float>(), ws.data_ptr(), need, stream_of(grads[0])),
                 "qlin_grad_clip");
  };
  if (error_if_nonfinite) {
    run(std::numeric_limits<double>::infinity());  // the norm alone
    const float n = norm.item<float>();
    TORCH_CHECK(std::isfinite(n), "the global norm of the gradients is ", n, "; they are not clipped");
  }
  run(max_norm);
  for (size_t k = 0; k < grads.size(); ++k) {
    if (dense[k].is_same(grads[k])) grads[k].unsafeGetTensorImpl()->bump_version();  // changed in place
    else grads[k].copy_(dense[k]);
  }
  return norm;
}

}  // namespace

void register_mx(pybind11::module& m) {
  namespace py = pybind11;
  m.def("mx_quantize", &mx_quantize, "four weight components -> 4-bit buffer");
  m.def("mx_dequantize",
        [](const at::Tensor& mx, int64_t n, int64_t k, const py::object& dtype) {
          return mx_dequantize(mx, n, k, torch::python::detail::py_object_to_dtype(dtype));
        },
        "4-bit buffer -> four weight components");
  m.def("mx_linear", &mx_linear, "quaternion linear layer on 4-bit weights (see qlin_b200.h)", py::arg("x"),
        py::arg("mx"), py::arg("out_groups"), py::arg("in_groups"), py::arg("bias") = py::none(),
        py::arg("lora_a") = py::none(), py::arg("lora_b") = py::none(), py::arg("lora_scale") = 0.0,
        py::call_guard<py::gil_scoped_release>());
  m.def("clip_grad_norm", &clip_grad_norm, "global norm of the parameters' gradients, clipped in place");
}
