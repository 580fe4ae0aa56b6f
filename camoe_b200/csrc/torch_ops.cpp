// The expert layer and the adapters as torch calls (camoe_b200/experts.py,
// camoe_b200/adapters.py): argument checks, output allocation, the current stream
// and the autograd nodes around the C ABI of include/camoe_experts.h.
//
// These operators are one to three launches of a few microseconds each, which the
// same glue in Python and ctypes does not keep up with: a combine of one token
// takes 10.9 us of host time in Python and 5.7 here (4 us on the device), forward
// and backward of the sort 84 and 56 us (29 us on the device for 8192 tokens).
//
// A call whose arguments it cannot take returns None; the Python caller then
// says what is wrong with them.
#include <torch/extension.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>

#include <stdexcept>
#include <string>

#include "camoe_experts.h"

extern "C" const char* camoe_wkv7_strerror(int code);

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A non-zero status of the C ABI; camoe_b200._lib raises it as its CamoeError (out of
// a backward torch turns it into a plain RuntimeError).
struct Status : std::runtime_error {
  int code;
  explicit Status(int c)
      : std::runtime_error("camoe_wkv7 error " + std::to_string(c) + ": " + camoe_wkv7_strerror(c)), code(c) {}
};
void check(int status) {
  if (status != 0) throw Status(status);
}
void* stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
int dtype_of(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 ? 0 : 1; }
bool is_float(const Tensor& t) { return t.scalar_type() == torch::kBFloat16 || t.scalar_type() == torch::kFloat32; }
bool fits(const Tensor& t, at::IntArrayRef shape, c10::ScalarType type, const c10::Device& device) {
  return t.scalar_type() == type && t.device() == device && t.sizes() == shape && t.is_contiguous();
}
bool aligned(std::initializer_list<const Tensor*> ts) {
  uintptr_t all = 0;
  for (const Tensor* t : ts) all |= reinterpret_cast<uintptr_t>(t->data_ptr());
  return (all & 15u) == 0;
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->requires_grad()) return true;
  return false;
}
// Forward-mode tangents, which the kernels would drop.
void no_tangents(const char* call, std::initializer_list<const Tensor*> ts) {
  for (const Tensor* t : ts)
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), call, " has no forward-mode derivative");
}
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor bytes(size_t n, const Tensor& like) {
  return n > 0 ? at::empty({static_cast<int64_t>(n)}, like.options().dtype(torch::kUInt8)) : Tensor();
}

// a gradient as the kernels take it
Tensor packed(const Tensor& g) {
  const Tensor t = g.contiguous();
  return aligned({&t}) ? t : t.clone();
}

// A gradient of a backward that is recorded (create_graph): the kernels have no
// derivative of it, so going back through it is an error.  from: what it depends on.
struct Once : torch::autograd::Function<Once> {
  static Tensor forward(AutogradContext*, const Tensor& gradient, const Tensor&) { return gradient.detach(); }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "the expert layer's operators are differentiable once: their gradients have no gradient");
    return {};
  }
};
void once(Tensor& gradient, std::initializer_list<const Tensor*> from) {
  if (!at::GradMode::is_enabled() || !gradient.defined()) return;
  for (const Tensor* t : from)
    if (t->requires_grad()) {
      gradient = Once::apply(gradient, *t);
      return;
    }
}

// ---- tokens to their experts and back

struct Sorted {
  Tensor xs, offsets, position, source;
};

Sorted sort(const Tensor& x, const Tensor& index, int64_t E) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t N = x.size(0), C = x.size(1), k = index.size(1);
  const auto ints = index.options().dtype(torch::kInt32);
  Sorted r{at::empty({N * k, C}, x.options()), at::empty({E + 1}, ints), at::empty({N, k}, ints),
           at::empty({N * k}, ints)};
  const size_t need = camoe_ex_dispatch_work_bytes(N, k, E);
  const Tensor work = bytes(need, x);
  check(camoe_ex_dispatch(x.data_ptr(), dtype_of(x), index.data_ptr(), static_cast<int>(index.element_size()),
                          r.xs.data_ptr(), r.offsets.data_ptr<int32_t>(), r.position.data_ptr<int32_t>(),
                          r.source.data_ptr<int32_t>(), ptr(work), need, N, k, E, C, stream_of(x)));
  return r;
}

Tensor sum_rows(const Tensor& rows, const Tensor& weight, const Tensor& position) {
  const c10::cuda::CUDAGuard guard(rows.device());
  const int64_t N = position.size(0), k = position.size(1), C = rows.size(1);
  Tensor out = at::empty({N, C}, rows.options());
  check(camoe_ex_combine(rows.data_ptr(), dtype_of(rows), static_cast<const float*>(ptr(weight)),
                         position.data_ptr<int32_t>(), out.data_ptr(), N, k, C, stream_of(rows)));
  return out;
}

struct DispatchFn : torch::autograd::Function<DispatchFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& index, int64_t E, Sorted* plan) {
    *plan = sort(x, index, E);
    ctx->save_for_backward({plan->position});
    return plan->xs;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    out[0] = sum_rows(packed(grads[0]), Tensor(), ctx->get_saved_variables()[0]);
    once(out[0], {&grads[0]});
    return out;
  }
};

py::object dispatch(const Tensor& x, const Tensor& index, int64_t E) {
  if (x.dim() != 2 || index.dim() != 2 || !x.is_cuda() || !is_float(x) || !x.is_contiguous() ||
      (index.scalar_type() != torch::kInt64 && index.scalar_type() != torch::kInt32) || !index.is_contiguous() ||
      index.device() != x.device() || index.size(0) != x.size(0) || E < 1 || E > 1024 || index.size(1) < 1 ||
      index.size(1) > 64)
    return py::none();
  no_tangents("expert_dispatch", {&x});
  Sorted r;
  if (wants_grad({&x}))
    r.xs = DispatchFn::apply(x, index, E, &r);
  else
    r = sort(x, index, E);
  return py::make_tuple(r.xs, r.offsets, r.position, r.source);
}

struct CombineFn : torch::autograd::Function<CombineFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& ys, const Tensor& weight, const Tensor& offsets,
                        const Tensor& position) {
    ctx->save_for_backward({ys, weight, offsets, position});
    return sum_rows(ys, weight, position);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &ys = saved[0], &weight = saved[1], &offsets = saved[2], &position = saved[3];
    const c10::cuda::CUDAGuard guard(ys.device());
    const Tensor dout = packed(grads[0]);
    if (ctx->needs_input_grad(0)) out[0] = at::empty_like(ys);
    if (ctx->needs_input_grad(1)) out[1] = at::empty_like(weight);
    check(camoe_ex_combine_bwd(dout.data_ptr(), dtype_of(ys), ys.data_ptr(), weight.data_ptr<float>(),
                               offsets.data_ptr<int32_t>(), position.data_ptr<int32_t>(), ptr(out[0]),
                               static_cast<float*>(ptr(out[1])), position.size(0), position.size(1),
                               offsets.size(0) - 1, ys.size(1), stream_of(ys)));
    once(out[0], {&grads[0], &weight});
    once(out[1], {&grads[0], &ys});
    return out;
  }
};

py::object combine(const Tensor& ys, const Tensor& weight, const Tensor& offsets, const Tensor& position,
                   const Tensor& source) {
  if (!ys.is_cuda() || ys.dim() != 2 || !is_float(ys) || !ys.is_contiguous() || position.dim() != 2 ||
      offsets.dim() != 1 || offsets.size(0) < 2 || offsets.size(0) > 1025)
    return py::none();
  const int64_t N = position.size(0), k = position.size(1);
  const auto device = ys.device();
  if (k < 1 || k > 64 || ys.size(0) != N * k || !fits(weight, {N, k}, torch::kFloat32, device) ||
      !fits(position, {N, k}, torch::kInt32, device) ||
      !fits(offsets, {offsets.size(0)}, torch::kInt32, device) || !fits(source, {N * k}, torch::kInt32, device))
    return py::none();
  no_tangents("expert_combine", {&ys, &weight});
  return py::cast(wants_grad({&ys, &weight}) ? CombineFn::apply(ys, weight, offsets, position)
                                             : sum_rows(ys, weight, position));
}

// ---- the experts' products

struct Hidden {
  Tensor ys, h, low;
};

// `low`: h to 8 bits below bf16, for a backward that takes its root
Hidden ffn_forward(const Tensor& xs, const Tensor& w_up, const Tensor& w_down, const Tensor& offsets, bool low) {
  const c10::cuda::CUDAGuard guard(xs.device());
  const int64_t R = xs.size(0), C = xs.size(1), E = w_up.size(0), F = w_up.size(1);
  Hidden r{at::empty({R, C}, xs.options()), at::empty({R, F}, xs.options()), Tensor()};
  if (low) r.low = at::empty({R, (F + 15) / 16 * 16}, xs.options().dtype(torch::kInt8));
  check(camoe_ex_ffn_fwd(xs.data_ptr(), w_up.data_ptr(), w_down.data_ptr(), offsets.data_ptr<int32_t>(),
                         r.h.data_ptr(), ptr(r.low), r.ys.data_ptr(), R, E, C, F, stream_of(xs)));
  return r;
}

struct FfnFn : torch::autograd::Function<FfnFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& xs, const Tensor& w_up, const Tensor& w_down,
                        const Tensor& offsets) {
    const Hidden r = ffn_forward(xs, w_up, w_down, offsets, xs.requires_grad() || w_up.requires_grad());
    ctx->save_for_backward({xs, w_up, w_down, offsets, r.h, r.low});
    return r.ys;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list out(4);
    if (!grads[0].defined()) return out;
    const auto saved = ctx->get_saved_variables();
    const Tensor &xs = saved[0], &w_up = saved[1], &w_down = saved[2], &offsets = saved[3], &h = saved[4];
    const c10::cuda::CUDAGuard guard(xs.device());
    const Tensor dys = packed(grads[0]);
    for (int i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) out[i] = at::empty_like(saved[i]);
    const Tensor dpre = out[0].defined() || out[1].defined() ? at::empty_like(h) : Tensor();
    check(camoe_ex_ffn_bwd(dys.data_ptr(), xs.data_ptr(), w_up.data_ptr(), w_down.data_ptr(),
                           offsets.data_ptr<int32_t>(), h.data_ptr(), ptr(saved[5]), ptr(dpre), ptr(out[0]),
                           ptr(out[1]), ptr(out[2]), xs.size(0), w_up.size(0), xs.size(1), w_up.size(1),
                           stream_of(xs)));
    for (int i = 0; i < 2; ++i) once(out[i], {&grads[0], &xs, &w_up, &w_down});
    once(out[2], {&grads[0], &xs, &w_up});
    return out;
  }
};

py::object ffn(const Tensor& xs, const Tensor& w_up, const Tensor& w_down, const Tensor& offsets) {
  if (xs.dim() != 2 || w_up.dim() != 3 || !xs.is_cuda()) return py::none();
  const int64_t R = xs.size(0), C = xs.size(1), E = w_up.size(0), F = w_up.size(1);
  const auto device = xs.device();
  if (!fits(xs, {R, C}, torch::kBFloat16, device) || !fits(w_up, {E, F, C}, torch::kBFloat16, device) ||
      !fits(w_down, {E, C, F}, torch::kBFloat16, device) || !fits(offsets, {E + 1}, torch::kInt32, device) ||
      E < 1 || E > 1024 || C < 8 || F < 8 || C % 8 != 0 || F % 8 != 0 || !aligned({&xs, &w_up, &w_down}))
    return py::none();
  no_tangents("expert_ffn", {&xs, &w_up, &w_down});
  return py::cast(wants_grad({&xs, &w_up, &w_down}) ? FfnFn::apply(xs, w_up, w_down, offsets)
                                                    : ffn_forward(xs, w_up, w_down, offsets, false).ys);
}

// ---- adapters

py::object adapter_linear(const Tensor& x, const Tensor& weight, const Tensor& down, const Tensor& up,
                          const Tensor& adapter, const std::optional<Tensor>& scale) {
  if (x.dim() != 2 || weight.dim() != 2 || down.dim() != 3 || !x.is_cuda()) return py::none();
  const int64_t N = x.size(0), C = x.size(1), M = weight.size(0), L = down.size(0), D = down.size(1);
  const auto device = x.device();
  if (!fits(x, {N, C}, torch::kBFloat16, device) || !fits(weight, {M, C}, torch::kBFloat16, device) ||
      !fits(down, {L, D, C}, torch::kBFloat16, device) || !fits(up, {L, M, D}, torch::kBFloat16, device) ||
      !fits(adapter, {N}, torch::kInt32, device) || (scale && !fits(*scale, {L}, torch::kFloat32, device)) ||
      C < 8 || M < 8 || D < 8 || C % 8 != 0 || M % 8 != 0 || D % 8 != 0 || D > 256 || L < 1 || L > 1024 ||
      !aligned({&x, &weight, &down, &up}) || wants_grad({&x, &weight, &down, &up}) || (scale && wants_grad({&*scale})))
    return py::none();
  no_tangents("adapter_linear", {&x, &weight, &down, &up});
  if (scale) no_tangents("adapter_linear", {&*scale});
  const c10::cuda::CUDAGuard guard(device);
  Tensor y = at::empty({N, M}, x.options());
  const size_t need = camoe_ad_work_bytes(N, C, M, D, L);
  const Tensor work = bytes(need, x);
  check(camoe_ad_linear(x.data_ptr(), weight.data_ptr(), down.data_ptr(), up.data_ptr(), adapter.data_ptr<int32_t>(),
                        scale ? scale->data_ptr<float>() : nullptr, y.data_ptr(), ptr(work), need, N, C, M, D, L,
                        stream_of(x)));
  return py::cast(y);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      std::rethrow_exception(p);
    } catch (const Status& e) {
      try {
        py::module_::import("camoe_b200._lib").attr("check")(e.code);
      } catch (py::error_already_set& raised) {
        raised.restore();
      }
    }
  });
  m.def("dispatch", &dispatch);
  m.def("combine", &combine);
  m.def("ffn", &ffn);
  m.def("adapter_linear", &adapter_linear);
}
