// Autograd nodes of linear_act and distill_ce, and the call of top_logits
// (ops.nn, ops.loss).
//
// The kernels of both take tens of microseconds at the sizes of a classifier's
// head.  As Python autograd functions their host path took longer than that: the
// backward runs on the engine's thread, which waits for the interpreter and then
// runs it from cold caches (measured: 39 us in a function that takes 12 us when
// it is called in a loop).  These nodes make the same calls of libcerebro_hip.so
// without the interpreter.  Arguments are checked by the Python callers.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <initializer_list>
#include <optional>

#include "../hip/nodes_api.h"

using torch::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

static hipStream_t stream_of(const Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

// sizes go to the kernels as int
static void ints(const char* name, std::initializer_list<int64_t> sizes) {
  for (int64_t n : sizes)
    TORCH_CHECK_VALUE(n <= INT32_MAX, name, ": ", n, " rows or columns are more than 2^31 - 1");
}

static void done(int rc, const char* name) {
  TORCH_CHECK(rc == 0, name, " failed with hipError ", rc);
}

// What a tracer would record of these calls are the empty outputs, and what a dual
// number would get is no tangent, that is a derivative of zero: both are refused.
static void eager_and_reverse(const char* name, std::initializer_list<const Tensor*> inputs) {
  using c10::impl::TorchDispatchModeKey;
  using c10::impl::TorchDispatchModeTLS;
  TORCH_CHECK_NOT_IMPLEMENTED(
      !torch::jit::tracer::isTracing() && !TorchDispatchModeTLS::get_mode(TorchDispatchModeKey::PROXY),
      name, " cannot be traced");
  for (const Tensor* t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t->defined() || !t->_fw_grad(0).defined(), name,
                                " has no forward-mode derivative");
}

static void once(const char* name) {
  TORCH_CHECK(!at::GradMode::is_enabled(), name,
              " has no second derivative (its backward ran with create_graph=True)");
}

static Tensor floats(const Tensor& like, int64_t n) {
  return n > 0 ? at::empty({n}, like.options().dtype(at::kFloat)) : Tensor();
}

static float* fptr(const Tensor& t) { return t.defined() ? t.data_ptr<float>() : nullptr; }

// All that a backward reads goes through SavedVariable: hooks on saved tensors
// (offload, checkpoints) see it, and an input that was written in between is
// refused.  An inference tensor counts no writes; it is copied.  What a hook gives
// back is read by kernels: other sizes, types or devices are refused, another layout
// is copied (elements of a row adjacent, a matrix's pitch at least its width).
class Saved {
  SavedVariable v_;
  at::ScalarType type_ = at::kFloat;
  at::DimVector sizes_;

 public:
  Saved() = default;
  explicit Saved(const Tensor& t)
      : v_(t.defined() && t.is_inference() ? t.clone() : t, false) {
    if (!t.defined()) return;
    type_ = t.scalar_type();
    sizes_ = t.sizes();
  }

  Tensor unpack(const c10::Device& device) const {
    const Tensor t = v_.unpack();
    if (!t.defined()) return t;
    TORCH_CHECK(t.scalar_type() == type_ && t.sizes() == sizes_ && t.device() == device &&
                    t.layout() == at::kStrided,
                "a hook on saved tensors gave back ", t.scalar_type(), " ", t.sizes(), " on ",
                t.device(), " for ", type_, " ", at::IntArrayRef(sizes_), " on ", device);
    const int64_t last = t.dim() - 1;
    const bool adjacent = last < 0 || ((t.size(last) <= 1 || t.stride(last) == 1) &&
                                       (last != 1 || t.stride(0) >= t.size(1)));
    return adjacent ? t : t.clone(at::MemoryFormat::Contiguous);
  }

  void free() { v_.reset_data(); }
};

// ---------------------------------------------------------------------------
struct Dense {
  Tensor work, grad;            // the arena's rows [G, n]
  int64_t w_off, b_off;         // elements in a row; b_off < 0: no bias
  int64_t M, N, K, G, act;
  bool bf16;

  char* at_(const Tensor& t, int64_t off) const {
    return off < 0 ? nullptr : static_cast<char*>(t.data_ptr()) + off * t.element_size();
  }
};

struct LinearActBackward : public Node {
  Dense p;
  Saved x, derivative;          // act'(z)

  variable_list apply(variable_list&& grads) override {
    variable_list out(3);
    const Tensor g0 = grads[0];
    if (!g0.defined()) return out;
    once("linear_act");
    const Tensor xv = x.unpack(p.work.device());
    Tensor d = derivative.unpack(p.work.device());
    if (d.defined()) d = d.contiguous();
    const c10::OptionalDeviceGuard guard(xv.device());
    const Tensor dy = g0.contiguous();
    const bool need_dx = task_should_compute_output(0);
    const int64_t n = cer_dense_ws(1, p.M, p.N, p.K, p.G, p.bf16, p.act);
    TORCH_CHECK(n >= 0, "linear_act: sizes out of range");
    // one temporary: the workspace and dz
    const Tensor tmp = floats(xv, n + (p.act ? p.M * p.G * p.N : 0));
    if (need_dx) out[0] = at::empty({p.M, p.G * p.K}, xv.options());
    done((p.bf16 ? cer_dense_bwd : cer_dense_bwd_f32)(
             dy.data_ptr(), d.defined() ? d.data_ptr() : nullptr, p.act ? fptr(tmp) + n : nullptr,
             xv.data_ptr(), xv.stride(0), p.at_(p.work, p.w_off), p.work.stride(0),
             need_dx ? out[0].data_ptr() : nullptr, (float*)p.at_(p.grad, p.w_off),
             p.grad.stride(0), (float*)p.at_(p.grad, p.b_off), p.grad.stride(0), p.M, p.N, p.K,
             p.G, p.act, n ? fptr(tmp) : nullptr, n, stream_of(xv)),
         "cer_dense_bwd");
    if (task_should_compute_output(2)) out[2] = g0;
    return out;
  }

  void release_variables() override {
    x.free();
    derivative.free();
  }
};

// x [M, G K] and residual [M, G N] with adjacent columns; w_off, b_off: the
// parameters' elements in the arena's rows
static Tensor linear_act(const Tensor& x, const std::optional<Tensor>& anchor,
                         const std::optional<Tensor>& residual, const Tensor& work,
                         const std::optional<Tensor>& grad, int64_t w_off, int64_t b_off, int64_t N,
                         int64_t K, int64_t act, bool train) {
  eager_and_reverse("linear_act",
                    {&x, anchor ? &*anchor : &x, residual ? &*residual : &x, &work});
  ints("linear_act", {x.size(0), x.size(1), work.size(0) * N});
  // statistics live behind the parameters and have no gradient
  TORCH_CHECK_VALUE(w_off >= 0 && w_off + N * K <= work.size(1) && b_off + N <= work.size(1),
                    "linear_act: the weight or bias is no trainable parameter of its arena");
  const c10::OptionalDeviceGuard guard(x.device());
  Dense p{work, grad.value_or(Tensor()), w_off, b_off, x.size(0), N, K, work.size(0), act,
          x.scalar_type() == at::kBFloat16};
  const int64_t n = cer_dense_ws(0, p.M, N, K, p.G, p.bf16, act);
  TORCH_CHECK_VALUE(n >= 0 && (!train || cer_dense_ws(1, p.M, N, K, p.G, p.bf16, act) >= 0),
                    "linear_act: M=", p.M, " N=", N, " K=", K, " G=", p.G,
                    " is beyond the kernels' 32-bit offsets and grids");
  const Tensor ws = floats(x, n);
  Tensor y = at::empty({p.M, p.G * N}, x.options());
  Tensor d;
  if (train && act)
    d = at::empty({p.M, p.G * N}, x.options().dtype(act > 6 ? at::kFloat : at::kByte));
  done((p.bf16 ? cer_dense_fwd : cer_dense_fwd_f32)(
           x.data_ptr(), x.stride(0), p.at_(work, w_off), work.stride(0), p.at_(work, b_off),
           work.stride(0), residual ? residual->data_ptr() : nullptr,
           residual ? residual->stride(0) : 0, y.data_ptr(), d.defined() ? d.data_ptr() : nullptr,
           p.M, N, K, p.G, act, fptr(ws), n, stream_of(x)),
       "cer_dense_fwd");
  if (train) {
    auto node = std::shared_ptr<LinearActBackward>(new LinearActBackward(),
                                                   torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, anchor.value_or(Tensor()),
                                                             residual.value_or(Tensor())));
    node->p = std::move(p);
    node->x = Saved(x);
    node->derivative = Saved(d);
    torch::autograd::set_history(y, node);
  }
  return y;
}

// ---------------------------------------------------------------------------
struct Teacher {
  Tensor labels, val, idx, alpha, tau;
  double alpha0, tau0;
};

// read again in the backward, beside sums that the forward made of them
struct SavedTeacher {
  Saved labels, val, idx, alpha, tau;
  double alpha0 = 0, tau0 = 0;

  SavedTeacher() = default;
  explicit SavedTeacher(const Teacher& t)
      : labels(t.labels), val(t.val), idx(t.idx), alpha(t.alpha), tau(t.tau), alpha0(t.alpha0),
        tau0(t.tau0) {}

  Teacher unpack(const c10::Device& device) const {
    Teacher t{labels.unpack(device).contiguous(), val.unpack(device), idx.unpack(device),
              alpha.unpack(device), tau.unpack(device), alpha0, tau0};
    if (t.alpha.defined()) t.alpha = t.alpha.contiguous();
    if (t.tau.defined()) t.tau = t.tau.contiguous();
    return t;
  }
};

struct DistillBackward : public Node {
  SavedTeacher teacher;
  Saved z, stats;
  Saved finished;               // the gradient for a unit loss gradient
  c10::Device device = c10::kCUDA;
  int64_t G;
  bool unit;

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    once("distill_ce");
    if (unit) {
      const Tensor d = finished.unpack(device);
      // a graph that is kept may be run again: the caller may write its gradient
      out[0] = torch::autograd::get_current_graph_task_keep_graph() ? d.clone() : d;
      return out;
    }
    const Tensor zv = z.unpack(device);
    const Tensor sums = stats.unpack(device).contiguous();
    const Teacher t = teacher.unpack(device);
    const c10::OptionalDeviceGuard guard(zv.device());
    const Tensor dloss = grads[0].contiguous();
    const bool bf16 = zv.scalar_type() == at::kBFloat16;
    out[0] = at::empty({zv.size(0), zv.size(1)}, zv.options());
    done((bf16 ? cer_distill_bwd : cer_distill_bwd_f32)(
             zv.data_ptr(), zv.stride(0), t.labels.data_ptr<int>(), t.val.data_ptr(),
             t.val.scalar_type() == at::kFloat, t.val.stride(0), t.val.stride(1),
             t.idx.data_ptr<int>(), t.idx.stride(0), t.idx.stride(1), fptr(t.alpha), t.alpha0,
             fptr(t.tau), t.tau0, fptr(dloss), fptr(sums), out[0].data_ptr(), zv.size(0), G,
             zv.size(1) / G, t.val.size(2), stream_of(zv)),
         "cer_distill_bwd");
    return out;
  }

  void release_variables() override {
    z.free();
    stats.free();
    finished.free();
    teacher = SavedTeacher();
  }
};

static Tensor distill_ce(const Tensor& z, const Tensor& labels, const Tensor& acc, int64_t G,
                         const Tensor& val, const Tensor& idx, const std::optional<Tensor>& alpha,
                         double alpha0, const std::optional<Tensor>& tau, double tau0, bool unit,
                         bool train) {
  eager_and_reverse("distill_ce", {&z, &val, alpha ? &*alpha : &z, tau ? &*tau : &z});
  const bool bf16 = z.scalar_type() == at::kBFloat16;
  const int64_t B = z.size(0), N = z.size(1) / G;
  ints("distill_ce", {B, G, N});
  const c10::OptionalDeviceGuard guard(z.device());
  const int64_t n = cer_distill_ws(B, G, N, bf16);
  TORCH_CHECK_VALUE(n >= 0, "distill_ce: B=", B, " G=", G, " N=", N,
                    " is beyond the kernels' grids");
  Tensor loss = at::empty({G}, z.options().dtype(at::kFloat));
  Tensor buf = floats(z, 4 * G * B + n);        // stats for the backward, workspace
  Tensor d;
  if (train && unit) d = at::empty({B, z.size(1)}, z.options());
  Teacher t{labels, val, idx, alpha.value_or(Tensor()), tau.value_or(Tensor()), alpha0, tau0};
  done((bf16 ? cer_distill_fwd : cer_distill_fwd_f32)(
           z.data_ptr(), z.stride(0), labels.data_ptr<int>(), val.data_ptr(),
           val.scalar_type() == at::kFloat, val.stride(0), val.stride(1), idx.data_ptr<int>(),
           idx.stride(0), idx.stride(1), fptr(t.alpha), alpha0, fptr(t.tau), tau0, fptr(buf),
           d.defined() ? d.data_ptr() : nullptr, fptr(loss), acc.data_ptr<float>(), B, G, N,
           val.size(2), fptr(buf) + 4 * G * B, n, stream_of(z)),
       "cer_distill_fwd");
  if (train) {
    auto node = std::shared_ptr<DistillBackward>(new DistillBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(z));
    node->G = G;
    node->unit = unit;
    node->device = z.device();
    if (unit) {
      node->finished = Saved(d);
    } else {
      node->z = Saved(z);
      node->teacher = SavedTeacher(t);
      node->stats = Saved(buf.narrow(0, 0, 4 * G * B));
    }
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

// ---------------------------------------------------------------------------
static std::tuple<Tensor, Tensor> top_logits(const Tensor& z, int64_t G, int64_t k) {
  eager_and_reverse("top_logits", {});
  const bool bf16 = z.scalar_type() == at::kBFloat16;
  const int64_t B = z.size(0), N = z.size(1) / G;
  ints("top_logits", {B * G, N});
  const c10::OptionalDeviceGuard guard(z.device());
  const int64_t n = cer_top_ws(B, G, N, k, bf16);
  TORCH_CHECK_VALUE(n >= 0, "top_logits: B=", B, " G=", G, " N=", N, " k=", k,
                    " is beyond the kernels' grids");
  Tensor val = at::empty({G, B, k}, z.options());
  Tensor idx = at::empty({G, B, k}, z.options().dtype(at::kInt));
  Tensor ws = n > 0 ? at::empty({n}, z.options().dtype(at::kLong)) : Tensor();
  done((bf16 ? cer_top_logits : cer_top_logits_f32)(
           z.data_ptr(), z.stride(0), val.data_ptr(), idx.data_ptr<int>(), B, G, N, k,
           ws.defined() ? ws.data_ptr<int64_t>() : nullptr, n > 0 ? n : 0, stream_of(z)),
       "cer_top_logits");
  return {val, idx};
}

PYBIND11_MODULE(cerebro_nodes, m) {
  m.def("top_logits", &top_logits);
  m.def("linear_act", &linear_act);
  m.def("distill_ce", &distill_ce);
}
