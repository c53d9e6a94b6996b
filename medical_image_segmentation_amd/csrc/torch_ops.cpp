// The autograd nodes of group_norm_act and linear_act in C++ over the C-ABI.  A small training call of these operators is
// bound by the host: as Python nodes forward and backward took 125-140 us, of which the kernels were 20-50 (the engine
// runs a node's backward on a thread of its own, which has to take the interpreter's lock for a Python one).
// Arguments are checked by the Python functions that call in here (functional.py); scratch comes from torch's caching
// allocator, whose blocks belong to the stream, or to the graph being captured.
#include <torch/extension.h>

#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>

#include <unordered_set>
#include <vector>

#include "../../include/misamd.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

int dtype_of(const Tensor& t) { return t.scalar_type() == at::kFloat ? MIS_F32 : MIS_BF16; }
mis_stream_t stream() { return (mis_stream_t)c10::hip::getCurrentHIPStream().stream(); }
Tensor scratch(size_t bytes, const Tensor& like) { return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)); }
template <typename T = void> T* ptr(const Tensor& t) { return t.defined() ? (T*)t.data_ptr() : nullptr; }
Tensor dense(const Maybe& t) { return t && t->defined() ? t->contiguous() : Tensor(); }

// Which inputs want a gradient in this pass: a node has edges only for the tensors that were given.
struct Wanted {
  AutogradContext* ctx;
  size_t edge = 0;
  bool next(bool given) { return given && ctx->needs_input_grad(edge++); }
};

void check(int rc, const char* name) {
  TORCH_CHECK(rc == MIS_OK, name, " failed (status ", rc, "): ", mis_last_error());
}

// A backward pass under capture must not reach a leaf whose gradient node was made on the default stream, which cannot join
// a capture: the node lives as long as any graph that uses the leaf, here one from before the capture.  (The engine would
// wait on that stream at the end of the pass and the capture would end with the process.)  Looked at are all leaves that this
// pass will reach from the running node on, behind views, casts and other operations too; only under capture, so that
// walking the graph costs an eager pass nothing.
void refuse_stale_leaves(const char* name) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  const auto running = torch::autograd::get_current_node();
  if (!running) return;
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();       // empty: all nodes are executed
  std::vector<torch::autograd::Node*> todo{running.get()};
  std::unordered_set<torch::autograd::Node*> seen;
  while (!todo.empty()) {
    torch::autograd::Node* node = todo.back();
    todo.pop_back();
    for (const auto& edge : node->next_edges()) {
      torch::autograd::Node* next = edge.function.get();
      if (!next || !seen.insert(next).second) continue;
      if (wanted && !wanted->empty()) {
        const auto found = wanted->find(next);
        if (found == wanted->end() || !found->second.should_execute()) continue;
      }
      if (!next->next_edges().empty()) {
        todo.push_back(next);
        continue;
      }
      const auto made_on = next->stream();
      TORCH_CHECK(!made_on || made_on->id() != c10::hip::getDefaultHIPStream(made_on->device_index()).id(), name,
                  ": an eager graph of the same leaf is alive; drop the tensors that hold it (outputs, losses) before capturing "
                  "a backward pass");
    }
  }
}

// Gradients that raise when they are differentiated with respect to what they were formed from: the backward is not
// differentiable itself.
variable_list once(variable_list grads, bool twice, const variable_list& from, const char* name) {
  if (!twice) return grads;
  at::AutoGradMode grad_mode(true);
  std::shared_ptr<torch::autograd::Node> error(
      new torch::autograd::Error(std::string(name) + " is differentiable once", torch::autograd::collect_next_edges(from)),
      torch::autograd::deleteNode);
  for (auto& g : grads)
    if (g.defined()) {
      g = g.detach();
      torch::autograd::set_history(g, error);
    }
  return grads;
}

struct GroupNormAct : torch::autograd::Function<GroupNormAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Maybe& weight, const Maybe& bias, int64_t groups, double eps,
                        int64_t act) {
    c10::DeviceGuard guard(x.device());
    const Tensor w = dense(weight), b = dense(bias);
    const int64_t B = x.size(0), C = x.size(1), HW = x.size(2) * x.size(3);
    TORCH_CHECK(B <= INT32_MAX && C <= INT32_MAX, "group_norm_act: ", B, " samples of ", C, " channels are too many");
    Tensor y = at::empty_like(x, at::MemoryFormat::ChannelsLast);
    Tensor stats = at::empty({B, groups, 2}, x.options().dtype(at::kDouble));
    if (x.numel()) {
      const Tensor ws = scratch(mis_group_norm_act_fwd_workspace_bytes(dtype_of(x), B, HW, C, groups), x);
      check(mis_group_norm_act_fwd(ptr(x), dtype_of(x), B, HW, C, groups, ptr<float>(w), ptr<float>(b), eps, act, ptr(y),
                                   ptr<double>(stats), ptr(ws), stream()), "mis_group_norm_act_fwd");
    }
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["groups"] = groups;
    ctx->saved_data["act"] = act;
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
    const int64_t groups = ctx->saved_data["groups"].toInt(), act = ctx->saved_data["act"].toInt();
    const bool twice = at::GradMode::is_enabled();         // create_graph=True
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(x.device());
    refuse_stale_leaves("group_norm_act");
    const int64_t B = x.size(0), C = x.size(1), HW = x.size(2) * x.size(3);
    const bool some = x.numel() > 0;
    Tensor dx, dw, db;
    Wanted wanted{ctx};
    if (wanted.next(true)) dx = at::empty_like(x, at::MemoryFormat::ChannelsLast);
    const auto f32 = x.options().dtype(at::kFloat);
    if (wanted.next(w.defined())) dw = some ? at::empty({C}, f32) : at::zeros({C}, f32);
    if (wanted.next(b.defined())) db = some ? at::empty({C}, f32) : at::zeros({C}, f32);
    if (some) {
      const Tensor dy = grad[0].to(x.scalar_type()).contiguous(at::MemoryFormat::ChannelsLast);
      const Tensor ws = scratch(mis_group_norm_act_bwd_workspace_bytes(dtype_of(x), B, HW, C, groups), x);
      check(mis_group_norm_act_bwd(ptr(x), ptr(dy), dtype_of(x), B, HW, C, groups, ptr<float>(w), ptr<float>(b),
                                   ptr<double>(stats), act, ptr(dx), ptr<float>(dw), ptr<float>(db), ptr(ws), stream()),
            "mis_group_norm_act_bwd");
    }
    return once({dx, dw, db, Tensor(), Tensor(), Tensor()}, twice, {x, w, b, grad[0]}, "group_norm_act");
  }
};

// [..., n] -> rows of n consecutive elements and their stride; a copy only where the strides need one
Tensor as_rows(const Tensor& t, int64_t n, int64_t& ld) {
  ld = n;
  if (!t.defined() || t.is_contiguous()) return t;
  Tensor r = t.reshape({-1, n});
  if ((n > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < n)) r = r.contiguous();
  if (r.size(0) > 1) ld = r.stride(0);
  return r;
}

struct LinearAct : torch::autograd::Function<LinearAct> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& residual,
                        int64_t act) {
    c10::DeviceGuard guard(x.device());
    const int64_t N = weight.size(0), K = weight.size(1), M = x.numel() / K;
    const Tensor w = weight.contiguous(), b = dense(bias);
    int64_t ldx, ldr;
    const Tensor rows = as_rows(x, K, ldx), res = as_rows(residual ? *residual : Tensor(), N, ldr);
    auto shape = x.sizes().vec();
    shape.back() = N;
    Tensor y = at::empty(shape, x.options());
    if (M) {
      const Tensor ws = scratch(mis_linear_act_fwd_workspace_bytes(dtype_of(x), M, N, K), x);
      check(mis_linear_act_fwd(ptr(rows), ldx, ptr(w), ptr<float>(b), ptr(res), ldr, dtype_of(x), M, N, K, act, ptr(y), ptr(ws),
                               stream()), "mis_linear_act_fwd");
    }
    ctx->save_for_backward({x, w, b});
    ctx->saved_data["act"] = act;
    ctx->saved_data["residual"] = res.defined();
    return y;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const int64_t act = ctx->saved_data["act"].toInt();
    const bool twice = at::GradMode::is_enabled();         // create_graph=True
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(x.device());
    refuse_stale_leaves("linear_act");
    const int64_t N = w.size(0), K = w.size(1), M = x.numel() / K;
    Tensor dx, dw, db, dr;
    Wanted wanted{ctx};
    const bool need_x = wanted.next(true), need_w = wanted.next(true), need_b = wanted.next(b.defined());
    if (wanted.next(ctx->saved_data["residual"].toBool())) dr = grad[0];
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_w) dw = M ? at::empty({N, K}, x.options()) : at::zeros({N, K}, x.options());
    const auto f32 = x.options().dtype(at::kFloat);
    if (need_b) db = M ? at::empty({N}, f32) : at::zeros({N}, f32);
    if (M && (need_x || need_w || need_b)) {
      int64_t ldx, ldd;
      const Tensor rows = as_rows(x, K, ldx), dy = as_rows(grad[0].to(x.scalar_type()), N, ldd);
      const Tensor ws = scratch(mis_linear_act_bwd_workspace_bytes(dtype_of(x), M, N, K, act), x);
      check(mis_linear_act_bwd(ptr(rows), ldx, ptr(w), ptr<float>(b), ptr(dy), ldd, dtype_of(x), M, N, K, act, ptr(dx), ptr(dw),
                               ptr<float>(db), ptr(ws), stream()), "mis_linear_act_bwd");
    }
    return once({dx, dw, db, dr, Tensor()}, twice, {x, w, b, grad[0]}, "linear_act");
  }
};

Tensor group_norm_act(const Tensor& x, const Maybe& weight, const Maybe& bias, int64_t groups, double eps, int64_t act) {
  return GroupNormAct::apply(x, weight, bias, groups, eps, act);
}

Tensor linear_act(const Tensor& x, const Tensor& weight, const Maybe& bias, const Maybe& residual, int64_t act) {
  return LinearAct::apply(x, weight, bias, residual, act);
}

// The types, devices, shapes and strides of parameters: what an optimizer's tables of them hold good for.  A Parameter stays
// the same object when its module is converted (Module.to, .bfloat16) or its .data replaced, so these are compared at every
// step; in C++, since the interpreter would take as long for it as the step's launches.
class Layouts {
 public:
  explicit Layouts(std::vector<Tensor> params) : params_(std::move(params)) {
    for (const Tensor& p : params_) kept_.push_back({p.scalar_type(), p.device(), p.sizes().vec(), p.strides().vec()});
  }
  bool hold() const {
    for (size_t i = 0; i < params_.size(); i++) {
      const Tensor& p = params_[i];
      const One& k = kept_[i];
      if (p.scalar_type() != k.type || p.device() != k.device || p.sizes() != at::IntArrayRef(k.sizes) ||
          p.strides() != at::IntArrayRef(k.strides))
        return false;
    }
    return true;
  }

 private:
  struct One {
    at::ScalarType type;
    at::Device device;
    std::vector<int64_t> sizes, strides;
  };
  std::vector<Tensor> params_;
  std::vector<One> kept_;
};

// Whether the values of an optimizer's `state` are still these dicts, in this order, and hold these entries one dict after the
// other (None: any): a user may clear the state, or put other dicts or tensors in its place.  Dicts keep their order, so
// nothing is looked up by its key.
bool state_holds(const pybind11::dict& state, const pybind11::list& dicts, const pybind11::list& entries) {
  const Py_ssize_t n = PyList_GET_SIZE(dicts.ptr()), m = PyList_GET_SIZE(entries.ptr());
  if (PyDict_Size(state.ptr()) != n) return false;
  PyObject *key, *value, *entry;
  Py_ssize_t at = 0, e = 0;
  for (Py_ssize_t i = 0; PyDict_Next(state.ptr(), &at, &key, &value); i++) {
    if (value != PyList_GET_ITEM(dicts.ptr(), i) || !PyDict_Check(value)) return false;
    for (Py_ssize_t in = 0; PyDict_Next(value, &in, &key, &entry); e++) {
      if (e >= m) return false;
      PyObject* held = PyList_GET_ITEM(entries.ptr(), e);
      if (held != Py_None && held != entry) return false;
    }
  }
  return e == m;
}

// The pointers [parameter, gradient, parameter, ...] of parameters whose gradients lie in the same memory order, type and
// device; empty if one does not (the caller then looks at them one by one).
std::vector<int64_t> step_pointers(const std::vector<Tensor>& params, int64_t device) {
  std::vector<int64_t> out;
  out.reserve(2 * params.size());
  for (const Tensor& p : params) {
    const Tensor& g = p.grad();
    if (!g.defined() || g.is_sparse() || g.scalar_type() != p.scalar_type() || g.get_device() != device ||
        p.get_device() != device || !(g.is_contiguous() && p.is_contiguous()) || g.sizes() != p.sizes())
      return {};
    out.push_back((int64_t)p.data_ptr());
    out.push_back((int64_t)g.data_ptr());
  }
  return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("group_norm_act", &group_norm_act, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("linear_act", &linear_act, pybind11::call_guard<pybind11::gil_scoped_release>());
  m.def("step_pointers", &step_pointers);
  m.def("state_holds", &state_holds);
  pybind11::class_<Layouts>(m, "Layouts").def(pybind11::init<std::vector<Tensor>>()).def("hold", &Layouts::hold);
}
