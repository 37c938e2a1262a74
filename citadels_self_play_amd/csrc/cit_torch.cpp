// The training operators' path from torch to the C ABI (include/citadels.h):
// outputs and workspaces from torch's allocator, the current stream, and the
// autograd nodes.  ops.py checks the arguments of the linear layer and the
// policy loss; what it hands over is of the shapes, types and devices that it
// says.  Lists of gradients, which may be long, are checked here.
//
// The nodes are C++ because a backward pass runs on torch's own thread for the
// device: a Python one has to be woken there with the interpreter's lock, in
// another core's caches (64 x 418 -> 512, forward and backward, host time:
// 109 us with Python nodes, 58 with these; a ReLU's own takes 46).
#include <hip/hip_runtime_api.h>
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <c10/hip/HIPStream.h>

#include <mutex>
#include <optional>

#include "../../include/citadels.h"

namespace {

using at::Tensor;
using torch::autograd::collect_next_edges;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

struct NativeError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

// The library's entry points, by address: the one that is loaded, whichever file it came from.
struct Api {
  decltype(&cit_linear_forward_work_bytes) linear_forward_work_bytes;
  decltype(&cit_linear_forward) linear_forward;
  decltype(&cit_linear_backward_work_bytes) linear_backward_work_bytes;
  decltype(&cit_linear_backward) linear_backward;
  decltype(&cit_policy_loss_work_bytes) policy_loss_work_bytes;
  decltype(&cit_policy_loss) policy_loss;
  decltype(&cit_policy_loss_backward) policy_loss_backward;
  decltype(&cit_clip_grad_norm_work_bytes) clip_grad_norm_work_bytes;
  decltype(&cit_clip_grad_norm) clip_grad_norm;
} api;

void check(int rc, const char* what) {
  if (rc) throw NativeError(std::string(what) + " failed with code " + std::to_string(rc));
}

int type_of(const Tensor& t) {
  return t.scalar_type() == at::kFloat ? CIT_FP32 : t.scalar_type() == at::kBFloat16 ? CIT_BF16 : CIT_FP16;
}
const void* address(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* writable(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }

// The device as the current one, and its current stream.
struct On {
  c10::DeviceGuard guard;
  hipStream_t stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};

Tensor workspace(size_t bytes, const Tensor& like) {
  return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : Tensor();
}

// A number of the capture that the stream is part of; 0: none.
unsigned long long capture_of(hipStream_t stream) {
  hipStreamCaptureStatus s = hipStreamCaptureStatusNone;
  unsigned long long id = 0;
  if (hipStreamGetCaptureInfo(stream, &s, &id) != hipSuccess) {
    (void)hipGetLastError();             // not the next launch's
    return 0;
  }
  return s == hipStreamCaptureStatusNone ? 0 : id + 1;
}
bool capturing(hipStream_t stream) { return capture_of(stream) != 0; }

// `t` as [rows][width] with its entries side by side, and the elements between rows.
Tensor as_rows(const Tensor& t, int64_t rows, int64_t width, int64_t& ld) {
  const Tensor r = t.resolve_neg(), m = r.dim() == 2 ? r : r.reshape({rows, width});
  ld = width;
  if (m.is_contiguous()) return m;
  if ((width > 1 && m.stride(1) != 1) || (rows > 1 && m.stride(0) < width)) return m.contiguous();
  if (rows > 1) ld = m.stride(0);
  return m;
}

bool wanted(const Tensor& t) { return t.defined() && t.requires_grad(); }

void first_only(const char* what) {
  if (at::GradMode::is_enabled())
    throw std::runtime_error(std::string("ops.") + what +
                             " has first derivatives only: its backward pass cannot run with create_graph=True");
}
// A backward pass under capture hands its gradients to its leaves' nodes, on the streams that these were made on.  A
// node that an eager graph keeps alive has a stream outside the capture, and torch's engine, joining the two, would
// end the process: refused while that is still an error.
void leaves_in_capture(const torch::autograd::Node& node, hipStream_t stream, const char* what) {
  if (!capturing(stream)) return;
  for (size_t i = 0; i < node.num_outputs(); i++) {
    const auto& leaf = node.next_edge(i).function;
    if (!leaf || !node.task_should_compute_output(i) || !dynamic_cast<torch::autograd::AccumulateGrad*>(leaf.get()))
      continue;
    const std::optional<c10::Stream> s = leaf->stream();
    if (!s) continue;
    const hipStream_t other = c10::hip::HIPStream(c10::hip::HIPStream::UNCHECKED, *s).stream();
    if (other != stream && (!other || !capturing(other)))
      throw std::runtime_error(std::string("ops.") + what +
                               ": a backward pass cannot be captured while an eager graph of the same leaves is alive");
  }
}

// torch.func's and vmap's tensors stand for others and have no memory; nor have batched gradients.
void own_memory(std::initializer_list<Tensor> given, const char* what) {
  for (const Tensor& t : given)
    if (t.defined() && !t.has_storage())
      throw py::value_error(std::string("ops.") + what + " takes no tensors of torch.func or vmap");
}
void one_gradient(const Tensor& t, const char* what) {
  if (!t.has_storage())
    throw std::runtime_error(std::string("ops.") + what +
                             ": its backward pass takes one gradient, not a batch of them (is_grads_batched, vmap)");
}

void no_tangent(std::initializer_list<Tensor> given, const char* what) {
  for (const Tensor& t : given)
    if (t.defined() && t._fw_grad(0).defined())
      throw std::runtime_error(std::string("ops.") + what + " has no forward-mode derivatives");
}

// ---- linear ---------------------------------------------------------------------

struct LinearBackward : torch::autograd::Node {
  SavedVariable x, w, z;                 // z: the pre-activation, or y itself (own_y)
  bool own_y = false;
  std::vector<int64_t> shape;            // of x
  int64_t M = 0, N = 0, K = 0;
  int act = 0;

  std::string name() const override { return "LinearBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(), w.reset_data(), z.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(4);
    const Tensor& dy = grads[0];
    if (!dy.defined()) return out;
    first_only("linear");
    one_gradient(dy, "linear");
    const On on(dy);
    leaves_in_capture(*this, on.stream, "linear");
    const bool nx = task_should_compute_output(0), nw = task_should_compute_output(1),
               nb = task_should_compute_output(2);
    if (task_should_compute_output(3)) out[3] = dy;
    if (!(nx || nw || nb)) return out;
    Tensor vx = nw ? x.unpack() : Tensor(), vw = nx ? w.unpack() : Tensor();
    Tensor vz = act ? z.unpack(own_y ? shared_from_this() : nullptr) : Tensor();
    const auto make = [&](at::IntArrayRef size, bool yes) {
      return !yes ? Tensor() : M && N ? at::empty(size, dy.options()) : at::zeros(size, dy.options());
    };
    out[0] = make(shape, nx), out[1] = make({N, K}, nw), out[2] = make({N}, nb);
    if (!(M && N)) return out;
    int64_t ldy, ldx = K, ldw = K;
    const Tensor d = as_rows(dy, M, N, ldy);
    if (nw) vx = as_rows(vx, M, K, ldx);
    if (nx) vw = as_rows(vw, N, K, ldw);
    if (vz.defined()) vz = vz.contiguous();
    const int t = type_of(dy);
    const void *px = address(vx), *pw = address(vw);
    void *dx = writable(out[0]), *dw = writable(out[1]), *db = writable(out[2]);
    const size_t n = api.linear_backward_work_bytes(px, ldx, pw, ldw, dx, dw, db, M, N, K, t, act);
    const Tensor work = workspace(n, dy);
    check(api.linear_backward(address(d), ldy, address(vz), px, ldx, pw, ldw, dx, dw, db, M, N, K, t, act,
                              writable(work), n, on.stream),
          "cit_linear_backward");
    return out;
  }
};

Tensor linear(const Tensor& x, const Tensor& w, const Maybe& bias, const Maybe& residual, int act) {
  const Tensor b = bias.value_or(Tensor()), r = residual.value_or(Tensor());
  own_memory({x, w, b, r}, "linear");
  std::shared_ptr<LinearBackward> node;
  if (at::GradMode::is_enabled() && (wanted(x) || wanted(w) || wanted(b) || wanted(r))) {
    node = std::shared_ptr<LinearBackward>(new LinearBackward(), torch::autograd::deleteNode);
    node->set_next_edges(collect_next_edges(x, w, b, r));
  }
  no_tangent({x, w, b, r}, "linear");
  const int64_t K = w.size(1), N = w.size(0);
  int64_t M = 1;
  for (int64_t i = 0; i + 1 < x.dim(); i++) M *= x.size(i);
  std::vector<int64_t> shape = x.sizes().vec();
  // relu without a residual leaves its sign in y (fp16 aside, where a small y rounds to 0); other activations need
  // the pre-activation
  const bool own_y = act == 1 && !r.defined() && x.scalar_type() != at::kHalf;
  Tensor y, z;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const On on(x);
    std::vector<int64_t> size = shape;
    size.back() = N;
    y = at::empty(size, x.options());
    if (node && act && !own_y) z = at::empty({M, N}, x.options());
    if (M && N) {
      int64_t ldx, ldw, ldr = N;
      const Tensor vx = as_rows(x, M, K, ldx), vw = as_rows(w, N, K, ldw);
      const Tensor vr = r.defined() ? as_rows(r, M, N, ldr) : r, vb = b.defined() ? b.contiguous() : b;
      const int t = type_of(x);
      const size_t n = api.linear_forward_work_bytes(M, N, K, t);
      const Tensor work = workspace(n, x);
      check(api.linear_forward(address(vx), ldx, address(vw), ldw, address(vb), address(vr), ldr, writable(y),
                               writable(z), M, N, K, t, act, writable(work), n, on.stream),
            "cit_linear_forward");
    }
  }
  if (node) {
    torch::autograd::set_history(y, node);
    if (wanted(w)) node->x = SavedVariable(x, false);
    if (wanted(x)) node->w = SavedVariable(w, false);
    if (act) node->z = own_y ? SavedVariable(y, true) : SavedVariable(z, false);
    node->own_y = own_y, node->act = act;
    node->M = M, node->N = N, node->K = K;
    node->shape = std::move(shape);
  }
  return y;
}

// ---- policy loss ------------------------------------------------------------------

struct Scalars {
  double low, high, beta;
};

// The entry points' common arguments; `keep` holds what they point to.
struct PolicyArgs {
  Tensor logits, ref, mask;
  const int64_t *offsets, *actions;
  const float *old, *adv, *weights;
  int64_t ld, ld_ref, ld_mask, total, rows;
  int width, type;

  PolicyArgs(const Tensor& l, const Tensor& q, const Tensor& m, const Tensor& off, const Tensor& act, const Tensor& o,
             const Tensor& a, const Tensor& w) {
    rows = act.size(0), total = 0, width = 0;
    ld = ld_ref = ld_mask = 0;
    if (off.defined()) {
      total = l.size(0);
      logits = l.contiguous();
      if (q.defined()) ref = q.contiguous();
      if (m.defined()) mask = m.contiguous();
    } else {
      width = (int)l.size(1);
      ld_ref = ld_mask = width;
      logits = as_rows(l, rows, width, ld);
      if (q.defined()) ref = as_rows(q, rows, width, ld_ref);
      if (m.defined()) mask = as_rows(m, rows, width, ld_mask);
    }
    offsets = static_cast<const int64_t*>(address(off)), actions = static_cast<const int64_t*>(address(act));
    old = static_cast<const float*>(address(o)), adv = static_cast<const float*>(address(a));
    weights = static_cast<const float*>(address(w));
    type = type_of(l);
  }
  size_t bytes() const { return api.policy_loss_work_bytes(rows, width, offsets != nullptr); }
};

// The forward kernel has a row's probabilities in hand, so it writes the
// gradient for an upstream gradient of 1 in the same pass over the logits; the
// backward kernel reads the upstream gradient on the device and computes the
// gradient again only where it is something else.
struct PolicyLossBackward : torch::autograd::Node {
  SavedVariable given[8];                // logits, ref, mask, offsets, actions, old, adv, weights
  Scalars s;
  Tensor held;                           // the gradient for an upstream gradient of 1
  unsigned long long made_in = 0;        // the capture that it was made in; 0: none

  std::string name() const override { return "PolicyLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& v : given) v.reset_data();
    held.reset();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!grads[0].defined() || !task_should_compute_output(0)) return out;
    first_only("policy_loss");
    one_gradient(grads[0], "policy_loss");
    Tensor v[8];
    for (int i = 0; i < 8; i++) v[i] = given[i].unpack();
    const On on(v[0]);
    leaves_in_capture(*this, on.stream, "policy_loss");
    // The forward pass's gradient goes to one backward pass, its owner from then on, that runs as often as the forward
    // pass does: an eager one after an eager one, or one of the same capture.  Any other works the gradient out again in
    // memory of its own: a graph's replays would go on writing into an eager pass's, whoever has it by then, and
    // what a graph keeps for itself may be anything when another one is replayed.
    const bool ready = held.defined() && made_in == capture_of(on.stream);
    Tensor grad = ready ? std::move(held) : at::empty(v[0].sizes(), v[0].options());
    if (ready) held = Tensor();
    out[0] = grad;
    const PolicyArgs a(v[0], v[1], v[2], v[3], v[4], v[5], v[6], v[7]);
    if (!a.rows) {
      grad.zero_();
      return out;
    }
    const Tensor up = grads[0].scalar_type() == at::kFloat ? grads[0] : grads[0].to(at::kFloat);
    const size_t n = a.bytes();
    const Tensor work = workspace(n, grad);
    check(api.policy_loss_backward(address(a.logits), a.ld, address(a.ref), a.ld_ref,
                                   static_cast<const uint8_t*>(address(a.mask)), a.ld_mask, a.offsets, a.total, a.rows,
                                   a.width, a.actions, a.old, a.adv, a.weights, s.low, s.high, s.beta, a.type,
                                   static_cast<const float*>(address(up)), ready, writable(grad), writable(work), n,
                                   on.stream),
          "cit_policy_loss_backward");
    return out;
  }
};

std::tuple<Tensor, Tensor, Tensor> policy_loss(const Tensor& logits, const Maybe& ref, const Maybe& mask,
                                               const Maybe& offsets, const Tensor& actions, const Tensor& old,
                                               const Tensor& adv, const Maybe& weights, double low, double high,
                                               double beta) {
  const Tensor given[8] = {logits, ref.value_or(Tensor()), mask.value_or(Tensor()), offsets.value_or(Tensor()),
                           actions, old, adv, weights.value_or(Tensor())};
  for (const Tensor& t : given) own_memory({t}, "policy_loss");
  std::shared_ptr<PolicyLossBackward> node;
  if (at::GradMode::is_enabled() && wanted(logits)) {
    node = std::shared_ptr<PolicyLossBackward>(new PolicyLossBackward(), torch::autograd::deleteNode);
    node->set_next_edges(collect_next_edges(logits));
  }
  no_tangent({logits}, "policy_loss");
  Tensor loss, logp, kl, grad;
  unsigned long long made_in = 0;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    const On on(logits);
    const PolicyArgs a(given[0], given[1], given[2], given[3], given[4], given[5], given[6], given[7]);
    const auto f32 = logits.options().dtype(at::kFloat);
    loss = at::empty({}, f32), logp = at::empty({a.rows}, f32), kl = at::empty({a.rows}, f32);
    if (node) {
      grad = a.rows ? at::empty(logits.sizes(), logits.options()) : at::zeros(logits.sizes(), logits.options());
      made_in = capture_of(on.stream);
    }
    const size_t n = a.bytes();
    const Tensor work = workspace(n, logits);
    check(api.policy_loss(address(a.logits), a.ld, address(a.ref), a.ld_ref, static_cast<const uint8_t*>(address(a.mask)),
                          a.ld_mask, a.offsets, a.total, a.rows, a.width, a.actions, a.old, a.adv, a.weights, low, high,
                          beta, a.type, static_cast<float*>(writable(loss)), static_cast<float*>(writable(logp)),
                          static_cast<float*>(writable(kl)), writable(grad), writable(work), n, on.stream),
          "cit_policy_loss");
  }
  if (node) {
    torch::autograd::set_history(loss, node);
    for (int i = 0; i < 8; i++)
      if (given[i].defined()) node->given[i] = SavedVariable(i && given[i].requires_grad() ? given[i].detach() : given[i], false);
    node->s = Scalars{low, high, beta};
    node->held = std::move(grad);
    node->made_in = made_in;
  }
  return {loss, logp, kl};
}

// ---- gradient norm ------------------------------------------------------------------

// The tensors of a Python list: dense ones of the kernels' types on one device.
std::vector<Tensor> listed(const py::list& from, const std::string& what) {
  std::vector<Tensor> out;
  out.reserve(from.size());
  for (const py::handle& h : from) {
    if (!THPVariable_Check(h.ptr())) throw py::value_error(what + " must be a tensor");
    out.push_back(THPVariable_Unpack(h.ptr()));
  }
  for (const Tensor& t : out) {
    if (t.layout() != at::kStrided || t.is_neg() || !t.has_storage()) throw py::value_error(what + " must be a dense tensor");
    const at::ScalarType dt = t.scalar_type();
    if (dt != at::kFloat && dt != at::kBFloat16 && dt != at::kHalf)
      throw py::value_error(what + "s must be fp32, bf16 or fp16, not " +
                            py::str(py::reinterpret_borrow<py::object>(from[&t - out.data()]).attr("dtype")).cast<std::string>());
    if (t.device() != out[0].device()) throw py::value_error(what + "s must be on one device");
  }
  return out;
}

typedef std::vector<std::pair<uintptr_t, uintptr_t>> Spans;

// Start and end of the tensors that hold something.
Spans spans_of(const std::vector<Tensor>& list) {
  Spans s;
  s.reserve(list.size());
  for (const Tensor& t : list)
    if (t.numel()) s.emplace_back((uintptr_t)t.const_data_ptr(), (uintptr_t)t.const_data_ptr() + t.nbytes());
  return s;
}
bool disjoint(Spans s) {
  std::sort(s.begin(), s.end());
  for (size_t i = 1; i < s.size(); i++)
    if (s[i].first < s[i - 1].second) return false;
  return true;
}

enum { NORM = 0, CHECK = 1, CLIP = 2 };  // the norm alone; the same after clip's checks; clip

// The norm of `grads` (not empty), and their clipping into `out` (None: in place).
Tensor clip_grad_norm(const py::list& given, double max_norm, const py::object& into, int mode) {
  const std::vector<Tensor> grads = listed(given, "a gradient");
  std::vector<Tensor> flat, outs;
  flat.reserve(grads.size());
  {
    at::NoGradGuard none;
    for (const Tensor& t : grads) flat.push_back(t.is_contiguous() ? t : t.contiguous());
  }
  const Spans spans = spans_of(flat);
  if (mode != NORM && into.is_none()) {
    std::vector<uintptr_t> at;
    for (size_t i = 0; i < grads.size(); i++) {
      const Tensor& t = grads[i];
      if (!t.is_same(flat[i]))
        for (int64_t d = 0; d < t.dim(); d++)
          if (t.stride(d) == 0 && t.size(d) > 1)
            throw py::value_error("a gradient whose elements share memory cannot be clipped in place: give out=");
      if (t.numel()) at.push_back((uintptr_t)t.const_data_ptr());
    }
    std::sort(at.begin(), at.end());
    if (!disjoint(spans) || std::adjacent_find(at.begin(), at.end()) != at.end())
      throw py::value_error("a gradient is listed twice, or two share memory");
    outs = flat;
  } else if (mode != NORM) {
    outs = listed(py::list(into), "an out tensor");
    if (outs.size() != grads.size())
      throw py::value_error(std::to_string(grads.size()) + " gradients, " + std::to_string(outs.size()) +
                            " tensors in out");
    for (size_t i = 0; i < outs.size(); i++)
      if (!outs[i].is_contiguous() || outs[i].sizes() != grads[i].sizes() ||
          (outs[i].scalar_type() != grads[i].scalar_type() && outs[i].scalar_type() != at::kFloat))
        throw py::value_error("an out tensor must be contiguous, of its gradient's shape, and of its type or fp32");
    if (outs[0].device() != grads[0].device()) throw py::value_error("out tensors must be on the gradients' device");
    const Spans to = spans_of(outs);
    Spans both = to;
    both.insert(both.end(), spans.begin(), spans.end());
    if (!disjoint(both)) {
      // gradients may share memory among themselves, and one may be its own out tensor
      bool bad = !disjoint(to);
      for (size_t i = 0; i < flat.size() && !bad; i++) {
        if (!flat[i].numel() || (flat[i].const_data_ptr() == outs[i].const_data_ptr() &&
                                 flat[i].scalar_type() == outs[i].scalar_type()))
          continue;
        Spans with = to;
        with.emplace_back((uintptr_t)flat[i].const_data_ptr(), (uintptr_t)flat[i].const_data_ptr() + flat[i].nbytes());
        bad = !disjoint(with);
      }
      if (bad) throw py::value_error("out tensors share memory with one another or with other gradients");
    }
  }
  if (!flat[0].is_cuda())
    throw py::value_error("tensors must be on the GPU (there is no CPU path), not on " + flat[0].device().str());
  const size_t n = flat.size();
  std::vector<const void*> from(n);
  std::vector<void*> to(n);
  std::vector<int64_t> sizes(n);
  std::vector<int32_t> types(n), out_types(n);
  for (size_t i = 0; i < n; i++) {
    from[i] = flat[i].const_data_ptr(), sizes[i] = flat[i].numel(), types[i] = type_of(flat[i]);
    if (mode == CLIP) to[i] = outs[i].mutable_data_ptr(), out_types[i] = type_of(outs[i]);
  }
  py::gil_scoped_release release;
  at::NoGradGuard none;
  const On on(flat[0]);
  const Tensor norm = at::empty({}, flat[0].options().dtype(at::kFloat));
  const size_t bytes = api.clip_grad_norm_work_bytes((int)n);
  const Tensor work = workspace(bytes, norm);
  check(api.clip_grad_norm(from.data(), mode == CLIP ? to.data() : nullptr, sizes.data(), types.data(),
                           mode == CLIP ? out_types.data() : nullptr, (int)n, max_norm,
                           static_cast<float*>(writable(norm)), writable(work), bytes, on.stream),
        "cit_clip_grad_norm");
  if (mode == CLIP)
    for (size_t i = 0; i < n; i++) {
      if (into.is_none() && !grads[i].is_same(flat[i])) grads[i].copy_(flat[i]);
      else if (!outs[i].is_inference()) torch::autograd::impl::bump_version(outs[i]);
    }
  return norm;
}

PyObject* native_error = nullptr;        // _lib.NativeError

void bind(py::object error, const std::map<std::string, uint64_t>& at) {
  native_error = error.release().ptr();
  const auto take = [&](auto& f, const char* name) {
    f = reinterpret_cast<std::remove_reference_t<decltype(f)>>(at.at(name));
  };
  take(api.linear_forward_work_bytes, "cit_linear_forward_work_bytes");
  take(api.linear_forward, "cit_linear_forward");
  take(api.linear_backward_work_bytes, "cit_linear_backward_work_bytes");
  take(api.linear_backward, "cit_linear_backward");
  take(api.policy_loss_work_bytes, "cit_policy_loss_work_bytes");
  take(api.policy_loss, "cit_policy_loss");
  take(api.policy_loss_backward, "cit_policy_loss_backward");
  take(api.clip_grad_norm_work_bytes, "cit_clip_grad_norm_work_bytes");
  take(api.clip_grad_norm, "cit_clip_grad_norm");
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const NativeError& e) {
      PyErr_SetString(native_error ? native_error : PyExc_RuntimeError, e.what());
    }
  });
  m.def("bind", &bind);
  m.def("linear", &linear, py::call_guard<py::gil_scoped_release>());
  m.def("policy_loss", &policy_loss, py::call_guard<py::gil_scoped_release>());
  m.def("clip_grad_norm", &clip_grad_norm);
}
