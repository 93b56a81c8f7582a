// Autograd nodes of the token operators (multiyolov5_amd/utils/tokens.py): checks, descriptors, results and the backward call in C++, so that a
// training pass neither enters the interpreter twice nor takes its lock on the engine's thread.  A pass over small tensors is bound by the
// host: with the nodes in Python it took 88 / 128 / 137 us (layer norm, rope, attention), the kernels of a 4097 x 1003 layer norm 40.
// The arithmetic stays behind the C ABI of include/myolo.h; the entry points are handed over by the ctypes binding (bind), so both sides
// use one library.
#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <array>
#include <cmath>
#include <map>
#include <sstream>
#include <unordered_set>
#include "../../include/myolo.h"

namespace {

using at::Tensor;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Error : std::runtime_error { using std::runtime_error::runtime_error; };
template <class... A> [[noreturn]] void fail(const A&... a) {
  std::ostringstream o;
  (o << ... << a);
  throw Error(o.str());
}
#define NEED(cond, ...) do { if (!(cond)) fail(__VA_ARGS__); } while (0)

struct Entries {
  decltype(&myolo_layernorm_fwd) ln_fwd;
  decltype(&myolo_layernorm_bwd) ln_bwd;
  decltype(&myolo_layernorm_ws_bytes) ln_ws;
  decltype(&myolo_rope) rope;
  decltype(&myolo_attn_fwd) attn_fwd;
  decltype(&myolo_attn_bwd) attn_bwd;
  decltype(&myolo_attn_ws_bytes) attn_ws;
} lib{};

void check(int rc, const char* what) {
  if (rc) fail("libmyolo ", what, " failed with error ", rc, rc == MYOLO_EINVAL ? " (invalid argument)" : "");
}
// launches go to the tensors' device and its current stream, whatever the current device is
struct On {
  c10::DeviceGuard guard;
  void* stream;
  explicit On(const Tensor& t) : guard(t.device()), stream(c10::hip::getCurrentHIPStream(t.get_device()).stream()) {}
};
int dtype_of(const Tensor& t) { return t.scalar_type() == at::kHalf ? MYOLO_F16 : MYOLO_F32; }
void same_device(const Tensor& t, std::initializer_list<const Tensor*> others) {
  for (const Tensor* o : others)
    NEED(!o->defined() || o->device() == t.device(), "tensors on ", t.device(), " and ", o->device(), " in one call");
}
bool wants_grad(std::initializer_list<const Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : ts)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}
// the kernels form no tangents: a result without one would pass for a constant downstream
void no_forward_mode(const char* what, std::initializer_list<const Tensor*> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const Tensor* t : ts)
    NEED(!t->defined() || !t->_fw_grad(0).defined(), what, ": no derivatives in forward mode (a dual tensor)");
}
// torch.jit.trace records torch's own calls: the results' empty() without the launches that fill them
void not_traced(const char* what) { NEED(!torch::jit::tracer::isTracing(), what, ": a call cannot be traced (its kernels would be missing from the trace)"); }
void first_order_only(const char* what) {
  NEED(!at::GradMode::is_enabled(), what, ": the backward pass cannot itself be recorded for a second derivative (create_graph)");
}
// A leaf that an eager graph on the default stream still holds has its gradient's node there: the engine would make that stream wait for the one
// being captured, which no capture survives (the error ends the process).  Refused while the capture is still whole: the node's own edges, and
// whatever this pass is going to run behind them (a leaf under a projection, a part of the graph recorded before the capture).
void capturable(const torch::autograd::Node& n, const Tensor& like, const char* what) {
  using torch::autograd::Node;
  const c10::DeviceGuard guard(like.device());
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() == c10::hip::CaptureStatus::None) return;
  if (c10::hip::getCurrentHIPStream(like.get_device()).id() == 0) return;
  auto check_stream = [&](Node* f) {
    const auto s = f->stream();
    NEED(!s || s->id() != 0, what,
         ": backward captured while an eager graph of the same leaf lives on the default stream: drop that graph, or capture with detached leaves");
  };
  const auto* exec = torch::autograd::get_current_graph_task_exec_info();      // (empty: a pass over everything)
  std::unordered_set<Node*> seen;
  std::vector<Node*> todo;
  auto push = [&](const Node& f) {
    for (const auto& e : f.next_edges()) {
      Node* next = e.function.get();
      if (!next) continue;
      if (exec && !exec->empty()) {
        const auto it = exec->find(next);
        if (it == exec->end() || !it->second.should_execute()) continue;
      }
      if (seen.insert(next).second) todo.push_back(next);
    }
  };
  for (const auto& e : n.next_edges())
    if (dynamic_cast<torch::autograd::AccumulateGrad*>(e.function.get())) check_stream(e.function.get());
  push(n);
  while (!todo.empty()) {
    Node* f = todo.back();
    todo.pop_back();
    check_stream(f);
    push(*f);
  }
}
Tensor empty(at::IntArrayRef shape, const Tensor& like) { return at::empty(shape, like.options()); }
Tensor floats(int64_t n, const Tensor& like) { return at::empty({n}, like.options().dtype(at::kFloat)); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor of(const OptTensor& t) { return t.has_value() ? *t : Tensor(); }
// t with its values in its memory: a lazily negated view (the imaginary part of a conjugate) is written out, a tensor without memory refused
Tensor plain(const Tensor& t, const char* what) {
  if (!t.defined()) return t;
  NEED(!t._is_zerotensor(), what, ": a tensor without storage");
  return t.is_neg() ? t.resolve_neg() : t;
}
// What a node saved may come back from saved-tensor hooks in any layout (save_on_cpu: contiguous; a user's: anything), so a backward lays it out
// again as its kernels read it; only its values, type, shape and device are taken for granted, and those are checked.
Tensor saved_as(const Tensor& t, at::IntArrayRef shape, at::ScalarType dtype, const at::Device& device, const char* what) {
  NEED(t.defined() && t.sizes() == shape && t.scalar_type() == dtype && t.device() == device, what, ": a tensor saved as ", dtype, " ", shape, " on ", device,
       " came back as ", t.scalar_type(), " ", t.sizes(), " on ", t.device());
  return plain(t, what);
}

// ---- layer norm ----------------------------------------------------------------------------------------------------------------------
// leading dimensions merged where their strides allow, padded to three; false where they do not reduce to three strides
bool lead(const Tensor& t, myolo_tensor& d) {
  const int64_t c = t.size(-1);
  if (c > 1 && t.stride(-1) != 1) return false;
  int64_t n[3], s[3];
  int k = 0;
  const int64_t most = int64_t(1) << 31;
  for (int64_t i = 0; i + 1 < t.dim(); ++i) {
    const int64_t ni = t.size(i), si = t.stride(i);
    if (ni == 1) continue;
    if (ni >= most) return false;
    if (k && s[k - 1] == ni * si && n[k - 1] * ni < most) { n[k - 1] *= ni; s[k - 1] = si; continue; }
    if (k == 3) return false;
    n[k] = ni;
    s[k++] = si;
  }
  if (k >= 2 && n[k - 1] * n[k - 2] >= most) return false;
  int64_t N[3] = {1, 1, 1}, S[3];
  for (int i = 0; i < k; ++i) { N[3 - k + i] = n[i]; S[3 - k + i] = s[i]; }
  if (!k) S[2] = c;
  for (int i = (k ? 2 - k : 1); i >= 0; --i) S[i] = N[i + 1] * S[i + 1];
  d = myolo_tensor{t.data_ptr(), (int32_t)N[0], (int32_t)N[1], (int32_t)N[2], (int32_t)c, S[0], S[1], S[2], dtype_of(t), 0};
  return true;
}
// the tensor whose rows d describes: x itself, or a copy
Tensor rows_of(const Tensor& x, myolo_tensor& d) {
  if (lead(x, d)) return x;
  Tensor y = x.contiguous();
  NEED(lead(y, d), "layer_norm: more than 2^31 - 1 rows in one dimension");
  return y;
}
// the rows of the contiguous tensor t, numbered as d numbers its own
myolo_tensor rows_like(const Tensor& t, const myolo_tensor& d) {
  return myolo_tensor{ptr(t), d.n, d.h, d.w, d.c, (int64_t)d.h * d.w * d.c, (int64_t)d.w * d.c, d.c, d.dtype, 0};
}
bool same_rows(const myolo_tensor& a, const myolo_tensor& b) { return a.n == b.n && a.h == b.h && a.w == b.w; }

struct LayerNormBackward : torch::autograd::Node {
  SavedVariable x, w, saved;
  std::vector<int64_t> shape;
  at::TensorOptions like;
  bool has_w;
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    first_order_only("layer_norm");
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor()};
    no_forward_mode("layer_norm", {&g[0]});
    const int64_t c = shape.back();
    const auto dtype = like.dtype().toScalarType();
    const at::Device device = like.device();
    const Tensor raw = saved_as(x.unpack(), shape, dtype, device, "layer_norm");
    const Tensor W = has_w ? saved_as(w.unpack(), {c}, at::kFloat, device, "layer_norm").contiguous() : Tensor();
    const Tensor S = saved_as(saved.unpack(), {2 * (raw.numel() / c)}, at::kFloat, device, "layer_norm").contiguous();
    capturable(*this, raw, "layer_norm");
    myolo_tensor xd, gd;
    const Tensor X = rows_of(raw, xd);
    Tensor go = plain(g[0], "layer_norm");
    if (go.scalar_type() != X.scalar_type()) go = go.to(X.scalar_type());
    go = rows_of(go, gd);
    if (!same_rows(gd, xd)) {
      go = go.contiguous();
      gd = rows_like(go, xd);
    }
    Tensor gx, gw, gb, ws;
    if (task_should_compute_output(0)) gx = empty(X.sizes(), X);
    if (task_should_compute_output(1)) gw = floats(xd.c, X);
    if (task_should_compute_output(2)) gb = floats(xd.c, X);
    int64_t nb = 0;
    if (gw.defined() || gb.defined()) nb = lib.ln_ws((int64_t)xd.n * xd.h * xd.w, xd.c);
    if (nb) ws = floats(nb / 4, X);
    const myolo_tensor gxd = rows_like(gx, xd);
    On on(X);
    check(lib.ln_bwd(&gd, &xd, (const float*)ptr(S), (const float*)ptr(W), gx.defined() ? &gxd : nullptr, 0, (float*)ptr(gw), (float*)ptr(gb), 0,
                     (float*)ptr(ws), nb, on.stream),
          "myolo_layernorm_bwd");
    return {gx, gw, gb};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data();
    w.reset_data();
    saved.reset_data();
  }
  std::string name() const override { return "LayerNormBackward"; }
};

Tensor layer_norm(const Tensor& x_, const OptTensor& w_, const OptTensor& b_, double eps) {
  not_traced("layer_norm");
  const Tensor x = plain(x_, "layer_norm"), w = plain(of(w_), "layer_norm"), b = plain(of(b_), "layer_norm");
  NEED(x.dim() > 0 && x.size(-1) >= 1, "layer_norm: no channels in a tensor of shape ", x.sizes());
  NEED(x.size(-1) <= MYOLO_LAYERNORM_MAX_C, "layer_norm: ", x.size(-1), " channels (at most ", MYOLO_LAYERNORM_MAX_C, ")");
  NEED(eps >= 0.0 && std::isfinite(eps), "layer_norm: eps must be a number >= 0, got ", eps);
  for (const Tensor* p : {&w, &b})
    NEED(!p->defined() || (p->scalar_type() == at::kFloat && p->dim() == 1 && p->size(0) == x.size(-1) && p->is_cuda()),
         "layer_norm: weight and bias are fp32 tensors of ", x.size(-1), " values on the GPU, got ", p->scalar_type(), " ", p->sizes());
  same_device(x, {&w, &b});
  no_forward_mode("layer_norm", {&x, &w, &b});
  const bool train = wants_grad({&x, &w, &b});
  Tensor X, out, saved, W, B;
  {
    at::NoGradGuard off;
    myolo_tensor xd;
    X = rows_of(x, xd);
    W = w.defined() ? w.contiguous() : w;
    B = b.defined() ? b.contiguous() : b;
    out = empty(x.sizes(), x);
    if (train) saved = floats(2 * (int64_t)xd.n * xd.h * xd.w, x);
    const myolo_tensor od = rows_like(out, xd);
    On on(x);
    check(lib.ln_fwd(&xd, (const float*)ptr(W), (const float*)ptr(B), (float)eps, &od, (float*)ptr(saved), on.stream), "myolo_layernorm_fwd");
  }
  if (train) {
    std::shared_ptr<LayerNormBackward> fn(new LayerNormBackward(), torch::autograd::deleteNode);
    fn->set_next_edges(torch::autograd::collect_next_edges(x, w, b));
    fn->shape = x.sizes().vec();
    fn->like = x.options();
    fn->has_w = W.defined();
    fn->x = SavedVariable(X, false);
    if (W.defined()) fn->w = SavedVariable(W, false);
    fn->saved = SavedVariable(saved, false);
    torch::autograd::set_history(out, fn);
  }
  return out;
}

// ---- [b, l, h, d] views --------------------------------------------------------------------------------------------------------------
// {batch, token, head} strides; a dimension of one element has none that matters
void strides3(int64_t* s, const Tensor& t) {
  for (int i = 0; i < 3; ++i) s[i] = t.size(i) > 1 ? t.stride(i) : 0;
}

// ---- rotary positions ----------------------------------------------------------------------------------------------------------------
struct RopeSpec {
  std::array<double, MYOLO_ROPE_MAX_PAIRS> turns;
  std::array<int32_t, MYOLO_ROPE_MAX_PAIRS> axis;
  int npair, naxis;
  bool interleaved;
};
Tensor adjacent(const Tensor& t) { return t.size(-1) > 1 && t.stride(-1) != 1 ? t.contiguous() : t; }

std::pair<Tensor, Tensor> turn(Tensor q, Tensor k, const Tensor& pos, const RopeSpec& s, bool inverse) {
  q = adjacent(q);
  Tensor qo = empty(q.sizes(), q), ko;
  myolo_rope_desc d{};
  d.q = ptr(q); d.qo = ptr(qo); d.pos = (const int64_t*)ptr(pos);
  strides3(d.qs, q);
  strides3(d.qos, qo);
  if (k.defined()) {
    k = adjacent(k);
    ko = empty(k.sizes(), k);
    d.k = ptr(k); d.ko = ptr(ko); d.hk = (int32_t)k.size(2);
    strides3(d.ks, k);
    strides3(d.kos, ko);
  }
  d.ps[0] = pos.dim() == 3 && pos.size(0) > 1 ? pos.stride(0) : 0;
  d.ps[1] = pos.stride(-2);
  d.ps[2] = pos.stride(-1);
  d.turns = s.turns.data(); d.axis = s.axis.data();
  d.b = (int32_t)q.size(0); d.l = (int32_t)q.size(1); d.hq = (int32_t)q.size(2); d.d = (int32_t)q.size(3);
  d.npair = s.npair; d.naxis = s.naxis; d.interleaved = s.interleaved; d.inverse = inverse; d.dtype = dtype_of(q);
  On on(q);
  check(lib.rope(&d, on.stream), "myolo_rope");
  return {qo, ko};
}

struct RopeBackward : torch::autograd::Node {
  SavedVariable pos;
  RopeSpec spec;
  std::vector<int64_t> qs, ks, ps;
  at::TensorOptions like;
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    first_order_only("rope_axes");
    const bool has_k = !ks.empty();
    for (const Tensor& t : g) no_forward_mode("rope_axes", {&t});
    const Tensor P = saved_as(pos.unpack(), ps, at::kLong, like.device(), "rope_axes");     // (once: a checkpoint hands every saved tensor out a single time)
    capturable(*this, P, "rope_axes");
    if (!g[0].defined() && !(has_k && g[1].defined())) return {Tensor(), Tensor()};
    auto grad = [&](const Tensor& t_, const std::vector<int64_t>& shape) {
      const Tensor t = plain(t_, "rope_axes");
      return !t.defined() ? at::zeros(shape, like) : t.scalar_type() == like.dtype() ? t : t.to(like);
    };
    auto r = turn(grad(g[0], qs), has_k ? grad(g[1], ks) : Tensor(), P, spec, true);
    return {task_should_compute_output(0) ? r.first : Tensor(), task_should_compute_output(1) ? r.second : Tensor()};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    pos.reset_data();
  }
  std::string name() const override { return "RopeAxesBackward"; }
};

// turns, axis: addresses of sum(sections) values each
std::pair<Tensor, OptTensor> rope_axes(const Tensor& q_, const OptTensor& k_, const Tensor& pos_, int64_t turns, int64_t axis, int npair, int naxis,
                                       bool interleaved) {
  not_traced("rope_axes");
  const Tensor q = plain(q_, "rope_axes"), k = plain(of(k_), "rope_axes"), pos = plain(pos_, "rope_axes");
  NEED(!k.defined() || (k.size(0) == q.size(0) && k.size(1) == q.size(1) && k.size(3) == q.size(3) && k.size(2) >= 1),
       "rope_axes: q ", q.sizes(), " and k ", k.sizes(), " differ in more than their heads");
  NEED(q.size(2) >= 1 && q.size(3) >= 1, "rope_axes: q ", q.sizes());
  for (int i = 0; i < 4; ++i) NEED(q.size(i) < (int64_t(1) << 31) && (!k.defined() || k.size(i) < (int64_t(1) << 31)), "rope_axes: q ", q.sizes(), " is too large");
  NEED(2 * npair <= q.size(3) && npair <= MYOLO_ROPE_MAX_PAIRS, "rope_axes: ", npair, " pairs in ", q.size(3), " channels (at most ", MYOLO_ROPE_MAX_PAIRS, ")");
  NEED((pos.dim() == 2 || pos.dim() == 3) && pos.size(-2) == q.size(1) && pos.size(-1) == naxis &&
           (pos.dim() == 2 || pos.size(0) == 1 || pos.size(0) == q.size(0)),
       "rope_axes: pos ", pos.sizes(), " for ", q.size(1), " tokens, ", naxis, " axes and a batch of ", q.size(0));
  same_device(q, {&k, &pos});
  no_forward_mode("rope_axes", {&q, &k});
  RopeSpec s;
  s.npair = npair; s.naxis = naxis; s.interleaved = interleaved;
  std::copy_n(reinterpret_cast<const double*>(turns), npair, s.turns.begin());
  std::copy_n(reinterpret_cast<const int32_t*>(axis), npair, s.axis.begin());
  std::pair<Tensor, Tensor> r;
  {
    at::NoGradGuard off;
    r = turn(q, k, pos, s, false);
  }
  if (wants_grad({&q, &k})) {
    std::shared_ptr<RopeBackward> fn(new RopeBackward(), torch::autograd::deleteNode);
    fn->set_next_edges(torch::autograd::collect_next_edges(q, k));
    fn->pos = SavedVariable(pos, false);
    fn->spec = s;
    fn->qs = q.sizes().vec();
    fn->ps = pos.sizes().vec();
    if (k.defined()) fn->ks = k.sizes().vec();
    fn->like = q.options();
    if (k.defined()) torch::autograd::set_history(variable_list{r.first, r.second}, fn);
    else torch::autograd::set_history(r.first, fn);
  }
  return {r.first, k.defined() ? OptTensor(r.second) : std::nullopt};
}

// ---- attention -----------------------------------------------------------------------------------------------------------------------
// t as the kernels read it -- adjacent channels, base and strides multiples of 16 bytes -- copied where it is not
Tensor side(const Tensor& t) {
  bool ok = (t.stride(3) == 1 || t.size(3) <= 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int i = 0; i < 3 && ok; ++i) ok = t.size(i) <= 1 || t.stride(i) * t.element_size() % 16 == 0;
  return ok ? t : t.clone(at::MemoryFormat::Contiguous);
}
void attn_fill(myolo_attn_desc& d, const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& res, const Tensor& lse,
               const Tensor& lens, const Tensor& starts) {
  d.q = ptr(q); d.k = ptr(k); d.v = ptr(v); d.o = ptr(o); d.o_res = ptr(res); d.lse = (float*)ptr(lse);
  d.lens = (const int*)ptr(lens); d.starts = (const int*)ptr(starts);
  strides3(d.qs, q);
  strides3(d.ks, k);
  strides3(d.vs, v);
  strides3(d.os, o);
}
Tensor scratch(myolo_attn_desc& d, int backward, const Tensor& like) {
  d.ws_bytes = lib.attn_ws(&d, backward);
  Tensor ws = d.ws_bytes ? at::empty({d.ws_bytes}, like.options().dtype(at::kByte)) : Tensor();
  d.ws = ptr(ws);
  return ws;
}

struct WindowAttentionBackward : torch::autograd::Node {
  SavedVariable q, k, v, o, res, lse, lens, starts;
  myolo_attn_desc shape;                                    // sizes and options; no addresses
  at::TensorOptions like;
  bool has_lens, has_starts;
  variable_list apply(variable_list&& g) override {
    std::lock_guard<std::mutex> lock(mutex_);
    first_order_only("window_attention");
    if (!g[0].defined()) return {Tensor(), Tensor(), Tensor()};
    no_forward_mode("window_attention", {&g[0]});
    const auto dtype = like.dtype().toScalarType();
    const at::Device device = like.device();
    const int64_t b = shape.b, lq = shape.lq, lk = shape.lk, hq = shape.hq, hk = shape.hk, dim = shape.d;
    auto back = [&](const Tensor& t, at::IntArrayRef sizes, at::ScalarType type) { return saved_as(t, sizes, type, device, "window_attention"); };
    const Tensor Q = side(back(q.unpack(), {b, lq, hq, dim}, dtype)), K = side(back(k.unpack(), {b, lk, hk, dim}, dtype)),
                 V = side(back(v.unpack(), {b, lk, hk, dim}, dtype));
    // (the residual is addressed by o's strides: both dense, as the forward wrote them)
    const Tensor O = side(back(o.unpack(shared_from_this()), {b, lq, hq, dim}, dtype).contiguous());
    const Tensor R = dtype == at::kHalf ? side(back(res.unpack(), {b, lq, hq, dim}, dtype).contiguous()) : Tensor();
    const Tensor S = back(lse.unpack(), {b * hq * lq}, at::kFloat).contiguous();
    const Tensor N = has_lens ? back(lens.unpack(), {b}, at::kInt).contiguous() : Tensor(), P = has_starts ? back(starts.unpack(), {b}, at::kInt).contiguous() : Tensor();
    capturable(*this, Q, "window_attention");
    Tensor go = plain(g[0], "window_attention");
    go = side(go.scalar_type() == Q.scalar_type() ? go : go.to(Q.scalar_type()));
    const bool want_q = task_should_compute_output(0), want_k = task_should_compute_output(1), want_v = task_should_compute_output(2);
    myolo_attn_desc d = shape;
    attn_fill(d, Q, K, V, O, R, S, N, P);
    d.go = ptr(go);
    strides3(d.gos, go);
    Tensor gq, gk, gv;
    if (want_q) {
      gq = empty(Q.sizes(), Q);
      d.gq = ptr(gq);
      strides3(d.gqs, gq);
    }
    if (want_k || want_v) {
      gk = empty(K.sizes(), K);
      gv = empty(V.sizes(), V);
      d.gk = ptr(gk);
      d.gv = ptr(gv);
      strides3(d.gks, gk);
      strides3(d.gvs, gv);
    }
    const Tensor ws = scratch(d, 1, Q);
    On on(Q);
    check(lib.attn_bwd(&d, on.stream), "myolo_attn_bwd");
    return {gq, want_k ? gk : Tensor(), want_v ? gv : Tensor()};
  }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q, &k, &v, &o, &res, &lse, &lens, &starts}) s->reset_data();
  }
  std::string name() const override { return "WindowAttentionBackward"; }
};

Tensor window_attention(const Tensor& q_, const Tensor& k_, const Tensor& v_, int64_t window, int64_t sinks, bool causal, const OptTensor& lens_,
                        const OptTensor& starts_, std::optional<double> scale_) {
  not_traced("window_attention");
  const Tensor q = plain(q_, "window_attention"), k = plain(k_, "window_attention"), v = plain(v_, "window_attention");
  Tensor lens = plain(of(lens_), "window_attention"), starts = plain(of(starts_), "window_attention");
  const int64_t b = q.size(0), lq = q.size(1), hq = q.size(2), dim = q.size(3), lk = k.size(1), hk = k.size(2);
  NEED(k.sizes() == v.sizes() && k.size(0) == b && k.size(3) == dim, "window_attention: q ", q.sizes(), ", k ", k.sizes(), ", v ", v.sizes());
  NEED(hk >= 1 && hq >= 1 && hq % hk == 0, "window_attention: ", hq, " query heads over ", hk, " key heads");
  NEED(dim % 8 == 0 && dim >= 8 && dim <= 128, "window_attention: head dimension ", dim, " (a multiple of 8 up to 128)");
  NEED(window >= 0 && sinks >= 0, "window_attention: window ", window, ", sinks ", sinks);
  NEED(std::max({lq * (hq / hk), lk, window}) <= MYOLO_ATTN_MAX_LEN && b * hq < (1 << 24), "window_attention: sequence, window or batch too long");
  const double scale = scale_.has_value() ? *scale_ : 1.0 / std::sqrt((double)dim);
  NEED(scale > 0.0 && std::isfinite(scale), "window_attention: scale ", scale);
  for (const Tensor* t : {&lens, &starts})
    NEED(!t->defined() || (t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == b && t->is_cuda()),
         "window_attention: lens and starts are int32 tensors of ", b, " values on the GPU, got ", t->scalar_type(), " ", t->sizes());
  same_device(q, {&k, &v, &lens, &starts});
  no_forward_mode("window_attention", {&q, &k, &v});
  const bool train = wants_grad({&q, &k, &v});
  myolo_attn_desc shape{};
  shape.b = (int32_t)b; shape.lq = (int32_t)lq; shape.lk = (int32_t)lk; shape.hq = (int32_t)hq; shape.hk = (int32_t)hk; shape.d = (int32_t)dim;
  shape.dtype = dtype_of(q); shape.causal = causal; shape.window = (int32_t)window; shape.sinks = (int32_t)std::min(sinks, lk); shape.scale = (float)scale;
  Tensor Q, K, V, out, res, lse;
  {
    at::NoGradGuard off;
    Q = side(q);
    K = side(k);
    V = side(v);
    if (lens.defined()) lens = lens.contiguous();
    if (starts.defined()) starts = starts.contiguous();
    out = empty(q.sizes(), q);
    if (train) {
      lse = floats(b * hq * lq, q);
      if (q.scalar_type() == at::kHalf) res = empty(q.sizes(), q);
    }
    myolo_attn_desc d = shape;
    attn_fill(d, Q, K, V, out, res, lse, lens, starts);
    const Tensor ws = scratch(d, 0, q);
    On on(q);
    check(lib.attn_fwd(&d, on.stream), "myolo_attn_fwd");
  }
  if (train) {
    std::shared_ptr<WindowAttentionBackward> fn(new WindowAttentionBackward(), torch::autograd::deleteNode);
    fn->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
    fn->q = SavedVariable(Q, false);
    fn->k = SavedVariable(K, false);
    fn->v = SavedVariable(V, false);
    if (res.defined()) fn->res = SavedVariable(res, false);
    fn->lse = SavedVariable(lse, false);
    if ((fn->has_lens = lens.defined())) fn->lens = SavedVariable(lens, false);
    if ((fn->has_starts = starts.defined())) fn->starts = SavedVariable(starts, false);
    fn->shape = shape;
    fn->like = q.options();
    torch::autograd::set_history(out, fn);
    fn->o = SavedVariable(out, true);
  }
  return out;
}

// addresses of the C entry points, by name
void bind(const std::map<std::string, int64_t>& f) {
  auto at = [&](const char* n) { return reinterpret_cast<void*>(f.at(n)); };
  lib.ln_fwd = (decltype(lib.ln_fwd))at("myolo_layernorm_fwd");
  lib.ln_bwd = (decltype(lib.ln_bwd))at("myolo_layernorm_bwd");
  lib.ln_ws = (decltype(lib.ln_ws))at("myolo_layernorm_ws_bytes");
  lib.rope = (decltype(lib.rope))at("myolo_rope");
  lib.attn_fwd = (decltype(lib.attn_fwd))at("myolo_attn_fwd");
  lib.attn_bwd = (decltype(lib.attn_bwd))at("myolo_attn_bwd");
  lib.attn_ws = (decltype(lib.attn_ws))at("myolo_attn_ws_bytes");
}

}  // namespace

PYBIND11_MODULE(_token_autograd, m) {
  static PyObject* error = py::object(py::module_::import("multiyolov5_amd._lib").attr("MyoloError")).release().ptr();
  py::register_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const Error& e) {
      PyErr_SetString(error, e.what());
    }
  });
  m.def("bind", &bind);
  using free_lock = py::call_guard<py::gil_scoped_release>;      // (a launch may wait for the queue)
  m.def("layer_norm", &layer_norm, free_lock());
  m.def("rope_axes", &rope_axes, free_lock());
  m.def("window_attention", &window_attention, free_lock());
}
