// dvgr_torch.cpp -- autograd nodes of the question-side operators (inputs.embed_tokens, losses.distillation_loss,
// attention.cross_attention) around their C ABI.
//
// A small call of these is bound by the host: autograd runs a backward on a thread of its own, and a Python function there costs
// more than the kernels (a question batch's embedding, forward and backward: 125 us with Python nodes).  The module holds no
// kernel and does not link the library: `bind` gets the addresses of the entry points of whichever build was loaded.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/graph_task.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <cmath>
#include <mutex>
#include <unordered_set>

#include "../../include/dvgr_attn.h"
#include "../../include/dvgr_head.h"
#include "../../include/dvgr_inputs.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

struct Entry {
  decltype(&dvgr_embed_forward) embed_forward;
  decltype(&dvgr_embed_workspace_bytes) embed_workspace_bytes;
  decltype(&dvgr_embed_backward) embed_backward;
  decltype(&dvgr_distill_workspace_bytes) distill_workspace_bytes;
  decltype(&dvgr_distill_forward) distill_forward;
  decltype(&dvgr_distill_backward) distill_backward;
  decltype(&dvgr_attn_check) attn_check;
  decltype(&dvgr_attn_forward_workspace_bytes) attn_forward_workspace_bytes;
  decltype(&dvgr_attn_backward_workspace_bytes) attn_backward_workspace_bytes;
  decltype(&dvgr_attn_forward) attn_forward;
  decltype(&dvgr_attn_backward) attn_backward;
} E{};

void bind(const std::unordered_map<std::string, uintptr_t>& at) {
#define DVGR_BIND(name) E.name = reinterpret_cast<decltype(E.name)>(at.at("dvgr_" #name))
  DVGR_BIND(embed_forward); DVGR_BIND(embed_workspace_bytes); DVGR_BIND(embed_backward);
  DVGR_BIND(distill_workspace_bytes); DVGR_BIND(distill_forward); DVGR_BIND(distill_backward);
  DVGR_BIND(attn_check); DVGR_BIND(attn_forward_workspace_bytes); DVGR_BIND(attn_backward_workspace_bytes);
  DVGR_BIND(attn_forward); DVGR_BIND(attn_backward);
#undef DVGR_BIND
}

void check(int code, const char* what) {
  if (code == 0) return;
  const char* why = code == DVGR_E_DIMS ? "DVGR_E_DIMS (unsupported dimensions)" : code == DVGR_E_NULL ? "DVGR_E_NULL (null pointer)"
                  : code == DVGR_E_WORKSPACE ? "DVGR_E_WORKSPACE (workspace buffer too small)" : code == DVGR_E_ALIGN ? "DVGR_E_ALIGN (misaligned pointer)"
                  : code == DVGR_E_KIND ? "DVGR_E_KIND (unknown element / reduction kind)" : nullptr;
  TORCH_CHECK(code > 0 || why, what, " failed: ", code);
  TORCH_CHECK(code > 0, what, " failed: ", why);
  TORCH_CHECK(false, what, " failed: hipError_t ", code);
}

// What these nodes do not do and would not notice: an output without the tangent of its inputs reads as a constant, a trace would record
// the output's allocation alone.
void refuse_modes(const char* what, std::initializer_list<const Tensor*> inputs) {
  TORCH_CHECK(!torch::jit::tracer::isTracing(), what, " cannot be traced");
  for (const Tensor* t : inputs)
    TORCH_CHECK(!t->_fw_grad(/*level=*/0).defined(), what, " has no forward-mode derivative; got an input with a tangent");
}

int elem_code(const Tensor& t, const char* what) {
  TORCH_CHECK(t.is_cuda(), what, " runs on a ROCm device only (no CPU fallback); got a tensor on ", t.device());
  switch (t.scalar_type()) {
    case at::kFloat: return DVGR_ELEM_F32;
    case at::kBFloat16: return DVGR_ELEM_BF16;
    case at::kHalf: return DVGR_ELEM_F16;
    default: TORCH_CHECK(false, what, " takes fp32, bf16 and fp16 tensors; got ", t.scalar_type());
  }
}

hipStream_t stream_of(const Tensor& t) { return at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream(); }
Tensor bytes_on(const Tensor& t, size_t n) { return at::empty({(int64_t)n}, t.options().dtype(at::kByte)); }

// ---- captured backwards ---------------------------------------------------------------------------------------------------------
// autograd runs a node on the stream where it was made, and keeps one accumulation node for a leaf while any graph of it lives.  A
// backward that is captured and runs into a node of the default stream would draw that stream into the capture, which it cannot be
// part of and which ends the process: it is refused instead.  (Other streams join the capture and leave it again; wrappers that keep
// accumulation nodes make them on one.)  So the nodes in front of an operator are looked through, down to the leaves, while its backward is
// captured (and only then), whatever stands between it and them: views, copies, other operators.
bool outside_capture(Node* n) {
  const auto s = n->stream();                                       // (none: not a device's)
  return s && at::hip::HIPStreamMasqueradingAsCUDA(at::hip::HIPStreamMasqueradingAsCUDA::UNCHECKED, *s).stream() == nullptr;
}
bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }
// the nodes that the running backward reaches from `todo`, each once, until `found` says yes to one
template <typename F> bool reaches(std::vector<Node*> todo, F found) {
  const auto* wanted = torch::autograd::get_current_graph_task_exec_info();        // (without entries: all of them)
  std::unordered_set<Node*> seen;
  while (!todo.empty()) {
    Node* n = todo.back();
    todo.pop_back();
    if (!n || !seen.insert(n).second) continue;
    if (wanted && !wanted->empty()) {
      const auto it = wanted->find(n);
      if (it == wanted->end() || !it->second.should_execute()) continue;
    }
    if (found(n)) return true;
    for (const auto& e : n->next_edges()) todo.push_back(e.function.get());
  }
  return false;
}
// `n` is about to run: refuses if its gradients go on into such a node
void refuse_capture(const char* what, Node* n) {
  if (!capturing()) return;
  std::vector<Node*> from;
  for (size_t i = 0; i < n->num_outputs(); ++i)
    if (n->task_should_compute_output(i)) from.push_back(n->next_edge(i).function.get());
  TORCH_CHECK(!reaches(std::move(from), outside_capture), what, ": this backward is being captured while a graph of the same leaves lives that was "
              "made on the default stream: drop that graph's outputs (or detach them) before the capture");
}
// the same for the node of a Python autograd function, from inside its backward
void refuse_capture_here(const std::string& what) {
  if (const auto n = torch::autograd::get_current_node()) refuse_capture(what.c_str(), n.get());
}
// test aids: the leaves that a backward of `t` ends in; would a captured backward of `t` be refused
std::vector<Tensor> dbg_leaves(const Tensor& t) {
  std::vector<Tensor> out;
  reaches({t.grad_fn().get()}, [&](Node* n) {
    if (const auto* a = dynamic_cast<torch::autograd::AccumulateGrad*>(n)) out.push_back(a->variable);
    return false;
  });
  return out;
}
bool dbg_refuses_capture(const Tensor& t) { return reaches({t.grad_fn().get()}, outside_capture); }

struct OpNode : Node {
  const char* what = "";
  virtual variable_list gradients(variable_list&& grads) = 0;
  // do the gradients depend on the upstream gradient alone?  Otherwise on the inputs too, one of which wants a gradient: there is a node.
  virtual bool linear() const { return false; }
  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    if (!grads[0].defined()) return variable_list(num_outputs());
    refuse_capture(what, this);
    const bool again = at::GradMode::is_enabled() && (!linear() || grads[0].requires_grad());
    at::NoGradGuard no_grad;
    const c10::DeviceGuard guard(grads[0].device());
    variable_list out = gradients(std::move(grads));
    if (!again) return out;
    at::AutoGradMode grad(true);                                    // differentiating a gradient again says so, if it comes to it
    for (Tensor& t : out)
      if (t.defined()) t = t.detach().set_requires_grad(true);
    torch::autograd::DelayedError err(std::string(what) + ": its gradient cannot be differentiated again", (int64_t)out.size());
    return err.apply(std::move(out));
  }
};

template <typename N> std::shared_ptr<N> make_node() { return std::shared_ptr<N>(new N(), torch::autograd::deleteNode); }

// ---- token embedding ---------------------------------------------------------------------------------------------------------
struct EmbedNode : OpNode {
  SavedVariable tokens_;
  int64_t vocab, wd, padding;
  int elem;
  float scale;
  std::string name() const override { return "EmbedTokensBackward"; }
  bool linear() const override { return true; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    tokens_.reset_data();
  }
  variable_list gradients(variable_list&& grads) override {
    const Tensor tokens = tokens_.unpack(), g = grads[0].contiguous();
    const int64_t n = tokens.numel();
    Tensor out = at::empty({vocab, wd}, g.options());
    const size_t bytes = E.embed_workspace_bytes(n, vocab, (int)wd, elem);
    const Tensor ws = bytes_on(g, bytes);
    check(E.embed_backward(g.data_ptr(), tokens.data_ptr<int64_t>(), n, vocab, (int)wd, elem, scale, padding, out.data_ptr(), ws.data_ptr(), bytes,
                           stream_of(g)), "dvgr_embed_backward");
    return {out};
  }
};

Tensor embed_tokens(const Tensor& table, Tensor tokens, double scale, std::optional<int64_t> padding_idx, const OptTensor& bad) {
  const char* what = "embed_tokens";
  refuse_modes(what, {&table});
  const int elem = elem_code(table, what);
  TORCH_CHECK(table.dim() == 2 && table.size(0) > 0 && table.size(1) > 0, what, ": the table is (vocab, wd), not empty; got ", table.sizes());
  const int64_t vocab = table.size(0), wd = table.size(1);
  TORCH_CHECK(wd < (1ll << 31), what, ": rows of up to 2^31 - 1 elements; got ", wd);
  TORCH_CHECK(at::isIntegralType(tokens.scalar_type(), false), what, ": tokens are integers; got ", tokens.scalar_type());
  TORCH_CHECK(tokens.device() == table.device(), what, ": the tokens are on ", tokens.device(), ", the table is on ", table.device());
  TORCH_CHECK(!bad || (bad->scalar_type() == at::kInt && bad->numel() == 1 && bad->device() == table.device()), what,
              ": `bad` is one int32 on the table's device");
  int64_t padding = -1;
  if (padding_idx) {
    padding = *padding_idx + (*padding_idx < 0 ? vocab : 0);
    TORCH_CHECK(padding >= 0 && padding < vocab, what, ": padding_idx ", *padding_idx, " is outside a table of ", vocab, " rows");
  }
  const c10::DeviceGuard guard(table.device());
  const hipStream_t st = stream_of(table);
  Tensor y;
  {
    at::NoGradGuard no_grad;
    if (tokens.scalar_type() != at::kLong) tokens = tokens.to(at::kLong);
    tokens = tokens.contiguous();
    const Tensor rows = table.contiguous();
    at::DimVector shape(tokens.sizes());
    shape.push_back(wd);
    y = at::empty(shape, table.options());
    check(E.embed_forward(rows.data_ptr(), vocab, (int)wd, elem, tokens.data_ptr<int64_t>(), tokens.numel(), (float)scale, y.data_ptr(),
                          bad ? bad->data_ptr<int32_t>() : nullptr, st), "dvgr_embed_forward");
  }
  if (at::GradMode::is_enabled() && table.requires_grad()) {
    auto n = make_node<EmbedNode>();
    n->set_next_edges(torch::autograd::collect_next_edges(table));
    n->what = what;
    n->tokens_ = SavedVariable(tokens, false);
    n->vocab = vocab; n->wd = wd; n->padding = padding; n->elem = elem; n->scale = (float)scale;
    torch::autograd::set_history(y, n);
  }
  return y;
}

// ---- distillation -------------------------------------------------------------------------------------------------------------
struct DistillNode : OpNode {
  SavedVariable logits_, values_, indices_, stats_;
  int reduction;
  float temperature;
  std::string name() const override { return "DistillationLossBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    logits_.reset_data(); values_.reset_data(); indices_.reset_data(); stats_.reset_data();
  }
  variable_list gradients(variable_list&& grads) override {
    const Tensor z = logits_.unpack(), v = values_.unpack(), i = indices_.unpack(), stats = stats_.unpack(), g = grads[0].contiguous();
    const int64_t R = z.size(0), C = z.size(1);
    Tensor out = at::empty({R, C}, z.options());
    check(E.distill_backward(z.data_ptr(), R > 1 ? z.stride(0) : C, elem_code(z, what), R, C, v.data_ptr(), elem_code(v, what), i.data_ptr<int64_t>(), (int)v.size(1),
                             temperature, stats.data_ptr<float>(), g.data_ptr<float>(), reduction ? 0 : 1, out.data_ptr(), C, stream_of(z)),
          "dvgr_distill_backward");
    return {out};
  }
};

// logits (R, C) with rows any distance apart, values and indices (R, K)
Tensor distillation_loss(Tensor z, Tensor v, Tensor i, double temperature, int64_t reduction) {
  const char* what = "distillation_loss";
  refuse_modes(what, {&z});
  const int elem = elem_code(z, what), elem_v = elem_code(v, what);
  const c10::DeviceGuard guard(z.device());
  const hipStream_t st = stream_of(z);
  const int64_t R = z.size(0), C = z.size(1), K = v.size(1);
  if (z.stride(1) != 1 || (R > 1 && z.stride(0) < C)) z = z.contiguous();      // (differentiable: its node passes the gradient on)
  Tensor rows, total, stats;
  {
    at::NoGradGuard no_grad;
    v = v.detach().contiguous();
    if (i.scalar_type() != at::kLong) i = i.to(at::kLong);
    i = i.contiguous();
    const auto f32 = z.options().dtype(at::kFloat);
    rows = at::empty({R}, f32);
    if (reduction) total = at::empty({}, f32);
    stats = at::empty({R + 1, 4}, f32);
    const size_t bytes = E.distill_workspace_bytes(R, C);
    const Tensor ws = bytes ? bytes_on(z, bytes) : Tensor();
    check(E.distill_forward(z.data_ptr(), R > 1 ? z.stride(0) : C, elem, R, C, v.data_ptr(), elem_v, i.data_ptr<int64_t>(), (int)K, (float)temperature,
                            (int)reduction, rows.data_ptr<float>(), reduction ? total.data_ptr<float>() : nullptr, stats.data_ptr<float>(),
                            bytes ? ws.data_ptr() : nullptr, bytes, st), "dvgr_distill_forward");
  }
  Tensor out = reduction ? total : rows;
  if (at::GradMode::is_enabled() && z.requires_grad()) {
    auto n = make_node<DistillNode>();
    n->set_next_edges(torch::autograd::collect_next_edges(z));
    n->what = what;
    n->logits_ = SavedVariable(z, false); n->values_ = SavedVariable(v, false); n->indices_ = SavedVariable(i, false);
    n->stats_ = SavedVariable(stats, false);
    n->reduction = (int)reduction; n->temperature = (float)temperature;
    torch::autograd::set_history(out, n);
  }
  return out;
}

// ---- cross attention ------------------------------------------------------------------------------------------------------------
// `t`, or a copy whose heads start at multiples of 16 bytes (the stride of a dimension of one element does not count)
Tensor ready(const Tensor& t) {
  const int64_t per = 16 / t.element_size();
  const auto off = [&](int d) { return t.size(d) > 1 && t.stride(d) % per != 0; };
  if ((t.size(3) > 1 && t.stride(3) != 1) || off(2) || off(1) || off(0) || ((uintptr_t)t.data_ptr() & 15) ||
      (t.size(1) > 1 && t.stride(1) * (int64_t)t.element_size() >= (1ll << 32)))
    return t.clone(at::MemoryFormat::Contiguous);
  return t;
}
dvgr_attn_view view(const Tensor& t) {
  const auto stride = [&](int d) { return t.size(d) > 1 ? t.stride(d) : 0; };
  return {t.data_ptr(), stride(0), stride(1), stride(2)};
}

dvgr_attn_problem problem(const Tensor& q, const Tensor& k, const Tensor& v, const Tensor& o, const Tensor& o_lo, const Tensor& lens, const Tensor& mask,
                          float scale, const Tensor& lse) {
  dvgr_attn_problem a{};
  a.B = (int32_t)q.size(0); a.Lq = (int32_t)q.size(1); a.Lk = (int32_t)k.size(1); a.H = (int32_t)q.size(2); a.Hk = (int32_t)k.size(2);
  a.Dh = (int32_t)q.size(3);
  a.elem = elem_code(q, "cross_attention");
  a.scale = scale;
  a.q = view(q); a.k = view(k); a.v = view(v); a.o = view(o);
  a.o_lo = o_lo.defined() ? o_lo.data_ptr() : nullptr;
  a.lens = lens.defined() ? lens.data_ptr<int64_t>() : nullptr;
  if (mask.defined()) { a.mask = reinterpret_cast<const uint8_t*>(mask.data_ptr()); a.mask_stride = mask.stride(0); }
  a.lse = lse.defined() ? lse.data_ptr<float>() : nullptr;
  return a;
}

struct AttendNode : OpNode {
  SavedVariable q_, k_, v_, o_, o_lo_, lse_, lens_, mask_;
  float scale;
  std::string name() const override { return "CrossAttentionBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable* s : {&q_, &k_, &v_, &o_, &o_lo_, &lse_, &lens_, &mask_}) s->reset_data();
  }
  variable_list gradients(variable_list&& grads) override {
    const Tensor q = q_.unpack(), k = k_.unpack(), v = v_.unpack(), o = o_.unpack(shared_from_this()), lse = lse_.unpack(), g = ready(grads[0]);
    const dvgr_attn_problem a = problem(q, k, v, o, o_lo_.unpack(), lens_.unpack(), mask_.unpack(), scale, lse);
    const bool wq = task_should_compute_output(0), wk = task_should_compute_output(1), wv = task_should_compute_output(2);
    dvgr_attn_grads gr{};
    gr.g_o = view(g);
    Tensor gq, gk, gv;
    if (wq) { gq = at::empty(q.sizes(), q.options()); gr.g_q = view(gq); }
    if (wk || wv) {
      gk = at::empty(k.sizes(), k.options()); gv = at::empty(v.sizes(), v.options());
      gr.g_k = view(gk); gr.g_v = view(gv);
    }
    const size_t bytes = E.attn_backward_workspace_bytes(&a);
    const Tensor ws = bytes_on(q, bytes);
    check(E.attn_backward(&a, &gr, ws.data_ptr(), bytes, stream_of(q)), "dvgr_attn_backward");
    return {gq, wk ? gk : Tensor(), wv ? gv : Tensor()};
  }
};

Tensor cross_attention(const Tensor& q, const Tensor& k, const Tensor& v, const OptTensor& lens_, const OptTensor& mask_, std::optional<double> scale_) {
  const char* what = "cross_attention";
  refuse_modes(what, {&q, &k, &v});
  elem_code(q, what);
  TORCH_CHECK(q.dim() == 4 && k.dim() == 4 && k.sizes() == v.sizes() && q.size(0) == k.size(0) && q.size(3) == k.size(3), what,
              ": q (B, Lq, H, Dh), k and v (B, Lk, Hk, Dh); got ", q.sizes(), ", ", k.sizes(), ", ", v.sizes());
  TORCH_CHECK(k.scalar_type() == q.scalar_type() && v.scalar_type() == q.scalar_type() && k.device() == q.device() && v.device() == q.device(), what,
              ": q, k and v have one type and are on one device");
  const int64_t B = q.size(0), Lq = q.size(1), H = q.size(2), Dh = q.size(3), Lk = k.size(1), Hk = k.size(2);
  TORCH_CHECK(H > 0 && Hk > 0 && H % Hk == 0, what, ": the query heads (", H, ") are a multiple of the key heads (", Hk, ")");
  TORCH_CHECK(Dh % 8 == 0 && Dh >= 8 && Dh <= 128, what, ": the head size is a multiple of 8 up to 128; got ", Dh);
  for (const int64_t s : {B, Lq, Lk, H}) TORCH_CHECK(s < (1ll << 30), what, ": a dimension of ", s, " is too large");
  const double scale = scale_ ? *scale_ : 1.0 / std::sqrt((double)Dh);
  TORCH_CHECK(scale >= 1e-30 && scale <= 1e30, what, ": scale is a positive number, 1e-30 to 1e30; got ", scale);
  const c10::DeviceGuard guard(q.device());
  const hipStream_t st = stream_of(q);
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  Tensor lens, mask, o, o_lo, lse, qr, kr, vr;
  {
    at::NoGradGuard no_grad;
    if (lens_) {
      TORCH_CHECK(lens_->dim() == 1 && lens_->size(0) == B && lens_->device() == q.device() &&
                  (lens_->scalar_type() == at::kLong || lens_->scalar_type() == at::kInt), what,
                  ": lens is (B) int64 or int32 on q's device; got ", lens_->sizes(), " ", lens_->scalar_type(), " on ", lens_->device());
      lens = lens_->to(at::kLong).contiguous();
    }
    if (mask_) {
      TORCH_CHECK(mask_->dim() == 2 && mask_->size(0) == B && mask_->size(1) == Lk && mask_->device() == q.device() && mask_->scalar_type() == at::kBool,
                  what, ": mask is (B, Lk) bool on q's device; got ", mask_->sizes(), " ", mask_->scalar_type(), " on ", mask_->device());
      mask = mask_->stride(1) == 1 ? *mask_ : mask_->contiguous();
    }
    qr = ready(q); kr = ready(k); vr = ready(v);
    o = at::empty({B, Lq, H, Dh}, q.options());
    if (grad) {
      lse = at::empty({B, H, Lq}, q.options().dtype(at::kFloat));
      if (q.scalar_type() != at::kFloat) o_lo = at::empty({B, Lq, H, Dh}, q.options());
    }
    const dvgr_attn_problem a = problem(qr, kr, vr, o, o_lo, lens, mask, (float)scale, lse);
    check(E.attn_check(&a), "dvgr_attn_check");
    const size_t bytes = E.attn_forward_workspace_bytes(&a);
    const Tensor ws = bytes ? bytes_on(q, bytes) : Tensor();
    check(E.attn_forward(&a, bytes ? ws.data_ptr() : nullptr, bytes, st), "dvgr_attn_forward");
  }
  if (grad) {
    auto n = make_node<AttendNode>();
    n->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
    n->what = what;
    n->q_ = SavedVariable(qr, false); n->k_ = SavedVariable(kr, false); n->v_ = SavedVariable(vr, false);
    n->o_lo_ = SavedVariable(o_lo, false); n->lse_ = SavedVariable(lse, false); n->lens_ = SavedVariable(lens, false); n->mask_ = SavedVariable(mask, false);
    n->scale = (float)scale;
    torch::autograd::set_history(o, n);
    n->o_ = SavedVariable(o, true);
  }
  return o;
}

}  // namespace

PYBIND11_MODULE(_dvgr_torch, m) {
  m.def("bind", &bind);
  m.def("embed_tokens", &embed_tokens);
  m.def("distillation_loss", &distillation_loss);
  m.def("cross_attention", &cross_attention);
  m.def("refuse_capture", &refuse_capture_here);
  m.def("dbg_leaves", &dbg_leaves);
  m.def("dbg_refuses_capture", &dbg_refuses_capture);
}
