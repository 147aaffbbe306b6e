// The token operators in native code (included by bind.cpp): arguments in their plain form, launch, and the graph node that calls the backward launch.
// What bounds a small training call is the host: through Python autograd functions a layer norm's forward and backward pass took 150 us of host time for 33 us of kernels, most
// of it in the hand-overs between the autograd engine's thread and the interpreter.
// Forms that a function does not take (None is returned) go to the Python path of fovi_b200/tokens.py, which gives the same values from the same kernels.
#pragma once
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>

#include <math.h>

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

struct TokenAbi {
  decltype(&fovi_status_string) status = nullptr;
  decltype(&fovi_last_cuda_error) cuda_error = nullptr;
  decltype(&fovi_layer_norm_forward) norm = nullptr;
  decltype(&fovi_layer_norm_workspace_bytes) norm_work = nullptr;
  decltype(&fovi_layer_norm_backward) norm_back = nullptr;
  decltype(&fovi_rotary) rotary = nullptr;
  decltype(&fovi_attention_workspace_bytes) attend_work = nullptr;
  decltype(&fovi_attention_forward) attend = nullptr;
  decltype(&fovi_attention_backward) attend_back = nullptr;
} tok;

// The stream that the engine has made current on this thread for the device of a backward call.
void* stream_of(const at::Tensor& t) {
  const c10::impl::VirtualGuardImpl guard(c10::DeviceType::CUDA);
  return guard.getStream(t.device()).native_handle();
}
void launched(int rc, const char* what) {
  TORCH_CHECK(rc == FOVI_OK, what, ": ", tok.status(rc), rc == FOVI_ERR_CUDA ? std::string(" (") + tok.cuda_error() + ")" : std::string());
}
// A gradient's own gradient is not built: in a graph that is kept for one, a node that says so.
void once(variable_list& grads, const variable_list& from, const char* name) {
  if (!at::GradMode::is_enabled()) return;
  bool any = false;
  for (const auto& t : from) any = any || (t.defined() && t.requires_grad());
  if (!any) return;
  for (auto& g : grads)
    if (g.defined()) {
      auto stop = std::make_shared<torch::autograd::Error>(std::string(name) + ": the gradient cannot be differentiated again", torch::autograd::collect_next_edges(from));
      torch::autograd::set_history(g, stop);
    }
}
void* out_ptr(const at::Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
bool real_type(const at::Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
bool needs_graph(const at::Tensor& a, const at::Tensor* b = nullptr, const at::Tensor* c = nullptr) {
  return at::GradMode::is_enabled() && (a.requires_grad() || (b && b->requires_grad()) || (c && c->requires_grad()));
}
// A tensor with a tangent: the Python path names the derivative that is not built, where this one would lose it.
bool has_tangent(const at::Tensor& t) { return t._fw_grad(/*level=*/0).defined(); }
at::Tensor or_none(const at::Tensor* t) { return t ? *t : at::Tensor(); }

// ------------------------------------------------------------------------------------------------------------ layer norm
struct LayerNormNode : Node {
  SavedVariable x, w;
  at::Tensor stats;
  at::DimVector shape[2];                // of the weight and the bias: C values, in whatever shape
  std::string name() const override { return "FoviLayerNormBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    x.reset_data(); w.reset_data(); stats.reset();
  }
  variable_list apply(variable_list&& in) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!in[0].defined()) return out;
    const at::Tensor xv = x.unpack(), wv = w.unpack();
    const variable_list from = {in[0], xv, wv};
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor g = in[0].contiguous();
      const int64_t C = xv.size(-1), rows = xv.numel() / C;
      const int dev = xv.get_device();
      if (task_should_compute_output(0)) out[0] = fresh(xv.sizes(), xv.scalar_type(), dev);
      for (int i = 1; i < 3; ++i)
        if (task_should_compute_output(i)) out[i] = fresh(shape[i - 1], at::kFloat, dev);
      const bool sums = out[1].defined() || out[2].defined();
      const int64_t bytes = sums ? tok.norm_work(rows, (int)C) : 0;
      const at::Tensor work = sums ? fresh({bytes}, at::kByte, dev) : at::Tensor();
      launched(tok.norm_back(xv.const_data_ptr(), code_of(xv.scalar_type()), rows, (int)C, C, g.const_data_ptr(), code_of(g.scalar_type()), C,
                             wv.defined() ? wv.const_data_ptr<float>() : nullptr, stats.const_data_ptr<float>(), out_ptr(out[0]), (float*)out_ptr(out[1]),
                             (float*)out_ptr(out[2]), out_ptr(work), bytes, stream_of(xv)),
               "fovi_layer_norm_backward");
    }
    once(out, from, "layer_norm");
    return out;
  }
};

// x, weight or None, bias or None, eps, device, stream
BODY(layer_norm, 6)
  const at::Tensor* x = plain(v[0], dev);
  if (!x || !real_type(*x) || x->dim() < 1 || x->numel() == 0 || !x->is_contiguous()) GENERAL;
  const int64_t C = x->size(-1), rows = x->numel() / C;
  const float *wp, *bp;
  if (C > INT32_MAX || !bias_arg(v[1], dev, C, &wp) || !bias_arg(v[2], dev, C, &bp)) GENERAL;
  const double eps = PyFloat_AsDouble(v[3]);
  if (PyErr_Occurred()) return nullptr;
  if (!(eps >= 0)) GENERAL;
  const at::Tensor *w = wp ? plain(v[1], dev) : nullptr, *b = bp ? plain(v[2], dev) : nullptr;
  if (has_tangent(*x) || (w && has_tangent(*w)) || (b && has_tangent(*b))) GENERAL;
  at::Tensor y;
  int rcode;
  {
    Release r;
    const bool graph = needs_graph(*x, w, b);
    at::Tensor stats;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      y = fresh(x->sizes(), x->scalar_type(), dev);
      if (graph) stats = fresh({rows, 2}, at::kFloat, dev);
    }
    const int type = code_of(x->scalar_type());
    rcode = tok.norm(x->const_data_ptr(), type, rows, (int)C, C, wp, bp, (float)eps, y.mutable_data_ptr(), type, (float*)out_ptr(stats), st);
    if (graph && !rcode) {
      std::shared_ptr<LayerNormNode> node(new LayerNormNode(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*x, or_none(w), or_none(b)));
      node->x = SavedVariable(*x, false);
      node->w = SavedVariable(or_none(w), false);
      if (w) node->shape[0] = w->sizes();
      if (b) node->shape[1] = b->sizes();
      node->stats = stats;
      torch::autograd::set_history(y, node);
    }
  }
  return status_or(rcode, y);
END

// ------------------------------------------------------------------------------------------------------------ rotary positions
struct Turn {
  int axes = 0, prefix = 0, interleaved = 0;
  int32_t pairs[4] = {0, 0, 0, 0};
};
int turn(const at::Tensor& x, const at::Tensor& pos, const at::Tensor& f, const Turn& t, bool inverse, const at::Tensor& y, void* st) {
  const int64_t strides[3] = {x.stride(0), x.stride(1), x.stride(2)};
  return tok.rotary(x.const_data_ptr(), code_of(x.scalar_type()), (int)x.size(0), (int)x.size(1), (int)x.size(2), (int)x.size(3), strides, pos.const_data_ptr<float>(),
                    pos.dim() == 2 ? 0 : pos.stride(0), t.axes, t.pairs, f.const_data_ptr<float>(), t.prefix, t.interleaved, inverse, y.mutable_data_ptr(), st);
}

struct RotaryNode : Node {
  SavedVariable pos, f;
  Turn how;
  std::string name() const override { return "FoviRotaryBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    pos.reset_data(); f.reset_data();
  }
  variable_list apply(variable_list&& in) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(1);
    if (!in[0].defined() || !task_should_compute_output(0)) return out;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor g = in[0].stride(3) == 1 ? in[0] : in[0].contiguous(), p = pos.unpack(), fr = f.unpack();
      out[0] = fresh(g.sizes(), g.scalar_type(), g.get_device());
      launched(turn(g, p, fr, how, true, out[0], stream_of(g)), "fovi_rotary");
    }
    once(out, {in[0]}, "rotary");
    return out;
  }
};

// x, positions, frequencies, pairs per axis (tuple), prefix, interleaved, device, stream
BODY(rotary, 8)
  const at::Tensor *x = plain(v[0], dev), *pos = plain(v[1], dev), *f = plain(v[2], dev);
  if (!x || !pos || !f || !PyTuple_CheckExact(v[3]) || !real_type(*x) || x->dim() != 4 || x->numel() == 0 || x->stride(3) != 1 || pos->scalar_type() != at::kFloat ||
      f->scalar_type() != at::kFloat || !pos->is_contiguous() || !f->is_contiguous() || (pos->dim() != 2 && pos->dim() != 3))
    GENERAL;
  Turn t;
  t.axes = (int)PyTuple_GET_SIZE(v[3]);
  if (t.axes < 1 || t.axes > 4) GENERAL;
  int64_t P = 0;
  for (int i = 0; i < t.axes; ++i) {
    const long n = num(PyTuple_GET_ITEM(v[3], i));
    if (PyErr_Occurred()) return nullptr;
    if (n < 0 || n > INT32_MAX / 8) GENERAL;
    t.pairs[i] = (int32_t)n;
    P += n;
  }
  const long prefix = num(v[4]), inter = num(v[5]);
  if (PyErr_Occurred()) return nullptr;
  const int64_t B = x->size(0), L = x->size(1);
  if (prefix < 0 || prefix > L || 2 * P > x->size(3) || f->numel() != P || pos->size(-1) != t.axes || pos->size(-2) != L - prefix || (pos->dim() == 3 && pos->size(0) != B) ||
      B > INT32_MAX || L > INT32_MAX || x->size(2) > INT32_MAX || x->size(3) > INT32_MAX || needs_graph(*pos, f) || has_tangent(*x) ||
      has_tangent(*pos) || has_tangent(*f))
    GENERAL;
  t.prefix = (int)prefix; t.interleaved = (int)inter;
  at::Tensor y;
  int rcode;
  {
    Release r;
    {
      at::AutoDispatchBelowADInplaceOrView below;
      y = fresh(x->sizes(), x->scalar_type(), dev);
    }
    rcode = turn(*x, *pos, *f, t, false, y, st);
    if (!rcode && needs_graph(*x)) {
      std::shared_ptr<RotaryNode> node(new RotaryNode(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*x));
      node->pos = SavedVariable(*pos, false);
      node->f = SavedVariable(*f, false);
      node->how = t;
      torch::autograd::set_history(y, node);
    }
  }
  return status_or(rcode, y);
END

// ------------------------------------------------------------------------------------------------------------ attention
// Channels contiguous, and bf16 rows as the tensor copies want them (tokens.py copies what is not).
bool rows_plain(const at::Tensor& t) {
  if (t.stride(3) != 1) return false;
  if (t.scalar_type() != at::kBFloat16 || t.size(3) % 8) return true;
  return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15) == 0 && (t.size(1) == 1 || (t.stride(1) % 8 == 0 && t.stride(1) > 0)) &&
         (t.size(2) == 1 || t.stride(2) % 8 == 0) && (t.size(0) == 1 || t.stride(0) % 8 == 0);
}
void put_strides(int64_t* s, const at::Tensor& t) { for (int i = 0; i < 3; ++i) s[i] = t.stride(i); }

struct AttentionNode : Node {
  SavedVariable q, k, v, o, lengths, mask;
  at::Tensor lse;
  float scale = 0.f;
  std::string name() const override { return "FoviAttentionBackward"; }
  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    q.reset_data(); k.reset_data(); v.reset_data(); o.reset_data(); lengths.reset_data(); mask.reset_data(); lse.reset();
  }
  variable_list apply(variable_list&& in) override {
    std::lock_guard<std::mutex> lock(mutex_);
    variable_list out(3);
    if (!in[0].defined()) return out;
    const at::Tensor qv = q.unpack(), kv = k.unpack(), vv = v.unpack(), ov = o.unpack(shared_from_this()), len = lengths.unpack(), mk = mask.unpack();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const at::Tensor g = rows_plain(in[0]) ? in[0] : in[0].clone(at::MemoryFormat::Contiguous);
      const int dev = qv.get_device(), type = code_of(qv.scalar_type());
      const int B = (int)qv.size(0), Lq = (int)qv.size(1), H = (int)qv.size(2), D = (int)qv.size(3), Lk = (int)kv.size(1), Hkv = (int)kv.size(2);
      if (task_should_compute_output(0)) out[0] = fresh(qv.sizes(), qv.scalar_type(), dev);
      at::Tensor dv;
      if (task_should_compute_output(1)) out[1] = fresh(kv.sizes(), kv.scalar_type(), dev);
      if (out[1].defined() || task_should_compute_output(2)) dv = fresh(kv.sizes(), kv.scalar_type(), dev);
      const int64_t bytes = tok.attend_work(type, B, Lq, Lk, H, Hkv, D, 1);
      const at::Tensor work = fresh({bytes}, at::kByte, dev);
      int64_t s[12];
      put_strides(s, qv); put_strides(s + 3, kv); put_strides(s + 6, vv); put_strides(s + 9, g);
      launched(tok.attend_back(qv.const_data_ptr(), kv.const_data_ptr(), vv.const_data_ptr(), ov.const_data_ptr(), g.const_data_ptr(), type, B, Lq, Lk, H, Hkv, D, s,
                               len.defined() ? len.const_data_ptr<int32_t>() : nullptr, mk.defined() ? (const uint8_t*)mk.const_data_ptr() : nullptr, scale,
                               lse.const_data_ptr<float>(), out_ptr(out[0]), out_ptr(out[1]), out_ptr(dv), work.mutable_data_ptr(), bytes, stream_of(qv)),
               "fovi_attention_backward");
      if (task_should_compute_output(2)) out[2] = dv;
    }
    once(out, {in[0], qv, kv, vv}, "cross_attention");
    return out;
  }
};

// q, k, v, key_lengths or None, key_mask or None, scale or None, device, stream
BODY(attention, 8)
  const at::Tensor *q = plain(v[0], dev), *k = plain(v[1], dev), *s = plain(v[2], dev), *len = nullptr, *mask = nullptr;
  if (!q || !k || !s || !real_type(*q) || k->scalar_type() != q->scalar_type() || s->scalar_type() != q->scalar_type() || q->dim() != 4 || k->dim() != 4 ||
      s->sizes() != k->sizes() || k->size(0) != q->size(0) || k->size(3) != q->size(3) || q->numel() == 0 || k->numel() == 0)
    GENERAL;
  const int64_t B = q->size(0), Lq = q->size(1), H = q->size(2), D = q->size(3), Lk = k->size(1), Hkv = k->size(2);
  if (H % Hkv || D > 128 || B > INT32_MAX || Lq > INT32_MAX || Lk > INT32_MAX || H > INT32_MAX || !rows_plain(*q) || !rows_plain(*k) || !rows_plain(*s) ||
      has_tangent(*q) || has_tangent(*k) || has_tangent(*s))
    GENERAL;
  if (v[3] != Py_None && (!(len = plain(v[3], dev)) || len->scalar_type() != at::kInt || len->dim() != 1 || len->size(0) != B || !len->is_contiguous())) GENERAL;
  if (v[4] != Py_None &&
      (!(mask = plain(v[4], dev)) || mask->scalar_type() != at::kBool || mask->dim() != 2 || mask->size(0) != B || mask->size(1) != Lk || !mask->is_contiguous()))
    GENERAL;
  const double scale = v[5] == Py_None ? 1.0 / sqrt((double)D) : PyFloat_AsDouble(v[5]);
  if (PyErr_Occurred()) return nullptr;
  if (!std::isfinite(scale)) GENERAL;
  at::Tensor o;
  int rcode;
  {
    Release r;
    const bool graph = needs_graph(*q, k, s);
    const int type = code_of(q->scalar_type());
    at::Tensor lse, work;
    const int64_t bytes = tok.attend_work(type, (int)B, (int)Lq, (int)Lk, (int)H, (int)Hkv, (int)D, 0);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      o = fresh(q->sizes(), q->scalar_type(), dev);
      if (graph) lse = fresh({B, H, Lq}, at::kFloat, dev);
      if (bytes > 0) work = fresh({bytes}, at::kByte, dev);
    }
    int64_t st9[9];
    put_strides(st9, *q); put_strides(st9 + 3, *k); put_strides(st9 + 6, *s);
    rcode = tok.attend(q->const_data_ptr(), k->const_data_ptr(), s->const_data_ptr(), type, (int)B, (int)Lq, (int)Lk, (int)H, (int)Hkv, (int)D, st9,
                       len ? len->const_data_ptr<int32_t>() : nullptr, mask ? (const uint8_t*)mask->const_data_ptr() : nullptr, (float)scale, o.mutable_data_ptr(),
                       (float*)out_ptr(lse), out_ptr(work), bytes, st);
    if (graph && !rcode) {
      std::shared_ptr<AttentionNode> node(new AttentionNode(), torch::autograd::deleteNode);
      node->set_next_edges(torch::autograd::collect_next_edges(*q, *k, *s));
      node->q = SavedVariable(*q, false); node->k = SavedVariable(*k, false); node->v = SavedVariable(*s, false);
      node->lengths = SavedVariable(or_none(len), false); node->mask = SavedVariable(or_none(mask), false);
      node->lse = lse; node->scale = (float)scale;
      torch::autograd::set_history(o, node);
      node->o = SavedVariable(o, true);
    }
  }
  return status_or(rcode, o);
END

}  // namespace
