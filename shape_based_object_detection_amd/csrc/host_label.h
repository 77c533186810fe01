// The label-vocabulary operators' calls (operators.Loss.topk_distill_loss, operators.Logits.process_logits,
// operators.Embedding.scaled_embedding) in C++: argument forms, allocations, launches and C++ autograd nodes,
// so that a call costs its launches and not the interpreter.  Part of _sbodhost (hostpack.cpp).
//
// Each returns the result; None when an argument needs a conversion, a copy, a check's error or a device
// change (core.py's path converts or raises: the errors live in one place); an int for a failing sbod status.
#pragma once

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/VirtualGuardImpl.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>
#include <unordered_set>
#include <vector>

#include "sbod.h"

namespace sbod_label {

inline int label_dt(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return SBOD_DT_F32;
    case at::kBFloat16: return SBOD_DT_BF16;
    case at::kHalf: return SBOD_DT_F16;
    default: return -1;
  }
}
inline bool is_id(const at::Tensor &t) { return t.scalar_type() == at::kLong || t.scalar_type() == at::kInt; }
inline bool wants(const at::Tensor &t) { return t.defined() && t.requires_grad() && at::GradMode::is_enabled(); }
// core._constant refuses it: a derivative of either mode would be dropped.
inline bool varies(const at::Tensor &t) { return wants(t) || t._fw_grad(0).defined(); }
// [n, v] whose rows are contiguous and apart, as core._rows_of takes them without a copy.
inline bool good_rows(const at::Tensor &t) {
  return t.dim() == 2 && (t.stride(1) == 1 || t.size(1) <= 1) && (t.size(0) <= 1 || t.stride(0) >= t.size(1));
}
inline int64_t row_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
// core._empty_rows
inline at::Tensor empty_rows(const at::Tensor &t) {
  const int64_t n = t.size(0), v = t.size(1), es = t.element_size(), per = 16 / es;
  const int64_t shift = static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) / es;
  const int64_t ld = v + (row_stride(t) - v) % per;
  if (shift == 0 && ld == v) return at::empty({n, v}, t.options());
  return at::empty({n * ld + shift}, t.options()).as_strided({n, v}, {ld, 1}, shift);
}
inline const at::Tensor *tensor_of(PyObject *o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }
inline void *ptr_of(const at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
inline PyObject *wrap_status(int st, at::Tensor &&t) {
  return st != SBOD_OK ? PyLong_FromLong(st) : THPVariable_Wrap(std::move(t));
}

// core.differentiable_once
inline at::Tensor once(at::Tensor grad) {
  if (!at::GradMode::is_enabled()) return grad;
  at::Tensor g = grad.detach();
  g.set_requires_grad(true);
  const auto late = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice a function that is differentiable once", 1);
  return (*late)({g})[0];
}

// foreign_leaves(t): whether a leaf below t has a gradient node that was made on another stream than the current one
// (a graph from before still holds it).  Such a backward pass synchronises the two streams.
inline PyObject *foreign_leaves_call(PyObject *const *a, Py_ssize_t n) {
  const at::Tensor *t = n == 1 ? tensor_of(a[0]) : nullptr;
  if (!t) {
    PyErr_SetString(PyExc_TypeError, "foreign_leaves: expected a tensor");
    return nullptr;
  }
  const c10::Stream now = c10::impl::VirtualGuardImpl(t->device().type()).getStream(t->device());
  std::shared_ptr<torch::autograd::Node> top = t->grad_fn();
  if (!top) top = torch::autograd::impl::try_get_grad_accumulator(*t);
  std::vector<torch::autograd::Node *> todo;
  std::unordered_set<torch::autograd::Node *> seen;
  if (top) todo.push_back(top.get());
  while (!todo.empty()) {
    torch::autograd::Node *node = todo.back();
    todo.pop_back();
    if (!seen.insert(node).second) continue;
    if (dynamic_cast<torch::autograd::AccumulateGrad *>(node)) {
      const auto made = node->stream();
      if (made && made->device() == now.device() && *made != now) Py_RETURN_TRUE;
    }
    for (const auto &e : node->next_edges())
      if (e.is_valid()) todo.push_back(e.function.get());
  }
  Py_RETURN_FALSE;
}

// ------------------------------------------------------------------------------------------ distillation
struct DistillCall {
  at::Tensor ids, top, lse, w;
  int dt, top_dt, reduction, status = 0;
  float temperature;
  bool want;
  int64_t unit;   // data pointer of core.unit_grad(device), 0 if none yet
  void *stream;
};

struct DistillFn : public torch::autograd::Function<DistillFn> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &x, DistillCall *c) {
    const int64_t n = x.size(0), v = x.size(1);
    const int k = static_cast<int>(c->top.size(1));
    const int64_t nst = sbod_distill_stats_bytes(n, v, k, c->dt) / sizeof(float);
    const size_t nb = sbod_distill_workspace_bytes(n, v, k, c->dt);
    const auto f32 = x.options().dtype(at::kFloat);
    at::Tensor kept = at::empty({nst + 1}, f32), ws = at::empty({static_cast<int64_t>(nb)}, x.options().dtype(at::kByte));
    const bool red = c->reduction != SBOD_REDUCE_NONE;
    at::Tensor out = red ? at::empty({}, f32) : at::empty({n}, f32), grad;
    // (float16 gradients at upstream 1 would underflow before a loss scale reaches them)
    if (c->want && red && c->dt != SBOD_DT_F16) grad = empty_rows(x);
    float *stats = kept.data_ptr<float>();
    c->status = sbod_distill_fwd(x.data_ptr(), c->dt, n, v, row_stride(x), c->ids.data_ptr(),
                                 c->ids.scalar_type() == at::kLong, c->top.data_ptr(), c->top_dt, k,
                                 static_cast<float *>(ptr_of(c->lse)), static_cast<float *>(ptr_of(c->w)), c->temperature,
                                 c->reduction, red ? nullptr : out.data_ptr<float>(), red ? out.data_ptr<float>() : nullptr,
                                 stats + nst, stats, ptr_of(grad), grad.defined() ? row_stride(grad) : 0, ws.data_ptr(), nb,
                                 c->stream);
    if (c->want) {
      ctx->save_for_backward({x, c->ids, c->top, c->lse, c->w, kept});
      ctx->saved_data["grad"] = grad;
      ctx->saved_data["stream"] = reinterpret_cast<int64_t>(c->stream);
      ctx->saved_data["unit"] = c->unit;
      ctx->saved_data["form"] = std::vector<int64_t>{c->dt, c->top_dt, c->reduction};
      ctx->saved_data["temperature"] = static_cast<double>(c->temperature);
      ctx->set_materialize_grads(false);
    }
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list go) {
    if (go.empty() || !go[0].defined()) return {at::Tensor(), at::Tensor()};
    auto saved = ctx->get_saved_variables();
    auto &sd = ctx->saved_data;
    const at::Tensor &x = saved[0], &ids = saved[1], &top = saved[2], &lse = saved[3], &w = saved[4], &kept = saved[5];
    at::Tensor grad, g = go[0];
    const auto it = sd.find("grad");   // (a second backward of a retained graph computes its own)
    if (it != sd.end()) {
      grad = it->second.toTensor();
      sd.erase(it);
    }
    const bool written = grad.defined();
    const int64_t unit = sd["unit"].toInt();
    if (written && unit != 0 && reinterpret_cast<int64_t>(g.data_ptr()) == unit) return {once(std::move(grad)), at::Tensor()};
    if (!written) grad = empty_rows(x);
    if (g.scalar_type() != at::kFloat || !g.is_contiguous()) g = g.detach().to(at::kFloat).contiguous();
    const auto form = sd["form"].toIntVector();
    const float *stats = kept.data_ptr<float>();
    const int st = sbod_distill_bwd(x.data_ptr(), static_cast<int>(form[0]), x.size(0), x.size(1), row_stride(x), ids.data_ptr(),
                                    ids.scalar_type() == at::kLong, top.data_ptr(), static_cast<int>(form[1]),
                                    static_cast<int>(top.size(1)), static_cast<float *>(ptr_of(lse)),
                                    static_cast<float *>(ptr_of(w)), static_cast<float>(sd["temperature"].toDouble()),
                                    static_cast<int>(form[2]), stats + (kept.numel() - 1), stats, g.data_ptr<float>(), written,
                                    grad.data_ptr(), row_stride(grad), reinterpret_cast<void *>(sd["stream"].toInt()));
    if (st != SBOD_OK) throw std::runtime_error(std::string("sbod_distill_bwd: ") + sbod_last_error());
    return {once(std::move(grad)), at::Tensor()};
  }
};

// label_distill(logits, ids, top, lse | None, weights | None, temperature, reduction, unit_ptr | None, stream)
inline PyObject *label_distill_call(PyObject *const *a, Py_ssize_t n) {
  if (n != 9) {
    PyErr_SetString(PyExc_TypeError, "label_distill: expected 9 arguments");
    return nullptr;
  }
  const at::Tensor *x = tensor_of(a[0]), *ids = tensor_of(a[1]), *top = tensor_of(a[2]), *lse = tensor_of(a[3]), *w = tensor_of(a[4]);
  if (!x || !ids || !top || (!lse && a[3] != Py_None) || (!w && a[4] != Py_None) || !PyFloat_Check(a[5])) Py_RETURN_NONE;
  DistillCall c;
  c.temperature = static_cast<float>(PyFloat_AS_DOUBLE(a[5]));
  c.reduction = static_cast<int>(PyLong_AsLong(a[6]));
  c.unit = a[7] == Py_None ? 0 : static_cast<int64_t>(reinterpret_cast<intptr_t>(PyLong_AsVoidPtr(a[7])));
  c.stream = PyLong_AsVoidPtr(a[8]);
  if (PyErr_Occurred()) return nullptr;
  const auto vec = [&](const at::Tensor *t) {
    return !t || (t->dim() == 1 && t->size(0) == x->size(0) && t->scalar_type() == at::kFloat && t->is_contiguous() &&
                  t->device() == x->device() && !varies(*t));
  };
  if (!x->is_cuda() || (c.dt = label_dt(*x)) < 0 || (c.top_dt = label_dt(*top)) < 0 || !is_id(*ids) || !good_rows(*x) ||
      x->size(1) < 1 || ids->dim() != 2 || !ids->is_contiguous() || !top->is_contiguous() || ids->sizes() != top->sizes() ||
      ids->size(0) != x->size(0) || ids->size(1) < 1 || ids->size(1) > 1024 || ids->device() != x->device() ||
      top->device() != x->device() || varies(*top) || !vec(lse) || !vec(w) ||
      !(c.temperature >= 1e-30f && c.temperature <= 1e30f))
    Py_RETURN_NONE;
  c.ids = *ids, c.top = top->detach();
  if (lse) c.lse = lse->detach();
  if (w) c.w = w->detach();
  c.want = wants(*x);
  const c10::DeviceGuard guard(x->device());
  at::Tensor out = DistillFn::apply(*x, &c);
  return wrap_status(c.status, std::move(out));
}

// ------------------------------------------------------------------------------------------ embedding
struct EmbedCall {
  at::Tensor ids;
  int dt, status = 0;
  float scale;
  int64_t pad;
  void *stream;
};

struct EmbedFn : public torch::autograd::Function<EmbedFn> {
  static at::Tensor forward(torch::autograd::AutogradContext *ctx, const at::Tensor &w, EmbedCall *c) {
    auto sizes = c->ids.sizes().vec();
    sizes.push_back(w.size(1));
    at::Tensor out = at::empty(sizes, w.options());
    c->status = sbod_embed_fwd(w.data_ptr(), c->dt, w.size(0), w.size(1), c->ids.data_ptr(), c->ids.scalar_type() == at::kLong,
                               c->ids.numel(), c->scale, out.data_ptr(), c->stream);
    ctx->save_for_backward({c->ids});
    ctx->saved_data["form"] = std::vector<int64_t>{w.size(0), w.size(1), c->dt, c->pad, reinterpret_cast<int64_t>(c->stream)};
    ctx->saved_data["scale"] = static_cast<double>(c->scale);
    ctx->set_materialize_grads(false);
    return out;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx, torch::autograd::variable_list go) {
    if (go.empty() || !go[0].defined()) return {at::Tensor(), at::Tensor()};
    const at::Tensor ids = ctx->get_saved_variables()[0], g = go[0].contiguous();
    const auto form = ctx->saved_data["form"].toIntVector();
    const int64_t v = form[0], d = form[1], n = ids.numel();
    at::Tensor grad = at::empty({v, d}, g.options());
    const size_t nb = sbod_embed_bwd_workspace_bytes(n, v, d);
    at::Tensor ws = at::empty({static_cast<int64_t>(nb)}, g.options().dtype(at::kByte));
    const int st = sbod_embed_bwd(g.data_ptr(), static_cast<int>(form[2]), v, d, ids.data_ptr(), ids.scalar_type() == at::kLong, n,
                                  form[3], static_cast<float>(ctx->saved_data["scale"].toDouble()), grad.data_ptr(),
                                  ws.data_ptr(), nb, reinterpret_cast<void *>(form[4]));
    if (st != SBOD_OK) throw std::runtime_error(std::string("sbod_embed_bwd: ") + sbod_last_error());
    return {once(std::move(grad)), at::Tensor()};
  }
};

// label_embed(ids, weight, scale, padding id | None, stream)
inline PyObject *label_embed_call(PyObject *const *a, Py_ssize_t n) {
  if (n != 5) {
    PyErr_SetString(PyExc_TypeError, "label_embed: expected 5 arguments");
    return nullptr;
  }
  const at::Tensor *ids = tensor_of(a[0]), *w = tensor_of(a[1]);
  if (!ids || !w || !PyFloat_Check(a[2]) || (a[3] != Py_None && !PyLong_Check(a[3]))) Py_RETURN_NONE;
  EmbedCall c;
  const double scale = PyFloat_AS_DOUBLE(a[2]);
  c.scale = static_cast<float>(scale);
  int beyond = 0;   // (an id beyond 64 bits: core.py's error)
  c.pad = a[3] == Py_None ? -1 : PyLong_AsLongLongAndOverflow(a[3], &beyond);
  c.stream = PyLong_AsVoidPtr(a[4]);
  if (PyErr_Occurred()) return nullptr;
  if (!w->is_cuda() || (c.dt = label_dt(*w)) < 0 || !is_id(*ids) || ids->device() != w->device() || w->dim() != 2 ||
      !w->is_contiguous() || !ids->is_contiguous() || !std::isfinite(scale) || beyond || w->size(0) < 1 ||
      (a[3] != Py_None && (c.pad < 0 || c.pad >= w->size(0))))
    Py_RETURN_NONE;
  c.ids = *ids;
  const c10::DeviceGuard guard(w->device());
  at::Tensor out = EmbedFn::apply(*w, &c);
  return wrap_status(c.status, std::move(out));
}

// ------------------------------------------------------------------------------------------ logits
// label_logits(logits, history | None, history_len | None, prompt_len | None, repetition, presence, frequency,
//              bias | None, bias_ids | None, bias_values | None, allowed | None, out | None, stream)
inline PyObject *label_logits_call(PyObject *const *a, Py_ssize_t n_args) {
  if (n_args != 13) {
    PyErr_SetString(PyExc_TypeError, "label_logits: expected 13 arguments");
    return nullptr;
  }
  const at::Tensor *x = tensor_of(a[0]);
  if (!x || !x->is_cuda() || !good_rows(*x) || x->size(1) < 1 || varies(*x)) Py_RETURN_NONE;
  const int dt = label_dt(*x);
  if (dt < 0) Py_RETURN_NONE;
  const int64_t n = x->size(0), v = x->size(1);
  bool ok = true;
  const at::Tensor *none = nullptr;
  // an optional tensor on the logits' device
  const auto opt = [&](PyObject *o) -> const at::Tensor * {
    if (o == Py_None) return none;
    const at::Tensor *t = tensor_of(o);
    if (!t || t->device() != x->device() || varies(*t)) ok = false;
    // (in place, an argument in the logits' own storage: core.py's path looks at where)
    if (ok && a[11] == a[0] && t->is_alias_of(*x)) ok = false;
    return ok ? t : none;
  };
  const at::Tensor *hist = opt(a[1]), *hlen = opt(a[2]), *plen = opt(a[3]), *bias = opt(a[7]), *bids = opt(a[8]), *bval = opt(a[9]),
                   *mask = opt(a[10]);
  // per row, or one row for all
  const auto rows = [&](const at::Tensor *t, int64_t cols) {
    if (!t) return;
    if (t->dim() == 1) ok = ok && t->is_contiguous();
    else ok = ok && t->dim() == 2 && t->size(0) == n && (t->size(1) <= 1 || t->stride(1) == 1);
    ok = ok && (cols < 0 || t->size(-1) == cols);
  };
  const auto ld = [&](const at::Tensor *t) { return t && t->dim() == 2 ? t->stride(0) : 0; };
  const auto cols = [&](const at::Tensor *t) { return t && t->dim() > 0 ? t->size(-1) : 0; };
  rows(hist, -1), rows(bias, v), rows(bids, -1), rows(bval, bids ? cols(bids) : -1), rows(mask, -1);
  const auto lens = [&](const at::Tensor *t) {
    ok = ok && (!t || (hist && t->dim() == 1 && t->size(0) == n && t->scalar_type() == at::kInt && t->is_contiguous()));
  };
  lens(hlen), lens(plen);
  float scalar[3] = {1.f, 0.f, 0.f};
  const float *per_row[3] = {nullptr, nullptr, nullptr};
  for (int i = 0; ok && i < 3; ++i) {
    if (PyFloat_Check(a[4 + i])) {
      scalar[i] = static_cast<float>(PyFloat_AS_DOUBLE(a[4 + i]));
    } else {
      const at::Tensor *t = tensor_of(a[4 + i]);
      ok = t && t->device() == x->device() && !varies(*t) && t->dim() == 1 && t->size(0) == n && t->scalar_type() == at::kFloat &&
           t->is_contiguous();
      if (ok) per_row[i] = t->data_ptr<float>();
    }
  }
  int kind = SBOD_MASK_NONE;
  if (ok && mask) {
    kind = mask->scalar_type() == at::kBool ? SBOD_MASK_BYTES : SBOD_MASK_BITS;
    ok = kind == SBOD_MASK_BYTES ? cols(mask) == v : mask->scalar_type() == at::kInt && cols(mask) >= (v + 31) / 32;
  }
  ok = ok && (!hist || (is_id(*hist) && cols(hist) < (1 << 29))) && cols(bids) <= 4096 && (!bids == !bval) && (!bids || (is_id(*bids) && bval->scalar_type() == at::kFloat)) &&
       (!bias || bias->scalar_type() == at::kFloat || bias->scalar_type() == x->scalar_type()) &&
       (per_row[0] || (scalar[0] > 0.f && std::isfinite(scalar[0]))) && (a[11] == Py_None || a[11] == a[0]);
  if (!ok) Py_RETURN_NONE;
  void *stream = PyLong_AsVoidPtr(a[12]);
  if (PyErr_Occurred()) return nullptr;
  const c10::DeviceGuard guard(x->device());
  const at::NoGradGuard no_grad;
  at::Tensor out = a[11] == Py_None ? empty_rows(*x) : *x;
  const int st = sbod_logits_process(x->data_ptr(), dt, n, v, row_stride(*x), hist ? hist->data_ptr() : nullptr,
                                     hist && hist->scalar_type() == at::kLong, cols(hist), ld(hist),
                                     hlen ? hlen->data_ptr<int32_t>() : nullptr, plen ? plen->data_ptr<int32_t>() : nullptr, per_row[0],
                                     per_row[1], per_row[2], scalar[0], scalar[1], scalar[2], bias ? bias->data_ptr() : nullptr,
                                     bias ? label_dt(*bias) : 0, ld(bias), bids ? bids->data_ptr() : nullptr,
                                     bids && bids->scalar_type() == at::kLong, bval ? bval->data_ptr<float>() : nullptr,
                                     static_cast<int>(cols(bids)), ld(bids), ld(bval), mask ? mask->data_ptr() : nullptr, kind, ld(mask),
                                     out.data_ptr(), row_stride(out), stream);
  if (st == SBOD_OK && a[11] == a[0]) {   // in place: the caller's own object, and its version counted
    x->unsafeGetTensorImpl()->bump_version();
    Py_INCREF(a[0]);
    return a[0];
  }
  return wrap_status(st, std::move(out));
}

// Nothing that ATen throws passes the interpreter.
template <PyObject *(*kCall)(PyObject *const *, Py_ssize_t)>
PyObject *guarded(PyObject *, PyObject *const *a, Py_ssize_t n) {
  try {
    return kCall(a, n);
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

}  // namespace sbod_label
