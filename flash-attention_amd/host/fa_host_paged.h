// The calls of the paged cache and of the norm in front of it, made natively (included by fa_host.cpp, whose rules hold here: a call that fails a
// check returns None and the binding runs it, and raises what it has to).  A decode step is a handful of such calls whose kernels take 4 to 15 us: what
// the host takes decides.  us of a pass among others with the binding's own calls / with these:
//   norm of a prompt of 61 tokens 28.0 / 6.1, its training step on 8 x 511 .. 1021 tokens 194 / 79 (kernels 30; an empty native function's takes 54), a
//   decode step of 32 sequences stored 29.1 / 5.9, attention of one token 23.9 / 7.8, eviction of 32 sequences' one key with two copies 28.7 / 16.1.
#pragma once

#include <ATen/core/grad_mode.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>

namespace {

struct PagedLibrary {
  int (*qk_norm)(const fa_qk_norm_args*);
  int (*qk_norm_bwd)(const fa_qk_norm_args*);
  size_t (*qk_norm_bwd_workspace_bytes)(const fa_qk_norm_args*);
  int (*append)(const fa_paged_append_args*, const fa_paged_scales*);
  int (*fwd)(const fa_paged_fwd_args*, const fa_paged_scales*, const fa_paged_prefix*);
  size_t (*fwd_workspace_bytes)(const fa_paged_fwd_args*, const fa_paged_scales*, const fa_paged_prefix*);
  int (*read)(const fa_paged_read_args*, const fa_paged_scales*);
  int (*key_weights)(const fa_paged_fwd_args*);
  int (*evict)(const fa_paged_evict_args*);
  size_t (*evict_workspace_bytes)(const fa_paged_evict_args*);
} g_paged;
bool g_paged_bound = false;

// bind_paged(addresses of the ten entry points above, in their order)
PyObject* py_bind_paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr int kEntries = 10;
  if (n != kEntries) return PyErr_Format(PyExc_TypeError, "bind_paged takes %d addresses", kEntries);
  void* f[kEntries];
  for (int i = 0; i < kEntries; i++) {
    f[i] = PyLong_AsVoidPtr(a[i]);
    if (!f[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  static_assert(sizeof(g_paged) == sizeof(f), "a pointer each");
  memcpy(&g_paged, f, sizeof(f));
  g_paged_bound = true;
  Py_RETURN_NONE;
}

int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kHalf ? FA_FP16 : t.scalar_type() == at::kBFloat16 ? FA_BF16 : -1; }
bool needs_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!c10::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}
bool small(int64_t n) { return n >= 0 && n <= INT32_MAX; }
at::TensorOptions plain(const at::Tensor& t) { return t.options().memory_format(at::MemoryFormat::Contiguous).requires_grad(false); }

// (rows, heads, dim), or (batch, seqlen, heads, dim) with evenly strided rows, as the kernels read them
struct Rows {
  char* p;
  int64_t rows, heads, dim, row_stride, head_stride;
};
bool rows_of(const at::Tensor& t, const at::Tensor& like, Rows* r) {
  const int d = (int)t.dim();
  if ((d != 3 && d != 4) || !t.is_cuda() || t.device() != like.device() || t.scalar_type() != like.scalar_type() || t.stride(d - 1) != 1) return false;
  if (d == 4 && t.size(0) > 1 && t.stride(0) != t.size(1) * t.stride(1)) return false;
  r->p = static_cast<char*>(ptr(t));
  r->rows = d == 4 ? t.size(0) * t.size(1) : t.size(0);
  r->heads = t.size(d - 2);
  r->dim = t.size(d - 1);
  r->row_stride = t.stride(d - 3);
  r->head_stride = t.stride(d - 2);
  const auto ok = [](int64_t s) { return s >= 0 && s % 8 == 0 && s < ((int64_t)1 << 24); };
  return ok(r->row_stride) && ok(r->head_stride) && reinterpret_cast<uintptr_t>(r->p) % 16 == 0 && small(r->rows) && small(r->heads);
}
bool norm_ok(const at::Tensor* qw, const at::Tensor* kw, const at::Tensor& like, int64_t dim) {
  auto one = [&](const at::Tensor* w) {
    return w && w->device() == like.device() && (w->scalar_type() == like.scalar_type() || w->scalar_type() == at::kFloat) && w->dim() == 1 && w->size(0) == dim &&
           w->is_contiguous();
  };
  return one(qw) && one(kw) && qw->scalar_type() == kw->scalar_type();
}
bool angles_ok(const at::Tensor* c, const at::Tensor* s, const at::Tensor& like, int64_t dim) {
  if (!c && !s) return true;
  auto one = [&](const at::Tensor* t) {
    return t && t->device() == like.device() && t->scalar_type() == like.scalar_type() && t->dim() == 2 && t->size(1) == dim / 2 && t->size(0) > 0 && small(t->size(0)) &&
           t->is_contiguous() && reinterpret_cast<uintptr_t>(ptr(*t)) % 8 == 0;
  };
  return one(c) && one(s) && c->size(0) == s->size(0);
}
bool positions_ok(const at::Tensor* p, const at::Tensor& like, int64_t rows) {
  return !p || (p->device() == like.device() && p->scalar_type() == at::kInt && p->numel() == rows && p->is_contiguous());
}
bool dim_ok(int64_t d) { return d == 16 || d == 32 || d == 64 || d == 128; }

// ---- norm and rotation of q and k
void fill_norm(fa_qk_norm_args* f, const at::Tensor& q, const Rows& rq, const Rows& rk, const at::Tensor& qw, const at::Tensor& kw, const at::Tensor* cos,
               const at::Tensor* sin, const at::Tensor* positions, int64_t seqlen, double eps) {
  memset(f, 0, sizeof(*f));
  f->struct_bytes = sizeof(*f);
  f->dtype = dtype_of(q);
  f->q = rq.p; f->q_row_stride = rq.row_stride; f->q_head_stride = rq.head_stride;
  f->k = rk.p; f->k_row_stride = rk.row_stride; f->k_head_stride = rk.head_stride;
  f->q_weight = ptr(qw); f->k_weight = ptr(kw);
  f->weight_dtype = qw.scalar_type() == at::kFloat ? FA_FP32 : f->dtype;
  if (cos) { f->cos_table = ptr(*cos); f->sin_table = ptr(*sin); f->table_rows = (int32_t)cos->size(0); }
  if (positions) f->positions = (const int32_t*)ptr(*positions);
  f->n_rows = rq.rows;
  f->nheads_q = (int32_t)rq.heads; f->nheads_k = (int32_t)rk.heads; f->head_dim = (int32_t)rq.dim;
  f->seqlen = (int32_t)seqlen;
  f->eps = (float)eps;
  f->stream = stream_of(q);
}
const at::Tensor* given(const at::Tensor& t) { return t.defined() ? &t : nullptr; }

struct QkNormRotary : public torch::autograd::Function<QkNormRotary> {
  static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& qw, const at::Tensor& kw,
                                                const at::Tensor& cos, const at::Tensor& sin, const at::Tensor& positions, int64_t seqlen, double eps) {
    Rows rq, rk;
    TORCH_CHECK(rows_of(q, q, &rq) && rows_of(k, q, &rk));  // (looked at by the caller)
    at::Tensor qo = at::empty(q.sizes(), plain(q)), ko = at::empty(k.sizes(), plain(k));
    fa_qk_norm_args f;
    fill_norm(&f, q, rq, rk, qw, kw, given(cos), given(sin), given(positions), seqlen, eps);
    f.q_out = ptr(qo); f.q_out_row_stride = rq.heads * rq.dim; f.q_out_head_stride = rq.dim;
    f.k_out = ptr(ko); f.k_out_row_stride = rk.heads * rk.dim; f.k_out_head_stride = rk.dim;
    const int rc = g_paged.qk_norm(&f);
    TORCH_CHECK(rc == 0, "flash_attn_gfx950 error ", rc, ": ", g_lib.last_error());
    if (ctx) {
      ctx->save_for_backward({q, k, qw, kw, cos, sin, positions});
      ctx->saved_data["seqlen"] = seqlen;
      ctx->saved_data["eps"] = eps;
    }
    return {qo, ko};
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const at::Tensor &q = saved[0], &k = saved[1], &qw = saved[2], &kw = saved[3];
    Rows rq, rk, gq, gk;
    at::Tensor dqo = grads[0], dko = grads[1];
    // (a clone: contiguous() hands a contiguous tensor back whose address is the fault)
    if (!rows_of(dqo, q, &gq)) dqo = dqo.clone(at::MemoryFormat::Contiguous);
    if (!rows_of(dko, q, &gk)) dko = dko.clone(at::MemoryFormat::Contiguous);
    TORCH_CHECK(rows_of(q, q, &rq) && rows_of(k, q, &rk) && rows_of(dqo, q, &gq) && rows_of(dko, q, &gk), "apply_qk_norm_rotary: gradients of another dtype or device");
    at::Tensor dq = at::empty(q.sizes(), plain(q)), dk = at::empty(k.sizes(), plain(k)), dqw = at::empty(qw.sizes(), plain(qw)), dkw = at::empty(kw.sizes(), plain(kw));
    fa_qk_norm_args f;
    fill_norm(&f, q, rq, rk, qw, kw, given(saved[4]), given(saved[5]), given(saved[6]), ctx->saved_data["seqlen"].toInt(), ctx->saved_data["eps"].toDouble());
    f.dq_out = gq.p; f.dq_out_row_stride = gq.row_stride; f.dq_out_head_stride = gq.head_stride;
    f.dk_out = gk.p; f.dk_out_row_stride = gk.row_stride; f.dk_out_head_stride = gk.head_stride;
    f.dq = ptr(dq); f.dq_row_stride = rq.heads * rq.dim; f.dq_head_stride = rq.dim;
    f.dk = ptr(dk); f.dk_row_stride = rk.heads * rk.dim; f.dk_head_stride = rk.dim;
    f.dq_weight = ptr(dqw); f.dk_weight = ptr(dkw);
    at::Tensor ws = at::empty({(int64_t)g_paged.qk_norm_bwd_workspace_bytes(&f)}, plain(q).dtype(at::kByte));
    f.workspace = ptr(ws);
    f.workspace_bytes = (size_t)ws.numel();
    const int rc = g_paged.qk_norm_bwd(&f);
    TORCH_CHECK(rc == 0, "flash_attn_gfx950 error ", rc, ": ", g_lib.last_error());
    torch::autograd::variable_list out = {dq, dk, dqw, dkw};
    if (c10::GradMode::is_enabled())  // (a graph of the gradients was asked for: differentiating through it raises)
      out = torch::autograd::DelayedError("trying to differentiate twice a function that can be differentiated once: apply_qk_norm_rotary", 4)(std::move(out));
    out.resize(9);
    return out;
  }
};

// qk_norm_rotary(q, k, q_weight, k_weight, cos, sin, positions, eps) -> (q', k') or None
PyObject* qk_norm_rotary(PyObject* const* a, Py_ssize_t n) {
  if (n != 8) return PyErr_Format(PyExc_TypeError, "qk_norm_rotary takes 8 arguments");
  bool ok = true;
  const at::Tensor *q = tensor(a[0], ok), *k = tensor(a[1], ok), *qw = tensor(a[2], ok), *kw = tensor(a[3], ok), *cos = tensor(a[4], ok), *sin = tensor(a[5], ok),
                   *pos = tensor(a[6], ok);
  double eps;
  Rows rq, rk;
  if (!ok || !g_paged_bound || !on_current_device(q) || !k || !as_double(a[7], &eps) || !(eps >= 0) || dtype_of(*q) < 0 || q->dim() != k->dim() || !rows_of(*q, *q, &rq) ||
      !rows_of(*k, *q, &rk) || rq.rows != rk.rows || rq.rows <= 0 || rq.heads <= 0 || rk.heads <= 0 || rq.dim != rk.dim || !dim_ok(rq.dim) ||
      (q->dim() == 4 && (q->size(0) != k->size(0) || q->size(1) != k->size(1))) || !norm_ok(qw, kw, *q, rq.dim) || !angles_ok(cos, sin, *q, rq.dim) ||
      !positions_ok(pos, *q, rq.rows) || (cos && cos->requires_grad()) || (sin && sin->requires_grad()))
    Py_RETURN_NONE;
  const int64_t seqlen = q->dim() == 4 ? q->size(1) : q->size(0);
  if (cos && !pos && seqlen > cos->size(0)) Py_RETURN_NONE;
  torch::autograd::variable_list out;
  const bool grad = needs_grad({q, k, qw, kw});
  const at::Tensor none;
  {
    pybind11::gil_scoped_release no_gil;
    const at::Tensor &c = cos ? *cos : none, &s = sin ? *sin : none, &p = pos ? *pos : none;
    out = grad ? QkNormRotary::apply(*q, *k, *qw, *kw, c, s, p, seqlen, eps) : QkNormRotary::forward(nullptr, *q, *k, *qw, *kw, c, s, p, seqlen, eps);
  }
  PyObject *o0 = THPVariable_Wrap(std::move(out[0])), *o1 = THPVariable_Wrap(std::move(out[1]));
  PyObject* r = o0 && o1 ? PyTuple_Pack(2, o0, o1) : nullptr;
  Py_XDECREF(o0);
  Py_XDECREF(o1);
  return r;
}

// ---- the paged cache
// The exponents of a cache in 8 bits, beside its tensors (both or neither)
struct Scales {
  const at::Tensor *k = nullptr, *v = nullptr;
  fa_paged_scales s;
  const fa_paged_scales* get() {
    if (!k) return nullptr;
    s = fa_paged_scales{(uint32_t)sizeof(s), 0, ptr(*k), ptr(*v)};
    return &s;
  }
};
// Fills a cache's fields; false where the binding would refuse (or copy) something.
bool fill_cache(fa_paged_cache* c, const at::Tensor* k, const at::Tensor* v, bool needs_v, const at::Tensor* table, const at::Tensor* lens, int64_t max_k,
                const at::Tensor* weights, const at::Tensor* positions, const Scales& scales = Scales()) {
  memset(c, 0, sizeof(*c));
  if (!g_paged_bound || !on_current_device(k) || (scales.k ? k->scalar_type() != at::kFloat8_e4m3fn : dtype_of(*k) < 0) || !scales.k != !scales.v || k->dim() != 4 ||
      k->stride(3) != 1 || !dim_ok(k->size(3)) || (needs_v && !v))
    return false;
  if (v && (v->device() != k->device() || v->scalar_type() != k->scalar_type() || v->sizes() != k->sizes() || v->stride(3) != 1)) return false;
  if (!table || table->device() != k->device() || table->scalar_type() != at::kInt || table->dim() != 2 || (table->stride(1) != 1 && table->size(1) != 1)) return false;
  const int64_t batch = table->size(0), cols = table->size(1);
  if (batch <= 0 || cols <= 0 || !small(batch) || !small(cols) || !lens || lens->device() != k->device() || lens->scalar_type() != at::kInt || lens->dim() != 1 ||
      lens->size(0) != batch || !lens->is_contiguous() || !small(k->size(0)) || !small(k->size(1)) || !small(k->size(2)) || k->numel() == 0 || max_k <= 0)
    return false;
  auto beside = [&](const at::Tensor* t, at::ScalarType type) {
    return !t || (t->device() == k->device() && t->scalar_type() == type && t->dim() == 3 && t->size(0) == k->size(0) && t->size(1) == k->size(2) &&
                  t->size(2) == k->size(1) && t->is_contiguous());
  };
  if (!beside(weights, at::kFloat) || !beside(positions, at::kInt) || !beside(scales.k, at::kByte) || !beside(scales.v, at::kByte)) return false;
  c->k_cache = ptr(*k);
  c->k_page_stride = k->stride(0); c->k_slot_stride = k->stride(1); c->k_head_stride = k->stride(2);
  if (v) {
    c->v_cache = ptr(*v);
    c->v_page_stride = v->stride(0); c->v_slot_stride = v->stride(1); c->v_head_stride = v->stride(2);
  }
  c->page_table = (const int32_t*)ptr(*table);
  c->table_row_stride = batch > 1 ? table->stride(0) : cols;
  c->seqlens_k = (const int32_t*)ptr(*lens);
  c->n_pages = (int32_t)k->size(0); c->page_size = (int32_t)k->size(1); c->table_cols = (int32_t)cols;
  c->batch = (int32_t)batch; c->nheads_k = (int32_t)k->size(2); c->head_dim = (int32_t)k->size(3);
  c->nheads_q = c->nheads_k;
  c->max_seqlen_k = (int32_t)(max_k < INT32_MAX ? max_k : INT32_MAX);
  if (weights) c->key_weights = (float*)ptr(*weights);
  if (positions) c->key_positions = (int32_t*)ptr(*positions);
  return true;
}
bool fill_queries(fa_paged_cache* c, const at::Tensor* q, const at::Tensor& k, const at::Tensor* cu, int64_t max_q) {
  if (!q || !cu || !q->is_cuda() || q->device() != k.device() || dtype_of(*q) < 0 || (k.scalar_type() != at::kFloat8_e4m3fn && q->scalar_type() != k.scalar_type()) ||
      q->dim() != 3 || q->size(2) != k.size(3) || q->stride(2) != 1 || q->size(1) <= 0 || !small(q->size(1)) || q->size(1) % k.size(2) != 0 || !small(q->size(0)) || max_q <= 0 || !is_cu(cu, k) || cu->size(0) != (int64_t)c->batch + 1)
    return false;
  c->cu_seqlens_q = (const int32_t*)ptr(*cu);
  c->nheads_q = (int32_t)q->size(1);
  c->total_q = (int32_t)q->size(0);
  c->max_seqlen_q = (int32_t)max_q;
  return true;
}

// paged_append(q, k, v, k_cache, v_cache, table, cu, seqlens, q_weight, k_weight, cos, sin, positions, eps, key_weights, key_positions[, k_scales, v_scales])
// -> the new q, True without one, or None
PyObject* paged_append(PyObject* const* a, Py_ssize_t n) {
  if (n != 16 && n != 18) return PyErr_Format(PyExc_TypeError, "paged_append takes 16 or 18 arguments");
  bool ok = true;
  const at::Tensor* t[13];
  for (int i = 0; i < 13; i++) t[i] = tensor(a[i], ok);
  const at::Tensor *q = t[0], *k = t[1], *v = t[2], *kc = t[3], *cu = t[6], *qw = t[8], *kw = t[9], *cos = t[10], *sin = t[11], *pos = t[12];
  const at::Tensor *weights = tensor(a[14], ok), *positions = tensor(a[15], ok);
  Scales scales;
  if (n == 18) scales.k = tensor(a[16], ok), scales.v = tensor(a[17], ok);
  fa_paged_append_args f;
  memset(&f, 0, sizeof(f));
  double eps;
  Rows rk, rv, rq;
  if (!ok || !as_double(a[13], &eps) || needs_grad({q, k, v, qw, kw}) || !k || !v || !kc || !t[5] || kc->dim() != 4 || t[5]->dim() != 2 ||
      !fill_cache(&f.cache, kc, t[4], true, t[5], t[7], t[5]->size(1) * kc->size(1), weights, positions, scales) || dtype_of(*k) < 0 || k->device() != kc->device() ||
      (!scales.k && k->scalar_type() != kc->scalar_type()) || k->dim() != 3 || v->dim() != 3 || !rows_of(*k, *k, &rk) || !rows_of(*v, *k, &rv) || rk.heads != kc->size(2) ||
      rv.heads != rk.heads || rk.dim != kc->size(3) || rv.dim != rk.dim || rv.rows != rk.rows || !is_cu(cu, *kc) || cu->size(0) != (int64_t)f.cache.batch + 1 ||
      ((qw || kw) && !norm_ok(qw, kw, *k, rk.dim)) || !angles_ok(cos, sin, *k, rk.dim) || !positions_ok(pos, *k, rk.rows))
    Py_RETURN_NONE;
  if (q && (q->dim() != 3 || !rows_of(*q, *k, &rq) || rq.rows != rk.rows || rq.dim != rk.dim || rq.heads <= 0 || rq.heads % rk.heads != 0)) Py_RETURN_NONE;
  f.struct_bytes = sizeof(f);
  f.dtype = dtype_of(*k);
  f.cache.cu_seqlens_q = (const int32_t*)ptr(*cu);
  f.cache.total_q = (int32_t)rk.rows;
  f.cache.max_seqlen_q = (int32_t)(rk.rows > 0 ? rk.rows : 1);
  f.k = rk.p; f.k_row_stride = rk.row_stride; f.k_head_stride = rk.head_stride;
  f.v = rv.p; f.v_row_stride = rv.row_stride; f.v_head_stride = rv.head_stride;
  if (kw) {
    f.q_weight = ptr(*qw); f.k_weight = ptr(*kw);
    f.weight_dtype = kw->scalar_type() == at::kFloat ? FA_FP32 : f.dtype;
  }
  if (cos) { f.cos_table = ptr(*cos); f.sin_table = ptr(*sin); f.table_rows = (int32_t)cos->size(0); }
  if (pos) f.positions = (const int32_t*)ptr(*pos);
  f.eps = (float)eps;
  f.stream = stream_of(*kc);
  at::Tensor qo;
  if (q) {
    qo = at::empty(q->sizes(), plain(*q));
    f.cache.nheads_q = (int32_t)rq.heads;
    f.q = rq.p; f.q_row_stride = rq.row_stride; f.q_head_stride = rq.head_stride;
    f.q_out = ptr(qo); f.q_out_row_stride = rq.heads * rq.dim; f.q_out_head_stride = rq.dim;
  }
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_paged.append(&f, scales.get());
  Py_END_ALLOW_THREADS
  if (rc != 0) return refused(rc);
  if (!q) Py_RETURN_TRUE;
  return THPVariable_Wrap(std::move(qo));
}

// paged_fwd(q, k_cache, v_cache, table, cu, seqlens, max_q, max_k, scale or None, causal, return_lse[, k_scales, v_scales[, cu_groups, prefix_lens, max_prefix]])
// -> out, (out, lse) or None
PyObject* paged_fwd(PyObject* const* a, Py_ssize_t n) {
  if (n != 11 && n != 13 && n != 16) return PyErr_Format(PyExc_TypeError, "paged_fwd takes 11, 13 or 16 arguments");
  bool ok = true;
  const at::Tensor* t[6];
  for (int i = 0; i < 6; i++) t[i] = tensor(a[i], ok);
  const at::Tensor *q = t[0], *kc = t[1], *vc = t[2];
  fa_paged_fwd_args f;
  memset(&f, 0, sizeof(f));
  int64_t mq, mk;
  double scale = 0;
  int32_t causal, want_lse;
  Scales scales;
  if (n > 11) scales.k = tensor(a[11], ok), scales.v = tensor(a[12], ok);
  if (!ok || !as_int(a[6], &mq) || !as_int(a[7], &mk) || (a[8] != Py_None && !as_double(a[8], &scale)) || !as_flag(a[9], &causal) || !as_flag(a[10], &want_lse) ||
      needs_grad({q, kc, vc}) || !fill_cache(&f.cache, kc, vc, true, t[3], t[5], mk, nullptr, nullptr, scales) || !fill_queries(&f.cache, q, *kc, t[4], mq))
    Py_RETURN_NONE;
  fa_paged_prefix prefix;
  memset(&prefix, 0, sizeof(prefix));
  if (n == 16) {
    const at::Tensor *groups = tensor(a[13], ok), *lens = tensor(a[14], ok);
    int64_t most;
    const auto ints = [&](const at::Tensor* x) { return x && x->device() == kc->device() && x->scalar_type() == at::kInt && x->dim() == 1 && x->is_contiguous(); };
    if (!ok || !ints(groups) || !ints(lens) || lens->size(0) != f.cache.batch || groups->size(0) < 2 ||
        groups->size(0) > (int64_t)f.cache.batch + 1 || !as_int(a[15], &most))
      Py_RETURN_NONE;
    prefix = fa_paged_prefix{(uint32_t)sizeof(prefix), (int32_t)(groups->size(0) - 1), (int32_t)most, 0, (const int32_t*)ptr(*groups),
                             (const int32_t*)ptr(*lens)};
  }
  if (a[8] == Py_None) scale = 1 / std::sqrt((double)f.cache.head_dim);
  at::Tensor o = at::empty(q->sizes(), plain(*q)), lse, ws;
  f.struct_bytes = sizeof(f);
  f.dtype = dtype_of(*q);
  f.q = ptr(*q); f.q_row_stride = q->stride(0); f.q_head_stride = q->stride(1);
  f.o = ptr(o); f.o_row_stride = q->size(1) * q->size(2); f.o_head_stride = q->size(2);
  if (want_lse) {
    lse = at::empty({f.cache.batch, q->size(1), (mq + 15) / 16 * 16}, plain(*q).dtype(at::kFloat));
    f.softmax_lse = (float*)ptr(lse);
  }
  f.softmax_scale = (float)scale;
  f.is_causal = causal;
  const fa_paged_scales* const s8 = scales.get();
  const fa_paged_prefix* const px = n == 16 ? &prefix : nullptr;
  f.workspace_bytes = g_paged.fwd_workspace_bytes(&f, s8, px);
  if (f.workspace_bytes) {
    ws = at::empty({(int64_t)f.workspace_bytes}, plain(*q).dtype(at::kByte));
    f.workspace = ptr(ws);
  }
  f.stream = stream_of(*q);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_paged.fwd(&f, s8, px);
  Py_END_ALLOW_THREADS
  if (rc != 0) return refused(rc);
  PyObject* po = THPVariable_Wrap(std::move(o));
  if (!want_lse || !po) return po;
  PyObject* pl = THPVariable_Wrap(std::move(lse));
  PyObject* r = pl ? PyTuple_Pack(2, po, pl) : nullptr;
  Py_DECREF(po);
  Py_XDECREF(pl);
  return r;
}

// paged_read(k_cache, v_cache, table, cu, seqlens, total, dtype (0 fp16, 1 bf16), k_scales, v_scales) -> (k, v) or None
PyObject* paged_read(PyObject* const* a, Py_ssize_t n) {
  if (n != 9) return PyErr_Format(PyExc_TypeError, "paged_read takes 9 arguments");
  bool ok = true;
  const at::Tensor* t[5];
  for (int i = 0; i < 5; i++) t[i] = tensor(a[i], ok);
  const at::Tensor *kc = t[0], *vc = t[1], *cu = t[3];
  Scales scales;
  scales.k = tensor(a[7], ok);
  scales.v = tensor(a[8], ok);
  fa_paged_read_args f;
  memset(&f, 0, sizeof(f));
  int64_t total, dtype;
  if (!ok || !as_int(a[5], &total) || !as_int(a[6], &dtype) || (dtype != FA_FP16 && dtype != FA_BF16) || total < 0 || !kc || !t[2] || kc->dim() != 4 || t[2]->dim() != 2 ||
      needs_grad({kc, vc}) || !fill_cache(&f.cache, kc, vc, true, t[2], t[4], t[2]->size(1) * kc->size(1), nullptr, nullptr, scales) ||
      (!scales.k && dtype_of(*kc) != dtype) || !is_cu(cu, *kc) || cu->size(0) != (int64_t)f.cache.batch + 1)
    Py_RETURN_NONE;
  const at::TensorOptions as = plain(*kc).dtype(dtype == FA_FP16 ? at::kHalf : at::kBFloat16);
  at::Tensor k = at::empty({total, kc->size(2), kc->size(3)}, as), v = at::empty({total, kc->size(2), kc->size(3)}, as);
  f.struct_bytes = sizeof(f);
  f.dtype = (int32_t)dtype;
  f.cache.cu_seqlens_q = (const int32_t*)ptr(*cu);
  f.cache.total_q = (int32_t)total;
  f.cache.max_seqlen_q = (int32_t)(total > 0 ? total : 1);
  f.k_out = ptr(k); f.v_out = ptr(v);
  f.k_row_stride = f.v_row_stride = kc->size(2) * kc->size(3);
  f.k_head_stride = f.v_head_stride = kc->size(3);
  f.stream = stream_of(*kc);
  int rc;
  const fa_paged_scales* const s8 = scales.get();
  Py_BEGIN_ALLOW_THREADS
  rc = g_paged.read(&f, s8);
  Py_END_ALLOW_THREADS
  if (rc != 0) return refused(rc);
  PyObject *pk = THPVariable_Wrap(std::move(k)), *pv = THPVariable_Wrap(std::move(v));
  PyObject* r = pk && pv ? PyTuple_Pack(2, pk, pv) : nullptr;
  Py_XDECREF(pk);
  Py_XDECREF(pv);
  return r;
}

// paged_key_weights(q, lse, k_cache, key_weights, table, cu, seqlens, max_q, max_k, scale or None, causal) -> True or None
PyObject* paged_key_weights(PyObject* const* a, Py_ssize_t n) {
  if (n != 11) return PyErr_Format(PyExc_TypeError, "paged_key_weights takes 11 arguments");
  bool ok = true;
  const at::Tensor* t[7];
  for (int i = 0; i < 7; i++) t[i] = tensor(a[i], ok);
  const at::Tensor *q = t[0], *lse = t[1], *kc = t[2], *weights = t[3];
  fa_paged_fwd_args f;
  memset(&f, 0, sizeof(f));
  int64_t mq, mk;
  double scale = 0;
  int32_t causal;
  if (!ok || !as_int(a[7], &mq) || !as_int(a[8], &mk) || (a[9] != Py_None && !as_double(a[9], &scale)) || !as_flag(a[10], &causal) || !weights || !lse ||
      needs_grad({q, kc}) || !fill_cache(&f.cache, kc, nullptr, false, t[4], t[6], mk, weights, nullptr) || !fill_queries(&f.cache, q, *kc, t[5], mq) ||
      lse->device() != q->device() || lse->scalar_type() != at::kFloat || !lse->is_contiguous() || lse->dim() != 3 || lse->size(0) != f.cache.batch ||
      lse->size(1) != q->size(1) || lse->size(2) != (mq + 15) / 16 * 16)
    Py_RETURN_NONE;
  if (a[9] == Py_None) scale = 1 / std::sqrt((double)f.cache.head_dim);
  f.struct_bytes = sizeof(f);
  f.dtype = dtype_of(*q);
  f.q = ptr(*q); f.q_row_stride = q->stride(0); f.q_head_stride = q->stride(1);
  f.softmax_lse = (float*)ptr(*lse);
  f.softmax_scale = (float)scale;
  f.is_causal = causal;
  f.stream = stream_of(*q);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_paged.key_weights(&f);
  Py_END_ALLOW_THREADS
  if (rc != 0) return refused(rc);
  Py_RETURN_TRUE;
}

// paged_evict(k_cache, v_cache, key_weights, key_positions, table, seqlens, next_positions, budget, recent, max_k) -> the new lengths or None
PyObject* paged_evict(PyObject* const* a, Py_ssize_t n) {
  if (n != 10) return PyErr_Format(PyExc_TypeError, "paged_evict takes 10 arguments");
  bool ok = true;
  const at::Tensor* t[7];
  for (int i = 0; i < 7; i++) t[i] = tensor(a[i], ok);
  fa_paged_evict_args f;
  memset(&f, 0, sizeof(f));
  int64_t budget, recent, mk;
  if (!ok || !as_int(a[7], &budget) || !as_int(a[8], &recent) || !as_int(a[9], &mk) || needs_grad({t[0], t[1]}) || !t[2] || !t[3] || !t[6] ||
      !fill_cache(&f.cache, t[0], t[1], true, t[4], t[5], mk, t[2], t[3]) || t[6]->device() != t[0]->device() || t[6]->scalar_type() != at::kInt || t[6]->dim() != 1 ||
      t[6]->size(0) != f.cache.batch || !t[6]->is_contiguous())
    Py_RETURN_NONE;
  at::Tensor lens = at::empty({f.cache.batch}, plain(*t[5]));
  f.struct_bytes = sizeof(f);
  f.budget = (int32_t)budget;
  f.recent = (int32_t)recent;
  f.next_positions = (const int32_t*)ptr(*t[6]);
  f.new_seqlens_k = (int32_t*)ptr(lens);
  f.workspace_bytes = g_paged.evict_workspace_bytes(&f);
  at::Tensor ws = at::empty({(int64_t)(f.workspace_bytes > 4 ? f.workspace_bytes : 4)}, plain(*t[0]).dtype(at::kByte));
  f.workspace = ptr(ws);
  f.stream = stream_of(*t[0]);
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = g_paged.evict(&f);
  Py_END_ALLOW_THREADS
  if (rc != 0) return refused(rc);
  return THPVariable_Wrap(std::move(lens));
}

}  // namespace
