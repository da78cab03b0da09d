// Host side of the plain calls of a decode step's operators (dan_amd/paged.py,
// dan_amd/readout.py): a CPython module that reads torch tensors and fills the argument
// structures of include/dan_paged.h and include/dan_readout.h in C++.
//
// A decode step's kernels take a few microseconds, about as much as Python needs to look its
// tensors over. Each function here takes the arguments of the Python function of its name,
// and makes the call if everything about it is plain: tensors of the current device, of the
// types and layouts that the kernels read in place, with no gradient or tangent to refuse.
// Otherwise it returns None, having done nothing, and the Python function goes on: it copies
// what lies unaligned, guards another device, and raises what is to be raised. Host time of a
// call, Python alone / through here, us: append 12.3 / 5.8, attend in one launch 10.0 / 5.1,
// log probabilities 14.7 / 9.8, with their gradient 98 / 62 (of which torch's engine takes 39 for
// any gradient; in C++ the backward needs no hand-over of the interpreter's lock to its thread).
#include "calls.h"
#include "dan_paged.h"
#include "dan_readout.h"

namespace {

// The library's entry points (bind).
struct Library {
  int (*append)(const DanPagedAppendArgs *, void *);
  int (*attn)(const DanPagedAttnArgs *, void *);
  int64_t (*attn_bytes)(int32_t, int32_t, int32_t, int32_t, int32_t, int32_t);
  int (*logprobs)(const DanLogprobsArgs *, void *);
  int (*grad)(const DanLogprobsGradArgs *, void *);
  int64_t (*logprobs_bytes)(int32_t, int32_t, int32_t, int32_t);
  const char *(*last_error)(void);
} lib;

// The cache, table and scales of both calls.
bool cache_ok(const Tensor &kc, const Tensor &vc, const Tensor &ks, const Tensor &vs, const Tensor &table, at::ScalarType dtype, int index) {
  const auto kind = kc.scalar_type();
  if (kc.dim() != 4 || kc.sizes() != vc.sizes() || kind != vc.scalar_type() || (kind != dtype && kind != at::kFloat8_e4m3fn)) return false;
  if (!plain(kc, index) || !plain(vc, index) || !rows_ok(kc) || !rows_ok(vc)) return false;
  if (table.dim() != 2 || table.scalar_type() != at::kInt || !plain(table, index) || (table.size(1) > 1 && table.stride(1) != 1)) return false;
  for (int i = 0; i < 4; ++i)
    if (!fits(kc.size(i))) return false;
  if (!fits(table.size(0)) || !fits(table.size(1))) return false;
  if (kind != at::kFloat8_e4m3fn) return !ks.defined() && !vs.defined();
  for (const Tensor *t : {&ks, &vs})
    if (!t->defined() || t->numel() != 1 || t->scalar_type() != at::kFloat || !plain(*t, index)) return false;
  return true;
}

// append(q, k, v, cos, sin, k_cache, v_cache, table, places, seqs, rope_rows, q_norm_weight, k_norm_weight, eps, norm, k_scale, v_scale):
// norm a DanFrontNorm; q not None. q [H, N, D], or None.
PyObject *append(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, k, v, cos, sin, kc, vc, table, places, seqs, rope, qw, kw, ks, vs;
  Tensor *to[] = {&q, &k, &v, &cos, &sin, &kc, &vc, &table, &places, &seqs, &rope, &qw, &kw, nullptr, nullptr, &ks, &vs};
  if (nargs != 17) Py_RETURN_NONE;
  for (int i = 0; i < 17; ++i)
    if (to[i] && !tensor_of(args[i], *to[i])) Py_RETURN_NONE;
  if (!PyFloat_Check(args[13]) || !PyLong_Check(args[14])) Py_RETURN_NONE;
  if (!q.defined() || !k.defined() || !v.defined() || !kc.defined() || !vc.defined() || !table.defined() || !places.defined() ||
      !k.is_cuda() || k.get_device() != c10::hip::current_device())
    Py_RETURN_NONE;
  const int index = k.get_device();
  const auto dtype = k.scalar_type();
  const int64_t norm = PyLong_AsLong(args[14]);
  if (norm < DAN_FRONT_NORM_NONE || norm > DAN_FRONT_NORM_RMS_ZERO_CENTERED) Py_RETURN_NONE;
  if (!is16(dtype) || k.dim() != 3 || q.dim() != 3 || v.sizes() != k.sizes() || q.size(0) != k.size(0) || q.size(2) != k.size(2) ||
      q.scalar_type() != dtype || v.scalar_type() != dtype || grads_of({&q, &k, &v, &kc, &vc, &cos, &sin, &ks, &vs}))
    Py_RETURN_NONE;
  const int64_t n = k.size(0), h = q.size(1), hkv = k.size(1), d = k.size(2);
  if (!fits(n) || !fits(h) || !fits(hkv) || n == 0 || !cache_ok(kc, vc, ks, vs, table, dtype, index) || kc.size(1) != hkv || kc.size(3) != d)
    Py_RETURN_NONE;
  for (const Tensor *t : {&q, &k, &v})
    if (!plain(*t, index) || !rows_ok(*t)) Py_RETURN_NONE;
  for (const Tensor *t : {&kc, &vc})
    for (int i = 0; i < 3; ++i)
      if (t->stride(i) == 0) Py_RETURN_NONE;
  if (!index_ok(places, n, index) || (seqs.defined() ? !index_ok(seqs, n, index) : table.size(0) < n) || (rope.defined() && !index_ok(rope, n, index)))
    Py_RETURN_NONE;
  DanPagedAppendArgs a = {};
  if (cos.defined()) {
    if (!sin.defined() || cos.dim() != 2 || sin.sizes() != cos.sizes() || sin.strides() != cos.strides() || (!rope.defined() && cos.size(0) != n) ||
        (cos.scalar_type() != dtype && cos.scalar_type() != at::kFloat) || sin.scalar_type() != cos.scalar_type() || !plain(cos, index) ||
        !plain(sin, index) || !rows_ok(cos) || !rows_ok(sin) || cos.size(1) == 0 || cos.stride(0) < cos.size(1) || !fits(cos.size(0)) || !fits(cos.size(1)))
      Py_RETURN_NONE;
    a.rotary_dim = (int32_t)cos.size(1);
    a.num_rope_rows = (int32_t)cos.size(0);
    a.cs_stride_tok = cos.stride(0);
  } else if (sin.defined()) {
    Py_RETURN_NONE;
  }
  if (norm != DAN_FRONT_NORM_NONE) {
    if (grads_of({&qw, &kw})) Py_RETURN_NONE;
    for (const Tensor *t : {&qw, &kw})
      if (!t->defined() || t->dim() != 1 || t->size(0) != d || t->scalar_type() != dtype || !plain(*t, index) || !rows_ok(*t)) Py_RETURN_NONE;
    a.q_norm_weight = at_of(qw);
    a.k_norm_weight = at_of(kw);
  }
  const Tensor out = at::empty_strided({h, n, d}, {d, h * d, 1}, q.options().requires_grad(false));
  a.abi_version = DAN_PAGED_ABI_VERSION;
  a.dtype = code_of(dtype);
  a.cache_dtype = code_of(kc.scalar_type());
  a.table_dtype = cos.defined() ? code_of(cos.scalar_type()) : a.dtype;
  a.num_tokens = (int32_t)n;
  a.num_heads = (int32_t)h;
  a.num_kv_heads = (int32_t)hkv;
  a.head_dim = (int32_t)d;
  a.norm = (int32_t)norm;
  a.page_size = (int32_t)kc.size(2);
  a.num_pages = (int32_t)kc.size(0);
  a.table_width = (int32_t)table.size(1);
  a.num_seqs = (int32_t)table.size(0);
  a.eps = (float)PyFloat_AS_DOUBLE(args[13]);
  a.q = at_of(q); a.q_stride_tok = q.stride(0); a.q_stride_head = q.stride(1);
  a.k = at_of(k); a.k_stride_tok = k.stride(0); a.k_stride_head = k.stride(1);
  a.v = at_of(v); a.v_stride_tok = v.stride(0); a.v_stride_head = v.stride(1);
  a.cos = at_of(cos); a.sin = at_of(sin);
  a.q_out = at_of(out); a.qo_stride_tok = h * d; a.qo_stride_head = d;
  a.k_cache = kc.mutable_data_ptr(); a.kc_stride_page = kc.stride(0); a.kc_stride_head = kc.stride(1); a.kc_stride_tok = kc.stride(2);
  a.v_cache = vc.mutable_data_ptr(); a.vc_stride_page = vc.stride(0); a.vc_stride_head = vc.stride(1); a.vc_stride_tok = vc.stride(2);
  a.k_scale = static_cast<const float *>(at_of(ks));
  a.v_scale = static_cast<const float *>(at_of(vs));
  a.table = static_cast<const int32_t *>(at_of(table)); a.table_stride = table.stride(0);
  a.places = static_cast<const int32_t *>(at_of(places));
  a.seqs = static_cast<const int32_t *>(at_of(seqs));
  a.rope_rows = static_cast<const int32_t *>(at_of(rope));
  check(lib.append(&a, c10::hip::getCurrentHIPStream(index).stream()), "dan_paged_append", lib.last_error);
  for (const Tensor *t : {&kc, &vc})  // a backward that has saved a cache must not take the new rows for the old
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// attend(q, k_cache, v_cache, table, lens, scale, k_scale, v_scale, max_len, return_lse): scale None or a float,
// max_len None or an int. out [H, B, D], with return_lse (out, lse [H, B]), or None.
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, kc, vc, table, lens, ks, vs;
  Tensor *to[] = {&q, &kc, &vc, &table, &lens, nullptr, &ks, &vs};
  if (nargs != 10) Py_RETURN_NONE;
  for (int i = 0; i < 8; ++i)
    if (to[i] && !tensor_of(args[i], *to[i])) Py_RETURN_NONE;
  if (!q.defined() || !kc.defined() || !vc.defined() || !table.defined() || !lens.defined() || !q.is_cuda() ||
      q.get_device() != c10::hip::current_device() || (args[5] != Py_None && !PyFloat_Check(args[5])) || (args[8] != Py_None && !PyLong_Check(args[8])))
    Py_RETURN_NONE;
  const int index = q.get_device();
  const auto dtype = q.scalar_type();
  if (!is16(dtype) || q.dim() != 3 || !plain(q, index) || !rows_ok(q) || grads_of({&q, &kc, &vc, &ks, &vs}) || !cache_ok(kc, vc, ks, vs, table, dtype, index))
    Py_RETURN_NONE;
  const int64_t h = q.size(0), b = q.size(1), d = q.size(2), hkv = kc.size(1), page = kc.size(2), holds = table.size(1) * page;
  int overflow = 0;
  const int64_t most = args[8] == Py_None ? holds : PyLong_AsLongLongAndOverflow(args[8], &overflow);
  const double scale = args[5] == Py_None ? 1.0 / std::sqrt((double)d) : PyFloat_AS_DOUBLE(args[5]);
  if (!fits(h) || !fits(b) || b == 0 || kc.size(3) != d || hkv == 0 || h == 0 || h % hkv || table.size(0) != b || !index_ok(lens, b, index) ||
      overflow || most < 0 || most > holds || !fits(most) || !(scale > 0) || !std::isfinite(scale))
    Py_RETURN_NONE;
  const int want = PyObject_IsTrue(args[9]);
  if (want < 0) return nullptr;
  const int kind = code_of(kc.scalar_type());
  const Tensor out = at::empty_strided({h, b, d}, {d, h * d, 1}, q.options().requires_grad(false));
  Tensor lse, ws;
  if (want) lse = at::empty_strided({h, b}, {1, h}, q.options().dtype(at::kFloat).requires_grad(false));
  const int64_t need = lib.attn_bytes(kind, (int32_t)b, (int32_t)h, (int32_t)hkv, (int32_t)d, (int32_t)most);
  if (need > 0) ws = at::empty({need}, q.options().dtype(at::kByte).requires_grad(false));
  DanPagedAttnArgs a = {};
  a.abi_version = DAN_PAGED_ABI_VERSION;
  a.dtype = code_of(dtype);
  a.cache_dtype = kind;
  a.num_seqs = (int32_t)b;
  a.num_heads = (int32_t)h;
  a.num_kv_heads = (int32_t)hkv;
  a.head_dim = (int32_t)d;
  a.page_size = (int32_t)page;
  a.num_pages = (int32_t)kc.size(0);
  a.table_width = (int32_t)table.size(1);
  a.max_len = (int32_t)most;
  a.scale = (float)scale;
  a.q = at_of(q); a.q_stride_seq = q.stride(1); a.q_stride_head = q.stride(0);
  a.out = at_of(out); a.o_stride_seq = h * d; a.o_stride_head = d;
  a.lse = static_cast<float *>(at_of(lse));
  a.k_cache = at_of(kc); a.kc_stride_page = kc.stride(0); a.kc_stride_head = kc.stride(1); a.kc_stride_tok = kc.stride(2);
  a.v_cache = at_of(vc); a.vc_stride_page = vc.stride(0); a.vc_stride_head = vc.stride(1); a.vc_stride_tok = vc.stride(2);
  a.k_scale = static_cast<const float *>(at_of(ks));
  a.v_scale = static_cast<const float *>(at_of(vs));
  a.table = static_cast<const int32_t *>(at_of(table)); a.table_stride = table.stride(0);
  a.lens = static_cast<const int32_t *>(at_of(lens));
  a.workspace = at_of(ws); a.workspace_bytes = need > 0 ? need : 0;
  check(lib.attn(&a, c10::hip::getCurrentHIPStream(index).stream()), "dan_paged_attn", lib.last_error);
  if (!want) return THPVariable_Wrap(out);
  THPObjectPtr x(THPVariable_Wrap(out)), y(THPVariable_Wrap(lse));
  return x && y ? PyTuple_Pack(2, x.get(), y.get()) : nullptr;
  END_HANDLE_TH_ERRORS
}

// What forward gives: undefined where it was not asked for. rest: what rounding took from lse.
struct Outputs {
  Tensor logprobs, lse, rest, entropy, top_logprobs, top_ids;
};

Outputs logprobs_forward(const Tensor &x, const Tensor &tokens, int64_t top, bool entropy, bool rest) {
  const int64_t n = x.size(0), vocab = x.size(1);
  const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
  Outputs o;
  o.logprobs = at::empty(tokens.sizes(), f32);
  o.lse = at::empty({n}, f32);
  if (rest) o.rest = at::empty({n}, f32);
  if (entropy) o.entropy = at::empty({n}, f32);
  if (top) {
    o.top_logprobs = at::empty({n, top}, f32);
    o.top_ids = at::empty({n, top}, f32.dtype(at::kLong));
  }
  const int code = code_of(x.scalar_type());
  const int64_t need = lib.logprobs_bytes(code, (int32_t)n, (int32_t)vocab, (int32_t)top);
  const Tensor ws = at::empty({need}, f32.dtype(at::kByte));
  DanLogprobsArgs a = {};
  a.abi_version = DAN_READOUT_ABI_VERSION;
  a.dtype = code;
  a.rows = (int32_t)n;
  a.vocab = (int32_t)vocab;
  a.labels = tokens.dim() == 2 ? (int32_t)tokens.size(1) : 1;
  a.top = (int32_t)top;
  a.logits = at_of(x); a.logits_stride = x.stride(0);
  a.tokens = static_cast<const int64_t *>(at_of(tokens)); a.tokens_stride = tokens.stride(0);
  a.logprobs = static_cast<float *>(at_of(o.logprobs));
  a.logsumexp = static_cast<float *>(at_of(o.lse));
  a.entropy = static_cast<float *>(at_of(o.entropy));
  a.top_logprobs = static_cast<float *>(at_of(o.top_logprobs));
  a.top_ids = static_cast<int64_t *>(at_of(o.top_ids));
  a.workspace = at_of(ws); a.workspace_bytes = need;
  a.logsumexp_rest = static_cast<float *>(at_of(o.rest));
  check(lib.logprobs(&a, c10::hip::getCurrentHIPStream(x.get_device()).stream()), "dan_logprobs_fwd", lib.last_error);
  return o;
}

// check_capture(device index, name), for a backward that runs in Python
PyObject *py_check_capture(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  if (nargs != 2) return PyErr_Format(PyExc_TypeError, "check_capture takes a device index and a name");
  const long index = PyLong_AsLong(args[0]);
  if (index == -1 && PyErr_Occurred()) return nullptr;
  const char *name = PyUnicode_AsUTF8(args[1]);
  if (!name) return nullptr;
  check_capture((int)index, name);
  Py_RETURN_NONE;
  END_HANDLE_TH_ERRORS
}

struct Logprobs : torch::autograd::Function<Logprobs> {
  static variable_list forward(torch::autograd::AutogradContext *ctx, const Tensor &x, const Tensor &tokens, int64_t top, bool entropy) {
    const Outputs o = logprobs_forward(x, tokens, top, entropy, true);
    ctx->save_for_backward({x, tokens, o.lse, o.entropy, o.top_ids, o.rest});
    ctx->saved_data["top"] = top;
    ctx->saved_data["entropy"] = entropy;
    ctx->set_materialize_grads(false);
    variable_list out = {o.logprobs, o.lse};
    if (entropy) out.push_back(o.entropy);
    if (top) {
      out.push_back(o.top_logprobs);
      out.push_back(o.top_ids);
      ctx->mark_non_differentiable({o.top_ids});
    }
    return out;
  }
  static variable_list backward(torch::autograd::AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &tokens = saved[1];
    const int64_t top = ctx->saved_data["top"].toInt();
    const bool entropy = ctx->saved_data["entropy"].toBool();
    Tensor g[4];  // of logprobs, logsumexp, entropy, top_logprobs
    bool any = false, again = false;
    for (int i = 0, at = 0; i < 4; ++i) {
      if ((i == 2 && !entropy) || (i == 3 && !top)) continue;
      g[i] = grads[at++];
      any |= g[i].defined();
      again |= g[i].defined() && g[i].requires_grad();
    }
    if (!any) return {Tensor(), Tensor(), Tensor(), Tensor()};
    check_capture(x.get_device());
    again = (again || x.requires_grad()) && at::GradMode::is_enabled();
    Tensor grad;
    {
      at::NoGradGuard guard;
      const int64_t n = x.size(0), vocab = x.size(1);
      grad = at::empty({n, vocab}, x.options().requires_grad(false));
      for (Tensor &t : g)
        if (t.defined()) t = t.detach().contiguous();
      DanLogprobsGradArgs a = {};
      a.abi_version = DAN_READOUT_ABI_VERSION;
      a.dtype = code_of(x.scalar_type());
      a.rows = (int32_t)n;
      a.vocab = (int32_t)vocab;
      a.labels = tokens.dim() == 2 ? (int32_t)tokens.size(1) : 1;
      a.top = (int32_t)top;
      a.logits = at_of(x); a.logits_stride = x.stride(0);
      a.tokens = static_cast<const int64_t *>(at_of(tokens)); a.tokens_stride = tokens.stride(0);
      a.logsumexp = static_cast<const float *>(at_of(saved[2]));
      a.entropy = static_cast<const float *>(at_of(saved[3]));
      a.top_ids = static_cast<const int64_t *>(at_of(saved[4]));
      a.g_logprobs = static_cast<const float *>(at_of(g[0]));
      a.g_logsumexp = static_cast<const float *>(at_of(g[1]));
      a.g_entropy = static_cast<const float *>(at_of(g[2]));
      a.g_top = static_cast<const float *>(at_of(g[3]));
      a.grad = at_of(grad); a.grad_stride = vocab;
      a.logsumexp_rest = static_cast<const float *>(at_of(saved[5]));
      // (the engine has made the gradients' device the thread's)
      check(lib.grad(&a, c10::hip::getCurrentHIPStream(x.get_device()).stream()), "dan_logprobs_bwd", lib.last_error);
    }
    return {differentiable_once(grad, again, "token_logprobs is differentiable once"), Tensor(), Tensor(), Tensor()};
  }
};

// logprobs(logits, tokens, top, entropy): the five outputs, None where not asked for; or None.
PyObject *logprobs(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, tokens;
  if (nargs != 4 || !tensor_of(args[0], x) || !tensor_of(args[1], tokens) || !x.defined() || !tokens.defined() || !PyLong_Check(args[2])) Py_RETURN_NONE;
  if (!x.is_cuda() || x.get_device() != c10::hip::current_device()) Py_RETURN_NONE;
  const int index = x.get_device();
  const auto dtype = x.scalar_type();
  if (x.dim() != 2 || !(is16(dtype) || dtype == at::kFloat) || !plain(x, index) || !plain(tokens, index) || tokens.scalar_type() != at::kLong ||
      tokens.dim() < 1 || tokens.dim() > 2)
    Py_RETURN_NONE;
  const int64_t n = x.size(0), vocab = x.size(1);
  int overflow = 0;
  const int64_t top = PyLong_AsLongLongAndOverflow(args[2], &overflow);
  if (n == 0 || vocab == 0 || !fits(n) || !fits(vocab) || x.stride(1) != 1 || tokens.size(0) != n ||
      (tokens.dim() == 2 && (!fits(tokens.size(1)) || tokens.stride(1) != 1)) || overflow || top < 0 || top > DAN_READOUT_MAX_TOP || top > vocab ||
      (top && vocab > DAN_READOUT_MAX_TOP_VOCAB))
    Py_RETURN_NONE;
  const int entropy = PyObject_IsTrue(args[3]);
  if (entropy < 0) return nullptr;
  Outputs o;
  if (grads_of({&x})) {
    const variable_list out = Logprobs::apply(x, tokens, top, entropy);
    o.logprobs = out[0];
    o.lse = out[1];
    if (entropy) o.entropy = out[2];
    if (top) {
      o.top_logprobs = out[2 + entropy];
      o.top_ids = out[3 + entropy];
    }
  } else {
    o = logprobs_forward(x, tokens, top, entropy, false);
  }
  THPObjectPtr tuple(PyTuple_New(5));
  if (!tuple) return nullptr;
  const Tensor *out[] = {&o.logprobs, &o.lse, &o.entropy, &o.top_logprobs, &o.top_ids};
  for (int i = 0; i < 5; ++i) {
    PyObject *t = out[i]->defined() ? THPVariable_Wrap(*out[i]) : Py_NewRef(Py_None);
    if (!t) return nullptr;
    PyTuple_SET_ITEM(tuple.get(), i, t);
  }
  return tuple.release();
  END_HANDLE_TH_ERRORS
}

// bind(addresses of dan_paged_append, dan_paged_attn, dan_paged_attn_workspace_size, dan_logprobs_fwd, dan_logprobs_bwd,
// dan_logprobs_workspace_size, dan_tree_attn_last_error)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  void *at[7];
  if (nargs != 7) return PyErr_Format(PyExc_TypeError, "bind takes 7 addresses");
  for (int i = 0; i < 7; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is NULL", i);
  }
  lib.append = reinterpret_cast<decltype(lib.append)>(at[0]);
  lib.attn = reinterpret_cast<decltype(lib.attn)>(at[1]);
  lib.attn_bytes = reinterpret_cast<decltype(lib.attn_bytes)>(at[2]);
  lib.logprobs = reinterpret_cast<decltype(lib.logprobs)>(at[3]);
  lib.grad = reinterpret_cast<decltype(lib.grad)>(at[4]);
  lib.logprobs_bytes = reinterpret_cast<decltype(lib.logprobs_bytes)>(at[5]);
  lib.last_error = reinterpret_cast<decltype(lib.last_error)>(at[6]);
  Py_RETURN_NONE;
}

#define DAN_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {DAN_METHOD(append), DAN_METHOD(attend), DAN_METHOD(logprobs), DAN_METHOD(bind),
                         {"check_capture", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(py_check_capture)), METH_FASTCALL, nullptr}, {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode_calls(void) { return PyModule_Create(&module); }
