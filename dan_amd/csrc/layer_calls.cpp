// Host side of the plain calls of what adapters are trained and served with (dan_amd/norm.py,
// dan_amd/adapters.py, attend_train of dan_amd/attention.py): a CPython module that reads torch tensors
// and fills the argument structures of include/dan_norm.h, dan_adapt.h and dan_tree_grad.h in C++, as
// decode_calls.cpp does for a decode step.
//
// add_norm and adapt take the arguments of the Python functions of their names, make the call if
// everything about it is plain, with its autograd node where a gradient is wanted, and return None
// otherwise, having done nothing: the Python function goes on. attend is called by attend_train with what
// it has prepared for the batch. Host time of a
// pass, Python alone / through here, us: adapt 17.4 / 8.7, add_norm 13.4 / 6.7, add_norm with its gradient 102 / 70,
// attend_train with its gradient 174 / 85 (torch's engine takes about 39 of any gradient).
#include "calls.h"
#include "dan_adapt.h"
#include "dan_fp8.h"
#include "dan_norm.h"
#include "dan_tree_grad.h"

namespace {

using torch::autograd::AutogradContext;

struct Library {
  int (*norm)(const DanNormArgs *, void *);
  int (*norm_grad)(const DanNormGradArgs *, void *);
  int64_t (*norm_grad_bytes)(int32_t, int32_t);
  int (*adapt)(const DanAdaptArgs *, void *);
  int (*adapt_grad)(const DanAdaptGradArgs *, void *);
  int64_t (*adapt_bytes)(int32_t, int32_t, int32_t, int32_t);
  int64_t (*adapt_grad_bytes)(int32_t, int32_t, int32_t, int32_t, int32_t);
  int (*attn_lse)(const DanTreeAttnArgs *, float *, void *);
  int (*attn_grad)(const DanTreeGradArgs *, void *);
  int64_t (*fp8_tiled_bytes)(int32_t, int32_t);
  const char *(*last_error)(void);
} lib;

void *stream_of(const Tensor &t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
Tensor bytes(int64_t n, const Tensor &like) { return at::empty({n}, like.options().dtype(at::kByte).requires_grad(false)); }
Tensor rows_like(const Tensor &t, int64_t n, int64_t k) { return at::empty({n, k}, t.options().requires_grad(false)); }
// A gradient as the kernels read it.
Tensor readable(const Tensor &t) { return rows_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous); }
// A tensor that may be missing, as an argument of an autograd function (whose edges, and needs_input_grad, count the ones given).
using Maybe = std::optional<Tensor>;
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

bool dense_ok(const Tensor &t) { return t.is_contiguous() && aligned(t.const_data_ptr()); }

// ---------------------------------------------------------------- add_norm
struct NormOut {
  Tensor out, stream, codes, scale, rstd;
};
struct NormForm {
  int64_t norm, layout;  // layout: DanFp8Layout, or -1 without codes
  double eps;
  bool out;
};
NormOut norm_forward(const Tensor &x, const Tensor &residual, const Tensor &weight, const NormForm &f, bool rstd) {
  const int64_t n = x.size(0), k = x.size(1);
  NormOut o;
  DanNormArgs a = {};
  if (residual.defined()) {
    o.stream = rows_like(x, n, k);
    a.residual = at_of(residual); a.residual_stride = residual.stride(0);
    a.stream = at_of(o.stream); a.stream_stride = k;
  }
  if (f.out) {
    o.out = rows_like(x, n, k);
    a.out = at_of(o.out); a.out_stride = k;
  }
  const auto f32 = x.options().dtype(at::kFloat).requires_grad(false);
  if (f.layout >= 0) {
    o.scale = at::empty({n, 1}, f32);
    o.codes = f.layout == DAN_FP8_LAYOUT_ROWS ? at::empty({n, k}, f32.dtype(at::kFloat8_e4m3fn)) : bytes(lib.fp8_tiled_bytes((int32_t)n, (int32_t)k), x);
    a.codes = at_of(o.codes);
    a.scale = static_cast<float *>(at_of(o.scale));
    a.layout = (int32_t)f.layout;
  }
  if (rstd) {
    o.rstd = at::empty({n}, f32);
    a.rstd = static_cast<float *>(at_of(o.rstd));
  }
  a.abi_version = DAN_NORM_ABI_VERSION;
  a.dtype = code_of(x.scalar_type());
  a.rows = (int32_t)n; a.cols = (int32_t)k;
  a.norm = (int32_t)f.norm; a.eps = (float)f.eps;
  a.x = at_of(x); a.x_stride = x.stride(0);
  a.weight = at_of(weight);
  check(lib.norm(&a, stream_of(x)), "dan_add_norm", lib.last_error);
  return o;
}

struct AddNorm : torch::autograd::Function<AddNorm> {
  static variable_list forward(AutogradContext *ctx, const Tensor &x, const Maybe &other, const Tensor &weight, double eps, int64_t norm) {
    const Tensor residual = other.value_or(Tensor());
    const NormOut o = norm_forward(x, residual, weight, {norm, -1, eps, true}, true);
    ctx->save_for_backward({residual.defined() ? o.stream : x, weight, o.rstd});
    ctx->saved_data["norm"] = norm;
    ctx->set_materialize_grads(false);
    if (residual.defined()) return {o.out, o.stream};
    return {o.out};
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &s = saved[0], &weight = saved[1];
    const bool two = grads.size() > 1;
    const Tensor g = grads[0], gs = two ? grads[1] : Tensor();
    const bool need_x = ctx->needs_input_grad(0), need_r = two && ctx->needs_input_grad(1), need_w = ctx->needs_input_grad(two ? 2 : 1);
    bool again = at::GradMode::is_enabled() && (s.requires_grad() || weight.requires_grad());
    for (const Tensor &t : grads) again |= at::GradMode::is_enabled() && t.defined() && t.requires_grad();
    Tensor ds, dw;
    if (!g.defined()) {
      ds = gs;  // the sum alone was used
      again = false;
    } else {
      check_capture(s.get_device(), "add_norm");
      at::NoGradGuard guard;
      const int64_t n = s.size(0), k = s.size(1);
      const Tensor gr = readable(g.detach()), gsr = gs.defined() ? readable(gs.detach()) : Tensor();
      ds = rows_like(s, n, k);
      Tensor ws;
      DanNormGradArgs a = {};
      if (need_w) {
        dw = at::empty({k}, s.options().requires_grad(false));
        a.workspace_bytes = lib.norm_grad_bytes((int32_t)n, (int32_t)k);
        ws = bytes(a.workspace_bytes, s);
        a.workspace = at_of(ws);
        a.dw = at_of(dw);
      }
      a.abi_version = DAN_NORM_ABI_VERSION;
      a.dtype = code_of(s.scalar_type());
      a.rows = (int32_t)n; a.cols = (int32_t)k;
      a.norm = (int32_t)ctx->saved_data["norm"].toInt();
      a.s = at_of(s); a.s_stride = s.stride(0);
      a.weight = at_of(weight);
      a.rstd = static_cast<const float *>(at_of(saved[2]));
      a.g = at_of(gr); a.g_stride = gr.stride(0);
      if (gsr.defined()) {
        a.g_stream = at_of(gsr); a.g_stream_stride = gsr.stride(0);
      }
      a.ds = at_of(ds); a.ds_stride = k;
      check(lib.norm_grad(&a, stream_of(s)), "dan_add_norm_grad", lib.last_error);
    }
    const char *message = "add_norm is differentiable once";
    ds = differentiable_once(ds, again, message);
    return {need_x ? ds : Tensor(), need_r ? ds : Tensor(), differentiable_once(dw, again, message), Tensor(), Tensor()};
  }
};

PyObject *wrap(const Tensor &t) { return t.defined() ? THPVariable_Wrap(t) : Py_NewRef(Py_None); }
PyObject *tuple_of(std::initializer_list<const Tensor *> ts) {
  THPObjectPtr tuple(PyTuple_New((Py_ssize_t)ts.size()));
  if (!tuple) return nullptr;
  Py_ssize_t i = 0;
  for (const Tensor *t : ts) {
    PyObject *o = wrap(*t);
    if (!o) return nullptr;
    PyTuple_SET_ITEM(tuple.get(), i++, o);
  }
  return tuple.release();
}

// add_norm(x, residual, weight, eps, norm, layout, out): norm a DAN_NORM_*, layout a DAN_FP8_LAYOUT_* or -1. (out, stream, codes,
// scale), None where not made (stream: also where it is x itself); or None.
PyObject *add_norm(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor x, residual, weight;
  if (nargs != 7 || !tensor_of(args[0], x) || !tensor_of(args[1], residual) || !tensor_of(args[2], weight) || !x.defined() || !weight.defined() ||
      !PyFloat_Check(args[3]) || !PyLong_Check(args[4]) || !PyLong_Check(args[5]) || !PyBool_Check(args[6]))
    Py_RETURN_NONE;
  if (!x.is_cuda() || x.get_device() != c10::hip::current_device()) Py_RETURN_NONE;
  const int index = x.get_device();
  const NormForm f = {PyLong_AsLong(args[4]), PyLong_AsLong(args[5]), PyFloat_AsDouble(args[3]), args[6] == Py_True};
  if (f.norm < 0 || f.norm > DAN_NORM_ZERO_CENTERED || f.layout > DAN_FP8_LAYOUT_TILED || (f.layout < 0 && !f.out) || !(f.eps >= 0) ||
      !std::isfinite((float)f.eps))
    Py_RETURN_NONE;
  if (x.dim() != 2 || !is16(x.scalar_type()) || !plain(x, index) || !rows_ok(x)) Py_RETURN_NONE;
  const int64_t n = x.size(0), k = x.size(1);
  if (n == 0 || n >= 1 << 24 || (f.layout == DAN_FP8_LAYOUT_TILED && k > 1024 && n > (1 << 24) - 256) || k == 0 || k > DAN_NORM_MAX_COLS || k % (f.layout < 0 ? 8 : 16)) Py_RETURN_NONE;
  if (residual.defined() && (residual.sizes() != x.sizes() || residual.scalar_type() != x.scalar_type() || !plain(residual, index) || !rows_ok(residual)))
    Py_RETURN_NONE;
  if (weight.dim() != 1 || weight.size(0) != k || weight.scalar_type() != x.scalar_type() || !plain(weight, index) || !dense_ok(weight)) Py_RETURN_NONE;
  NormOut o;
  if (grads_of({&x, &residual, &weight})) {
    if (f.layout >= 0) Py_RETURN_NONE;
    const variable_list out = AddNorm::apply(x, maybe(residual), weight, f.eps, f.norm);
    o.out = out[0];
    if (residual.defined()) o.stream = out[1];
  } else {
    o = norm_forward(x, residual, weight, f, false);
  }
  return tuple_of({&o.out, &o.stream, &o.codes, &o.scale});
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- adapt
int64_t ranks_of(int64_t rank) { return rank <= 16 ? 16 : rank <= 32 ? 32 : rank <= 64 ? 64 : 128; }

Tensor adapt_forward(const Tensor &y, const Tensor &x, const Tensor &ad, const Tensor &bd, const Tensor &index, const Tensor &scale, double value, Tensor *down) {
  const int64_t n = x.size(0), n_in = x.size(1), n_out = y.size(1), rank = ad.size(1);
  const Tensor out = rows_like(x, n, n_out);
  DanAdaptArgs a = {};
  if (down) {
    *down = at::empty({n, ranks_of(rank)}, x.options().dtype(at::kFloat).requires_grad(false));
    a.down = static_cast<float *>(at_of(*down));
  }
  a.workspace_bytes = lib.adapt_bytes((int32_t)n, (int32_t)n_in, (int32_t)rank, (int32_t)ad.size(0));
  const Tensor ws = bytes(a.workspace_bytes, x);
  a.workspace = at_of(ws);
  a.abi_version = DAN_ADAPT_ABI_VERSION;
  a.dtype = code_of(x.scalar_type());
  a.rows = (int32_t)n; a.n_in = (int32_t)n_in; a.n_out = (int32_t)n_out; a.rank = (int32_t)rank; a.adapters = (int32_t)ad.size(0);
  a.x = at_of(x); a.x_stride = x.stride(0);
  a.y = at_of(y); a.y_stride = y.stride(0);
  a.a = at_of(ad); a.b = at_of(bd);
  a.index = static_cast<const int32_t *>(at_of(index));
  a.scale = static_cast<const float *>(at_of(scale)); a.scale_value = (float)value;
  a.out = at_of(out); a.out_stride = n_out;
  check(lib.adapt(&a, stream_of(x)), "dan_adapt", lib.last_error);
  return out;
}

struct Adapt : torch::autograd::Function<Adapt> {
  static Tensor forward(AutogradContext *ctx, const Tensor &y, const Tensor &x, const Tensor &a, const Tensor &b, const Maybe &rows, const Maybe &factors, double value) {
    const Tensor index = rows.value_or(Tensor()), scale = factors.value_or(Tensor());
    Tensor down;
    const Tensor out = adapt_forward(y, x, a, b, index, scale, value, &down);
    ctx->save_for_backward({x, a, b, down, index, scale});
    ctx->saved_data["value"] = value;
    ctx->set_materialize_grads(false);
    return out;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    const Tensor g = grads[0];
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &ad = saved[1], &bd = saved[2], &down = saved[3], &index = saved[4], &scale = saved[5];
    const bool need_y = ctx->needs_input_grad(0), need_x = ctx->needs_input_grad(1), need_a = ctx->needs_input_grad(2), need_b = ctx->needs_input_grad(3);
    if (!g.defined()) return variable_list(7);
    Tensor dx, da, db;
    bool again = false;
    if (need_x || need_a || need_b) {
      check_capture(x.get_device(), "adapt");
      again = at::GradMode::is_enabled() && (g.requires_grad() || x.requires_grad() || ad.requires_grad() || bd.requires_grad());
      at::NoGradGuard guard;
      const int64_t n = x.size(0), n_in = x.size(1), n_out = bd.size(1), rank = ad.size(1), count = ad.size(0);
      const Tensor gr = readable(g.detach());
      if (need_x) dx = rows_like(x, n, n_in);
      if (need_a) da = at::empty(ad.sizes(), ad.options().requires_grad(false));
      if (need_b) db = at::empty(bd.sizes(), bd.options().requires_grad(false));
      DanAdaptGradArgs a = {};
      a.workspace_bytes = lib.adapt_grad_bytes((int32_t)n, (int32_t)n_in, (int32_t)n_out, (int32_t)rank, (int32_t)count);
      const Tensor ws = bytes(a.workspace_bytes, x);
      a.workspace = at_of(ws);
      a.abi_version = DAN_ADAPT_ABI_VERSION;
      a.dtype = code_of(x.scalar_type());
      a.rows = (int32_t)n; a.n_in = (int32_t)n_in; a.n_out = (int32_t)n_out; a.rank = (int32_t)rank; a.adapters = (int32_t)count;
      a.x = at_of(x); a.x_stride = x.stride(0);
      a.g = at_of(gr); a.g_stride = gr.stride(0);
      a.a = at_of(ad); a.b = at_of(bd);
      a.index = static_cast<const int32_t *>(at_of(index));
      a.scale = static_cast<const float *>(at_of(scale)); a.scale_value = (float)ctx->saved_data["value"].toDouble();
      a.down = static_cast<const float *>(at_of(down));
      a.dx = at_of(dx); a.dx_stride = n_in;
      a.da = at_of(da); a.db = at_of(db);
      check(lib.adapt_grad(&a, stream_of(x)), "dan_adapt_grad", lib.last_error);
    }
    const char *message = "adapt is differentiable once";
    return {need_y ? g : Tensor(), differentiable_once(dx, again, message), differentiable_once(da, again, message), differentiable_once(db, again, message),
            Tensor(), Tensor(), Tensor()};
  }
};

// adapt(y, x, a, b, index, scale): out; or None.
PyObject *adapt(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor y, x, a, b, index, scale;
  if (nargs != 6 || !tensor_of(args[0], y) || !tensor_of(args[1], x) || !tensor_of(args[2], a) || !tensor_of(args[3], b) || !tensor_of(args[4], index) ||
      !y.defined() || !x.defined() || !a.defined() || !b.defined())
    Py_RETURN_NONE;
  double value = 0;
  if (PyFloat_Check(args[5])) {
    value = PyFloat_AsDouble(args[5]);
    if (!std::isfinite((float)value)) Py_RETURN_NONE;
  } else if (!tensor_of(args[5], scale) || !scale.defined()) {
    Py_RETURN_NONE;
  }
  if (!x.is_cuda() || x.get_device() != c10::hip::current_device()) Py_RETURN_NONE;
  const int dev = x.get_device();
  const auto dtype = x.scalar_type();
  if (!is16(dtype) || x.dim() != 2 || y.dim() != 2 || a.dim() != 3 || b.dim() != 3) Py_RETURN_NONE;
  for (const Tensor *t : {&y, &x, &a, &b})
    if (t->scalar_type() != dtype || !plain(*t, dev)) Py_RETURN_NONE;
  const int64_t n = x.size(0), n_in = x.size(1), n_out = y.size(1), count = a.size(0), rank = a.size(1);
  if (!rows_ok(x) || !rows_ok(y) || !dense_ok(a) || !dense_ok(b) || y.size(0) != n || a.size(2) != n_in || b.size(0) != count || b.size(1) != n_out ||
      b.size(2) != rank || n == 0 || n > 1 << 20 || n_in == 0 || n_out == 0 || n_in % 8 || n_out % 8 || !fits(n_in) || !fits(n_out) || rank == 0 ||
      rank > DAN_ADAPT_MAX_RANK || count == 0 || !fits(count))
    Py_RETURN_NONE;
  if (index.defined() ? !index_ok(index, n, dev) : count != 1) Py_RETURN_NONE;
  if (scale.defined() && (scale.scalar_type() != at::kFloat || scale.dim() != 1 || scale.size(0) != count || !plain(scale, dev) || !scale.is_contiguous() ||
                          (at::GradMode::is_enabled() && scale.requires_grad())))
    Py_RETURN_NONE;
  const Tensor out = grads_of({&y, &x, &a, &b}) ? Adapt::apply(y, x, a, b, maybe(index), maybe(scale), value) : adapt_forward(y, x, a, b, index, scale, value, nullptr);
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---------------------------------------------------------------- tree attention
// What attend_train has prepared for a batch: both argument structures without the call's own tensors, and the sizes
// of their workspaces. `tables`: device tensors that they point to. `pasts`: the prefixes' own.
struct Prepared {
  DanTreeAttnArgs forward;
  DanTreeGradArgs backward;
  int64_t forward_bytes, backward_bytes;
  bool zero;  // some row is in no segment
};

struct TreeAttention : torch::autograd::Function<TreeAttention> {
  static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v, const Prepared *prepared, const variable_list *tables,
                        const variable_list *pasts) {
    const int64_t h = q.size(0), n = q.size(1), d = q.size(2);
    const auto options = q.options().requires_grad(false);
    const Tensor out = prepared->zero ? at::zeros({n, h, d}, options) : at::empty({n, h, d}, options);
    const Tensor lse = at::empty({h, n}, options.dtype(at::kFloat)), ws = bytes(prepared->forward_bytes, q);
    DanTreeAttnArgs a = prepared->forward;
    a.q = at_of(q); a.q_stride_head = q.stride(0); a.q_stride_tok = q.stride(1);
    a.k = at_of(k); a.k_stride_head = k.stride(0); a.k_stride_tok = k.stride(1);
    a.v = at_of(v); a.v_stride_head = v.stride(0); a.v_stride_tok = v.stride(1);
    a.out = at_of(out); a.o_stride_head = d; a.o_stride_tok = h * d;
    a.workspace = at_of(ws); a.workspace_bytes = prepared->forward_bytes;
    check(lib.attn_lse(&a, static_cast<float *>(at_of(lse)), stream_of(q)), "dan_tree_attn_fwd_lse", lib.last_error);
    const Tensor view = out.transpose(0, 1);
    variable_list saved = {q, k, v, view, lse};
    saved.insert(saved.end(), pasts->begin(), pasts->end());  // what the backward pass reads has to be what this one read
    ctx->save_for_backward(std::move(saved));
    ctx->saved_data["tables"] = c10::List<Tensor>(*tables);
    ctx->saved_data["prepared"] = std::string(reinterpret_cast<const char *>(prepared), sizeof *prepared);
    ctx->set_materialize_grads(false);
    return view;
  }
  static variable_list backward(AutogradContext *ctx, variable_list grads) {
    if (!grads[0].defined()) return variable_list(6);
    const variable_list saved = ctx->get_saved_variables();
    const Tensor &q = saved[0], &k = saved[1], &v = saved[2], &out = saved[3], &lse = saved[4];
    check_capture(q.get_device(), "attend_train");
    Prepared prepared;
    memcpy(static_cast<void *>(&prepared), ctx->saved_data["prepared"].toStringRef().data(), sizeof prepared);
    const bool again = at::GradMode::is_enabled() && (grads[0].requires_grad() || q.requires_grad() || k.requires_grad() || v.requires_grad());
    Tensor d[3];
    {
      at::NoGradGuard guard;
      const Tensor g = rows_ok(grads[0]) && grads[0].stride(1) < 1 << 25 ? grads[0].detach() : grads[0].detach().clone(at::MemoryFormat::Contiguous);
      const Tensor *like[] = {&q, &k, &v};
      const auto options = q.options().requires_grad(false);
      for (int i = 0; i < 3; ++i) {
        const int64_t heads = like[i]->size(0), n = like[i]->size(1), dim = like[i]->size(2);
        d[i] = (prepared.zero ? at::zeros({n, heads, dim}, options) : at::empty({n, heads, dim}, options)).transpose(0, 1);
      }
      const Tensor ws = bytes(prepared.backward_bytes, q);
      DanTreeGradArgs a = prepared.backward;
      a.q = at_of(q); a.q_stride_head = q.stride(0); a.q_stride_tok = q.stride(1);
      a.k = at_of(k); a.k_stride_head = k.stride(0); a.k_stride_tok = k.stride(1);
      a.v = at_of(v); a.v_stride_head = v.stride(0); a.v_stride_tok = v.stride(1);
      a.out = at_of(out); a.o_stride_head = out.stride(0); a.o_stride_tok = out.stride(1);
      a.grad = at_of(g); a.g_stride_head = g.stride(0); a.g_stride_tok = g.stride(1);
      a.lse = static_cast<const float *>(at_of(lse));
      a.dq = at_of(d[0]); a.dq_stride_head = d[0].stride(0); a.dq_stride_tok = d[0].stride(1);
      a.dk = at_of(d[1]); a.dk_stride_head = d[1].stride(0); a.dk_stride_tok = d[1].stride(1);
      a.dv = at_of(d[2]); a.dv_stride_head = d[2].stride(0); a.dv_stride_tok = d[2].stride(1);
      a.workspace = at_of(ws); a.workspace_bytes = prepared.backward_bytes;
      check(lib.attn_grad(&a, stream_of(q)), "dan_tree_attn_bwd", lib.last_error);
    }
    for (int i = 0; i < 3; ++i)
      d[i] = ctx->needs_input_grad(i) ? differentiable_once(d[i], again, "attend_train is differentiable once") : Tensor();
    return {d[0], d[1], d[2], Tensor(), Tensor(), Tensor()};
  }
};

bool list_of(PyObject *o, variable_list &to) {
  if (!PyTuple_Check(o)) return false;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(o); ++i) {
    if (!THPVariable_Check(PyTuple_GET_ITEM(o, i))) return false;
    to.push_back(THPVariable_Unpack(PyTuple_GET_ITEM(o, i)));
  }
  return true;
}

// attend(q, k, v, forward, forward workspace bytes, backward, backward workspace bytes, zero, tables, pasts): `forward` and `backward`
// are the argument structures' bytes. The output; or None.
PyObject *attend(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  Tensor q, k, v;
  if (nargs != 10 || !tensor_of(args[0], q) || !tensor_of(args[1], k) || !tensor_of(args[2], v) || !q.defined() || !k.defined() || !v.defined()) Py_RETURN_NONE;
  if (!q.is_cuda() || q.get_device() != c10::hip::current_device() || !is16(q.scalar_type())) Py_RETURN_NONE;
  for (const Tensor *t : {&q, &k, &v})
    if (t->dim() != 3 || t->scalar_type() != q.scalar_type() || !plain(*t, q.get_device()) || !rows_ok(*t) || t->stride(1) >= 1 << 25) Py_RETURN_NONE;
  Prepared prepared;
  if (!PyBytes_Check(args[3]) || PyBytes_GET_SIZE(args[3]) != (Py_ssize_t)sizeof prepared.forward || !PyBytes_Check(args[5]) ||
      PyBytes_GET_SIZE(args[5]) != (Py_ssize_t)sizeof prepared.backward)
    return PyErr_Format(PyExc_TypeError, "attend takes the two argument structures as bytes");
  memset(static_cast<void *>(&prepared), 0, sizeof prepared);
  memcpy(&prepared.forward, PyBytes_AS_STRING(args[3]), sizeof prepared.forward);
  memcpy(&prepared.backward, PyBytes_AS_STRING(args[5]), sizeof prepared.backward);
  prepared.forward_bytes = PyLong_AsLongLong(args[4]);
  prepared.backward_bytes = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  const DanTreeAttnArgs &f = prepared.forward;
  if (q.size(0) != f.num_heads || q.size(1) != f.num_tokens || q.size(2) != f.head_dim || k.size(0) != f.num_kv_heads || k.size(1) != f.num_tokens ||
      k.size(2) != f.head_dim || v.sizes() != k.sizes() || code_of(q.scalar_type()) != f.in_dtype)
    Py_RETURN_NONE;
  prepared.zero = args[7] == Py_True;
  variable_list tables, pasts;
  if (!list_of(args[8], tables) || !list_of(args[9], pasts)) return PyErr_Format(PyExc_TypeError, "attend takes two tuples of tensors");
  return THPVariable_Wrap(TreeAttention::apply(q, k, v, &prepared, &tables, &pasts));
  END_HANDLE_TH_ERRORS
}

// bind(the addresses of Library's functions, in its order)
PyObject *bind(PyObject *, PyObject *const *args, Py_ssize_t nargs) {
  constexpr int kCount = 11;
  void *at[kCount];
  if (nargs != kCount) return PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kCount);
  for (int i = 0; i < kCount; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "address %d is NULL", i);
  }
  static_assert(sizeof lib == sizeof at, "one address each");
  memcpy(static_cast<void *>(&lib), at, sizeof at);
  Py_RETURN_NONE;
}

#define DAN_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {DAN_METHOD(add_norm), DAN_METHOD(adapt), DAN_METHOD(attend), DAN_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_layer_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__layer_calls(void) { return PyModule_Create(&module); }
