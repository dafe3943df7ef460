// Python binding of include/csm_ops.h for torch tensors: looks into the tensors, checks them against each other, allocates outputs and scratch
// memory, and makes one C call on the tensors' device and its current stream.  What needs no tensor is checked by the C entries themselves.  In
// Python the same work (some forty attribute reads, the argument pack, a ctypes call) took 4 us a call, more than most decode-step kernels run.
#include <torch/csrc/autograd/python_variable.h>
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <cmath>
#include <limits>
#include <stdexcept>
#include <string>
#include <vector>
#include "../../../include/csm_ops.h"

namespace {

struct Refused { PyObject* type; std::string text; };   // type nullptr: the Python error is set already
[[noreturn]] void refuse(const std::string& text) { throw Refused{PyExc_ValueError, text}; }
void need(bool ok, const char* text) { if (!ok) refuse(text); }

// The tensors of one call: all on one GPU, with values in their memory, none that asks for a derivative.
struct Call {
  int device = -1;
  c10::OptionalDeviceGuard guard;   // the tensors' device is current from the first of them on, until the call returns
  void* stream() const { return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA((c10::DeviceIndex)device).stream(); }
  const at::Tensor& take(const char* name, PyObject* o) {
    if (!THPVariable_Check(o)) throw Refused{PyExc_TypeError, std::string(name) + " must be a tensor"};
    const at::Tensor& t = THPVariable_Unpack(o);
    if (!t.is_cuda()) {
      if (device < 0) throw Refused{PyExc_RuntimeError, "csm_hf_amd operators need tensors on the GPU (no CPU fallback)"};
      refuse(std::string(name) + " is not on the GPU of the other tensors");
    }
    if (device < 0) {
      device = (int)t.get_device();
      guard.reset_device(t.device());
    }
    if (t.get_device() != device) refuse(std::string(name) + " is on cuda:" + std::to_string(t.get_device()) + ", expected cuda:" + std::to_string(device));
    if (t.requires_grad() && at::GradMode::is_enabled())
      throw Refused{PyExc_RuntimeError, std::string(name) + " requires a gradient: this operator has no backward pass (call it under torch.no_grad())"};
    if (c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(0).defined())
      throw Refused{PyExc_RuntimeError, std::string(name) + " has a forward-mode tangent: this operator has no derivative"};
    if (t.layout() != at::kStrided) refuse(std::string(name) + " must be a dense tensor");
    // wrappers of function transforms (vmap, jvp) have no memory of their own; a lazily negated view holds other values than it stands for
    if (!t.has_storage()) throw Refused{PyExc_RuntimeError, std::string(name) + " is a tensor inside a function transform: this operator cannot be transformed"};
    if (t.is_neg()) refuse(std::string(name) + " is a negated view: pass its resolve_neg()");
    return t;
  }
  const at::Tensor* maybe(const char* name, PyObject* o) { return o == Py_None ? nullptr : &take(name, o); }
};

int32_t i32(const char* name, int64_t v) {
  if (v < std::numeric_limits<int32_t>::min() || v > std::numeric_limits<int32_t>::max()) refuse(std::string(name) + " = " + std::to_string(v) + " is out of range");
  return (int32_t)v;
}
int32_t py_i32(const char* name, PyObject* o) {
  PyObject* n = PyNumber_Index(o);
  if (!n) throw Refused{nullptr, ""};
  int over = 0;
  const int64_t v = PyLong_AsLongLongAndOverflow(n, &over);
  Py_DECREF(n);
  if (over) refuse(std::string(name) + " is out of range");
  return i32(name, v);
}
float py_float(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Refused{nullptr, ""};
  return (float)v;
}
int dtype_of(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? CSM_OPS_F32 : t.scalar_type() == at::kBFloat16 ? CSM_OPS_BF16 : -1; }
int64_t step(const at::Tensor& t, int64_t d, int64_t alone) { return t.size(d) > 1 ? t.stride(d) : alone; }   // a dimension of one: its stride means nothing
const int32_t* ints(const char* name, const at::Tensor& t, int64_t n) {
  if (t.scalar_type() != at::kInt || t.dim() != 1 || t.size(0) != n || !t.is_contiguous()) refuse(std::string(name) + " must be a contiguous int32 tensor of shape (" + std::to_string(n) + ",)");
  return (const int32_t*)t.data_ptr();
}

// what a call wrote: autograd notices when it has saved the tensor for a backward pass (inference tensors have no version to raise)
void written(const at::Tensor& t) { if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); }

void paged(Call& call, csm_ops_paged_t& c, PyObject* k_obj, PyObject* v_obj, PyObject* table_obj, PyObject* lens_obj, PyObject* cu_obj, int64_t rows) {
  const at::Tensor &k = call.take("k_cache", k_obj), &v = call.take("v_cache", v_obj), &table = call.take("page_table", table_obj), &lens = call.take("seq_lens", lens_obj);
  need(k.dim() == 4 && dtype_of(k) >= 0 && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type(),
       "k_cache and v_cache must be float32 or bfloat16 tensors [n_pages, n_kv, page_size, head_dim] of one shape and dtype");
  need((k.stride(3) == 1 && v.stride(3) == 1) || k.size(3) == 1, "the last dimension of k_cache and v_cache must be contiguous");
  c.k = k.data_ptr(); c.v = v.data_ptr(); c.dtype = dtype_of(k);
  c.n_pages = i32("n_pages", k.size(0)); c.n_kv = i32("n_kv", k.size(1)); c.page_size = i32("page_size", k.size(2)); c.head_dim = i32("head_dim", k.size(3));
  c.k_page_stride = step(k, 0, 0); c.k_head_stride = step(k, 1, 0); c.k_slot_stride = step(k, 2, 0);
  c.v_page_stride = step(v, 0, 0); c.v_head_stride = step(v, 1, 0); c.v_slot_stride = step(v, 2, 0);
  need(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1), "page_table must be an int32 tensor [n_seqs, pages] with contiguous rows");
  c.n_seqs = i32("n_seqs", table.size(0)); c.table_width = i32("pages", table.size(1));
  c.page_table = (const int32_t*)table.data_ptr(); c.table_stride = step(table, 0, table.size(1));
  c.seq_lens = ints("seq_lens", lens, c.n_seqs);
  c.rows = i32("rows", rows);
  const at::Tensor* cu = call.maybe("cu_rows", cu_obj);
  c.cu_rows = cu ? ints("cu_rows", *cu, (int64_t)c.n_seqs + 1) : nullptr;
  if (!cu && rows != c.n_seqs) refuse("without cu_rows every sequence has one row: " + std::to_string(rows) + " rows, " + std::to_string(c.n_seqs) + " sequences");
}

// [rows, heads, dim] with contiguous heads
int64_t row_stride(const char* name, const at::Tensor& t, at::IntArrayRef sizes, at::ScalarType type) {
  if (t.scalar_type() != type || t.sizes() != sizes) refuse(std::string(name) + " must be a " + (type == at::kFloat ? "float32" : "bfloat16") + " tensor [" + std::to_string(sizes[0]) + ", " + std::to_string(sizes[1]) + ", " + std::to_string(sizes[2]) + "]");
  if (t.numel() && ((sizes[2] > 1 && t.stride(2) != 1) || (sizes[1] > 1 && t.stride(1) != sizes[2]))) refuse(std::string("the heads of a row of ") + name + " must be contiguous");
  return step(t, 0, sizes[1] * sizes[2]);
}

void done(int rc) {
  if (!rc) return;
  const std::string text = csm_ops_last_error();
  if (rc == CSM_OPS_ERR_CAPACITY) refuse("csm_ops capacity error: " + text);
  throw Refused{PyExc_RuntimeError, "csm_ops error " + std::to_string(rc) + ": " + text};
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& r) {
    if (r.type) PyErr_SetString(r.type, r.text.c_str());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}
PyObject* result(PyObject* given, const at::Tensor& t) {
  if (given == Py_None) return THPVariable_Wrap(t);
  Py_INCREF(given);
  return given;
}
void arguments(Py_ssize_t n, Py_ssize_t want) { if (n != want) throw Refused{PyExc_TypeError, std::to_string(want) + " arguments"}; }

// qkv, cos, sin, k_cache, v_cache, page_table, seq_lens, cu_rows | None, pos_offset, q_out | None
PyObject* rope_append(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    arguments(n, 10);
    Call call;
    csm_ops_rope_append_t a{};
    const at::Tensor &qkv = call.take("qkv", o[0]), &cos = call.take("cos", o[1]), &sin = call.take("sin", o[2]);
    a.x_dtype = dtype_of(qkv);
    need(a.x_dtype >= 0 && qkv.dim() == 2 && (qkv.size(1) <= 1 || qkv.stride(1) == 1), "qkv must be a float32 or bfloat16 tensor [rows, (n_q + 2 n_kv) * head_dim] with contiguous rows");
    paged(call, a.c, o[3], o[4], o[5], o[6], o[7], qkv.size(0));
    const int64_t hd = a.c.head_dim, n_kv = a.c.n_kv, width = qkv.size(1), n_q = hd ? width / hd - 2 * n_kv : 0;
    if (n_q < 1 || width != (n_q + 2 * n_kv) * hd) refuse("qkv rows of " + std::to_string(width) + " elements are not n_q + 2 * " + std::to_string(n_kv) + " heads of " + std::to_string(hd));
    if (cos.scalar_type() != at::kFloat || sin.scalar_type() != at::kFloat || cos.dim() != 2 || cos.size(1) != hd / 2 || sin.sizes() != cos.sizes() || !cos.is_contiguous() || !sin.is_contiguous())
      refuse("cos and sin must be contiguous float32 tensors [positions, " + std::to_string(hd / 2) + "]");
    const int64_t sizes[3] = {qkv.size(0), n_q, hd};
    const at::Tensor* given = call.maybe("q_out", o[9]);
    const at::Tensor q = given ? *given : at::empty(sizes, qkv.options());
    a.q_out_stride = row_stride("q_out", q, sizes, qkv.scalar_type());
    a.qkv = qkv.data_ptr(); a.q_out = q.data_ptr(); a.qkv_stride = step(qkv, 0, width); a.n_q = i32("n_q", n_q);
    a.cos = (const float*)cos.data_ptr(); a.sin = (const float*)sin.data_ptr();
    a.rope_positions = i32("positions", cos.size(0)); a.pos_offset = py_i32("pos_offset", o[8]);
    done(csm_ops_paged_rope_append(&a, call.stream()));
    written(THPVariable_Unpack(o[3])); written(THPVariable_Unpack(o[4])); written(q);
    return result(o[9], q);
  });
}

// q, k_cache, v_cache, page_table, seq_lens, prefix_table | None, prefix_len, cu_rows | None, scale | None, out | None
PyObject* prefix_attention(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    arguments(n, 10);
    Call call;
    csm_ops_attention_t a{};
    const at::Tensor& q = call.take("q", o[0]);
    a.x_dtype = dtype_of(q);
    need(a.x_dtype >= 0 && q.dim() == 3, "q must be a float32 or bfloat16 tensor [rows, n_q, head_dim]");
    paged(call, a.c, o[1], o[2], o[3], o[4], o[7], q.size(0));
    if (q.size(2) != a.c.head_dim) refuse("q has heads of " + std::to_string(q.size(2)) + ", the cache of " + std::to_string(a.c.head_dim));
    const at::Tensor* given = call.maybe("out", o[9]);
    const at::Tensor out = given ? *given : at::empty(q.sizes(), q.options());
    a.q_stride = row_stride("q", q, q.sizes(), q.scalar_type());
    a.out_stride = row_stride("out", out, q.sizes(), q.scalar_type());
    a.q = q.data_ptr(); a.out = out.data_ptr(); a.n_q = i32("n_q", q.size(1));
    if (const at::Tensor* t = call.maybe("prefix_table", o[5])) {
      a.prefix_pages = i32("prefix pages", t->numel());
      a.prefix_table = ints("prefix_table", *t, t->numel());
    }
    a.prefix_len = py_i32("prefix_len", o[6]);
    a.scale = o[8] == Py_None ? (float)(1.0 / std::sqrt((double)q.size(2))) : py_float(o[8]);
    done(csm_ops_paged_attention_workspace(&a, &a.workspace_bytes));
    at::Tensor scratch;
    if (a.workspace_bytes) {
      scratch = at::empty({(int64_t)a.workspace_bytes}, q.options().dtype(at::kByte));
      a.workspace = scratch.data_ptr();
    }
    done(csm_ops_paged_prefix_attention(&a, call.stream()));
    written(out);
    return result(o[9], out);
  });
}

// logits, uniform, temperature, topk, top_p, min_p (numbers or tensors)
PyObject* sample(PyObject*, PyObject* const* o, Py_ssize_t n) {
  return guarded([&] {
    arguments(n, 6);
    Call call;
    csm_ops_sample_t a{};
    const at::Tensor& logits = call.take("logits", o[0]);
    a.x_dtype = dtype_of(logits);
    need(a.x_dtype >= 0 && logits.dim() >= 1, "logits must be a float32 or bfloat16 tensor [..., V]");
    const int64_t V = logits.size(-1), rows = V ? logits.numel() / V : 0;
    need(V > 0, "logits must have entries");
    const auto lead = logits.sizes().slice(0, logits.dim() - 1);
    const at::Tensor rows_of = logits.dim() == 2 && (V <= 1 || logits.stride(1) == 1) ? logits : logits.reshape({rows, V}).contiguous();
    at::Tensor kept[5];   // flattened copies live until the launch is queued
    auto per_row = [&](int i, const char* name, PyObject* obj, at::ScalarType type) -> const void* {
      const at::Tensor& t = call.take(name, obj);
      if (t.scalar_type() != type || t.numel() != rows || (t.dim() > 1 && t.sizes() != lead)) refuse(std::string(name) + " must be a " + (type == at::kInt ? "int32" : "float32") + " tensor with one value per row");
      kept[i] = t.is_contiguous() ? t : t.contiguous();
      return kept[i].data_ptr();
    };
    a.uniform = (const float*)per_row(0, "uniform", o[1], at::kFloat);
    if (THPVariable_Check(o[2])) a.temperatures = (const float*)per_row(1, "temperature", o[2], at::kFloat); else a.temperature = py_float(o[2]);
    if (THPVariable_Check(o[3])) a.topks = (const int32_t*)per_row(2, "topk", o[3], at::kInt); else a.topk = py_i32("topk", o[3]);
    if (THPVariable_Check(o[4])) a.top_ps = (const float*)per_row(3, "top_p", o[4], at::kFloat); else a.top_p = py_float(o[4]);
    if (THPVariable_Check(o[5])) a.min_ps = (const float*)per_row(4, "min_p", o[5], at::kFloat); else a.min_p = py_float(o[5]);
    std::vector<int64_t> sizes(lead.begin(), lead.end());
    sizes.push_back(1);
    const at::Tensor out = at::empty(sizes, logits.options().dtype(at::kInt));
    a.logits = rows_of.data_ptr(); a.logits_stride = step(rows_of, 0, V); a.rows = i32("rows", rows); a.V = i32("V", V); a.out = (int32_t*)out.data_ptr();
    done(csm_ops_sample_workspace(&a, &a.workspace_bytes));
    at::Tensor scratch;
    if (a.workspace_bytes) {
      scratch = at::empty({(int64_t)a.workspace_bytes}, logits.options().dtype(at::kByte));
      a.workspace = scratch.data_ptr();
    }
    done(csm_ops_sample_filtered(&a, call.stream()));
    return THPVariable_Wrap(out);
  });
}

PyMethodDef methods[] = {{"rope_append", (PyCFunction)(void*)rope_append, METH_FASTCALL, nullptr},
                         {"prefix_attention", (PyCFunction)(void*)prefix_attention, METH_FASTCALL, nullptr},
                         {"sample", (PyCFunction)(void*)sample, METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_ops_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__ops_binding(void) {
  PyObject* m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "built_for", CSM_BINDING_STAMP) < 0) Py_CLEAR(m);   // compared with what is installed when it is loaded
  return m;
}
