// The host side of the row and rotary ops in native code: the checks, the outputs and the launches of one call.
//
// What such a pass costs is the host's work: the rotary op forward and backward on 16 tokens took 135 us of Python, where the
// kernels of 14336 tokens take 58, and takes 70 to 83 this way; permute and unpermute of 14593 tokens forward and backward took
// 140 and take 100, which is what their kernels take.  Each function here takes the call as the op got it, and either makes it whole --
// allocates, launches, returns the outputs -- or returns None and has touched nothing: anything but plain CUDA tensors of one device
// with the shapes, types and strides that the kernels read in place (a subclass, a transform's wrapper, a tensor that would
// first be copied or moved, anything to be refused) is the general path's, in native.py, which warns, copies and raises.
// No state is kept between calls.  The library's entry points come in through bind(), from the library that _lib.py loaded.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/hip/HIPStream.h>
#include <pybind11/pybind11.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <initializer_list>
#include <optional>
#include <string>
#include <type_traits>

#include "wallx_mi355.h"

namespace {

struct Entry {
  decltype(&wx_last_error_string) last_error;
  decltype(&wx_mrope_apply) rope;
  decltype(&wx_mrope_apply_bwd) rope_bwd;
  decltype(&wx_mrope_apply_positions) rope_positions;
  decltype(&wx_mrope_apply_packed) rope_packed;
  decltype(&wx_mrope_table_width) table_width;
  decltype(&wx_partition_workspace_bytes) partition_bytes;
  decltype(&wx_partition_build) partition;
  decltype(&wx_permute_rows) permute;
  decltype(&wx_unpermute_rows) unpermute;
  decltype(&wx_unpermute_rows_bwd_clear) unpermute_bwd;
  decltype(&wx_qk_norm_rope) norm_rope;
  decltype(&wx_qk_norm_rope_bwd_workspace_bytes) norm_rope_bwd_bytes;
  decltype(&wx_qk_norm_rope_bwd) norm_rope_bwd;
  decltype(&wx_attention_workspace_bytes) attention_bytes;
  decltype(&wx_attention_fwd) attention;
  decltype(&wx_attention_bwd_workspace_bytes) attention_bwd_bytes;
  decltype(&wx_attention_bwd) attention_bwd;
  decltype(&wx_kv_cache_write) cache_write;
  decltype(&wx_cached_attention) cached_attention;
  decltype(&wx_paged_kv_resize) paged_resize;
  decltype(&wx_paged_kv_write) paged_write;
  decltype(&wx_paged_attention_workspace_bytes) paged_bytes;
  decltype(&wx_paged_attention) paged_attention;
} entry;
const char* const kNames[] = {"wx_last_error_string", "wx_mrope_apply", "wx_mrope_apply_bwd", "wx_mrope_apply_positions",
                              "wx_mrope_apply_packed", "wx_mrope_table_width", "wx_partition_workspace_bytes", "wx_partition_build",
                              "wx_permute_rows", "wx_unpermute_rows", "wx_unpermute_rows_bwd_clear", "wx_qk_norm_rope",
                              "wx_qk_norm_rope_bwd_workspace_bytes", "wx_qk_norm_rope_bwd", "wx_attention_workspace_bytes", "wx_attention_fwd",
                              "wx_attention_bwd_workspace_bytes", "wx_attention_bwd", "wx_kv_cache_write", "wx_cached_attention",
                              "wx_paged_kv_resize", "wx_paged_kv_write", "wx_paged_attention_workspace_bytes", "wx_paged_attention"};
constexpr int kEntries = sizeof(kNames) / sizeof(kNames[0]);
static_assert(sizeof(Entry) == kEntries * sizeof(void*), "a name per entry point");

// A tensor that is what it looks like: strided CUDA memory, no wrapper, no pending conjugation or negation, no tangent of forward-mode
// differentiation (what is launched here would drop it) -- and, as what is allocated inside a transform is a wrapper whatever the inputs
// are, outside of all transforms.
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  for (const c10::DispatchKey transform : {c10::DispatchKey::FuncTorchDynamicLayerFrontMode, c10::DispatchKey::Functionalize})
    if (c10::impl::tls_is_dispatch_key_included(transform)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || t.is_conj() || t.is_neg()) return nullptr;
  constexpr c10::DispatchKeySet wrappers({c10::DispatchKey::Python, c10::DispatchKey::PythonTLSSnapshot, c10::DispatchKey::FuncTorchBatched,
                                          c10::DispatchKey::FuncTorchGradWrapper, c10::DispatchKey::Functionalize,
                                          c10::DispatchKey::ZeroTensor, c10::DispatchKey::Batched});
  if (t.key_set().has_any(wrappers) || !t.has_storage() || t._fw_grad(0).defined()) return nullptr;
  return &t;
}

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? WX_F32 : t == at::kHalf ? WX_F16 : t == at::kBFloat16 ? WX_BF16 : -1;
}

void* ptr(const at::Tensor& t) { return t.numel() == 0 ? nullptr : t.data_ptr(); }

wx_stream_t stream_of(const at::Tensor& t) { return reinterpret_cast<wx_stream_t>(c10::hip::getCurrentHIPStream(t.get_device()).stream()); }

// Runs `f` without the interpreter lock (a launch waits where the queue is full) and with the device of `t` current; the
// library's statuses become Python errors here, C++ exceptions (an allocation that fails) in the functions' own frames.
template <typename F>
bool run(const at::Tensor& t, F f) {
  int rc = 0;
  std::string error;
  {
    const pybind11::gil_scoped_release no_gil;
    const c10::DeviceGuard guard(t.device());
    rc = f();
    if (rc != 0) error = entry.last_error();
  }
  if (rc != 0) PyErr_Format(PyExc_RuntimeError, "wallx_mi355: %s (status %d)", error.c_str(), rc);
  return rc == 0;
}

bool to_int(PyObject* o, int64_t& v) {
  if (!PyLong_CheckExact(o)) return false;
  int overflow = 0;
  v = PyLong_AsLongLongAndOverflow(o, &overflow);
  return overflow == 0;
}

bool section_of(PyObject* o, int sec[3]) {
  if (!PyList_CheckExact(o) && !PyTuple_CheckExact(o)) return false;
  if (PySequence_Fast_GET_SIZE(o) != 3) return false;
  for (int i = 0; i < 3; ++i) {
    int64_t v;
    if (!to_int(PySequence_Fast_GET_ITEM(o, i), v) || v < 0 || v > 1024) return false;
    sec[i] = static_cast<int>(v);
  }
  return true;
}

bool layout_of(PyObject* o, int& layout) {
  if (!PyUnicode_CheckExact(o)) return false;
  if (PyUnicode_CompareWithASCIIString(o, "hf") == 0) layout = WX_MROPE_HF;
  else if (PyUnicode_CompareWithASCIIString(o, "csrc") == 0) layout = WX_MROPE_CSRC;
  else return false;
  return true;
}

PyObject* none() { Py_RETURN_NONE; }

PyObject* wrap(const at::Tensor& t) { return THPVariable_Wrap(t); }

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
  PyObject* const x = wrap(a);
  PyObject* const y = x ? wrap(b) : nullptr;
  PyObject* const r = y ? PyTuple_Pack(2, x, y) : nullptr;
  Py_XDECREF(x);
  Py_XDECREF(y);
  return r;
}

// rope(form, q, k, a, b, section, layout, backward) -> (q_out, k_out) or None.
// form 0: a, b = cos, sin [3, B, S, D]; 1: a, b = position_ids [3, B, S], inv_freq [D / 2]; 2: a = the packed table, b = None.
PyObject* rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t form, backward;
  int sec[3], layout;
  if (n != 8 || !entry.rope || !to_int(args[0], form) || !to_int(args[7], backward) || !section_of(args[5], sec) || !layout_of(args[6], layout)) return none();
  const at::Tensor *q = plain(args[1]), *k = plain(args[2]), *a = plain(args[3]), *b = form == 2 ? a : plain(args[4]);
  if (!q || !k || !a || !b || q->dim() != 4 || k->dim() != 4) return none();
  const int64_t B = q->size(0), Hq = q->size(1), S = q->size(2), D = q->size(3), Hk = k->size(1);
  if (k->size(0) != B || k->size(2) != S || k->size(3) != D || q->stride(3) != 1 || k->stride(3) != 1) return none();
  if (Hq > INT32_MAX || Hk > INT32_MAX || D > INT32_MAX) return none();
  const at::ScalarType dt = q->scalar_type();
  const int code = dtype_code(dt);
  if (code < 0 || k->scalar_type() != dt || k->device() != q->device() || a->device() != q->device() || b->device() != q->device()) return none();
  if (!a->is_contiguous() || !b->is_contiguous()) return none();
  if (form == 0) {
    for (const at::Tensor* t : {a, b})
      if (t->dim() != 4 || t->size(0) != 3 || t->size(1) != B || t->size(2) != S || t->size(3) != D || t->scalar_type() != dt) return none();
  } else if (form == 1) {
    if (a->dim() != 3 || a->size(0) != 3 || a->size(1) != B || a->size(2) != S || a->scalar_type() != at::kLong) return none();
    if (b->dim() != 1 || b->size(0) != D / 2 || b->scalar_type() != at::kFloat) return none();
  } else if (form == 2) {
    const int width = entry.table_width(static_cast<int>(D), sec, layout);
    if (width < 0 || a->dim() != 2 || a->size(0) != B * S || a->size(1) != width || a->scalar_type() != at::kInt || dt != at::kBFloat16) return none();
  } else {
    return none();
  }
  at::Tensor qo, ko;
  const bool ok = run(*q, [&] {
    qo = at::empty(q->sizes(), q->options());
    ko = at::empty(k->sizes(), k->options());
    const int64_t sq[3] = {q->stride(0), q->stride(1), q->stride(2)}, sk[3] = {k->stride(0), k->stride(1), k->stride(2)};
    const int64_t so[3] = {qo.stride(0), qo.stride(1), qo.stride(2)}, st[3] = {ko.stride(0), ko.stride(1), ko.stride(2)};
    const int hq = static_cast<int>(Hq), hk = static_cast<int>(Hk), d = static_cast<int>(D);
    const wx_stream_t stream = stream_of(*q);
    if (form == 0)
      return (backward ? entry.rope_bwd : entry.rope)(ptr(*q), ptr(*k), ptr(*a), ptr(*b), ptr(qo), ptr(ko), B, S, hq, hk, d, sq, sk, so, st, sec, layout, code, stream);
    if (form == 1)
      return entry.rope_positions(ptr(*q), ptr(*k), static_cast<const int64_t*>(ptr(*a)), static_cast<const float*>(ptr(*b)), ptr(qo), ptr(ko), B, S, hq, hk, d,
                                  sq, sk, so, st, sec, layout, code, backward != 0, stream);
    return entry.rope_packed(ptr(*q), ptr(*k), static_cast<const uint32_t*>(ptr(*a)), ptr(qo), ptr(ko), B, S, hq, hk, d, sq, sk, so, st, sec, layout, code,
                             backward != 0, stream);
  });
  return ok ? pair(qo, ko) : nullptr;
  END_HANDLE_TH_ERRORS
}

// permute(input [T, H], indices int32 [T, K], num_out_tokens, histograms, status, experts) -> (permuted, row_id_map) or None.
// The scratch is the caller's, and large enough (else the general path makes another), or with None this call's own; no status
// word with None.
PyObject* permute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t num_out, experts;
  if (n != 6 || !entry.partition || !to_int(args[2], num_out) || !to_int(args[5], experts)) return none();
  const at::Tensor *x = plain(args[0]), *ids = plain(args[1]), *hist = args[3] == Py_None ? nullptr : plain(args[3]),
                   *status = args[4] == Py_None ? nullptr : plain(args[4]);
  if (!x || !ids || (args[3] != Py_None && !hist) || (args[4] != Py_None && !status)) return none();
  if (x->dim() != 2 || ids->dim() != 2 || !x->is_contiguous() || !ids->is_contiguous()) return none();
  const int64_t T = ids->size(0), K = ids->size(1), H = x->size(1);
  const int code = dtype_code(x->scalar_type());
  if (code < 0 || ids->scalar_type() != at::kInt || x->size(0) != T || T <= 0 || K <= 0 || K > 128 || H <= 0 || num_out < 0) return none();
  for (const at::Tensor* t : {ids, hist, status})
    if (t && t->device() != x->device()) return none();
  const int64_t need = static_cast<int64_t>(entry.partition_bytes(T * K));
  if ((hist && (!hist->is_contiguous() || hist->numel() * hist->element_size() < need)) || (status && status->numel() < 1)) return none();
  at::Tensor out, map;
  const bool ok = run(*x, [&] {
    const at::TensorOptions i32 = ids->options();
    map = at::empty({T * K}, i32);
    at::Tensor offsets = at::empty({experts + 1}, i32);
    out = at::empty({num_out > 0 ? num_out : T * K, H}, x->options());
    const at::Tensor scratch = hist ? *hist : at::empty({need}, x->options().dtype(at::kByte));
    const wx_stream_t stream = stream_of(*x);
    const int rc = entry.partition(ptr(*ids), WX_I32, T, static_cast<int>(K), static_cast<int>(experts), num_out, static_cast<int32_t*>(ptr(map)), nullptr,
                                   static_cast<int32_t*>(offsets.data_ptr()), status ? static_cast<int32_t*>(status->data_ptr()) : nullptr, ptr(scratch),
                                   static_cast<size_t>(scratch.numel()) * scratch.element_size(), stream);
    return rc != 0 ? rc : entry.permute(ptr(*x), ptr(out), static_cast<const int32_t*>(ptr(map)), T, static_cast<int>(K), H, code, stream);
  });
  return ok ? pair(out, map) : nullptr;
  END_HANDLE_TH_ERRORS
}

// unpermute(input, row_id_map int32, probs fp32 [T, K] or None, T, K) -> output [T, H] or None.
PyObject* unpermute(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t T, K;
  if (n != 5 || !entry.unpermute || !to_int(args[3], T) || !to_int(args[4], K)) return none();
  const at::Tensor *x = plain(args[0]), *map = plain(args[1]), *probs = args[2] == Py_None ? nullptr : plain(args[2]);
  if (!x || !map || (args[2] != Py_None && !probs) || x->dim() != 2 || !x->is_contiguous() || !map->is_contiguous()) return none();
  const int code = dtype_code(x->scalar_type());
  if (code < 0 || T <= 0 || K <= 0 || K > 128 || map->scalar_type() != at::kInt || map->numel() < T * K || map->device() != x->device()) return none();
  if (probs && (!probs->is_contiguous() || probs->scalar_type() != at::kFloat || probs->device() != x->device() || probs->numel() == 0)) return none();
  at::Tensor out;
  const bool ok = run(*x, [&] {
    out = at::empty({T, x->size(1)}, x->options());
    return entry.unpermute(ptr(*x), ptr(out), static_cast<const int32_t*>(ptr(*map)), probs && K > 1 ? static_cast<const float*>(ptr(*probs)) : nullptr, T,
                           static_cast<int>(K), x->size(1), code, stream_of(*x));
  });
  return ok ? wrap(out) : nullptr;
  END_HANDLE_TH_ERRORS
}

// unpermute_bwd(grad [T, H], input_fwd [R, H], row_id_map int32, probs fp32 [T, K] or None) -> act_grad [R, H], or with probs
// (act_grad, their gradient [T, K]), or None.  Without probs: one expert per token.  (A single weight per token, whose
// gradient is zeros, is the general path's.)
PyObject* unpermute_bwd(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 4 || !entry.unpermute_bwd) return none();
  const at::Tensor *g = plain(args[0]), *x = plain(args[1]), *map = plain(args[2]), *probs = args[3] == Py_None ? nullptr : plain(args[3]);
  if (!g || !x || !map || (args[3] != Py_None && !probs) || g->dim() != 2 || x->dim() != 2 || !g->is_contiguous() || !x->is_contiguous() ||
      !map->is_contiguous())
    return none();
  const int64_t T = g->size(0), K = probs ? (probs->dim() == 2 ? probs->size(1) : 0) : 1;
  if (probs && (K < 2 || K > 128 || probs->size(0) != T || !probs->is_contiguous() || probs->scalar_type() != at::kFloat || probs->device() != g->device()))
    return none();
  const int code = dtype_code(g->scalar_type());
  if (code < 0 || x->scalar_type() != g->scalar_type() || map->scalar_type() != at::kInt || x->size(1) != g->size(1) || g->numel() == 0 || x->numel() == 0 ||
      map->numel() < T * K || x->device() != g->device() || map->device() != g->device())
    return none();
  at::Tensor out, prob_grad;
  const bool ok = run(*g, [&] {
    out = at::empty({x->size(0), g->size(1)}, g->options());
    if (probs) prob_grad = at::empty({T, K}, probs->options());
    return entry.unpermute_bwd(ptr(*g), ptr(*x), ptr(out), out.size(0), probs ? static_cast<float*>(ptr(prob_grad)) : nullptr,
                               static_cast<const int32_t*>(ptr(*map)), probs ? static_cast<const float*>(ptr(*probs)) : nullptr, T, static_cast<int>(K),
                               g->size(1), code, stream_of(*g));
  });
  return !ok ? nullptr : (probs ? pair(out, prob_grad) : wrap(out));
  END_HANDLE_TH_ERRORS
}

// ---- the norm of q and k with the rotary embedding, attention, the cache.  Forward and backward are autograd nodes of their own here:
// a Python autograd.Function around native calls costs 50 us of a training pass, as much as the norm's kernels on 5000 tokens take.

using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

// [B, H, S, D] as the kernels read it through strides: contiguous heads, rows on 16 bytes
bool rows16(const at::Tensor& t) {
  if (t.dim() != 4 || (t.stride(3) != 1 && t.size(3) != 1)) return false;
  const int64_t unit = 16 / t.element_size();
  for (int i = 0; i < 3; ++i)
    if (t.size(i) > 1 && (t.stride(i) % unit != 0 || t.stride(i) < 0)) return false;
  return t.numel() == 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
}
at::Tensor as_rows16(const at::Tensor& t) { return rows16(t) ? t : t.clone(at::MemoryFormat::Contiguous); }

bool packed16(const at::Tensor& t) { return t.is_contiguous() && (t.numel() == 0 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0); }

struct RowStrides {
  int64_t v[3];
  explicit RowStrides(const at::Tensor& t) {
    for (int i = 0; i < 3; ++i) v[i] = t.size(i) > 1 ? t.stride(i) : 0;
  }
};

// [B, H, S, D] over token-major memory, no view of anything: a caller may write into it in place
at::Tensor token_major(int64_t B, int64_t H, int64_t S, int64_t D, const at::TensorOptions& options) {
  return at::empty_strided({B, H, S, D}, {S * H * D, D, H * D, 1}, options);
}

// As run(), for code under an autograd node: the library's errors are exceptions there.
template <typename F>
void launch(const at::Tensor& t, F f) {
  const c10::DeviceGuard guard(t.device());
  const int rc = f();
  TORCH_CHECK(rc == 0, "wallx_mi355: ", entry.last_error(), " (status ", rc, ")");
}

// A backward pass under capture must not hand its gradients to a node that was made on the default stream, as the accumulation into a
// leaf is whose eager graph still lives: the engine makes that node's stream wait for the capturing one, which HIP does not allow the
// default stream (id 0), and what is left of the capture ends the process.  Called before the first launch, under the node at work.
void check_capture(const at::Tensor& t) {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  if (hipStreamIsCapturing(reinterpret_cast<hipStream_t>(stream_of(t)), &status) != hipSuccess || status != hipStreamCaptureStatusActive) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  for (const auto& edge : node->next_edges())
    if (const auto made = edge.function ? edge.function->stream() : std::nullopt)
      TORCH_CHECK(made->id() != 0, "a backward pass is captured while an earlier graph of the same leaves, made on the default stream, is alive: drop "
                                   "that graph's outputs first, or capture the gradients of detached copies");
}

bool optional(PyObject* o, const at::Tensor*& t) {
  t = nullptr;
  return o == Py_None || (t = plain(o)) != nullptr;
}
bool to_double(PyObject* o, double& v) {
  if (!PyFloat_CheckExact(o)) return false;
  v = PyFloat_AS_DOUBLE(o);
  return true;
}
bool needs_grad(std::initializer_list<const at::Tensor*> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const at::Tensor* t : ts)
    if (t && t->requires_grad()) return true;
  return false;
}
PyObject* wrap_all(const variable_list& v) { return v.size() == 1 ? wrap(v[0]) : pair(v[0], v[1]); }

// What a graph of gradients (create_graph) gets of a backward pass that is not differentiable itself: its gradients, as results of a node that
// hangs on everything they were made from and raises where a second derivative is asked through it.
struct NoSecond : torch::autograd::Function<NoSecond> {
  static variable_list forward(AutogradContext* ctx, at::TensorList grads_and_from, int64_t count, const std::string& what) {
    ctx->saved_data["what"] = what;
    variable_list out;
    for (int64_t i = 0; i < count; ++i) out.push_back(grads_and_from[i].view_as(grads_and_from[i]));
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list&) {
    TORCH_CHECK(false, ctx->saved_data["what"].toStringRef(), "'s backward is not differentiable");
  }
};
void no_second(variable_list& grads, std::initializer_list<variable_list> from, const char* what) {
  variable_list all;
  for (const at::Tensor& g : grads)
    if (g.defined()) all.push_back(g);
  const int64_t count = static_cast<int64_t>(all.size());
  for (const variable_list& list : from)
    for (const at::Tensor& t : list)
      if (t.defined()) all.push_back(t);
  const variable_list held = NoSecond::apply(at::TensorList(all), count, std::string(what));
  size_t i = 0;
  for (at::Tensor& g : grads)
    if (g.defined()) g = held[i++];
}

struct NormRope : torch::autograd::Function<NormRope> {
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k, const Variable& wq, const Variable& wk, const Variable& source,
                               const std::optional<at::Tensor>& inv_freq, at::IntArrayRef section, double eps, int64_t layout) {
    const at::Tensor freq = inv_freq.value_or(at::Tensor());
    at::Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
    const int sec[3] = {static_cast<int>(section[0]), static_cast<int>(section[1]), static_cast<int>(section[2])};
    launch(q, [&] {
      return entry.norm_rope(ptr(q), ptr(k), ptr(wq), ptr(wk), static_cast<float>(eps), ptr(source), freq.defined() ? static_cast<const float*>(ptr(freq)) : nullptr,
                             ptr(qo), ptr(ko), q.size(0), q.size(2), static_cast<int>(q.size(1)), static_cast<int>(k.size(1)), static_cast<int>(q.size(3)),
                             RowStrides(q).v, RowStrides(k).v, sec, static_cast<int>(layout), dtype_code(q.scalar_type()), stream_of(q));
    });
    if (ctx) {
      ctx->save_for_backward({q, k, wq, wk, source, freq});
      ctx->saved_data["section"] = section.vec();
      ctx->saved_data["eps"] = eps;
      ctx->saved_data["layout"] = layout;
    }
    return {qo, ko};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    variable_list out = gradients(ctx, saved, grads);
    if (at::GradMode::is_enabled()) no_second(out, {grads, {saved[0], saved[1], saved[2], saved[3]}}, "qk_norm_rope");
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& saved, const variable_list& grads) {
    const at::NoGradGuard no_grad;
    const at::Tensor q = as_rows16(saved[0]), k = as_rows16(saved[1]);  // (saved-tensor hooks may hand them back in another order)
    const at::Tensor &wq = saved[2], &wk = saved[3], &source = saved[4], &freq = saved[5];
    const std::vector<int64_t> section = ctx->saved_data["section"].toIntVector();
    const int sec[3] = {static_cast<int>(section[0]), static_cast<int>(section[1]), static_cast<int>(section[2])};
    const int layout = static_cast<int>(ctx->saved_data["layout"].toInt());
    variable_list out(9);
    launch(q, [&] {
      const at::Tensor gq = as_rows16(grads[0]), gk = as_rows16(grads[1]);
      const at::Tensor* like[4] = {&q, &k, &wq, &wk};
      for (int i = 0; i < 4; ++i)
        if (ctx->needs_input_grad(i)) out[i] = at::empty(like[i]->sizes(), q.options());
      const int D = static_cast<int>(q.size(3));
      const bool weights = out[2].defined() || out[3].defined();
      const size_t bytes = weights ? entry.norm_rope_bwd_bytes(D) : 0;
      const at::Tensor work = weights ? at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)) : at::Tensor();
      auto at_ = [&](int i) { return out[i].defined() ? ptr(out[i]) : nullptr; };
      return entry.norm_rope_bwd(ptr(gq), ptr(gk), ptr(q), ptr(k), ptr(wq), ptr(wk), static_cast<float>(ctx->saved_data["eps"].toDouble()), ptr(source),
                                 freq.defined() ? static_cast<const float*>(ptr(freq)) : nullptr, at_(0), at_(1), at_(2), at_(3), q.size(0), q.size(2),
                                 static_cast<int>(q.size(1)), static_cast<int>(k.size(1)), D, RowStrides(gq).v, RowStrides(gk).v, RowStrides(q).v,
                                 RowStrides(k).v, sec, layout, dtype_code(q.scalar_type()), weights ? ptr(work) : nullptr, bytes, stream_of(q));
    });
    return out;
  }
};

// norm_rope(q, k, q_weight, k_weight, source, inv_freq or None, section, eps, layout) -> (q_out, k_out) or None.
PyObject* norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int sec[3], layout;
  double eps;
  const at::Tensor* freq;
  if (n != 9 || !entry.norm_rope || !optional(args[5], freq) || !section_of(args[6], sec) || !to_double(args[7], eps) || !layout_of(args[8], layout)) return none();
  const at::Tensor *q = plain(args[0]), *k = plain(args[1]), *wq = plain(args[2]), *wk = plain(args[3]), *source = plain(args[4]);
  if (!q || !k || !wq || !wk || !source || !rows16(*q) || !rows16(*k)) return none();
  const int64_t B = q->size(0), S = q->size(2), D = q->size(3);
  const at::ScalarType dt = q->scalar_type();
  if (k->size(0) != B || k->size(2) != S || k->size(3) != D || dtype_code(dt) < 0 || q->size(1) > INT32_MAX || k->size(1) > INT32_MAX || D > INT32_MAX) return none();
  for (const at::Tensor* t : {k, wq, wk, source, freq})
    if (t && t->device() != q->device()) return none();
  for (const at::Tensor* w : {wq, wk})
    if (w->scalar_type() != dt || w->dim() != 1 || w->size(0) != D || !packed16(*w)) return none();
  if (k->scalar_type() != dt || !packed16(*source)) return none();
  if (freq) {
    if (source->dim() != 3 || source->size(0) != 3 || source->size(1) != B || source->size(2) != S || source->scalar_type() != at::kLong) return none();
    if (freq->dim() != 1 || freq->size(0) != D / 2 || freq->scalar_type() != at::kFloat || !freq->is_contiguous() || freq->numel() == 0) return none();
  } else {
    const int width = entry.table_width(static_cast<int>(D), sec, layout);
    if (width < 0 || source->dim() != 2 || source->size(0) != B * S || source->size(1) != width || source->scalar_type() != at::kInt || dt != at::kBFloat16) return none();
  }
  const int64_t section[3] = {sec[0], sec[1], sec[2]};
  const std::optional<at::Tensor> inv_freq = freq ? std::optional<at::Tensor>(*freq) : std::nullopt;
  variable_list out;
  {
    const pybind11::gil_scoped_release no_gil;
    out = needs_grad({q, k, wq, wk}) ? NormRope::apply(*q, *k, *wq, *wk, *source, inv_freq, at::IntArrayRef(section, 3), eps, static_cast<int64_t>(layout))
                                     : NormRope::forward(nullptr, *q, *k, *wq, *wk, *source, inv_freq, at::IntArrayRef(section, 3), eps, layout);
  }
  return wrap_all(out);
  END_HANDLE_TH_ERRORS
}

const int32_t* ints(const at::Tensor& t) { return t.defined() ? static_cast<const int32_t*>(ptr(t)) : nullptr; }

struct Attention : torch::autograd::Function<Attention> {
  static variable_list forward(AutogradContext* ctx, const Variable& q, const Variable& k, const Variable& v, const std::optional<at::Tensor>& key_ranges,
                               const std::optional<at::Tensor>& key_lengths, bool causal, double scale) {
    const at::Tensor ranges = key_ranges.value_or(at::Tensor()), lengths = key_lengths.value_or(at::Tensor());
    const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3), Hk = k.size(1), Sk = k.size(2);
    at::Tensor out, lse, rest;
    launch(q, [&] {
      out = token_major(B, Hq, Sq, D, q.options());
      if (ctx) lse = at::empty({B, Hk, Sq * (Hq / Hk)}, q.options().dtype(at::kFloat));
      if (ctx) rest = at::empty({B, Sq, Hq, D}, q.options().dtype(at::kByte));
      const size_t bytes = entry.attention_bytes(B, static_cast<int>(Hq), static_cast<int>(Hk), Sq, Sk, static_cast<int>(D));
      const at::Tensor work = bytes ? at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)) : at::Tensor();
      return entry.attention(ptr(q), ptr(k), ptr(v), ptr(out), ctx ? static_cast<float*>(ptr(lse)) : nullptr, ctx ? ptr(rest) : nullptr, ints(ranges), ints(lengths), causal, B,
                             static_cast<int>(Hq), static_cast<int>(Hk), Sq, Sk, static_cast<int>(D), RowStrides(q).v, RowStrides(k).v, RowStrides(v).v,
                             static_cast<float>(scale), dtype_code(q.scalar_type()), bytes ? ptr(work) : nullptr, bytes, stream_of(q));
    });
    if (ctx) {
      ctx->save_for_backward({q, k, v, out, lse, rest, ranges, lengths});
      ctx->saved_data["causal"] = causal;
      ctx->saved_data["scale"] = scale;
    }
    return {out};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    const variable_list saved = ctx->get_saved_variables();
    check_capture(saved[0]);
    variable_list out = gradients(ctx, saved, grads);
    if (at::GradMode::is_enabled()) no_second(out, {grads, {saved[0], saved[1], saved[2]}}, "attention");
    return out;
  }
  static variable_list gradients(AutogradContext* ctx, const variable_list& saved, const variable_list& grads) {
    const at::NoGradGuard no_grad;
    const at::Tensor q = as_rows16(saved[0]), k = as_rows16(saved[1]), v = as_rows16(saved[2]);  // (see above)
    const at::Tensor &out = saved[3], &lse = saved[4], &rest = saved[5], &ranges = saved[6], &lengths = saved[7];
    const int64_t B = q.size(0), Hq = q.size(1), Sq = q.size(2), D = q.size(3), Hk = k.size(1), Sk = k.size(2);
    at::Tensor dq, dk, dv;
    launch(q, [&] {
      const at::Tensor g = as_rows16(grads[0]);
      dq = token_major(B, Hq, Sq, D, q.options());
      dk = token_major(B, Hk, Sk, D, q.options());
      dv = token_major(B, Hk, Sk, D, q.options());
      at::Tensor tokens = out.transpose(1, 2);
      if (!packed16(tokens)) tokens = tokens.clone(at::MemoryFormat::Contiguous);
      const size_t bytes = entry.attention_bwd_bytes(B, static_cast<int>(Hq), static_cast<int>(Hk), Sq, Sk, static_cast<int>(D));
      const at::Tensor work = bytes ? at::empty({static_cast<int64_t>(bytes)}, q.options().dtype(at::kByte)) : at::Tensor();
      return entry.attention_bwd(ptr(q), ptr(k), ptr(v), ptr(tokens), static_cast<const float*>(ptr(lse)), ptr(rest), ptr(g), ptr(dq), ptr(dk), ptr(dv), ints(ranges),
                                 ints(lengths), ctx->saved_data["causal"].toBool(), B, static_cast<int>(Hq), static_cast<int>(Hk), Sq, Sk, static_cast<int>(D),
                                 RowStrides(q).v, RowStrides(k).v, RowStrides(v).v, RowStrides(g).v, static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                 dtype_code(q.scalar_type()), bytes ? ptr(work) : nullptr, bytes, stream_of(q));
    });
    variable_list r(7);
    if (ctx->needs_input_grad(0)) r[0] = dq;
    if (ctx->needs_input_grad(1)) r[1] = dk;
    if (ctx->needs_input_grad(2)) r[2] = dv;
    return r;
  }
};

// The mask and the scale that attention's two forms share.
struct MaskArgs {
  const at::Tensor *ranges, *lengths;
  bool causal;
  double scale;
  bool from(PyObject* r, PyObject* l, PyObject* c, PyObject* s, const at::Tensor& q) {
    if (!optional(r, ranges) || !optional(l, lengths) || !PyBool_Check(c)) return false;
    causal = c == Py_True;
    scale = 1.0 / std::sqrt(static_cast<double>(q.size(3)));
    if (s != Py_None && !to_double(s, scale)) return false;
    const int64_t B = q.size(0), S = q.size(2);
    if (ranges && (ranges->dim() != 3 || ranges->size(0) != B || ranges->size(1) != S || ranges->size(2) != 2 || ranges->scalar_type() != at::kInt || !packed16(*ranges)))
      return false;
    if (lengths && (lengths->dim() != 1 || lengths->size(0) != B || lengths->scalar_type() != at::kInt || !lengths->is_contiguous())) return false;
    for (const at::Tensor* t : {ranges, lengths})
      if (t && t->device() != q.device()) return false;
    return true;
  }
};
bool attention_type(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }
bool heads_fit(int64_t Hq, int64_t Hk) { return Hk > 0 && Hq % Hk == 0 && Hq <= INT32_MAX; }

// attention(q, k, v, key_ranges, key_lengths, causal, scale) -> out or None.
PyObject* attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !entry.attention) return none();
  const at::Tensor *q = plain(args[0]), *k = plain(args[1]), *v = plain(args[2]);
  MaskArgs m;
  if (!q || !k || !v || !rows16(*q) || !rows16(*k) || !rows16(*v) || !m.from(args[3], args[4], args[5], args[6], *q)) return none();
  if (!k->sizes().equals(v->sizes()) || k->size(0) != q->size(0) || k->size(3) != q->size(3) || !heads_fit(q->size(1), k->size(1)) || q->size(3) > 1024) return none();
  if (!attention_type(q->scalar_type()) || k->scalar_type() != q->scalar_type() || v->scalar_type() != q->scalar_type() || k->device() != q->device() ||
      v->device() != q->device())
    return none();
  const std::optional<at::Tensor> ranges = m.ranges ? std::optional<at::Tensor>(*m.ranges) : std::nullopt,
                                  lengths = m.lengths ? std::optional<at::Tensor>(*m.lengths) : std::nullopt;
  variable_list out;
  {
    const pybind11::gil_scoped_release no_gil;
    out = needs_grad({q, k, v}) ? Attention::apply(*q, *k, *v, ranges, lengths, m.causal, m.scale) : Attention::forward(nullptr, *q, *k, *v, ranges, lengths, m.causal, m.scale);
  }
  return wrap(out[0]);
  END_HANDLE_TH_ERRORS
}

// k_cache, v_cache, k_scale, v_scale on q's device in the layout that the kernels take
bool cache_of(PyObject* const* args, const at::Tensor& q, const at::Tensor* (&c)[4]) {
  for (int i = 0; i < 4; ++i) {
    if ((c[i] = plain(args[i])) == nullptr || !packed16(*c[i]) || c[i]->device() != q.device()) return false;
    if (c[i]->scalar_type() != (i < 2 ? at::kFloat8_e4m3fn : at::kFloat)) return false;
  }
  if (c[0]->dim() != 4 || !c[1]->sizes().equals(c[0]->sizes()) || c[0]->size(0) != q.size(0) || c[0]->size(3) != q.size(3) || q.size(3) > 1024) return false;
  for (int i = 2; i < 4; ++i)
    if (!c[i]->sizes().equals(c[0]->sizes().slice(0, 3))) return false;
  return true;
}

// cached_attention(q, k_cache, v_cache, k_scale, v_scale, key_ranges, key_lengths, causal, scale) -> out or None.
PyObject* cached_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 9 || !entry.cached_attention) return none();
  const at::Tensor *q = plain(args[0]), *c[4];
  MaskArgs m;
  if (!q || !rows16(*q) || !cache_of(args + 1, *q, c) || !m.from(args[5], args[6], args[7], args[8], *q)) return none();
  if (!attention_type(q->scalar_type()) || !heads_fit(q->size(1), c[0]->size(1)) || needs_grad({q})) return none();
  const int64_t B = q->size(0), Hq = q->size(1), Sq = q->size(2), D = q->size(3), Hk = c[0]->size(1), C = c[0]->size(2);
  at::Tensor out;
  const bool ok = run(*q, [&] {
    out = token_major(B, Hq, Sq, D, q->options());
    const size_t bytes = entry.attention_bytes(B, static_cast<int>(Hq), static_cast<int>(Hk), Sq, C, static_cast<int>(D));
    const at::Tensor work = bytes ? at::empty({static_cast<int64_t>(bytes)}, q->options().dtype(at::kByte)) : at::Tensor();
    return entry.cached_attention(ptr(*q), ptr(*c[0]), ptr(*c[1]), static_cast<const float*>(ptr(*c[2])), static_cast<const float*>(ptr(*c[3])), ptr(out),
                                  m.ranges ? ints(*m.ranges) : nullptr, m.lengths ? ints(*m.lengths) : nullptr, m.causal, B, static_cast<int>(Hq),
                                  static_cast<int>(Hk), Sq, C, static_cast<int>(D), RowStrides(*q).v, static_cast<float>(m.scale),
                                  dtype_code(q->scalar_type()), bytes ? ptr(work) : nullptr, bytes, stream_of(*q));
  });
  return ok ? wrap(out) : nullptr;
  END_HANDLE_TH_ERRORS
}

// cache_write(k, v, k_cache, v_cache, k_scale, v_scale, start, lengths) -> True or None.
PyObject* cache_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 8 || !entry.cache_write) return none();
  const at::Tensor *k = plain(args[0]), *v = plain(args[1]), *c[4], *start = plain(args[6]), *lengths;
  if (!k || !v || !start || !optional(args[7], lengths) || !rows16(*k) || !rows16(*v) || !cache_of(args + 2, *k, c)) return none();
  if (!v->sizes().equals(k->sizes()) || c[0]->size(1) != k->size(1) || k->size(1) > INT32_MAX || !attention_type(k->scalar_type()) || v->scalar_type() != k->scalar_type() ||
      v->device() != k->device() || needs_grad({k, v}))
    return none();
  for (const at::Tensor* t : {start, lengths})
    if (t && (t->dim() != 1 || t->size(0) != k->size(0) || t->scalar_type() != at::kInt || !t->is_contiguous() || t->device() != k->device())) return none();
  const bool ok = run(*k, [&] {
    return entry.cache_write(ptr(*k), ptr(*v), ptr(*c[0]), ptr(*c[1]), static_cast<float*>(ptr(*c[2])), static_cast<float*>(ptr(*c[3])), ints(*start),
                             lengths ? ints(*lengths) : nullptr, k->size(0), static_cast<int>(k->size(1)), k->size(2), c[0]->size(2), static_cast<int>(k->size(3)),
                             RowStrides(*k).v, RowStrides(*v).v, dtype_code(k->scalar_type()), stream_of(*k));
  });
  if (!ok) return nullptr;
  for (const at::Tensor* t : c)
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();  // (written in place, as an in-place op would)
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// ---- the paged cache
void written(const at::Tensor* t) {  // in place, as an in-place op would
  if (t && !t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
}
bool is_ints(const at::Tensor* t, int64_t dim, const at::Tensor& like) {
  return t && t->dim() == dim && t->scalar_type() == at::kInt && t->is_contiguous() && t->device() == like.device();
}

// paged_resize(lengths, wanted, page_table, free_pages, free_count, page_size, max_tokens) -> (lengths, free_count, starts, slots, positions) or None.
PyObject* paged_resize(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  int64_t page_size, max_tokens;
  if (n != 7 || !entry.paged_resize || !to_int(args[5], page_size) || !to_int(args[6], max_tokens)) return none();
  const at::Tensor *lengths = plain(args[0]), *wanted = plain(args[1]), *table = plain(args[2]), *stack = plain(args[3]), *count = plain(args[4]);
  if (!lengths || !is_ints(lengths, 1, *lengths) || !is_ints(wanted, 1, *lengths) || !is_ints(table, 2, *lengths) || !is_ints(stack, 1, *lengths) ||
      !is_ints(count, 1, *lengths))
    return none();
  const int64_t R = lengths->size(0);
  if (wanted->size(0) != R || table->size(0) != R || count->size(0) != 1 || page_size <= 0 || page_size > INT32_MAX || max_tokens < 0) return none();
  at::Tensor out[5];
  const bool ok = run(*lengths, [&] {
    // (an allocation each: as parts of one, 4.3 us a call for 6.1, each grew over its neighbours and kept them)
    const int64_t sizes[5] = {R, 1, R + 1, max_tokens, max_tokens};
    for (int i = 0; i < 5; ++i) out[i] = at::empty({sizes[i]}, i < 4 ? lengths->options() : lengths->options().dtype(at::kLong));
    auto to = [&](int i) { return static_cast<int32_t*>(ptr(out[i])); };
    return entry.paged_resize(ints(*lengths), ints(*wanted), static_cast<int32_t*>(ptr(*table)), static_cast<int32_t*>(ptr(*stack)), ints(*count), to(0), to(1), to(2),
                              to(3), static_cast<int64_t*>(ptr(out[4])), R, table->size(1), stack->size(0), static_cast<int>(page_size), max_tokens, stream_of(*lengths));
  });
  if (!ok) return nullptr;
  written(table);
  written(stack);
  PyObject* const r = PyTuple_New(5);
  for (int i = 0; r && i < 5; ++i) PyTuple_SET_ITEM(r, i, wrap(out[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

// k_pages, v_pages, k_scale, v_scale on q's device in the layout that the kernels take: e4m3 with scales, or q's type without
bool pages_of(PyObject* const* args, const at::Tensor& q, const at::Tensor* (&c)[4]) {
  for (int i = 0; i < 4; ++i)
    if (i < 2 ? (c[i] = plain(args[i])) == nullptr : !optional(args[i], c[i])) return false;
  if ((c[2] == nullptr) != (c[3] == nullptr) || c[0]->dim() != 4 || !c[1]->sizes().equals(c[0]->sizes()) || c[0]->size(3) != q.size(3) || q.size(3) > 1024) return false;
  for (int i = 0; i < 4; ++i) {
    if (!c[i]) continue;
    if (!packed16(*c[i]) || c[i]->device() != q.device()) return false;
    if (c[i]->scalar_type() != (i >= 2 ? at::kFloat : c[2] ? at::kFloat8_e4m3fn : q.scalar_type())) return false;
    if (i >= 2 && !c[i]->sizes().equals(c[0]->sizes().slice(0, 3))) return false;
  }
  return c[0]->size(1) <= INT32_MAX && c[0]->size(2) > 0 && c[0]->size(2) <= INT32_MAX;
}
float* floats(const at::Tensor* t) { return t ? static_cast<float*>(t->data_ptr()) : nullptr; }

// paged_write(k, v, k_pages, v_pages, k_scale, v_scale, slots) -> True or None.
PyObject* paged_write(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 7 || !entry.paged_write) return none();
  const at::Tensor *k = plain(args[0]), *v = plain(args[1]), *c[4], *slots = plain(args[6]);
  if (!k || !v || !slots || !rows16(*k) || !rows16(*v) || !attention_type(k->scalar_type()) || !pages_of(args + 2, *k, c)) return none();
  if (!v->sizes().equals(k->sizes()) || v->scalar_type() != k->scalar_type() || v->device() != k->device() || c[0]->size(1) != k->size(1) ||
      needs_grad({k, v, c[0], c[1], c[2], c[3]}))
    return none();
  const int64_t B = k->size(0), S = k->size(2);
  if (!(is_ints(slots, 1, *k) && slots->size(0) == B * S) && !(is_ints(slots, 2, *k) && slots->size(0) == B && slots->size(1) == S)) return none();
  const bool ok = run(*k, [&] {
    return entry.paged_write(ptr(*k), ptr(*v), ptr(*c[0]), ptr(*c[1]), floats(c[2]), floats(c[3]), ints(*slots), B, static_cast<int>(k->size(1)), S, c[0]->size(0),
                             static_cast<int>(c[0]->size(2)), static_cast<int>(k->size(3)), RowStrides(*k).v, RowStrides(*v).v, dtype_code(k->scalar_type()),
                             stream_of(*k));
  });
  if (!ok) return nullptr;
  for (const at::Tensor* t : c) written(t);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// paged_attention(q, k_pages, v_pages, k_scale, v_scale, page_table, lengths, starts, causal, scale) -> out or None.
PyObject* paged_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  const at::Tensor *q, *c[4], *table, *lengths, *starts;
  if (n != 10 || !entry.paged_attention || !(q = plain(args[0])) || !rows16(*q) || !attention_type(q->scalar_type()) || !pages_of(args + 1, *q, c)) return none();
  if (!is_ints(table = plain(args[5]), 2, *q) || !is_ints(lengths = plain(args[6]), 1, *q) || !optional(args[7], starts) || !PyBool_Check(args[8])) return none();
  double scale = 1.0 / std::sqrt(static_cast<double>(q->size(3)));
  if (args[9] != Py_None && !to_double(args[9], scale)) return none();
  const int64_t B = q->size(0), Hq = q->size(1), S = q->size(2), D = q->size(3), Hk = c[0]->size(1), R = table->size(0);
  if (!heads_fit(Hq, Hk) || lengths->size(0) != R || (starts ? !is_ints(starts, 1, *q) || starts->size(0) != R + 1 : R != B) ||
      needs_grad({q, c[0], c[1], c[2], c[3]}))
    return none();
  at::Tensor out;
  const bool ok = run(*q, [&] {
    out = token_major(B, Hq, S, D, q->options());
    const size_t bytes = entry.paged_bytes(B * S, static_cast<int>(Hq), static_cast<int>(Hk), static_cast<int>(D));
    const at::Tensor work = bytes ? at::empty({static_cast<int64_t>(bytes)}, q->options().dtype(at::kByte)) : at::Tensor();
    return entry.paged_attention(ptr(*q), ptr(*c[0]), ptr(*c[1]), floats(c[2]), floats(c[3]), ptr(out), ints(*table), ints(*lengths), starts ? ints(*starts) : nullptr,
                                 args[8] == Py_True, B, static_cast<int>(Hq), static_cast<int>(Hk), S, R, table->size(1), c[0]->size(0), static_cast<int>(c[0]->size(2)),
                                 static_cast<int>(D), RowStrides(*q).v, static_cast<float>(scale), dtype_code(q->scalar_type()), bytes ? ptr(work) : nullptr, bytes,
                                 stream_of(*q));
  });
  return ok ? wrap(out) : nullptr;
  END_HANDLE_TH_ERRORS
}

// names() -> the entry points in the order bind() takes their addresses in.
PyObject* names(PyObject*, PyObject*) {
  PyObject* const r = PyTuple_New(kEntries);
  for (int i = 0; r && i < kEntries; ++i) PyTuple_SET_ITEM(r, i, PyUnicode_FromString(kNames[i]));
  return r;
}

PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != kEntries) return PyErr_Format(PyExc_TypeError, "bind takes %d addresses", kEntries);
  void* at[kEntries];
  for (int i = 0; i < kEntries; ++i) {
    at[i] = PyLong_AsVoidPtr(args[i]);
    if (!at[i]) {
      if (!PyErr_Occurred()) PyErr_SetString(PyExc_ValueError, "null address");
      return nullptr;
    }
  }
  static_assert(std::is_trivially_copyable_v<Entry>);
  memcpy(&entry, at, sizeof(entry));
  return none();
}

// capture_check(tensor): check_capture for the backward of a node in Python.
PyObject* capture_check(PyObject*, PyObject* const* args, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (const at::Tensor* t = n == 1 ? plain(args[0]) : nullptr) check_capture(*t);
  return none();
  END_HANDLE_TH_ERRORS
}

#define WX_FAST(f) reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(f)), METH_FASTCALL
PyMethodDef methods[] = {{"rope", WX_FAST(rope), nullptr},
                         {"capture_check", WX_FAST(capture_check), nullptr},
                         {"permute", WX_FAST(permute), nullptr},
                         {"unpermute", WX_FAST(unpermute), nullptr},
                         {"unpermute_bwd", WX_FAST(unpermute_bwd), nullptr},
                         {"norm_rope", WX_FAST(norm_rope), nullptr},
                         {"attention", WX_FAST(attention), nullptr},
                         {"cached_attention", WX_FAST(cached_attention), nullptr},
                         {"cache_write", WX_FAST(cache_write), nullptr},
                         {"paged_resize", WX_FAST(paged_resize), nullptr},
                         {"paged_write", WX_FAST(paged_write), nullptr},
                         {"paged_attention", WX_FAST(paged_attention), nullptr},
                         {"bind", WX_FAST(bind), nullptr},
                         {"names", names, METH_NOARGS, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_wallx_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__wallx_host() { return PyModule_Create(&module); }
