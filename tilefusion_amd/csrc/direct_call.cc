// Python module tilefusion_amd._direct: the ops called without the work that the dispatcher does for any op from Python.
//
// A call of torch.ops.tilefusion.* from Python costs ~2 us beside the launch (matching the arguments to the schema,
// boxing them, three dispatch keys under which nothing is done), as much as the launch of a small kernel.  The functions
// here take a call only where the dispatcher would do nothing but call what is registered for the CUDA key: plain
// device tensors, no gradient asked for, nothing that watches or rewrites ops (see `plain`).  Otherwise they
// return False (None), having done nothing, and the wrapper in tilefusion_amd/ops goes through torch.ops, as it does for
// torch.compile and torch.jit.script.  What is called is the dispatcher's CUDA kernel of the op, an implementation that a
// program registers in place of the library's included.
// us a call in a loop, through torch.ops / as here: gemm 128 x 64 x 256 4.6 / 3.7; fused 16384 x 128 x 128 x 128 4.7 / 4.4 and decoding
// 32 x 1999 x 64 9.4 / 9.4, whose kernels take as long; rows of 16 x 4096 quantised and multiplied with 4096 channels in 8 bits 17.5 / 9.5.
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/Context.h>
#include <ATen/PythonTorchFunctionTLS.h>
#include <ATen/core/dispatch/Dispatcher.h>
#include <ATen/hip/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/GradMode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <optional>
#include <string>

namespace {

// Dispatch keys above CUDA that plain tensors come with: nothing is done under them where no gradient is asked for, unless a
// program registers something there (has_observer).
const c10::DispatchKeySet kPassed =
    c10::DispatchKeySet(c10::DispatchKey::AutogradCUDA) | c10::DispatchKeySet(c10::DispatchKey::ADInplaceOrView) |
    c10::DispatchKeySet(c10::DispatchKey::BackendSelect);
const c10::DispatchKeySet kCuda(c10::DispatchKey::CUDA);

// The ops of torch_bind.cc (loaded by the package before this module).
template <typename Signature>
c10::TypedOperatorHandle<Signature> find_op(const char* name) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<Signature>();
}
using AttentionOp = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, double, bool);

// A program has registered something under the keys that are passed.
bool has_observer(const c10::OperatorHandle& op) {
  return op.hasKernelForAnyDispatchKey(kPassed) || op.hasKernelForDispatchKey(c10::DispatchKey::Autograd);
}

// Takes the tensors out of args[0 .. n); false unless every one is an ordinary torch.Tensor (no subclass) on a GPU that
// wants no gradient, and no mode, transform, autocast, tracer, profiler or observer of `op` is to see the call.
bool plain(const c10::OperatorHandle& op, PyObject* const* args, int n, at::Tensor* out) {
  c10::DispatchKeySet keys;
  for (int i = 0; i < n; ++i) {
    if (!THPVariable_CheckExact(args[i])) return false;
    const at::Tensor& t = THPVariable_Unpack(args[i]);
    if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided) return false;
    if (t.requires_grad() || t._fw_grad(0).defined()) return false;
    keys = keys | t.key_set();
    out[i] = t;   // (held while the interpreter is unlocked)
  }
  const auto local = c10::impl::tls_local_dispatch_key_set();
  keys = ((keys | local.included_) - local.excluded_) - (kPassed | kCuda);
  return keys.highestFunctionalityKey() == c10::DispatchKey::Undefined && !at::impl::torch_function_mode_enabled() &&
         !at::hasCallbacks() && !has_observer(op);
}

// ints only (a bool, a numpy number or a tensor is the dispatcher's business)
bool ints(PyObject* const* args, int n, int64_t* out) {
  for (int i = 0; i < n; ++i) {
    if (!PyLong_CheckExact(args[i])) return false;
    out[i] = PyLong_AsLongLong(args[i]);
    if (out[i] == -1 && PyErr_Occurred()) {
      PyErr_Clear();
      return false;
    }
  }
  return true;
}

struct NoGil {   // as the dispatcher: other threads run while a call is prepared
  PyThreadState* state = PyEval_SaveThread();
  ~NoGil() { PyEval_RestoreThread(state); }
};

// at::empty(shape, like.options()) for a tensor that `plain` has passed: the same allocator and tensor, without the dispatcher's way to
// them (0.3 us instead of 0.7).
at::Tensor empty_output(at::IntArrayRef shape, const at::Tensor& like) {
  const auto& context = at::globalContext();
  if (context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()) return at::empty(shape, like.options());
  return at::Tensor(at::detail::empty_cuda(shape, like.scalar_type(), like.device(), c10::nullopt));
}

at::Tensor empty_output(at::IntArrayRef shape, const at::Tensor& like, at::ScalarType type) {
  const auto& context = at::globalContext();
  if (context.deterministicAlgorithms() && context.deterministicFillUninitializedMemory()) return at::empty(shape, like.options().dtype(type));
  return at::Tensor(at::detail::empty_cuda(shape, type, like.device(), c10::nullopt));
}

// at::empty_like(like), which gives a dense tensor its strides, also the ones that address nothing (of extents of 1).
at::Tensor empty_output_like(const at::Tensor& like) {
  int64_t in_order = 1;
  for (int64_t i = like.dim() - 1; i >= 0; --i) {
    if (like.stride(i) != in_order) return at::empty_like(like);
    in_order *= like.size(i);
  }
  return empty_output(like.sizes(), like);
}

bool is_half_type(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

PyObject* gemm(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[3];
  int64_t i[5];
  using Op = void(const at::Tensor&, const at::Tensor&, at::Tensor&, int64_t, int64_t, int64_t, int64_t, int64_t);
  static const auto op = find_op<Op>("tilefusion::gemm");
  if (nargs != 8 || !plain(op, args, 3, t) || !ints(args + 3, 5, i)) Py_RETURN_FALSE;
  {
    NoGil unlocked;
    op.redispatch(kCuda, t[0], t[1], t[2], i[0], i[1], i[2], i[3], i[4]);
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* fused_two_gemms(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[4];
  int64_t i[4];
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, int64_t, int64_t, int64_t, int64_t);
  static const auto op = find_op<Op>("tilefusion::fused_two_gemms");
  if (nargs != 8 || !plain(op, args, 4, t) || !ints(args + 4, 4, i)) Py_RETURN_FALSE;
  for (const at::Tensor& x : t)   // (other types: the wrapper's own errors)
    if (!is_half_type(x) || x.scalar_type() != t[0].scalar_type()) Py_RETURN_FALSE;
  {
    NoGil unlocked;
    op.redispatch(kCuda, t[0], t[1], t[2], t[3], i[0], i[1], i[2], i[3]);
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

PyObject* scatter_nd(PyObject*, PyObject* const* args, Py_ssize_t nargs) {   // data, updates, indices
  HANDLE_TH_ERRORS
  at::Tensor t[3];
  static const auto op = find_op<void(const at::Tensor&, at::Tensor&, const at::Tensor&)>("tilefusion::scatter_nd");
  if (nargs != 3 || !plain(op, args, 3, t)) Py_RETURN_FALSE;
  {
    NoGil unlocked;
    op.redispatch(kCuda, t[0], t[1], t[2]);
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (query, key [.., D, Lkv], value, tile_length_q, tile_length_kv, tile_hidden_qk, tile_hidden_v, softmax_scale, causal)
// -> output, or None
PyObject* flash_attention(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[3];
  int64_t tile[4];
  static const auto op = find_op<AttentionOp>("tilefusion::flash_attention_fwd");
  static const auto op_kt = find_op<AttentionOp>("tilefusion::flash_attention_fwd_kt");
  if (nargs != 9 || !plain(op, args, 3, t) || has_observer(op_kt) || !ints(args + 3, 4, tile) || !PyFloat_CheckExact(args[7]) ||
      !PyBool_Check(args[8]))
    Py_RETURN_NONE;
  const at::Tensor &q = t[0], &k = t[1], &v = t[2];
  if (q.dim() < 2 || k.dim() < 2 || v.dim() < 2) Py_RETURN_NONE;
  const int64_t extent[4] = {q.size(-2), v.size(-2), q.size(-1), v.size(-1)};
  for (int i = 0; i < 4; ++i)
    if (tile[i] <= 0 || extent[i] % tile[i] != 0) Py_RETURN_NONE;
  const double scale = PyFloat_AS_DOUBLE(args[7]);
  const bool causal = args[8] == Py_True;
  at::Tensor out;
  {
    NoGil unlocked;
    at::DimVector shape(q.sizes());
    shape.back() = v.size(-1);
    out = empty_output(shape, q);
    // (a [D, Lkv] matrix in order is no [Lkv, D] one in order, unless one of the two is 1, or there is nothing in it)
    const bool kt = k.is_contiguous() && k.size(-1) > 1 && k.size(-2) > 1 && k.numel() > 0;
    if (kt)
      op_kt.redispatch(kCuda, q.contiguous(), k, v.contiguous(), out, scale, causal);
    else
      op.redispatch(kCuda, q.contiguous(), k.transpose(-1, -2).contiguous(), v.contiguous(), out, scale, causal);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (query, key, value, num_splits, softmax_scale or None) -> output, or None
PyObject* flash_decode(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[3];
  int64_t num_splits;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, int64_t, double);
  static const auto op = find_op<Op>("tilefusion::flash_decode");
  if (nargs != 5 || !plain(op, args, 3, t) || !ints(args + 3, 1, &num_splits)) Py_RETURN_NONE;
  if (args[4] != Py_None && !PyFloat_CheckExact(args[4])) Py_RETURN_NONE;
  const at::Tensor &q = t[0], &k = t[1], &v = t[2];
  if (q.dim() < 1 || q.size(-1) < 1) Py_RETURN_NONE;
  const double scale = args[4] == Py_None ? 1.0 / std::sqrt((double)q.size(-1)) : PyFloat_AS_DOUBLE(args[4]);
  at::Tensor out;
  {
    NoGil unlocked;
    out = empty_output_like(q);
    op.redispatch(kCuda, q.contiguous(), k.contiguous(), v.contiguous(), out, num_splits, scale);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// ---- products whose results do not leave as they are: matrices, contiguous as they come -------
bool matrices(const at::Tensor* t, int n) {
  for (int i = 0; i < n; ++i)
    if (t[i].dim() != 2 || !t[i].is_contiguous()) return false;
  return true;
}
bool vectors(const at::Tensor* t, int n) {
  for (int i = 0; i < n; ++i)
    if (t[i].dim() != 1 || !t[i].is_contiguous()) return false;
  return true;
}
bool text(PyObject* arg, c10::string_view* out) {
  Py_ssize_t n = 0;
  if (!PyUnicode_CheckExact(arg)) return false;
  const char* const p = PyUnicode_AsUTF8AndSize(arg, &n);
  if (p == nullptr) {
    PyErr_Clear();
    return false;
  }
  *out = c10::string_view(p, (size_t)n);
  return true;
}
PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
  PyObject* const out = PyTuple_New((Py_ssize_t)tensors.size());
  if (out == nullptr) return nullptr;
  Py_ssize_t i = 0;
  for (const at::Tensor& t : tensors) PyTuple_SET_ITEM(out, i++, THPVariable_Wrap(t));
  return out;
}

// (x) -> (q, scale), or None
PyObject* quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[1], q, scale;
  static const auto op = find_op<void(const at::Tensor&, at::Tensor&, at::Tensor&)>("tilefusion::quantize_rows");
  if (nargs != 1 || !plain(op, args, 1, t) || !matrices(t, 1)) Py_RETURN_NONE;
  {
    NoGil unlocked;
    q = empty_output(t[0].sizes(), t[0], at::kChar);
    scale = empty_output({t[0].size(0)}, t[0], at::kFloat);
    op.redispatch(kCuda, t[0], q, scale);
  }
  return tuple_of({q, scale});
  END_HANDLE_TH_ERRORS
}

// (A, B, scale_a, scale_b, C)
PyObject* gemm_int8(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[5];
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&);
  static const auto op = find_op<Op>("tilefusion::gemm_int8");
  if (nargs != 5 || !plain(op, args, 5, t) || !matrices(t, 2) || !vectors(t + 2, 2)) Py_RETURN_FALSE;
  {
    NoGil unlocked;
    op.redispatch(kCuda, t[0], t[1], t[2], t[3], t[4]);
  }
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// (x, w_gate, w_up, activation, keep) -> (h,) or (h, gate, up), or None
PyObject* gated_ffn(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[3], h;
  std::optional<at::Tensor> gate, up;
  c10::string_view activation;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, c10::string_view, at::Tensor&, const std::optional<at::Tensor>&,
                  const std::optional<at::Tensor>&);
  static const auto op = find_op<Op>("tilefusion::gated_ffn");
  if (nargs != 5 || !plain(op, args, 3, t) || !matrices(t, 3) || !text(args[3], &activation) || !PyBool_Check(args[4])) Py_RETURN_NONE;
  if (t[0].size(1) != t[1].size(1) || t[0].size(1) == 0) Py_RETURN_NONE;   // (the wrapper's own errors)
  const bool keep = args[4] == Py_True;
  {
    NoGil unlocked;
    const int64_t shape[2] = {t[0].size(0), t[1].size(0)};
    h = empty_output(shape, t[0]);
    if (keep) {
      gate = empty_output(shape, t[0]);
      up = empty_output(shape, t[0]);
    }
    op.redispatch(kCuda, t[0], t[1], t[2], activation, h, gate, up);
  }
  return keep ? tuple_of({h, *gate, *up}) : tuple_of({h});
  END_HANDLE_TH_ERRORS
}

// (hidden, weight, target, ignore_index) -> (loss, lse), or None
PyObject* linear_cross_entropy(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[3], loss, lse;
  int64_t ignore_index;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, at::Tensor&, at::Tensor&);
  static const auto op = find_op<Op>("tilefusion::linear_cross_entropy");
  if (nargs != 4 || !plain(op, args, 3, t) || !matrices(t, 2) || !vectors(t + 2, 1) || !ints(args + 3, 1, &ignore_index)) Py_RETURN_NONE;
  if (t[0].size(1) != t[1].size(1) || t[0].size(1) == 0 || t[2].size(0) != t[0].size(0)) Py_RETURN_NONE;
  {
    NoGil unlocked;
    loss = empty_output({t[0].size(0)}, t[0], at::kFloat);
    lse = empty_output({t[0].size(0)}, t[0], at::kFloat);
    op.redispatch(kCuda, t[0], t[1], t[2], ignore_index, loss, lse);
  }
  return tuple_of({loss, lse});
  END_HANDLE_TH_ERRORS
}

// (grad_h, x, w_gate, w_up, gate, up, activation) -> (grad_x, grad_w [2, F, K]), or None
PyObject* gated_ffn_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[6], grad_x, grad_w;
  c10::string_view activation;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, c10::string_view,
                  const std::optional<at::Tensor>&, const std::optional<at::Tensor>&);
  static const auto op = find_op<Op>("tilefusion::gated_ffn_backward");
  if (nargs != 7 || !plain(op, args, 6, t) || !matrices(t, 6) || !text(args[6], &activation)) Py_RETURN_NONE;
  const at::Tensor &x = t[1], &w = t[2];
  if (x.size(1) != w.size(1) || x.size(1) == 0) Py_RETURN_NONE;   // (the wrapper's own errors)
  for (int i : {0, 4, 5})
    if (t[i].size(1) != w.size(0)) Py_RETURN_NONE;
  {
    NoGil unlocked;
    grad_x = empty_output(x.sizes(), x);
    grad_w = empty_output({2 * w.size(0), w.size(1)}, x);
    op.redispatch(kCuda, t[0], x, w, t[3], t[4], t[5], activation, grad_x, grad_w);
    grad_w = grad_w.view({2, w.size(0), w.size(1)});
  }
  return tuple_of({grad_x, grad_w});
  END_HANDLE_TH_ERRORS
}

// (grad_loss, hidden, weight, target, lse, ignore_index) -> (grad_hidden, grad_weight), or None
PyObject* linear_cross_entropy_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[5], grad_hidden, grad_weight;
  int64_t ignore_index;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t, const std::optional<at::Tensor>&,
                  const std::optional<at::Tensor>&);
  static const auto op = find_op<Op>("tilefusion::linear_cross_entropy_backward");
  if (nargs != 6 || !plain(op, args, 5, t) || !vectors(t, 1) || !matrices(t + 1, 2) || !vectors(t + 3, 2) || !ints(args + 5, 1, &ignore_index))
    Py_RETURN_NONE;
  const at::Tensor &hidden = t[1], &weight = t[2];
  if (hidden.size(1) != weight.size(1) || hidden.size(1) == 0) Py_RETURN_NONE;
  for (int i : {0, 3, 4})
    if (t[i].size(0) != hidden.size(0)) Py_RETURN_NONE;
  {
    NoGil unlocked;
    grad_hidden = empty_output(hidden.sizes(), hidden);
    grad_weight = empty_output(weight.sizes(), weight);
    op.redispatch(kCuda, t[0], hidden, weight, t[3], t[4], ignore_index, grad_hidden, grad_weight);
  }
  return tuple_of({grad_hidden, grad_weight});
  END_HANDLE_TH_ERRORS
}

// ---- attention over packed sequences and paged caches: [n, heads, D], rows in one piece at 16-byte boundaries as they come ----
bool rows_in_place(const at::Tensor* t, int n) {
  for (int i = 0; i < n; ++i)
    if (t[i].dim() != 3 || t[i].stride(2) != 1 || t[i].stride(0) % 8 != 0 || t[i].stride(1) % 8 != 0 || reinterpret_cast<uintptr_t>(t[i].data_ptr()) % 16 != 0 ||
        !is_half_type(t[i]))
      return false;
  return true;
}
// ... and near enough to one another for attention over packed sequences (as the C entry points have it); what is not, the wrapper copies
bool within_reach(const at::Tensor& query, const at::Tensor& key, const at::Tensor& value) {
  constexpr int64_t kToken = 1 << 24;
  const int64_t group = key.size(1) > 0 ? query.size(1) / key.size(1) : 1;
  return query.stride(0) < kToken && key.stride(0) < kToken && value.stride(0) < kToken &&
         (group <= 1 || (query.stride(1) < (1ll << 31) && 33 * query.stride(0) + group * query.stride(1) < (1ll << 31) - query.size(2)));
}
bool scale_of(PyObject* arg, const at::Tensor& query, double* out) {
  if (arg != Py_None && !PyFloat_CheckExact(arg)) return false;
  *out = arg == Py_None ? 1.0 / std::sqrt((double)query.size(2)) : PyFloat_AS_DOUBLE(arg);
  return query.size(2) > 0;
}
// A tensor or None; false: something else, or a tensor that is not plain (as `plain` has it).
bool plain_or_none(const c10::OperatorHandle& op, PyObject* arg, std::optional<at::Tensor>* out) {
  if (arg == Py_None) return true;
  at::Tensor t[1];
  if (!plain(op, &arg, 1, t)) return false;
  *out = t[0];
  return true;
}

// (query, key_cache, value_cache, page_table, lengths, softmax_scale or None) -> output, or None
PyObject* flash_decode_paged(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[5], out;
  double scale;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, double, at::Tensor&);
  static const auto op = find_op<Op>("tilefusion::flash_decode_paged");
  if (nargs != 6 || !plain(op, args, 5, t) || !rows_in_place(t, 1) || !scale_of(args[5], t[0], &scale)) Py_RETURN_NONE;
  {
    NoGil unlocked;
    out = empty_output(t[0].sizes(), t[0]);
    op.redispatch(kCuda, t[0], t[1], t[2], t[3], t[4], scale, out);
  }
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// (query, key, value, cos, sin, key_cache, value_cache, page_table, lengths, offsets or None, interleaved, keep) -> (query,) or (query, key), or None
PyObject* append_paged_kv(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[9], query;
  std::optional<at::Tensor> offsets, key;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, at::Tensor&, const at::Tensor&,
                  const at::Tensor&, const std::optional<at::Tensor>&, bool, at::Tensor&, const std::optional<at::Tensor>&);
  static const auto op = find_op<Op>("tilefusion::append_paged_kv");
  if (nargs != 12 || !plain(op, args, 9, t) || !rows_in_place(t, 3) || !t[3].is_contiguous() || !t[4].is_contiguous() ||
      !plain_or_none(op, args[9], &offsets) || !PyBool_Check(args[10]) || !PyBool_Check(args[11]))
    Py_RETURN_NONE;
  const bool keep = args[11] == Py_True;
  {
    NoGil unlocked;
    query = empty_output(t[0].sizes(), t[0]);
    if (keep) key = empty_output(t[1].sizes(), t[1]);
    op.redispatch(kCuda, t[0], t[1], t[2], t[3], t[4], t[5], t[6], t[7], t[8], offsets, args[10] == Py_True, query, key);
  }
  return keep ? tuple_of({query, *key}) : tuple_of({query});
  END_HANDLE_TH_ERRORS
}

// (query, key, value, offsets, kv_offsets or None, softmax_scale or None, causal, keep) -> (out,) or (out, lse), or None
PyObject* flash_attention_packed(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[4], out;
  std::optional<at::Tensor> kv_offsets, lse;
  double scale;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&, double, bool, at::Tensor&,
                  const std::optional<at::Tensor>&);
  static const auto op = find_op<Op>("tilefusion::flash_attention_packed");
  if (nargs != 8 || !plain(op, args, 4, t) || !rows_in_place(t, 3) || !within_reach(t[0], t[1], t[2]) || !plain_or_none(op, args[4], &kv_offsets) ||
      !scale_of(args[5], t[0], &scale) || !PyBool_Check(args[6]) || !PyBool_Check(args[7]))
    Py_RETURN_NONE;
  const bool keep = args[7] == Py_True;
  {
    NoGil unlocked;
    out = empty_output(t[0].sizes(), t[0]);
    if (keep) lse = empty_output({t[0].size(1), t[0].size(0)}, t[0], at::kFloat);
    op.redispatch(kCuda, t[0], t[1], t[2], t[3], kv_offsets, scale, args[6] == Py_True, out, lse);
  }
  return keep ? tuple_of({out, *lse}) : tuple_of({out});
  END_HANDLE_TH_ERRORS
}

// (grad_out, query, key, value, out, lse, offsets, kv_offsets or None, softmax_scale or None, causal) -> (grad_query, grad_key, grad_value), or None
PyObject* flash_attention_packed_backward(PyObject*, PyObject* const* args, Py_ssize_t nargs) {
  HANDLE_TH_ERRORS
  at::Tensor t[7];
  std::optional<at::Tensor> kv_offsets, grads[3];
  double scale;
  using Op = void(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                  const std::optional<at::Tensor>&, double, bool, const std::optional<at::Tensor>&, const std::optional<at::Tensor>&,
                  const std::optional<at::Tensor>&);
  static const auto op = find_op<Op>("tilefusion::flash_attention_packed_backward");
  if (nargs != 10 || !plain(op, args, 7, t) || !rows_in_place(t, 5) || !within_reach(t[1], t[2], t[3]) || !t[0].is_contiguous() || !t[4].is_contiguous() || !t[5].is_contiguous() ||
      !plain_or_none(op, args[7], &kv_offsets) || !scale_of(args[8], t[1], &scale) || !PyBool_Check(args[9]))
    Py_RETURN_NONE;
  {
    NoGil unlocked;
    for (int i = 0; i < 3; ++i) grads[i] = empty_output(t[1 + i].sizes(), t[1 + i]);
    op.redispatch(kCuda, t[0], t[1], t[2], t[3], t[4], t[5], t[6], kv_offsets, scale, args[9] == Py_True, grads[0], grads[1], grads[2]);
  }
  return tuple_of({*grads[0], *grads[1], *grads[2]});
  END_HANDLE_TH_ERRORS
}

template <PyObject* (*kFunction)(PyObject*, PyObject* const*, Py_ssize_t)>
constexpr PyMethodDef method(const char* name) {
  return {name, (PyCFunction)(void (*)(void))kFunction, METH_FASTCALL, nullptr};
}
PyMethodDef methods[] = {method<gemm>("gemm"), method<fused_two_gemms>("fused_two_gemms"), method<scatter_nd>("scatter_nd"),
                         method<flash_attention>("flash_attention"), method<flash_decode>("flash_decode"),
                         method<quantize_rows>("quantize_rows"), method<gemm_int8>("gemm_int8"), method<gated_ffn>("gated_ffn"),
                         method<gated_ffn_backward>("gated_ffn_backward"), method<linear_cross_entropy>("linear_cross_entropy"),
                         method<linear_cross_entropy_backward>("linear_cross_entropy_backward"),
                         method<flash_decode_paged>("flash_decode_paged"), method<append_paged_kv>("append_paged_kv"),
                         method<flash_attention_packed>("flash_attention_packed"),
                         method<flash_attention_packed_backward>("flash_attention_packed_backward"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_direct", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__direct() { return PyModule_Create(&module); }
