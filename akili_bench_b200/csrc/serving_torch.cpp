// serving_torch.cpp — the torch side of include/akili_serving.h: a CPython
// module that checks tensors, makes the outputs and calls libakili.so.
//
// The operators of a decode step run for a few microseconds, so the front end
// has to cost less than that: checking and filling the argument blocks from
// Python took 15 to 25 us a call; here a call takes the host 3.5 to 5 us, the
// launch included (tree_attention, with its tensor maps and two launches, 8.5).
// akili_bench_b200/serving.py
// holds the documented functions; each passes its arguments on by position.
// Wrong types, shapes and devices raise TypeError or ValueError; a refusal of
// the C entry raises abi.AkiliError.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Stream.h>
#include <torch/csrc/autograd/VariableTypeUtils.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <limits>
#include <memory>
#include <optional>
#include <string>

#include "../../include/akili_serving.h"

namespace {

// Thrown with a Python exception set.
struct PyError {};

[[noreturn]] void fail(PyObject* type, const std::string& what) {
  PyErr_SetString(type, what.c_str());
  throw PyError{};
}

// Sets module.cls(*args); takes `args`.
void raise(const char* module, const char* cls, PyObject* args) {
  PyObject* m = args ? PyImport_ImportModule(module) : nullptr;
  PyObject* c = m ? PyObject_GetAttrString(m, cls) : nullptr;
  if (c) PyErr_SetObject(c, args);
  Py_XDECREF(c);
  Py_XDECREF(m);
  Py_XDECREF(args);
}

[[noreturn]] void refuse(const char* op, int code) {
  raise("akili_bench_b200.abi", "AkiliError", Py_BuildValue("(si)", op, code));
  throw PyError{};
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) fail(PyExc_TypeError, std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw PyError{};
  return v;
}

uint32_t size32(int64_t v, const char* name) {
  if (v < 0 || v > 0xffffffffll) fail(PyExc_ValueError, std::string(name) + " does not fit 32 bits");
  return static_cast<uint32_t>(v);
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw PyError{};
  return v;
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw PyError{};
  return v != 0;
}

uint64_t addr(const at::Tensor& t) { return reinterpret_cast<uint64_t>(t.const_data_ptr()); }

std::string text(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

uint32_t element(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return AKILI_DTYPE_F32;
    case at::kHalf: return AKILI_DTYPE_F16;
    case at::kBFloat16: return AKILI_DTYPE_BF16;
    default: fail(PyExc_TypeError, std::string("unsupported dtype ") + at::toString(t.scalar_type()));
  }
}

// A CUDA tensor on the current device.
void on_device(const at::Tensor& t) {
  if (!t.is_cuda() || t.get_device() != c10::cuda::current_device())
    fail(PyExc_ValueError, "serving ops take CUDA tensors on the current device");
}

void rank_is(const at::Tensor& t, int64_t rank, const char* layout) {
  if (t.dim() != rank) fail(PyExc_ValueError, layout);
}

// Values of the type and on the device of `first`, last axis contiguous.
void values(const at::Tensor& first, const at::Tensor& t, const char* name) {
  if (t.scalar_type() != first.scalar_type() || t.device() != first.device())
    fail(PyExc_ValueError, std::string(name) + " must have the type and the device of the first tensor");
  if (t.dim() < 1 || (t.stride(-1) != 1 && t.size(-1) != 1))
    fail(PyExc_ValueError, "the last axis of " + std::string(name) + " must be contiguous");
}

void shape_is(const at::Tensor& t, std::initializer_list<int64_t> want, const char* name) {
  const at::IntArrayRef w(want);
  bool ok = t.dim() == static_cast<int64_t>(w.size());
  for (size_t i = 0; ok && i < w.size(); ++i) ok = w[i] < 0 || t.size(i) == w[i];
  if (!ok) fail(PyExc_ValueError, std::string(name) + " has shape " + text(t.sizes()) + ", expected " + text(w) + " (-1: any)");
}

// An index tensor; rows may be strided, the last axis not.
uint64_t index(const at::Tensor& t, const at::Tensor& first, std::initializer_list<int64_t> want, const char* name,
               at::ScalarType type = at::kInt) {
  if (t.scalar_type() != type || t.device() != first.device())
    fail(PyExc_ValueError, std::string(name) + " must be " + at::toString(type) + " on the device of the first tensor");
  shape_is(t, want, name);
  if (t.numel() && t.stride(-1) != 1 && t.size(-1) != 1)
    fail(PyExc_ValueError, "the last axis of " + std::string(name) + " must be contiguous");
  return addr(t);
}

// The stream of a call.  What the call allocates comes from that stream's
// memory: a block that the allocator takes back from the caller's current
// stream may still be read or written by what is queued there, which this
// stream does not wait for.  The caller goes on to use the result on its own
// stream, which the allocator is told.
class CallStream {
 public:
  explicit CallStream(PyObject* o) : caller_(c10::cuda::getCurrentCUDAStream()), handle_(caller_.stream()) {
    if (o == Py_None) return;
    const c10::cuda::CUDAStream s = given(o, caller_.device_index());
    handle_ = s.stream();
    if (handle_ != caller_.stream()) guard_.emplace(s);
  }
  bool capturing() const {  // (the call's stream is the current one)
    return c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None;
  }
  akili_stream_t handle() const { return reinterpret_cast<akili_stream_t>(handle_); }
  at::Tensor empty(at::IntArrayRef sizes, const at::TensorOptions& options) const {
    at::Tensor t = at::empty(sizes, options);
    if (guard_) t.record_stream(caller_);
    return t;
  }

 private:
  static c10::cuda::CUDAStream given(PyObject* o, c10::DeviceIndex device) {
    if (THPStream_Check(o)) {
      const auto* s = reinterpret_cast<const THPStream*>(o);
      if (s->device_type != static_cast<int64_t>(c10::DeviceType::CUDA) || s->device_index != device)
        fail(PyExc_ValueError, "stream must be a CUDA stream of the current device");
      return c10::cuda::CUDAStream::unpack3(s->stream_id, device, c10::DeviceType::CUDA);
    }
    PyObject* h = PyObject_GetAttrString(o, "cuda_stream");
    if (!h) throw PyError{};
    void* p = PyLong_AsVoidPtr(h);
    Py_DECREF(h);
    if (!p && PyErr_Occurred()) throw PyError{};
    return c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(p), device);
  }

  c10::cuda::CUDAStream caller_;
  cudaStream_t handle_;
  std::optional<c10::cuda::CUDAStreamGuard> guard_;
};

template <size_t n>
void strides(int64_t (&to)[n], const at::Tensor& t, int64_t from = 0) {
  for (size_t i = 0; i < n; ++i) to[i] = t.stride(from + static_cast<int64_t>(i));
}

// A tensor that was given and is written: a backward pass that saved its old
// values has to notice.
void written(const at::Tensor& t) {
  if (!t.is_inference()) torch::autograd::increment_version(t);
}

// The operators have no autograd formulas.  Where an input is part of a graph
// the results are too, behind a node that raises in a backward pass: they
// would look like constants otherwise.  Made before the launch, which a
// refusal (a leaf written in place, say) must not follow.
class Untaught {
 public:
  Untaught(const char* name, std::initializer_list<const at::Tensor*> inputs,
           std::initializer_list<PyObject*> given = {}) {
    if (!at::GradMode::is_enabled()) return;
    torch::autograd::edge_list edges;
    for (const at::Tensor* t : inputs)
      if (t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
    if (edges.empty()) return;
    for (PyObject* o : given)
      if (o != Py_None) torch::autograd::check_inplace(THPVariable_Unpack(o), true);
    node_ = std::make_shared<torch::autograd::NotImplemented>(name, std::move(edges));
  }
  // A result, in a tensor that was `given` or a new one.
  void result(const at::Tensor& t, PyObject* given = Py_None) const {
    if (given != Py_None) written(t);
    if (!node_) return;
    const torch::autograd::Edge edge(node_, node_->add_input_metadata(t));
    if (given != Py_None) torch::autograd::impl::rebase_history(t, edge);
    else torch::autograd::impl::set_gradient_edge(t, edge);
  }

 private:
  std::shared_ptr<torch::autograd::Node> node_;
};

constexpr const char* kRopeGradient = "ops.rope (it is ops.rope of the gradients with inverse=True)";

at::Tensor given_or_like(PyObject* o, const at::Tensor& like, const char* name, const CallStream& st) {
  if (o == Py_None) return st.empty(like.sizes(), like.options());
  const at::Tensor& t = tensor(o, name);
  values(like, t, name);
  if (t.sizes() != like.sizes())
    fail(PyExc_ValueError, std::string(name) + " has shape " + text(t.sizes()) + ", expected " + text(like.sizes()));
  return t;
}

void rope_common(akili_rope_arg_t& a, const at::Tensor& q, const at::Tensor& k, const at::Tensor& pos,
                 const at::Tensor& table, bool interleaved, bool inverse) {
  on_device(q);
  values(q, q, "q");
  values(q, k, "k");
  if (q.dim() != 3 || k.dim() != 3 || q.size(0) != k.size(0) || q.size(2) != k.size(2))
    fail(PyExc_ValueError, "q and k are [tokens, heads, head_dim] with the same tokens and head_dim");
  if (table.dim() != 2 || table.scalar_type() != at::kFloat || !table.is_contiguous() || table.device() != q.device())
    fail(PyExc_ValueError, "table is a contiguous fp32 [max_positions, rot_dim] tensor on the device of q");
  a.dtype = element(q);
  a.flags = (interleaved ? AKILI_ROPE_INTERLEAVED : 0u) | (inverse ? AKILI_ROPE_INVERSE : 0u);
  a.tokens = size32(q.size(0), "tokens");
  a.q_heads = size32(q.size(1), "q_heads");
  a.k_heads = size32(k.size(1), "k_heads");
  a.head_dim = size32(q.size(2), "head_dim");
  a.rot_dim = size32(table.size(1), "rot_dim");
  a.max_positions = size32(table.size(0), "max_positions");
  a.q_addr = addr(q);
  a.k_addr = addr(k);
  a.positions_addr = index(pos, q, {q.size(0)}, "positions");
  a.table_addr = addr(table);
  strides(a.q_stride, q);
  strides(a.k_stride, k);
}

// (q, k, positions, table, interleaved, inverse, q_out, k_out, stream)
PyObject* rope(PyObject* const* v) {
  akili_rope_arg_t a = {};
  const at::Tensor &q = tensor(v[0], "q"), &k = tensor(v[1], "k");
  rope_common(a, q, k, tensor(v[2], "positions"), tensor(v[3], "table"), truth(v[4]), truth(v[5]));
  const CallStream st(v[8]);
  const at::Tensor q_out = given_or_like(v[6], q, "q_out", st), k_out = given_or_like(v[7], k, "k_out", st);
  a.q_out_addr = addr(q_out);
  a.k_out_addr = addr(k_out);
  strides(a.q_out_stride, q_out);
  strides(a.k_out_stride, k_out);
  const Untaught history(kRopeGradient, {&q, &k}, {v[6], v[7]});
  if (const int rc = akili_rope(&a, st.handle())) refuse("rope", rc);
  history.result(q_out, v[6]);
  history.result(k_out, v[7]);
  return Py_BuildValue("(NN)", THPVariable_Wrap(q_out), THPVariable_Wrap(k_out));
}

// (q, k, v, positions, table, slots, k_pages, v_pages, interleaved, q_out, k_out, stream)
PyObject* rope_append(PyObject* const* v) {
  akili_rope_arg_t a = {};
  const at::Tensor &q = tensor(v[0], "q"), &k = tensor(v[1], "k"), &val = tensor(v[2], "v"),
                   &kp = tensor(v[6], "k_pages"), &vp = tensor(v[7], "v_pages");
  rope_common(a, q, k, tensor(v[3], "positions"), tensor(v[4], "table"), truth(v[8]), false);
  values(q, val, "v");
  values(q, kp, "k_pages");
  values(q, vp, "v_pages");
  shape_is(val, {k.size(0), k.size(1), k.size(2)}, "v");
  shape_is(kp, {-1, -1, k.size(1), k.size(2)}, "k_pages");
  shape_is(vp, {kp.size(0), kp.size(1), k.size(1), k.size(2)}, "v_pages");
  a.slots_addr = index(tensor(v[5], "slots"), q, {q.size(0)}, "slots", at::kLong);
  const CallStream st(v[11]);
  const at::Tensor q_out = given_or_like(v[9], q, "q_out", st);
  a.q_out_addr = addr(q_out);
  strides(a.q_out_stride, q_out);
  a.v_addr = addr(val);
  a.k_pages_addr = addr(kp);
  a.v_pages_addr = addr(vp);
  a.num_pages = size32(kp.size(0), "num_pages");
  a.page_size = size32(kp.size(1), "page_size");
  strides(a.v_stride, val);
  strides(a.k_page_stride, kp);
  strides(a.v_page_stride, vp);
  if (v[10] != Py_None) {
    const at::Tensor& k_out = tensor(v[10], "k_out");
    values(q, k_out, "k_out");
    shape_is(k_out, {k.size(0), k.size(1), k.size(2)}, "k_out");
    a.k_out_addr = addr(k_out);
    strides(a.k_out_stride, k_out);
  }
  const Untaught history("ops.rope_append", {&q, &k, &val}, {v[9], v[10]});
  if (const int rc = akili_rope_append(&a, st.handle())) refuse("rope_append", rc);
  history.result(q_out, v[9]);
  if (v[10] != Py_None) history.result(THPVariable_Unpack(v[10]), v[10]);
  // (a cache that carried history would hold every step's graph)
  written(kp);
  written(vp);
  return THPVariable_Wrap(q_out);
}

// (max_positions, rot_dim, scaling, base, factor, original_positions, low, high, amplitude, stream)
PyObject* rope_table(PyObject* const* v) {
  akili_rope_table_arg_t a = {};
  const CallStream st(v[9]);
  const at::Tensor t = st.empty({integer(v[0]), integer(v[1])},
                                at::TensorOptions(at::kFloat).device(at::kCUDA, c10::cuda::current_device()));
  a.max_positions = size32(t.size(0), "max_positions");
  a.rot_dim = size32(t.size(1), "rot_dim");
  a.scaling = static_cast<uint32_t>(integer(v[2]));
  a.base = number(v[3]);
  a.factor = number(v[4]);
  a.original_positions = number(v[5]);
  a.low = number(v[6]);
  a.high = number(v[7]);
  a.amplitude = number(v[8]);
  a.table_addr = addr(t);
  if (const int rc = akili_rope_table(&a, st.handle())) refuse("rope_table", rc);
  return THPVariable_Wrap(t);
}

// 0 stands for the default in the C entries.  A given scale that is 0 in fp32
// becomes the smallest positive one, which weighs all visible keys alike: it
// moves a weight by less than 2^-20 for any finite score.
float scale_of(PyObject* o) {
  if (o == Py_None) return 0.0f;
  const float s = static_cast<float>(number(o));
  return s != 0.0f ? s : std::numeric_limits<float>::denorm_min();
}

PyObject* with_lse(const at::Tensor& out, const at::Tensor& lse) {
  if (!lse.defined()) return THPVariable_Wrap(out);
  return Py_BuildValue("(NN)", THPVariable_Wrap(out), THPVariable_Wrap(lse));
}

// (q, k, v, cu_q, cu_k, softmax_scale, causal, out, return_lse, stream)
PyObject* prompt_attention(PyObject* const* v) {
  akili_prompt_attention_arg_t a = {};
  const at::Tensor &q = tensor(v[0], "q"), &k = tensor(v[1], "k"), &val = tensor(v[2], "v"), &cu_q = tensor(v[3], "cu_q");
  const at::Tensor& cu_k = v[4] == Py_None ? cu_q : tensor(v[4], "cu_k");
  on_device(q);
  rank_is(q, 3, "q is [total_q, q_heads, head_dim]");
  values(q, q, "q");
  values(q, k, "k");
  values(q, val, "v");
  rank_is(k, 3, "k and v are [total_k, kv_heads, head_dim]");
  shape_is(k, {-1, -1, q.size(2)}, "k");
  shape_is(val, {k.size(0), k.size(1), k.size(2)}, "v");
  a.cu_q_addr = index(cu_q, q, {-1}, "cu_q");
  a.cu_k_addr = index(cu_k, q, {cu_q.size(0)}, "cu_k");
  if (cu_q.size(0) == 0) fail(PyExc_ValueError, "cu_q has batch + 1 entries");
  const CallStream st(v[9]);
  const at::Tensor out = given_or_like(v[7], q, "out", st);
  at::Tensor lse;
  if (truth(v[8])) lse = st.empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  a.dtype = element(q);
  a.q_heads = size32(q.size(1), "q_heads");
  a.kv_heads = size32(k.size(1), "kv_heads");
  a.head_dim = size32(q.size(2), "head_dim");
  a.batch = size32(cu_q.size(0) - 1, "batch");
  a.total_q = size32(q.size(0), "total_q");
  a.total_k = size32(k.size(0), "total_k");
  a.causal = truth(v[6]);
  a.softmax_scale = scale_of(v[5]);
  a.q_addr = addr(q);
  a.k_addr = addr(k);
  a.v_addr = addr(val);
  a.o_addr = addr(out);
  a.lse_addr = lse.defined() ? addr(lse) : 0;
  strides(a.q_stride, q);
  strides(a.k_stride, k);
  strides(a.v_stride, val);
  strides(a.o_stride, out);
  const Untaught history("ops.prompt_attention", {&q, &k, &val}, {v[7]});
  if (const int rc = akili_prompt_attention(&a, st.handle())) refuse("prompt_attention", rc);
  history.result(out, v[7]);
  if (lse.defined()) history.result(lse);
  return with_lse(out, lse);
}

// (parents, cu_q, words, stream)
PyObject* tree_mask(PyObject* const* v) {
  akili_tree_mask_arg_t a = {};
  const at::Tensor &parents = tensor(v[0], "parents"), &cu_q = tensor(v[1], "cu_q");
  on_device(parents);
  a.parents_addr = index(parents, parents, {-1}, "parents");
  a.cu_q_addr = index(cu_q, parents, {-1}, "cu_q");
  if (cu_q.size(0) == 0) fail(PyExc_ValueError, "cu_q has batch + 1 entries");
  a.mask_words = size32(integer(v[2]), "mask_words");
  a.batch = size32(cu_q.size(0) - 1, "batch");
  a.total_q = size32(parents.size(0), "total_q");
  const CallStream st(v[3]);
  const at::Tensor mask = st.empty({parents.size(0), static_cast<int64_t>(a.mask_words)}, parents.options());
  a.mask_addr = addr(mask);
  if (const int rc = akili_tree_mask(&a, st.handle())) refuse("tree_mask", rc);
  return THPVariable_Wrap(mask);
}

void tree_common(akili_tree_attention_arg_t& a, const at::Tensor& q, const at::Tensor& kp, const at::Tensor& table,
                 const at::Tensor& lens) {
  on_device(q);
  rank_is(q, 3, "q is [total_q, q_heads, head_dim]");
  values(q, q, "q");
  values(q, kp, "k_pages");
  shape_is(kp, {-1, -1, -1, q.size(2)}, "k_pages");
  a.context_lens_addr = index(lens, q, {-1}, "context_lens");
  a.page_table_addr = index(table, q, {lens.size(0), -1}, "page_table");
  a.dtype = element(q);
  a.q_heads = size32(q.size(1), "q_heads");
  a.kv_heads = size32(kp.size(2), "kv_heads");
  a.head_dim = size32(q.size(2), "head_dim");
  a.batch = size32(lens.size(0), "batch");
  a.total_q = size32(q.size(0), "total_q");
  a.num_pages = size32(kp.size(0), "num_pages");
  a.page_size = size32(kp.size(1), "page_size");
  a.max_pages = size32(table.size(1), "max_pages");
  a.page_table_stride = table.stride(0);
}

// (q, k_pages, v_pages, page_table, context_lens, cu_q, mask, softmax_scale, out, return_lse, workspace, stream)
PyObject* tree_attention(PyObject* const* v) {
  akili_tree_attention_arg_t a = {};
  const at::Tensor &q = tensor(v[0], "q"), &kp = tensor(v[1], "k_pages"), &vp = tensor(v[2], "v_pages");
  tree_common(a, q, kp, tensor(v[3], "page_table"), tensor(v[4], "context_lens"));
  values(q, vp, "v_pages");
  shape_is(vp, {kp.size(0), kp.size(1), kp.size(2), kp.size(3)}, "v_pages");
  a.cu_q_addr = index(tensor(v[5], "cu_q"), q, {static_cast<int64_t>(a.batch) + 1}, "cu_q");
  if (v[6] != Py_None) {
    const at::Tensor& mask = tensor(v[6], "mask");
    a.mask_addr = index(mask, q, {q.size(0), -1}, "mask");
    // (a mask of no words has no address, which would be no mask at all)
    if (mask.size(1) == 0 && q.size(0) > 0) fail(PyExc_ValueError, "mask rows have at least one word");
    a.mask_words = size32(mask.size(1), "mask_words");
    a.mask_stride = mask.stride(0);
  }
  const CallStream st(v[11]);
  const at::Tensor out = given_or_like(v[8], q, "out", st);
  at::Tensor lse;
  if (truth(v[9])) lse = st.empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat));
  at::Tensor ws;
  if (v[10] != Py_None) {
    ws = tensor(v[10], "workspace");
    if (ws.device() != q.device() || !ws.is_contiguous())
      fail(PyExc_ValueError, "workspace is a contiguous tensor on the device of q");
  } else if (st.capturing()) {
    // A graph's own memory: the stream's scratch belongs to its eager calls,
    // which a replay on another stream would not be ordered with.
    uint64_t n = 0;
    if (const int rc = akili_tree_attention_workspace(&a, &n)) refuse("tree_attention", rc);
    ws = st.empty({static_cast<int64_t>(n)}, q.options().dtype(at::kByte));
  }
  if (ws.defined()) {
    a.workspace = addr(ws);
    a.workspace_bytes = static_cast<uint64_t>(ws.nbytes());
  }
  a.softmax_scale = scale_of(v[7]);
  a.q_addr = addr(q);
  a.k_pages_addr = addr(kp);
  a.v_pages_addr = addr(vp);
  a.o_addr = addr(out);
  a.lse_addr = lse.defined() ? addr(lse) : 0;
  strides(a.q_stride, q);
  strides(a.o_stride, out);
  strides(a.k_page_stride, kp);
  strides(a.v_page_stride, vp);
  const Untaught history("ops.tree_attention", {&q, &kp, &vp}, {v[8]});
  if (const int rc = akili_tree_attention(&a, st.handle())) refuse("tree_attention", rc);
  history.result(out, v[8]);
  if (lse.defined()) history.result(lse);
  return with_lse(out, lse);
}

// (q, k_pages, page_table, context_lens)
PyObject* tree_attention_workspace(PyObject* const* v) {
  akili_tree_attention_arg_t a = {};
  tree_common(a, tensor(v[0], "q"), tensor(v[1], "k_pages"), tensor(v[2], "page_table"), tensor(v[3], "context_lens"));
  uint64_t n = 0;
  if (const int rc = akili_tree_attention_workspace(&a, &n)) refuse("tree_attention_workspace", rc);
  return PyLong_FromUnsignedLongLong(n);
}

// (k_pages, v_pages, page_table, context_lens, accepted, n_accepted, new_lens, stream); pages with or without layers
PyObject* cache_accept(PyObject* const* v) {
  akili_cache_accept_arg_t a = {};
  const at::Tensor &kp = tensor(v[0], "k_pages"), &vp = tensor(v[1], "v_pages"), &table = tensor(v[2], "page_table"),
                   &lens = tensor(v[3], "context_lens"), &acc = tensor(v[4], "accepted");
  on_device(kp);
  values(kp, kp, "k_pages");
  values(kp, vp, "v_pages");
  const int64_t lead = kp.dim() - 4;
  if ((lead != 0 && lead != 1) || vp.sizes() != kp.sizes())
    fail(PyExc_ValueError, "k_pages and v_pages are [layers, num_pages, page_size, kv_heads, head_dim]");
  a.context_lens_addr = index(lens, kp, {-1}, "context_lens");
  a.page_table_addr = index(table, kp, {lens.size(0), -1}, "page_table");
  a.accepted_addr = index(acc, kp, {lens.size(0), -1}, "accepted");
  a.n_accepted_addr = index(tensor(v[5], "n_accepted"), kp, {lens.size(0)}, "n_accepted");
  const CallStream st(v[7]);
  const at::Tensor out = v[6] == Py_None ? st.empty(lens.sizes(), lens.options()) : tensor(v[6], "new_lens");
  a.new_lens_addr = index(out, kp, {lens.size(0)}, "new_lens");
  a.elem_bytes = static_cast<uint32_t>(kp.element_size());
  a.layers = lead ? size32(kp.size(0), "layers") : 1;
  a.batch = size32(lens.size(0), "batch");
  a.num_pages = size32(kp.size(lead), "num_pages");
  a.page_size = size32(kp.size(lead + 1), "page_size");
  a.kv_heads = size32(kp.size(lead + 2), "kv_heads");
  a.head_dim = size32(kp.size(lead + 3), "head_dim");
  a.max_pages = size32(table.size(1), "max_pages");
  a.max_accepted = size32(acc.size(1), "max_accepted");
  a.k_pages_addr = addr(kp);
  a.v_pages_addr = addr(vp);
  a.page_table_stride = table.stride(0);
  a.accepted_stride = acc.stride(0);
  for (int64_t i = 0; i < 4; ++i) {
    a.k_page_stride[i] = i - 1 + lead < 0 ? 0 : kp.stride(i - 1 + lead);
    a.v_page_stride[i] = i - 1 + lead < 0 ? 0 : vp.stride(i - 1 + lead);
  }
  if (const int rc = akili_cache_accept(&a, st.handle())) refuse("cache_accept", rc);
  written(kp);
  written(vp);
  if (v[6] != Py_None) written(out);
  return THPVariable_Wrap(out);
}

// Argument count, and exceptions of C++ and torch as Python's.
template <PyObject* (*f)(PyObject* const*), Py_ssize_t n>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != n) {
    PyErr_Format(PyExc_TypeError, "%zd arguments expected, got %zd", n, count);
    return nullptr;
  }
  try {
    return f(args);
  } catch (const PyError&) {
    return nullptr;
  } catch (const c10::OutOfMemoryError& e) {
    raise("torch", "OutOfMemoryError", Py_BuildValue("(s)", e.what_without_backtrace()));
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

template <PyObject* (*f)(PyObject* const*), Py_ssize_t n>
PyMethodDef method(const char* name) {
  return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&entry<f, n>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<rope, 9>("rope"),
                         method<rope_append, 12>("rope_append"),
                         method<rope_table, 10>("rope_table"),
                         method<prompt_attention, 10>("prompt_attention"),
                         method<tree_mask, 4>("tree_mask"),
                         method<tree_attention, 12>("tree_attention"),
                         method<tree_attention_workspace, 4>("tree_attention_workspace"),
                         method<cache_accept, 8>("cache_accept"),
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_serving", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__serving(void) { return PyModule_Create(&module); }
