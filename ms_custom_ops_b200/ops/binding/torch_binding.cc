// Python binding of the operators that a serving loop calls for every layer of every step (rope_and_cache,
// chunk_attention) or step (verify_draft_tokens): torch tensors to operator descriptors without a Python object per
// field.  The same work through ctypes took 20 us per call on the host, several times what the small kernels take.
//
// Each function takes its operator's arguments in registration order and returns the operator's result, or the status
// code of the operator layer as an int (the caller raises what belongs to it).
#include <ATen/ATen.h>
#include <Python.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <limits>
#include <string>

#include "ms_custom_ops_c.h"

namespace {

[[noreturn]] void TypeError(const std::string &msg) {
  PyErr_SetString(PyExc_TypeError, msg.c_str());
  throw python_error();
}

// Descriptors of one call.  Every device tensor has to be on the first one's device.
class Call {
 public:
  Call(PyObject *first, const char *name) {
    if (!THPVariable_Check(first)) TypeError(std::string(name) + " must be a torch CUDA tensor");
    const at::Tensor &t = THPVariable_Unpack(first);
    if (!t.is_cuda()) throw std::runtime_error(std::string(name) + " must be a CUDA tensor (only lengths are read on the host)");
    device_ = t.get_device();
  }
  c10::DeviceIndex device() const { return static_cast<c10::DeviceIndex>(device_); }

  MsTensorDesc *Add(const at::Tensor &t, const char *name, bool host) {
    const bool cuda = t.is_cuda();
    if (!cuda && !host && t.numel() != 0)
      throw std::runtime_error(std::string(name) + " must be a CUDA tensor (only lengths are read on the host)");
    if (cuda && t.get_device() != device_)
      throw std::runtime_error(std::string("all tensors must be on one device, but ") + name + " is on cuda:" +
                               std::to_string(t.get_device()) + " instead of cuda:" + std::to_string(device_));
    if (t.dim() > MS_MAX_DIMS) TORCH_CHECK_VALUE(false, "tensors of more than 8 dimensions are not supported");
    MsTensorDesc *d = &desc_[used_++];
    d->data = t.data_ptr();
    switch (t.scalar_type()) {
      case at::kHalf: d->dtype = MSCO_DTYPE_F16; break;
      case at::kBFloat16: d->dtype = MSCO_DTYPE_BF16; break;
      case at::kChar: d->dtype = MSCO_DTYPE_I8; break;
      case at::kFloat: d->dtype = MSCO_DTYPE_F32; break;
      case at::kInt: d->dtype = MSCO_DTYPE_I32; break;
      case at::kLong: d->dtype = MSCO_DTYPE_I64; break;
      default: TypeError(std::string("unsupported dtype of ") + name);
    }
    d->ndim = static_cast<int32_t>(t.dim());
    for (int64_t i = 0; i < t.dim(); ++i) {
      d->shape[i] = t.size(i);
      d->strides[i] = t.stride(i);
    }
    d->on_host = cuda ? 0 : 1;
    d->reserved = 0;
    return d;
  }
  MsTensorDesc *Add(PyObject *o, const char *name, bool host = false) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) TypeError(std::string(name) + " must be a torch tensor");
    return Add(THPVariable_Unpack(o), name, host);
  }

 private:
  MsTensorDesc desc_[24];
  int used_ = 0;
  int64_t device_ = 0;
};

void CheckArgs(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) TypeError("takes " + std::to_string(want) + " arguments, got " + std::to_string(got));
}
double Number(PyObject *o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}
long long Integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}
int Truth(PyObject *o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw python_error();
  return v;
}
void *StreamOf(const Call &c) { return c10::cuda::getCurrentCUDAStream(c.device()).stream(); }

PyObject *RopeAndCache(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CheckArgs(n, 18);
  Call c(a[0], "query");
  const c10::cuda::CUDAGuard guard(c.device());
  const at::Tensor &query = THPVariable_Unpack(a[0]);
  at::Tensor out = at::empty(query.sizes(), query.options());
  MsTensorDesc *d[10];
  static const char *names[10] = {"query", "key", "value", "key_cache", "value_cache", "slot_mapping", "positions", "cos_sin",
                                  "q_weight", "k_weight"};
  for (int i = 0; i < 10; ++i) d[i] = c.Add(a[i], names[i]);
  MsTensorDesc *kd = c.Add(a[13], "k_descale"), *ko = c.Add(a[14], "k_offset"), *vd = c.Add(a[15], "v_descale"),
               *vo = c.Add(a[16], "v_offset"), *oob = c.Add(a[17], "oob_count"), *od = c.Add(out, "query_out", false);
  const int rc = ms_custom_ops_rope_and_cache(d[0], d[1], d[2], d[3], d[4], d[5], d[6], d[7], d[8], d[9], Number(a[10]),
                                              Truth(a[11]), Integer(a[12]), kd, ko, vd, vo, oob, od, StreamOf(c));
  if (rc != MSCO_OK) return PyLong_FromLong(rc);
  return THPVariable_Wrap(std::move(out));
  END_HANDLE_TH_ERRORS
}

// query, key_cache, value_cache, block_tables, q_seq_lens, context_lens, qk_scale, window_size, input_layout, k_descale,
// k_offset, v_descale, v_offset, out, return_lse, oob_count -> (out, lse or None)
PyObject *ChunkAttention(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CheckArgs(n, 16);
  Call c(a[0], "query");
  const c10::cuda::CUDAGuard guard(c.device());
  const at::Tensor &query = THPVariable_Unpack(a[0]);
  MsChunkAttentionArgs args;
  args.query = c.Add(a[0], "query");
  args.key_cache = c.Add(a[1], "key_cache");
  args.value_cache = c.Add(a[2], "value_cache");
  args.block_tables = c.Add(a[3], "block_tables");
  args.q_seq_lens = c.Add(a[4], "q_seq_lens", true);
  args.context_lens = c.Add(a[5], "context_lens", true);
  args.qk_scale = Number(a[6]);
  args.window_size = Integer(a[7]);
  args.input_layout = Integer(a[8]);
  args.k_descale = c.Add(a[9], "k_descale");
  args.k_offset = c.Add(a[10], "k_offset");
  args.v_descale = c.Add(a[11], "v_descale");
  args.v_offset = c.Add(a[12], "v_offset");
  args.oob_count = c.Add(a[15], "oob_count");
  // the checks and the plan first: shapes are what they should be when the outputs are made
  size_t bytes = 0;
  int rc = ms_custom_ops_chunk_attention_workspace_size(&args, &bytes);
  if (rc != MSCO_OK) return PyLong_FromLong(rc);
  const bool given = a[13] != Py_None;
  if (given && !THPVariable_Check(a[13])) TypeError("out must be a torch CUDA tensor");
  at::Tensor out = given ? THPVariable_Unpack(a[13]) : at::empty(query.sizes(), query.options());
  at::Tensor lse, workspace;
  if (Truth(a[14])) lse = at::empty({query.size(0), query.size(1)}, query.options().dtype(at::kFloat));
  // from the allocator, per call: it belongs to this call's stream, or to the graph that is being captured
  if (bytes != 0) workspace = at::empty({static_cast<int64_t>(bytes)}, query.options().dtype(at::kByte));
  rc = ms_custom_ops_chunk_attention(&args, c.Add(out, "out", false), lse.defined() ? c.Add(lse, "lse", false) : nullptr,
                                     bytes != 0 ? workspace.data_ptr() : nullptr, bytes, StreamOf(c));
  if (rc != MSCO_OK) return PyLong_FromLong(rc);
  int64_t rows = 0;
  const int32_t *lens = static_cast<const int32_t *>(args.q_seq_lens->data);
  for (int64_t i = 0; i < args.q_seq_lens->shape[0]; ++i) rows += lens[i];
  if (rows < query.size(0)) {
    if (!given) out.narrow(0, rows, query.size(0) - rows).zero_();
    if (lse.defined()) lse.narrow(0, rows, query.size(0) - rows).fill_(-std::numeric_limits<double>::infinity());
  }
  PyObject *l = Py_None;
  if (lse.defined()) l = THPVariable_Wrap(std::move(lse)); else Py_INCREF(l);
  PyObject *o = a[13];
  if (given) Py_INCREF(o); else o = THPVariable_Wrap(std::move(out));
  return Py_BuildValue("(NN)", o, l);
  END_HANDLE_TH_ERRORS
}

// target_probs, draft_probs, draft_tokens, uniform, draft_lens -> (tokens, accepted)
PyObject *VerifyDraftTokens(PyObject *, PyObject *const *a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  CheckArgs(n, 5);
  Call c(a[0], "target_probs");
  const c10::cuda::CUDAGuard guard(c.device());
  MsTensorDesc *t = c.Add(a[0], "target_probs"), *d = c.Add(a[1], "draft_probs"), *tok = c.Add(a[2], "draft_tokens"),
               *u = c.Add(a[3], "uniform"), *len = c.Add(a[4], "draft_lens");
  int32_t dtype = 0, ndim = 0;
  int64_t shape[MS_MAX_DIMS];
  int rc = ms_custom_ops_verify_draft_tokens_infer(t, d, tok, u, len, &dtype, &ndim, shape);
  if (rc != MSCO_OK) return PyLong_FromLong(rc);
  const auto options = THPVariable_Unpack(a[0]).options().dtype(at::kInt);
  at::Tensor tokens = at::empty({shape[0], shape[1]}, options), accepted = at::empty({shape[0]}, options);
  rc = ms_custom_ops_verify_draft_tokens(t, d, tok, u, len, c.Add(tokens, "tokens", false), c.Add(accepted, "accepted", false),
                                         StreamOf(c));
  if (rc != MSCO_OK) return PyLong_FromLong(rc);
  return Py_BuildValue("(NN)", THPVariable_Wrap(std::move(tokens)), THPVariable_Wrap(std::move(accepted)));
  END_HANDLE_TH_ERRORS
}

PyMethodDef g_methods[] = {
    {"rope_and_cache", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(RopeAndCache)), METH_FASTCALL, nullptr},
    {"chunk_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(ChunkAttention)), METH_FASTCALL, nullptr},
    {"verify_draft_tokens", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(VerifyDraftTokens)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_torch_binding", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__torch_binding(void) { return PyModule_Create(&g_module); }
