// The short calls' way from Python to the C ABI: checks of arguments, output allocation and launch in one native step.
//
// A decode step's kernels take 5 to 10 us; asking eleven tensors for shape, strides, type and device from Python takes
// as long again.  Each function here makes exactly the checks of the Python function of the same operator (ops.py) and
// launches, or returns False: nothing is launched when a check does not hold, and the Python function then goes on with
// its own checks, which say what is wrong, and with the rare forms that are not taken here.  It returns False too when the
// library reports an error, for the Python function to make the call again and raise it; a first launch of two may then
// run twice, which writes the same.  Nothing is kept from call to call but what a plan holds.  Host time of a call, checks
// in Python and here: multi-axis append 13.7 and 6.8 us, decode with first tokens 10.4 and 5.0, prefill with first tokens
// 11.9 and 5.2, shared-prefix decode 11.2 and 7.9 (two launches, three tensor maps, a look at the stream's capture).
#include <Python.h>
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>
#include <cstring>
#include <new>

#include "piekv.h"

namespace {

constexpr int kDevices = 64;
decltype(&piekv_rope_axes) rope_axes_fn = nullptr;
decltype(&piekv_shared_prefix_run) shared_prefix_fn = nullptr;
decltype(&piekv_decode_run_opt) decode_fn = nullptr;
decltype(&piekv_prefill_run_opt) prefill_fn = nullptr;
int32_t *error_words[kDevices] = {nullptr};

// A plain tensor on CUDA device `device` (-1: any), or nullptr.
const at::Tensor *tensor_on(PyObject *o, int device) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor &t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || (device >= 0 && t.get_device() != device)) return nullptr;
  return &t;
}
int dtype_code(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return PIEKV_F32;
    case at::kHalf: return PIEKV_F16;
    case at::kBFloat16: return PIEKV_BF16;
    default: return -1;
  }
}
bool fits(int64_t n) { return n >= 0 && n <= INT_MAX; }
// [tokens, heads, head_dim] with neighbouring elements in a row
bool is_rows(const at::Tensor &t) { return t.dim() == 3 && (t.stride(2) == 1 || t.size(2) <= 1); }
bool is_i32(const at::Tensor *t) { return t != nullptr && t->scalar_type() == at::kInt && t->is_contiguous(); }
bool is_pool(const at::Tensor *t) { return t != nullptr && t->dim() == 5 && t->size(1) == 2 && t->is_contiguous() && fits(t->size(0)); }
bool is_current(int device) { return device >= 0 && device < kDevices && c10::cuda::current_device() == device; }
void *stream_of(int device) { return c10::cuda::getCurrentCUDAStream(device).stream(); }

// `out` as given (contiguous, shaped and typed like q), or a new one; undefined when what was given does not do.
at::Tensor output_like(const at::Tensor &q, PyObject *given) {
  if (given == Py_None) return at::empty(q.sizes(), q.options());
  const at::Tensor *out = tensor_on(given, q.get_device());
  if (out == nullptr || out->sizes() != q.sizes() || out->scalar_type() != q.scalar_type() || !out->is_contiguous())
    return at::Tensor();
  return *out;
}

PyObject *declined() { Py_RETURN_FALSE; }

// set_error_word(device, address)
PyObject *set_error_word(PyObject *, PyObject *args) {
  int device;
  unsigned long long address;
  if (!PyArg_ParseTuple(args, "iK", &device, &address)) return nullptr;
  if (device >= 0 && device < kDevices) error_words[device] = reinterpret_cast<int32_t *>(address);
  Py_RETURN_NONE;
}

// bind(rope_axes, shared_prefix_run, decode_run_opt, prefill_run_opt): addresses of the library's functions
PyObject *bind(PyObject *, PyObject *args) {
  unsigned long long a, b, c, d;
  if (!PyArg_ParseTuple(args, "KKKK", &a, &b, &c, &d)) return nullptr;
  rope_axes_fn = reinterpret_cast<decltype(rope_axes_fn)>(a);
  shared_prefix_fn = reinterpret_cast<decltype(shared_prefix_fn)>(b);
  decode_fn = reinterpret_cast<decltype(decode_fn)>(c);
  prefill_fn = reinterpret_cast<decltype(prefill_fn)>(d);
  Py_RETURN_NONE;
}

// rope_axes_append(piekv_rope_axes_table as bytes, q, k, v, pos_ids, batch_indices, positions, pool, kv_indices, kv_indptr, q_out | None)
PyObject *rope_axes_append(PyObject *, PyObject *const *o, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 11) {
    PyErr_SetString(PyExc_TypeError, "rope_axes_append takes 11 arguments");
    return nullptr;
  }
  if (!PyObject_CheckBuffer(o[0])) return declined();
  Py_buffer given_table;
  if (PyObject_GetBuffer(o[0], &given_table, PyBUF_SIMPLE) != 0) return nullptr;
  piekv_rope_axes_table table;  // a copy: the caller's may change once the interpreter runs other threads
  const bool is_table = given_table.len == (Py_ssize_t)sizeof(table);
  if (is_table) std::memcpy(&table, given_table.buf, sizeof(table));
  PyBuffer_Release(&given_table);
  if (!is_table) return declined();
  const at::Tensor *k = tensor_on(o[2], -1);
  if (k == nullptr || !is_rows(*k)) return declined();
  const int device = k->get_device(), dtype = dtype_code(*k);
  if (dtype < 0 || !is_current(device) || error_words[device] == nullptr) return declined();
  const at::Tensor *q = tensor_on(o[1], device), *v = tensor_on(o[3], device), *pos = tensor_on(o[4], device),
                   *batch_indices = tensor_on(o[5], device), *positions = tensor_on(o[6], device),
                   *pool = tensor_on(o[7], device), *indices = tensor_on(o[8], device), *indptr = tensor_on(o[9], device);
  const int64_t n = k->size(0), hkv = k->size(1), d = k->size(2);
  if (q == nullptr || !is_rows(*q) || q->size(0) != n || q->size(2) != d || q->scalar_type() != k->scalar_type()) return declined();
  if (v == nullptr || !is_rows(*v) || v->sizes() != k->sizes() || v->scalar_type() != k->scalar_type()) return declined();
  if (pos == nullptr || pos->scalar_type() != at::kInt || pos->dim() != 2 || pos->size(0) != table.num_axes || pos->size(1) < n ||
      (n > 1 && pos->stride(1) != 1))
    return declined();
  if (!is_pool(pool) || pool->size(3) != hkv || pool->size(4) != d || pool->scalar_type() != k->scalar_type()) return declined();
  if (!is_i32(batch_indices) || !is_i32(positions) || !is_i32(indices) || !is_i32(indptr)) return declined();
  if (batch_indices->numel() < n || positions->numel() < n || indptr->numel() < 1) return declined();
  if (2 * (int64_t)table.half > d || !fits(n) || !fits(hkv) || !fits(d) || !fits(q->size(1)) || !fits(pool->size(2)) ||
      !fits(indptr->numel()))
    return declined();
  at::Tensor out;
  if (o[10] == Py_None) {
    out = at::empty(q->sizes(), q->options());
  } else {
    const at::Tensor *given = tensor_on(o[10], device);
    if (given == nullptr || !is_rows(*given) || given->sizes() != q->sizes() || given->scalar_type() != q->scalar_type())
      return declined();
    out = *given;
  }
  piekv_rope_axes_args a{};
  a.q = q->data_ptr();
  a.k = k->data_ptr();
  a.v = v->data_ptr();
  a.q_out = out.data_ptr();
  a.q_stride_n = q->stride(0);
  a.q_stride_h = q->stride(1);
  a.k_stride_n = k->stride(0);
  a.k_stride_h = k->stride(1);
  a.v_stride_n = v->stride(0);
  a.v_stride_h = v->stride(1);
  a.q_out_stride_n = out.stride(0);
  a.q_out_stride_h = out.stride(1);
  a.pos = static_cast<const int32_t *>(pos->data_ptr());
  a.pos_stride = pos->stride(0);
  a.batch_indices = static_cast<const int32_t *>(batch_indices->data_ptr());
  a.positions = static_cast<const int32_t *>(positions->data_ptr());
  a.pool = pool->data_ptr();
  a.kv_indices = static_cast<const int32_t *>(indices->data_ptr());
  a.kv_indptr = static_cast<const int32_t *>(indptr->data_ptr());
  a.err = error_words[device];
  a.nnz = (int32_t)n;
  a.batch = (int32_t)(indptr->numel() - 1);
  a.num_qo_heads = (int32_t)q->size(1);
  a.num_kv_heads = (int32_t)hkv;
  a.head_dim = (int32_t)d;
  a.page_size = (int32_t)pool->size(2);
  a.num_pages = (int32_t)pool->size(0);
  a.dtype = dtype;
  void *stream = stream_of(device);
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = rope_axes_fn(&a, &table, stream);
  Py_END_ALLOW_THREADS;
  if (status != 0) return declined();
  return THPVariable_Wrap(out);
  END_HANDLE_TH_ERRORS
}

// What a plan fixes about its runs.
struct Plan {
  int device;
  bool prefix;  // a shared-prefix run; otherwise a call with a window and first tokens, `options`
  piekv_shared_prefix_args args;
  piekv_attn_options options;
  const int32_t *qo_indptr;  // of a prefill call
  int causal;
};
const char *const kPlanName = "pie_b200.plan";
void free_plan(PyObject *capsule) { delete static_cast<Plan *>(PyCapsule_GetPointer(capsule, kPlanName)); }

// plan(device, piekv_shared_prefix_args as bytes, piekv_attn_options as bytes | None, qo_indptr address, causal): with
// options the plan of a call with a window and first tokens, which uses the tables, sizes, workspace, err and sm_scale of the struct
PyObject *make_plan(PyObject *, PyObject *args) {
  int device, causal = 0;
  unsigned long long qo_indptr = 0;
  Py_buffer a, opt;
  std::memset(&opt, 0, sizeof(opt));
  if (!PyArg_ParseTuple(args, "iy*z*|Ki", &device, &a, &opt, &qo_indptr, &causal)) return nullptr;
  PyObject *capsule = nullptr;
  if (a.len != (Py_ssize_t)sizeof(piekv_shared_prefix_args) || (opt.buf != nullptr && opt.len != (Py_ssize_t)sizeof(piekv_attn_options))) {
    PyErr_SetString(PyExc_ValueError, "plan: struct sizes differ from the library's");
  } else if (Plan *plan = new (std::nothrow) Plan()) {
    plan->device = device;
    plan->prefix = opt.buf == nullptr;
    std::memcpy(&plan->args, a.buf, sizeof(plan->args));
    if (opt.buf != nullptr) std::memcpy(&plan->options, opt.buf, sizeof(plan->options));
    plan->qo_indptr = reinterpret_cast<const int32_t *>(qo_indptr);
    plan->causal = causal;
    capsule = PyCapsule_New(plan, kPlanName, free_plan);
    if (capsule == nullptr) delete plan;
  } else {
    PyErr_NoMemory();
  }
  PyBuffer_Release(&a);
  if (opt.buf != nullptr) PyBuffer_Release(&opt);
  return capsule;
}

// What the runs of a plan ask of q, pool and out; `rows` is q's first size.  False: declined.
bool fill(const Plan &plan, int64_t rows, PyObject *q_object, PyObject *pool_object, PyObject *given, piekv_shared_prefix_args &a,
          at::Tensor &out) {
  const at::Tensor *q = tensor_on(q_object, plan.device), *pool = tensor_on(pool_object, plan.device);
  if (q == nullptr || !is_rows(*q) || !is_pool(pool) || !is_current(plan.device)) return false;
  a = plan.args;
  const int dtype = dtype_code(*q);
  if (dtype < 0 || dtype_code(*pool) != dtype || (plan.prefix && dtype != a.dtype)) return false;
  if (q->size(0) != rows || q->size(1) != a.num_qo_heads || q->size(2) != a.head_dim) return false;
  if (pool->size(2) != a.page_size || pool->size(3) != a.num_kv_heads || pool->size(4) != a.head_dim) return false;
  // the wrapper keeps a shared-prefix plan that a captured call points to
  if (plan.prefix && c10::cuda::currentStreamCaptureStatusMayInitCtx() != c10::cuda::CaptureStatus::None) return false;
  out = output_like(*q, given);
  if (!out.defined()) return false;
  a.dtype = dtype;
  a.q = q->data_ptr();
  a.q_stride_n = q->stride(0);
  a.q_stride_h = q->stride(1);
  a.pool = pool->data_ptr();
  a.num_pages = (int32_t)pool->size(0);
  a.out = out.data_ptr();
  return true;
}
PyObject *result(const at::Tensor &out, PyObject *given) {
  if (given == Py_None) return THPVariable_Wrap(out);
  Py_INCREF(given);
  return given;
}

// decode_run(plan, q, pool, out | None)
PyObject *decode_run(PyObject *, PyObject *const *o, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 4) {
    PyErr_SetString(PyExc_TypeError, "decode_run takes 4 arguments");
    return nullptr;
  }
  const auto *plan = static_cast<const Plan *>(PyCapsule_GetPointer(o[0], kPlanName));
  if (plan == nullptr) return nullptr;
  piekv_shared_prefix_args a;
  at::Tensor out;
  if (!fill(*plan, plan->args.batch, o[1], o[2], o[3], a, out)) return declined();
  void *stream = stream_of(plan->device);
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = plan->prefix
               ? shared_prefix_fn(&a, stream)
               : decode_fn(a.q, a.q_stride_n, a.q_stride_h, a.pool, a.out, nullptr, a.kv_indptr, a.kv_indices, a.kv_last_page_len, a.batch,
                           a.num_qo_heads, a.num_kv_heads, a.head_dim, a.page_size, a.num_pages, a.dtype, a.sm_scale, a.workspace,
                           a.workspace_bytes, a.err, stream, &plan->options);
  Py_END_ALLOW_THREADS;
  if (status != 0) return declined();
  return result(out, o[3]);
  END_HANDLE_TH_ERRORS
}

// prefill_run(plan, (query tokens, pages) that the device's work list was built for, q, pool, out | None)
PyObject *prefill_run(PyObject *, PyObject *const *o, Py_ssize_t count) {
  HANDLE_TH_ERRORS
  if (count != 5) {
    PyErr_SetString(PyExc_TypeError, "prefill_run takes 5 arguments");
    return nullptr;
  }
  const auto *plan = static_cast<const Plan *>(PyCapsule_GetPointer(o[0], kPlanName));
  if (plan == nullptr) return nullptr;
  long long rows, pages;
  if (!PyTuple_Check(o[1])) return declined();  // not built yet
  if (!PyArg_ParseTuple(o[1], "LL", &rows, &pages)) return nullptr;
  piekv_shared_prefix_args a;
  at::Tensor out;
  if (plan->qo_indptr == nullptr || !fits(rows) || !fill(*plan, rows, o[2], o[3], o[4], a, out) || a.num_pages != pages) return declined();
  void *stream = stream_of(plan->device);
  int status;
  Py_BEGIN_ALLOW_THREADS;
  status = prefill_fn(a.q, a.q_stride_n, a.q_stride_h, a.pool, a.out, nullptr, plan->qo_indptr, a.kv_indptr, a.kv_indices,
                      a.kv_last_page_len, nullptr, 0, plan->causal, 1, a.batch, (int32_t)rows, a.num_qo_heads, a.num_kv_heads, a.head_dim,
                      a.page_size, a.num_pages, a.dtype, a.sm_scale, a.workspace, a.workspace_bytes, a.err, stream, &plan->options);
  Py_END_ALLOW_THREADS;
  if (status != 0) return declined();
  return result(out, o[4]);
  END_HANDLE_TH_ERRORS
}

PyMethodDef methods[] = {
    {"bind", bind, METH_VARARGS, nullptr},
    {"set_error_word", set_error_word, METH_VARARGS, nullptr},
    {"rope_axes_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(rope_axes_append)), METH_FASTCALL, nullptr},
    {"plan", make_plan, METH_VARARGS, nullptr},
    {"prefill_run", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(prefill_run)), METH_FASTCALL, nullptr},
    {"decode_run", reinterpret_cast<PyCFunction>(reinterpret_cast<void *>(decode_run)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject *PyInit__calls() {
  PyObject *m = PyModule_Create(&module);
  // ops.py compares it with the torch that is loaded
  if (m != nullptr && PyModule_AddStringConstant(m, "torch_version", PIEKV_TORCH_VERSION) != 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
