// hc_host.cpp -- the serving calls' arguments from tensors, without Python.
//
// A call of kernels.paged_kv_append and its like takes 15 us in Python:
// about 50 attribute reads of 50 ns, 30 ctypes conversions, an allocation; the
// launch itself takes 2.  A decode step's kernels are shorter than that.  From
// here the call takes 5 us (8 with two launches).  The functions read the same arguments from the tensors themselves, check them
// in the same way and make the same C-ABI call. They answer NotImplemented
// for anything but the plain case -- another device, a view that has to be
// copied, an argument that is refused, an error of the call -- and the
// Python form then does the whole call again from the start and raises what
// there is to raise: every refusal comes from one place. All refusals are made
// before a launch, so nothing runs twice.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include "heliocuda.h"

namespace {

// the library's functions, by address (the library is loaded by ctypes)
decltype(&hpc_paged_kv_append) f_append;
decltype(&hpc_attention_workspace_bytes) f_attention_bytes;
decltype(&hpc_paged_attention) f_paged;
decltype(&hpc_prompt_attention) f_prompt;
decltype(&hpc_logits_topk_workspace_bytes) f_logits_bytes;
decltype(&hpc_logits_topk) f_logits;

PyObject* not_handled() {
  PyErr_Clear();
  Py_RETURN_NOTIMPLEMENTED;
}

// Not the plain case.
struct Other {};

const at::Tensor& tensor(PyObject* o) {
  if (!THPVariable_CheckExact(o)) throw Other();
  return THPVariable_Unpack(o);
}
bool none(PyObject* o) { return o == Py_None; }
void need(bool ok) {
  if (!ok) throw Other();
}
int64_t integer(PyObject* o) {
  need(PyLong_CheckExact(o));
  const int64_t v = PyLong_AsLongLong(o);
  need(v != -1 || !PyErr_Occurred());
  return v;
}
double number(PyObject* o) {
  need(PyFloat_CheckExact(o) || PyLong_CheckExact(o));
  const double v = PyFloat_AsDouble(o);
  need(v != -1.0 || !PyErr_Occurred());
  return v;
}
int dtype_id(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return HPC_DTYPE_F32;
    case at::kHalf: return HPC_DTYPE_F16;
    case at::kBFloat16: return HPC_DTYPE_BF16;
    default: throw Other();
  }
}
// Contiguous, of a type, on the device.
const at::Tensor& flat(PyObject* o, at::ScalarType type, int dev) {
  const at::Tensor& t = tensor(o);
  need(t.scalar_type() == type && t.is_cuda() && t.get_device() == dev && t.is_contiguous());
  return t;
}
// A list that may be left out: its address, and its length if `count` is not negative.
const void* list(PyObject* o, at::ScalarType type, int dev, int64_t count) {
  if (none(o)) return nullptr;
  const at::Tensor& t = flat(o, type, dev);
  need(count < 0 || t.numel() == count);
  return t.const_data_ptr();
}
// [rows][heads][dim], heads and elements contiguous within a row; its row stride.
struct Rows {
  const void* p;
  size_t stride;
};
Rows rows3(const at::Tensor& t, int dev, int64_t rows, int64_t heads, int64_t dim) {
  need(t.is_cuda() && t.dim() == 3 && t.get_device() == dev && t.size(0) == rows && t.size(1) == heads && t.size(2) == dim);
  const auto st = t.strides();
  const void* p = t.const_data_ptr();
  need(st[2] == 1 && (st[1] == dim || heads <= 1) && st[0] % 8 == 0 && st[0] >= heads * dim &&
       reinterpret_cast<uintptr_t>(p) % 16 == 0);
  return {p, size_t(st[0])};
}

struct Cache {
  const at::Tensor &k, &v;
  int dev;
  int64_t pages, page_size, heads, dim;
};
Cache cache(PyObject* ko, PyObject* vo) {
  const at::Tensor &k = tensor(ko), &v = tensor(vo);
  need(k.is_cuda() && v.is_cuda() && k.dim() == 4 && k.sizes() == v.sizes() && k.scalar_type() == v.scalar_type() &&
       k.get_device() == v.get_device() && k.is_contiguous() && v.is_contiguous());
  return {k, v, int(k.get_device()), k.size(0), k.size(1), k.size(2), k.size(3)};
}

struct Batch {
  const int32_t *table, *starts, *lens;
  size_t width, seqs;
};
Batch batch(PyObject* table, PyObject* starts, PyObject* lens, int dev) {
  const at::Tensor &t = flat(table, at::kInt, dev), &s = flat(starts, at::kInt, dev), &l = flat(lens, at::kInt, dev);
  const int64_t seqs = l.numel();
  need(t.dim() == 2 && t.size(0) == seqs && s.numel() == seqs + 1);
  return {t.const_data_ptr<int32_t>(), s.const_data_ptr<int32_t>(), l.const_data_ptr<int32_t>(), size_t(t.size(1)),
          size_t(seqs)};
}

void current(int dev) { need(c10::cuda::current_device() == dev); }

// Device memory for the length of one call, handed on in stream order.
struct Workspace {
  void* p;
  Workspace(size_t n, cudaStream_t st) : p(c10::cuda::CUDACachingAllocator::raw_alloc_with_stream(n, st)) {}
  ~Workspace() { c10::cuda::CUDACachingAllocator::raw_delete(p); }
  Workspace(const Workspace&) = delete;
};

template <class F>
int unlocked(F&& call) {
  int code;
  Py_BEGIN_ALLOW_THREADS
  code = call();
  Py_END_ALLOW_THREADS
  return code;
}

template <class F>
PyObject* plain_case(F&& f) {
  if (!f_append) return not_handled();
  try {
    return f();
  } catch (...) {
    return not_handled();
  }
}

at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, int dev) {
  return at::empty(sizes, at::TensorOptions().dtype(type).device(at::kCUDA, dev));
}

// k, v, key_cache, value_cache, page_table, query_starts, kv_lens, q, inv_freq, q_norm, k_norm, norm_v, eps, q_out
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return plain_case([&]() -> PyObject* {
    need(n == 14);
    const Cache c = cache(a[2], a[3]);
    current(c.dev);
    const Batch b = batch(a[4], a[5], a[6], c.dev);
    const at::Tensor &k = tensor(a[0]), &v = tensor(a[1]);
    const int cache_type = dtype_id(c.k.scalar_type()), type = dtype_id(k.scalar_type());
    need(k.dim() == 3 && v.scalar_type() == k.scalar_type());
    const int64_t rows = k.size(0);
    const Rows kr = rows3(k, c.dev, rows, c.heads, c.dim), vr = rows3(v, c.dev, rows, c.heads, c.dim);
    Rows qr{nullptr, 0};
    int64_t heads = c.heads;
    at::Tensor made;
    const at::Tensor* out = nullptr;
    if (!none(a[7])) {
      const at::Tensor& q = tensor(a[7]);
      need(q.dim() == 3 && q.scalar_type() == k.scalar_type());
      heads = q.size(1);
      qr = rows3(q, c.dev, rows, heads, c.dim);
      if (none(a[13])) {
        made = empty({rows, heads, c.dim}, c.k.scalar_type(), c.dev);
        out = &made;
      } else {
        out = &flat(a[13], c.k.scalar_type(), c.dev);
        need(out->sizes() == q.sizes());
      }
    }
    const at::Tensor* freq = none(a[8]) ? nullptr : &flat(a[8], at::kDouble, c.dev);
    const size_t half = freq ? size_t(freq->numel()) : 0;
    const auto qn = static_cast<const float*>(list(a[9], at::kFloat, c.dev, c.dim));
    const auto kn = static_cast<const float*>(list(a[10], at::kFloat, c.dev, c.dim));
    const int norm_v = PyObject_IsTrue(a[11]);
    need(norm_v >= 0);
    const float eps = float(number(a[12]));
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(c.dev)).stream();
    need(unlocked([&] {
           return f_append(kr.p, kr.stride, vr.p, vr.stride, qr.p, qr.stride, type, size_t(rows), size_t(heads),
                           size_t(c.heads), size_t(c.dim), half ? freq->const_data_ptr<double>() : nullptr, half, qn, kn,
                           norm_v, eps, c.k.data_ptr(), c.v.data_ptr(), cache_type, size_t(c.pages), size_t(c.page_size),
                           b.table, b.width, b.starts, b.lens, b.seqs, out ? out->data_ptr() : nullptr, st);
         }) == HPC_OK);
    if (!out) Py_RETURN_NONE;
    return made.defined() ? THPVariable_Wrap(made) : Py_NewRef(a[13]);
  });
}

// The attention calls' output: `out`, or a new tensor of out_dtype or q's type.
struct Out {
  at::Tensor made;
  void* p;
  int type;
};
Out attention_out(PyObject* out, PyObject* out_dtype, const at::Tensor& q, int dev) {
  if (!none(out)) {
    const at::Tensor& t = tensor(out);
    need(t.is_cuda() && t.get_device() == dev && t.is_contiguous() && t.sizes() == q.sizes());
    return {at::Tensor(), t.data_ptr(), dtype_id(t.scalar_type())};
  }
  at::ScalarType type = q.scalar_type();
  if (!none(out_dtype)) {
    need(THPDtype_Check(out_dtype));
    type = reinterpret_cast<THPDtype*>(out_dtype)->scalar_type;
  }
  const int id = dtype_id(type);
  at::Tensor t = empty(q.sizes(), type, dev);
  void* const p = t.data_ptr();
  return {std::move(t), p, id};
}

// q, key_cache, value_cache, page_table, query_starts, kv_lens, max_query_len, scale, window, out, out_dtype
PyObject* paged(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return plain_case([&]() -> PyObject* {
    need(n == 11);
    const Cache c = cache(a[1], a[2]);
    current(c.dev);
    const Batch b = batch(a[3], a[4], a[5], c.dev);
    const at::Tensor& q = tensor(a[0]);
    need(q.dim() == 3 && q.scalar_type() == c.k.scalar_type());
    const int type = dtype_id(q.scalar_type());
    const int64_t rows = q.size(0), heads = q.size(1), most = integer(a[6]), window = integer(a[8]);
    const Rows qr = rows3(q, c.dev, rows, heads, c.dim);
    const float scale = float(number(a[7]));
    size_t bytes = 0;
    need(most >= 0 && window >= 0 && f_attention_bytes(size_t(heads), size_t(c.heads), size_t(c.dim), &bytes) == HPC_OK);
    const Out out = attention_out(a[9], a[10], q, c.dev);
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(c.dev)).stream();
    const Workspace ws(bytes, st);
    need(unlocked([&] {
           return f_paged(qr.p, qr.stride, c.k.const_data_ptr(), c.v.const_data_ptr(), type, size_t(c.pages),
                          size_t(c.page_size), b.table, b.width, b.starts, b.lens, b.seqs, size_t(rows), size_t(heads),
                          size_t(c.heads), size_t(c.dim), size_t(most), scale, size_t(window), ws.p, bytes, out.p, out.type,
                          nullptr, st);
         }) == HPC_OK);
    return out.made.defined() ? THPVariable_Wrap(out.made) : Py_NewRef(a[9]);
  });
}

// q, k, v, query_starts, max_query_len, scale, window, out, out_dtype
PyObject* prompt(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return plain_case([&]() -> PyObject* {
    need(n == 9);
    const at::Tensor &q = tensor(a[0]), &k = tensor(a[1]), &v = tensor(a[2]);
    need(q.is_cuda() && q.dim() == 3 && k.dim() == 3 && k.sizes() == v.sizes() && k.scalar_type() == q.scalar_type() &&
         v.scalar_type() == q.scalar_type());
    const int dev = int(q.get_device()), type = dtype_id(q.scalar_type());
    current(dev);
    const int64_t rows = q.size(0), heads = q.size(1), dim = q.size(2), kv_heads = k.size(1);
    const int64_t most = integer(a[4]), window = integer(a[6]);
    const Rows qr = rows3(q, dev, rows, heads, dim), kr = rows3(k, dev, rows, kv_heads, dim),
               vr = rows3(v, dev, rows, kv_heads, dim);
    const at::Tensor& starts = flat(a[3], at::kInt, dev);
    const float scale = float(number(a[5]));
    size_t bytes = 0;
    need(starts.numel() >= 1 && most >= 0 && window >= 0 &&
         f_attention_bytes(size_t(heads), size_t(kv_heads), size_t(dim), &bytes) == HPC_OK);
    const Out out = attention_out(a[7], a[8], q, dev);
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream();
    const Workspace ws(bytes, st);
    need(unlocked([&] {
           return f_prompt(qr.p, qr.stride, kr.p, kr.stride, vr.p, vr.stride, type, starts.const_data_ptr<int32_t>(),
                           size_t(starts.numel() - 1), size_t(rows), size_t(heads), size_t(kv_heads), size_t(dim),
                           size_t(most), scale, size_t(window), ws.p, bytes, out.p, out.type, nullptr, st);
         }) == HPC_OK);
    return out.made.defined() ? THPVariable_Wrap(out.made) : Py_NewRef(a[7]);
  });
}

// logits, k, history, history_starts, prompt_lens, repetition, frequency, presence, bias_ids, bias_values, bias_starts, allowed
PyObject* logits(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return plain_case([&]() -> PyObject* {
    need(n == 12);
    const at::Tensor& x = tensor(a[0]);
    need(x.is_cuda() && x.dim() == 2 && x.scalar_type() == at::kFloat);
    const int dev = int(x.get_device());
    current(dev);
    const int64_t rows = x.size(0), vocab = x.size(1), k = integer(a[1]);
    need(k >= 1 && rows >= 1 && x.stride(1) == 1 && x.stride(0) >= vocab);
    const int64_t stride = rows > 1 ? x.stride(0) : vocab;
    need(none(a[2]) == none(a[3]) && none(a[8]) == none(a[10]) && none(a[8]) == none(a[9]));
    const size_t hist_n = none(a[2]) ? 0 : size_t(tensor(a[2]).numel()), bias_n = none(a[8]) ? 0 : size_t(tensor(a[8]).numel());
    size_t mask_stride = 0;
    if (!none(a[11])) {
      const at::Tensor& m = tensor(a[11]);
      need(m.dim() == 2 && m.size(0) == rows);
      mask_stride = size_t(m.size(1));
    }
    const auto i32 = [&](int i, int64_t count) { return static_cast<const int32_t*>(list(a[i], at::kInt, dev, count)); };
    const auto f32 = [&](int i, int64_t count) { return static_cast<const float*>(list(a[i], at::kFloat, dev, count)); };
    const int32_t *hist = i32(2, -1), *hist_starts = i32(3, rows + 1), *prompt_lens = i32(4, rows);
    const float *rep = f32(5, rows), *freq = f32(6, rows), *pres = f32(7, rows);
    const int32_t* bias_ids = i32(8, -1);
    const float* bias_vals = f32(9, int64_t(bias_n));
    const int32_t *bias_starts = i32(10, rows + 1), *allowed = i32(11, -1);
    size_t bytes = 0;
    need(f_logits_bytes(size_t(rows), size_t(vocab), size_t(k), &bytes) == HPC_OK);
    const at::Tensor ids = empty({rows, k}, at::kInt, dev), vals = empty({rows, k}, at::kFloat, dev);
    const cudaStream_t st = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(dev)).stream();
    {
      const Workspace ws(bytes, st);
      need(unlocked([&] {
             return f_logits(x.const_data_ptr<float>(), size_t(stride), size_t(rows), size_t(vocab), size_t(k), hist, hist_n,
                             hist_starts, prompt_lens, rep, freq, pres, bias_ids, bias_vals, bias_n, bias_starts,
                             reinterpret_cast<const uint32_t*>(allowed), mask_stride, ws.p, bytes, ids.data_ptr<int32_t>(),
                             vals.data_ptr<float>(), st);
           }) == HPC_OK);
    }
    PyObject* i = THPVariable_Wrap(ids);
    PyObject* v = THPVariable_Wrap(vals);
    return i && v ? Py_BuildValue("(NN)", i, v) : nullptr;
  });
}

// The library's functions by their addresses, in the order of the variables above.
PyObject* bind(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 6) {
    PyErr_SetString(PyExc_TypeError, "bind: six addresses");
    return nullptr;
  }
  void* p[6];
  for (int i = 0; i < 6; ++i) {
    p[i] = PyLong_AsVoidPtr(a[i]);
    if (!p[i]) return PyErr_Occurred() ? nullptr : PyErr_Format(PyExc_ValueError, "bind: address %d is null", i);
  }
  f_append = reinterpret_cast<decltype(f_append)>(p[0]);
  f_attention_bytes = reinterpret_cast<decltype(f_attention_bytes)>(p[1]);
  f_paged = reinterpret_cast<decltype(f_paged)>(p[2]);
  f_prompt = reinterpret_cast<decltype(f_prompt)>(p[3]);
  f_logits_bytes = reinterpret_cast<decltype(f_logits_bytes)>(p[4]);
  f_logits = reinterpret_cast<decltype(f_logits)>(p[5]);
  Py_RETURN_NONE;
}

#define HC_METHOD(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {HC_METHOD(append), HC_METHOD(paged), HC_METHOD(prompt), HC_METHOD(logits), HC_METHOD(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() {
  PyObject* m = PyModule_Create(&module);
  // the versions whose interfaces were compiled in; the caller compares them before its first call
  if (m && PyModule_AddStringConstant(m, "built_for", HC_BUILT_FOR) < 0) Py_CLEAR(m);
  return m;
}
