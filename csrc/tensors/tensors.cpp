// The checks of the ops whose calls are short, in one native call each: asked of
// the tensors one by one from Python, the questions take longer than the launch.
//
// Each function returns the numbers that its launch needs, or None for any call
// that is not what almost every one is; foundry_b200/ops then looks at it in detail
// and says what is wrong with it, or finds that it is allowed all the same.
#include <ATen/core/Tensor.h>
#include <torch/csrc/autograd/python_variable.h>

#include <Python.h>

#include <cstdint>
#include <exception>

namespace {

// All of `n` arguments as tensors; missing ones (None) are null where `optional` allows them.
bool tensors(PyObject* const* args, int n, const at::Tensor** out, bool optional = false) {
  for (int i = 0; i < n; ++i) {
    if (optional && args[i] == Py_None) {
      out[i] = nullptr;
      continue;
    }
    if (!THPVariable_Check(args[i])) return false;
    out[i] = &THPVariable_Unpack(args[i]);
  }
  return true;
}

int64_t address(const at::Tensor& t) { return reinterpret_cast<int64_t>(t.const_data_ptr()); }

PyObject* numbers(const int64_t* v, int n) {
  PyObject* t = PyTuple_New(n);
  for (int i = 0; t && i < n; ++i) {
    PyObject* x = PyLong_FromLongLong(v[i]);
    if (!x) {
      Py_DECREF(t);
      return nullptr;
    }
    PyTuple_SET_ITEM(t, i, x);
  }
  return t;
}

// decode(q, k_cache, v_cache, block_tables, seq_lens, out, device, page):
// (batch, q heads, kv heads, blocks, table width, the six addresses, row strides of q and out)
PyObject* decode(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 8) {
    PyErr_SetString(PyExc_TypeError, "decode takes six tensors, the device and the page size");
    return nullptr;
  }
  const int64_t device = PyLong_AsLongLong(args[6]), page = PyLong_AsLongLong(args[7]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor* t[6];
    if (!tensors(args, 6, t)) Py_RETURN_NONE;
    const at::Tensor &q = *t[0], &k = *t[1], &v = *t[2], &table = *t[3], &lens = *t[4], &out = *t[5];
    if (q.dim() != 3 || k.dim() != 4 || table.dim() != 2 || lens.dim() != 1) Py_RETURN_NONE;
    const int64_t b = q.size(0), n_q = q.size(1), blocks = k.size(0), n_kv = k.size(1), width = table.size(1);
    for (int i = 0; i < 6; ++i) {
      const bool index = i == 3 || i == 4;
      if (t[i]->scalar_type() != (index ? at::kInt : at::kBFloat16) || !t[i]->is_contiguous() ||
          t[i]->get_device() != device)
        Py_RETURN_NONE;
    }
    if (q.size(2) != 128 || k.size(2) != page || k.size(3) != 128 || out.sizes() != q.sizes() ||
        v.sizes() != k.sizes() || table.size(0) != b || lens.size(0) != b)
      Py_RETURN_NONE;
    if (blocks <= 0 || width <= 0 || width > 1 << 24 || blocks >= int64_t{1} << 31 || n_kv >= 1 << 16 ||
        (blocks + 1) * n_kv * page >= int64_t{1} << 31 || b >= 1 << 30 || b * n_kv >= 1 << 30 ||
        b * n_kv * (width / 2 + 2) >= 1 << 30)
      Py_RETURN_NONE;
    const int64_t r[13] = {b,           n_q,            n_kv,          blocks,       width,     address(q), address(k),
                           address(v), address(table), address(lens), address(out), n_q * 128, n_q * 128};
    if ((r[5] | r[6] | r[7] | r[10]) & 15) Py_RETURN_NONE;
    return numbers(r, 13);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

// rows(logits, ids, logprobs, entropy, top_logprobs, top_ids, device): (kind, rows, vocabulary,
// alternatives, row stride, the six addresses); kind 0 bf16, 1 fp16, 2 fp32. All but logits may be None.
PyObject* rows(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != 7) {
    PyErr_SetString(PyExc_TypeError, "rows takes six tensors and the device");
    return nullptr;
  }
  const int64_t device = PyLong_AsLongLong(args[6]);
  if (PyErr_Occurred()) return nullptr;
  try {
    const at::Tensor* t[6];
    if (!THPVariable_Check(args[0]) || !tensors(args, 6, t, true)) Py_RETURN_NONE;
    const at::Tensor& x = *t[0];
    if (x.dim() != 2 || x.get_device() != device || x.stride(1) != 1) Py_RETURN_NONE;
    const auto type = x.scalar_type();
    const int kind = type == at::kBFloat16 ? 0 : type == at::kHalf ? 1 : type == at::kFloat ? 2 : -1;
    const int64_t rows = x.size(0), vocab = x.size(1);
    if (kind < 0 || vocab <= 0 || vocab >= 1 << 30 || rows >= 1 << 30 || !t[1] != !t[2] || !t[4] != !t[5])
      Py_RETURN_NONE;
    int64_t k = 0;
    if (t[5]) {
      if (t[5]->dim() != 2) Py_RETURN_NONE;
      k = t[5]->size(1);
    }
    int64_t r[11] = {kind, rows, vocab, k, x.stride(0), address(x)};
    for (int i = 1; i < 6; ++i) {
      r[5 + i] = 0;
      if (!t[i]) continue;
      const at::Tensor& o = *t[i];
      const bool index = i == 1 || i == 5;
      if (o.scalar_type() != (index ? at::kInt : at::kFloat) || o.dim() != (i < 4 ? 1 : 2) || o.size(0) != rows ||
          (i >= 4 && o.size(1) != k) || !o.is_contiguous() || o.get_device() != device)
        Py_RETURN_NONE;
      r[5 + i] = address(o);
    }
    return numbers(r, 11);
  } catch (const std::exception&) {
    Py_RETURN_NONE;
  }
}

PyMethodDef methods[] = {
    {"decode", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(decode)), METH_FASTCALL,
     "The numbers of a decode attention call, or None."},
    {"rows", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rows)), METH_FASTCALL,
     "The numbers of a token_logprobs call, or None."},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_tensors", "Checks of short ops' tensors.", -1, methods};

}  // namespace

PyMODINIT_FUNC PyInit__tensors() { return PyModule_Create(&module); }
