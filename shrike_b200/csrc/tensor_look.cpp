// What a call over 8-bit cache pages asks of its tensors, as a Python module: a dozen questions in one call.
//
// A store of one token takes the GPU 2 us and its launch 2 more; asking torch from Python for every tensor's type, device, sizes
// and address took another 3 to 4.  Each function answers None when anything does not fit, and the caller (quantised_cache.py)
// then looks up what, and says so; nothing is kept from one call for the next.
#include <Python.h>

#include <torch/csrc/autograd/python_variable.h>

#include "cache_q8_call.cuh"

namespace {

constexpr int MOST_HEAD_DIM = 256;

const at::Tensor* tensor_of(PyObject* x) { return THPVariable_Check(x) ? &THPVariable_Unpack(x) : nullptr; }
long long device_of(const at::Tensor& t) { return t.is_cuda() ? t.get_device() : t.is_cpu() ? -1 : -2; }
bool on_16_bytes(const at::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
at::ScalarType element(long long dtype) { return dtype == 0 ? at::kFloat : at::kBFloat16; }
bool dense(const at::Tensor& t, at::ScalarType type, long long device) {
  return t.scalar_type() == type && device_of(t) == device && t.is_contiguous();
}
// A vector of `count` int32.
bool ints(const at::Tensor& t, long long count, long long device) { return dense(t, at::kInt, device) && t.numel() == count; }

bool pages_fit(const at::Tensor& codes, const at::Tensor& scales) {
  return codes.dim() == 4 && codes.scalar_type() == at::kChar && scales.scalar_type() == at::kFloat && scales.dim() == 3 &&
         scales.size(0) == codes.size(0) && scales.size(1) == codes.size(2) && scales.size(2) == codes.size(1) && codes.is_contiguous() &&
         scales.is_contiguous() && codes.device() == scales.device();
}
// Head sizes that the kernels take, and slots that are 32-bit numbers.
bool served(const at::Tensor& codes) {
  const long long dim = codes.size(3);
  return dim % 16 == 0 && dim >= 16 && dim <= MOST_HEAD_DIM && codes.size(0) * codes.size(1) <= 0x7fffffffll;
}
// Keys' and values' pages, each of which a QuantisedPages has looked at.
bool both_fit(const at::Tensor& keys, const at::Tensor& values, long long device) {
  return keys.dim() == 4 && keys.sizes() == values.sizes() && served(keys) && device_of(keys) == device && device_of(values) == device &&
         on_16_bytes(keys) && on_16_bytes(values);
}
// [n, width] rows whose elements lie side by side.
bool rows(const at::Tensor& t, at::ScalarType type, long long n, long long width, long long device) {
  return t.dim() == 2 && t.size(0) == n && t.size(1) == width && t.scalar_type() == type && device_of(t) == device &&
         (width <= 1 || t.stride(1) == 1) && (n <= 1 || t.stride(0) >= 0);
}

// Runs `body` with the tensors of args[0 ... TENSORS) and the numbers behind them; None where one is no tensor, or where torch
// has no answer (a tensor without memory, say).
template <int TENSORS, int NUMBERS, typename Body>
PyObject* with_arguments(PyObject* const* args, Py_ssize_t count, Body body) {
  if (count != TENSORS + NUMBERS) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  const at::Tensor* t[TENSORS];
  for (int i = 0; i < TENSORS; ++i)
    if ((t[i] = tensor_of(args[i])) == nullptr) Py_RETURN_NONE;
  unsigned long long x[NUMBERS + 1];
  for (int i = 0; i < NUMBERS; ++i) {
    x[i] = PyLong_AsUnsignedLongLongMask(args[TENSORS + i]);
    if (x[i] == static_cast<unsigned long long>(-1) && PyErr_Occurred()) return nullptr;
  }
  try {
    return body(t, x);
  } catch (...) {
    Py_RETURN_NONE;
  }
}

// pages(codes, scales) -> (pages, page size, kv heads, head size)
PyObject* look_pages(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return with_arguments<2, 0>(args, count, [](auto& t, auto&) -> PyObject* {
    if (!pages_fit(*t[0], *t[1])) Py_RETURN_NONE;
    const at::Tensor& codes = *t[0];
    return Py_BuildValue("(LLLL)", static_cast<long long>(codes.size(0)), static_cast<long long>(codes.size(1)), static_cast<long long>(codes.size(2)),
                         static_cast<long long>(codes.size(3)));
  });
}

// cache(k, v, key codes, key scales, value codes, value scales, slots, device, type, stream, stores) -> the launcher's arguments,
// empty for no rows
PyObject* look_cache(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return with_arguments<7, 4>(args, count, [](auto& t, auto& x) -> PyObject* {
    const at::Tensor &k = *t[0], &v = *t[1], &codes = *t[2], &key_scales = *t[3], &value_codes = *t[4], &value_scales = *t[5], &slots = *t[6];
    const long long device = static_cast<long long>(x[0]), stores = static_cast<long long>(x[3]);
    if (!both_fit(codes, value_codes, device) || k.dim() != 2) Py_RETURN_NONE;
    const long long n = stores ? k.size(0) : slots.numel(), width = codes.size(2) * codes.size(3);
    const at::ScalarType type = element(static_cast<long long>(x[1]));
    if (!ints(slots, n, device) || !rows(k, type, n, width, device) || !rows(v, type, n, width, device) || n > 0x7fffffffll) Py_RETURN_NONE;
    if (!stores && !(k.is_contiguous() && v.is_contiguous() && on_16_bytes(k) && on_16_bytes(v))) Py_RETURN_NONE;
    if (n == 0) return PyBytes_FromStringAndSize(nullptr, 0);
    const ShrikeCacheQ8 call{k.data_ptr(), v.data_ptr(), codes.data_ptr(), value_codes.data_ptr(), key_scales.data_ptr(), value_scales.data_ptr(),
                             slots.data_ptr(), reinterpret_cast<void*>(static_cast<uintptr_t>(x[2])), n > 1 ? k.stride(0) : width, n > 1 ? v.stride(0) : width, static_cast<int>(x[1]),
                             static_cast<int>(n), static_cast<int>(codes.size(2)), static_cast<int>(codes.size(3)), static_cast<int>(codes.size(0)),
                             static_cast<int>(codes.size(1))};
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&call), sizeof(call));
  });
}

// attention(q, out, key codes, key scales, value codes, value scales, block table, query starts, context lengths, device, type,
// heads, kv heads, head size) -> (tokens, sequences, blocks a sequence, out's address, (the addresses that a launch begins with))
PyObject* look_attention(PyObject*, PyObject* const* args, Py_ssize_t count) {
  return with_arguments<9, 5>(args, count, [](auto& t, auto& x) -> PyObject* {
    const at::Tensor &q = *t[0], &out = *t[1], &codes = *t[2], &key_scales = *t[3], &value_codes = *t[4], &value_scales = *t[5], &table = *t[6],
                     &starts = *t[7], &context = *t[8];
    const long long device = static_cast<long long>(x[0]), heads = static_cast<long long>(x[2]), kv_heads = static_cast<long long>(x[3]),
                    dim = static_cast<long long>(x[4]);
    const at::ScalarType type = element(static_cast<long long>(x[1]));
    if (!both_fit(codes, value_codes, device) || codes.size(2) != kv_heads || codes.size(3) != dim || kv_heads <= 0 || heads <= 0 || heads % kv_heads ||
        q.dim() != 2 || q.size(1) != heads * dim || q.sizes() != out.sizes() || !dense(q, type, device) || !dense(out, type, device) ||
        !on_16_bytes(q) || !on_16_bytes(out) || table.dim() != 2 || !dense(table, at::kInt, device))
      Py_RETURN_NONE;
    const long long sequences = table.size(0);
    if (!ints(starts, sequences + 1, device) || !ints(context, sequences, device)) Py_RETURN_NONE;
    auto at = [](const at::Tensor& y) { return static_cast<unsigned long long>(reinterpret_cast<uintptr_t>(y.data_ptr())); };
    return Py_BuildValue("LLLK(KKKKKKKK)", static_cast<long long>(q.size(0)), sequences, static_cast<long long>(table.size(1)), at(out), at(q), at(codes),
                         at(key_scales), at(value_codes), at(value_scales), at(table), at(starts), at(context));
  });
}

template <typename F> PyCFunction function(F f) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }
PyMethodDef methods[] = {{"pages", function(look_pages), METH_FASTCALL, nullptr},
                         {"cache", function(look_cache), METH_FASTCALL, nullptr},
                         {"attention", function(look_attention), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "shrike_tensor_look", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_shrike_tensor_look() { return PyModule_Create(&module); }
