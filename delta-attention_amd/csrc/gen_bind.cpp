// The Python entry of the generation calls (delta_attention.ops.sample_tokens):
// the checks of their tensors and the packing of the C ABI's structs, as one
// extension function each, for the same reason as the 8-bit cache's: a decode
// step's calls are shorter on the GPU than their checks in Python.
#include "bind_common.h"

namespace {

// The library's functions, handed over once by bind().
int (*g_sample)(const da_sample_args*, void*);
size_t (*g_sample_bytes)(int, int, int);

double number(PyObject* o, const char* what) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) throw PythonError();
  REQUIRE(x == x, what, ": a number is needed");
  return x;
}

// A setting of the rows: a device tensor of one entry or one per row, or a number
// in [lo, hi].
const float* setting(PyObject* o, int64_t B, c10::Device dev, const char* what, double lo, double hi, int32_t& per_row,
                     float& value) {
  if (THPVariable_Check(o)) return entries<float>(o, B, at::kFloat, dev, what, per_row);
  const double x = number(o, what);
  REQUIRE(x >= lo && x <= hi, what, ": ", x, " is not in [", lo, ", ", hi, "]");
  value = (float)x;
  return nullptr;
}

// (logits, u, temperature, top_k, top_p, min_p) -> (tokens, log-probabilities)
PyObject* sample(PyObject* const* a) {
  const at::Tensor &l0 = tensor(a[0], "logits"), &u = tensor(a[1], "u");
  const c10::Device dev = l0.device();
  da_sample_args x{};
  REQUIRE(l0.dim() == 2 && l0.size(1) > 0, "logits are [rows, tokens], got ", l0.sizes());
  const at::ScalarType type = l0.scalar_type();
  REQUIRE(type == at::kBFloat16 || type == at::kHalf || type == at::kFloat, "dtype ", type,
          " is not supported (bfloat16, float16, float32)");
  x.dtype = type == at::kFloat ? DA_FP32 : dtype_code(type);
  const int64_t B = l0.size(0);
  x.B = narrow(B, "rows");
  x.V = narrow(l0.size(1), "tokens");
  REQUIRE(u.scalar_type() == at::kFloat && u.dim() == 1 && u.numel() == B && u.is_contiguous() && u.device() == dev,
          "u: a contiguous float32 tensor of ", B, " entries on ", dev, " is needed, got ", u.scalar_type(), u.sizes(),
          " on ", u.device());
  on_gpu(dev);
  const double inf = std::numeric_limits<float>::max();
  x.temperature_dev = setting(a[2], B, dev, "temperature", 0, inf, x.temperature_per_row, x.temperature);
  if (THPVariable_Check(a[3])) x.top_k_dev = entries<int32_t>(a[3], B, at::kInt, dev, "top_k", x.top_k_per_row);
  else x.top_k = narrow(integer(a[3]), "top_k");
  x.top_p_dev = setting(a[4], B, dev, "top_p", 0, 1, x.top_p_per_row, x.top_p);
  x.min_p_dev = setting(a[5], B, dev, "min_p", 0, 1, x.min_p_per_row, x.min_p);
  const On on(dev);
  const at::Tensor logits = l0.stride(1) == 1 || x.V == 1 ? l0 : l0.contiguous();
  at::Tensor tokens = at::empty({B}, logits.options().dtype(at::kLong));
  at::Tensor logprobs = at::empty({B}, logits.options().dtype(at::kFloat));
  if (B > 0) {
    at::Tensor ws;
    x.logits = logits.data_ptr();
    x.row_stride = logits.stride(0);
    x.u = (const float*)u.data_ptr();
    x.tokens = (int64_t*)tokens.data_ptr();
    x.logprobs = (float*)logprobs.data_ptr();
    const size_t bytes = g_sample_bytes(x.B, x.V, x.dtype);
    if (bytes > 0) {
      ws = at::empty({(int64_t)bytes}, logits.options().dtype(at::kByte));
      x.workspace = ws.data_ptr();
      x.workspace_bytes = (int64_t)bytes;
    }
    check(g_sample(&x, on.stream()), "da_sample");
  }
  PyObject* result = PyTuple_New(2);
  if (!result) throw PythonError();
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(tokens)));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(logprobs)));
  return result;
}

// (addresses of da_sample, da_sample_workspace_bytes; _lib.check)
PyObject* bind(PyObject* const* a) {
  auto address = [](PyObject* o) { return (void*)(uintptr_t)integer(o); };
  g_sample = (decltype(g_sample))address(a[0]);
  g_sample_bytes = (decltype(g_sample_bytes))address(a[1]);
  Py_XSETREF(g_check, new_ref(a[2]));
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", (PyCFunction)(void (*)(void))entry<bind, 3>, METH_FASTCALL, nullptr},
    {"sample", (PyCFunction)(void (*)(void))entry<sample, 6>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_gen_ext", "The generation calls.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__gen_ext(void) { return PyModule_Create(&g_module); }
