// The Python entry of the generation calls (delta_attention.ops.sample_tokens and
// prefix_attention):
// the checks of their tensors and the packing of the C ABI's structs, as one
// extension function each, for the same reason as the 8-bit cache's: a decode
// step's calls are shorter on the GPU than their checks in Python.
#include "bind_common.h"

namespace {

// The library's functions, handed over once by bind().
int (*g_sample)(const da_sample_args*, void*);
size_t (*g_sample_bytes)(int, int, int);
int (*g_prefix)(const da_prefix_attn_args*, void*);
size_t (*g_prefix_bytes)(int, int, int, int, int, int, int, int);

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

// Key counts: a device tensor (one entry, or one for each of N), or a number up to
// the capacity; None is all of them.
const int32_t* counts(PyObject* o, int64_t N, int32_t most, c10::Device dev, const char* what, int32_t& per, int32_t& value) {
  value = most;
  if (o == Py_None || THPVariable_Check(o)) return entries<int32_t>(o, N, at::kInt, dev, what, per);
  const int64_t n = integer(o);
  REQUIRE(n >= 0 && n <= most, what, ": ", n, " of ", most, " keys");
  value = (int32_t)n;
  return nullptr;
}

// (q, k_prefix, v_prefix, k, v, n_prefix, n_keys, sm_scale, out or None) -> out
PyObject* prefix(PyObject* const* a) {
  const char* names[] = {"q", "k_prefix", "v_prefix", "k", "v"};
  const at::Tensor* t[5];
  for (int i = 0; i < 5; ++i) {
    t[i] = &tensor(a[i], names[i]);
    REQUIRE(t[i]->dim() == 4, names[i], ": four dimensions are needed, got ", t[i]->sizes());
    REQUIRE(t[i]->scalar_type() == t[0]->scalar_type(), names[i], " and q have different types");
    REQUIRE(t[i]->device() == t[0]->device(), "all tensors must be on one device");
  }
  const at::Tensor &q0 = *t[0], &kp0 = *t[1], &k0 = *t[3];
  const c10::Device dev = q0.device();
  da_prefix_attn_args x{};
  const int64_t B = q0.size(0), P = kp0.size(0), Hkv = kp0.size(1), D = q0.size(3);
  REQUIRE(P > 0 && B % P == 0, "a batch of ", B, " sequences does not share ", P, " prefixes alike");
  REQUIRE(Hkv > 0 && q0.size(1) > 0 && q0.size(1) % Hkv == 0, q0.size(1), " query heads of ", Hkv, " kv heads");
  REQUIRE(kp0.size(3) == D && t[2]->sizes() == kp0.sizes(), "k_prefix and v_prefix are [prefixes, kv heads, keys, ", D,
          "], got ", kp0.sizes(), " and ", t[2]->sizes());
  REQUIRE(k0.size(0) == B && k0.size(1) == Hkv && k0.size(3) == D && t[4]->sizes() == k0.sizes(), "k and v are [", B, ", ",
          Hkv, ", keys, ", D, "], got ", k0.sizes(), " and ", t[4]->sizes());
  x.dtype = dtype_code(q0.scalar_type());
  on_gpu(dev);
  x.B = narrow(B, "sequences"), x.P = narrow(P, "prefixes"), x.Hq = narrow(q0.size(1), "heads");
  x.Hkv = narrow(Hkv, "kv heads"), x.s = narrow(q0.size(2), "rows"), x.D = narrow(D, "head_dim");
  x.max_prefix = narrow(kp0.size(2), "prefix keys"), x.max_keys = narrow(k0.size(2), "keys");
  x.n_prefix_dev = counts(a[5], P, x.max_prefix, dev, "n_prefix", x.n_prefix_per, x.n_prefix);
  x.n_keys_dev = counts(a[6], B, x.max_keys, dev, "n_keys", x.n_keys_per_seq, x.n_keys);
  x.sm_scale = (float)number(a[7], "sm_scale");
  const On on(dev);
  at::Tensor in[5], out, ws;
  for (int i = 0; i < 5; ++i) {
    // (keys that share their places, as one key read as many does, are copied too)
    const bool apart = i == 0 || t[i]->size(2) <= 1 || t[i]->stride(2) >= D;
    in[i] = apart ? ready(*t[i]) : t[i]->clone(at::MemoryFormat::Contiguous);
  }
  if (a[8] == Py_None) {
    out = at::empty_like(in[0]);
  } else {
    out = tensor(a[8], "out");
    REQUIRE(out.sizes() == q0.sizes() && out.scalar_type() == q0.scalar_type() && out.device() == dev && out.stride(3) == 1,
            "out: a tensor like q is needed");
  }
  if (B > 0 && x.s > 0) {
    x.q = in[0].data_ptr(), x.k_prefix = in[1].data_ptr(), x.v_prefix = in[2].data_ptr();
    x.k = in[3].data_ptr(), x.v = in[4].data_ptr(), x.out = out.data_ptr();
    strides3(x.q_str, in[0]), strides3(x.kp_str, in[1]), strides3(x.vp_str, in[2]);
    strides3(x.k_str, in[3]), strides3(x.v_str, in[4]), strides3(x.o_str, out);
    const size_t bytes = g_prefix_bytes(x.B, x.P, x.Hq, x.Hkv, x.s, x.D, x.max_prefix, x.max_keys);
    if (bytes > 0) {
      ws = at::empty({(int64_t)bytes}, q0.options().dtype(at::kByte));
      x.workspace = ws.data_ptr();
      x.workspace_bytes = (int64_t)bytes;
    }
    check(g_prefix(&x, on.stream()), "da_prefix_attn_fwd");
  }
  if (a[8] != Py_None) return new_ref(a[8]);
  return THPVariable_Wrap(out);
}

// (addresses of da_sample, da_sample_workspace_bytes, da_prefix_attn_fwd,
// da_prefix_attn_workspace_bytes; _lib.check)
PyObject* bind(PyObject* const* a) {
  auto address = [](PyObject* o) { return (void*)(uintptr_t)integer(o); };
  g_sample = (decltype(g_sample))address(a[0]);
  g_sample_bytes = (decltype(g_sample_bytes))address(a[1]);
  g_prefix = (decltype(g_prefix))address(a[2]);
  g_prefix_bytes = (decltype(g_prefix_bytes))address(a[3]);
  Py_XSETREF(g_check, new_ref(a[4]));
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", (PyCFunction)(void (*)(void))entry<bind, 5>, METH_FASTCALL, nullptr},
    {"sample", (PyCFunction)(void (*)(void))entry<sample, 6>, METH_FASTCALL, nullptr},
    {"prefix", (PyCFunction)(void (*)(void))entry<prefix, 9>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_gen_ext", "The generation calls.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__gen_ext(void) { return PyModule_Create(&g_module); }
