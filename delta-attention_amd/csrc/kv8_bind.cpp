// The Python entry of the 8-bit cache's calls (delta_attention.ops.kv8_*): the
// checks of their tensors and the packing of the C ABI's structs, as one
// extension function each. A decode step's append takes 3 us on the GPU and one
// of its rows 8; the same checks and calls from Python take 8 and 11 us of the
// host's time, here 1 to 2.
#include "bind_common.h"

namespace {

// The library's functions and _lib.check, handed over once by bind().
int (*g_write)(const da_kv8_write_args*, void*);
int (*g_read)(const da_kv8_read_args*, void*);
int (*g_attn)(const da_kv8_attn_args*, void*);
size_t (*g_attn_bytes)(int, int, int, int, int, int, int, int);

// One layer's cache: the tuple (k, v, k_scale, v_scale) of ops.KV8.
da_kv8_cache cache_of(PyObject* o, c10::Device dev) {
  REQUIRE(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 4, "an ops.KV8 cache is needed");
  const at::Tensor &k = tensor(PyTuple_GET_ITEM(o, 0), "cache.k"), &v = tensor(PyTuple_GET_ITEM(o, 1), "cache.v"),
                   &ks = tensor(PyTuple_GET_ITEM(o, 2), "cache.k_scale"), &vs = tensor(PyTuple_GET_ITEM(o, 3), "cache.v_scale");
  REQUIRE(k.dim() == 4 && v.dim() == 5 && ks.dim() == 3 && vs.dim() == 3, "a cache's tensors have 4, 5, 3 and 3 dimensions");
  const int64_t B = k.size(0), H = k.size(1), cap = k.size(2), D = k.size(3), nb = cap / 64;
  REQUIRE(H >= 1, "a cache has one kv head at least");
  REQUIRE(cap % 64 == 0 && v.sizes() == at::IntArrayRef({B, H, nb, D, 64}) && ks.sizes() == at::IntArrayRef({B, H, nb}) &&
              vs.sizes() == ks.sizes(), "a cache's shapes do not belong together: ", k.sizes(), v.sizes(), ks.sizes(), vs.sizes());
  REQUIRE(k.scalar_type() == at::kFloat8_e4m3fn && v.scalar_type() == at::kFloat8_e4m3fn && ks.scalar_type() == at::kFloat &&
              vs.scalar_type() == at::kFloat, "a cache's codes are float8_e4m3fn, its scales float32");
  REQUIRE(k.stride(3) == 1 && k.stride(2) == D && v.stride(4) == 1 && v.stride(3) == 64 && v.stride(2) == D * 64 &&
              (nb <= 1 || (ks.stride(2) == 1 && vs.stride(2) == 1)),
          "a cache's tokens, blocks and scales must be contiguous within a head");
  REQUIRE(k.device() == dev && v.device() == dev && ks.device() == dev && vs.device() == dev,
          "all tensors must be on one device");
  return da_kv8_cache{k.data_ptr(), v.data_ptr(), (float*)ks.data_ptr(), (float*)vs.data_ptr(),
                      {k.stride(0), k.stride(1)}, {v.stride(0), v.stride(1)}, {ks.stride(0), ks.stride(1)},
                      {vs.stride(0), vs.stride(1)}, narrow(B, "sequences"), narrow(H, "kv heads"),
                      narrow(cap, "capacity"), narrow(D, "head_dim")};
}

// (cache, k, v, pos, counts)
PyObject* write(PyObject* const* a) {
  const at::Tensor &k0 = tensor(a[1], "k"), &v0 = tensor(a[2], "v");
  const c10::Device dev = k0.device();
  da_kv8_write_args x{};
  x.cache = cache_of(a[0], dev);
  const int64_t B = x.cache.B;
  REQUIRE(k0.dim() == 4 && k0.sizes() == v0.sizes() && k0.size(0) == B && k0.size(2) == x.cache.Hkv && k0.size(3) == x.cache.D,
          "k and v are [", B, ", S, ", x.cache.Hkv, ", ", x.cache.D, "], got ", k0.sizes(), " and ", v0.sizes());
  REQUIRE(k0.scalar_type() == v0.scalar_type(), "k and v have different types");
  REQUIRE(v0.device() == dev, "all tensors must be on one device");
  x.dtype = dtype_code(k0.scalar_type());
  on_gpu(dev);
  x.S = narrow(k0.size(1), "tokens");
  if (THPVariable_Check(a[3])) {
    x.pos_dev = entries<int64_t>(a[3], B, at::kLong, dev, "pos", x.pos_per_seq);
  } else {
    x.pos = integer(a[3]);
    REQUIRE(x.pos >= 0 && x.pos <= (int64_t)x.cache.cap - x.S, "rows ", x.pos, " .. ", x.pos, " + ", x.S,
            " do not fit a cache of ", x.cache.cap);
  }
  x.counts_dev = entries<int32_t>(a[4], B, at::kInt, dev, "counts", x.counts_per_seq);
  if (B == 0 || x.S == 0) Py_RETURN_NONE;
  const On on(dev);
  const at::Tensor k = ready(k0), v = ready(v0);
  x.k = k.data_ptr();
  x.v = v.data_ptr();
  strides3(x.k_str, k);
  strides3(x.v_str, v);
  check(g_write(&x, on.stream()), "da_kv8_write");
  Py_RETURN_NONE;
}

// (cache, start, n, n_keys, dtype, (k out, v out) or None) -> (k, v)
PyObject* read(PyObject* const* a) {
  const bool given = a[5] != Py_None;
  REQUIRE(PyTuple_Check(a[0]) && PyTuple_GET_SIZE(a[0]) == 4, "an ops.KV8 cache is needed");
  const c10::Device dev = tensor(PyTuple_GET_ITEM(a[0], 0), "cache.k").device();
  da_kv8_read_args x{};
  x.cache = cache_of(a[0], dev);
  const int64_t start = integer(a[1]), n = integer(a[2]), B = x.cache.B;
  REQUIRE(start >= 0 && n >= 0 && start <= x.cache.cap - n, "rows ", start, " .. ", start, " + ", n, " of a cache of ", x.cache.cap);
  at::Tensor k, v;
  if (given) {
    REQUIRE(PyTuple_Check(a[5]) && PyTuple_GET_SIZE(a[5]) == 2, "out: two tensors are needed");
    k = tensor(PyTuple_GET_ITEM(a[5], 0), "k");
    v = tensor(PyTuple_GET_ITEM(a[5], 1), "v");
    REQUIRE(k.sizes() == at::IntArrayRef({B, (int64_t)x.cache.Hkv, n, (int64_t)x.cache.D}) && v.sizes() == k.sizes() &&
                k.scalar_type() == v.scalar_type() && k.stride(3) == 1 && v.stride(3) == 1,
            "the results are two [", B, ", ", x.cache.Hkv, ", ", n, ", ", x.cache.D, "] tensors of one type, got ", k.sizes(), v.sizes());
    REQUIRE(k.device() == dev && v.device() == dev, "all tensors must be on one device");
    x.dtype = dtype_code(k.scalar_type());
    on_gpu(dev);
  } else {
    REQUIRE(THPDtype_Check(a[4]), "dtype: a torch.dtype is needed");
    const at::ScalarType type = ((THPDtype*)a[4])->scalar_type;
    x.dtype = dtype_code(type);
    on_gpu(dev);
    // (two allocations: views of one would share a version, and keep each other's memory)
    const auto options = at::TensorOptions().dtype(type).device(dev);
    k = at::empty({B, x.cache.Hkv, n, x.cache.D}, options);
    v = at::empty({B, x.cache.Hkv, n, x.cache.D}, options);
  }
  x.n_keys_dev = entries<int32_t>(a[3], B, at::kInt, dev, "n_keys", x.n_keys_per_seq);
  if (B > 0 && n > 0) {
    x.start = (int32_t)start;
    x.n = (int32_t)n;
    x.k = k.data_ptr();
    x.v = v.data_ptr();
    strides3(x.k_str, k);
    strides3(x.v_str, v);
    const On on(dev);
    check(g_read(&x, on.stream()), "da_kv8_read");
  }
  if (given) return new_ref(a[5]);
  PyObject* result = PyTuple_New(2);
  if (!result) throw PythonError();
  PyTuple_SET_ITEM(result, 0, THPVariable_Wrap(std::move(k)));
  PyTuple_SET_ITEM(result, 1, THPVariable_Wrap(std::move(v)));
  return result;
}

// (q, cache, n_keys, window, sink, sm_scale, out or None, add or None) -> out
PyObject* attention(PyObject* const* a) {
  const at::Tensor& q0 = tensor(a[0], "q");
  const c10::Device dev = q0.device();
  da_kv8_attn_args x{};
  x.cache = cache_of(a[1], dev);
  const int64_t B = x.cache.B, cap = x.cache.cap;
  REQUIRE(q0.dim() == 4 && q0.size(0) == B && q0.size(3) == x.cache.D && q0.size(1) > 0 && q0.size(1) % x.cache.Hkv == 0,
          "q is [", B, ", heads (a multiple of ", x.cache.Hkv, "), rows, ", x.cache.D, "], got ", q0.sizes());
  x.dtype = dtype_code(q0.scalar_type());
  on_gpu(dev);
  x.Hq = narrow(q0.size(1), "heads");
  x.s = narrow(q0.size(2), "rows");
  x.n_keys = x.cache.cap;
  if (THPVariable_Check(a[2])) {
    x.n_keys_dev = entries<int32_t>(a[2], B, at::kInt, dev, "n_keys", x.n_keys_per_seq);
  } else {
    const int64_t n = integer(a[2]);
    REQUIRE(n >= 0 && n <= cap, n, " keys in a cache of ", cap);
    x.n_keys = (int32_t)n;
  }
  const int64_t window = integer(a[3]), sink = integer(a[4]);
  x.window = (int32_t)std::min(std::max<int64_t>(window, 0), cap);
  x.sink = (int32_t)std::min(std::max<int64_t>(sink, 0), cap);
  const double scale = PyFloat_AsDouble(a[5]);
  if (scale == -1.0 && PyErr_Occurred()) throw PythonError();
  x.sm_scale = (float)scale;
  const On on(dev);
  const at::Tensor q = ready(q0);
  at::Tensor out, add, ws;
  if (a[6] == Py_None) {
    out = at::empty_like(q);
  } else {
    out = tensor(a[6], "out");
    REQUIRE(out.sizes() == q.sizes() && out.scalar_type() == q.scalar_type() && out.device() == dev && out.stride(3) == 1,
            "out: a tensor like q is needed");
  }
  if (a[7] != Py_None) {
    const at::Tensor& t = tensor(a[7], "add");
    REQUIRE(t.sizes() == q.sizes() && t.scalar_type() == q.scalar_type() && t.device() == dev, "add: a tensor like q is needed");
    add = ready(t);
    x.addend = add.data_ptr();
    strides3(x.add_str, add);
  }
  if (B > 0 && x.s > 0) {
    x.q = q.data_ptr();
    x.out = out.data_ptr();
    strides3(x.q_str, q);
    strides3(x.o_str, out);
    const size_t bytes = g_attn_bytes(x.cache.B, x.Hq, x.cache.Hkv, x.s, x.cache.D, x.n_keys, x.window, x.sink);
    if (bytes > 0) {
      ws = at::empty({(int64_t)bytes}, q.options().dtype(at::kByte));
      x.workspace = ws.data_ptr();
      x.workspace_bytes = (int64_t)bytes;
    }
    check(g_attn(&x, on.stream()), "da_kv8_attn_fwd");
  }
  if (a[6] != Py_None) return new_ref(a[6]);
  return THPVariable_Wrap(out);
}

// (addresses of da_kv8_write, da_kv8_read, da_kv8_attn_fwd,
// da_kv8_attn_workspace_bytes; _lib.check)
PyObject* bind(PyObject* const* a) {
  auto address = [](PyObject* o) { return (void*)(uintptr_t)integer(o); };
  g_write = (decltype(g_write))address(a[0]);
  g_read = (decltype(g_read))address(a[1]);
  g_attn = (decltype(g_attn))address(a[2]);
  g_attn_bytes = (decltype(g_attn_bytes))address(a[3]);
  Py_XSETREF(g_check, new_ref(a[4]));
  Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", (PyCFunction)(void (*)(void))entry<bind, 5>, METH_FASTCALL, nullptr},
    {"write", (PyCFunction)(void (*)(void))entry<write, 5>, METH_FASTCALL, nullptr},
    {"read", (PyCFunction)(void (*)(void))entry<read, 6>, METH_FASTCALL, nullptr},
    {"attention", (PyCFunction)(void (*)(void))entry<attention, 8>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_kv8_ext", "The 8-bit cache's calls.", -1, g_methods,
                        nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__kv8_ext(void) { return PyModule_Create(&g_module); }
