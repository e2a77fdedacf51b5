// binding.cpp -- the serving operators' calls from Python (_binding.so): checks of
// the tensors, allocation of outputs and the C-ABI call in one step.  A decode
// step's kernels run for 4 to 20 us, and the same work through ctypes and the
// tensors' Python methods took 11 to 17 us a call; here it is 4 to 6.  Arguments
// are positional; serving.py holds the public functions and their documentation.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <exception>

#include "../../include/qgemm_b200.h"

namespace {

using at::Tensor;

// A failed check: the ValueError is set, the call returns null.
struct Refused {};

[[noreturn]] void refuse(const char* where, const char* what) {
  PyErr_Format(PyExc_ValueError, "%s: %s", where, what);
  throw Refused{};
}
const Tensor& tensor(PyObject* o, const char* where, const char* what) {
  if (!THPVariable_Check(o)) refuse(where, what);
  return THPVariable_Unpack(o);
}
bool given(PyObject* o) { return o != Py_None; }
int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Refused{};
  return v;
}
// A number that the C-ABI takes as int32.
int32_t small(PyObject* o, const char* where) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse(where, "a size exceeds 2^31 - 1");
  return (int32_t)v;
}
int32_t fits(int64_t v, const char* where) {
  if (v > INT32_MAX) refuse(where, "a size exceeds 2^31 - 1");
  return (int32_t)v;
}
// On the GPU that the call goes by.
bool on(const Tensor& t, c10::DeviceIndex device) { return t.is_cuda() && t.get_device() == device; }
bool ints(const Tensor& t, c10::DeviceIndex device, int64_t dims = 1) {
  return t.scalar_type() == at::kInt && t.dim() == dims && on(t, device) && t.is_contiguous();
}
template <typename P = int32_t>
P* ptr(const Tensor& t) { return static_cast<P*>(t.data_ptr()); }
// The call's device, and its stream: the current one, or the one given (a
// cudaStream_t as an integer), which is made current so that outputs are allocated
// for it.
struct Place {
  c10::cuda::OptionalCUDAGuard device;
  c10::cuda::OptionalCUDAStreamGuard guard;
  void* stream;
  Place(PyObject* s, const Tensor& t) {
    if (given(s)) {
      void* p = PyLong_AsVoidPtr(s);
      if (!p && PyErr_Occurred()) throw Refused{};
      guard.reset_stream(c10::cuda::getStreamFromExternal(static_cast<cudaStream_t>(p), t.get_device()));
      stream = p;
    } else {
      device.set_device(t.device());
      stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
    }
  }
};
Tensor make(at::IntArrayRef sizes, at::ScalarType type, const Tensor& like) {
  return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt);
}
// Tensors of one dimension in one allocation, each on a 16-byte boundary: a plan's
// six, made one by one, took 3 us longer.
template <size_t N>
void make_together(Tensor (&out)[N], const int64_t (&sizes)[N], const at::ScalarType (&types)[N], const Tensor& like) {
  int64_t at[N], bytes = 0;
  for (size_t i = 0; i < N; ++i) {
    at[i] = bytes;
    bytes += (sizes[i] * (int64_t)c10::elementSize(types[i]) + 15) / 16 * 16;
  }
  const Tensor whole = make({bytes}, at::kByte, like);
  for (size_t i = 0; i < N; ++i) {
    out[i] = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(whole.storage()), whole.key_set(),
                                                      c10::scalarTypeToTypeMeta(types[i]));
    c10::TensorImpl* t = out[i].unsafeGetTensorImpl();
    t->set_storage_offset(at[i] / (int64_t)c10::elementSize(types[i]));
    t->set_sizes_contiguous({sizes[i]});
  }
}
// (status, result...): serving.py turns a status other than 0 into its error.
PyObject* done(int status, std::initializer_list<const Tensor*> out) {
  PyObject* r = PyTuple_New((Py_ssize_t)out.size() + 1);
  if (!r) return nullptr;
  PyTuple_SET_ITEM(r, 0, PyLong_FromLong(status));
  Py_ssize_t i = 1;
  for (const Tensor* t : out) {
    PyObject* o = t->defined() ? THPVariable_Wrap(*t) : Py_NewRef(Py_None);
    if (!o) { Py_DECREF(r); return nullptr; }
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}
// Runs a call's body; nothing of C++ leaves it.
template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refused&) {
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}
bool count_is(Py_ssize_t n, Py_ssize_t want, const char* where) {
  if (n == want) return true;
  PyErr_Format(PyExc_TypeError, "%s: %zd arguments expected", where, want);
  return false;
}
// A KVCache's description: the C-ABI's, and the GPU it lies on (-1: none).
struct Cache {
  qgemm_kv_cache_t c;
  int64_t device;
};
const Cache* cache_of(PyObject* o, const char* where) {
  if (!PyBytes_Check(o) || PyBytes_GET_SIZE(o) != (Py_ssize_t)sizeof(Cache)) refuse(where, "not a KVCache");
  const Cache* c = reinterpret_cast<const Cache*>(PyBytes_AS_STRING(o));
  if (c->device < 0) refuse(where, "the cache must be on a GPU");
  return c;
}

// kv_cache(type, k, v, k_scales, v_scales) -> bytes of a Cache
PyObject* kv_cache(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (!count_is(n, 5, "KVCache")) return nullptr;
  return guarded([&]() -> PyObject* {
    const char* codes = "k and v must be contiguous uint8 tensors of one shape [blocks, heads, block, head_dim]";
    const char* scales = "k_scales and v_scales must be contiguous uint8 [blocks, heads]";
    const Tensor &k = tensor(a[1], "KVCache", codes), &v = tensor(a[2], "KVCache", codes);
    const Tensor &ks = tensor(a[3], "KVCache", scales), &vs = tensor(a[4], "KVCache", scales);
    for (const Tensor* t : {&k, &v})
      if (t->dim() != 4 || t->scalar_type() != at::kByte || !t->is_contiguous() || t->sizes() != k.sizes() ||
          t->device() != k.device())
        refuse("KVCache", codes);
    for (const Tensor* t : {&ks, &vs})
      if (t->dim() != 2 || t->scalar_type() != at::kByte || !t->is_contiguous() || t->size(0) != k.size(0) ||
          t->size(1) != k.size(1) || t->device() != k.device())
        refuse("KVCache", scales);
    Cache whole;
    std::memset(&whole, 0, sizeof(whole));
    whole.device = k.is_cuda() ? k.get_device() : -1;
    qgemm_kv_cache_t& c = whole.c;
    c.type = small(a[0], "KVCache");
    c.block = fits(k.size(2), "KVCache"); c.heads = fits(k.size(1), "KVCache"); c.head_dim = fits(k.size(3), "KVCache");
    c.blocks = k.size(0);
    c.k = ptr<uint8_t>(k); c.v = ptr<uint8_t>(v); c.k_scales = ptr<uint8_t>(ks); c.v_scales = ptr<uint8_t>(vs);
    return PyBytes_FromStringAndSize(reinterpret_cast<const char*>(&whole), sizeof(whole));
  });
}

// kv_plan(lens, new, table, free_list, free_count, block, tokens, out, stream) ->
// (status, starts, lens, slots, positions, runs, counts); out: None or those six
PyObject* kv_plan(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr const char* W = "kv_plan";
  if (!count_is(n, 9, W)) return nullptr;
  return guarded([&]() -> PyObject* {
    const char* what =
        "lens, new, table [requests, width], free_list and free_count must be contiguous int32 CUDA tensors on one GPU";
    const Tensor &lens = tensor(a[0], W, what), &news = tensor(a[1], W, what), &table = tensor(a[2], W, what);
    const Tensor &list = tensor(a[3], W, what), &count = tensor(a[4], W, what);
    const auto gpu = lens.is_cuda() ? lens.get_device() : -1;
    if (!ints(lens, gpu) || !ints(news, gpu) || !ints(table, gpu, 2) || !ints(list, gpu) || !ints(count, gpu))
      refuse(W, what);
    const int32_t requests = fits(table.size(0), W), width = fits(table.size(1), W);
    if (lens.numel() != requests || news.numel() != requests || count.numel() != 1)
      refuse(W, "new, table and free_count must have one entry per request, row per request, and one element");
    const int32_t block = small(a[5], W), tokens = small(a[6], W);
    const int32_t most = qgemm_kv_max_runs(requests, tokens, block);
    if (most < 0) refuse(W, "block must be 16, 32, 64 or 128 and tokens not negative");
    const Place place(a[8], lens);
    Tensor o[6];
    const int64_t sizes[6] = {requests + 1ll, requests, tokens, tokens, most + 1ll, 4};
    if (given(a[7])) {
      if (!PyTuple_Check(a[7]) || PyTuple_GET_SIZE(a[7]) != 6) refuse(W, "out must be a KVPlan");
      for (int i = 0; i < 6; ++i) {
        o[i] = tensor(PyTuple_GET_ITEM(a[7], i), W, "out must hold tensors");
        if (o[i].numel() != sizes[i] || o[i].scalar_type() != (i == 2 ? at::kLong : at::kInt) || !on(o[i], gpu) ||
            !o[i].is_contiguous())
          refuse(W, "out was made for other sizes or another GPU");
      }
    } else {
      make_together(o, sizes, {at::kInt, at::kInt, at::kLong, at::kInt, at::kInt, at::kInt}, lens);
    }
    const int st = qgemm_kv_plan_bounded(block, requests, ptr(lens), ptr(news), ptr(table), width, ptr(list),
                                         fits(list.numel(), W), ptr(count), tokens, ptr(o[1]), ptr(o[0]),
                                         ptr<int64_t>(o[2]), ptr(o[3]), ptr(o[4]), ptr(o[5]), place.stream);
    return done(st, {&o[0], &o[1], &o[2], &o[3], &o[4], &o[5]});
  });
}

// bf16 [tokens, heads, head_dim] rows with any spacing of tokens and heads.
void check_rows(const Tensor& t, const Cache* c, const char* where, const char* what) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 3 || !on(t, c->device) || t.size(2) != c->c.head_dim)
    refuse(where, what);
  if (t.stride(2) != 1 && t.numel()) refuse(where, "the head_dim values of a row must lie together");
}

// kv_append(cache, k, v, slots, runs, stream) -> (status,)
PyObject* kv_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr const char* W = "kv_append";
  if (!count_is(n, 6, W)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache* cache = cache_of(a[0], W);
    const qgemm_kv_cache_t* c = &cache->c;
    const char* what = "k and v must be bf16 [tokens, heads, head_dim] of the cache, on its GPU";
    const char* index =
        "slots (int64) and runs (int32, with an end mark) must be contiguous on the cache's GPU, one slot a token";
    const Tensor &k = tensor(a[1], W, what), &v = tensor(a[2], W, what);
    const Tensor &slots = tensor(a[3], W, index), &runs = tensor(a[4], W, index);
    check_rows(k, cache, W, what);
    check_rows(v, cache, W, what);
    if (k.size(1) != c->heads || v.size(1) != c->heads || v.size(0) != k.size(0)) refuse(W, what);
    if (slots.scalar_type() != at::kLong || !on(slots, cache->device) || slots.numel() != k.size(0) ||
        !slots.is_contiguous() || !ints(runs, cache->device) || runs.numel() < 1)
      refuse(W, index);
    const Place place(a[5], k);
    const int st = qgemm_kv_append(c, ptr<uint16_t>(k), ptr<uint16_t>(v), k.stride(0), k.stride(1), v.stride(0),
                                   v.stride(1), fits(k.size(0), W), ptr<int64_t>(slots), ptr(runs),
                                   fits(runs.numel() - 1, W), place.stream);
    return done(st, {});
  });
}

// kv_attention(cache, q, starts, lens, table, max_new, scale, window, causal, lse, out,
// workspace, stream) -> (status, out, lse or None)
PyObject* kv_attention(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr const char* W = "kv_attention";
  if (!count_is(n, 13, W)) return nullptr;
  return guarded([&]() -> PyObject* {
    const Cache* cache = cache_of(a[0], W);
    const qgemm_kv_cache_t* c = &cache->c;
    const auto gpu = cache->device;
    const char* rows = "q must be bf16 [tokens, heads, head_dim] with the cache's head_dim, on its GPU";
    const char* index = "starts, lens and table [requests, width] must be contiguous int32 on the cache's GPU";
    const Tensor& q = tensor(a[1], W, rows);
    const Tensor &starts = tensor(a[2], W, index), &lens = tensor(a[3], W, index), &table = tensor(a[4], W, index);
    check_rows(q, cache, W, rows);
    if (!ints(starts, gpu) || !ints(lens, gpu) || !ints(table, gpu, 2)) refuse(W, index);
    if (starts.numel() != lens.numel() + 1 || table.size(0) != lens.numel())
      refuse(W, "starts needs requests + 1 entries and table a row per request");
    const double scale = PyFloat_AsDouble(a[6]);
    if (scale == -1.0 && PyErr_Occurred()) throw Refused{};
    const int lse = PyObject_IsTrue(a[9]), causal = PyObject_IsTrue(a[8]);
    if (lse < 0 || causal < 0) throw Refused{};
    const Place place(a[12], q);
    Tensor out, z;
    if (given(a[10])) {
      out = tensor(a[10], W, "out must be a tensor");
      if (out.sizes() != q.sizes() || out.scalar_type() != at::kBFloat16 || !on(out, gpu) || !out.is_contiguous())
        refuse(W, "out must be contiguous bf16 of q's shape on its GPU");
    } else {
      out = make(q.sizes(), at::kBFloat16, q);
    }
    if (lse) z = make({q.size(0), q.size(1)}, at::kFloat, q);
    const Tensor& ws = tensor(a[11], W, "workspace must be a tensor");
    if (!on(ws, gpu) || !ws.is_contiguous()) refuse(W, "workspace must be contiguous on the cache's GPU");
    const int st = qgemm_kv_attention(
        c, ptr<uint16_t>(q), q.stride(0), q.stride(1), fits(q.size(1), W), fits(lens.numel(), W), ptr(starts), ptr(lens),
        ptr(table), fits(table.size(1), W), fits(q.size(0), W), small(a[5], W), (float)scale, small(a[7], W), causal,
        ptr<uint16_t>(out), lse ? ptr<float>(z) : nullptr, ws.data_ptr(), ws.nbytes(), place.stream);
    return done(st, {&out, &z});
  });
}

// residual_norm(y, residual, post, pre, post_bias, pre_bias, gate, alpha, kind, eps,
// residual_out, h, stream) -> (status, residual_out, h or None)
PyObject* residual_norm(PyObject*, PyObject* const* a, Py_ssize_t n) {
  constexpr const char* W = "residual_norm";
  if (!count_is(n, 13, W)) return nullptr;
  return guarded([&]() -> PyObject* {
    const char* stream_rows = "residual must be contiguous bf16 or float32 [tokens, width] on the GPU";
    const char* rows = "y and h must be contiguous bf16 [tokens, width] on residual's GPU";
    const char* weights = "post, pre and their biases must be contiguous bf16 [width] on residual's GPU";
    const char* gates = "gate must be bf16 [width] or [tokens, width] on residual's GPU";
    const Tensor& r = tensor(a[1], W, stream_rows);
    const auto type = r.scalar_type();
    if (r.dim() != 2 || (type != at::kBFloat16 && type != at::kFloat) || !r.is_cuda() || !r.is_contiguous())
      refuse(W, stream_rows);
    const int64_t width = r.size(1);
    const auto gpu = r.get_device();
    qgemm_residual_norm_t p;
    std::memset(&p, 0, sizeof(p));
    p.kind = small(a[8], W);
    p.tokens = fits(r.size(0), W); p.width = fits(width, W);
    p.residual_f32 = type == at::kFloat;
    p.residual = r.data_ptr();
    auto row = [&](PyObject* o) -> uint16_t* {
      if (!given(o)) return nullptr;
      const Tensor& t = tensor(o, W, rows);
      if (t.scalar_type() != at::kBFloat16 || t.sizes() != r.sizes() || !on(t, gpu) || !t.is_contiguous()) refuse(W, rows);
      return ptr<uint16_t>(t);
    };
    auto weight = [&](PyObject* o) -> const uint16_t* {
      if (!given(o)) return nullptr;
      const Tensor& t = tensor(o, W, weights);
      if (t.scalar_type() != at::kBFloat16 || t.dim() != 1 || t.numel() != width || !on(t, gpu) || !t.is_contiguous())
        refuse(W, weights);
      return ptr<uint16_t>(t);
    };
    p.y = row(a[0]);
    const bool has_y = given(a[0]);
    p.post = weight(a[2]); p.pre = weight(a[3]); p.post_bias = weight(a[4]); p.pre_bias = weight(a[5]);
    if (given(a[6])) {
      const Tensor& g = tensor(a[6], W, gates);
      const bool each = g.dim() == 2;
      if (g.scalar_type() != at::kBFloat16 || !on(g, gpu) || (each ? g.sizes() != r.sizes() : g.dim() != 1 || g.numel() != width) ||
          (g.stride(-1) != 1 && width > 1))
        refuse(W, gates);
      p.gate = ptr<uint16_t>(g);
      p.gate_stride = each ? g.stride(0) : 0;
    }
    p.alpha = (float)PyFloat_AsDouble(a[7]);
    p.eps = (float)PyFloat_AsDouble(a[9]);
    if (PyErr_Occurred()) throw Refused{};
    const Place place(a[12], r);
    Tensor out, h;
    if (!has_y) {
      out = r;
    } else if (given(a[10])) {
      out = tensor(a[10], W, "residual_out must be like residual, on its GPU");
      if (out.sizes() != r.sizes() || out.scalar_type() != type || !on(out, gpu) || !out.is_contiguous())
        refuse(W, "residual_out must be like residual, on its GPU");
    } else {
      out = make(r.sizes(), type, r);
    }
    p.residual_out = out.data_ptr();
    if (p.pre || given(a[3])) {
      if (given(a[11])) {
        p.h = row(a[11]);
        h = THPVariable_Unpack(a[11]);
      } else {
        h = make(r.sizes(), at::kBFloat16, r);
        p.h = ptr<uint16_t>(h);
      }
    }
    return done(qgemm_residual_norm(&p, place.stream), {&out, &h});
  });
}

PyMethodDef methods[] = {
    {"kv_cache", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv_cache)), METH_FASTCALL, nullptr},
    {"kv_plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv_plan)), METH_FASTCALL, nullptr},
    {"kv_append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv_append)), METH_FASTCALL, nullptr},
    {"kv_attention", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(kv_attention)), METH_FASTCALL, nullptr},
    {"residual_norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(residual_norm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() { return PyModule_Create(&module); }
