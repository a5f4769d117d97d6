// The Python operators of the paged cache, in C++: argument checks, allocations and the call into the C ABI.  A step of generation is a few short calls a
// block; written in Python, one took 13 us of host time where the kernels take 7.  The kernels themselves are reached through the C ABI alone, whose
// functions this module is handed (init): it links to neither the library nor CUDA's tools.
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include "hyperattn_b200.h"

namespace {

using at::Tensor;

struct Abi {
  int (*append)(const ha_paged_params*, void*);
  int (*attn)(const ha_paged_params*, void*);
  int (*gather)(const ha_paged_params*, void*);
  int (*maps)(const ha_paged_params*, void*);
  int64_t (*workspace)(const ha_paged_params*);
} abi;

// What a PagedCache is to these functions: its parameters as checked, its tensors, the status words of its device.
struct Handle {
  ha_paged_params p;
  std::vector<Tensor> pages;
  std::vector<const void*> at;
  at::ScalarType dtype;
  at::Device device{at::kCPU};
  const volatile int32_t* failed;
  bool mapped = false;
  alignas(64) char maps[HA_PAGED_MAPS_BYTES];
};

struct Refused : std::exception {
  std::string text;
  explicit Refused(std::string t) : text(std::move(t)) {}
  const char* what() const noexcept override { return text.c_str(); }
};
inline void want(bool ok, const char* text) {
  if (C10_UNLIKELY(!ok)) throw Refused(text);
}

const char* NAME = "hyperattention_b200.paged_cache";
Handle& handle_of(PyObject* o) {
  void* h = PyCapsule_GetPointer(o, NAME);
  want(h != nullptr, "not a cache");
  return *static_cast<Handle*>(h);
}
const Tensor& tensor_of(PyObject* o, const char* text) {
  want(THPVariable_Check(o), text);
  return THPVariable_Unpack(o);
}

// Common to the calls: the cache's pages where they were, the table and the lengths of B sequences.
ha_paged_params start(Handle& h, const Tensor& table, const Tensor& lengths, const Tensor* counts, int64_t B) {
  for (size_t i = 0; i < h.pages.size(); ++i) want(h.pages[i].data_ptr() == h.at[i], "the pages have moved: make a new PagedCache");
  want(h.device.is_cuda(), "tensors must be CUDA tensors (there is no CPU implementation)");
  want(table.dim() == 2 && table.size(0) == B && table.scalar_type() == at::kInt && (table.stride(1) == 1 || table.size(1) <= 1),
       "table must be int32 [batch, columns], rows contiguous");
  want(lengths.dim() == 1 && lengths.size(0) == B && lengths.scalar_type() == at::kInt && lengths.is_contiguous(), "lengths must be contiguous int32 [batch]");
  want(table.device() == h.device && lengths.device() == h.device, "all tensors must be on one device");
  ha_paged_params p = h.p;
  if (counts) {
    want(counts->dim() == 1 && counts->size(0) == B && counts->scalar_type() == at::kInt && counts->is_contiguous() && counts->device() == h.device,
         "counts must be contiguous int32 [batch]");
    p.counts = static_cast<const int32_t*>(counts->data_ptr());
  }
  want(B <= INT32_MAX && table.size(1) <= INT32_MAX, "too many sequences or columns");
  p.B = (int32_t)B;
  p.columns = (int32_t)table.size(1);
  p.table_sb = table.size(0) > 1 ? table.stride(0) : table.size(1);
  p.table = static_cast<const int32_t*>(table.data_ptr());
  p.lengths = static_cast<const int32_t*>(lengths.data_ptr());
  return p;
}

void want_rows(const Handle& h, const Tensor& t, int64_t B, int64_t n, int64_t heads, const char* shape, const char* type) {
  want(t.dim() == 4 && t.size(0) == B && t.size(1) == n && t.size(2) == heads && t.size(3) == h.p.d, shape);
  want(t.scalar_type() == h.dtype && t.device() == h.device, type);
  want(!(t.requires_grad() && at::GradMode::is_enabled()), "the operators of the paged cache have no gradient: call them under torch.no_grad()");
}
// rows that are not contiguous are copied, as in HyperAttention
Tensor rows(const Tensor& t) { return t.dim() == 0 || t.size(t.dim() - 1) <= 1 || t.stride(t.dim() - 1) == 1 ? t : t.contiguous(); }

// (at::empty without its way through the dispatcher)
Tensor dense(const Handle& h, at::IntArrayRef shape, at::ScalarType type) { return at::detail::empty_cuda(shape, type, h.device, std::nullopt); }

int run(int (*fn)(const ha_paged_params*, void*), const Handle& h, const ha_paged_params& p) {
  c10::cuda::OptionalCUDAGuard guard;
  if (c10::cuda::current_device() != h.device.index()) guard.set_index(h.device.index());
  return fn(&p, c10::cuda::getCurrentCUDAStream(h.device.index()).stream());
}

PyObject* answer(int rc, std::initializer_list<const Tensor*> out) {
  if (rc != HA_OK) return PyLong_FromLong(rc);
  if (out.size() == 1) {
    const Tensor& t = **out.begin();
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
  }
  PyObject* r = PyTuple_New((Py_ssize_t)out.size());
  Py_ssize_t i = 0;
  for (const Tensor* t : out) {
    PyObject* o = Py_None;
    if (t->defined()) o = THPVariable_Wrap(*t);
    else Py_INCREF(o);
    PyTuple_SET_ITEM(r, i++, o);
  }
  return r;
}

template <typename F>
PyObject* guarded(F f) {
  try {
    return f();
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_AssertionError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    // (torch's own class of it)
    PyObject* mod = PyImport_ImportModule("torch");
    PyObject* type = mod ? PyObject_GetAttrString(mod, "OutOfMemoryError") : nullptr;
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(mod);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

const Tensor* maybe(PyObject* o, const char* text) { return o == Py_None ? nullptr : &tensor_of(o, text); }

// init(addresses of ha_paged_append, ha_paged_attn, ha_paged_gather, ha_paged_maps, ha_paged_attn_workspace_bytes)
PyObject* ext_init(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n == 5, "init takes five addresses");
    void* f[5];
    for (int i = 0; i < 5; ++i) f[i] = PyLong_AsVoidPtr(a[i]);
    if (PyErr_Occurred()) return nullptr;
    abi.append = reinterpret_cast<decltype(abi.append)>(f[0]);
    abi.attn = reinterpret_cast<decltype(abi.attn)>(f[1]);
    abi.gather = reinterpret_cast<decltype(abi.gather)>(f[2]);
    abi.maps = reinterpret_cast<decltype(abi.maps)>(f[3]);
    abi.workspace = reinterpret_cast<decltype(abi.workspace)>(f[4]);
    Py_RETURN_NONE;
  });
}

// open(bytes of ha_paged_params with what the cache decides, host address of the host's status word or 0, pages ...) -> capsule
PyObject* ext_open(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n >= 4 && PyBytes_Check(a[0]) && PyBytes_GET_SIZE(a[0]) == sizeof(ha_paged_params), "open takes parameters");
    auto h = std::make_unique<Handle>();
    memcpy(&h->p, PyBytes_AS_STRING(a[0]), sizeof(h->p));
    h->dtype = h->p.dtype == HA_BF16 ? at::kBFloat16 : at::kHalf;
    h->failed = static_cast<const volatile int32_t*>(PyLong_AsVoidPtr(a[1]));
    if (PyErr_Occurred()) return nullptr;
    for (Py_ssize_t i = 2; i < n; ++i) {
      h->pages.push_back(tensor_of(a[i], "pages must be tensors"));
      h->at.push_back(h->pages.back().data_ptr());
    }
    h->device = h->pages[0].device();
    PyObject* c = PyCapsule_New(h.get(), NAME, [](PyObject* o) { delete static_cast<Handle*>(PyCapsule_GetPointer(o, NAME)); });
    if (c) h.release();
    return c;
  });
}

bool failed(const Handle& h) { return h.failed && *h.failed != 0; }

// append(handle, k, v, table, lengths, counts, rope, q, return_keys) -> q, or (q, k); an int: a status; NotImplemented: an earlier launch has failed
PyObject* ext_append(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n == 9, "append takes nine arguments");
    const int keys = PyObject_IsTrue(a[8]);
    if (keys < 0) return nullptr;
    Handle& h = handle_of(a[0]);
    if (failed(h)) Py_RETURN_NOTIMPLEMENTED;
    const Tensor k = rows(tensor_of(a[1], "k must be a tensor")), v = rows(tensor_of(a[2], "v must be a tensor"));
    const Tensor *counts = maybe(a[5], "counts must be a tensor"), *rope = maybe(a[6], "rope must be a tensor"), *q0 = maybe(a[7], "q must be a tensor");
    want(k.dim() == 4, "k must be [batch, tokens, heads, head_dim]");
    const int64_t B = k.size(0), m = k.size(1);
    ha_paged_params p = start(h, tensor_of(a[3], "table must be a tensor"), tensor_of(a[4], "lengths must be a tensor"), counts, B);
    want_rows(h, k, B, m, p.Hk, "k must be [batch, tokens, K/V heads, head_dim] of the cache", "k must have the type and device of the cache");
    want_rows(h, v, B, m, p.Hk, "v must be [batch, tokens, K/V heads, head_dim] of the cache", "v must have the type and device of the cache");
    want(m <= INT32_MAX, "too many tokens");
    p.n = (int32_t)m;
    p.k = k.data_ptr();
    p.v = v.data_ptr();
    p.k_sb = k.stride(0), p.k_sn = k.stride(1), p.k_sh = k.stride(2);
    p.v_sb = v.stride(0), p.v_sn = v.stride(1), p.v_sh = v.stride(2);
    Tensor q, q_out, k_out;
    if (q0) {
      q = rows(*q0);
      want(q.dim() == 4 && q.size(2) % p.Hk == 0 && q.size(2) <= INT32_MAX, "query heads must be a multiple of the key/value heads");
      want_rows(h, q, B, m, q.size(2), "q must be [batch, tokens, heads, head_dim] of the cache", "q must have the type and device of the cache");
      q_out = dense(h, q.sizes(), h.dtype);
      p.H = (int32_t)q.size(2);
      p.q = q.data_ptr();
      p.q_out = q_out.data_ptr();
      p.q_sb = q.stride(0), p.q_sn = q.stride(1), p.q_sh = q.stride(2);
    }
    if (rope) {
      want(rope->dim() == 3 && rope->size(2) == 2 && rope->is_contiguous() && rope->device() == h.device, "rope must be contiguous [positions, rot / 2, 2]");
      want((rope->scalar_type() == at::kFloat || rope->scalar_type() == h.dtype) && 2 * rope->size(1) <= p.d && rope->size(0) <= INT32_MAX,
           "rope must be fp32 or of the cache's type, for at most head_dim elements");
      want(rope->size(0) > 0 || rope->size(1) == 0 || B * m == 0, "rope must have the tokens' positions");     // (an empty tensor has no address, which would mean no rotation)
      p.rope = rope->data_ptr();
      p.rot = (int32_t)(2 * rope->size(1));
      p.rope_rows = (int32_t)rope->size(0);
      p.rope_dtype = rope->scalar_type() == at::kFloat ? HA_FP32 : p.dtype;
    }
    if (keys) {
      k_out = dense(h, k.sizes(), h.dtype);
      p.k_out = k_out.data_ptr();
    }
    const int rc = run(abi.append, h, p);
    return keys ? answer(rc, {&q_out, &k_out}) : answer(rc, {&q_out});
  });
}

// attn(handle, q, table, lengths, counts, scale) -> (o, lse)
PyObject* ext_attn(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n == 6, "attn takes six arguments");
    Handle& h = handle_of(a[0]);
    if (failed(h)) Py_RETURN_NOTIMPLEMENTED;
    const Tensor* counts = maybe(a[4], "counts must be a tensor");
    const double scale = PyFloat_AsDouble(a[5]);
    if (PyErr_Occurred()) return nullptr;
    Tensor q = tensor_of(a[1], "q must be a tensor");
    want(q.dim() == 4 && q.size(2) > 0 && q.size(2) % h.p.Hk == 0 && q.size(2) <= INT32_MAX, "q must be [batch, tokens, heads, head_dim], heads a multiple of the K/V heads");
    const int64_t B = q.size(0), m = q.size(1), H = q.size(2);
    ha_paged_params p = start(h, tensor_of(a[2], "table must be a tensor"), tensor_of(a[3], "lengths must be a tensor"), counts, B);
    want_rows(h, q, B, m, H, "q must be [batch, tokens, heads, head_dim] of the cache", "q must have the type and device of the cache");
    want(m <= INT32_MAX, "too many tokens");
    // rows that the kernel's 16-byte loads cannot read are copied
    if (q.stride(3) != 1 || (reinterpret_cast<uintptr_t>(q.data_ptr()) | (uintptr_t)(2 * (q.stride(0) | q.stride(1) | q.stride(2)))) % 16 != 0)
      q = q.clone(at::MemoryFormat::Contiguous);
    p.n = (int32_t)m;
    p.H = (int32_t)H;
    p.scale = (float)scale;
    p.q = q.data_ptr();
    p.q_sb = q.stride(0), p.q_sn = q.stride(1), p.q_sh = q.stride(2);
    const Tensor o = dense(h, {B, m, H, p.d}, h.dtype), lse = dense(h, {B, H, m}, at::kFloat);
    if (o.numel() == 0) return answer(HA_OK, {&o, &lse});
    p.o = o.data_ptr();
    p.lse = static_cast<float*>(lse.data_ptr());
    c10::cuda::OptionalCUDAGuard guard;
    if (c10::cuda::current_device() != h.device.index()) guard.set_index(h.device.index());
    if (p.bits == 16) {
      if (!h.mapped) {
        const int rc = abi.maps(&p, h.maps);
        if (rc != HA_OK) return PyLong_FromLong(rc);
        h.mapped = true;
      }
      p.maps = h.maps;
    }
    const int64_t bytes = abi.workspace(&p);
    if (bytes < 0) return PyLong_FromLongLong(bytes);
    Tensor ws;                                  // (free once the launches are enqueued: same stream)
    if (bytes > 0) {
      ws = dense(h, {bytes}, at::kByte);
      p.workspace = ws.data_ptr();
      p.workspace_bytes = bytes;
    }
    return answer(abi.attn(&p, c10::cuda::getCurrentCUDAStream(h.device.index()).stream()), {&o, &lse});
  });
}

// gather(handle, table, lengths, rows) -> (k, v)
PyObject* ext_gather(PyObject*, PyObject* const* a, Py_ssize_t n) {
  return guarded([&]() -> PyObject* {
    want(n == 4, "gather takes four arguments");
    Handle& h = handle_of(a[0]);
    if (failed(h)) Py_RETURN_NOTIMPLEMENTED;
    const Tensor& table = tensor_of(a[1], "table must be a tensor");
    const int64_t count = PyLong_AsLongLong(a[3]);
    if (PyErr_Occurred()) return nullptr;
    want(table.dim() == 2 && count >= 0 && count <= INT32_MAX, "table must be int32 [batch, columns], rows a number");
    ha_paged_params p = start(h, table, tensor_of(a[2], "lengths must be a tensor"), nullptr, table.size(0));
    const Tensor k = dense(h, {p.B, p.Hk, count, p.d}, h.dtype), v = dense(h, {p.B, p.Hk, count, p.d}, h.dtype);
    p.rows = (int32_t)count;
    p.k_out = k.data_ptr();
    p.v_out = v.data_ptr();
    return answer(run(abi.gather, h, p), {&k, &v});
  });
}

PyMethodDef methods[] = {{"init", (PyCFunction)(void*)ext_init, METH_FASTCALL, nullptr},       {"open", (PyCFunction)(void*)ext_open, METH_FASTCALL, nullptr},
                         {"append", (PyCFunction)(void*)ext_append, METH_FASTCALL, nullptr},   {"attn", (PyCFunction)(void*)ext_attn, METH_FASTCALL, nullptr},
                         {"gather", (PyCFunction)(void*)ext_gather, METH_FASTCALL, nullptr},   {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_paged_ext", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__paged_ext() { return PyModule_Create(&module); }
