// The speculative-decoding calls from Python, over torch tensors.
//
// A speculative step is a handful of short launches per token, so what a call
// costs on the host counts: checking a dozen tensors and converting them for
// ctypes took 10 to 15 us per call where this takes about 1.  It calls
// the C ABI of include/nwd.h (libnwd.so, beside this module) and nothing else
// of the library; torch provides the tensors, the current stream and the
// memory for outputs and workspaces.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <string>

#include "nwd.h"

namespace {

PyObject* g_error = nullptr;  // NwdError(status, message)

struct Refused {};  // a Python error is set

[[noreturn]] void refuse(PyObject* type, const std::string& what) {
  PyErr_SetString(type, what.c_str());
  throw Refused();
}

void check(int status) {
  if (status == NWD_OK) return;
  const std::string what = std::string(nwd_status_name(status)) + ": " + nwd_last_error();
  PyObject* e = PyObject_CallFunction(g_error, "is", status, what.c_str());
  if (e) {
    PyErr_SetObject(g_error, e);
    Py_DECREF(e);
  }
  throw Refused();
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse(PyExc_TypeError, std::string(name) + " must be a torch.Tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.is_cuda()) refuse(PyExc_ValueError, std::string(name) + " must be a CUDA tensor");
  return t;
}

std::string text(at::IntArrayRef shape) {
  std::string s = "(";
  for (size_t i = 0; i < shape.size(); i++) s += (i ? ", " : "") + std::to_string(shape[i]);
  return s + (shape.size() == 1 ? ",)" : ")");
}

// The pointer of a contiguous tensor of this type, shape and device.
template <typename T>  // (may be const)
T* pointer(PyObject* o, const char* name, at::ScalarType type, at::IntArrayRef shape, int device) {
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != type)
    refuse(PyExc_TypeError, std::string(name) + " must be torch." + c10::toString(type) + ", got torch." +
                                c10::toString(t.scalar_type()));
  if (t.get_device() != device)
    refuse(PyExc_ValueError, std::string(name) + " is on cuda:" + std::to_string(t.get_device()) +
                                 ", not on cuda:" + std::to_string(device));
  if (t.sizes() != shape)
    refuse(PyExc_ValueError,
           std::string(name) + " must have shape " + text(shape) + ", got " + text(t.sizes()));
  if (!t.is_contiguous()) refuse(PyExc_ValueError, std::string(name) + " must be contiguous");
  return static_cast<T*>(t.data_ptr());
}

uint64_t number(PyObject* o, const char* name) {
  const unsigned long long v = PyLong_AsUnsignedLongLong(o);
  if (v == (unsigned long long)-1 && PyErr_Occurred()) throw Refused();
  (void)name;
  return v;
}
uint32_t number32(PyObject* o, const char* name) {
  const uint64_t v = number(o, name);
  if (v > 0xffffffffull)
    refuse(PyExc_ValueError, std::string(name) + " is too large: " + std::to_string(v));
  return (uint32_t)v;
}

constexpr at::ScalarType F16 = at::kHalf, F32 = at::kFloat, I32 = at::kInt, I64 = at::kLong;

template <typename F>
PyObject* guarded(F&& f) {
  try {
    return f();
  } catch (const Refused&) {
    return nullptr;
  } catch (const c10::Error& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
    return nullptr;
  }
}

bool expect(Py_ssize_t got, Py_ssize_t want) {
  if (got == want) return true;
  PyErr_Format(PyExc_TypeError, "expected %zd arguments, got %zd", want, got);
  return false;
}

// tree(q, k_new | None, v_new | None, k_pool, v_pool, row_offset, seq_len, parents, o, n_heads,
//      n_kv_heads, head_dim, tree_len | None, scale, workspace, ws_bytes, err, capacity | None)
PyObject* tree(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!expect(n_args, 18)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& q = tensor(a[0], "q");
    const int dev = q.get_device();
    const at::Tensor& par = tensor(a[7], "parents");
    if (par.dim() != 2)
      refuse(PyExc_ValueError, "parents must be [batch, n_nodes], got " + text(par.sizes()));
    const int64_t batch = par.size(0), n = par.size(1);
    const uint32_t n_heads = number32(a[9], "n_heads"), n_kv = number32(a[10], "n_kv_heads"),
                   hd = number32(a[11], "head_dim");
    const double scale = PyFloat_AsDouble(a[13]);
    if (scale == -1.0 && PyErr_Occurred()) throw Refused();
    const int64_t qo[4] = {batch, n, n_heads, hd}, kv[4] = {batch, n, n_kv, hd}, one[1] = {batch};
    const bool append = a[1] != Py_None;
    const at::Tensor &kp = tensor(a[3], "k_pool"), &vp = tensor(a[4], "v_pool");
    const int64_t row = (int64_t)n_kv * hd;
    if (row == 0 || kp.numel() % row || vp.numel() != kp.numel())
      refuse(PyExc_ValueError, "k_pool and v_pool must hold the same whole number of rows");
    const uint64_t rows = (uint64_t)(kp.numel() / row);
    const auto* qp = pointer<uint16_t>(a[0], "q", F16, qo, dev);
    const uint16_t *kn = nullptr, *vn = nullptr;
    if (append) {
      kn = pointer<uint16_t>(a[1], "k_new", F16, kv, dev);
      vn = pointer<uint16_t>(a[2], "v_new", F16, kv, dev);
    }
    auto* k = pointer<uint16_t>(a[3], "k_pool", F16, kp.sizes(), dev);
    auto* v = pointer<uint16_t>(a[4], "v_pool", F16, vp.sizes(), dev);
    const auto* off = pointer<int64_t>(a[5], "row_offset", I64, one, dev);
    const auto* len = pointer<int32_t>(a[6], append ? "pos" : "seq_len", I32, one, dev);
    const auto* pr = pointer<int32_t>(a[7], "parents", I32, par.sizes(), dev);
    auto* op = pointer<uint16_t>(a[8], "o", F16, qo, dev);
    const auto* tl =
        a[12] == Py_None ? nullptr : pointer<int32_t>(a[12], "tree_len", I32, one, dev);
    const auto* cap =
        a[17] == Py_None ? nullptr : pointer<int32_t>(a[17], "capacity", I32, one, dev);
    void* ws = reinterpret_cast<void*>(number(a[14], "workspace"));
    size_t ws_bytes = number(a[15], "ws_bytes");
    auto* err = reinterpret_cast<uint32_t*>(number(a[16], "err"));
    if (batch > 0xffffffffll || n > 0xffffffffll) refuse(PyExc_ValueError, "parents is too large");
    if (batch == 0 || n == 0) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard on(dev);
    at::Tensor own;
    if (!ws) {
      check(nwd_attn_tree_workspace_size((uint32_t)batch, (uint32_t)n, n_heads, n_kv, hd, &ws_bytes));
      own = at::empty({(int64_t)ws_bytes}, q.options().dtype(at::kByte));
      ws = own.data_ptr();
    }
    void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    if (append)
      check(nwd_kv_append_attn_tree_bounded(qp, kn, vn, k, v, rows, off, len, cap, pr, tl, op,
                                            (uint32_t)batch, (uint32_t)n, n_heads, n_kv, hd,
                                            (float)scale, ws, ws_bytes, err, stream));
    else
      check(nwd_attn_tree(qp, k, v, rows, off, len, pr, tl, op, (uint32_t)batch, (uint32_t)n,
                          n_heads, n_kv, hd, (float)scale, ws, ws_bytes, err, stream));
    Py_RETURN_NONE;
  });
}

// verify(tokens, parents, tree_len | None, target_probs, draft_probs | None, u, w, path | None,
//        n_accepted | None, next_token | None, err) -> (path, n_accepted, next_token)
PyObject* verify(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!expect(n_args, 11)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& target = tensor(a[3], "target_probs");
    if (target.dim() != 3)
      refuse(PyExc_ValueError,
             "target_probs must be [batch, n_nodes, vocab], got " + text(target.sizes()));
    const int dev = target.get_device();
    const int64_t batch = target.size(0), n = target.size(1), vocab = target.size(2);
    const int64_t bn[2] = {batch, n}, one[1] = {batch};
    const auto* tk = pointer<int32_t>(a[0], "tokens", I32, bn, dev);
    const auto* pr = pointer<int32_t>(a[1], "parents", I32, bn, dev);
    const auto* tl = a[2] == Py_None ? nullptr : pointer<int32_t>(a[2], "tree_len", I32, one, dev);
    const auto* tp = pointer<float>(a[3], "target_probs", F32, target.sizes(), dev);
    const auto* dp =
        a[4] == Py_None ? nullptr : pointer<float>(a[4], "draft_probs", F32, target.sizes(), dev);
    const auto* u = pointer<float>(a[5], "u", F32, bn, dev);
    const auto* w = pointer<float>(a[6], "w", F32, one, dev);
    auto* err = reinterpret_cast<uint32_t*>(number(a[10], "err"));
    if (batch > 0xffffffffll || n > 0xffffffffll || vocab > 0xffffffffll)
      refuse(PyExc_ValueError, "target_probs is too large");
    const c10::cuda::CUDAGuard on(dev);
    const bool given = a[7] != Py_None;
    at::Tensor path, count, token;
    if (!given) {
      const auto opt = target.options().dtype(I32);
      path = at::empty({batch, n}, opt);
      count = at::empty({batch}, opt);
      token = at::empty({batch}, opt);
    } else {
      path = tensor(a[7], "path");
      count = tensor(a[8], "n_accepted");
      token = tensor(a[9], "next_token");
      pointer<int32_t>(a[7], "path", I32, bn, dev);
      pointer<int32_t>(a[8], "n_accepted", I32, one, dev);
      pointer<int32_t>(a[9], "next_token", I32, one, dev);
    }
    if (batch)
      check(nwd_verify_tree(tk, pr, tl, tp, dp, u, w, static_cast<int32_t*>(path.data_ptr()),
                          static_cast<int32_t*>(count.data_ptr()),
                          static_cast<int32_t*>(token.data_ptr()), (uint32_t)batch, (uint32_t)n,
                          (uint32_t)vocab, err, c10::cuda::getCurrentCUDAStream(dev).stream()));
    if (given) {
      PyObject* out = PyTuple_Pack(3, a[7], a[8], a[9]);
      return out;
    }
    PyObject* out = PyTuple_New(3);
    if (!out) return nullptr;
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(path)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(count)));
    PyTuple_SET_ITEM(out, 2, THPVariable_Wrap(std::move(token)));
    return out;
  });
}

// The pools of a list, all of the first one's shape and on `dev`; that shape.
std::vector<uint16_t*> pool_pointers(PyObject* list, int dev, at::IntArrayRef* shape) {
  if (!PyList_Check(list)) refuse(PyExc_TypeError, "pools must be a list");
  const Py_ssize_t count = PyList_GET_SIZE(list);
  std::vector<uint16_t*> ptrs((size_t)count);
  if (count == 0) return ptrs;
  const at::Tensor& first = tensor(PyList_GET_ITEM(list, 0), "pool");
  if (first.dim() != 3)
    refuse(PyExc_ValueError, "pools must be [rows, n_kv, hd], got " + text(first.sizes()));
  for (Py_ssize_t i = 0; i < count; i++) {
    ptrs[i] = pointer<uint16_t>(PyList_GET_ITEM(list, i), "pool", F16, first.sizes(), dev);
    for (Py_ssize_t j = 0; j < i; j++)
      if (ptrs[j] == ptrs[i] && first.numel())
        refuse(PyExc_ValueError, "pools must differ from one another");
  }
  *shape = first.sizes();
  if (first.size(1) > 0xffffffffll || first.size(2) > 0xffffffffll)
    refuse(PyExc_ValueError, "pools are too large");
  return ptrs;
}

// commit(pools (a list), row_offset, pos, path, n_accepted, err): 16 pools per launch
PyObject* commit(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!expect(n_args, 6)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& path = tensor(a[3], "path");
    if (path.dim() != 2)
      refuse(PyExc_ValueError, "path must be [batch, n_nodes], got " + text(path.sizes()));
    const int dev = path.get_device();
    const int64_t batch = path.size(0), n = path.size(1);
    const int64_t one[1] = {batch};
    const auto* off = pointer<int64_t>(a[1], "row_offset", I64, one, dev);
    const auto* pos = pointer<int32_t>(a[2], "pos", I32, one, dev);
    const auto* pp = pointer<int32_t>(a[3], "path", I32, path.sizes(), dev);
    const auto* na = pointer<int32_t>(a[4], "n_accepted", I32, one, dev);
    auto* err = reinterpret_cast<uint32_t*>(number(a[5], "err"));
    at::IntArrayRef shape;
    const std::vector<uint16_t*> ptrs = pool_pointers(a[0], dev, &shape);
    const Py_ssize_t count = (Py_ssize_t)ptrs.size();
    if (batch > 0xffffffffll || n > 0xffffffffll) refuse(PyExc_ValueError, "path is too large");
    if (batch == 0 || n == 0 || count == 0 || !ptrs[0]) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard on(dev);
    void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    for (Py_ssize_t i = 0; i < count; i += 16)
      check(nwd_kv_commit(ptrs.data() + i, (uint32_t)std::min<Py_ssize_t>(16, count - i),
                          (uint64_t)shape[0], off, pos, pp, na, (uint32_t)batch, (uint32_t)n,
                          (uint32_t)shape[1], (uint32_t)shape[2], err, stream));
    Py_RETURN_NONE;
  });
}

// The pointers of a list of tensors of one type and shape; nullptr for None where
// that is allowed.
template <typename T>
std::vector<T*> pointers(PyObject* list, const char* name, at::ScalarType type, size_t count,
                         at::IntArrayRef shape, int dev, bool optional = false) {
  if (!PyList_Check(list) || (size_t)PyList_GET_SIZE(list) != count)
    refuse(PyExc_TypeError, std::string(name) + " must be a list with an entry per layer");
  std::vector<T*> ptrs(count);
  for (size_t i = 0; i < count; i++) {
    PyObject* o = PyList_GET_ITEM(list, (Py_ssize_t)i);
    ptrs[i] = optional && o == Py_None ? nullptr : pointer<T>(o, name, type, shape, dev);
  }
  return ptrs;
}

// commit_layers(pools (K, V, K, V ..), row_offsets, lengths, capacities, tree_lens (or None; lists,
//               an entry per layer), path, n_accepted, err): 32 layers per launch
PyObject* commit_layers(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  if (!expect(n_args, 8)) return nullptr;
  return guarded([&]() -> PyObject* {
    const at::Tensor& path = tensor(a[5], "path");
    if (path.dim() != 2)
      refuse(PyExc_ValueError, "path must be [batch, n_nodes], got " + text(path.sizes()));
    const int dev = path.get_device();
    const int64_t batch = path.size(0), n = path.size(1);
    const int64_t one[1] = {batch};
    at::IntArrayRef shape;
    const std::vector<uint16_t*> ptrs = pool_pointers(a[0], dev, &shape);
    if (ptrs.size() % 2) refuse(PyExc_ValueError, "a layer has two pools");
    const size_t layers = ptrs.size() / 2;
    const auto off = pointers<const int64_t>(a[1], "row_offset", I64, layers, one, dev);
    const auto len = pointers<int32_t>(a[2], "lengths", I32, layers, one, dev);
    const auto cap = pointers<const int32_t>(a[3], "capacity", I32, layers, one, dev);
    const auto tree = pointers<const int32_t>(a[4], "tree_len", I32, layers, one, dev, true);
    const auto* pp = pointer<int32_t>(a[5], "path", I32, path.sizes(), dev);
    const auto* na = pointer<int32_t>(a[6], "n_accepted", I32, one, dev);
    auto* err = reinterpret_cast<uint32_t*>(number(a[7], "err"));
    if (batch > 0xffffffffll || n > 0xffffffffll) refuse(PyExc_ValueError, "path is too large");
    if (batch == 0 || n == 0 || layers == 0 || !ptrs[0]) Py_RETURN_NONE;
    const c10::cuda::CUDAGuard on(dev);
    void* stream = c10::cuda::getCurrentCUDAStream(dev).stream();
    for (size_t i = 0; i < layers; i += 32)
      check(nwd_kv_commit_layers(ptrs.data() + 2 * i, (uint32_t)std::min<size_t>(32, layers - i),
                                 (uint64_t)shape[0], off.data() + i, len.data() + i,
                                 cap.data() + i, tree.data() + i, pp, na, (uint32_t)batch,
                                 (uint32_t)n, (uint32_t)shape[1], (uint32_t)shape[2], err, stream));
    Py_RETURN_NONE;
  });
}

PyObject* set_error(PyObject*, PyObject* type) {
  Py_INCREF(type);
  Py_XSETREF(g_error, type);
  Py_RETURN_NONE;
}

PyMethodDef methods[] = {
    {"tree", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(tree)), METH_FASTCALL, nullptr},
    {"verify", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(verify)), METH_FASTCALL, nullptr},
    {"commit", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(commit)), METH_FASTCALL, nullptr},
    {"commit_layers", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(commit_layers)),
     METH_FASTCALL, nullptr},
    {"set_error", set_error, METH_O, nullptr},
    {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_nwd_torch",
                      "The speculative-decoding calls of libnwd.so over torch tensors.", -1, methods,
                      nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__nwd_torch() { return PyModule_Create(&module); }
