// lf_host.cpp — the host's part of a repeated call of the operators for different lengths (loopfuse_amd/packed.py, paged.py), as a
// Python module: what a call launches depends on shapes, strides, dtypes, alignment and device of its operands, its plan, its sizes and
// the environment switches alone.  The first call of such a signature goes through the Python module, which checks it and leaves here the parameter
// block and the launches (`keep`); the next ones form the signature, the results and the block here.  A function returns None where nothing is
// kept for the signature, or for operands that are no plain GPU tensors: the Python module then takes the call, or refuses it.
//   The kernels of small calls run for 3 ... 6 us.  us a call, with the same steps in Python / here: extend_tables 10.9 / 6.2, packed_layout, two launches, 16.4 / 7.0, store_kv of 64 rows 8.3 / 4.6,
// attention_packed of 3 short prompts 10.9 / 6.8, attention_shared of 2 requests, two launches, 15.5 / 10.9, a training step of 24 short sequences, 121 us of
// kernels, 135 / 123.
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstring>
#include <memory>
#include <mutex>
#include <string>
#include <unordered_map>
#include <utility>
#include <vector>

#include "lf_ragged_params.h"
#include "lf_shim.h"

namespace {

constexpr size_t kMaxKept = 512;
constexpr size_t kMaxBlock = 1024;

struct Entry {                       // the launches of one signature
  std::string block;                 // parameter block, its pointers still to be set
  std::string items;                 // lf_launch_item [count]
  int count = 0;
  PyObject* record = nullptr;        // what the operator's last_launch becomes
  PyObject* owner = nullptr;         // keeps the kernels alive
  std::vector<long long> more;       // what the operator keeps beside it
  ~Entry() {                         // (with the GIL)
    Py_XDECREF(record);
    Py_XDECREF(owner);
  }
};

// Leaked on purpose: destructors of tensors and Python objects must not run behind the end of the runtimes.
std::unordered_map<std::string, std::shared_ptr<Entry>>& kept = *new std::unordered_map<std::string, std::shared_ptr<Entry>>;
struct {
  PyObject *os = nullptr, *environ = nullptr, *variables = nullptr, *switches = nullptr, *checks = nullptr, *last = nullptr, *fail = nullptr, *step = nullptr;
  int (*launch)(const lf_launch_item*, int, void*, void*) = nullptr;
} env;

// Partial results of a step, one buffer per device and stream: steps on one stream are ordered; a step's launches are made under the lock.
std::mutex& scratch_lock = *new std::mutex;
std::unordered_map<std::string, at::Tensor>& scratch = *new std::unordered_map<std::string, at::Tensor>;

PyObject* none() { Py_RETURN_NONE; }

template <class T>
void put(std::string& s, const T& x) {
  s.append(reinterpret_cast<const char*>(&x), sizeof(x));
}

bool put_plain(std::string& s, PyObject* o) {
  if (o == Py_None) {
    s += 'N';
  } else if (PyBool_Check(o)) {
    s += o == Py_True ? 'T' : 'F';
  } else if (PyLong_CheckExact(o)) {
    int overflow = 0;
    const long long x = PyLong_AsLongLongAndOverflow(o, &overflow);
    if (overflow) return false;
    s += 'i';
    put(s, x);
  } else if (PyFloat_CheckExact(o)) {
    s += 'f';
    put(s, PyFloat_AS_DOUBLE(o));
  } else if (PyUnicode_CheckExact(o)) {
    Py_ssize_t n = 0;
    const char* p = PyUnicode_AsUTF8AndSize(o, &n);
    if (!p) {
      PyErr_Clear();
      return false;
    }
    s += 's';
    put(s, n);
    s.append(p, n);
  } else {
    return false;
  }
  return true;
}

// a plain GPU tensor: no subclass, no wrapper of a transform, nothing pending, no tangent
const at::Tensor* plain(PyObject* o) {
  if (!THPVariable_CheckExact(o)) return nullptr;
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.defined() || !t.is_cuda() || t.layout() != at::kStrided || !t.has_storage() || t.is_neg() || t.is_conj() ||
      t.unsafeGetTensorImpl()->is_python_dispatch() || t.unsafeGetTensorImpl()->has_symbolic_sizes_strides() ||
      t.key_set().has(at::DispatchKey::Functionalize) || t._fw_grad(0).defined())
    return nullptr;
  return &t;
}

bool put_tensor(std::string& s, PyObject* o, int& device, bool aligned) {
  if (o == Py_None) {
    s += 'N';
    return true;
  }
  const at::Tensor* t = plain(o);
  if (!t) return false;
  if (device < 0) {
    device = c10::hip::current_device();
    put(s, device);
  }
  if (t->get_device() != device || (aligned && reinterpret_cast<uintptr_t>(t->const_data_ptr()) % 16)) return false;
  s += 't';
  put(s, t->scalar_type());
  put(s, t->dim());
  for (int64_t n : t->sizes()) put(s, n);
  for (int64_t n : t->strides()) put(s, n);
  return true;
}

PyObject *names[7], *name_environ, *name_record;        // fields of a plan; attributes

// The signature of a call: `n` tensors, of which the first `data` are read 16 bytes at a time, a plan (or null) and further sizes.
// False: not to be kept.
bool signature(std::string& s, char kind, PyObject* const* tensors, int n, int data, PyObject* plan, PyObject* const* more, int count) {
  if (!env.variables) return false;
  PyObject* now = PyObject_GetAttr(env.os, name_environ);
  Py_XDECREF(now);
  if (now != env.environ || PyDict_Contains(env.variables, env.checks) != 0) {
    PyErr_Clear();
    return false;
  }
  int device = -1;
  s.reserve(512);
  s += kind;
  for (int i = 0; i < n; ++i)
    if (!put_tensor(s, tensors[i], device, i < data)) return false;
  if (device < 0) return false;
  if (plan)
    for (PyObject* name : names) {
      PyObject* x = PyObject_GetAttr(plan, name);
      const bool ok = x && put_plain(s, x);
      Py_XDECREF(x);
      if (!ok) {
        PyErr_Clear();
        return false;
      }
    }
  for (int i = 0; i < count; ++i)
    if (!put_plain(s, more[i])) return false;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(env.switches); ++i)
    if (PyObject* x = PyDict_GetItemWithError(env.variables, PyTuple_GET_ITEM(env.switches, i))) {
      if (!PyBytes_Check(x)) return false;
      put(s, i);
      put(s, PyBytes_GET_SIZE(x));
      s.append(PyBytes_AS_STRING(x), PyBytes_GET_SIZE(x));
    }
  return !PyErr_Occurred();
}

std::shared_ptr<Entry> find(char kind, PyObject* const* tensors, int n, int data, PyObject* plan, PyObject* const* more, int count) {
  std::string s;
  if (!signature(s, kind, tensors, n, data, plan, more, count)) {
    PyErr_Clear();
    return nullptr;
  }
  auto it = kept.find(s);
  return it == kept.end() ? nullptr : it->second;
}

struct Block {
  alignas(16) char bytes[kMaxBlock];
  explicit Block(const Entry& e) { std::memcpy(bytes, e.block.data(), e.block.size()); }
  template <class T>
  T* as() {
    return reinterpret_cast<T*>(bytes);
  }
};

template <class T = void>
T* at_(PyObject* o) {
  return o == Py_None ? nullptr : static_cast<T*>(THPVariable_Unpack(o).data_ptr());
}

// a result of the call; throws where it is no memory of the GPU (a mode that makes other tensors)
at::Tensor made(at::IntArrayRef sizes, const at::TensorOptions& options) {
  at::Tensor t = at::empty(sizes, options);
  TORCH_CHECK(t.is_cuda() && !t.unsafeGetTensorImpl()->is_python_dispatch(), "loopfuse_amd: results must be plain tensors on the GPU");
  return t;
}
at::TensorOptions like(const at::Tensor& t) { return at::TensorOptions().dtype(t.scalar_type()).device(t.device()); }

void* stream_of(const at::Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }

// the launches, without the GIL; false: the error is set.  `told`: last_launch says so
bool launch(const Entry& e, Block& block, void* stream, bool told = true) {
  int rc;
  Py_BEGIN_ALLOW_THREADS
  rc = env.launch(reinterpret_cast<const lf_launch_item*>(e.items.data()), e.count, block.bytes, stream);
  Py_END_ALLOW_THREADS
  if (rc) {
    Py_XDECREF(PyObject_CallFunction(env.fail, "i", rc));
    return false;
  }
  return !told || PyObject_SetAttr(env.last, name_record, e.record) == 0;
}

// Room for partial results, under scratch_lock: a captured call has its own, the graph's.
at::Tensor partial_results(long long floats, const at::Tensor& q, void* stream) {
  if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) return made({floats}, like(q).dtype(at::kFloat));
  std::string where;
  put(where, q.get_device());
  put(where, stream);
  at::Tensor& t = scratch[where];
  if (!t.defined() || t.numel() < floats) t = made({std::max<int64_t>(floats, 1 << 20)}, like(q).dtype(at::kFloat));
  return t;
}

// ---- module functions ------------------------------------------------------------------------------------------

// setup(os, environ, variables, switches, checks, last, fail, step, launch)
PyObject* setup(PyObject*, PyObject* const* a, Py_ssize_t n) {
  if (n != 9 || !PyDict_Check(a[2]) || !PyTuple_Check(a[3])) {
    PyErr_SetString(PyExc_TypeError, "setup: 9 arguments");
    return nullptr;
  }
  PyObject** to[] = {&env.os, &env.environ, &env.variables, &env.switches, &env.checks, &env.last, &env.fail, &env.step};
  for (int i = 0; i < 8; ++i) {
    Py_INCREF(a[i]);
    Py_XDECREF(*to[i]);
    *to[i] = a[i];
  }
  env.launch = reinterpret_cast<decltype(env.launch)>(PyLong_AsVoidPtr(a[8]));
  if (PyErr_Occurred()) return nullptr;
  return none();
}

// key(kind, data, ints, plan, more): the signature as bytes, None: not to be kept
PyObject* key(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 5 || !PyUnicode_Check(a[0]) || !PyTuple_Check(a[1]) || !PyTuple_Check(a[2]) || !PyTuple_Check(a[4])) {
    PyErr_SetString(PyExc_TypeError, "key: kind, data, ints, plan, more");
    return nullptr;
  }
  std::vector<PyObject*> tensors;
  for (int k = 1; k < 3; ++k)
    for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[k]); ++i) tensors.push_back(PyTuple_GET_ITEM(a[k], i));
  std::vector<PyObject*> more;
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[4]); ++i) more.push_back(PyTuple_GET_ITEM(a[4], i));
  std::string s;
  const char* kind = PyUnicode_AsUTF8(a[0]);
  if (!kind) return nullptr;
  if (!signature(s, kind[0], tensors.data(), (int)tensors.size(), (int)PyTuple_GET_SIZE(a[1]), a[3] == Py_None ? nullptr : a[3], more.data(), (int)more.size())) {
    PyErr_Clear();
    return none();
  }
  return PyBytes_FromStringAndSize(s.data(), s.size());
  END_HANDLE_TH_ERRORS
}

// keep(key, block, items, record, owner, more)
PyObject* keep(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (n != 6 || !PyBytes_Check(a[0]) || !PyBytes_Check(a[1]) || !PyBytes_Check(a[2]) || !PyTuple_Check(a[5]) ||
      PyBytes_GET_SIZE(a[1]) > (Py_ssize_t)kMaxBlock || PyBytes_GET_SIZE(a[2]) % sizeof(lf_launch_item)) {
    PyErr_SetString(PyExc_TypeError, "keep: key, block, items, record, owner, more");
    return nullptr;
  }
  auto e = std::make_shared<Entry>();
  e->block.assign(PyBytes_AS_STRING(a[1]), PyBytes_GET_SIZE(a[1]));
  e->items.assign(PyBytes_AS_STRING(a[2]), PyBytes_GET_SIZE(a[2]));
  e->count = (int)(e->items.size() / sizeof(lf_launch_item));
  for (Py_ssize_t i = 0; i < PyTuple_GET_SIZE(a[5]); ++i) e->more.push_back(PyLong_AsLongLong(PyTuple_GET_ITEM(a[5], i)));
  if (PyErr_Occurred()) return nullptr;
  Py_INCREF(e->record = a[3]);
  Py_INCREF(e->owner = a[4]);
  if (kept.size() >= kMaxKept) kept.clear();
  kept[std::string(PyBytes_AS_STRING(a[0]), PyBytes_GET_SIZE(a[0]))] = std::move(e);
  return none();
  END_HANDLE_TH_ERRORS
}

PyObject* clear(PyObject*, PyObject*) {
  kept.clear();
  return none();
}

PyObject* size(PyObject*, PyObject*) { return PyLong_FromSize_t(kept.size()); }

bool takes(Py_ssize_t n, Py_ssize_t want) {
  if (n != want) PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", want, n);
  return n == want;
}

// Does the node that made the tensor, and that its gradient goes to, belong to a stream outside the capture?  A captured backward that reaches such
// a node would have its stream wait inside the capture, which ends the process.
bool node_elsewhere(const at::Tensor& t) {
  const std::shared_ptr<torch::autograd::Node> node = t.requires_grad() ? t.grad_fn() : nullptr;
  const auto stream = node ? node->stream() : std::nullopt;
  if (!stream) return false;
  // (torch's nodes name the device type CUDA, its HIP streams HIP)
  const c10::hip::HIPStream its(c10::hip::HIPStream::UNCHECKED,
                                c10::Stream(c10::Stream::UNSAFE, c10::Device(c10::DeviceType::HIP, stream->device_index()), stream->id()));
  if (its.stream() == nullptr) return true;            // (the default stream is never captured, and not to be asked while another is)
  const c10::hip::HIPStreamGuard guard(its);
  return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::Active;
}

// elsewhere(tensor) -> node_elsewhere
PyObject* elsewhere(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 1)) return nullptr;
  return PyBool_FromLong(THPVariable_Check(a[0]) && node_elsewhere(THPVariable_Unpack(a[0])));
  END_HANDLE_TH_ERRORS
}

// extend_tables(cached, new, table, free, page_size, total) -> PagedStep; more: entries of the one allocation, then of its five parts
PyObject* extend_tables(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 6)) return nullptr;
  auto e = find('t', a, 4, 0, nullptr, a + 4, 2);
  if (!e) return none();
  const at::Tensor& cached = THPVariable_Unpack(a[0]);
  at::Tensor all = made({e->more[0]}, like(cached));
  Block block(*e);
  auto* p = block.as<LfTablesParamsHost>();
  p->cached = at_<int32_t>(a[0]);
  p->fresh = at_<int32_t>(a[1]);
  p->table = at_(a[2]);
  p->free = at_(a[3]);
  int32_t* at = all.mutable_data_ptr<int32_t>();
  int32_t** to[] = {&p->offsets, &p->lengths, &p->pages, &p->slots, &p->positions};
  for (int i = 0; i < 5; at += e->more[1 + i], ++i) *to[i] = at;
  if (!launch(*e, block, stream_of(cached))) return nullptr;
  // five tensors in one storage: plain ones, not views that autograd follows
  PyObject* parts = PyTuple_New(5);
  if (!parts) return nullptr;
  int64_t first = 0;
  for (int i = 0; i < 5; first += e->more[1 + i], ++i) {
    auto t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
    t.unsafeGetTensorImpl()->set_sizes_contiguous({e->more[1 + i]});
    t.unsafeGetTensorImpl()->set_storage_offset(first);
    PyObject* x = THPVariable_Wrap(std::move(t));
    if (!x) {
      Py_DECREF(parts);
      return nullptr;
    }
    PyTuple_SET_ITEM(parts, i, x);
  }
  // (the order of the fields: offsets, lengths, slots, positions, pages)
  PyObject* pages = PyTuple_GET_ITEM(parts, 2);
  PyTuple_SET_ITEM(parts, 2, PyTuple_GET_ITEM(parts, 3));
  PyTuple_SET_ITEM(parts, 3, PyTuple_GET_ITEM(parts, 4));
  PyTuple_SET_ITEM(parts, 4, pages);
  PyObject* args = PyTuple_Pack(1, parts);
  PyObject* step = args ? PyTuple_Type.tp_new(reinterpret_cast<PyTypeObject*>(env.step), args, nullptr) : nullptr;
  Py_XDECREF(args);
  Py_DECREF(parts);
  return step;
  END_HANDLE_TH_ERRORS
}

// packed_layout(offsets, total) -> (tiles, caps); owner: a tuple whose second item is caps; more: entries of the lists, numbers in all
PyObject* packed_layout(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 2)) return nullptr;
  auto e = find('l', a, 1, 0, nullptr, a + 1, 1);
  if (!e) return none();
  const at::Tensor& offsets = THPVariable_Unpack(a[0]);
  at::Tensor all = made({e->more[1]}, like(offsets));
  Block block(*e);
  auto* p = block.as<LfPackedPlanParamsHost>();
  p->offsets = at_<int32_t>(a[0]);
  p->tiles = static_cast<LfPackedTileHost*>(all.mutable_data_ptr());
  p->sorted = reinterpret_cast<int32_t*>(p->tiles + e->more[0]);
  if (!launch(*e, block, stream_of(offsets), false)) return nullptr;
  auto tiles = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(all.storage()), all.key_set(), all.dtype());
  tiles.unsafeGetTensorImpl()->set_sizes_contiguous({e->more[0], 4});
  PyObject* x = THPVariable_Wrap(std::move(tiles));
  if (!x) return nullptr;
  PyObject* r = PyTuple_Pack(2, x, PyTuple_GET_ITEM(e->owner, 1));
  Py_DECREF(x);
  return r;
  END_HANDLE_TH_ERRORS
}

// store_kv(k, v, k_pool, v_pool, slots) -> True
PyObject* store_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 5)) return nullptr;
  auto e = find('s', a, 5, 4, nullptr, nullptr, 0);
  if (!e) return none();
  Block block(*e);
  auto* p = block.as<LfStoreParamsHost>();
  p->k = at_(a[0]);
  p->v = at_(a[1]);
  p->k_pool = at_(a[2]);
  p->v_pool = at_(a[3]);
  p->slots = at_<int32_t>(a[4]);
  if (!launch(*e, block, stream_of(THPVariable_Unpack(a[0])))) return nullptr;
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// attention_shared(q, k_pool, v_pool, out, table, lengths, prefix_table, v_table, prefix_v_table, plan, prefix_len) -> O;
// more: floats of scratch, and the bytes in front of part_ml, pre_acc and pre_ml in it
PyObject* attention_shared(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 11)) return nullptr;
  auto e = find('h', a, 9, 4, a[9], a + 10, 1);
  if (!e) return none();
  const at::Tensor& q = THPVariable_Unpack(a[0]);
  const at::Tensor out = a[3] == Py_None ? made(q.sizes(), like(q)) : THPVariable_Unpack(a[3]);
  Block block(*e);
  auto* p = block.as<LfSharedParamsHost>();
  p->attn.q = at_(a[0]);
  p->attn.k = at_(a[1]);
  p->attn.v = at_(a[2]);
  p->attn.o = out.mutable_data_ptr();
  p->lengths = at_<int32_t>(a[5]);
  p->attn.k_table = at_(a[4]);
  p->attn.v_table = a[7] == Py_None ? p->attn.k_table : at_(a[7]);
  p->prefix_k = at_(a[6]);
  p->prefix_v = a[8] == Py_None ? p->prefix_k : at_(a[8]);
  void* stream = stream_of(q);
  int rc;
  {
    // (without the GIL: whoever holds the lock needs nothing of Python's)
    pybind11::gil_scoped_release without;
    std::lock_guard<std::mutex> lock(scratch_lock);
    const at::Tensor room = partial_results(e->more[0], q, stream);
    char* at = static_cast<char*>(room.mutable_data_ptr());
    p->attn.part_acc = reinterpret_cast<float*>(at);
    p->attn.part_ml = reinterpret_cast<float*>(at + e->more[1]);
    p->pre_acc = reinterpret_cast<float*>(at + e->more[2]);
    p->pre_ml = reinterpret_cast<float*>(at + e->more[3]);
    rc = env.launch(reinterpret_cast<const lf_launch_item*>(e->items.data()), e->count, block.bytes, stream);
  }
  if (rc) {
    Py_XDECREF(PyObject_CallFunction(env.fail, "i", rc));
    return nullptr;
  }
  if (PyObject_SetAttr(env.last, name_record, e->record)) return nullptr;
  if (a[3] == Py_None) return THPVariable_Wrap(out);
  Py_INCREF(a[3]);
  return a[3];
  END_HANDLE_TH_ERRORS
}

// attention_packed(q, k, v, out, lse, tiles, plan, total, entries, train) -> O, or with `train` (O, lse, low), both made here;
// more: bytes in front of the list of tiles
PyObject* attention_packed(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 10)) return nullptr;
  auto e = find('p', a, 6, 4, a[6], a + 7, 3);
  if (!e) return none();
  const bool train = a[9] == Py_True;
  const at::Tensor& q = THPVariable_Unpack(a[0]);
  const at::Tensor out = a[3] == Py_None ? made(q.sizes(), like(q)) : THPVariable_Unpack(a[3]);
  at::Tensor lse, low;
  Block block(*e);
  auto* p = block.as<LfPackedAttnParamsHost>();
  p->attn.q = at_(a[0]);
  p->attn.k = at_(a[1]);
  p->attn.v = at_(a[2]);
  p->attn.o = out.mutable_data_ptr();
  if (train) {
    lse = made({q.size(1), q.size(0)}, like(q).dtype(at::kFloat));
    low = made(q.sizes(), like(q));
    p->attn.part_ml = lse.mutable_data_ptr<float>();
    p->low = low.mutable_data_ptr();
  } else {
    p->attn.part_ml = at_<float>(a[4]);
  }
  p->tiles = reinterpret_cast<const LfPackedTileHost*>(at_<char>(a[5]) + e->more[0]);
  if (!launch(*e, block, stream_of(q))) return nullptr;
  if (train) {
    PyObject* r = PyTuple_New(3);
    if (!r) return nullptr;
    const at::Tensor* parts[] = {&out, &lse, &low};
    for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(*parts[i]));
    return r;
  }
  if (a[3] == Py_None) return THPVariable_Wrap(out);
  Py_INCREF(a[3]);
  return a[3];
  END_HANDLE_TH_ERRORS
}

// attention_packed_backward(q, k, v, o, dout, low, lse, tiles, plan, total, entries) -> (dq, dk, dv), False where dS has no room;
// more: bytes in front of the two lists of tiles, elements of dS, calls until room for dS is looked for again (-1: never)
PyObject* attention_packed_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 11)) return nullptr;
  auto e = find('b', a, 8, 6, a[8], a + 9, 2);
  if (!e || e->more[3] == 0) return none();
  if (e->more[3] > 0) --e->more[3];
  const at::Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]), &lse = THPVariable_Unpack(a[6]);
  const at::Tensor dq = made(q.sizes(), like(q)), dk = made(k.sizes(), like(k)), dv = made(k.sizes(), like(k)), delta = made(lse.sizes(), like(lse));
  Block block(*e);
  auto* p = block.as<LfPackedBwdParamsHost>();
  p->bwd.q = at_(a[0]);
  p->bwd.k = at_(a[1]);
  p->bwd.v = at_(a[2]);
  p->bwd.o = at_(a[3]);
  p->bwd.dout = at_(a[4]);
  p->bwd.lse = at_<float>(a[6]);
  p->bwd.dq = dq.mutable_data_ptr();
  p->bwd.dk = dk.mutable_data_ptr();
  p->bwd.dv = dv.mutable_data_ptr();
  p->bwd.delta = delta.mutable_data_ptr<float>();
  p->dkdv_tiles = reinterpret_cast<const LfPackedTileHost*>(at_<char>(a[7]) + e->more[0]);
  p->dq_tiles = reinterpret_cast<const LfPackedTileHost*>(at_<char>(a[7]) + e->more[1]);
  p->low = at_(a[5]);
  at::Tensor ds;
  if (e->more[2]) {
    // last: it may take what room is left, which the results need and it does not
    try {
      ds = made({e->more[2]}, like(q));
    } catch (const c10::OutOfMemoryError&) {
      Py_RETURN_FALSE;
    }
    p->bwd.ds = ds.mutable_data_ptr();
  }
  if (!launch(*e, block, stream_of(q))) return nullptr;
  PyObject* r = PyTuple_New(3);
  if (!r) return nullptr;
  const at::Tensor* parts[] = {&dq, &dk, &dv};
  for (int i = 0; i < 3; ++i) PyTuple_SET_ITEM(r, i, THPVariable_Wrap(*parts[i]));
  return r;
  END_HANDLE_TH_ERRORS
}

// tensors as a tuple, None in the place of one that is not defined
PyObject* tuple_of(std::initializer_list<const at::Tensor*> parts) {
  PyObject* r = PyTuple_New(parts.size());
  Py_ssize_t i = 0;
  if (r)
    for (const at::Tensor* t : parts) PyTuple_SET_ITEM(r, i++, t->defined() ? THPVariable_Wrap(*t) : none());
  return r;
}

// rotate_heads(q, k, table, q_weight, k_weight, positions, eps, pairs) -> (q, k)
PyObject* rotate_heads(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 8)) return nullptr;
  auto e = find('r', a, 6, 5, nullptr, a + 6, 2);
  if (!e) return none();
  const at::Tensor &q = THPVariable_Unpack(a[0]), &k = THPVariable_Unpack(a[1]);
  const at::Tensor q_out = made(q.sizes(), like(q)), k_out = made(k.sizes(), like(k));
  Block block(*e);
  auto* p = block.as<LfRotateParamsHost>();
  p->q = at_(a[0]);
  p->k = at_(a[1]);
  p->table = at_<float>(a[2]);
  p->q_weight = at_(a[3]);
  p->k_weight = at_(a[4]);
  p->positions = at_<int32_t>(a[5]);
  p->q_out = q_out.mutable_data_ptr();
  p->k_out = k_out.mutable_data_ptr();
  if (!launch(*e, block, stream_of(q))) return nullptr;
  return tuple_of({&q_out, &k_out});
  END_HANDLE_TH_ERRORS
}

// rotate_backward(dq_out, dk_out, q, k, table, q_weight, k_weight, positions, eps, pairs, of q_weight, of k_weight) -> (dq, dk, dq_weight, dk_weight);
// more: floats of the weights' partial sums
PyObject* rotate_backward(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 12)) return nullptr;
  auto e = find('R', a, 8, 7, nullptr, a + 8, 4);
  if (!e) return none();
  const at::Tensor &dq_out = THPVariable_Unpack(a[0]), &dk_out = THPVariable_Unpack(a[1]);
  const at::Tensor dq = made(dq_out.sizes(), like(dq_out)), dk = made(dk_out.sizes(), like(dk_out));
  at::Tensor parts, dw[2];
  Block block(*e);
  auto* p = block.as<LfRotateBwdParamsHost>();
  p->dq_out = at_(a[0]);
  p->dk_out = at_(a[1]);
  p->q = at_(a[2]);
  p->k = at_(a[3]);
  p->table = at_<float>(a[4]);
  p->q_weight = at_(a[5]);
  p->k_weight = at_(a[6]);
  p->positions = at_<int32_t>(a[7]);
  p->dq = dq.mutable_data_ptr();
  p->dk = dk.mutable_data_ptr();
  for (int i = 0; i < 2; ++i)
    if (a[10 + i] == Py_True) {
      const at::Tensor& w = THPVariable_Unpack(a[5 + i]);
      dw[i] = made(w.sizes(), like(w));
      (i ? p->dk_weight : p->dq_weight) = dw[i].mutable_data_ptr();
    }
  if (e->more[0]) {
    parts = made({e->more[0]}, like(dq_out).dtype(at::kFloat));
    p->parts = parts.mutable_data_ptr<float>();
  }
  if (!launch(*e, block, stream_of(dq_out))) return nullptr;
  return tuple_of({&dq, &dk, &dw[0], &dw[1]});
  END_HANDLE_TH_ERRORS
}

// The gradients of rotate_heads as a node of the graph: a node in Python takes 19 us more of the host (6001 rows of 16 and 4 heads of 64 with gradients 95 / 76 us, 26 of them the kernels; the rest is torch's
// engine).  Where its launches are not kept, or what it returns
// is to be part of a graph, it calls `differentiate` (rotary._differentiate).
PyObject* differentiate = nullptr;
struct RotateNode : torch::autograd::Node {
  torch::autograd::SavedVariable q, k, table, q_weight, k_weight, positions;
  bool norm = false, pairs = false;
  double eps = 0.0;

  std::string name() const override { return "RotateHeadsBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (torch::autograd::SavedVariable* v : {&q, &k, &table, &q_weight, &k_weight, &positions}) v->reset_data();
  }

  torch::autograd::variable_list apply(torch::autograd::variable_list&& grads) override {
    at::Tensor saved[6];
    {
      std::lock_guard<std::mutex> lock(mutex_);
      const torch::autograd::SavedVariable* from[] = {&q, &k, &table, &q_weight, &k_weight, &positions};
      for (int i = 0; i < 6; ++i) saved[i] = from[i]->unpack();
    }
    for (int i = 0; i < 2; ++i)
      if (!grads[i].defined()) grads[i] = input_metadata(i).zeros_like();
    pybind11::gil_scoped_acquire gil;
    auto wrap = [](const at::Tensor& t) { return t.defined() ? THPVariable_Wrap(t) : none(); };
    PyObject* a[12] = {wrap(grads[0]), wrap(grads[1]), wrap(saved[0]), wrap(saved[1]), wrap(saved[2]), wrap(saved[3]), wrap(saved[4]), wrap(saved[5]),
                       norm ? PyFloat_FromDouble(eps) : none(), PyBool_FromLong(pairs), PyBool_FromLong(saved[3].defined() && task_should_compute_output(2)),
                       PyBool_FromLong(saved[4].defined() && task_should_compute_output(3))};
    PyObject* r = nullptr;
    bool made_all = true;
    for (PyObject* x : a) made_all = made_all && x;
    if (made_all) {
      if (c10::GradMode::is_enabled())
        r = none();
      else
        r = rotate_backward(nullptr, a, 12);
      if (r == Py_None) {
        Py_DECREF(r);
        r = PyObject_Vectorcall(differentiate, a, 12, nullptr);
      }
    }
    for (PyObject* x : a) Py_XDECREF(x);
    torch::autograd::variable_list res(4);
    if (r)
      for (int i = 0; i < 4; ++i) {
        PyObject* x = PyTuple_GET_ITEM(r, i);
        if (x != Py_None) res[i] = THPVariable_Unpack(x);
      }
    Py_XDECREF(r);
    if (!r) {
      python_error e;
      e.persist();
      throw std::move(e);
    }
    return res;
  }
};

// rotate(q, k, table, q_weight, k_weight, positions, eps, pairs, differentiate) -> (q, k), with gradients where they are asked for
PyObject* rotate(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 9)) return nullptr;
  bool train = false;
  if (c10::GradMode::is_enabled()) {
    if (THPVariable_Check(a[2]) && THPVariable_Unpack(a[2]).requires_grad()) return none();      // (refused)
    for (int i : {0, 1, 3, 4}) train = train || (THPVariable_Check(a[i]) && THPVariable_Unpack(a[i]).requires_grad());
  }
  if (!train) return rotate_heads(nullptr, a, 8);
  if (!plain(a[0]) || (a[6] != Py_None && !PyFloat_CheckExact(a[6])) || !PyBool_Check(a[7]) || c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None) return none();
  PyObject* out = rotate_heads(nullptr, a, 8);
  if (!out || out == Py_None) return out;
  pybind11::object owned = pybind11::reinterpret_steal<pybind11::object>(out);
  if (!differentiate) Py_INCREF(differentiate = a[8]);
  at::Tensor in[6];
  for (int i = 0; i < 6; ++i)
    if (a[i] != Py_None) in[i] = THPVariable_Unpack(a[i]);
  const std::shared_ptr<RotateNode> node(new RotateNode(), torch::autograd::deleteNode);
  node->set_next_edges(torch::autograd::collect_next_edges(in[0], in[1], in[3], in[4]));
  node->norm = a[6] != Py_None;
  node->eps = node->norm ? PyFloat_AS_DOUBLE(a[6]) : 0.0;
  node->pairs = a[7] == Py_True;
  // (in the order in which rotary._Rotate saves them: a recomputation may take either path, and what it saves is matched by its place)
  const std::pair<torch::autograd::SavedVariable*, const at::Tensor*> saved[] = {{&node->q, &in[0]}, {&node->k, &in[1]}, {&node->positions, &in[5]},
                                                                                 {&node->table, &in[2]}, {&node->q_weight, &in[3]}, {&node->k_weight, &in[4]}};
  for (int i = node->norm ? 0 : 2; i < 6; ++i) *saved[i].first = torch::autograd::SavedVariable(*saved[i].second, false);
  for (int i = 0; i < 2; ++i) torch::autograd::set_history(THPVariable_Unpack(PyTuple_GET_ITEM(out, i)), node);
  return owned.release().ptr();
  END_HANDLE_TH_ERRORS
}

// append_kv(q, k, v, k_pool, v_pool, k_scales, v_scales, table, q_weight, k_weight, slots, positions, eps, pairs) -> q, without positions True; the pools are those
// of 16-bit rows, or the codes with their scales
PyObject* append_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 14)) return nullptr;
  auto e = find('a', a, 12, 10, nullptr, a + 12, 2);
  if (!e) return none();
  const at::Tensor& q = THPVariable_Unpack(a[0]);
  at::Tensor out;
  Block block(*e);
  auto* p = block.as<LfRotateParamsHost>();
  p->q = at_(a[0]);
  p->k = at_(a[1]);
  p->v = at_(a[2]);
  p->k_out = at_(a[3]);
  p->v_out = at_(a[4]);
  p->k_scales = at_<uint8_t>(a[5]);
  p->v_scales = at_<uint8_t>(a[6]);
  p->table = at_<float>(a[7]);
  p->q_weight = at_(a[8]);
  p->k_weight = at_(a[9]);
  p->slots = at_<int32_t>(a[10]);
  p->positions = at_<int32_t>(a[11]);
  if (a[11] != Py_None) {
    out = made(q.sizes(), like(q));
    p->q_out = out.mutable_data_ptr();
  }
  if (!launch(*e, block, stream_of(q))) return nullptr;
  if (out.defined()) return THPVariable_Wrap(out);
  Py_RETURN_TRUE;
  END_HANDLE_TH_ERRORS
}

// read_kv(k_pool, v_pool, k_scales, v_scales, slots, fp16) -> (k, v); more: the shape of either
PyObject* read_kv(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 6)) return nullptr;
  auto e = find('g', a, 5, 4, nullptr, a + 5, 1);
  if (!e) return none();
  const auto options = like(THPVariable_Unpack(a[0])).dtype(a[5] == Py_True ? at::kHalf : at::kBFloat16);
  const at::Tensor k = made({e->more[0], e->more[1], e->more[2]}, options), v = made(k.sizes(), options);
  Block block(*e);
  auto* p = block.as<LfReadParamsHost>();
  p->k_pool = at_(a[0]);
  p->v_pool = at_(a[1]);
  p->k_scales = at_<uint8_t>(a[2]);
  p->v_scales = at_<uint8_t>(a[3]);
  p->slots = at_<int32_t>(a[4]);
  p->k = k.mutable_data_ptr();
  p->v = v.mutable_data_ptr();
  if (!launch(*e, block, stream_of(k))) return nullptr;
  return tuple_of({&k, &v});
  END_HANDLE_TH_ERRORS
}

// attention_cached(q, k_codes, v_codes, k_scales, v_scales, out, table, lengths, offsets, positions, plan) -> O; more: floats of scratch, and the bytes in front of
// part_ml in it
PyObject* attention_cached(PyObject*, PyObject* const* a, Py_ssize_t n) {
  HANDLE_TH_ERRORS
  if (!takes(n, 11)) return nullptr;
  auto e = find('c', a, 10, 6, a[10], nullptr, 0);
  if (!e) return none();
  const at::Tensor& q = THPVariable_Unpack(a[0]);
  const at::Tensor out = a[5] == Py_None ? made(q.sizes(), like(q)) : THPVariable_Unpack(a[5]);
  Block block(*e);
  auto* p = block.as<LfCachedParamsHost>();
  p->q = at_(a[0]);
  p->k = at_<uint8_t>(a[1]);
  p->v = at_<uint8_t>(a[2]);
  p->k_scales = at_<uint8_t>(a[3]);
  p->v_scales = at_<uint8_t>(a[4]);
  p->o = out.mutable_data_ptr();
  p->table = at_(a[6]);
  p->lengths = at_<int32_t>(a[7]);
  p->offsets = at_<int32_t>(a[8]);
  p->positions = at_<int32_t>(a[9]);
  void* stream = stream_of(q);
  if (e->more[0]) {
    int rc;
    {
      // (without the GIL: whoever holds the lock needs nothing of Python's)
      pybind11::gil_scoped_release without;
      std::lock_guard<std::mutex> lock(scratch_lock);
      const at::Tensor room = partial_results(e->more[0], q, stream);
      p->part_acc = room.mutable_data_ptr<float>();
      p->part_ml = reinterpret_cast<float*>(reinterpret_cast<char*>(p->part_acc) + e->more[1]);
      rc = env.launch(reinterpret_cast<const lf_launch_item*>(e->items.data()), e->count, block.bytes, stream);
    }
    if (rc) {
      Py_XDECREF(PyObject_CallFunction(env.fail, "i", rc));
      return nullptr;
    }
    if (PyObject_SetAttr(env.last, name_record, e->record)) return nullptr;
  } else if (!launch(*e, block, stream)) {
    return nullptr;
  }
  if (a[5] == Py_None) return THPVariable_Wrap(out);
  Py_INCREF(a[5]);
  return a[5];
  END_HANDLE_TH_ERRORS
}

#define LF_FAST(f) {#f, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {LF_FAST(setup), LF_FAST(key), LF_FAST(keep), {"clear", clear, METH_NOARGS, nullptr}, {"size", size, METH_NOARGS, nullptr},
                         LF_FAST(elsewhere), LF_FAST(packed_layout), LF_FAST(extend_tables), LF_FAST(store_kv), LF_FAST(attention_shared), LF_FAST(attention_packed), LF_FAST(attention_packed_backward),
                         LF_FAST(rotate_heads), LF_FAST(rotate_backward), LF_FAST(rotate), LF_FAST(append_kv), LF_FAST(read_kv), LF_FAST(attention_cached),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_lf_host", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__lf_host() {
  const char* fields[] = {"mask", "window", "scale", "softcap", "k_paged", "v_paged", "denom_add"};
  for (int i = 0; i < 7; ++i)
    if (!(names[i] = PyUnicode_InternFromString(fields[i]))) return nullptr;
  if (!(name_environ = PyUnicode_InternFromString("environ")) || !(name_record = PyUnicode_InternFromString("record"))) return nullptr;
  return PyModule_Create(&module);
}
