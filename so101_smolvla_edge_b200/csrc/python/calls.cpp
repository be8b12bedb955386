// The Python side of the text tower's serving operators: tensor checks, the result's allocation, the
// current stream and the C ABI call (include/so101_b200_text.h), in one native step.
//
// These operators run once per layer and token, on kernels of 4 to 20 us. With the checks in Python and the call
// through ctypes, a call of attention_pages took 10.5 us of host time (the launch itself about 4), so
// that a decoding step waited for its host. ops.py keeps the names, defaults and documentation and hands its arguments on in order.
//
// Plain CPython functions (METH_FASTCALL): every one takes its arguments by position, raises ValueError for a
// tensor that the operator does not take, and passes a status other than SO101_OK to the `check` callable that
// the package registered (its exception types). C++ exceptions become Python ones at the boundary. The call is made with
// the tensors' device current: the library launches, looks up and records on the current one.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdarg>
#include <map>
#include <mutex>
#include <utility>
#include <vector>

#include "../../../include/so101_b200_text.h"

namespace {

PyObject* g_check = nullptr;      // check(status, name): raises
PyObject* g_workspace = nullptr;  // workspace(device, stream): makes and registers a workspace

struct Space {
  void* partials;
  int64_t bytes;
  int* tickets;
  int64_t n_tickets;
};
std::map<std::pair<int, int64_t>, Space> g_spaces;  // by device and stream; under the interpreter lock

// A Python error is already set.
struct Raised {};

[[noreturn]] void refuse(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  PyErr_FormatV(PyExc_ValueError, fmt, ap);
  va_end(ap);
  throw Raised{};
}

void status(int rc, const char* name) {
  if (rc == SO101_OK) return;
  PyObject* r = PyObject_CallFunction(g_check, "is", rc, name);
  if (r) {
    Py_DECREF(r);
    PyErr_Format(PyExc_RuntimeError, "%s: status %d", name, rc);
  }
  throw Raised{};
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{};
  return v;
}

int small(PyObject* o, const char* name) {
  const int64_t v = integer(o);
  if (v < INT32_MIN || v > INT32_MAX) refuse("%s is out of range", name);
  return static_cast<int>(v);
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) refuse("%s must be a tensor", name);
  return THPVariable_Unpack(o);
}

c10::Device cuda_device(const at::Tensor& t) {
  if (!t.is_cuda()) refuse("the B200 kernels take CUDA tensors only");
  return t.device();
}

struct Rows {
  void* p;
  int64_t ld;
};

// bf16 rows (rows, cols), any row stride.
Rows bf16_rows(const at::Tensor& t, const char* name, int64_t rows, int64_t cols, c10::Device dev) {
  if (t.scalar_type() != at::kBFloat16 || t.dim() != 2 || t.size(0) != rows || t.size(1) != cols || t.device() != dev)
    refuse("%s must be bf16 (%lld, %lld) on %s", name, static_cast<long long>(rows), static_cast<long long>(cols),
           dev.str().c_str());
  if (t.stride(1) != 1 && cols > 1) refuse("%s needs unit column stride", name);
  return {t.data_ptr(), rows > 1 ? t.stride(0) : cols};  // (a single row's stride may be anything)
}

// A contiguous int32 vector, or null where None is allowed.
const int* ints(PyObject* o, const char* name, c10::Device dev, int64_t* n, bool optional = false) {
  if (optional && o == Py_None) {
    *n = -1;
    return nullptr;
  }
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || t.dim() != 1 || !t.is_contiguous() || t.device() != dev)
    refuse("%s must be a contiguous int32 vector on %s", name, dev.str().c_str());
  *n = t.numel();
  return static_cast<const int*>(t.data_ptr());
}

struct Rope {
  const float* cos;
  const float* sin;
};

Rope rope(PyObject* c, PyObject* s, int64_t rows, int64_t half, c10::Device dev) {
  if (c == Py_None && s == Py_None) return {nullptr, nullptr};
  if (c == Py_None || s == Py_None) refuse("cos and sin come together");
  const float* p[2];
  PyObject* both[2] = {c, s};
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& t = tensor(both[i], i ? "sin" : "cos");
    if (t.scalar_type() != at::kFloat || t.dim() != 2 || t.size(0) != rows || t.size(1) != half || !t.is_contiguous() ||
        t.device() != dev)
      refuse("cos and sin must be contiguous float32 (%lld, %lld) on %s", static_cast<long long>(rows),
             static_cast<long long>(half), dev.str().c_str());
    p[i] = static_cast<const float*>(t.data_ptr());
  }
  return {p[0], p[1]};
}

float scale_of(PyObject* o, int hd) {
  if (o == Py_None) return static_cast<float>(1.0 / std::sqrt(static_cast<double>(hd)));
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised{};
  return static_cast<float>(v);
}

bool truth(PyObject* o) {
  const int v = PyObject_IsTrue(o);
  if (v < 0) throw Raised{};
  return v != 0;
}

// `out` where given, else fresh bf16 rows.
at::Tensor result(PyObject* o, int64_t rows, int64_t cols, c10::Device dev) {
  if (o != Py_None) return tensor(o, "out");
  return at::empty({rows, cols}, at::TensorOptions().dtype(at::kBFloat16).device(dev));
}

cudaStream_t stream_of(c10::Device dev) { return c10::cuda::getCurrentCUDAStream(dev.index()).stream(); }

// The cache behind a handle: (address of its so101_kv_pages, device index).
const so101_kv_pages* cache(PyObject* handle, c10::Device* dev) {
  if (!PyTuple_Check(handle) || PyTuple_GET_SIZE(handle) != 2) refuse("pages must be a KvPages");
  *dev = c10::Device(c10::kCUDA, static_cast<c10::DeviceIndex>(integer(PyTuple_GET_ITEM(handle, 1))));
  return static_cast<const so101_kv_pages*>(PyLong_AsVoidPtr(PyTuple_GET_ITEM(handle, 0)));
}

// Entries of a list of sequences given by starts (or one per row) and seqs.
int64_t entries(int64_t n_starts, int64_t n_seqs, int64_t rows) {
  const int64_t n = n_starts < 0 ? rows : n_starts - 1;
  if (n < 0 || (n_seqs >= 0 && n_seqs != n))
    refuse("starts has one entry more than there are sequences, seqs one per sequence");
  if (n > INT32_MAX) refuse("too many sequences");
  return n;
}

// What a graph under capture uses: (capture id, stream) -> its workspace. The graph may be replayed beside eager calls on its
// capture stream and beside other graphs captured there, so it has partials and tickets of its own, which it clears
// at its start and which live as long as it does (a CUDA user object holds them). The object's destructor may run on
// a thread of the driver's and make no CUDA calls: it hands them to the next call here.
using CaptureKey = std::pair<unsigned long long, int64_t>;
struct Held {
  at::Tensor memory;
  CaptureKey key;
};
std::map<CaptureKey, Space> g_captured;  // under the interpreter lock, as g_spaces
// (never destroyed: the driver may end the last graphs after this module's own objects are gone)
std::mutex& g_ended_lock = *new std::mutex;
std::vector<Held*>& g_ended = *new std::vector<Held*>;

void CUDART_CB graph_ended(void* held) {
  const std::lock_guard<std::mutex> lock(g_ended_lock);
  g_ended.push_back(static_cast<Held*>(held));
}

void clear_ended() {
  std::vector<Held*> ended;
  {
    const std::lock_guard<std::mutex> lock(g_ended_lock);
    ended.swap(g_ended);
  }
  for (Held* h : ended) {
    g_captured.erase(h->key);
    delete h;
  }
}

constexpr int64_t kSpaceBytes = int64_t(40) << 20, kSpaceTickets = 1184;

const Space& captured_space(c10::Device dev, cudaStream_t stream, unsigned long long id, cudaGraph_t graph) {
  const CaptureKey key(id, reinterpret_cast<int64_t>(stream));
  auto it = g_captured.find(key);
  if (it != g_captured.end()) return it->second;
  const auto bytes = at::TensorOptions().dtype(at::kByte).device(dev);
  const at::Tensor memory = at::empty({kSpaceBytes + kSpaceTickets * 4}, bytes);
  memory.narrow(0, kSpaceBytes, kSpaceTickets * 4).zero_();
  Held* held = new Held{memory, key};
  cudaUserObject_t object;
  cudaError_t e = cudaUserObjectCreate(&object, held, graph_ended, 1, cudaUserObjectNoDestructorSync);
  if (e != cudaSuccess) {
    delete held;
  } else {
    e = cudaGraphRetainUserObject(graph, object, 1, cudaGraphUserObjectMove);
    if (e != cudaSuccess) cudaUserObjectRelease(object, 1);
  }
  if (e != cudaSuccess) {
    PyErr_Format(PyExc_RuntimeError, "a workspace for the graph under capture: %s", cudaGetErrorString(e));
    throw Raised{};
  }
  char* at = static_cast<char*>(memory.data_ptr());
  return g_captured[key] = Space{at, kSpaceBytes, reinterpret_cast<int*>(at + kSpaceBytes), kSpaceTickets};
}

const Space& space(c10::Device dev, cudaStream_t stream) {
  clear_ended();
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  cudaGraph_t graph = nullptr;
  if (cudaStreamGetCaptureInfo(stream, &capture, &id, &graph) != cudaSuccess) cudaGetLastError();  // the launch will say
  else if (capture == cudaStreamCaptureStatusActive) return captured_space(dev, stream, id, graph);
  const std::pair<int, int64_t> key(dev.index(), reinterpret_cast<int64_t>(stream));
  auto it = g_spaces.find(key);
  if (it == g_spaces.end()) {
    PyObject* r = PyObject_CallFunction(g_workspace, "iL", key.first, static_cast<long long>(key.second));
    if (!r) throw Raised{};
    Py_DECREF(r);
    it = g_spaces.find(key);
    if (it == g_spaces.end()) {
      PyErr_SetString(PyExc_RuntimeError, "the workspace was not registered");
      throw Raised{};
    }
  }
  return it->second;
}

void need(Py_ssize_t got, Py_ssize_t want) {
  if (got != want) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", got, want);
    throw Raised{};
  }
}

template <PyObject* (*F)(PyObject* const*, Py_ssize_t)>
PyObject* guarded(PyObject*, PyObject* const* a, Py_ssize_t n) {
  try {
    return F(a, n);
  } catch (const Raised&) {
    return nullptr;
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
    return nullptr;
  }
}

PyObject* none() { Py_RETURN_NONE; }

// q, k, v, starts, max_len, n_heads, n_kv, cos, sin, scale, out
PyObject* attention_packed(PyObject* const* a, Py_ssize_t n) {
  need(n, 11);
  const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k"), &v = tensor(a[2], "v");
  const c10::Device dev = cuda_device(q);
  const int heads = small(a[5], "n_heads"), kv = small(a[6], "n_kv");
  if (k.dim() != 2 || kv < 1 || k.size(1) % kv) refuse("k must be (rows, n_kv * head_dim)");
  const int64_t rows = k.size(0), hd = k.size(1) / kv;
  const Rows rq = bf16_rows(q, "q", rows, heads * hd, dev), rk = bf16_rows(k, "k", rows, kv * hd, dev),
             rv = bf16_rows(v, "v", rows, kv * hd, dev);
  int64_t n_starts;
  const int* starts = ints(a[3], "starts", dev, &n_starts);
  const Rope r = rope(a[7], a[8], rows, hd / 2, dev);
  const c10::cuda::CUDAGuard current(dev);
  const at::Tensor out = result(a[10], rows, heads * hd, dev);
  const Rows ro = bf16_rows(out, "out", rows, heads * hd, dev);
  status(so101_attention_packed(rq.p, rq.ld, rk.p, rk.ld, rv.p, rv.ld, ro.p, ro.ld, rows, starts,
                                static_cast<int>(entries(n_starts, -1, rows)), integer(a[4]), heads, kv,
                                static_cast<int>(hd), scale_of(a[9], static_cast<int>(hd)), r.cos, r.sin, stream_of(dev)),
         "so101_attention_packed");
  return THPVariable_Wrap(out);
}

// pages, layer, k, v, starts, seqs, max_new, cos, sin
PyObject* kv_append(PyObject* const* a, Py_ssize_t n) {
  need(n, 9);
  c10::Device dev(c10::kCUDA, 0);
  const so101_kv_pages* c = cache(a[0], &dev);
  const at::Tensor &k = tensor(a[2], "k"), &v = tensor(a[3], "v");
  if (k.dim() != 2) refuse("k must be (rows, n_kv * head_dim)");
  const int64_t rows = k.size(0), width = static_cast<int64_t>(c->n_kv) * c->hd;
  const Rows rk = bf16_rows(k, "k", rows, width, dev), rv = bf16_rows(v, "v", rows, width, dev);
  int64_t n_starts, n_seqs;
  const int* starts = ints(a[4], "starts", dev, &n_starts, true);
  const int* seqs = ints(a[5], "seqs", dev, &n_seqs, true);
  const Rope r = rope(a[7], a[8], rows, c->hd / 2, dev);
  const c10::cuda::CUDAGuard current(dev);
  status(so101_kv_append(c, small(a[1], "layer"), rk.p, rk.ld, rv.p, rv.ld, rows, starts, seqs,
                         static_cast<int>(entries(n_starts, n_seqs, rows)), integer(a[6]), r.cos, r.sin, stream_of(dev)),
         "so101_kv_append");
  return none();
}

// pages, layer, starts, rows, seqs, first
PyObject* kv_read(PyObject* const* a, Py_ssize_t n) {
  need(n, 6);
  c10::Device dev(c10::kCUDA, 0);
  const so101_kv_pages* c = cache(a[0], &dev);
  int64_t n_starts, n_seqs, n_first;
  const int* starts = ints(a[2], "starts", dev, &n_starts);
  const int64_t rows = integer(a[3]), width = static_cast<int64_t>(c->n_kv) * c->hd;
  if (rows < 0) refuse("rows must not be negative");
  const int* seqs = ints(a[4], "seqs", dev, &n_seqs, true);
  const int* first = ints(a[5], "first", dev, &n_first, true);
  const int64_t count = entries(n_starts, n_seqs, rows);
  if (n_first >= 0 && n_first != count) refuse("first has one entry per sequence");
  const c10::cuda::CUDAGuard current(dev);
  const at::Tensor k = result(Py_None, rows, width, dev), v = result(Py_None, rows, width, dev);
  status(so101_kv_read(c, small(a[1], "layer"), starts, seqs, first, static_cast<int>(count), rows, k.data_ptr(), width,
                       v.data_ptr(), width, stream_of(dev)),
         "so101_kv_read");
  PyObject* both = PyTuple_New(2);
  if (!both) throw Raised{};
  PyTuple_SET_ITEM(both, 0, THPVariable_Wrap(k));
  PyTuple_SET_ITEM(both, 1, THPVariable_Wrap(v));
  return both;
}

// q, pages, layer, n_heads, starts, seqs, max_q, causal, cos, sin, scale, out
PyObject* attention_pages(PyObject* const* a, Py_ssize_t n) {
  need(n, 12);
  c10::Device dev(c10::kCUDA, 0);
  const so101_kv_pages* c = cache(a[1], &dev);
  const at::Tensor& q = tensor(a[0], "q");
  if (q.dim() != 2) refuse("q must be (rows, n_heads * head_dim)");
  const int heads = small(a[3], "n_heads");
  const int64_t rows = q.size(0), width = static_cast<int64_t>(heads) * c->hd;
  const Rows rq = bf16_rows(q, "q", rows, width, dev);
  int64_t n_starts, n_seqs;
  const int* starts = ints(a[4], "starts", dev, &n_starts, true);
  const int* seqs = ints(a[5], "seqs", dev, &n_seqs, true);
  const Rope r = rope(a[8], a[9], rows, c->hd / 2, dev);
  const c10::cuda::CUDAGuard current(dev);
  const at::Tensor out = result(a[11], rows, width, dev);
  const Rows ro = bf16_rows(out, "out", rows, width, dev);
  const cudaStream_t stream = stream_of(dev);
  const Space& ws = space(dev, stream);
  status(so101_attention_pages(rq.p, rq.ld, ro.p, ro.ld, rows, c, small(a[2], "layer"), heads, starts, seqs,
                               static_cast<int>(entries(n_starts, n_seqs, rows)), integer(a[6]), truth(a[7]),
                               scale_of(a[10], c->hd), r.cos, r.sin, ws.partials, ws.bytes, ws.tickets, ws.n_tickets,
                               stream),
         "so101_attention_pages");
  return THPVariable_Wrap(out);
}

// Two int32 vectors of one length (`second` null: one vector).
template <typename Call>
PyObject* lists(PyObject* const* a, Py_ssize_t n, const char* first, const char* second, const char* name, Call call) {
  need(n, second ? 3 : 2);
  c10::Device dev(c10::kCUDA, 0);
  const so101_kv_pages* c = cache(a[0], &dev);
  int64_t na, nb;
  const int* x = ints(a[1], first, dev, &na);
  const int* y = second ? ints(a[2], second, dev, &nb) : nullptr;
  if (second && na != nb) refuse("%s and %s have the same length", first, second);
  if (na > INT32_MAX) refuse("%s is too long", first);
  const c10::cuda::CUDAGuard current(dev);
  status(call(c, x, y, static_cast<int>(na), stream_of(dev)), name);
  return none();
}

PyObject* kv_reserve(PyObject* const* a, Py_ssize_t n) {
  return lists(a, n, "seqs", "tokens", "so101_kv_reserve", so101_kv_reserve);
}
PyObject* kv_fork(PyObject* const* a, Py_ssize_t n) {
  return lists(a, n, "parents", "children", "so101_kv_fork", so101_kv_fork);
}
PyObject* kv_copy(PyObject* const* a, Py_ssize_t n) { return lists(a, n, "src", "dst", "so101_kv_copy", so101_kv_copy); }
PyObject* kv_free(PyObject* const* a, Py_ssize_t n) {
  return lists(a, n, "seqs", nullptr, "so101_kv_free",
               [](const so101_kv_pages* c, const int* x, const int*, int m, cudaStream_t s) {
                 return so101_kv_free(c, x, m, s);
               });
}
PyObject* kv_compact(PyObject* const* a, Py_ssize_t n) {
  need(n, 1);
  c10::Device dev(c10::kCUDA, 0);
  const so101_kv_pages* c = cache(a[0], &dev);
  const c10::cuda::CUDAGuard current(dev);
  status(so101_kv_compact(c, stream_of(dev)), "so101_kv_compact");
  return none();
}

// check, workspace
PyObject* set_up(PyObject* const* a, Py_ssize_t n) {
  need(n, 2);
  Py_INCREF(a[0]);
  Py_INCREF(a[1]);
  Py_XSETREF(g_check, a[0]);
  Py_XSETREF(g_workspace, a[1]);
  return none();
}

// device, stream, partials, bytes, tickets, n_tickets
PyObject* add_workspace(PyObject* const* a, Py_ssize_t n) {
  need(n, 6);
  Space s;
  s.partials = reinterpret_cast<void*>(integer(a[2]));
  s.bytes = integer(a[3]);
  s.tickets = reinterpret_cast<int*>(integer(a[4]));
  s.n_tickets = integer(a[5]);
  g_spaces[{small(a[0], "device"), integer(a[1])}] = s;
  return none();
}

#define SO101_CALL(name) \
  { #name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(&guarded<name>)), METH_FASTCALL, nullptr }
PyMethodDef methods[] = {
    SO101_CALL(set_up),     SO101_CALL(add_workspace), SO101_CALL(attention_packed), SO101_CALL(attention_pages),
    SO101_CALL(kv_append),  SO101_CALL(kv_read),       SO101_CALL(kv_reserve),       SO101_CALL(kv_free),
    SO101_CALL(kv_fork),    SO101_CALL(kv_copy),       SO101_CALL(kv_compact),       {nullptr, nullptr, 0, nullptr}};
#undef SO101_CALL

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_calls", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

extern "C" __attribute__((visibility("default"))) PyObject* PyInit__calls() { return PyModule_Create(&module); }
