// Python binding of the calls that run once per layer and token (the q/k head
// pass and the 8-bit cache), for lara_b200.ops and lara_b200.kvquant.
//
// A decode step's kernels take 3 to 7 us each, and checking six to nine tensors
// in Python and converting up to forty arguments with ctypes took 7 to 11 us a
// call.  Here a call's tensors are read from their C++ objects and its checks
// cost well under a microsecond.  The functions take positional arguments (the
// Python functions order them), raise TypeError and ValueError for what the
// call cannot take, and return the status code of the C ABI (include/
// lara_b200.h), whose entry points they are given as addresses by init().
#define PY_SSIZE_T_CLEAN
#include <Python.h>

#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/version.h>

#include <cstdio>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "../../include/lara_b200.h"

namespace {

decltype(&lara_qk_norm_rope) f_norm_rope = nullptr;
decltype(&lara_kvq_append) f_append = nullptr;
decltype(&lara_kvq_append_qkv) f_append_qkv = nullptr;
decltype(&lara_kvq_read) f_read = nullptr;
decltype(&lara_gqa_decode_kvq) f_decode = nullptr;

struct BadType : std::runtime_error {
  using std::runtime_error::runtime_error;
};
struct BadValue : std::runtime_error {
  using std::runtime_error::runtime_error;
};

std::string text(const at::IntArrayRef& sizes) {
  std::string s = "(";
  for (size_t i = 0; i < sizes.size(); ++i) s += (i ? ", " : "") + std::to_string(sizes[i]);
  return s + (sizes.size() == 1 ? ",)" : ")");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw BadType(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}

int index_of(const at::Tensor& t) { return t.is_cuda() ? (int)t.get_device() : -1; }

// bf16 words, rows contiguous in the last dim, on device `index` (the check of
// ops._strided); returns the data pointer.
uint16_t* rows(const at::Tensor& t, const char* name, at::IntArrayRef shape, int index, bool written = false) {
  const at::ScalarType dt = t.scalar_type();
  if (dt != at::kBFloat16 && dt != at::kShort && dt != at::kUInt16)
    throw BadType(std::string(name) + " must hold bf16 words (bfloat16/int16/uint16), got " + at::toString(dt));
  if (index < 0 || index_of(t) != index)
    throw BadValue(std::string(name) + " must be on the CUDA device of the call, got " + t.device().str());
  if (t.sizes() != shape)
    throw BadValue(std::string(name) + " has shape " + text(t.sizes()) + ", expected " + text(shape));
  if (t.stride(-1) != 1) throw BadValue(std::string(name) + " must be contiguous in its last dimension");
  if (written)
    for (int64_t i = 0; i < t.dim(); ++i)
      if (t.stride(i) == 0 && t.size(i) > 1)
        throw BadValue(std::string(name) + " is written and must not repeat elements (a stride of 0)");
  return static_cast<uint16_t*>(t.data_ptr());
}

uint16_t* optional_row(PyObject* o, const char* name, int64_t d, int index) {
  return o == Py_None ? nullptr : rows(tensor(o, name), name, {d}, index);
}

int32_t* ints(PyObject* o, const char* name, int64_t n, int index) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, name);
  if (t.scalar_type() != at::kInt || index_of(t) != index || t.numel() != n || !t.is_contiguous())
    throw BadValue(std::string(name) + " must be a contiguous int32 tensor of length " + std::to_string(n) +
                   " on the pool's device");
  return static_cast<int32_t*>(t.data_ptr());
}

int checked_int(int64_t n, const char* name) {
  if (n > 0x7fffffff) throw BadValue(std::string(name) + " is too large");
  return (int)n;
}

const int32_t* block_table(PyObject* o, int64_t batch, int index, int* pages) {
  const at::Tensor& t = tensor(o, "block_table");
  if (t.scalar_type() != at::kInt || index_of(t) != index || t.dim() != 2 || !t.is_contiguous())
    throw BadValue("block_table must be a contiguous int32 [batch, pages_per_seq] tensor on the pool's device");
  if (t.size(0) != batch)
    throw BadValue("block_table has " + std::to_string(t.size(0)) + " rows for a batch of " + std::to_string(batch));
  *pages = checked_int(t.size(1), "block_table's pages per sequence");
  return static_cast<const int32_t*>(t.data_ptr());
}

struct Table {
  const float* p = nullptr;
  int max_pos = 0, rot = 0;
};

Table rope_table(PyObject* o, int index) {
  if (o == Py_None) return {};
  const at::Tensor& t = tensor(o, "cos_sin");
  if (t.scalar_type() != at::kFloat || index_of(t) != index || t.dim() != 2 || !t.is_contiguous())
    throw BadValue("cos_sin must be a contiguous float32 [max_pos, rot_dim] tensor on the same device");
  return {static_cast<const float*>(t.data_ptr()), checked_int(t.size(0), "cos_sin's positions"),
          checked_int(t.size(1), "rot_dim")};
}

void* workspace(PyObject* o, int index, size_t* bytes = nullptr) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, "workspace");
  if (index_of(t) != index || !t.is_contiguous()) throw BadValue("workspace must be a contiguous tensor on the same device");
  if (bytes)
    *bytes = t.nbytes();  // checked by the call
  else if (t.nbytes() < 256 || reinterpret_cast<uintptr_t>(t.data_ptr()) % 4)
    throw BadValue("workspace must hold at least 256 bytes, 4-byte aligned (ops.new_workspace)");
  return t.data_ptr();
}

double number(PyObject* o) {
  const double x = PyFloat_AsDouble(o);
  if (x == -1.0 && PyErr_Occurred()) {
    PyErr_Clear();
    throw BadType("a number is needed, got " + std::string(Py_TYPE(o)->tp_name));
  }
  return x;
}

long long integer(PyObject* o) {
  const long long x = PyLong_AsLongLong(o);
  if (x == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    throw BadType("a whole number is needed, got " + std::string(Py_TYPE(o)->tp_name));
  }
  return x;
}

bool truth(PyObject* o) {
  const int x = PyObject_IsTrue(o);
  if (x < 0) {
    PyErr_Clear();
    throw BadType("a truth value is needed, got " + std::string(Py_TYPE(o)->tp_name));
  }
  return x == 1;
}

const lara_kvq_pool* pool_of(PyObject* o) {
  return reinterpret_cast<const lara_kvq_pool*>(static_cast<uintptr_t>(integer(o)));
}

// Runs f; Python exceptions for C++ ones.
template <typename F>
PyObject* guarded(Py_ssize_t got, Py_ssize_t want, F f) {
  try {
    if (got != want) throw BadType("expected " + std::to_string(want) + " arguments");
    return PyLong_FromLong(f());
  } catch (const BadType& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const BadValue& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// Calls f(stream) with the device current, on its current stream, and without
// the interpreter's lock (a launch waits when the stream's queue is full).
template <typename F>
int launch(int index, F f) {
  const c10::cuda::CUDAGuard guard((c10::DeviceIndex)index);
  void* const stream = c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)index).stream();
  PyThreadState* const state = PyEval_SaveThread();
  const int rc = f(stream);
  PyEval_RestoreThread(state);
  return rc;
}

// q, k, q_out, k_out, positions, cos_sin, q_weight, k_weight, eps, interleaved, workspace
PyObject* norm_rope(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 11, [&] {
    const at::Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k");
    const int64_t nd = q.dim();
    if ((nd != 3 && nd != 4) || k.dim() != nd) throw BadValue("q and k must be [T, H, D] or [B, n, H, D]");
    const int index = index_of(q);
    const at::IntArrayRef qs = q.sizes();
    int64_t k_dims[4];
    for (int64_t i = 0; i < nd; ++i) k_dims[i] = qs[i];
    k_dims[nd - 2] = k.size(nd - 2);
    const at::IntArrayRef ks(k_dims, nd);
    uint16_t* qp = rows(q, "q", qs, index);
    uint16_t* kp = rows(k, "k", ks, index);
    const at::Tensor &qo = tensor(a[2], "q out"), &ko = tensor(a[3], "k out");
    uint16_t* qop = rows(qo, "q out", qs, index, true);
    uint16_t* kop = rows(ko, "k out", ks, index, true);
    const int64_t d = qs[nd - 1];
    const uint16_t* qw = optional_row(a[6], "q_weight", d, index);
    const uint16_t* kw = optional_row(a[7], "k_weight", d, index);
    const Table table = rope_table(a[5], index);
    const int64_t B = nd == 4 ? qs[0] : 1, n = qs[nd - 3];
    const int32_t* pos = nullptr;
    if (table.p) {
      if (a[4] == Py_None) throw BadValue("a rotation needs positions");
      const at::Tensor& p = tensor(a[4], "positions");
      if (p.scalar_type() != at::kInt || index_of(p) != index || p.sizes() != qs.slice(0, nd - 2) || !p.is_contiguous())
        throw BadValue("positions must be a contiguous int32 tensor of shape " + text(qs.slice(0, nd - 2)) +
                       " on the same device");
      pos = static_cast<const int32_t*>(p.data_ptr());
    }
    const float eps = (float)number(a[8]);
    const int inter = truth(a[9]), batch = checked_int(B, "batch"), tokens = checked_int(n, "n");
    const int hq = checked_int(qs[nd - 2], "heads"), hkv = checked_int(k_dims[nd - 2], "heads");
    const int head_dim = checked_int(d, "head_dim");
    void* const ws = workspace(a[10], index);
    return launch(index, [&](void* stream) {
      return f_norm_rope(qp, q.stride(0), q.stride(nd - 3), q.stride(nd - 2), kp, k.stride(0), k.stride(nd - 3),
                         k.stride(nd - 2), qop, qo.stride(0), qo.stride(nd - 3), qo.stride(nd - 2), kop, ko.stride(0),
                         ko.stride(nd - 3), ko.stride(nd - 2), batch, tokens, hq, hkv, head_dim, pos, table.p,
                         table.max_pos, table.rot, inter, qw, kw, eps, ws, stream);
    });
  });
}

// pool, device, block_table, starts, k, v, counts, new_lens, workspace
PyObject* append(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 9, [&] {
    const lara_kvq_pool* pool = pool_of(a[0]);
    const int index = checked_int(integer(a[1]), "device");
    const at::Tensor &k = tensor(a[4], "k_new"), &v = tensor(a[5], "v_new");
    if (k.dim() != 4) throw BadValue("k_new must be [B, Hkv, n, D]");
    const int64_t B = k.size(0), n = k.size(2);
    const int64_t shape[4] = {B, pool->n_kv_heads, n, pool->head_dim};
    const uint16_t* kp = rows(k, "k_new", shape, index);
    const uint16_t* vp = rows(v, "v_new", shape, index);
    int pages = 0;
    const int32_t* table = block_table(a[2], B, index, &pages);
    if (a[3] == Py_None) throw BadValue("starts must be a tensor");
    const int32_t* starts = ints(a[3], "starts", B, index);
    const int32_t* counts = ints(a[6], "counts", B, index);
    int32_t* new_lens = ints(a[7], "new_lens", B, index);
    const int batch = checked_int(B, "batch"), tokens = checked_int(n, "n");
    void* const ws = workspace(a[8], index);
    return launch(index, [&](void* stream) {
      return f_append(pool, table, pages, starts, counts, new_lens, kp, k.stride(0), k.stride(1), k.stride(2), vp,
                      v.stride(0), v.stride(1), v.stride(2), batch, tokens, ws, stream);
    });
  });
}

// pool, device, block_table, starts, q, k, v, q_out, positions, cos_sin, q_weight, k_weight, eps, interleaved,
// counts, new_lens, workspace
PyObject* append_qkv(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 17, [&] {
    const lara_kvq_pool* pool = pool_of(a[0]);
    const int index = checked_int(integer(a[1]), "device");
    const at::Tensor &q = tensor(a[4], "q"), &k = tensor(a[5], "k"), &v = tensor(a[6], "v"), &qo = tensor(a[7], "out");
    if (q.dim() != 4) throw BadValue("q must be [B, n, Hq, D]");
    const int64_t B = q.size(0), n = q.size(1), hq = q.size(2), d = pool->head_dim;
    const int64_t q_shape[4] = {B, n, hq, d}, kv_shape[4] = {B, n, pool->n_kv_heads, d};
    const uint16_t* qp = rows(q, "q", q_shape, index);
    const uint16_t* kp = rows(k, "k", kv_shape, index);
    const uint16_t* vp = rows(v, "v", kv_shape, index);
    uint16_t* qop = rows(qo, "out", q_shape, index, true);
    int pages = 0;
    const int32_t* blocks = block_table(a[2], B, index, &pages);
    if (a[3] == Py_None) throw BadValue("starts must be a tensor");
    const int32_t* starts = ints(a[3], "starts", B, index);
    const int32_t* positions = ints(a[8], "positions", B * n, index);
    const Table table = rope_table(a[9], index);
    const uint16_t* qw = optional_row(a[10], "q_weight", d, index);
    const uint16_t* kw = optional_row(a[11], "k_weight", d, index);
    const int32_t* counts = ints(a[14], "counts", B, index);
    int32_t* new_lens = ints(a[15], "new_lens", B, index);
    const float eps = (float)number(a[12]);
    const int inter = truth(a[13]), batch = checked_int(B, "batch"), tokens = checked_int(n, "n");
    const int heads = checked_int(hq, "heads");
    void* const ws = workspace(a[16], index);
    return launch(index, [&](void* stream) {
      return f_append_qkv(pool, blocks, pages, starts, counts, new_lens, qp, q.stride(0), q.stride(1), q.stride(2), kp,
                          k.stride(0), k.stride(1), k.stride(2), vp, v.stride(0), v.stride(1), v.stride(2), qop,
                          qo.stride(0), qo.stride(1), qo.stride(2), batch, tokens, heads, positions, table.p,
                          table.max_pos, table.rot, inter, qw, kw, eps, ws, stream);
    });
  });
}

// pool, device, block_table, seq_lens, n_tokens, starts, k_out, v_out, workspace
PyObject* read(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 9, [&] {
    const lara_kvq_pool* pool = pool_of(a[0]);
    const int index = checked_int(integer(a[1]), "device");
    const at::Tensor& lens = tensor(a[3], "seq_lens");
    const int64_t B = lens.numel(), n = integer(a[4]);
    const int64_t shape[4] = {B, pool->n_kv_heads, n, pool->head_dim};
    const at::Tensor &k = tensor(a[6], "k out"), &v = tensor(a[7], "v out");
    uint16_t* kp = rows(k, "k out", shape, index, true);
    uint16_t* vp = rows(v, "v out", shape, index, true);
    int pages = 0;
    const int32_t* table = block_table(a[2], B, index, &pages);
    const int32_t* seq_lens = ints(a[3], "seq_lens", B, index);
    const int32_t* starts = ints(a[5], "starts", B, index);
    const int batch = checked_int(B, "batch"), tokens = checked_int(n, "n_tokens");
    void* const ws = workspace(a[8], index);
    return launch(index, [&](void* stream) {
      return f_read(pool, table, pages, seq_lens, starts, kp, k.stride(0), k.stride(1), k.stride(2), vp, v.stride(0),
                    v.stride(1), v.stride(2), batch, tokens, ws, stream);
    });
  });
}

// pool, device, q, block_table, seq_lens, out, scale, workspace
PyObject* decode(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 8, [&] {
    const lara_kvq_pool* pool = pool_of(a[0]);
    const int index = checked_int(integer(a[1]), "device");
    const at::Tensor &q = tensor(a[2], "q"), &o = tensor(a[5], "out");
    if (q.dim() != 3) throw BadValue("q must be [B, Hq, D]");
    const int64_t B = q.size(0), hq = q.size(1);
    const int64_t shape[3] = {B, hq, pool->head_dim};
    const uint16_t* qp = rows(q, "q", shape, index);
    uint16_t* op = rows(o, "out", shape, index, true);
    if (!q.is_contiguous() || !o.is_contiguous()) throw BadValue("q and out must be contiguous");
    int pages = 0;
    const int32_t* table = block_table(a[3], B, index, &pages);
    if (a[4] == Py_None) throw BadValue("seq_lens must be a tensor");
    const int32_t* lens = ints(a[4], "seq_lens", B, index);
    size_t bytes = 0;
    void* ws = workspace(a[7], index, &bytes);
    const float scale = (float)number(a[6]);
    const int batch = checked_int(B, "batch"), heads = checked_int(hq, "heads");
    return launch(index, [&](void* stream) {
      return f_decode(qp, pool, table, pages, lens, op, batch, heads, scale, ws, bytes, stream);
    });
  });
}

// The addresses of the five C entry points, in the order of this file.
PyObject* init(PyObject*, PyObject* const* a, Py_ssize_t n_args) {
  return guarded(n_args, 5, [&] {
    f_norm_rope = reinterpret_cast<decltype(f_norm_rope)>(static_cast<uintptr_t>(integer(a[0])));
    f_append = reinterpret_cast<decltype(f_append)>(static_cast<uintptr_t>(integer(a[1])));
    f_append_qkv = reinterpret_cast<decltype(f_append_qkv)>(static_cast<uintptr_t>(integer(a[2])));
    f_read = reinterpret_cast<decltype(f_read)>(static_cast<uintptr_t>(integer(a[3])));
    f_decode = reinterpret_cast<decltype(f_decode)>(static_cast<uintptr_t>(integer(a[4])));
    return 0;
  });
}

#define LARA_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {LARA_METHOD(init), LARA_METHOD(norm_rope), LARA_METHOD(append), LARA_METHOD(append_qkv),
                         LARA_METHOD(read), LARA_METHOD(decode),    {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding() {
  PyObject* const m = PyModule_Create(&module);
  if (m && PyModule_AddStringConstant(m, "torch_version", TORCH_VERSION) < 0) {
    Py_DECREF(m);
    return nullptr;
  }
  return m;
}
