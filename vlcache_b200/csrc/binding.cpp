// Python binding of the ops whose device time is below what a call through ctypes takes: the argument checks, the
// allocations and the C-ABI call in one compiled function (a call of decode_attention_window took 20 us in Python
// and ctypes).  vlcache_b200/ops.py documents them; the kernels are in libvlcache_b200.so, whose C ABI is all
// that this file calls.
#include <Python.h>

#include <ATen/ops/empty.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <initializer_list>
#include <stdexcept>
#include <string>

#include "vlcache_b200.h"

namespace {

using at::Tensor;

// What the functions below throw; call() makes Python exceptions of them.
struct Refused : std::runtime_error {  // ValueError
  using std::runtime_error::runtime_error;
};
struct WrongType : std::runtime_error {  // TypeError
  using std::runtime_error::runtime_error;
};
struct Failed {  // vlcache_b200._lib.VLCError
  const char* function;
  int status;
};
struct Raised {};  // already set

void need(bool ok, const char* what) {
  if (!ok) throw Refused(what);
}
void need(bool ok, const char* name, const std::string& what) {
  if (!ok) throw Refused(std::string(name) + ": " + what);
}

// ---- Python arguments
const Tensor& tensor(PyObject* o, const char* name) {
  if (!THPVariable_Check(o)) throw WrongType(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
Tensor optional(PyObject* o, const char* name) { return o == Py_None ? Tensor() : tensor(o, name); }
int64_t integer(PyObject* o) {
  const long long v = PyLong_Check(o) ? PyLong_AsLongLong(o) : [&] {
    PyObject* n = PyNumber_Long(o);  // as int() takes it
    const long long x = n ? PyLong_AsLongLong(n) : -1;
    Py_XDECREF(n);
    return x;
  }();
  if (v == -1 && PyErr_Occurred()) throw Raised();
  return v;
}
int bounded(PyObject* o, const char* name, int64_t least, int64_t most) {
  const int64_t v = integer(o);
  need(v >= least && v <= most, name, std::to_string(least) + " .. " + std::to_string(most));
  return (int)v;
}
double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw Raised();
  return v;
}

// ---- checks
// Index of the CUDA device that all the tensors (undefined: none given) are on; the ops' last check.
int device_of(const Tensor& first, std::initializer_list<const Tensor*> others) {
  const at::Device device = first.device();
  if (!device.is_cuda()) throw Refused("vlcache_b200 ops run on CUDA tensors only (no CPU fallback)");
  for (const Tensor* t : others)
    if (t->defined() && t->device() != device)
      throw Refused("tensors on " + device.str() + " and " + t->device().str() + ": one call takes one device");
  return device.index();
}

// bf16 rows [sequences, tokens, heads, head_dim] (or [sequences, heads, head_dim]: one token) with contiguous heads,
// one sequence's tokens behind another's at one token stride.
struct Rows {
  int64_t seqs, tokens, heads, dim, stride;
};
Rows rows_of(const Tensor& t, const char* name) {
  const auto size = t.sizes(), stride = t.strides();
  const int n = (int)size.size();
  need(t.scalar_type() == at::kBFloat16 && (n == 3 || n == 4), name, "bf16 [sequences, tokens, heads, head_dim]");
  Rows r{size[0], n == 4 ? size[1] : 1, size[n - 2], size[n - 1], 0};
  need(stride[n - 1] == 1 && (r.heads <= 1 || stride[n - 2] == r.dim), name, "the heads of a token must be contiguous");
  const int64_t step = n == 4 ? stride[1] : stride[0];
  r.stride = r.tokens > 1 ? step : r.seqs > 1 ? stride[0] : r.heads * r.dim;
  need(r.tokens <= 1 || r.seqs <= 1 || stride[0] == r.tokens * step, name,
       "a sequence's tokens follow the one's before, at one token stride");
  return r;
}

const int32_t* ints_of(const Tensor& t, int64_t n, const char* name) {
  need(t.scalar_type() == at::kInt && t.is_contiguous() && t.numel() == n, name,
       "contiguous int32 [" + std::to_string(n) + "]");
  return (const int32_t*)t.data_ptr();
}

struct Tables {
  int32_t* data;
  int64_t stride;
  int width;
};
Tables tables_of(const Tensor& t, int64_t seqs) {
  need(t.scalar_type() == at::kInt && t.dim() == 2 && t.size(0) == seqs, "block_tables",
       "int32 [" + std::to_string(seqs) + ", width]");
  const int64_t width = t.size(1);
  need(width <= 1 || t.stride(1) == 1, "block_tables: rows must be contiguous");
  need(width <= 0x7fffffff, "block_tables: too wide");
  return Tables{(int32_t*)t.data_ptr(), seqs > 1 ? t.stride(0) : width, (int)width};
}

// The current stream of the device, made current for the call.
struct On {
  c10::cuda::OptionalCUDAGuard guard;
  void* stream;
  explicit On(int device) {
    if (device != c10::cuda::current_device()) guard.set_index(device);
    stream = c10::cuda::getCurrentCUDAStream(device).stream();
  }
};

void check(const char* function, int status) {
  if (status != VLC_OK) throw Failed{function, status};
}

at::TensorOptions like(const Tensor& t, at::ScalarType type) { return at::TensorOptions().dtype(type).device(t.device()); }

// A tensor of a part of a buffer, from byte `at` on (a multiple of the type's size): one allocation for several
// outputs, each some 1 us on the host.
Tensor part(const Tensor& buffer, int64_t at, at::ScalarType type, at::IntArrayRef sizes) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(buffer.storage()), buffer.key_set(),
                                                      c10::scalarTypeToTypeMeta(type));
  t.unsafeGetTensorImpl()->set_storage_offset(at / (int64_t)c10::elementSize(type));
  t.unsafeGetTensorImpl()->set_sizes_contiguous(sizes);
  return t;
}

// ---- the ops
PyObject* decode_attention_window(PyObject* const* a) {
  const Tensor &q = tensor(a[0], "q"), &k = tensor(a[1], "k_cache"), &v = tensor(a[2], "v_cache"),
               &tables = tensor(a[3], "block_tables"), &lens = tensor(a[4], "context_lens");
  Tensor out = optional(a[9], "out"), workspace = optional(a[10], "workspace");
  const Rows r = rows_of(q, "q");
  need(k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16 && k.dim() == 4 && k.sizes() == v.sizes() &&
           k.is_contiguous() && v.is_contiguous() && k.size(3) == r.dim,
       "k_cache / v_cache: contiguous bf16 [pages, block_size, num_kv_heads, head_dim]");
  const Tables t = tables_of(tables, r.seqs);
  const int32_t* const context_lens = ints_of(lens, r.seqs, "context_lens");
  const int max_len = bounded(a[5], "max_context_len", 0, 1 << 30);
  const float scale = (float)number(a[6]);
  const int window = bounded(a[7], "window", 0, 1 << 30), sinks = bounded(a[8], "sinks", 0, 1 << 30);
  for (const int64_t n : {r.seqs, r.tokens, r.heads, r.dim, k.size(1), k.size(2)})
    need(n <= 0x7fffffff, "sizes below 2^31");
  int64_t out_stride = r.heads * r.dim;
  if (out.defined()) {
    need(out.sizes() == q.sizes(), "out: q's shape");
    out_stride = rows_of(out, "out").stride;
  }
  need(!workspace.defined() || workspace.is_contiguous(), "workspace: contiguous");
  const On on(device_of(q, {&k, &v, &tables, &lens, &out, &workspace}));
  if (!out.defined()) out = at::empty(q.sizes(), like(q, at::kBFloat16));
  const int64_t bytes = vlc_decode_window_workspace_size((int)r.seqs, (int)r.tokens, (int)r.heads, (int)k.size(2), max_len,
                                                         window, sinks);
  if (bytes > 0 && (!workspace.defined() || (int64_t)workspace.nbytes() < bytes))
    workspace = at::empty({bytes}, like(q, at::kByte));
  check("vlc_decode_attn_window",
        vlc_decode_attn_window(q.data_ptr(), r.stride, (int)r.seqs, (int)r.tokens, (int)r.heads, k.data_ptr(),
                               v.data_ptr(), k.size(0), (int)k.size(1), (int)k.size(2), (int)r.dim, t.data, t.stride,
                               t.width, context_lens, max_len, window, sinks, scale, out.data_ptr(), out_stride,
                               workspace.defined() ? workspace.data_ptr() : nullptr,
                               workspace.defined() ? (int64_t)workspace.nbytes() : 0, on.stream));
  return THPVariable_Wrap(std::move(out));
}

// Tensors that are views of one buffer of ints, behind one another.
PyObject* tuple_of(std::initializer_list<Tensor> tensors) {
  PyObject* const out = PyTuple_New((Py_ssize_t)tensors.size());
  if (!out) throw Raised();
  Py_ssize_t i = 0;
  for (const Tensor& t : tensors) {
    PyObject* const o = THPVariable_Wrap(t);
    if (!o) {
      Py_DECREF(out);
      throw Raised();
    }
    PyTuple_SET_ITEM(out, i++, o);
  }
  return out;
}

PyObject* step_metadata(PyObject* const* a) {
  const Tensor &lens = tensor(a[0], "context_lens"), &fresh = tensor(a[1], "new_lens"),
               &tables = tensor(a[2], "block_tables"), &pages = tensor(a[3], "free_pages"),
               &count = tensor(a[4], "num_free");
  const int64_t b = lens.numel();
  need(b <= 65535, "at most 65535 sequences");
  const int32_t* const context_lens = ints_of(lens, b, "context_lens");
  const int32_t* const new_lens = ints_of(fresh, b, "new_lens");
  const Tables t = tables_of(tables, b);
  const int32_t* const free_pages = ints_of(pages, pages.numel(), "free_pages");
  const int32_t* const num_free = ints_of(count, 1, "num_free");
  need(pages.numel() <= 0x7fffffff, "free_pages: too many");
  const int block = bounded(a[5], "block_size", 1, 0x7fffffff), rows = bounded(a[6], "total_rows", 0, 1 << 30);
  const int window = bounded(a[7], "window", 0, 1 << 30), sinks = bounded(a[8], "sinks", 0, 1 << 30);
  const On on(device_of(lens, {&fresh, &tables, &pages, &count}));
  int64_t at = 0;
  const int64_t rows16 = (rows + 3) / 4 * 4;
  const Tensor buffer = at::empty({rows16 * 12 + (3 * b + 2) * 4}, like(lens, at::kByte));
  auto next = [&](at::ScalarType type, int64_t n, int64_t room) {
    const Tensor t = part(buffer, at, type, {n});
    at += room * (int64_t)c10::elementSize(type);
    return t;
  };
  const Tensor positions = next(at::kLong, rows, rows16), slots = next(at::kInt, rows, rows16);
  const Tensor cu_q = next(at::kInt, b + 1, b + 1), cu_k = next(at::kInt, b + 1, b + 1), after = next(at::kInt, b, b);
  check("vlc_step_metadata",
        vlc_step_metadata(context_lens, new_lens, (int)b, t.data, t.stride, t.width, block, window, sinks,
                          const_cast<int32_t*>(free_pages), (int)pages.numel(), const_cast<int32_t*>(num_free),
                          (int64_t*)positions.data_ptr(), (int32_t*)slots.data_ptr(), rows, (int32_t*)cu_q.data_ptr(),
                          (int32_t*)cu_k.data_ptr(), (int32_t*)after.data_ptr(), on.stream));
  return tuple_of({positions, slots, cu_q, cu_k, after});
}

struct Probs {
  int vocab, type;
  int64_t seq, row;  // strides
};
Probs probs_of(const Tensor& t, int64_t b, int64_t rows, const char* name) {
  const at::ScalarType type = t.scalar_type();
  const int kind = type == at::kFloat ? 0 : type == at::kBFloat16 ? 1 : type == at::kHalf ? 2 : -1;
  need(t.dim() == 3 && t.size(0) == b && t.size(1) == rows && kind >= 0, name,
       "fp32, bf16 or fp16 [" + std::to_string(b) + ", " + std::to_string(rows) + ", vocabulary]");
  need(t.size(2) > 0 && t.size(2) <= 1 << 18, name, "a vocabulary of 1 .. 2^18");
  need(t.size(2) == 1 || t.stride(2) == 1, name, "a row's values must be contiguous");
  return Probs{(int)t.size(2), kind, t.stride(0), t.stride(1)};
}

PyObject* verify_drafts(PyObject* const* a) {
  const Tensor &drafts = tensor(a[0], "drafts"), &target = tensor(a[1], "target_probs");
  const Tensor draft = optional(a[2], "draft_probs");
  const Tensor &u = tensor(a[3], "u"), &u_last = tensor(a[4], "u_last");
  const Tensor lens = optional(a[5], "context_lens"), tables = optional(a[6], "block_tables");
  need(drafts.scalar_type() == at::kLong && drafts.dim() == 2, "drafts: int64 [sequences, drafts]");
  const int64_t b = drafts.size(0), n = drafts.size(1);
  need(b <= 65535 && n <= 31, "at most 65535 sequences and 31 drafts");
  need(n <= 1 || drafts.stride(1) == 1, "drafts: a sequence's tokens must be contiguous");
  const Probs p = probs_of(target, b, n + 1, "target_probs");
  Probs q{};
  if (draft.defined()) {
    q = probs_of(draft, b, n, "draft_probs");
    need(q.vocab == p.vocab && q.type == p.type, "draft_probs: target_probs' vocabulary and type");
  }
  need(u.scalar_type() == at::kFloat && u.dim() == 2 && u.size(0) == b && u.size(1) == n && (n <= 1 || u.stride(1) == 1),
       "u", "fp32 [" + std::to_string(b) + ", " + std::to_string(n) + "]");
  need(u_last.scalar_type() == at::kFloat && u_last.dim() == 1 && u_last.size(0) == b && u_last.is_contiguous(), "u_last",
       "contiguous fp32 [" + std::to_string(b) + "]");
  const int32_t* const context_lens = lens.defined() ? ints_of(lens, b, "context_lens") : nullptr;
  Tables t{};
  int block = 0;
  need(tables.defined() || a[7] == Py_None, "block_size: with block_tables");
  if (tables.defined()) {
    need(lens.defined(), "block_tables: with context_lens");
    t = tables_of(tables, b);
    block = bounded(a[7], "block_size", 1, 0x7fffffff);
  }
  const On on(device_of(drafts, {&target, &draft, &u, &u_last, &lens, &tables}));
  const Tensor buffer = at::empty({b * ((n + 1) * 8 + 4)}, like(drafts, at::kByte));
  const Tensor tokens = part(buffer, 0, at::kLong, {b, n + 1}), emitted = part(buffer, b * (n + 1) * 8, at::kInt, {b});
  if (tables.defined())
    check("vlc_verify_stored_drafts",
          vlc_verify_stored_drafts((const int64_t*)drafts.data_ptr(), drafts.stride(0), (int)b, (int)n, target.data_ptr(),
                                   p.seq, p.row, draft.defined() ? draft.data_ptr() : nullptr, q.seq, q.row, p.vocab,
                                   p.type, (const float*)u.data_ptr(), u.stride(0), (const float*)u_last.data_ptr(),
                                   (int64_t*)tokens.data_ptr(), (int32_t*)emitted.data_ptr(),
                                   const_cast<int32_t*>(context_lens), t.data, t.stride, t.width, block, on.stream));
  else
    check("vlc_verify_drafts",
          vlc_verify_drafts((const int64_t*)drafts.data_ptr(), drafts.stride(0), (int)b, (int)n, target.data_ptr(), p.seq,
                            p.row, draft.defined() ? draft.data_ptr() : nullptr, q.seq, q.row, p.vocab, p.type,
                            (const float*)u.data_ptr(), u.stride(0), (const float*)u_last.data_ptr(),
                            (int64_t*)tokens.data_ptr(), (int32_t*)emitted.data_ptr(),
                            const_cast<int32_t*>(context_lens), on.stream));
  return tuple_of({tokens, emitted});
}

// ---- the module
// The exception class of that name, or null with an exception set.
PyObject* exception(const char* from, const char* name) {
  PyObject* const module = PyImport_ImportModule(from);
  PyObject* const type = module ? PyObject_GetAttrString(module, name) : nullptr;
  Py_XDECREF(module);
  return type;
}
void raise_failed(const Failed& f) {
  PyObject* const type = exception("vlcache_b200._lib", "VLCError");
  PyObject* const error = type ? PyObject_CallFunction(type, "si", f.function, f.status) : nullptr;
  if (error) PyErr_SetObject(type, error);
  Py_XDECREF(error);
  Py_XDECREF(type);
}
void raise_out_of_memory(const char* what) {
  PyObject* const type = exception("torch", "OutOfMemoryError");
  if (type) PyErr_SetString(type, what);
  Py_XDECREF(type);
}

template <PyObject* (*FUNCTION)(PyObject* const*), int ARGS>
PyObject* call(PyObject*, PyObject* const* args, Py_ssize_t n) {
  if (n != ARGS) {
    PyErr_Format(PyExc_TypeError, "%d arguments wanted, %zd given", ARGS, n);
    return nullptr;
  }
  try {
    return FUNCTION(args);
  } catch (const Refused& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const WrongType& e) {
    PyErr_SetString(PyExc_TypeError, e.what());
  } catch (const Failed& f) {
    raise_failed(f);
  } catch (const Raised&) {
  } catch (const c10::OutOfMemoryError& e) {
    raise_out_of_memory(e.what());
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  } catch (...) {
    PyErr_SetString(PyExc_RuntimeError, "unknown C++ exception");
  }
  return nullptr;
}

PyMethodDef kMethods[] = {
    {"decode_attention_window", (PyCFunction)(void (*)(void))call<decode_attention_window, 11>, METH_FASTCALL, nullptr},
    {"step_metadata", (PyCFunction)(void (*)(void))call<step_metadata, 9>, METH_FASTCALL, nullptr},
    {"verify_drafts", (PyCFunction)(void (*)(void))call<verify_drafts, 8>, METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_binding", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__binding(void) { return PyModule_Create(&kModule); }
