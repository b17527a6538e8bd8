// decode_binding.cpp -- Python calls of the decoding operators.
//
// A decoding step is a handful of launches of a few microseconds each, so the
// time of a call on the host is what a user waits for: a call of the public entry
// point takes 7.5 to 10 us (13.5 for an append and its read-back), where checks in
// Python and a call through ctypes took 15 to 30.  The module checks tensors, allocates the result, and calls the C entry points
// of libb200tx, whose addresses solution/_binding.py hands over (init).  It has
// no CUDA code of its own.
//
// Errors as in the wrappers of solution/kernels: RuntimeError where the
// inputs are not what the kernel runs on or the launch failed, ValueError
// where the call contradicts itself.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/ops/empty.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <cuda_runtime_api.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>

#include "b200tx.h"

namespace {

struct Entry {
  const char* (*last_error)();
  decltype(&b200tx_qk_norm_rope) qk_norm_rope;
  decltype(&b200tx_kv8_append) kv8_append;
  decltype(&b200tx_kv8_gather) kv8_gather;
  decltype(&b200tx_kv8_attention) kv8_attention;
  decltype(&b200tx_linear_w4) linear_w4;
  decltype(&b200tx_low_rank_add) low_rank_add;
  decltype(&b200tx_kv8_fork) kv8_fork;
  decltype(&b200tx_kv8_reserve) kv8_reserve;
  decltype(&b200tx_kv8_compact) kv8_compact;
  decltype(&b200tx_verify_draft) verify_draft;
} entry = {};

struct Refusal {
  PyObject* type;
  const char* text;
};

[[noreturn]] void ineligible(const char* text) { throw Refusal{PyExc_RuntimeError, text}; }

void require(bool ok, const char* text) {
  if (!ok) throw Refusal{PyExc_ValueError, text};
}

const at::Tensor* tensor(PyObject* o) { return THPVariable_Check(o) ? &THPVariable_Unpack(o) : nullptr; }

// An optional tensor argument: null for None, an error for anything else.
const at::Tensor* optional(PyObject* o, const char* text) {
  if (o == Py_None) return nullptr;
  const at::Tensor* t = tensor(o);
  require(t != nullptr, text);
  return t;
}

int64_t integer(PyObject* o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw python_error();
  return v;
}

double number(PyObject* o) {
  const double v = PyFloat_AsDouble(o);
  if (v == -1.0 && PyErr_Occurred()) throw python_error();
  return v;
}

template <typename T>
T* address(PyObject* o) {
  return o == Py_None ? nullptr : reinterpret_cast<T*>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(o)));
}

bool aligned(const at::Tensor& t) { return (reinterpret_cast<uintptr_t>(t.const_data_ptr()) & 15u) == 0; }

bool ready(const at::Tensor* t) { return t != nullptr && t->is_cuda() && !c10::GradMode::is_enabled(); }

bool packed_ok(const at::Tensor& t) {
  return t.dim() == 3 && (t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat) && t.numel() > 0 &&
         t.stride(2) == 1 && t.stride(0) % 8 == 0 && t.stride(1) % 8 == 0 && aligned(t);
}

int dtype(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? B200TX_F32 : B200TX_BF16; }

cudaStream_t stream_of(const at::Tensor& t) {
  if (t.get_device() != c10::cuda::current_device())
    ineligible("libb200tx launches on the current device: the operands are on another one (use torch.cuda.device(...))");
  return c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
}

void launched(int status, const char* what) {
  if (status == 0) return;
  PyErr_Format(PyExc_RuntimeError, "%s failed (status %d): %s", what, status, entry.last_error());
  throw python_error();
}

struct Span {
  uintptr_t begin, end;
};

// The addresses that a tensor lies within.
Span span(const at::Tensor& t) {
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  const uintptr_t begin = reinterpret_cast<uintptr_t>(t.const_data_ptr());
  return {begin, begin + static_cast<uintptr_t>(last + 1) * t.element_size()};
}

bool apart(const at::Tensor& a, const at::Tensor& b) {
  const Span x = span(a), y = span(b);
  return x.end <= y.begin || y.end <= x.begin;
}

// The rows of a packed tensor [B, T, W] in memory: `inner` rows at the smaller distance `near`,
// groups of them `far` apart.
struct Rows {
  int64_t inner, near, outer, far;
};

Rows rows(const at::Tensor& t) {
  const int64_t batch = t.size(0), tokens = t.size(1), b = t.stride(0), k = t.stride(1);
  return tokens > 1 && (batch == 1 || k <= b) ? Rows{tokens, k, batch, b} : Rows{batch, b, tokens, k};
}

// Whether no two rows share memory.
bool rows_once(const at::Tensor& t) {
  const Rows r = rows(t);
  const int64_t width = t.size(2), group = (r.inner > 1 ? (r.inner - 1) * r.near : 0) + width;
  return (r.inner == 1 || r.near >= width) && (r.outer == 1 || r.far >= group);
}

// Whether two packed tensors of one shape and type share no memory: they lie apart, or are columns
// of the same longer rows.
bool rows_apart(const at::Tensor& a, const at::Tensor& b) {
  if (apart(a, b)) return true;
  const Rows r = rows(a), other = rows(b);
  if (r.inner == 1 || r.inner != other.inner || r.near != other.near || r.near <= 0 ||
      (r.outer > 1 && (r.far != other.far || r.far % r.near != 0)))
    return false;
  const int64_t bytes = static_cast<int64_t>(reinterpret_cast<uintptr_t>(a.const_data_ptr()) -
                                             reinterpret_cast<uintptr_t>(b.const_data_ptr()));
  const int64_t row = r.near * a.element_size(), width = a.size(2) * a.element_size();
  const int64_t off = (bytes % row + row) % row;
  return off >= width && row - off >= width;
}

// `out` if the caller gave one (checked: it shares no memory with `like`, the input), else a new tensor.
at::Tensor result(PyObject* out, at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like, const char* text,
                  bool in_place = false) {
  if (out == Py_None) return at::empty(sizes, at::TensorOptions().dtype(type).device(like.device()));
  const at::Tensor* t = tensor(out);
  require(t != nullptr && t->sizes() == sizes && t->scalar_type() == type && t->device() == like.device() &&
              t->is_contiguous() && aligned(*t), text);
  require(apart(*t, like) || (in_place && t->const_data_ptr() == like.const_data_ptr() && like.is_contiguous()),
          "out shares memory with the input");
  return *t;
}

const float* norm_weight(PyObject* o, int64_t dim, const at::Tensor& like) {
  static const char* text = "the norm weights must be contiguous, 16-byte aligned float32 [head_dim] tensors on the input's device";
  const at::Tensor* w = optional(o, text);
  if (w == nullptr) return nullptr;
  require(w->scalar_type() == at::kFloat && w->dim() == 1 && w->size(0) == dim && w->is_contiguous() &&
              w->device() == like.device() && aligned(*w), text);
  return w->const_data_ptr<float>();
}

const int32_t* per_sequence(PyObject* o, int64_t batch, const at::Tensor& like, const char* text) {
  const at::Tensor* t = optional(o, text);
  if (t == nullptr) return nullptr;
  require(t->scalar_type() == at::kInt && t->dim() == 1 && t->size(0) == batch && t->is_contiguous() &&
              t->device() == like.device(), text);
  return t->const_data_ptr<int32_t>();
}

const char* const kSlots = "slots must be a contiguous int32 [B] tensor on the cache's device";
const char* const kCounts = "counts must be a contiguous int32 [B] tensor on the cache's device";
const char* const kBatch = "the batch is larger than the cache's slots";

// rope: (address of b200tx_rope, rotary, device index) or None
const b200tx_rope* rope_table(PyObject* o, int64_t dim, const at::Tensor& like) {
  if (o == Py_None) return nullptr;
  require(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 3, "rope must be a RotaryTable");
  const int64_t rotary = integer(PyTuple_GET_ITEM(o, 1));
  require(integer(PyTuple_GET_ITEM(o, 2)) == like.get_device(), "the rotation table must be on the input's device");
  require(rotary <= dim && rotary % (dim == 256 ? 16 : 8) == 0,
          "rotary must be a multiple of 8 (16 for head_dim 256) up to head_dim");
  return address<const b200tx_rope>(PyTuple_GET_ITEM(o, 0));
}

template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F f) {
  HANDLE_TH_ERRORS
  if (given != wanted) {
    PyErr_Format(PyExc_TypeError, "%zd arguments, %zd expected", given, wanted);
    return nullptr;
  }
  try {
    return f();
  } catch (const Refusal& r) {
    PyErr_SetString(r.type, r.text);
    return nullptr;
  }
  END_HANDLE_TH_ERRORS
}

// init({name: address}): the C entry points of the loaded libb200tx.
PyObject* init(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 1, [&]() -> PyObject* {
    auto take = [&](const char* name, auto& to) {
      PyObject* v = PyDict_GetItemString(args[0], name);
      require(v != nullptr, "an entry point is missing");
      to = reinterpret_cast<std::decay_t<decltype(to)>>(static_cast<uintptr_t>(PyLong_AsUnsignedLongLong(v)));
    };
    take("b200tx_last_error", entry.last_error);
    take("b200tx_qk_norm_rope", entry.qk_norm_rope);
    take("b200tx_kv8_append", entry.kv8_append);
    take("b200tx_kv8_gather", entry.kv8_gather);
    take("b200tx_kv8_attention", entry.kv8_attention);
    take("b200tx_linear_w4", entry.linear_w4);
    take("b200tx_low_rank_add", entry.low_rank_add);
    take("b200tx_kv8_fork", entry.kv8_fork);
    take("b200tx_kv8_reserve", entry.kv8_reserve);
    take("b200tx_kv8_compact", entry.kv8_compact);
    take("b200tx_verify_draft", entry.verify_draft);
    Py_RETURN_NONE;
  });
}

// qk_norm_rope_ok(qkv, heads, kv_heads)
int64_t rope_head_dim(PyObject* qkv, int64_t heads, int64_t kv_heads) {
  const at::Tensor* t = tensor(qkv);
  if (!ready(t) || !packed_ok(*t) || heads <= 0 || kv_heads <= 0 || kv_heads > heads) return 0;
  const int64_t total = heads + 2 * kv_heads, dim = t->size(2) / total;
  return t->size(2) % total == 0 && dim >= 8 && dim <= 256 && (dim & (dim - 1)) == 0 ? dim : 0;
}

PyObject* qk_norm_rope_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    return PyBool_FromLong(rope_head_dim(args[0], integer(args[1]), integer(args[2])) != 0);
  });
}

// qk_norm_rope(qkv, heads, kv_heads, q_weight, k_weight, eps, rope, positions, out) -> out
PyObject* qk_norm_rope(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const int64_t heads = integer(args[1]), kv_heads = integer(args[2]);
    const int64_t dim = rope_head_dim(args[0], heads, kv_heads);
    if (dim == 0) ineligible("sm100 qk norm + rotation is ineligible for the requested inputs");
    const at::Tensor& qkv = *tensor(args[0]);
    const float* qw = norm_weight(args[3], dim, qkv);
    const float* kw = norm_weight(args[4], dim, qkv);
    const b200tx_rope* rope = rope_table(args[6], dim, qkv);
    static const char* where = "positions must be an int32 or int64 [B, T] or [T] tensor on the input's device";
    const at::Tensor* pos = optional(args[7], where);
    if (pos != nullptr) {
      const bool flat = pos->dim() == 1;
      require((pos->scalar_type() == at::kInt || pos->scalar_type() == at::kLong) && pos->device() == qkv.device() &&
                  (flat || pos->dim() == 2) && pos->size(flat ? 0 : 1) == qkv.size(1) &&
                  (flat || pos->size(0) == qkv.size(0)) && (pos->stride(flat ? 0 : 1) == 1 || qkv.size(1) == 1), where);
    }
    at::Tensor out;
    if (args[8] == Py_None) {
      out = at::empty(qkv.sizes(), at::TensorOptions().dtype(qkv.scalar_type()).device(qkv.device()));
    } else {
      const at::Tensor* given = tensor(args[8]);
      require(given != nullptr && given->sizes() == qkv.sizes() && given->scalar_type() == qkv.scalar_type() &&
                  given->device() == qkv.device() && packed_ok(*given) &&
                  (given->const_data_ptr() != qkv.const_data_ptr() || given->strides() == qkv.strides()),
              "out must have qkv's shape, dtype and device, 16-byte aligned heads, and qkv's strides when it is qkv");
      out = *given;
      // in place every value is read and written by the same lane
      require(rows_once(out) && (out.const_data_ptr() == qkv.const_data_ptr() || rows_apart(out, qkv)),
              "out shares memory with qkv or with itself");
    }
    launched(entry.qk_norm_rope(qkv.const_data_ptr(), out.data_ptr(), dtype(qkv), qkv.size(0), qkv.size(1), heads, kv_heads,
                                dim, qkv.stride(0), qkv.stride(1), out.stride(0), out.stride(1), qw, kw,
                                static_cast<float>(number(args[5])), rope, pos == nullptr ? nullptr : pos->const_data_ptr(),
                                pos != nullptr && pos->scalar_type() == at::kLong,
                                pos != nullptr && pos->dim() == 2 ? pos->stride(0) : 0, stream_of(qkv)),
             "b200tx_qk_norm_rope");
    return THPVariable_Wrap(out);
  });
}

// A cache layer: (address of b200tx_kv8_cache, device index).
struct Layer {
  const b200tx_kv8_cache* view;
  int64_t device;
};

Layer layer_of(PyObject* o) {
  require(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2, "cache must be a Kv8Cache");
  return {address<const b200tx_kv8_cache>(PyTuple_GET_ITEM(o, 0)), integer(PyTuple_GET_ITEM(o, 1))};
}

bool append_fits(const Layer& c, const at::Tensor* qkv, int64_t heads) {
  return ready(qkv) && qkv->get_device() == c.device && packed_ok(*qkv) && heads >= c.view->kv_heads &&
         qkv->size(2) == (heads + 2 * c.view->kv_heads) * c.view->head_dim;
}

PyObject* kv8_append_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    return PyBool_FromLong(append_fits(layer_of(args[0]), tensor(args[1]), integer(args[2])));
  });
}

// kv8_append(layer, qkv, heads, q_weight, k_weight, eps, rope, slots, counts, out) -> q
PyObject* kv8_append(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 10, [&]() -> PyObject* {
    const Layer c = layer_of(args[0]);
    const int64_t heads = integer(args[2]);
    if (!append_fits(c, tensor(args[1]), heads)) ineligible("sm100 kv8 append is ineligible for the requested inputs");
    const at::Tensor& qkv = *tensor(args[1]);
    const int64_t dim = c.view->head_dim, batch = qkv.size(0);
    const float* qw = norm_weight(args[3], dim, qkv);
    const float* kw = norm_weight(args[4], dim, qkv);
    const b200tx_rope* rope = rope_table(args[6], dim, qkv);
    const int32_t* slots = per_sequence(args[7], batch, qkv, kSlots);
    const int32_t* counts = per_sequence(args[8], batch, qkv, kCounts);
    require(slots != nullptr || batch <= c.view->slots, kBatch);
    at::Tensor out = result(args[9], {batch, qkv.size(1), heads, dim}, at::kBFloat16, qkv,
                            "out must be a contiguous, 16-byte aligned bf16 [B, T, H, D] tensor");
    launched(entry.kv8_append(c.view, qkv.const_data_ptr(), dtype(qkv), out.data_ptr(), batch, qkv.size(1), heads,
                              qkv.stride(0), qkv.stride(1), slots, counts, qw, kw, static_cast<float>(number(args[5])), rope,
                              stream_of(qkv)),
             "b200tx_kv8_append");
    return THPVariable_Wrap(out);
  });
}

// kv8_gather(layer, codes, batch, most, tokens, slots, counts) -> (k, v)
PyObject* kv8_gather(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 7, [&]() -> PyObject* {
    const Layer c = layer_of(args[0]);
    const at::Tensor* codes = tensor(args[1]);
    if (!ready(codes)) ineligible("sm100 kv8 gather is ineligible for the requested inputs");
    const int64_t batch = integer(args[2]), most = integer(args[3]), tokens = integer(args[4]);
    require(batch > 0 && most > 0 && tokens >= 0, "max_tokens and the batch must be positive");
    const int32_t* slots = per_sequence(args[5], batch, *codes, kSlots);
    const int32_t* counts = per_sequence(args[6], batch, *codes, kCounts);
    require(slots != nullptr || batch <= c.view->slots, kBatch);
    const auto kind = at::TensorOptions().dtype(at::kBFloat16).device(codes->device());
    const int64_t shape[4] = {batch, most, c.view->kv_heads, c.view->head_dim};
    at::Tensor k = at::empty(shape, kind), v = at::empty(shape, kind);
    launched(entry.kv8_gather(c.view, k.data_ptr(), v.data_ptr(), batch, most, tokens, slots, counts, stream_of(*codes)),
             "b200tx_kv8_gather");
    PyObject* pk = THPVariable_Wrap(k);
    PyObject* pv = THPVariable_Wrap(v);
    PyObject* pair = PyTuple_Pack(2, pk, pv);
    Py_DECREF(pk);
    Py_DECREF(pv);
    return pair;
  });
}

bool attention_fits(const Layer& c, const at::Tensor* q) {
  return ready(q) && q->get_device() == c.device && q->scalar_type() == at::kBFloat16 && q->dim() == 4 && q->numel() > 0 &&
         q->size(3) == c.view->head_dim && q->size(2) % c.view->kv_heads == 0 && q->stride(3) == 1 &&
         q->stride(2) == c.view->head_dim && q->stride(1) % 8 == 0 && q->stride(0) % 8 == 0 && aligned(*q);
}

PyObject* kv8_attention_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 2, [&]() -> PyObject* { return PyBool_FromLong(attention_fits(layer_of(args[0]), tensor(args[1]))); });
}

// The id of the capture that the stream is in, 0 where it is in none.
unsigned long long capture_of(cudaStream_t stream) {
  cudaStreamCaptureStatus status = cudaStreamCaptureStatusNone;
  unsigned long long id = 0;
  const cudaError_t err = cudaStreamGetCaptureInfo_v2(stream, &status, &id, nullptr, nullptr, nullptr);
  if (err != cudaSuccess) {
    cudaGetLastError();  // it is told here; whoever asks next does not find it again
    ineligible("the stream's capture status cannot be read (another stream's capture, or an earlier CUDA error)");
  }
  return status == cudaStreamCaptureStatusNone ? 0 : id;
}

// A reference that is given up when it goes.
struct Owned {
  PyObject* o;
  explicit Owned(PyObject* p) : o(p) {
    if (o == nullptr) throw python_error();
  }
  Owned(const Owned&) = delete;
  ~Owned() { Py_DECREF(o); }
};

// kv8_attention(layer, q, scale or None, slots, counts, out, workspaces, make) -> context
// workspaces: {stream: uint8 tensor or None} of the calls outside of captures; make(stream) adds one
// and gives it, make(stream, capture) gives the one of the capture with that id.
PyObject* kv8_attention(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 8, [&]() -> PyObject* {
    const Layer c = layer_of(args[0]);
    if (!attention_fits(c, tensor(args[1]))) ineligible("sm100 kv8 attention is ineligible for the requested inputs");
    const at::Tensor& q = *tensor(args[1]);
    const int64_t batch = q.size(0), tokens = q.size(1), heads = q.size(2), dim = q.size(3);
    const double scale = args[2] == Py_None ? 1.0 / std::sqrt(static_cast<double>(dim)) : number(args[2]);
    require(scale > 0.0 && scale <= 1e30, "scale must be positive and finite");
    const int32_t* slots = per_sequence(args[3], batch, q, kSlots);
    const int32_t* counts = per_sequence(args[4], batch, q, kCounts);
    require(slots != nullptr || batch <= c.view->slots, kBatch);
    at::Tensor out = result(args[5], {batch, tokens, heads * dim}, at::kBFloat16, q,
                            "out must be a contiguous, 16-byte aligned bf16 [B, T, H * D] tensor", true);
    cudaStream_t stream = stream_of(q);
    const Owned key(PyLong_FromVoidPtr(stream));
    const unsigned long long capture = capture_of(stream);
    PyObject* held = capture == 0 ? PyDict_GetItemWithError(args[6], key.o) : nullptr;  // borrowed
    if (held == nullptr && PyErr_Occurred()) throw python_error();
    if (held != nullptr && held != Py_None) {
      Py_INCREF(held);
    } else if (capture == 0) {
      held = PyObject_CallOneArg(args[7], key.o);
    } else {
      const Owned id(PyLong_FromUnsignedLongLong(capture));
      held = PyObject_CallFunctionObjArgs(args[7], key.o, id.o, nullptr);
    }
    const Owned mine(held);
    const at::Tensor* given = tensor(mine.o);
    require(given != nullptr, "the workspace is not a tensor");
    const at::Tensor& work = *given;
    launched(entry.kv8_attention(c.view, q.const_data_ptr(), out.data_ptr(), batch, tokens, heads, q.stride(0), q.stride(1),
                                 slots, counts, static_cast<float>(scale), work.data_ptr(), work.numel(), stream),
             "b200tx_kv8_attention");
    return THPVariable_Wrap(out);
  });
}

bool linear_fits(const at::Tensor* x, const at::Tensor* packed, PyObject* bias, int64_t inner) {
  if (!ready(x) || packed == nullptr || x->scalar_type() != at::kBFloat16 || x->dim() < 1 || x->size(-1) != inner ||
      x->numel() == 0 || !x->is_contiguous() || !aligned(*x) || packed->device() != x->device())
    return false;
  if (bias == Py_None) return true;
  const at::Tensor* b = tensor(bias);
  return b != nullptr && b->scalar_type() == at::kFloat && b->dim() == 1 && b->size(0) == packed->size(0) &&
         b->is_contiguous() && b->device() == x->device();
}

PyObject* linear_w4_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    return PyBool_FromLong(linear_fits(tensor(args[0]), tensor(args[1]), args[2], integer(args[3])));
  });
}

// linear_w4(x, packed, scales, bias, inner, group, gelu, out_f32, out) -> out
PyObject* linear_w4(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const int64_t inner = integer(args[4]);
    if (!linear_fits(tensor(args[0]), tensor(args[1]), args[3], inner))
      ineligible("sm100 4-bit linear is ineligible for the requested operands");
    const at::Tensor& x = *tensor(args[0]);
    const at::Tensor& packed = *tensor(args[1]);
    const at::Tensor* scales = tensor(args[2]);
    require(scales != nullptr, "weight must be a W4Weight");
    const bool f32 = integer(args[7]) != 0;
    c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = packed.size(0);
    at::Tensor out = result(args[8], shape, f32 ? at::kFloat : at::kBFloat16, x,
                            "out has the wrong shape, dtype, device or layout");
    launched(entry.linear_w4(x.const_data_ptr(), inner, packed.const_data_ptr(), scales->const_data_ptr(),
                             args[3] == Py_None ? nullptr : tensor(args[3])->const_data_ptr<float>(), out.data_ptr(),
                             f32 ? B200TX_F32 : B200TX_BF16, x.numel() / inner, packed.size(0), inner, integer(args[5]),
                             integer(args[6]) != 0 ? B200TX_EPI_BIAS_GELU : B200TX_EPI_BIAS, stream_of(x)),
             "b200tx_linear_w4");
    return THPVariable_Wrap(out);
  });
}

bool low_rank_fits(const at::Tensor* x, const at::Tensor* base, const at::Tensor* down, const at::Tensor* up) {
  if (!ready(x) || base == nullptr || down == nullptr || up == nullptr || x->scalar_type() != at::kBFloat16 || x->dim() < 1 ||
      x->numel() == 0 || !x->is_contiguous() || !aligned(*x) || base->dim() != x->dim() || down->device() != x->device() ||
      base->device() != x->device() || !base->is_contiguous() || !aligned(*base) ||
      (base->scalar_type() != at::kBFloat16 && base->scalar_type() != at::kFloat))
    return false;
  const int64_t last = x->dim() - 1;
  return x->sizes().slice(0, last) == base->sizes().slice(0, last) && x->size(last) == down->size(2) &&
         base->size(last) == up->size(1);
}

PyObject* low_rank_add_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    return PyBool_FromLong(low_rank_fits(tensor(args[0]), tensor(args[1]), tensor(args[2]), tensor(args[3])));
  });
}

// low_rank_add(x, base, down, up, scales, indices, gelu, out_f32 or None, out) -> out
PyObject* low_rank_add(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 9, [&]() -> PyObject* {
    const at::Tensor *x = tensor(args[0]), *base = tensor(args[1]), *down = tensor(args[2]), *up = tensor(args[3]);
    if (!low_rank_fits(x, base, down, up)) ineligible("sm100 low-rank adapters are ineligible for the requested operands");
    const at::Tensor* scales = tensor(args[4]);
    require(scales != nullptr, "adapters must be a LowRankAdapters");
    const at::Tensor* indices = tensor(args[5]);
    const int64_t rows = x->numel() / x->size(-1);
    require(indices != nullptr && indices->scalar_type() == at::kInt && indices->is_contiguous() &&
                indices->device() == x->device() && indices->numel() > 0 && rows % indices->numel() == 0,
            "indices must be a contiguous int32 tensor on the input's device whose size divides the rows");
    const bool f32 = args[7] == Py_None ? base->scalar_type() == at::kFloat : integer(args[7]) != 0;
    const at::ScalarType type = f32 ? at::kFloat : at::kBFloat16;
    at::Tensor out = result(args[8], base->sizes(), type, *x, "out has the wrong shape, dtype, device or layout");
    require(args[8] == Py_None || apart(out, *base) || (out.const_data_ptr() == base->const_data_ptr() && type == base->scalar_type()),
            "out shares memory with base without being it");
    require(args[8] == Py_None || (apart(out, *down) && apart(out, *up) && apart(out, *scales) && apart(out, *indices)),
            "out shares memory with the adapters or indices");
    launched(entry.low_rank_add(x->const_data_ptr(), base->const_data_ptr(), dtype(*base), out.data_ptr(),
                                f32 ? B200TX_F32 : B200TX_BF16, down->const_data_ptr(), up->const_data_ptr(),
                                scales->const_data_ptr<float>(), indices->const_data_ptr<int32_t>(), indices->numel(), rows,
                                base->size(-1), x->size(-1), down->size(1), down->size(0),
                                integer(args[6]) != 0 ? B200TX_EPI_BIAS_GELU : B200TX_EPI_BIAS, stream_of(*x)),
             "b200tx_low_rank_add");
    return THPVariable_Wrap(out);
  });
}

// A pool of pages: (address of b200tx_kv8_pool, its refs).
struct Pool {
  const b200tx_kv8_pool* view;
  const at::Tensor* refs;
};

Pool pool_of(PyObject* o) {
  require(PyTuple_Check(o) && PyTuple_GET_SIZE(o) == 2, "pages must be a Kv8Pages");
  const Pool pool = {address<const b200tx_kv8_pool>(PyTuple_GET_ITEM(o, 0)), tensor(PyTuple_GET_ITEM(o, 1))};
  require(pool.refs != nullptr, "pages must be a Kv8Pages");
  if (!pool.refs->is_cuda()) ineligible("the pages of a cache are moved on an sm_100 CUDA device; there is no CPU fallback");
  return pool;
}

const int32_t* slot_list(PyObject* o, const at::Tensor& like, int64_t* size, const char* text) {
  const at::Tensor* t = tensor(o);
  require(t != nullptr && t->scalar_type() == at::kInt && t->dim() == 1 && t->is_contiguous() && t->device() == like.device(), text);
  *size = t->size(0);
  return t->const_data_ptr<int32_t>();
}

// kv8_fork(pool, source or None, target)
PyObject* kv8_fork(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 3, [&]() -> PyObject* {
    const Pool pool = pool_of(args[0]);
    int64_t pairs = 0, sources = 0;
    const int32_t* target = slot_list(args[2], *pool.refs, &pairs, "target must be a contiguous int32 [n] tensor on the cache's device");
    const int32_t* source = nullptr;
    if (args[1] != Py_None) {
      source = slot_list(args[1], *pool.refs, &sources, "source must be a contiguous int32 [n] tensor on the cache's device");
      require(sources == pairs, "source and target differ in size");
    }
    require(pairs <= 2048, "at most 2048 sequences at once");
    launched(entry.kv8_fork(pool.view, source, target, pairs, stream_of(*pool.refs)), "b200tx_kv8_fork");
    Py_RETURN_NONE;
  });
}

// kv8_reserve(pool, tokens, slots, counts) -> missing
PyObject* kv8_reserve(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 4, [&]() -> PyObject* {
    const Pool pool = pool_of(args[0]);
    const int64_t tokens = integer(args[1]);
    require(tokens >= 0, "tokens must not be negative");
    int64_t rows = pool.view->cache.slots;
    const int32_t* slots = nullptr;
    if (args[2] != Py_None) {
      slots = slot_list(args[2], *pool.refs, &rows, kSlots);
    } else if (args[3] != Py_None) {
      slot_list(args[3], *pool.refs, &rows, kCounts);
      require(rows <= pool.view->cache.slots, kBatch);
    }
    const int32_t* counts = per_sequence(args[3], rows, *pool.refs, kCounts);
    require(rows > 0 && rows <= 2048, "1 to 2048 sequences at once");
    at::Tensor missing = at::empty({rows}, at::TensorOptions().dtype(at::kInt).device(pool.refs->device()));
    launched(entry.kv8_reserve(pool.view, slots, counts, tokens, rows, missing.data_ptr<int32_t>(), stream_of(*pool.refs)),
             "b200tx_kv8_reserve");
    return THPVariable_Wrap(missing);
  });
}

// kv8_compact(pool) -> used
PyObject* kv8_compact(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 1, [&]() -> PyObject* {
    const Pool pool = pool_of(args[0]);
    at::Tensor used = at::empty({1}, at::TensorOptions().dtype(at::kInt).device(pool.refs->device()));
    launched(entry.kv8_compact(pool.view, used.data_ptr<int32_t>(), stream_of(*pool.refs)), "b200tx_kv8_compact");
    return THPVariable_Wrap(used);
  });
}

bool probabilities_fit(const at::Tensor* t, int64_t batch, int64_t tokens) {
  return t != nullptr && t->dim() == 3 && t->size(0) == batch && t->size(1) == tokens && t->size(2) > 0 &&
         (t->stride(2) == 1 || t->size(2) == 1) && (t->scalar_type() == at::kFloat || t->scalar_type() == at::kBFloat16);
}

bool verify_fits(const at::Tensor* target, const at::Tensor* drafted) {
  return target != nullptr && drafted != nullptr && target->is_cuda() && drafted->device() == target->device() &&
         drafted->dim() == 2 && drafted->size(0) > 0 && drafted->size(1) <= 1024 && drafted->is_contiguous() &&
         (drafted->scalar_type() == at::kInt || drafted->scalar_type() == at::kLong) &&
         probabilities_fit(target, drafted->size(0), drafted->size(1) + 1);
}

PyObject* verify_draft_ok(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 2, [&]() -> PyObject* { return PyBool_FromLong(verify_fits(tensor(args[0]), tensor(args[1]))); });
}

// verify_draft(target, drafted, uniform, draft, counts) -> (tokens, accepted)
PyObject* verify_draft(PyObject*, PyObject* const* args, Py_ssize_t n) {
  return guarded(n, 5, [&]() -> PyObject* {
    const at::Tensor *target = tensor(args[0]), *drafted = tensor(args[1]), *uniform = tensor(args[2]);
    if (!verify_fits(target, drafted)) ineligible("sm100 draft verification is ineligible for the requested inputs");
    const int64_t batch = drafted->size(0), tokens = drafted->size(1);
    require(uniform != nullptr && uniform->scalar_type() == at::kFloat && uniform->is_contiguous() && uniform->dim() == 2 &&
                uniform->size(0) == batch && uniform->size(1) == tokens + 1 && uniform->device() == target->device(),
            "uniform must be a contiguous float32 [B, T + 1] tensor on the input's device");
    static const char* text = "draft must be a [B, T, V] tensor of the target's dtype, device and vocabulary";
    const at::Tensor* draft = optional(args[3], text);
    require(draft == nullptr || (probabilities_fit(draft, batch, tokens) && draft->size(2) == target->size(2) &&
                                 draft->scalar_type() == target->scalar_type() && draft->device() == target->device()), text);
    const int32_t* counts =
        per_sequence(args[4], batch, *target, "counts must be a contiguous int32 [B] tensor on the input's device");
    at::Tensor out = at::empty({batch, tokens + 1}, drafted->options());
    at::Tensor accepted = at::empty({batch}, at::TensorOptions().dtype(at::kInt).device(target->device()));
    const bool given = draft != nullptr && tokens > 0;
    launched(entry.verify_draft(target->const_data_ptr(), target->stride(0), target->stride(1),
                                given ? draft->const_data_ptr() : nullptr, given ? draft->stride(0) : 0,
                                given ? draft->stride(1) : 0, dtype(*target), drafted->const_data_ptr(),
                                drafted->scalar_type() == at::kLong, uniform->const_data_ptr<float>(), counts, batch, tokens,
                                target->size(2), out.data_ptr(), accepted.data_ptr<int32_t>(), stream_of(*target)),
             "b200tx_verify_draft");
    const Owned first(THPVariable_Wrap(out)), second(THPVariable_Wrap(accepted));
    return PyTuple_Pack(2, first.o, second.o);
  });
}

#define B200TX_METHOD(name) \
  {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}

PyMethodDef methods[] = {
    B200TX_METHOD(init),
    B200TX_METHOD(qk_norm_rope_ok),
    B200TX_METHOD(qk_norm_rope),
    B200TX_METHOD(kv8_append_ok),
    B200TX_METHOD(kv8_append),
    B200TX_METHOD(kv8_gather),
    B200TX_METHOD(kv8_attention_ok),
    B200TX_METHOD(kv8_attention),
    B200TX_METHOD(linear_w4_ok),
    B200TX_METHOD(linear_w4),
    B200TX_METHOD(low_rank_add_ok),
    B200TX_METHOD(low_rank_add),
    B200TX_METHOD(kv8_fork),
    B200TX_METHOD(kv8_reserve),
    B200TX_METHOD(kv8_compact),
    B200TX_METHOD(verify_draft_ok),
    B200TX_METHOD(verify_draft),
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_decode_binding", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__decode_binding(void) { return PyModule_Create(&module); }
