// The host side of the paged step operators as a CPython extension module (deltakv_b200._step):
// argument checks, output allocation, the descriptors of include/dkv_b200.h and the call of the C
// entry, on the current stream of the tensors' device.
//
// Why it is not ctypes like the package's other entry points: a decode step calls these operators
// once a layer and their kernels take 3 to 10 us, so an eager step is bound by the host.  Reading
// shapes, strides, types and pointers of a handful of tensors through Python and filling a ctypes
// struct took 9 to 11 us a call (and the launch itself 2.5 to 4); here it takes about 2.
//
// The C entries are reached by the addresses that the Python side passes to bind(), so this module
// links against torch alone and the library has one loader (_lib.lib()).
#include <Python.h>

#include <ATen/ATen.h>
#include <ATen/MemoryOverlap.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <string>
#include <vector>

#include "../../include/dkv_b200.h"

namespace {

using at::Tensor;

int (*g_plan)(const dkv_step_plan_args *, dkv_stream_t);
int (*g_append)(const dkv_append_args *, const dkv_rotary *, dkv_stream_t);
int (*g_workspace)(const dkv_paged_decode_args *, int64_t *);
int (*g_attend)(const dkv_paged_decode_args *, dkv_stream_t);
// 8-bit pages
int (*g_append_quant)(const dkv_append_args *, const dkv_rotary *, const dkv_page_scales *, const dkv_page_scales *,
                      dkv_stream_t);
int (*g_scatter_quant)(const void *, int32_t, int64_t, int64_t, int64_t, const dkv_paged_cache *, const dkv_page_scales *,
                       const dkv_seq_batch *, int32_t *, dkv_stream_t);
int (*g_gather_quant)(const dkv_paged_cache *, const dkv_page_scales *, const dkv_seq_batch *, void *, int32_t, int64_t, int64_t,
                      int64_t, int32_t, int32_t *, dkv_stream_t);
int (*g_workspace_quant)(const dkv_paged_decode_args *, int32_t, int64_t *);
int (*g_attend_quant)(const dkv_paged_decode_args *, int32_t, const dkv_page_scales *, const dkv_page_scales *, dkv_stream_t);
int (*g_append_check)(const dkv_append_args *, dkv_stream_t);
int (*g_scatter_check)(int64_t, const dkv_paged_cache *, const dkv_seq_batch *, int32_t *, dkv_stream_t);
PyObject *g_raise;        // raises the package's error for a status code
PyObject *g_status_word;  // device index -> address of its status word
constexpr int kMaxDevices = 64;
int32_t *g_status[kMaxDevices];

// A Python exception on its way out.
struct Raised {
  PyObject *type;  // null: already set
  std::string text;
};
[[noreturn]] void value_error(const std::string &text) { throw Raised{PyExc_ValueError, text}; }
[[noreturn]] void type_error(const std::string &text) { throw Raised{PyExc_TypeError, text}; }

template <typename F>
PyObject *guarded(F f) {
  try {
    return f();
  } catch (const Raised &r) {
    if (r.type != nullptr) PyErr_SetString(r.type, r.text.c_str());
  } catch (const c10::OutOfMemoryError &e) {  // what torch itself raises for it
    PyObject *torch = PyImport_ImportModule("torch");
    PyObject *type = torch ? PyObject_GetAttrString(torch, "OutOfMemoryError") : nullptr;
    if (type != nullptr) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
    Py_XDECREF(torch);
  } catch (const c10::Error &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
  } catch (const std::exception &e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

// ---- arguments --------------------------------------------------------------------------
const Tensor &tensor(PyObject *o, const char *name) {
  if (!THPVariable_Check(o)) type_error(std::string(name) + " must be a tensor");
  return THPVariable_Unpack(o);
}
const Tensor *maybe(PyObject *o, const char *name) { return o == Py_None ? nullptr : &tensor(o, name); }
int64_t integer(PyObject *o) {
  const long long v = PyLong_AsLongLong(o);
  if (v == -1 && PyErr_Occurred()) throw Raised{nullptr, ""};
  return v;
}
const char *dtype_name(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return "torch.float32";
    case at::kHalf: return "torch.float16";
    case at::kBFloat16: return "torch.bfloat16";
    default: return c10::toString(t);
  }
}
int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return DKV_F32;
    case at::kHalf: return DKV_F16;
    case at::kBFloat16: return DKV_BF16;
    default: type_error(std::string("dtype ") + dtype_name(t) + " is not supported by the B200 kernels");
  }
}
bool is_code(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kChar; }
int code_of(at::ScalarType t) { return t == at::kFloat8_e4m3fn ? DKV_E4M3 : DKV_I8; }
std::string shape_text(const Tensor &t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + (t.dim() == 1 ? ",)" : ")");
}
// a new tensor straight from the device's allocator (the dispatcher's way to it costs as much again)
Tensor fresh_tensor(at::IntArrayRef sizes, at::ScalarType type, c10::Device device) {
  return Tensor(at::detail::empty_cuda(sizes, type, device, std::nullopt));
}
// [rows, heads, head_dim] like t, in t's order of rows and heads; head_dim stays contiguous, which empty_like
// does not promise where t's rows or heads lie over each other (broadcast, sliding windows)
Tensor fresh_like(const Tensor &t) {
  if (!t.is_contiguous()) {
    Tensor like = at::empty_like(t);
    if (like.stride(2) == 1 || like.size(2) == 1) return like;
  }
  return fresh_tensor(t.sizes(), t.scalar_type(), t.device());
}
void *ptr(const Tensor *t) { return t == nullptr ? nullptr : t->data_ptr(); }

// The device that all tensors must share, and its current stream.
struct Place {
  const char *where;
  c10::Device device;
  Place(const char *where_, const Tensor &first) : where(where_), device(first.device()) {
    if (!device.is_cuda()) value_error("deltakv_b200 kernels need CUDA tensors (there is no CPU path)");
  }
  void also(const Tensor *t) const {
    if (t == nullptr || t->device() == device) return;
    if (!t->is_cuda()) value_error("deltakv_b200 kernels need CUDA tensors (there is no CPU path)");
    value_error(std::string(where) + ": tensors on " + device.str() + " and " + t->device().str());
  }
  dkv_stream_t stream() const {
    return reinterpret_cast<dkv_stream_t>(c10::cuda::getCurrentCUDAStream(device.index()).stream());
  }
  int32_t *status() const {
    const int i = device.index();
    if (i >= 0 && i < kMaxDevices && g_status[i] != nullptr) return g_status[i];
    PyObject *r = PyObject_CallFunction(g_status_word, "i", i);
    if (r == nullptr) throw Raised{nullptr, ""};
    int32_t *p = static_cast<int32_t *>(PyLong_AsVoidPtr(r));
    Py_DECREF(r);
    if (p == nullptr) throw Raised{nullptr, ""};
    if (i >= 0 && i < kMaxDevices) g_status[i] = p;
    return p;
  }
};

void check(int rc, const char *entry) {
  if (rc == DKV_OK) return;
  PyObject *r = PyObject_CallFunction(g_raise, "is", rc, entry);
  Py_XDECREF(r);
  throw Raised{nullptr, ""};  // the call above raised
}

// Launches a look at a call's blocks, waits for what it records and raises it: f(status word) is the launch.
template <typename F>
void refuse(const Place &place, const char *look, F f) {
  Tensor word = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(place.device));
  check(f(word.data_ptr<int32_t>()), look);
  check(word.item<int32_t>(), place.where);
}

void int32_vector(const Tensor &t, const char *name, int64_t n) {  // n < 0: any length
  if (t.scalar_type() != at::kInt) type_error(std::string(name) + " must be int32");
  if (t.dim() != 1 || !t.is_contiguous() || (n >= 0 && t.numel() != n))
    value_error(std::string(name) + " must be a contiguous vector" + (n >= 0 ? " of " + std::to_string(n) : ""));
}

// [rows, heads, hd] with contiguous head_dim; heads < 0: any
void rows_of(const Tensor &t, const char *name, int64_t rows, int64_t heads, int64_t hd) {
  if (t.dim() != 3 || t.size(0) != rows || t.size(2) != hd || (heads >= 0 && t.size(1) != heads))
    value_error(std::string(name) + " " + shape_text(t) + " must be [" + std::to_string(rows) + ", " +
                (heads < 0 ? std::string("heads") : std::to_string(heads)) + ", " + std::to_string(hd) + "]");
  if (t.stride(2) != 1 && hd > 1) value_error(std::string(name) + " must have contiguous head_dim");
}

// A tensor that is written: no element of it may lie over another one of its own, and it may be the input
// but not lie across it (as far as the strides tell).
void written(const Tensor &t, const char *name, const Tensor *input, const char *input_name) {
  if (at::has_internal_overlap(t) == at::MemOverlap::Yes) value_error(std::string(name) + " has elements that share memory");
  if (input != nullptr && at::get_overlap_status(t, *input) == at::MemOverlapStatus::Partial)
    value_error(std::string(name) + " overlaps " + input_name + " without being it");
}

// a tensor that is written and another that must not lie over it (as far as the strides tell)
void apart(const Tensor &t, const char *name, const Tensor &other, const char *other_name) {
  const at::MemOverlapStatus s = at::get_overlap_status(t, other);
  if (s == at::MemOverlapStatus::Full || s == at::MemOverlapStatus::Partial)
    value_error(std::string(name) + " and " + other_name + " share memory");
}

dkv_paged_cache describe(const Tensor &t, int code) {
  dkv_paged_cache c;
  c.base = t.data_ptr();
  c.dtype = code;
  c.block_size = static_cast<int32_t>(t.size(1));
  c.n_heads = static_cast<int32_t>(t.size(2));
  c.head_dim = static_cast<int32_t>(t.size(3));
  c.num_blocks = t.size(0);
  c.stride_block = t.stride(0), c.stride_slot = t.stride(1), c.stride_head = t.stride(2);
  return c;
}
// checks the K and V pages, and describes them once they are known to be on the GPU; 8 bits: where scales come with them
struct Pages {
  const Tensor &k, &v;
  int code;
  int64_t heads, hd;
  Pages(const Tensor &k_, const Tensor &v_, bool scaled = false) : k(k_), v(v_) {
    if (k.dim() != 4 || v.dim() != 4)
      value_error("unsupported paged KV layout " + shape_text(k) + ", " + shape_text(v));
    if (k.scalar_type() != v.scalar_type() || k.size(1) != v.size(1) || k.size(2) != v.size(2) || k.size(3) != v.size(3))
      value_error("k_pages and v_pages must share dtype, block size, heads and head_dim");
    if (is_code(k.scalar_type()) && !scaled) type_error(std::string(dtype_name(k.scalar_type())) + " pages need kv_scales");
    if (scaled && !is_code(k.scalar_type()))
      type_error(std::string("kv_scales go with 8-bit pages (float8_e4m3fn or int8), not ") + dtype_name(k.scalar_type()));
    code = scaled ? code_of(k.scalar_type()) : dtype_code(k.scalar_type());
    heads = k.size(2), hd = k.size(3);
    if ((k.stride(3) != 1 || v.stride(3) != 1) && hd > 1) value_error("paged cache head_dim must be contiguous");
    if (k.size(1) > INT32_MAX || heads > INT32_MAX || hd > INT32_MAX) value_error("paged cache too large");
  }
};

// The scales of 8-bit pages: fp32 [num_blocks, heads], any strides.
void scales_of(const Tensor &t, const char *name, const Tensor &pages) {
  if (t.scalar_type() != at::kFloat) type_error(std::string(name) + " must be float32");
  if (t.dim() != 2 || t.size(0) != pages.size(0) || t.size(1) != pages.size(2))
    value_error(std::string(name) + " " + shape_text(t) + " must be [num_blocks, heads] = [" + std::to_string(pages.size(0)) +
                ", " + std::to_string(pages.size(2)) + "]");
}
dkv_page_scales describe_scales(const Tensor &t) { return {t.data_ptr<float>(), t.stride(0), t.stride(1)}; }

// kv_scales: None or a (K, V) pair of tensors
struct PairOfScales {
  const Tensor *k = nullptr, *v = nullptr;
  explicit PairOfScales(PyObject *o) {
    if (o == Py_None) return;
    if (!PyTuple_Check(o) || PyTuple_GET_SIZE(o) != 2) type_error("kv_scales must be a (k_scales, v_scales) tuple");
    k = &tensor(PyTuple_GET_ITEM(o, 0), "k_scales"), v = &tensor(PyTuple_GET_ITEM(o, 1), "v_scales");
  }
  explicit operator bool() const { return k != nullptr; }
  void check(const Pages &pages) const {
    if (k == nullptr) return;
    scales_of(*k, "k_scales", pages.k), scales_of(*v, "v_scales", pages.v);
  }
};

// a batch of sequences, as SeqBatchTensors holds it
struct Sequences {
  const Tensor &cu, &tables;
  const Tensor *lens;
  int64_t n, max_seq_len;
  Sequences(PyObject *cu_, PyObject *tables_, PyObject *lens_, PyObject *longest)
      : cu(tensor(cu_, "cu_seqlens")), tables(tensor(tables_, "block_tables")), lens(maybe(lens_, "table_lens")),
        n(cu.numel() - 1), max_seq_len(integer(longest)) {}
  void check_shapes() const {
    if (tables.dim() == 2 && tables.size(0) < n)
      value_error("block_tables has " + std::to_string(tables.size(0)) + " rows for " + std::to_string(n) +
                  " sequences");
    // without table_lens a row has as many entries as lie between two rows (SeqBatchTensors lays its tables out so)
    if (!lens && tables.dim() == 2 && tables.numel() > 0 && tables.stride(0) != tables.size(1))
      value_error("block_tables without table_lens must have rows that follow one another");
    if (lens && (lens->numel() < n || !lens->is_contiguous()))
      value_error("table_lens must be a contiguous vector of " + std::to_string(n));
    if (n < 0 || !cu.is_contiguous()) value_error("cu_seqlens must be a contiguous vector");
    if (max_seq_len < 0 || max_seq_len > INT32_MAX) value_error("max_seq_len must be in [0, 2**31)");
  }
  void check_types() const {
    if (cu.scalar_type() != at::kInt || tables.scalar_type() != at::kInt || (lens && lens->scalar_type() != at::kInt))
      type_error("sequence metadata must be int32");
    if (tables.dim() != 2 || (tables.stride(1) != 1 && tables.size(1) > 1))
      value_error("block_tables must be a row-major [n_seqs, max_blocks] int32 tensor");
  }
  dkv_seq_batch describe() const {
    dkv_seq_batch q;
    q.cu_seqlens = cu.data_ptr<int32_t>();
    q.block_tables = tables.data_ptr<int32_t>();
    q.table_lens = static_cast<int32_t *>(ptr(lens));
    q.positions = nullptr;
    q.table_stride = tables.stride(0);
    q.n_seqs = static_cast<int32_t>(n);
    q.max_seq_len = static_cast<int32_t>(max_seq_len);
    return q;
  }
};

// n elements of a vector as a tensor of their own on its storage (integers: nothing for autograd to know),
// without a dispatched call for each
Tensor vector_in(const Tensor &whole, int64_t offset, int64_t n) {
  Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::TensorImpl::VIEW, c10::Storage(whole.storage()),
                                                      whole.key_set(), whole.dtype());
  t.unsafeGetTensorImpl()->set_storage_offset(whole.storage_offset() + offset);
  t.unsafeGetTensorImpl()->set_sizes_contiguous(at::IntArrayRef(&n, 1));
  return t;
}

// ---- operators --------------------------------------------------------------------------
// plan(lengths, block_tables, block_size, rows, max_seq_len, new_lengths, table_lens, free_blocks)
//   -> (cu_seqlens, cu_new, table_lens, blocks_used, positions, slots)
PyObject *plan(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    if (count != 8) type_error("plan takes 8 arguments");
    const Tensor &lengths = tensor(a[0], "lengths"), &tables = tensor(a[1], "block_tables");
    const int64_t block_size = integer(a[2]), rows = integer(a[3]), max_seq_len = integer(a[4]);
    const Tensor *fresh = maybe(a[5], "new_lengths"), *held = maybe(a[6], "table_lens"),
                 *free_blocks = maybe(a[7], "free_blocks");
    const int64_t n = lengths.numel();
    int32_vector(lengths, "lengths", n);
    if (fresh) int32_vector(*fresh, "new_lengths", n);
    if (held) int32_vector(*held, "table_lens", n);
    if (free_blocks) int32_vector(*free_blocks, "free_blocks", -1);
    if (tables.scalar_type() != at::kInt) type_error("block_tables must be int32");
    if (tables.dim() != 2 || tables.size(0) != n || (tables.stride(1) != 1 && tables.size(1) > 1))
      value_error("block_tables must be a row-major [n_seqs, max_blocks] int32 tensor");
    const int64_t width = tables.size(1);
    if (n > 1 && tables.stride(0) < width) value_error("block_tables rows overlap: the plan writes them");
    if (block_size <= 0 || block_size > INT32_MAX || rows < 0 || rows > INT32_MAX || max_seq_len < 0 ||
        max_seq_len > INT32_MAX || width > INT32_MAX || n > INT32_MAX)
      value_error("block_size must be positive, rows and max_seq_len not negative, all below 2**31");
    apart(tables, "block_tables", lengths, "lengths");
    if (fresh) apart(tables, "block_tables", *fresh, "new_lengths");
    if (held) apart(tables, "block_tables", *held, "table_lens");
    if (free_blocks) apart(tables, "block_tables", *free_blocks, "free_blocks");
    const Place at_("plan_paged_step", lengths);
    at_.also(&tables), at_.also(fresh), at_.also(held), at_.also(free_blocks);
    const c10::DeviceGuard guard(at_.device);
    Tensor out = fresh_tensor({3 * n + 3 + rows}, at::kInt, at_.device);
    Tensor slots = fresh_tensor({rows}, at::kLong, at_.device);
    dkv_step_plan_args p;
    p.lengths = lengths.data_ptr<int32_t>();
    p.new_lengths = static_cast<int32_t *>(ptr(fresh));
    p.table_lens = static_cast<int32_t *>(ptr(held));
    p.free_blocks = static_cast<int32_t *>(ptr(free_blocks));
    p.n_free = free_blocks ? free_blocks->numel() : 0;
    p.block_tables = tables.data_ptr<int32_t>();
    p.table_stride = tables.stride(0);
    p.table_width = static_cast<int32_t>(width);
    p.n_seqs = static_cast<int32_t>(n);
    p.block_size = static_cast<int32_t>(block_size);
    p.n_rows = static_cast<int32_t>(rows);
    int32_t *base = out.data_ptr<int32_t>();
    p.cu_seqlens = base;
    p.cu_new = base + n + 1;
    p.table_lens_out = base + 2 * (n + 1);
    p.blocks_used = base + 3 * n + 2;
    p.positions = base + 3 * n + 3;
    p.slots = slots.data_ptr<int64_t>();
    p.status = at_.status();
    check(g_plan(&p, at_.stream()), "dkv_plan_paged_step");
    const int64_t sizes[5] = {n + 1, n + 1, n, 1, rows};
    PyObject *result = PyTuple_New(6);
    if (result == nullptr) throw Raised{nullptr, ""};
    for (int64_t i = 0, offset = 0; i < 5; offset += sizes[i++])
      PyTuple_SET_ITEM(result, i, THPVariable_Wrap(vector_in(out, offset, sizes[i])));
    PyTuple_SET_ITEM(result, 5, THPVariable_Wrap(slots));
    return result;
  });
}

// rope_ready(cos, sin, like): both fp32 and contiguous on like's device
PyObject *rope_ready(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    if (count != 3) type_error("rope_ready takes 3 arguments");
    const Tensor &c = tensor(a[0], "rope cos"), &s = tensor(a[1], "rope sin"), &like = tensor(a[2], "k");
    const bool ready = c.scalar_type() == at::kFloat && s.scalar_type() == at::kFloat && c.device() == like.device() &&
                       s.device() == like.device() && c.is_contiguous() && s.is_contiguous();
    return PyBool_FromLong(ready);
  });
}

// append(k, v, k_pages, v_pages, slots, q, positions, cos, sin, q_out, rotary_dim, interleaved, kv_scales, look)
//   -> q_out or None; rotary_dim None: the whole head; look: whether 8-bit pages' rows follow one another is seen first
PyObject *append(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    if (count != 14) type_error("append takes 14 arguments");
    const Tensor &k = tensor(a[0], "k"), &v = tensor(a[1], "v");
    const PairOfScales scales(a[12]);
    const Pages pages(tensor(a[2], "k_pages"), tensor(a[3], "v_pages"), static_cast<bool>(scales));
    const Tensor &slots = tensor(a[4], "slots");
    const Tensor *q = maybe(a[5], "q"), *positions = maybe(a[6], "positions"), *cos = maybe(a[7], "rope cos"),
                 *sin = maybe(a[8], "rope sin"), *q_out = maybe(a[9], "q_out");
    const int64_t rows = slots.numel(), rotary_dim = a[10] == Py_None ? pages.hd : integer(a[10]);
    const int crossed = PyObject_IsTrue(a[11]), look = PyObject_IsTrue(a[13]);
    if (crossed < 0 || look < 0) throw Raised{nullptr, ""};
    if ((a[10] != Py_None || crossed) && !cos) value_error("rotary_dim and interleaved say how rope turns: pass rope with them");
    if (slots.scalar_type() != at::kLong) type_error("slots must be int64");
    if (slots.dim() != 1 || !slots.is_contiguous()) value_error("slots must be a contiguous vector");
    written(pages.k, "k_pages", nullptr, ""), written(pages.v, "v_pages", nullptr, "");
    apart(pages.k, "k_pages", pages.v, "v_pages");
    if (scales) {
      scales.check(pages);
      written(*scales.k, "k_scales", nullptr, ""), written(*scales.v, "v_scales", nullptr, "");
      apart(*scales.k, "k_scales", *scales.v, "v_scales");
      if (pages.k.size(1) > 1024) value_error("8-bit pages have at most 1024 slots a block");
      dtype_code(k.scalar_type());  // any that the kernels read
    }
    rows_of(k, "k", rows, pages.heads, pages.hd);
    rows_of(v, "v", rows, pages.heads, pages.hd);
    if (v.scalar_type() != k.scalar_type() || (q && q->scalar_type() != k.scalar_type()))
      type_error("q, k and v must share a dtype");
    if (!scales && k.scalar_type() != pages.k.scalar_type() && k.scalar_type() != at::kFloat)
      type_error(std::string(dtype_name(k.scalar_type())) + " rows do not go into " +
                 dtype_name(pages.k.scalar_type()) + " pages (pass the pages' dtype or fp32)");
    if (cos) {
      if (!positions) value_error("rope needs positions");
      if (cos->dim() == 2 && cos->size(0) == 0) value_error("rope tables without positions");
      if (a[10] != Py_None && (rotary_dim <= 0 || rotary_dim > pages.hd || rotary_dim % 2))
        value_error("rotary_dim " + std::to_string(rotary_dim) + " must be even and in (0, head_dim]");
      int32_vector(*positions, "positions", rows);
    }
    if (!q && q_out) value_error("q_out without q");
    if (q) {
      if (!cos) value_error("q is only rotated: pass rope and positions with it");
      rows_of(*q, "q", rows, -1, pages.hd);
      if (q->size(1) > INT32_MAX) value_error("too many query heads");
      if (q_out) {
        rows_of(*q_out, "q_out", rows, q->size(1), pages.hd);
        if (q_out->scalar_type() != q->scalar_type()) type_error("q_out must have q's dtype");
        written(*q_out, "q_out", q, "q");
        apart(*q_out, "q_out", k, "k"), apart(*q_out, "q_out", v, "v");
      }
    }
    const Place at_("append_into_paged", k);
    at_.also(&v), at_.also(&pages.k), at_.also(&pages.v), at_.also(&slots), at_.also(q), at_.also(positions);
    at_.also(q_out), at_.also(cos), at_.also(sin), at_.also(scales.k), at_.also(scales.v);
    if (cos) {
      if (cos->dim() != 2 || cos->sizes() != sin->sizes() || 2 * cos->size(1) != rotary_dim)
        value_error("rope tables " + shape_text(*cos) + " do not cover " +
                    (a[10] == Py_None ? "head_dim " : "rotary_dim ") + std::to_string(rotary_dim));
      if (cos->size(0) > INT32_MAX) value_error("rope tables too long");
    }
    const c10::DeviceGuard guard(at_.device);
    Tensor made;
    if (q && !q_out) made = fresh_like(*q), q_out = &made;
    dkv_append_args p;
    p.k = k.data_ptr(), p.v = v.data_ptr(), p.q = ptr(q);
    p.in_dtype = dtype_code(k.scalar_type());
    p.n_q_heads = q ? static_cast<int32_t>(q->size(1)) : 0;
    p.n_rows = rows;
    p.k_stride_row = k.stride(0), p.k_stride_head = k.stride(1);
    p.v_stride_row = v.stride(0), p.v_stride_head = v.stride(1);
    p.q_stride_row = q ? q->stride(0) : 0, p.q_stride_head = q ? q->stride(1) : 0;
    p.q_out = ptr(q_out);
    p.q_out_stride_row = q ? q_out->stride(0) : 0, p.q_out_stride_head = q ? q_out->stride(1) : 0;
    p.slots = slots.data_ptr<int64_t>();
    p.positions = cos ? positions->data_ptr<int32_t>() : nullptr;
    p.rope_cos = static_cast<float *>(ptr(cos)), p.rope_sin = static_cast<float *>(ptr(sin));
    p.rope_max_pos = cos ? static_cast<int32_t>(cos->size(0)) : 0;
    p.k_pages = describe(pages.k, pages.code), p.v_pages = describe(pages.v, pages.code);
    p.status = at_.status();
    dkv_rotary rotary;
    rotary.dim = static_cast<int32_t>(rotary_dim), rotary.interleaved = crossed;
    if (scales) {
      if (look)
        refuse(at_, "dkv_append_paged_quant_check", [&](int32_t *word) {
          dkv_append_args rows = p;
          rows.status = word;
          return g_append_check(&rows, at_.stream());
        });
      const dkv_page_scales ks = describe_scales(*scales.k), vs = describe_scales(*scales.v);
      check(g_append_quant(&p, &rotary, &ks, &vs, at_.stream()), "dkv_append_paged_quant");
    } else {
      check(g_append(&p, &rotary, at_.stream()), "dkv_append_paged");
    }
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[9]);  // the caller's q_out, or None
    return a[9];
  });
}

// attend(q, k_pages, v_pages, cu_seqlens, block_tables, table_lens, max_seq_len, scale, out, return_lse,
//        kv_scales)
//   -> out, or (out, lse)
PyObject *attend(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    if (count != 11) type_error("attend takes 11 arguments");
    const Tensor &q = tensor(a[0], "q");
    const PairOfScales scales(a[10]);
    const Pages pages(tensor(a[1], "k_pages"), tensor(a[2], "v_pages"), static_cast<bool>(scales));
    const Sequences seqs(a[3], a[4], a[5], a[6]);
    const Tensor *out = maybe(a[8], "out");
    const int wanted = PyObject_IsTrue(a[9]);
    if (wanted < 0) throw Raised{nullptr, ""};
    const bool return_lse = wanted == 1;
    const int64_t n = seqs.n, hd = pages.hd;
    double scale = 1.0 / std::sqrt(static_cast<double>(hd > 0 ? hd : 1));
    if (a[7] != Py_None) {
      scale = PyFloat_AsDouble(a[7]);
      if (scale == -1.0 && PyErr_Occurred()) throw Raised{nullptr, ""};
    }
    rows_of(q, "q", n, -1, hd);
    const int64_t heads = q.size(1);
    scales.check(pages);
    const int q_code = dtype_code(q.scalar_type());
    if (!scales && q.scalar_type() != pages.k.scalar_type())
      type_error(std::string("q is ") + dtype_name(q.scalar_type()) + ", the pages are " +
                 dtype_name(pages.k.scalar_type()));
    if (hd > 256) value_error("head_dim " + std::to_string(hd) + " is above 256");
    if (heads == 0 || pages.heads == 0 || heads % pages.heads || heads > INT32_MAX)
      value_error(std::to_string(heads) + " query heads do not share " + std::to_string(pages.heads) +
                  " KV heads evenly");
    seqs.check_shapes();
    if (out) {
      rows_of(*out, "out", n, heads, hd);
      if (out->scalar_type() != q.scalar_type()) type_error("out must have q's dtype");
      written(*out, "out", &q, "q");
    }
    const Place at_("paged_decode_attention", q);
    at_.also(&pages.k), at_.also(&pages.v), at_.also(&seqs.cu), at_.also(&seqs.tables), at_.also(seqs.lens), at_.also(out);
    at_.also(scales.k), at_.also(scales.v);
    seqs.check_types();
    const c10::DeviceGuard guard(at_.device);
    Tensor made, lse, workspace;
    if (!out) made = fresh_like(q), out = &made;
    if (return_lse) lse = fresh_tensor({n, heads}, at::kFloat, at_.device);
    dkv_paged_decode_args p;
    p.q = q.data_ptr();
    p.q_stride_seq = q.stride(0), p.q_stride_head = q.stride(1);
    p.n_q_heads = static_cast<int32_t>(heads);
    p.scale = static_cast<float>(scale);
    p.seqs = seqs.describe();
    p.k_pages = describe(pages.k, pages.code), p.v_pages = describe(pages.v, pages.code);
    p.out = out->data_ptr();
    p.out_stride_seq = out->stride(0), p.out_stride_head = out->stride(1);
    p.lse = return_lse ? lse.data_ptr<float>() : nullptr;
    p.workspace = nullptr, p.workspace_bytes = 0;
    p.status = at_.status();
    int64_t bytes = 0;
    if (scales)
      check(g_workspace_quant(&p, q_code, &bytes), "dkv_paged_decode_quant_workspace_bytes");
    else
      check(g_workspace(&p, &bytes), "dkv_paged_decode_workspace_bytes");
    if (bytes > 0) {  // in stream order the allocator may give it away once the launches are queued
      workspace = fresh_tensor({bytes}, at::kByte, at_.device);
      p.workspace = workspace.data_ptr(), p.workspace_bytes = bytes;
    }
    if (scales) {
      const dkv_page_scales ks = describe_scales(*scales.k), vs = describe_scales(*scales.v);
      check(g_attend_quant(&p, q_code, &ks, &vs, at_.stream()), "dkv_paged_decode_attention_quant");
    } else {
      check(g_attend(&p, at_.stream()), "dkv_paged_decode_attention");
    }
    PyObject *first;
    if (made.defined()) {
      first = THPVariable_Wrap(made);
    } else {
      first = a[8];
      Py_INCREF(first);
    }
    if (!return_lse || first == nullptr) return first;
    return Py_BuildValue("(NN)", first, THPVariable_Wrap(lse));
  });
}

// 8-bit pages of K or V, [num_blocks, block_size, heads, head_dim], and their scales
void check_coded(const Tensor &pages, const Tensor &scales) {
  if (pages.dim() != 4) value_error("unsupported paged KV layout " + shape_text(pages));
  if (!is_code(pages.scalar_type()))
    type_error(std::string("page_scales go with 8-bit pages (float8_e4m3fn or int8), not ") + dtype_name(pages.scalar_type()));
  if (pages.stride(3) != 1 && pages.size(3) > 1) value_error("paged cache head_dim must be contiguous");
  if (pages.size(1) > 1024) value_error("8-bit pages have at most 1024 slots a block");
  if (pages.size(2) > INT32_MAX || pages.size(3) > INT32_MAX) value_error("paged cache too large");
  scales_of(scales, "page_scales", pages);
}

// scatter(delta, pages, page_scales, cu_seqlens, block_tables, table_lens, max_seq_len, look)
PyObject *scatter(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    if (count != 8) type_error("scatter takes 8 arguments");
    const int look = PyObject_IsTrue(a[7]);
    if (look < 0) throw Raised{nullptr, ""};
    const Tensor &delta = tensor(a[0], "delta"), &pages = tensor(a[1], "pages"), &scales = tensor(a[2], "page_scales");
    const Sequences seqs(a[3], a[4], a[5], a[6]);
    check_coded(pages, scales);
    if (delta.dim() != 3) value_error("delta " + shape_text(delta) + " must be [rows, heads, head_dim]");
    rows_of(delta, "delta", delta.size(0), pages.size(2), pages.size(3));
    const int code = dtype_code(delta.scalar_type());
    seqs.check_shapes();
    written(pages, "pages", nullptr, ""), written(scales, "page_scales", nullptr, "");
    const Place at_("scatter_into_paged_batched", pages);
    at_.also(&delta), at_.also(&scales), at_.also(&seqs.cu), at_.also(&seqs.tables), at_.also(seqs.lens);
    seqs.check_types();
    const c10::DeviceGuard guard(at_.device);
    const dkv_paged_cache cache = describe(pages, code_of(pages.scalar_type()));
    const dkv_page_scales s = describe_scales(scales);
    const dkv_seq_batch q = seqs.describe();
    if (look)
      refuse(at_, "dkv_scatter_paged_quant_check",
             [&](int32_t *word) { return g_scatter_check(delta.size(0), &cache, &q, word, at_.stream()); });
    check(g_scatter_quant(delta.data_ptr(), code, delta.size(0), delta.stride(0), delta.stride(1), &cache, &s, &q,
                          at_.status(), at_.stream()),
          "dkv_scatter_paged_quant");
    Py_RETURN_NONE;
  });
}

// gather(pages, page_scales, cu_seqlens, block_tables, table_lens, max_seq_len, rows, like, out) -> out
// like: a tensor of the type that a new out gets
PyObject *gather(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    if (count != 9) type_error("gather takes 9 arguments");
    const Tensor &pages = tensor(a[0], "pages"), &scales = tensor(a[1], "page_scales");
    const Sequences seqs(a[2], a[3], a[4], a[5]);
    const int64_t rows = integer(a[6]);
    const Tensor *out = maybe(a[8], "out");
    check_coded(pages, scales);
    if (rows < 0) value_error("rows must not be negative");
    if (out) {
      rows_of(*out, "out", rows, pages.size(2), pages.size(3));
      written(*out, "out", nullptr, "");
    }
    const at::ScalarType type = out ? out->scalar_type() : tensor(a[7], "like").scalar_type();
    const int code = dtype_code(type);
    seqs.check_shapes();
    const Place at_("gather_from_paged_batched", pages);
    at_.also(&scales), at_.also(&seqs.cu), at_.also(&seqs.tables), at_.also(seqs.lens), at_.also(out);
    seqs.check_types();
    const c10::DeviceGuard guard(at_.device);
    Tensor made;
    if (!out) made = fresh_tensor({rows, pages.size(2), pages.size(3)}, type, at_.device), out = &made;
    const dkv_paged_cache cache = describe(pages, code_of(pages.scalar_type()));
    const dkv_page_scales s = describe_scales(scales);
    const dkv_seq_batch q = seqs.describe();
    check(g_gather_quant(&cache, &s, &q, out->data_ptr(), code, rows, out->stride(0), out->stride(1), made.defined(),
                         at_.status(), at_.stream()),
          "dkv_gather_paged_quant");
    if (made.defined()) return THPVariable_Wrap(made);
    Py_INCREF(a[8]);
    return a[8];
  });
}

// bind(plan, append, workspace, attend, append_quant, scatter_quant, gather_quant, workspace_quant, attend_quant, append_check,
//      scatter_check, raise_error, status_word): entry addresses and callbacks
PyObject *bind(PyObject *, PyObject *const *a, Py_ssize_t count) {
  return guarded([&]() -> PyObject * {
    constexpr int kEntries = 11;
    if (count != kEntries + 2) type_error("bind takes 13 arguments");
    void *entry[kEntries];
    for (int i = 0; i < kEntries; ++i) {
      entry[i] = PyLong_AsVoidPtr(a[i]);
      if (entry[i] == nullptr) {
        if (PyErr_Occurred()) throw Raised{nullptr, ""};
        value_error("bind: an entry without an address");
      }
    }
    g_plan = reinterpret_cast<decltype(g_plan)>(entry[0]);
    g_append = reinterpret_cast<decltype(g_append)>(entry[1]);
    g_workspace = reinterpret_cast<decltype(g_workspace)>(entry[2]);
    g_attend = reinterpret_cast<decltype(g_attend)>(entry[3]);
    g_append_quant = reinterpret_cast<decltype(g_append_quant)>(entry[4]);
    g_scatter_quant = reinterpret_cast<decltype(g_scatter_quant)>(entry[5]);
    g_gather_quant = reinterpret_cast<decltype(g_gather_quant)>(entry[6]);
    g_workspace_quant = reinterpret_cast<decltype(g_workspace_quant)>(entry[7]);
    g_attend_quant = reinterpret_cast<decltype(g_attend_quant)>(entry[8]);
    g_append_check = reinterpret_cast<decltype(g_append_check)>(entry[9]);
    g_scatter_check = reinterpret_cast<decltype(g_scatter_check)>(entry[10]);
    Py_INCREF(a[kEntries]);
    Py_XSETREF(g_raise, a[kEntries]);
    Py_INCREF(a[kEntries + 1]);
    Py_XSETREF(g_status_word, a[kEntries + 1]);
    Py_RETURN_NONE;
  });
}

PyMethodDef kMethods[] = {
    {"bind", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(bind)), METH_FASTCALL, nullptr},
    {"plan", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(plan)), METH_FASTCALL, nullptr},
    {"rope_ready", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(rope_ready)), METH_FASTCALL, nullptr},
    {"append", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(append)), METH_FASTCALL, nullptr},
    {"attend", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(attend)), METH_FASTCALL, nullptr},
    {"scatter", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(scatter)), METH_FASTCALL, nullptr},
    {"gather", reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(gather)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_step", "Host side of the paged step operators.", -1, kMethods};

}  // namespace

PyMODINIT_FUNC PyInit__step() { return PyModule_Create(&kModule); }
