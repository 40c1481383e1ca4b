// Python module `deviceops_native`: the operators on device tensors (b2vx_*_noalloc of include/b2vx.h) for torch tensors.
//
// A decode step makes a dozen such calls of a few microseconds of GPU time each, so what a call costs the host counts: checks, outputs and
// workspaces are handled here, in one step between the interpreter and the library, with positional arguments only (deviceops.py has the
// keywords and the documentation).  Outputs and workspaces come from torch's caching allocator, work goes to the current stream
// of the tensors' device.
#include <Python.h>

#include <ATen/ATen.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>

#include <cstdint>
#include <initializer_list>
#include <stdexcept>
#include <string>

#include "b2vx.h"

namespace {

struct Refused {          // a status of the library
  b2vx_status status;
  std::string message;
};

void need(bool ok, const char* message) {
  if (!ok) throw std::invalid_argument(message);
}
[[noreturn]] void wrong(const std::string& message) { throw std::invalid_argument(message); }

int dtype_code(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return B2VX_DT_FLOAT32;
    case at::kHalf: return B2VX_DT_FLOAT16;
    case at::kBFloat16: return B2VX_DT_BFLOAT16;
    default: return 0;
  }
}

const at::Tensor& tensor(PyObject* o, const char* what) {
  if (!THPVariable_Check(o)) wrong(std::string(what) + " must be a tensor");
  const at::Tensor& t = THPVariable_Unpack(o);
  if (!t.has_storage()) wrong(std::string(what) + " has no memory of its own (a wrapper of torch.func, or not strided)");
  if (c10::GradMode::is_enabled() && t.requires_grad()) wrong(std::string(what) + " requires a gradient, which these operators do not have");
  if (t._fw_grad(0).defined()) wrong(std::string(what) + " carries a forward-mode gradient, which these operators do not have");
  // calls do not pass torch's dispatcher: a trace would keep their outputs as constants
  need(!torch::jit::tracer::isTracing(), "these operators cannot be traced");
  return t;
}
std::string shape_of(at::IntArrayRef s) {
  std::string r = "(";
  for (size_t i = 0; i < s.size(); ++i) r += (i ? ", " : "") + std::to_string(s[i]);
  return r + ")";
}

// Rows of float32, float16 or bfloat16 whose last dimension is contiguous; the distance between rows.
uint64_t rows_of(const at::Tensor& t, const char* what) {
  if (t.dim() != 2) wrong(std::string(what) + " must be a tensor of two dimensions");
  if (!dtype_code(t.scalar_type())) wrong(std::string(what) + " must have the type float32, float16 or bfloat16");
  if (t.size(1) > 1 && t.stride(1) != 1) wrong(std::string(what) + " must be contiguous along its last dimension");
  if (t.is_neg() || t.is_conj()) wrong(std::string(what) + " must not be a lazy view");
  return static_cast<uint64_t>(t.size(0) > 1 ? t.stride(0) : t.size(1));
}
// The address of a dense tensor of this type, shape and device; null for None.
void* dense(PyObject* o, const char* what, at::ScalarType type, at::IntArrayRef shape, const at::Device& device) {
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, what);
  if (t.scalar_type() != type) wrong(std::string(what) + " must have the type " + c10::toString(type));
  if (t.sizes() != shape) wrong(std::string(what) + " must have the shape " + shape_of(shape) + ", not " + shape_of(t.sizes()));
  if (!t.is_contiguous()) wrong(std::string(what) + " must be contiguous");
  if (t.device() != device) wrong(std::string(what) + " is on another device");
  return t.data_ptr();
}
void* tensor_scale(PyObject* o, long format, long count, const at::Device& device, const char* what) {
  if ((o != Py_None) != (format == B2VX_FP4_BLOCK16)) wrong(std::string(what) + " belongs to block16 and only to it");
  if (o == Py_None) return nullptr;
  const at::Tensor& t = tensor(o, what);
  if (t.numel() != count) wrong(std::string(what) + " must have " + std::to_string(count) + " elements");
  return dense(o, what, at::kFloat, t.sizes(), device);
}
at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, const at::Device& device) { return at::empty(shape, at::TensorOptions().dtype(type).device(device)); }
// Several dense tensors in one allocation, each on its own multiple of 256 bytes (a call of the allocator costs more than a view).
class Carver {
 public:
  explicit Carver(const at::Device& device) : device_(device) {}
  // Adds a tensor; returns its number.
  int add(at::IntArrayRef shape, at::ScalarType type) {
    int64_t n = 1;
    for (int64_t d : shape) n *= d;
    parts_[count_] = {bytes_, type};
    bytes_ += (n * static_cast<int64_t>(c10::elementSize(type)) + 255) / 256 * 256;
    return count_++;
  }
  at::Tensor take(int i, at::IntArrayRef shape) {
    if (!storage_.defined()) storage_ = empty({bytes_}, at::kByte, device_);
    const Part& p = parts_[i];
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(storage_.storage()), c10::DispatchKeySet(c10::DispatchKey::CUDA), c10::scalarTypeToTypeMeta(p.type));
    c10::TensorImpl* impl = t.unsafeGetTensorImpl();
    impl->set_storage_offset(p.at / static_cast<int64_t>(c10::elementSize(p.type)));
    impl->set_sizes_contiguous(shape);
    return t;
  }

 private:
  struct Part {
    int64_t at;
    at::ScalarType type;
  };
  at::Device device_;
  at::Tensor storage_;
  Part parts_[8] = {};
  int count_ = 0;
  int64_t bytes_ = 0;
};
at::Tensor output(PyObject* out, at::IntArrayRef shape, at::ScalarType type, const at::Device& device) {
  if (out == Py_None) return empty(shape, type, device);
  const at::Tensor& t = tensor(out, "out");
  rows_of(t, "out");
  if (t.sizes() != shape || t.device() != device) wrong("out must have the shape " + shape_of(shape) + " on " + device.str());
  need(t.size(0) <= 1 || t.stride(0) >= t.size(1), "out has rows that overlap");
  return t;
}
// An output of the caller's has been written: a graph that saved it for a backward pass notices.
void written(PyObject* out) {
  if (out == Py_None) return;
  const at::Tensor& t = THPVariable_Unpack(out);
  if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// A tensor's memory: rows of `width` bytes, `pitch` apart.
struct Memory {
  explicit Memory(const at::Tensor& t) : at(static_cast<const char*>(t.data_ptr())) {
    const int64_t size = static_cast<int64_t>(t.element_size());
    if (t.dim() == 2 && !t.is_contiguous()) {
      rows = t.size(0);
      pitch = t.stride(0) * size;
      width = t.size(1) * size;
    } else {
      width = t.numel() * size;
    }
  }
  const char* end() const { return at + (rows - 1) * pitch + width; }
  const char* at;
  int64_t rows = 1, pitch = 0, width;
};
// Rows of one pitch, such as columns of a larger tensor, may lie between one another; else the first to the last byte count.
bool overlap(const at::Tensor& ta, const at::Tensor& tb) {
  if (!ta.numel() || !tb.numel()) return false;
  const Memory a(ta), b(tb);
  if (a.at >= b.end() || b.at >= a.end()) return false;
  const int64_t pitch = a.rows > 1 ? a.pitch : b.pitch;
  if (pitch == 0 || (a.rows > 1 && b.rows > 1 && a.pitch != b.pitch)) return true;
  const int64_t apart = ((b.at - a.at) % pitch + pitch) % pitch;       // columns of b behind those of a
  return apart < a.width || apart + b.width > pitch;
}
// Refuses an output of the caller's that overlaps one of these arguments.
void apart(const at::Tensor& y, PyObject* out, PyObject* const* a, std::initializer_list<int> inputs) {
  if (out == Py_None) return;
  for (int i : inputs)
    if (a[i] != Py_None && overlap(y, tensor(a[i], "an input"))) wrong("out overlaps an input");
}
uint64_t row_stride(const at::Tensor& t) { return static_cast<uint64_t>(t.size(0) > 1 ? t.stride(0) : t.size(1)); }

// The device of a call as the current one, its current stream, and the place for a message.
struct Call {
  explicit Call(const at::Device& device) : guard((need(device.is_cuda(), "tensors must be on a GPU"), device)), stream(c10::cuda::getCurrentCUDAStream(device.index()).stream()) {}
  void operator()(b2vx_status st) const {
    if (st != B2VX_OK) throw Refused{st, err};
  }
  c10::cuda::CUDAGuard guard;
  cudaStream_t stream;
  mutable char err[256] = {0};
};

long number(PyObject* o) {
  const long v = PyLong_AsLong(o);
  if (v == -1 && PyErr_Occurred()) {
    PyErr_Clear();
    wrong("a whole number is needed");
  }
  return v;
}
at::ScalarType scalar_type(PyObject* o) {
  if (!THPDtype_Check(o) || !dtype_code(reinterpret_cast<THPDtype*>(o)->scalar_type)) wrong("the type must be float32, float16 or bfloat16");
  return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
int64_t block_of(long format) {
  need(format == B2VX_FP4_BLOCK32 || format == B2VX_FP4_BLOCK16, "unknown format");
  return format == B2VX_FP4_BLOCK32 ? 32 : 16;
}
int64_t index_rows(PyObject* row_index, const at::Tensor& x) { return row_index == Py_None ? x.size(0) : tensor(row_index, "row_index").numel(); }

// (x, format, scale, row_index) -> (codes, scales)
PyObject* quantize(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x");
  const long format = number(a[1]);
  const int64_t block = block_of(format);
  const uint64_t stride = rows_of(x, "x");
  const int64_t rows = index_rows(a[3], x), k = x.size(1);
  const at::Device device = x.device();
  void* scale = tensor_scale(a[2], format, 1, device, "scale");
  void* index = dense(a[3], "row_index", at::kInt, {rows}, device);
  Call call(device);
  const int64_t codes_shape[2] = {rows, (k + 31) / 32 * 16}, scales_shape[2] = {rows, (k + block - 1) / block};
  Carver carver(device);
  carver.add(codes_shape, at::kByte);
  carver.add(scales_shape, at::kByte);
  at::Tensor codes = carver.take(0, codes_shape), scales = carver.take(1, scales_shape);
  const b2vx_fp4_quantize_desc d = {static_cast<int32_t>(format), dtype_code(x.scalar_type()), static_cast<uint64_t>(x.size(0)), static_cast<uint64_t>(rows),
                                    static_cast<uint64_t>(k), stride, static_cast<uint64_t>(codes.size(1)), static_cast<uint64_t>(scales.size(1))};
  call(b2vx_fp4_quantize_noalloc(&d, x.data_ptr(), static_cast<const int32_t*>(index), static_cast<const float*>(scale), codes.data_ptr(), scales.data_ptr(),
                                 call.stream, call.err, sizeof(call.err)));
  PyObject* r = PyTuple_New(2);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(codes)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(scales)));
  return r;
}

// (codes, scales, k, format, scale, dtype, out) -> y
PyObject* dequantize(PyObject* const* a) {
  const at::Tensor& codes = tensor(a[0], "codes");
  const int64_t k = number(a[2]);
  const long format = number(a[3]);
  const int64_t block = block_of(format);
  need(codes.dim() == 2 && k >= 0, "codes must be a tensor of two dimensions");
  const int64_t rows = codes.size(0);
  const at::Device device = codes.device();
  void* c = dense(a[0], "codes", at::kByte, {rows, (k + 31) / 32 * 16}, device);
  void* s = dense(a[1], "scales", at::kByte, {rows, (k + block - 1) / block}, device);
  void* scale = tensor_scale(a[4], format, 1, device, "scale");
  Call call(device);
  at::Tensor y = output(a[6], {rows, k}, scalar_type(a[5]), device);
  apart(y, a[6], a, {0, 1, 4});
  const b2vx_fp4_dequantize_desc d = {static_cast<int32_t>(format), dtype_code(y.scalar_type()), static_cast<uint64_t>(rows), static_cast<uint64_t>(k),
                                      static_cast<uint64_t>(codes.size(1)), static_cast<uint64_t>((k + block - 1) / block), row_stride(y)};
  call(b2vx_fp4_dequantize_noalloc(&d, c, s, static_cast<const float*>(scale), y.data_ptr(), call.stream, call.err, sizeof(call.err)));
  written(a[6]);
  return THPVariable_Wrap(std::move(y));
}

// (scales [matrices][rows][blocks], format, gated) -> packed scales
PyObject* pack(PyObject* const* a) {
  const at::Tensor& scales = tensor(a[0], "scales");
  const long format = number(a[1]);
  const int64_t block = block_of(format);
  need(scales.dim() == 3 && scales.scalar_type() == at::kByte && scales.is_contiguous(), "scales must be a dense uint8 tensor");
  Call call(scales.device());
  const int32_t gated = number(a[2]) != 0;
  const uint64_t matrices = scales.size(0), n = gated ? scales.size(1) / 2 : scales.size(1), k = scales.size(2) * block;
  size_t bytes = 0;
  const b2vx_status st = b2vx_fp4_packed_scales_size_noalloc(static_cast<int32_t>(format), matrices, n, gated, k, &bytes);
  if (st != B2VX_OK) throw Refused{st, "more than 1024 matrices, or an extent out of range"};
  at::Tensor packed = empty({static_cast<int64_t>(bytes)}, at::kByte, scales.device());
  call(b2vx_fp4_pack_scales_noalloc(static_cast<int32_t>(format), matrices, n, gated, k, scales.data_ptr(), packed.data_ptr(), call.stream, call.err, sizeof(call.err)));
  return THPVariable_Wrap(std::move(packed));
}

// (x, w, packed scales or None, w_scale, format or 0, gated, offsets, row_index, bias, x_scale, dtype or None, out) -> y.  w: codes [..][n][k / 2] or
// 16-bit numbers [..][n][k].
PyObject* product(PyObject* const* a) {
  const at::Tensor& x = tensor(a[0], "x");
  const at::Tensor& w = tensor(a[1], "weight");
  const long format = number(a[4]), gated = number(a[5]);
  const uint64_t stride = rows_of(x, "x");
  const at::Device device = x.device();
  need(w.dim() == 2 || w.dim() == 3, "weight must have two or three dimensions");
  need(w.is_contiguous(), "weight must be contiguous");
  need(w.device() == device, "weight is on another device");
  const int64_t experts = w.dim() == 3 ? w.size(0) : 0, w_rows = w.size(-2), k = format ? w.size(-1) * 2 : w.size(-1);
  need(w.dim() == 2 || (experts > 0 && experts <= UINT32_MAX), "weight has no experts or too many");
  b2vx_linear_args p = {};
  if (format) {
    need(w.scalar_type() == at::kByte, "codes must have the type uint8");
    p.w_scales = tensor(a[2], "scales").data_ptr();
    p.w_scale = static_cast<const float*>(tensor_scale(a[3], format, experts ? experts : 1, device, "the weight's scale"));
  } else {
    need(w.scalar_type() == x.scalar_type(), "weight must be an Fp4Weight or a tensor of x's type");
  }
  p.x_scale = static_cast<const float*>(tensor_scale(a[9], format, 1, device, "x_scale"));
  need((a[6] != Py_None) == (experts > 0), "offsets belong to weights of experts and only to them");
  if (x.size(1) != k) wrong("x has " + std::to_string(x.size(1)) + " columns, the weight " + std::to_string(k));
  need(!gated || w_rows % 16 == 0, "the rows of a gated weight must be a multiple of 16");
  const int64_t rows = index_rows(a[7], x), n = gated ? w_rows / 2 : w_rows;
  p.offsets = static_cast<const int32_t*>(dense(a[6], "offsets", at::kInt, {experts + 1}, device));
  p.row_index = static_cast<const int32_t*>(dense(a[7], "row_index", at::kInt, {rows}, device));
  p.bias = static_cast<const float*>(experts ? dense(a[8], "bias", at::kFloat, {experts, w_rows}, device) : dense(a[8], "bias", at::kFloat, {w_rows}, device));
  Call call(device);
  at::Tensor y = output(a[11], {rows, n}, a[10] == Py_None ? x.scalar_type() : scalar_type(a[10]), device);
  apart(y, a[11], a, {0, 1, 2, 3, 6, 7, 8, 9});
  b2vx_linear_desc d = {};
  d.w_format = static_cast<int32_t>(format);
  d.x_dtype = dtype_code(x.scalar_type());
  d.y_dtype = dtype_code(y.scalar_type());
  d.gated = gated != 0;
  d.experts = static_cast<uint32_t>(experts);
  d.x_rows = x.size(0);
  d.rows = rows;
  d.n = n;
  d.k = k;
  d.x_stride = stride;
  d.y_stride = row_stride(y);
  p.x = x.data_ptr();
  p.w = w.data_ptr();
  p.y = y.data_ptr();
  at::Tensor workspace;
  if (!b2vx_linear_in_place_noalloc(&d, &p)) {
    call(b2vx_linear_workspace_size_noalloc(&d, &p.workspace_bytes, call.err, sizeof(call.err)));
    workspace = empty({static_cast<int64_t>(p.workspace_bytes)}, at::kByte, device);
    p.workspace = workspace.data_ptr();
  }
  call(b2vx_linear_noalloc(&d, &p, call.stream, call.err, sizeof(call.err)));
  written(a[11]);
  return THPVariable_Wrap(std::move(y));
}

// (logits, top_k, normalize) -> (ids, weights, offsets, row_index, slots)
PyObject* route(PyObject* const* a) {
  const at::Tensor& logits = tensor(a[0], "logits");
  const long top_k = number(a[1]), normalize = number(a[2]);
  const uint64_t stride = rows_of(logits, "logits");
  const int64_t tokens = logits.size(0), experts = logits.size(1);
  const at::Device device = logits.device();
  need(top_k >= 0 && top_k <= 1024, "top_k is out of range");
  need(experts <= UINT32_MAX, "logits has too many columns");
  Call call(device);
  const b2vx_route_desc d = {dtype_code(logits.scalar_type()), normalize != 0, static_cast<uint32_t>(experts), static_cast<uint32_t>(top_k), static_cast<uint64_t>(tokens), stride};
  size_t bytes = 0;
  call(b2vx_route_workspace_size_noalloc(&d, &bytes, call.err, sizeof(call.err)));
  const int64_t pairs[2] = {tokens, top_k}, rows[1] = {tokens * top_k}, starts[1] = {experts + 1}, work[1] = {static_cast<int64_t>(bytes)};
  at::Tensor workspace;
  if (bytes) workspace = empty(work, at::kByte, device);
  Carver carver(device);
  for (at::ScalarType type : {at::kInt, at::kFloat, at::kInt}) carver.add(pairs, type);
  carver.add(rows, at::kInt);
  carver.add(starts, at::kInt);
  at::Tensor ids = carver.take(0, pairs), weights = carver.take(1, pairs), slots = carver.take(2, pairs), row_index = carver.take(3, rows), offsets = carver.take(4, starts);
  call(b2vx_route_noalloc(&d, logits.data_ptr(), ids.data_ptr<int32_t>(), weights.data_ptr<float>(), offsets.data_ptr<int32_t>(), row_index.data_ptr<int32_t>(),
                          slots.data_ptr<int32_t>(), bytes ? workspace.data_ptr() : nullptr, bytes, call.stream, call.err, sizeof(call.err)));
  PyObject* r = PyTuple_New(5);
  PyTuple_SET_ITEM(r, 0, THPVariable_Wrap(std::move(ids)));
  PyTuple_SET_ITEM(r, 1, THPVariable_Wrap(std::move(weights)));
  PyTuple_SET_ITEM(r, 2, THPVariable_Wrap(std::move(offsets)));
  PyTuple_SET_ITEM(r, 3, THPVariable_Wrap(std::move(row_index)));
  PyTuple_SET_ITEM(r, 4, THPVariable_Wrap(std::move(slots)));
  return r;
}

// (z, slots, weights, residual, out) -> y
PyObject* combine(PyObject* const* a) {
  const at::Tensor& z = tensor(a[0], "z");
  const uint64_t stride = rows_of(z, "z");
  const at::Tensor& slots = tensor(a[1], "slots");
  need(slots.dim() == 2, "slots must be a tensor of two dimensions");
  need(slots.size(1) <= 1024, "top_k is out of range");
  const int64_t tokens = slots.size(0), top_k = slots.size(1), n = z.size(1);
  const at::Device device = z.device();
  const void* s = dense(a[1], "slots", at::kInt, {tokens, top_k}, device);
  need(a[2] != Py_None, "weights must be a tensor");
  const void* w = dense(a[2], "weights", at::kFloat, {tokens, top_k}, device);
  uint64_t r_stride = 0;
  const void* residual = nullptr;
  if (a[3] != Py_None) {
    const at::Tensor& r = tensor(a[3], "residual");
    r_stride = rows_of(r, "residual");
    need(r.scalar_type() == z.scalar_type() && r.device() == device && r.size(0) == tokens && r.size(1) == n, "residual must have z's type and device and a row of z's width for each token");
    residual = r.data_ptr();
  }
  Call call(device);
  at::Tensor y = output(a[4], {tokens, n}, z.scalar_type(), device);
  need(y.scalar_type() == z.scalar_type(), "out must have z's type");
  apart(y, a[4], a, {0, 1, 2});
  if (residual && residual != y.data_ptr()) apart(y, a[4], a, {3});
  else if (residual) need(r_stride == row_stride(y), "out overlaps the residual and has other rows");
  const b2vx_combine_desc d = {dtype_code(z.scalar_type()), static_cast<uint32_t>(top_k), static_cast<uint64_t>(tokens), static_cast<uint64_t>(n),
                               static_cast<uint64_t>(z.size(0)), stride, r_stride, row_stride(y)};
  call(b2vx_combine_noalloc(&d, z.data_ptr(), static_cast<const int32_t*>(s), static_cast<const float*>(w), residual, y.data_ptr(), call.stream, call.err, sizeof(call.err)));
  written(a[4]);
  return THPVariable_Wrap(std::move(y));
}

// (device index)
PyObject* check(PyObject* const* a) {
  Call call(at::Device(at::kCUDA, static_cast<c10::DeviceIndex>(number(a[0]))));
  b2vx_status st;
  Py_BEGIN_ALLOW_THREADS
  st = b2vx_device_check_noalloc(call.stream, call.err, sizeof(call.err));
  Py_END_ALLOW_THREADS
  call(st);
  Py_RETURN_NONE;
}

PyObject* attribute(const char* module, const char* name) {
  PyObject* m = PyImport_ImportModule(module);
  PyObject* a = m ? PyObject_GetAttrString(m, name) : nullptr;
  Py_XDECREF(m);
  return a;
}

template <PyObject* (*FN)(PyObject* const*), int ARGS>
PyObject* entry(PyObject*, PyObject* const* args, Py_ssize_t count) {
  if (count != ARGS) {
    PyErr_SetString(PyExc_TypeError, "wrong number of arguments");
    return nullptr;
  }
  try {
    return FN(args);
  } catch (const Refused& r) {
    PyObject* type = attribute("pyb2vx", "B2vxError");
    PyObject* error = type ? PyObject_CallFunction(type, "is", r.status, r.message.c_str()) : nullptr;
    if (error) PyErr_SetObject(type, error);
    Py_XDECREF(error);
    Py_XDECREF(type);
  } catch (const std::invalid_argument& e) {
    PyErr_SetString(PyExc_ValueError, e.what());
  } catch (const c10::OutOfMemoryError& e) {
    PyObject* type = attribute("torch", "OutOfMemoryError");
    if (type) PyErr_SetString(type, e.what_without_backtrace());
    Py_XDECREF(type);
  } catch (const std::exception& e) {
    PyErr_SetString(PyExc_RuntimeError, e.what());
  }
  return nullptr;
}

#define B2VX_ENTRY(fn, args) {#fn, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(entry<fn, args>)), METH_FASTCALL, nullptr}
PyMethodDef kMethods[] = {B2VX_ENTRY(quantize, 4), B2VX_ENTRY(dequantize, 7), B2VX_ENTRY(pack, 3), B2VX_ENTRY(product, 12),
                          B2VX_ENTRY(route, 3),    B2VX_ENTRY(combine, 5),    B2VX_ENTRY(check, 1), {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "deviceops_native", nullptr, -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_deviceops_native() { return PyModule_Create(&kModule); }
