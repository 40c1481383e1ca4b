// The entry points of the operators on device tensors: argument checks, workspace layout, launches.
#include <cuda_runtime.h>

#include <atomic>
#include <climits>
#include <cstdio>
#include <cstring>
#include <mutex>

#include "block_linear.cuh"
#include "experts.cuh"

namespace {

using namespace b2vx;

constexpr int kMaxDevices = 64;
constexpr uint64_t kMaxExtent = INT_MAX / 4;    // rows, columns
constexpr uint64_t kMaxStride = 1ull << 40;     // elements or bytes; keeps byte offsets of any row inside 63 bits

// Status words the products write a code to when they give up on a barrier, one per GPU, in page-locked memory of the library's own.
alignas(4096) int g_status[4096 / sizeof(int)];
struct PerDevice {
  std::atomic<bool> ready{false};
  int* status = nullptr;
  int sm_count = 0;
};
PerDevice g_devices[kMaxDevices];
std::mutex g_mutex;          // of the first call on each GPU
bool g_registered = false;

b2vx_status fail(char* err, size_t err_len, b2vx_status st, const char* msg) {
  if (err && err_len) std::snprintf(err, err_len, "%s", msg);
  return st;
}
b2vx_status launched(cudaError_t e, char* err, size_t err_len) {
  if (e == cudaSuccess) return B2VX_OK;
  cudaGetLastError();   // a refused launch is reported here and not by the caller's next call
  return fail(err, err_len, B2VX_CUDA_ERROR, cudaGetErrorString(e));
}
#define B2VX_NEED(cond, msg) \
  do { if (!(cond)) return fail(err, err_len, B2VX_INVALID_ARG, msg); } while (0)

bool is_float(int32_t t) { return t == B2VX_DT_FLOAT32 || t == B2VX_DT_FLOAT16 || t == B2VX_DT_BFLOAT16; }
bool is_fp4(int32_t f) { return f == B2VX_FP4_BLOCK32 || f == B2VX_FP4_BLOCK16; }
size_t size_of(int32_t t) { return t == B2VX_DT_FLOAT32 ? 4 : 2; }
bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
size_t round256(size_t n) { return (n + 255) & ~static_cast<size_t>(255); }

b2vx_status device(PerDevice** out, char* err, size_t err_len) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) {
    cudaGetLastError();
    return fail(err, err_len, B2VX_CUDA_ERROR, "no CUDA device");
  }
  PerDevice& d = g_devices[dev];
  if (!d.ready.load(std::memory_order_acquire)) {
    std::lock_guard<std::mutex> lock(g_mutex);
    // the first call may be one that is being captured, where registering memory is refused in other modes
    cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
    cudaError_t e = cudaThreadExchangeStreamCaptureMode(&mode);
    if (e == cudaSuccess) {
      if (!g_registered) e = cudaHostRegister(g_status, sizeof(g_status), cudaHostRegisterPortable | cudaHostRegisterMapped);
      void* p = nullptr;
      if (e == cudaSuccess) {
        g_registered = true;
        e = cudaHostGetDevicePointer(&p, g_status, 0);
      }
      if (e == cudaSuccess) e = cudaDeviceGetAttribute(&d.sm_count, cudaDevAttrMultiProcessorCount, dev);
      cudaThreadExchangeStreamCaptureMode(&mode);
      d.status = static_cast<int*>(p) + dev;
    }
    if (e != cudaSuccess) return launched(e, err, err_len);
    d.ready.store(true, std::memory_order_release);
  }
  *out = &d;
  return B2VX_OK;
}

int device_status(bool clear) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  volatile int* s = &g_status[dev];
  const int v = *s;
  if (clear) *s = 0;
  return v;
}

// The parts of a product's workspace.
struct Workspace {
  size_t codes = 0, scales = 0, between = 0, total = 0;
  uint64_t codes_pitch = 0;
};
Workspace workspace_of(const b2vx_linear_desc& d) {
  Workspace w;
  if (d.w_format) {
    w.codes_pitch = d.k / 2;
    w.codes = round256(d.rows * w.codes_pitch);
    const int experts = d.experts ? static_cast<int>(d.experts) : 1;
    w.scales = round256(static_cast<size_t>(expert_scale_tiles(d.rows, experts, tile_rows(d.rows, experts, d.w_format))) * scale_words(d.k, d.w_format) * kScaleTile);
  } else {
    w.codes_pitch = d.k * 2;
    w.codes = round256(d.rows * w.codes_pitch);
  }
  if (d.w_format) {   // whether there will be a row_index is not known here
    static const int32_t kSome = 0;
    QuantizeArgs q = {};
    q.x_rows = static_cast<long long>(d.x_rows); q.rows = static_cast<long long>(d.rows); q.k = static_cast<long long>(d.k);
    q.format = d.w_format; q.row_index = &kSome;
    w.between = round256(fp4_twice_bytes(q));
  }
  w.total = w.codes + w.scales + w.between;
  return w;
}

b2vx_status check_linear(const b2vx_linear_desc* d, char* err, size_t err_len) {
  B2VX_NEED(d, "null descriptor");
  B2VX_NEED(d->w_format == 0 || is_fp4(d->w_format), "w_format must be 0, B2VX_FP4_BLOCK32 or B2VX_FP4_BLOCK16");
  B2VX_NEED(is_float(d->x_dtype) && is_float(d->y_dtype), "x and y must be float32, float16 or bfloat16");
  B2VX_NEED(d->w_format || d->x_dtype != B2VX_DT_FLOAT32, "a product with 16-bit weights needs x of the weights' type, float16 or bfloat16");
  B2VX_NEED(d->gated == 0 || d->gated == 1, "gated must be 0 or 1");
  B2VX_NEED(!d->gated || d->n % 8 == 0, "n of a gated product must be a multiple of 8");
  B2VX_NEED(d->experts <= static_cast<uint32_t>(kMaxExperts), "at most 1024 experts");
  B2VX_NEED(d->n <= kMaxExtent && d->k <= kMaxExtent && d->rows <= kMaxExtent && d->x_rows <= kMaxExtent, "an extent is out of range");
  B2VX_NEED(d->k > 0, "k must not be zero");
  B2VX_NEED(d->w_format ? d->k % 32 == 0 : d->k % 8 == 0, "k must be a multiple of 32 for 4-bit and of 8 for 16-bit weights");
  B2VX_NEED(d->x_stride >= d->k && d->x_stride <= kMaxStride, "x_stride is smaller than a row or out of range");
  B2VX_NEED(d->y_stride >= d->n && d->y_stride <= kMaxStride, "y_stride is smaller than a row or out of range");
  // tiles of the product and scale tiles of its operands are counted in 32 bits, feature tiles divided as floats
  B2VX_NEED(d->n <= 1u << 27, "an extent is out of range");
  const int experts = d->experts ? static_cast<int>(d->experts) : 1;
  const double feature_tiles = static_cast<double>(weight_tiles(static_cast<long long>(d->n), d->gated)) + 1;
  double most = (static_cast<double>(d->rows) / 64 + experts) * feature_tiles;
  if (d->w_format) {
    const double words = static_cast<double>(scale_words(static_cast<long long>(d->k), d->w_format));
    const int bn = tile_rows(static_cast<long long>(d->rows), experts, d->w_format);
    const double x_tiles = static_cast<double>(expert_scale_tiles(static_cast<long long>(d->rows), experts, bn)) + 2;
    most = most > words * experts * feature_tiles ? most : words * experts * feature_tiles;
    most = most > words * x_tiles ? most : words * x_tiles;
  }
  B2VX_NEED(most < 2e9, "the product has too many tiles");
  return B2VX_OK;
}

}  // namespace

extern "C" b2vx_status b2vx_fp4_quantize_noalloc(const b2vx_fp4_quantize_desc* d, const void* x, const int32_t* row_index, const float* tensor_scale,
                                                 void* codes, void* scales, void* cuda_stream, char* err, size_t err_len) {
  B2VX_NEED(d, "null descriptor");
  B2VX_NEED(is_fp4(d->format), "format must be B2VX_FP4_BLOCK32 or B2VX_FP4_BLOCK16");
  B2VX_NEED(is_float(d->x_dtype), "x must be float32, float16 or bfloat16");
  B2VX_NEED(d->rows <= kMaxExtent && d->k <= kMaxExtent && d->x_rows <= kMaxExtent, "an extent is out of range");
  B2VX_NEED(d->x_stride >= d->k && d->x_stride <= kMaxStride, "x_stride is smaller than a row or out of range");
  const uint64_t block = fp4_block(d->format), k32 = (d->k + 31) / 32 * 32;
  B2VX_NEED(d->codes_pitch % 4 == 0 && d->codes_pitch >= k32 / 2 && d->codes_pitch <= kMaxStride, "codes_pitch must be a multiple of 4 that holds k rounded up to 32");
  B2VX_NEED(d->scales_pitch >= (d->k + block - 1) / block && d->scales_pitch <= kMaxStride, "scales_pitch is smaller than a row of scales");
  B2VX_NEED((tensor_scale != nullptr) == (d->format == B2VX_FP4_BLOCK16), "a tensor scale belongs to B2VX_FP4_BLOCK16 and only to it");
  B2VX_NEED(row_index || d->rows <= d->x_rows, "more rows than x has, and no row_index");
  if (d->rows == 0 || d->k == 0) return B2VX_OK;
  B2VX_NEED(codes && scales && (x || d->x_rows == 0), "null argument");
  B2VX_NEED(aligned(x, size_of(d->x_dtype)) && aligned(codes, 4) && aligned(row_index, 4) && aligned(tensor_scale, 4), "a pointer is not aligned");
  PerDevice* pd;
  b2vx_status st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  QuantizeArgs a = {};
  a.x = x; a.x_dtype = d->x_dtype;
  a.x_stride = static_cast<long long>(d->x_stride); a.x_rows = static_cast<long long>(d->x_rows);
  a.rows = static_cast<long long>(d->rows); a.k = static_cast<long long>(d->k);
  a.row_index = row_index; a.tensor_scale = tensor_scale; a.format = d->format;
  a.codes = static_cast<uint8_t*>(codes); a.codes_pitch = static_cast<long long>(d->codes_pitch);
  a.scales = static_cast<uint8_t*>(scales); a.scales_pitch = static_cast<long long>(d->scales_pitch);
  a.sm_count = pd->sm_count;
  return launched(launch_fp4_quantize(a, static_cast<cudaStream_t>(cuda_stream)), err, err_len);
}

extern "C" b2vx_status b2vx_fp4_dequantize_noalloc(const b2vx_fp4_dequantize_desc* d, const void* codes, const void* scales, const float* tensor_scale,
                                                   void* y, void* cuda_stream, char* err, size_t err_len) {
  B2VX_NEED(d, "null descriptor");
  B2VX_NEED(is_fp4(d->format), "format must be B2VX_FP4_BLOCK32 or B2VX_FP4_BLOCK16");
  B2VX_NEED(is_float(d->y_dtype), "y must be float32, float16 or bfloat16");
  B2VX_NEED(d->rows <= kMaxExtent && d->k <= kMaxExtent, "an extent is out of range");
  const uint64_t block = fp4_block(d->format), k32 = (d->k + 31) / 32 * 32;
  B2VX_NEED(d->codes_pitch % 4 == 0 && d->codes_pitch >= k32 / 2 && d->codes_pitch <= kMaxStride, "codes_pitch must be a multiple of 4 that holds k rounded up to 32");
  B2VX_NEED(d->scales_pitch >= (d->k + block - 1) / block && d->scales_pitch <= kMaxStride, "scales_pitch is smaller than a row of scales");
  B2VX_NEED(d->y_stride >= d->k && d->y_stride <= kMaxStride, "y_stride is smaller than a row or out of range");
  B2VX_NEED((tensor_scale != nullptr) == (d->format == B2VX_FP4_BLOCK16), "a tensor scale belongs to B2VX_FP4_BLOCK16 and only to it");
  if (d->rows == 0 || d->k == 0) return B2VX_OK;
  B2VX_NEED(codes && scales && y, "null argument");
  B2VX_NEED(aligned(y, size_of(d->y_dtype)) && aligned(codes, 4) && aligned(tensor_scale, 4), "a pointer is not aligned");
  PerDevice* pd;
  b2vx_status st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  return launched(launch_fp4_dequantize(static_cast<const uint8_t*>(codes), static_cast<long long>(d->codes_pitch), static_cast<const uint8_t*>(scales),
                                        static_cast<long long>(d->scales_pitch), tensor_scale, d->format, static_cast<long long>(d->rows),
                                        static_cast<long long>(d->k), y, d->y_dtype, static_cast<long long>(d->y_stride), pd->sm_count, static_cast<cudaStream_t>(cuda_stream)),
                  err, err_len);
}

extern "C" b2vx_status b2vx_fp4_packed_scales_size_noalloc(int32_t format, uint64_t matrices, uint64_t n, int32_t gated, uint64_t k, size_t* bytes) {
  if (!bytes || !is_fp4(format) || matrices > static_cast<uint64_t>(kMaxExperts) || n > kMaxExtent || k > kMaxExtent || (gated != 0 && gated != 1)) return B2VX_INVALID_ARG;
  *bytes = packed_scale_bytes(static_cast<long long>(matrices), static_cast<long long>(n), gated, static_cast<long long>(k), format);
  return B2VX_OK;
}

extern "C" b2vx_status b2vx_fp4_pack_scales_noalloc(int32_t format, uint64_t matrices, uint64_t n, int32_t gated, uint64_t k, const void* scales, void* packed,
                                                    void* cuda_stream, char* err, size_t err_len) {
  size_t bytes = 0;
  B2VX_NEED(b2vx_fp4_packed_scales_size_noalloc(format, matrices, n, gated, k, &bytes) == B2VX_OK, "unknown format or an extent out of range");
  if (bytes == 0) return B2VX_OK;
  B2VX_NEED(scales && packed, "null argument");
  B2VX_NEED(aligned(packed, 16), "packed must be 16-byte aligned");
  PerDevice* pd;
  b2vx_status st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  return launched(launch_fp4_pack_scales(static_cast<const uint8_t*>(scales), format, static_cast<long long>(matrices), static_cast<long long>(n), gated,
                                         static_cast<long long>(k), static_cast<uint8_t*>(packed), pd->sm_count, static_cast<cudaStream_t>(cuda_stream)),
                  err, err_len);
}

extern "C" b2vx_status b2vx_linear_workspace_size_noalloc(const b2vx_linear_desc* d, size_t* bytes, char* err, size_t err_len) {
  b2vx_status st = check_linear(d, err, err_len);
  if (st != B2VX_OK) return st;
  B2VX_NEED(bytes, "null argument");
  *bytes = workspace_of(*d).total;
  return B2VX_OK;
}

extern "C" int32_t b2vx_linear_in_place_noalloc(const b2vx_linear_desc* d, const b2vx_linear_args* a) {
  return d && a && d->w_format == 0 && !a->row_index && aligned(a->x, 16) && d->x_stride % 8 == 0;
}

extern "C" b2vx_status b2vx_linear_noalloc(const b2vx_linear_desc* d, const b2vx_linear_args* a, void* cuda_stream, char* err, size_t err_len) {
  b2vx_status st = check_linear(d, err, err_len);
  if (st != B2VX_OK) return st;
  B2VX_NEED(a, "null argument");
  const bool fp4 = d->w_format != 0, block16 = d->w_format == B2VX_FP4_BLOCK16;
  B2VX_NEED((a->offsets != nullptr) == (d->experts != 0), "offsets belong to a product with experts and only to it");
  B2VX_NEED((a->x_scale != nullptr) == block16 && (a->w_scale != nullptr) == block16, "tensor scales belong to B2VX_FP4_BLOCK16 and only to it");
  B2VX_NEED(a->row_index || d->rows <= d->x_rows, "more rows than x has, and no row_index");
  if (d->rows == 0 || d->n == 0) return B2VX_OK;
  B2VX_NEED(a->w && a->y && (a->x || d->x_rows == 0) && (!fp4 || a->w_scales), "null argument");
  B2VX_NEED(aligned(a->w, 16) && aligned(a->w_scales, 16) && aligned(a->x, size_of(d->x_dtype)) && aligned(a->y, size_of(d->y_dtype)), "a pointer is not aligned");
  B2VX_NEED(aligned(a->bias, 4) && aligned(a->x_scale, 4) && aligned(a->w_scale, 4) && aligned(a->offsets, 4) && aligned(a->row_index, 4), "a pointer is not aligned");
  const Workspace ws = workspace_of(*d);
  const bool direct = b2vx_linear_in_place_noalloc(d, a);
  if (!direct) {
    B2VX_NEED(a->workspace && aligned(a->workspace, 256), "a 256-byte aligned workspace is needed");
    B2VX_NEED(a->workspace_bytes >= ws.total, "the workspace is too small");
  }
  PerDevice* pd;
  st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  if (device_status(false) != 0) return fail(err, err_len, B2VX_DEVICE_TIMEOUT, "an earlier product gave up waiting on a barrier; see b2vx_device_check_noalloc");
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  uint8_t* codes = static_cast<uint8_t*>(a->workspace);
  LinearArgs l = {};
  l.format = d->w_format; l.x_dtype = d->x_dtype; l.y_dtype = d->y_dtype;
  l.rows = static_cast<long long>(d->rows); l.n = static_cast<long long>(d->n); l.k = static_cast<long long>(d->k);
  l.experts = d->experts ? static_cast<int>(d->experts) : 1;
  l.gated = d->gated;
  l.w = a->w; l.w_scales = static_cast<const uint8_t*>(a->w_scales);
  l.x_scale = a->x_scale; l.w_scale = a->w_scale; l.bias = a->bias; l.offsets = a->offsets;
  l.y = a->y; l.y_stride = static_cast<long long>(d->y_stride);
  l.after_operand = !direct;
  l.status = pd->status; l.sm_count = pd->sm_count;
  cudaError_t e = cudaSuccess;
  if (fp4 && !a->row_index && linear_raw(l.format, l.rows, l.n, l.k, l.experts, l.gated, l.sm_count) && !a->offsets) {
    l.raw = true;
    l.after_operand = false;
    l.x = a->x; l.x_pitch = static_cast<long long>(d->x_stride * size_of(d->x_dtype));
  } else if (fp4) {
    QuantizeArgs q = {};
    q.x = a->x; q.x_dtype = d->x_dtype;
    q.x_stride = static_cast<long long>(d->x_stride); q.x_rows = static_cast<long long>(d->x_rows);
    q.rows = l.rows; q.k = l.k; q.row_index = a->row_index; q.tensor_scale = a->x_scale; q.format = d->w_format;
    q.codes = codes; q.codes_pitch = static_cast<long long>(ws.codes_pitch);
    q.scales = codes + ws.codes; q.scales_pitch = 0;
    q.offsets = a->offsets; q.experts = l.experts;
    q.bn = tile_rows(l.rows, l.experts, l.format);
    q.scale_tiles = static_cast<int>(expert_scale_tiles(l.rows, l.experts, q.bn));
    q.sm_count = pd->sm_count;
    e = launch_fp4_operand(q, codes + ws.codes + ws.scales, s);
    l.x = codes; l.x_pitch = static_cast<long long>(ws.codes_pitch); l.x_scales = q.scales;
  } else if (direct) {
    l.x = a->x; l.x_pitch = static_cast<long long>(d->x_stride) * 2;
  } else {
    e = launch_gather_rows(a->x, static_cast<long long>(d->x_stride), static_cast<long long>(d->x_rows), a->row_index, l.rows, l.k, codes, pd->sm_count, s);
    l.x = codes; l.x_pitch = static_cast<long long>(ws.codes_pitch);
  }
  if (e != cudaSuccess) return launched(e, err, err_len);
  const char* why = "";
  e = launch_linear(l, s, &why);
  if (e != cudaSuccess && *why) return fail(err, err_len, B2VX_CUDA_ERROR, why);
  return launched(e, err, err_len);
}

extern "C" b2vx_status b2vx_route_workspace_size_noalloc(const b2vx_route_desc* d, size_t* bytes, char* err, size_t err_len) {
  B2VX_NEED(d && bytes, "null argument");
  B2VX_NEED(d->experts >= 1 && d->experts <= static_cast<uint32_t>(kMaxExperts), "experts must be 1 to 1024");
  B2VX_NEED(d->top_k >= 1 && d->top_k <= static_cast<uint32_t>(kMaxTopK) && d->top_k <= d->experts, "top_k must be 1 to 32 and at most experts");
  B2VX_NEED(d->tokens <= kMaxExtent && d->tokens * d->top_k <= static_cast<uint64_t>(INT_MAX), "too many tokens");
  *bytes = round256(route_workspace_bytes(static_cast<long long>(d->tokens), static_cast<int>(d->experts)));
  return B2VX_OK;
}

extern "C" b2vx_status b2vx_route_noalloc(const b2vx_route_desc* d, const void* logits, int32_t* ids, float* weights, int32_t* offsets, int32_t* row_index,
                                          int32_t* slots, void* workspace, size_t workspace_bytes, void* cuda_stream, char* err, size_t err_len) {
  size_t need = 0;
  b2vx_status st = b2vx_route_workspace_size_noalloc(d, &need, err, err_len);
  if (st != B2VX_OK) return st;
  B2VX_NEED(is_float(d->logits_dtype), "logits must be float32, float16 or bfloat16");
  B2VX_NEED(d->normalize == 0 || d->normalize == 1, "normalize must be 0 or 1");
  B2VX_NEED(d->logits_stride >= d->experts && d->logits_stride <= kMaxStride, "logits_stride is smaller than a row or out of range");
  B2VX_NEED(offsets, "null argument");
  B2VX_NEED(aligned(offsets, 4) && aligned(ids, 4) && aligned(weights, 4) && aligned(row_index, 4) && aligned(slots, 4), "a pointer is not aligned");
  cudaStream_t s = static_cast<cudaStream_t>(cuda_stream);
  PerDevice* pd;
  if (d->tokens == 0) {   // no rows: every expert starts at 0
    st = device(&pd, err, err_len);
    if (st != B2VX_OK) return st;
    return launched(cudaMemsetAsync(offsets, 0, (d->experts + 1) * sizeof(int32_t), s), err, err_len);
  }
  B2VX_NEED(logits && ids && weights && row_index && slots, "null argument");
  B2VX_NEED(aligned(logits, size_of(d->logits_dtype)), "a pointer is not aligned");
  B2VX_NEED(need == 0 || (workspace && aligned(workspace, 256) && workspace_bytes >= need), "a 256-byte aligned workspace of the told size is needed");
  st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  return launched(launch_route(*d, logits, ids, weights, offsets, row_index, slots, workspace, pd->sm_count, s), err, err_len);
}

extern "C" b2vx_status b2vx_combine_noalloc(const b2vx_combine_desc* d, const void* z, const int32_t* slots, const float* weights, const void* residual,
                                            void* y, void* cuda_stream, char* err, size_t err_len) {
  B2VX_NEED(d, "null descriptor");
  B2VX_NEED(is_float(d->dtype), "z must be float32, float16 or bfloat16");
  B2VX_NEED(d->tokens <= kMaxExtent && d->n <= kMaxExtent && d->z_rows <= static_cast<uint64_t>(INT_MAX) && d->top_k <= 1024, "an extent is out of range");
  B2VX_NEED(d->z_stride >= d->n && d->y_stride >= d->n && (!residual || d->residual_stride >= d->n), "a stride is smaller than a row");
  B2VX_NEED(d->z_stride <= kMaxStride && d->y_stride <= kMaxStride && d->residual_stride <= kMaxStride, "a stride is out of range");
  if (d->tokens == 0 || d->n == 0) return B2VX_OK;
  B2VX_NEED(y && (d->top_k == 0 || (slots && weights)) && (z || d->z_rows == 0), "null argument");
  B2VX_NEED(aligned(z, size_of(d->dtype)) && aligned(y, size_of(d->dtype)) && aligned(residual, size_of(d->dtype)) && aligned(slots, 4) && aligned(weights, 4), "a pointer is not aligned");
  PerDevice* pd;
  b2vx_status st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  return launched(launch_combine(*d, z, slots, weights, residual, y, pd->sm_count, static_cast<cudaStream_t>(cuda_stream)), err, err_len);
}

extern "C" b2vx_status b2vx_device_check_noalloc(void* cuda_stream, char* err, size_t err_len) {
  PerDevice* pd;
  b2vx_status st = device(&pd, err, err_len);
  if (st != B2VX_OK) return st;
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(cuda_stream));
  if (e != cudaSuccess) return fail(err, err_len, B2VX_CUDA_ERROR, cudaGetErrorString(e));
  if (device_status(true) != 0) return fail(err, err_len, B2VX_DEVICE_TIMEOUT, "a product gave up waiting on a barrier; its output is incomplete");
  return B2VX_OK;
}
