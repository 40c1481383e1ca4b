// Routing of tokens to experts, and the weighted sum of the experts' rows.
//
// Routing is a counting sort whose keys are made on the way.  A token chooses an expert at most once, so for 32 tokens an expert's
// pairs are one 32-bit mask: the number of a pair among those of its 32 tokens is a population count, and neither it nor the
// order of the result depends on the order in which masks were put together.
//   choose   a warp per token: top_k largest logits, weights, masks [32-token block][expert]
//   count    a thread per expert: pairs before each block, and the experts' first rows
//   place    a thread per pair
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "experts.cuh"
#include "pdl.cuh"

namespace b2vx {
namespace {

constexpr int kBlockTokens = 32;

template <typename T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
// Order of floats as unsigned numbers; NaN counts as -infinity, -0 as 0.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (!(v == v)) v = -__int_as_float(0x7f800000);
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order(uint32_t u) { return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u); }

// PER: logits a lane holds (experts / 32, rounded up).
template <typename T, int PER>
__global__ void __launch_bounds__(256) choose_kernel(const T* logits, long long stride, int tokens, int experts, int top_k, int normalize, int32_t* ids,
                                                     float* weights, uint32_t* masks) {
  extern __shared__ uint32_t mask[];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int e = threadIdx.x; e < experts; e += 256) mask[e] = 0;
  __syncthreads();
  for (int i = warp; i < kBlockTokens; i += 8) {
    const int t = blockIdx.x * kBlockTokens + i;
    if (t >= tokens) break;
    const T* row = logits + t * stride;
    uint32_t key[PER];      // 0: taken, or not there (below -infinity's)
#pragma unroll
    for (int j = 0; j < PER; ++j) key[j] = j * 32 + lane < experts ? order_of(as_float(row[j * 32 + lane])) : 0u;
    uint32_t top = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) top = max(top, key[j]);
    const float most = from_order(__reduce_max_sync(0xffffffffu, top));
    const bool none = most == -__int_as_float(0x7f800000);
    float total = 0.0f;
    if (!normalize) {
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (key[j]) {
          const float v = from_order(key[j]);
          total += v == most ? 1.0f : expf(v - most);
        }
#pragma unroll
      for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
    }
    float mine = 0.0f, chosen = 0.0f;
    int id = 0;
    for (int r = 0; r < top_k; ++r) {
      uint32_t best = 0;
      int at = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (key[j] > best) { best = key[j]; at = j; }
      const uint32_t all = __reduce_max_sync(0xffffffffu, best);
      const uint32_t e = __reduce_min_sync(0xffffffffu, best == all ? static_cast<uint32_t>(at * 32 + lane) : 0xffffffffu);
#pragma unroll
      for (int j = 0; j < PER; ++j)
        if (static_cast<uint32_t>(j * 32 + lane) == e) key[j] = 0;
      const float v = from_order(all);
      const float w = none ? 0.0f : (v == most ? 1.0f : expf(v - most));
      chosen += w;
      if (lane == r) { mine = w; id = static_cast<int>(e); }
    }
    if (normalize) total = chosen;
    if (lane < top_k) {
      ids[static_cast<long long>(t) * top_k + lane] = id;
      weights[static_cast<long long>(t) * top_k + lane] = none ? 0.0f : mine / total;
      atomicOr(&mask[id], 1u << i);
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += 256) masks[static_cast<long long>(blockIdx.x) * experts + e] = mask[e];
}

__global__ void __launch_bounds__(1024) count_kernel(const uint32_t* masks, int blocks, int experts, int32_t* before, int32_t* offsets) {
  __shared__ int sum[1024];
  pdl_trigger();
  pdl_wait();
  const int e = threadIdx.x;
  int n = 0;
  if (e < experts)
    for (int b = 0; b < blocks; ++b) {
      before[static_cast<long long>(b) * experts + e] = n;
      n += __popc(masks[static_cast<long long>(b) * experts + e]);
    }
  sum[e] = n;
  __syncthreads();
  for (int d = 1; d < 1024; d <<= 1) {
    const int v = e >= d ? sum[e - d] : 0;
    __syncthreads();
    sum[e] += v;
    __syncthreads();
  }
  if (e < experts) offsets[e + 1] = sum[e];
  if (e == 0) offsets[0] = 0;
}

__global__ void __launch_bounds__(256) place_kernel(const int32_t* ids, const uint32_t* masks, const int32_t* before, const int32_t* offsets, long long pairs,
                                                    int experts, int top_k, int32_t* row_index, int32_t* slots) {
  pdl_trigger();
  pdl_wait();
  const long long step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < pairs; i += step) {
    const int t = static_cast<int>(i / top_k), e = ids[i];
    const long long at = static_cast<long long>(t / kBlockTokens) * experts + e;
    const int slot = offsets[e] + before[at] + __popc(masks[at] & ((1u << (t % kBlockTokens)) - 1u));
    slots[i] = slot;
    row_index[slot] = t;
  }
}

template <typename T>
cudaError_t choose(const b2vx_route_desc& d, const void* logits, int32_t* ids, float* weights, uint32_t* masks, int blocks, cudaStream_t s) {
  const int per = (static_cast<int>(d.experts) + 31) / 32;
  auto* kernel = per <= 2 ? choose_kernel<T, 2> : per <= 4 ? choose_kernel<T, 4> : per <= 8 ? choose_kernel<T, 8> : per <= 16 ? choose_kernel<T, 16> : choose_kernel<T, 32>;
  return launch_pdl(kernel, dim3(blocks), dim3(256), d.experts * 4, s, static_cast<const T*>(logits), static_cast<long long>(d.logits_stride),
                    static_cast<int>(d.tokens), static_cast<int>(d.experts), static_cast<int>(d.top_k), d.normalize, ids, weights, masks);
}

// A thread owns eight neighbouring columns of a token (VEC: 16-byte loads) or one.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(const T* z, long long z_stride, long long z_rows, const int32_t* slots, const float* weights,
                                                      const T* residual, long long residual_stride, T* y, long long y_stride, long long tokens, int top_k,
                                                      int pieces) {
  constexpr int N = VEC ? 16 / sizeof(T) : 1;
  pdl_trigger();
  pdl_wait();
  const long long total = tokens * pieces, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const long long t = i / pieces;
    const int c = static_cast<int>(i - t * pieces) * N;
    float acc[N];
#pragma unroll
    for (int n = 0; n < N; ++n) acc[n] = 0.0f;
    alignas(16) T v[N];
    for (int j = 0; j < top_k; ++j) {
      const int slot = __ldg(slots + t * top_k + j);
      if (slot < 0 || slot >= z_rows) continue;
      const float w = __ldg(weights + t * top_k + j);
      const T* from = z + slot * z_stride + c;
      if constexpr (VEC) *reinterpret_cast<uint4*>(v) = __ldg(reinterpret_cast<const uint4*>(from));
      else v[0] = *from;
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n] = fmaf(w, as_float(v[n]), acc[n]);
    }
    if (residual) {
      const T* from = residual + t * residual_stride + c;
      if constexpr (VEC) *reinterpret_cast<uint4*>(v) = *reinterpret_cast<const uint4*>(from);
      else v[0] = *from;
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n] += as_float(v[n]);
    }
#pragma unroll
    for (int n = 0; n < N; ++n) {
      if constexpr (sizeof(T) == 4) v[n] = acc[n];
      else if constexpr (std::is_same<T, __half>::value) v[n] = __float2half_rn(acc[n]);
      else v[n] = __float2bfloat16_rn(acc[n]);
    }
    T* to = y + t * y_stride + c;
    if constexpr (VEC) *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(v);
    else *to = v[0];
  }
}

template <typename T>
cudaError_t combine(const b2vx_combine_desc& d, const void* z, const int32_t* slots, const float* weights, const void* residual, void* y, cudaStream_t s) {
  constexpr uint64_t N = 16 / sizeof(T);
  const bool vec = d.n % N == 0 && d.z_stride % N == 0 && d.y_stride % N == 0 && reinterpret_cast<uintptr_t>(z) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 16 == 0 && (!residual || (d.residual_stride % N == 0 && reinterpret_cast<uintptr_t>(residual) % 16 == 0));
  const int pieces = static_cast<int>(vec ? d.n / N : d.n);
  const long long total = static_cast<long long>(d.tokens) * pieces;
  const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>((total + 255) / 256, 148 * 8)));
  auto* kernel = vec ? combine_kernel<T, true> : combine_kernel<T, false>;
  return launch_pdl(kernel, dim3(grid), dim3(256), 0, s, static_cast<const T*>(z), static_cast<long long>(d.z_stride), static_cast<long long>(d.z_rows), slots,
                    weights, static_cast<const T*>(residual), static_cast<long long>(d.residual_stride), static_cast<T*>(y),
                    static_cast<long long>(d.y_stride), static_cast<long long>(d.tokens), static_cast<int>(d.top_k), pieces);
}

long long route_blocks(long long tokens) { return (tokens + kBlockTokens - 1) / kBlockTokens; }

}  // namespace

size_t route_workspace_bytes(long long tokens, int experts) { return static_cast<size_t>(route_blocks(tokens)) * experts * 8; }

cudaError_t launch_route(const b2vx_route_desc& d, const void* logits, int32_t* ids, float* weights, int32_t* offsets, int32_t* row_index,
                         int32_t* slots, void* workspace, cudaStream_t s) {
  const int blocks = static_cast<int>(route_blocks(static_cast<long long>(d.tokens))), experts = static_cast<int>(d.experts);
  uint32_t* masks = static_cast<uint32_t*>(workspace);
  int32_t* before = reinterpret_cast<int32_t*>(masks + static_cast<size_t>(blocks) * experts);
  cudaError_t e;
  if (d.logits_dtype == B2VX_DT_FLOAT32) e = choose<float>(d, logits, ids, weights, masks, blocks, s);
  else if (d.logits_dtype == B2VX_DT_FLOAT16) e = choose<__half>(d, logits, ids, weights, masks, blocks, s);
  else e = choose<__nv_bfloat16>(d, logits, ids, weights, masks, blocks, s);
  if (e != cudaSuccess) return e;
  e = launch_pdl(count_kernel, dim3(1), dim3(1024), 0, s, static_cast<const uint32_t*>(masks), blocks, experts, before, offsets);
  if (e != cudaSuccess) return e;
  const long long pairs = static_cast<long long>(d.tokens) * d.top_k;
  const int grid = static_cast<int>(std::min<long long>((pairs + 255) / 256, 148 * 8));
  return launch_pdl(place_kernel, dim3(grid), dim3(256), 0, s, static_cast<const int32_t*>(ids), static_cast<const uint32_t*>(masks), static_cast<const int32_t*>(before),
                    static_cast<const int32_t*>(offsets), pairs, experts, static_cast<int>(d.top_k), row_index, slots);
}

cudaError_t launch_combine(const b2vx_combine_desc& d, const void* z, const int32_t* slots, const float* weights, const void* residual, void* y,
                           cudaStream_t s) {
  if (d.dtype == B2VX_DT_FLOAT32) return combine<float>(d, z, slots, weights, residual, y, s);
  if (d.dtype == B2VX_DT_FLOAT16) return combine<__half>(d, z, slots, weights, residual, y, s);
  return combine<__nv_bfloat16>(d, z, slots, weights, residual, y, s);
}

}  // namespace b2vx
