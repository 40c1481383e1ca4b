// Routing of tokens to experts, and the weighted sum of the experts' rows.
//
// Routing is a counting sort whose keys are made on the way.  A token chooses an expert at most once, so for 32 tokens an expert's
// pairs are one 32-bit mask: the number of a pair among those of its 32 tokens is a population count, and neither it nor the
// order of the result depends on the order in which masks were put together.
// A warp chooses for one token; 32 tokens to a block.  Up to 128 tokens one block does everything (16 tokens, 8 of 128 experts: one
// launch, 3.2 us, instead of three); else
//   choose   ids, weights, masks [32-token block][expert]
//   before   a lane per expert, the blocks shared by 32 warps: pairs before each block, pairs of each expert
//   place    first rows of the experts from those, then a thread per pair
// Bound by latency, of the launches in the end: the 4 MB of logits of 8192 tokens and 256 experts are a microsecond.
#include <algorithm>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "block_linear.cuh"
#include "experts.cuh"
#include "pdl.cuh"

namespace b2vx {
namespace {

constexpr int kBlockTokens = 32;
constexpr int kOneBlockTokens = 128;

template <typename T>
__device__ __forceinline__ float as_float(T v) {
  if constexpr (sizeof(T) == 4) return v;
  else if constexpr (std::is_same<T, __half>::value) return __half2float(v);
  else return __bfloat162float(v);
}
// Order of floats as unsigned numbers; NaN counts as -infinity, -0 as 0.  A key above 0 stands for a logit that can be chosen: of 32-bit
// logits their order, of 16-bit ones their order in the upper half and 65535 minus the expert in the lower, so that one maximum
// finds both the largest logit and, among equals, the lowest expert.
__device__ __forceinline__ uint32_t order_of(float v) {
  if (!(v == v)) v = -__int_as_float(0x7f800000);
  const uint32_t b = __float_as_uint(v + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
template <typename T>
__device__ __forceinline__ uint32_t key_of(T v, int e) {
  if constexpr (sizeof(T) == 4) {
    return order_of(v);
  } else if constexpr (std::is_same<T, __half>::value) {
    const float f = as_float(v) + 0.0f;
    const uint32_t b = f == f ? __half_as_ushort(__float2half_rn(f)) : 0xfc00u;   // exact
    return ((b & 0x8000u ? ~b : b | 0x8000u) << 16) | (0xffffu - e);
  } else {
    return (order_of(as_float(v)) & 0xffff0000u) | (0xffffu - e);                 // the lower half of a bfloat16's order is all ones or zeros
  }
}
template <typename T>
__device__ __forceinline__ float value_of(uint32_t key) {
  if constexpr (std::is_same<T, __half>::value) {
    const uint32_t u = key >> 16;
    return __half2float(__ushort_as_half(static_cast<uint16_t>(u & 0x8000u ? u & 0x7fffu : ~u)));
  } else {
    const uint32_t u = sizeof(T) == 4 ? key : key & 0xffff0000u;
    return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : (sizeof(T) == 4 ? ~u : ~u & 0xffff0000u));
  }
}

// One token by one warp.  PER: logits a lane holds (experts / 32, rounded up).  Sets bit `bit` of the chosen experts' masks.
template <typename T, int PER>
__device__ __forceinline__ void choose(const T* row, long long t, int experts, int top_k, int normalize, int lane, int bit, int32_t* ids, float* weights,
                                       uint32_t* mask) {
  uint32_t key[PER];      // 0: taken, or not there
#pragma unroll
  for (int j = 0; j < PER; ++j) key[j] = j * 32 + lane < experts ? key_of(row[j * 32 + lane], j * 32 + lane) : 0u;
  uint32_t top = 0;
#pragma unroll
  for (int j = 0; j < PER; ++j) top = max(top, key[j]);
  const float most = value_of<T>(__reduce_max_sync(0xffffffffu, top));
  const bool none = most == -__int_as_float(0x7f800000);
  float total = 0.0f;
  if (!normalize) {
#pragma unroll
    for (int j = 0; j < PER; ++j)
      if (key[j]) {
        const float v = value_of<T>(key[j]);
        total += v == most ? 1.0f : expf(v - most);
      }
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  }
  uint32_t mine = 0;
  int id = 0;
  for (int r = 0; r < top_k; ++r) {
    uint32_t best = 0;
#pragma unroll
    for (int j = 0; j < PER; ++j) best = max(best, key[j]);
    const uint32_t all = __reduce_max_sync(0xffffffffu, best);
    uint32_t e;
    if constexpr (sizeof(T) == 2) {
      e = 0xffffu - (all & 0xffffu);
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = key[j] == all ? 0u : key[j];
    } else {
      uint32_t at = 0xffffffffu;
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) at = key[j] == all ? static_cast<uint32_t>(j * 32 + lane) : at;
      e = __reduce_min_sync(0xffffffffu, at);
#pragma unroll
      for (int j = 0; j < PER; ++j) key[j] = static_cast<uint32_t>(j * 32 + lane) == e ? 0u : key[j];
    }
    if (lane == r) { mine = all; id = static_cast<int>(e); }
  }
  const float v = value_of<T>(mine);
  const float w = none || lane >= top_k ? 0.0f : (v == most ? 1.0f : expf(v - most));
  if (normalize) {
    total = w;
#pragma unroll
    for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  }
  if (lane < top_k) {
    ids[t * top_k + lane] = id;
    weights[t * top_k + lane] = none ? 0.0f : w / total;
    atomicOr(&mask[id], 1u << bit);
  }
}

// Sums of all numbers before each thread's, over the block's 1024 threads.
__device__ __forceinline__ int sum_before(int n, int* warp_sums, int lane, int warp) {
  int sum = n;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, sum, d);
    if (lane >= d) sum += up;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    const int mine = warp_sums[lane];
    int all = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, all, d);
      if (lane >= d) all += up;
    }
    warp_sums[lane] = all - mine;
  }
  __syncthreads();
  return sum - n + warp_sums[warp];
}

// Everything, for up to kOneBlockTokens tokens.
template <typename T, int PER>
__global__ void __launch_bounds__(1024) route_kernel(const T* logits, long long stride, int tokens, int experts, int top_k, int normalize, int32_t* ids,
                                                     float* weights, int32_t* offsets, int32_t* row_index, int32_t* slots) {
  extern __shared__ uint32_t mask[];                    // [tokens / 32][experts], then first rows [experts]
  __shared__ int warp_sums[32];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, blocks = (tokens + kBlockTokens - 1) / kBlockTokens;
  int* first = reinterpret_cast<int*>(mask + blocks * experts);
  for (int i = threadIdx.x; i < blocks * experts; i += 1024) mask[i] = 0;
  __syncthreads();
  for (int t = warp; t < tokens; t += 32) choose<T, PER>(logits + t * stride, t, experts, top_k, normalize, lane, t & 31, ids, weights, mask + (t >> 5) * experts);
  __syncthreads();
  const int e = threadIdx.x;
  int n = 0;
  if (e < experts)
    for (int b = 0; b < blocks; ++b) n += __popc(mask[b * experts + e]);
  const int before = sum_before(n, warp_sums, lane, warp);
  if (e < experts) {
    first[e] = before;
    offsets[e] = before;
    if (e == experts - 1) offsets[experts] = before + n;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < tokens * top_k; i += 1024) {
    const int t = i / top_k, id = ids[i], block = t >> 5;
    int slot = first[id] + __popc(mask[block * experts + id] & ((1u << (t & 31)) - 1u));
    for (int b = 0; b < block; ++b) slot += __popc(mask[b * experts + id]);
    slots[i] = slot;
    row_index[slot] = t;
  }
}

template <typename T, int PER>
__global__ void __launch_bounds__(1024, PER <= 8 ? 2 : 1) choose_kernel(const T* logits, long long stride, int tokens, int experts, int top_k, int normalize, int32_t* ids,
                                                      float* weights, uint32_t* masks) {
  extern __shared__ uint32_t mask[];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * kBlockTokens + warp;
  for (int e = threadIdx.x; e < experts; e += 1024) mask[e] = 0;
  __syncthreads();
  if (t < tokens) choose<T, PER>(logits + t * stride, t, experts, top_k, normalize, lane, warp, ids, weights, mask);
  __syncthreads();
  for (int e = threadIdx.x; e < experts; e += 1024) masks[static_cast<long long>(blockIdx.x) * experts + e] = mask[e];
}

__global__ void __launch_bounds__(1024) before_kernel(const uint32_t* masks, int blocks, int experts, int32_t* before, int32_t* totals) {
  __shared__ int sums[32][33];
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
  const int share = (blocks + 31) / 32, b0 = warp * share, b1 = min(blocks, b0 + share);
  int n = 0;
  if (e < experts)
#pragma unroll 8
    for (int b = b0; b < b1; ++b) n += __popc(masks[static_cast<long long>(b) * experts + e]);
  sums[warp][lane] = n;
  __syncthreads();
  int sum = 0;
  for (int w = 0; w < warp; ++w) sum += sums[w][lane];
  if (e >= experts) return;
#pragma unroll 8
  for (int b = b0; b < b1; ++b) {
    before[static_cast<long long>(b) * experts + e] = sum;
    sum += __popc(masks[static_cast<long long>(b) * experts + e]);
  }
  if (warp == 31) totals[e] = sum;
}

__global__ void __launch_bounds__(1024) place_kernel(const int32_t* ids, const uint32_t* masks, const int32_t* before, const int32_t* totals, int pairs,
                                                     int experts, int top_k, int32_t* offsets, int32_t* row_index, int32_t* slots) {
  __shared__ int first[kMaxExperts], warp_sums[32];
  pdl_trigger();
  pdl_wait();
  const int e = threadIdx.x, n = e < experts ? totals[e] : 0;
  const int sum = sum_before(n, warp_sums, threadIdx.x & 31, threadIdx.x >> 5);
  first[e] = sum;
  if (blockIdx.x == 0 && e < experts) {
    offsets[e] = sum;
    if (e == experts - 1) offsets[experts] = sum + n;
  }
  __syncthreads();
  for (long long i = static_cast<long long>(blockIdx.x) * 1024 + threadIdx.x; i < pairs; i += static_cast<long long>(gridDim.x) * 1024) {
    const int t = static_cast<int>(i) / top_k, id = ids[i];
    const long long at = static_cast<long long>(t / kBlockTokens) * experts + id;
    const int slot = first[id] + before[at] + __popc(masks[at] & ((1u << (t % kBlockTokens)) - 1u));
    slots[i] = slot;
    row_index[slot] = t;
  }
}

template <typename T, int PER>
cudaError_t route(const b2vx_route_desc& d, const T* logits, int32_t* ids, float* weights, int32_t* offsets, int32_t* row_index, int32_t* slots,
                  void* workspace, int sm_count, cudaStream_t s) {
  const int tokens = static_cast<int>(d.tokens), experts = static_cast<int>(d.experts), top_k = static_cast<int>(d.top_k);
  const int blocks = (tokens + kBlockTokens - 1) / kBlockTokens;
  const long long stride = static_cast<long long>(d.logits_stride);
  if (tokens <= kOneBlockTokens)
    return launch_pdl(route_kernel<T, PER>, dim3(1), dim3(1024), (blocks + 1) * experts * 4, s, logits, stride, tokens, experts, top_k, d.normalize, ids, weights,
                      offsets, row_index, slots);
  uint32_t* masks = static_cast<uint32_t*>(workspace);
  int32_t* before = reinterpret_cast<int32_t*>(masks + static_cast<size_t>(blocks) * experts);
  int32_t* totals = before + static_cast<size_t>(blocks) * experts;
  cudaError_t e = launch_pdl(choose_kernel<T, PER>, dim3(blocks), dim3(1024), experts * 4, s, logits, stride, tokens, experts, top_k, d.normalize, ids, weights, masks);
  if (e != cudaSuccess) return e;
  e = launch_pdl(before_kernel, dim3((experts + 31) / 32), dim3(1024), 0, s, static_cast<const uint32_t*>(masks), blocks, experts, before, totals);
  if (e != cudaSuccess) return e;
  const int pairs = tokens * top_k;      // 1 to 2^31 - 1: no sum with it in 32 bits
  return launch_pdl(place_kernel, dim3(std::min((pairs - 1) / 1024 + 1, sm_count * 2)), dim3(1024), 0, s, static_cast<const int32_t*>(ids),
                    static_cast<const uint32_t*>(masks), static_cast<const int32_t*>(before), static_cast<const int32_t*>(totals), pairs, experts, top_k, offsets,
                    row_index, slots);
}
template <typename T>
cudaError_t route_typed(const b2vx_route_desc& d, const void* logits, int32_t* ids, float* weights, int32_t* offsets, int32_t* row_index, int32_t* slots,
                        void* workspace, int sm_count, cudaStream_t s) {
  const T* z = static_cast<const T*>(logits);
  if (d.experts <= 64) return route<T, 2>(d, z, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
  if (d.experts <= 128) return route<T, 4>(d, z, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
  if (d.experts <= 256) return route<T, 8>(d, z, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
  if (d.experts <= 512) return route<T, 16>(d, z, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
  return route<T, 32>(d, z, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
}

// The sum is bound by memory: z once.  blockDim.x threads share a token, each with 16 bytes of neighbouring columns (VEC) or one column at a
// time; four rows of z are asked for before the first is added.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) combine_kernel(const T* z, long long z_stride, int z_rows, const int32_t* slots, const float* weights,
                                                      const T* residual, long long residual_stride, T* y, long long y_stride, int tokens, int top_k,
                                                      int pieces) {
  constexpr int N = VEC ? 16 / sizeof(T) : 1, U = 4;
  struct alignas(VEC ? 16 : sizeof(T)) Piece {
    T v[N];
  };
  pdl_trigger();
  pdl_wait();
  for (int t = blockIdx.x * blockDim.y + threadIdx.y; t < tokens; t += gridDim.x * blockDim.y) {
    const int32_t* slot_row = slots + static_cast<long long>(t) * top_k;
    const float* weight_row = weights + static_cast<long long>(t) * top_k;
    for (int p = threadIdx.x; p < pieces; p += blockDim.x) {
      const long long c = static_cast<long long>(p) * N;
      Piece r;
      if (residual) r = *reinterpret_cast<const Piece*>(residual + t * residual_stride + c);
      float acc[N];
#pragma unroll
      for (int n = 0; n < N; ++n) acc[n] = 0.0f;
      for (int j0 = 0; j0 < top_k; j0 += U) {
        Piece v[U];
        float w[U];
        bool there[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int slot = j0 + u < top_k ? __ldg(slot_row + j0 + u) : -1;
          there[u] = slot >= 0 && slot < z_rows;
          w[u] = there[u] ? __ldg(weight_row + j0 + u) : 0.0f;
          if (there[u]) {
            const T* from = z + slot * z_stride + c;
            if constexpr (VEC) *reinterpret_cast<uint4*>(&v[u]) = __ldg(reinterpret_cast<const uint4*>(from));
            else v[u].v[0] = *from;
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (there[u])
#pragma unroll
            for (int n = 0; n < N; ++n) acc[n] = fmaf(w[u], as_float(v[u].v[n]), acc[n]);
      }
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const float sum = residual ? acc[n] + as_float(r.v[n]) : acc[n];
        if constexpr (sizeof(T) == 4) r.v[n] = sum;
        else if constexpr (std::is_same<T, __half>::value) r.v[n] = __float2half_rn(sum);
        else r.v[n] = __float2bfloat16_rn(sum);
      }
      *reinterpret_cast<Piece*>(y + t * y_stride + c) = r;
    }
  }
}

template <typename T>
cudaError_t combine(const b2vx_combine_desc& d, const void* z, const int32_t* slots, const float* weights, const void* residual, void* y, int sm_count,
                    cudaStream_t s) {
  constexpr uint64_t N = 16 / sizeof(T);
  const bool vec = d.n % N == 0 && d.z_stride % N == 0 && d.y_stride % N == 0 && reinterpret_cast<uintptr_t>(z) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(y) % 16 == 0 && (!residual || (d.residual_stride % N == 0 && reinterpret_cast<uintptr_t>(residual) % 16 == 0));
  const int pieces = static_cast<int>(vec ? d.n / N : d.n), tokens = static_cast<int>(d.tokens);
  int x = 8;                                     // threads to a token
  while (x < 256 && x < pieces) x *= 2;
  const int y_dim = 256 / x, grid = std::min((tokens + y_dim - 1) / y_dim, sm_count * 8);
  auto* kernel = vec ? combine_kernel<T, true> : combine_kernel<T, false>;
  return launch_pdl(kernel, dim3(grid), dim3(x, y_dim), 0, s, static_cast<const T*>(z), static_cast<long long>(d.z_stride), static_cast<int>(d.z_rows), slots,
                    weights, static_cast<const T*>(residual), static_cast<long long>(d.residual_stride), static_cast<T*>(y),
                    static_cast<long long>(d.y_stride), tokens, static_cast<int>(d.top_k), pieces);
}

}  // namespace

size_t route_workspace_bytes(long long tokens, int experts) {
  const size_t blocks = static_cast<size_t>((tokens + kBlockTokens - 1) / kBlockTokens);
  return tokens <= kOneBlockTokens ? 0 : (2 * blocks + 1) * experts * 4;
}

cudaError_t launch_route(const b2vx_route_desc& d, const void* logits, int32_t* ids, float* weights, int32_t* offsets, int32_t* row_index,
                         int32_t* slots, void* workspace, int sm_count, cudaStream_t s) {
  if (d.logits_dtype == B2VX_DT_FLOAT32) return route_typed<float>(d, logits, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
  if (d.logits_dtype == B2VX_DT_FLOAT16) return route_typed<__half>(d, logits, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
  return route_typed<__nv_bfloat16>(d, logits, ids, weights, offsets, row_index, slots, workspace, sm_count, s);
}

cudaError_t launch_combine(const b2vx_combine_desc& d, const void* z, const int32_t* slots, const float* weights, const void* residual, void* y,
                           int sm_count, cudaStream_t s) {
  if (d.dtype == B2VX_DT_FLOAT32) return combine<float>(d, z, slots, weights, residual, y, sm_count, s);
  if (d.dtype == B2VX_DT_FLOAT16) return combine<__half>(d, z, slots, weights, residual, y, sm_count, s);
  return combine<__nv_bfloat16>(d, z, slots, weights, residual, y, sm_count, s);
}

}  // namespace b2vx
