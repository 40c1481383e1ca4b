// Launchers of routing and of the weighted sum of expert rows (experts.cu), for device_ops.cu.
#ifndef B2VX_EXPERTS_CUH_
#define B2VX_EXPERTS_CUH_

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "b2vx.h"

namespace b2vx {

constexpr int kMaxTopK = 32;   // of a token: a lane for each

size_t route_workspace_bytes(long long tokens, int experts);
cudaError_t launch_route(const b2vx_route_desc& d, const void* logits, int32_t* ids, float* weights, int32_t* offsets, int32_t* row_index,
                         int32_t* slots, void* workspace, int sm_count, cudaStream_t s);
cudaError_t launch_combine(const b2vx_combine_desc& d, const void* z, const int32_t* slots, const float* weights, const void* residual, void* y,
                           int sm_count, cudaStream_t s);

}  // namespace b2vx
#endif  // B2VX_EXPERTS_CUH_
