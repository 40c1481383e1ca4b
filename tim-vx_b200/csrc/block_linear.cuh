// What the host entry points (device_ops.cu) and the kernels of the operators on device tensors share: formats, layouts, launchers.
#ifndef B2VX_BLOCK_LINEAR_CUH_
#define B2VX_BLOCK_LINEAR_CUH_

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

#include "b2vx.h"

namespace b2vx {

// Columns that share a scale.
__host__ __device__ constexpr int fp4_block(int format) { return format == B2VX_FP4_BLOCK16 ? 16 : 32; }

// Scales of a product's operand ("packed"): tiles of 128 rows x 4 blocks, 512 bytes each, which is the form the tensor pipe takes
// its scales in.  Row r's four bytes of a tile lie at (r % 32) * 16 + (r / 32) * 4: a copy of the tile into tensor memory puts rows
// 32 c .. 32 c + 31 into its column c.  Order: [pipeline stage of 256 columns][128-row tile][tile of the stage], so that what a stage
// needs of neighbouring row tiles is one piece of memory.
constexpr int kScaleTile = 512;
constexpr int kStageBytes = 128;                       // bytes of K per row and pipeline stage
constexpr int kMaxExperts = 1024;
__host__ __device__ constexpr int scale_words_per_stage(int format) { return 256 / (4 * fp4_block(format)); }   // 2 or 4
__host__ __device__ inline long long scale_words(long long k, int format) {
  return (k + 255) / 256 * scale_words_per_stage(format);
}
// 128-row tiles of a matrix with n features; those of a gated one hold 64 gate and 64 up rows, in turn eight of each.
__host__ __device__ inline long long weight_tiles(long long n, int gated) { return gated ? (n + 63) / 64 : (n + 127) / 128; }
__host__ __device__ inline size_t packed_scale_bytes(long long matrices, long long n, int gated, long long k, int format) {
  return static_cast<size_t>(matrices) * weight_tiles(n, gated) * scale_words(k, format) * kScaleTile;
}
// Rows of x in a tile of a product.  Up to 64 rows to a group: narrow tiles of one CTA.  More: tiles of two CTAs, as wide as leaves
// tensor memory for two accumulators and two slots of scales (twice as many of block16).
inline int tile_rows(long long rows, int experts, int format) {
  const long long groups = rows < experts ? rows : experts, mean = groups ? (rows + groups - 1) / groups : 0;
  return mean <= 64 ? 64 : (mean <= 128 ? 128 : (format == B2VX_FP4_BLOCK16 ? 192 : 224));
}
// Rows of each tile of a group: its rows in even shares.
__host__ __device__ inline int rows_of_tile(int count, int bn) {
  const int tiles = (count + bn - 1) / bn;
  return tiles ? ((count + tiles - 1) / tiles + 31) / 32 * 32 : 32;
}
// Packed scales of x: every tile's rows start on a scale tile of their own (an instruction takes its scales from an even column of tensor
// memory on, so 32-row steps inside a scale tile would not do).  Group e, whose first row is lo, starts at scale tile
// expert_scale_tile(lo, e); since floor(a + b) >= floor(a) + floor(b), the tiles of group e end where group e + 1 may start.
__host__ __device__ inline int expert_scale_tile(int lo, int e, int bn) { return (lo / bn + e) * ((bn + 127) / 128); }
__host__ __device__ inline long long expert_scale_tiles(long long rows, long long experts, int bn) { return (rows / bn + experts) * ((bn + 127) / 128); }

struct QuantizeArgs {
  const void* x;
  int x_dtype;
  long long x_stride;          // elements
  long long x_rows;            // rows of x (bound of row_index)
  long long rows, k;
  const int32_t* row_index;    // or null
  const float* tensor_scale;   // block16
  int format;
  uint8_t* codes;
  long long codes_pitch;       // bytes
  uint8_t* scales;
  long long scales_pitch;      // bytes; 0: packed, for a product
  const int32_t* offsets;      // packed: the groups, or null for one group of all rows
  int experts;
  int bn;                      // packed: rows of the product's tiles
  int scale_tiles;             // packed: expert_scale_tiles
  int sm_count;
};
cudaError_t launch_fp4_quantize(const QuantizeArgs& a, cudaStream_t s);
// The operand x of a product (packed scales; codes_pitch is k / 2, a multiple of 16): quantized in one step, or each row of x once and then
// copied to where row_index wants it.  `between`: fp4_twice_bytes bytes for that, aligned to 16.
size_t fp4_twice_bytes(const QuantizeArgs& a);
cudaError_t launch_fp4_operand(const QuantizeArgs& a, void* between, cudaStream_t s);
cudaError_t launch_fp4_dequantize(const uint8_t* codes, long long codes_pitch, const uint8_t* scales, long long scales_pitch,
                                  const float* tensor_scale, int format, long long rows, long long k, void* y, int y_dtype,
                                  long long y_stride, int sm_count, cudaStream_t s);
cudaError_t launch_fp4_pack_scales(const uint8_t* scales, int format, long long matrices, long long n, int gated, long long k, uint8_t* packed, int sm_count,
                                   cudaStream_t s);
// rows of 16-bit numbers, gathered: y[i] = x[row_index[i]] (zeros where the index is out of range), K contiguous in y
cudaError_t launch_gather_rows(const void* x, long long x_stride, long long x_rows, const int32_t* row_index, long long rows, long long k,
                               void* y, int sm_count, cudaStream_t s);

struct LinearArgs {
  int format;                  // 0: 16-bit numbers of x_dtype, else B2VX_FP4_*
  int x_dtype, y_dtype;
  long long rows;              // rows of the operand x and of y
  long long n, k;
  int experts;                 // groups; 1 with offsets == null: one product
  int gated;
  const void* x;               // codes or 16-bit numbers
  long long x_pitch;           // bytes
  const uint8_t* x_scales;     // packed
  const void* w;
  const uint8_t* w_scales;     // packed
  const float* x_scale;        // tensor scales, or null
  const float* w_scale;
  const float* bias;
  const int32_t* offsets;
  void* y;
  long long y_stride;          // elements
  bool raw;                    // x is rows of x_dtype numbers, x_pitch apart, that the product quantizes itself (linear_raw)
  bool after_operand;          // the kernel before this one in the stream made x and x_scales, and waited for all before it
  int* status;
  int sm_count;
};
cudaError_t launch_linear(const LinearArgs& a, cudaStream_t s, const char** why);
// Whether the product quantizes x itself: one matrix, up to 16 rows, a cluster for every tile, little to quantize for each CTA.
bool linear_raw(int format, long long rows, long long n, long long k, int experts, int gated, int sm_count);

}  // namespace b2vx
#endif  // B2VX_BLOCK_LINEAR_CUH_
