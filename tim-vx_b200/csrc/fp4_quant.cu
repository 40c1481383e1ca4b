// Rows of numbers to 4-bit block floating point and back, packing of scales, gathering of rows.
//
// Quantization reads every number once and writes half a byte and a scale's share for it: 8192 x 8192 bfloat16 numbers to block32 in 34 us,
// to block16 in 38 (26 are the bytes'), 32-bit numbers in 49 (46).  From 16 bits instructions bind, 65 - 68 % of the issue slots at 55 % of the warps; from 32 bits memory.
// Sixteen columns a lane: a block of block16, so that its scale, some forty instructions, is worked out once, or half a block of block32.
#include <algorithm>
#include <climits>

#include "block_linear.cuh"
#include "fp4.cuh"
#include "pdl.cuh"

namespace b2vx {
namespace {

constexpr int kWarps = 8;
// Blocks of a quantization kernel an SM: what 48 registers a thread leave, or 64 where 32-bit numbers would not fit beside block16's
// rounding (8192 x 8192 to block16: 50 us with four, 58 with five).  8192 x 8192 bfloat16 numbers by rows with five / four: to block32 34 / 42 us, to
// block16 38 / 42.  As a product's operand, where the place of the scales takes registers too, block16 wants four at every number of rows: 24 / 512 / 2048 / 8192 rows
// of 8192 columns and a product with 128 features 6.6 / 17.5 / 29.0 / 73.8 us with five, 6.5 / 16.3 / 24.8 / 62.4 with four.
constexpr int quantize_blocks(int format, size_t elem, bool packed) { return format == B2VX_FP4_BLOCK16 && (elem == 4 || packed) ? 4 : 5; }
// Rows that several rows of an operand refer to (a token's, for each of its experts) are quantized once and then copied, where that saves
// more than the second launch costs: measured at 8192 rows of 1408 columns taken four times each.
constexpr long long kTwiceElements = 1 << 22;
constexpr int kChunk = 512;   // columns of a warp per step, two k-blocks of the products

// Where the words of a row's scales lie in the first k-block's scale tiles of a product's operand; null: the row belongs to no group.
// Groups follow the product's rule, offsets cut to rising values among the rows: the first offset behind the row ends its group, and the largest of
// those before that one (the last, where they rise) begins it.
template <int FORMAT>
__device__ __forceinline__ uint8_t* packed_place(const QuantizeArgs& a, uint32_t row, int lane) {
  int e = 0, lo = 0, count = static_cast<int>(a.rows);
  if (a.offsets) {
    // of the offsets behind the first: the first that is behind the row, and how many are not
    int end = a.experts + 1, begun = 0;
    const int begin = a.offsets[0];
    for (int top = a.experts - lane; top > 0; top -= 4 * 32) {
      int v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) v[u] = top - u * 32 > 0 ? a.offsets[top - u * 32] : INT_MIN;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        if (v[u] > static_cast<int>(row)) {
          end = top - u * 32;
        } else {
          lo = max(lo, v[u]);
          begun += top - u * 32 > 0;
        }
      }
    }
    end = __reduce_min_sync(0xffffffffu, end);
    begun = __reduce_add_sync(0xffffffffu, begun);
    lo = __reduce_max_sync(0xffffffffu, lo);
    if (begin > static_cast<int>(row) || end > a.experts) return nullptr;
    if (begun != end - 1) {                                  // some behind the end are lower again
      lo = 0;
      for (int j = lane; j < end; j += 32) lo = max(lo, a.offsets[j]);
      lo = __reduce_max_sync(0xffffffffu, lo);
    }
    lo = max(lo, begin);
    e = end - 1;
    count = min(a.offsets[end], count) - lo;
  }
  const int in = static_cast<int>(row) - lo;            // row inside its group
  const int per = rows_of_tile(count, a.bn), i = in / per, r = in - i * per;
  const int at = expert_scale_tile(lo, e, a.bn) + i * ((a.bn + 127) / 128) + r / 128;
  return a.scales + static_cast<long long>(at) * (scale_words_per_stage(FORMAT) * kScaleTile) + (r % 32) * 16 + (r % 128 / 32) * 4;
}

// `split` warps share a row, each taking every split-th chunk.
template <typename T, int FORMAT, bool VEC, bool PACKED>
__global__ void __launch_bounds__(kWarps * 32, quantize_blocks(FORMAT, sizeof(T), PACKED)) quantize_kernel(const QuantizeArgs a, int chunks, int split) {
  constexpr int B = fp4_block(FORMAT), LANES = B / 16, PER = scale_words_per_stage(FORMAT);   // lanes to a block, words to a k-block
  pdl_wait();
  pdl_trigger();   // after the wait: a product behind this kernel may read its weights before its own wait
  __shared__ uint4 all_staging[VEC ? 1 : kWarps * 32 * (static_cast<int>(sizeof(Sixteen<T>)) / 16 + 1)];
  uint4* staging = all_staging + (VEC ? 0 : (threadIdx.x >> 5) * 32 * (sizeof(Sixteen<T>) / 16 + 1));
  const int lane = threadIdx.x & 31;
  const uint32_t warps = gridDim.x * kWarps, units = static_cast<uint32_t>(a.rows) * split;
  const TensorScale scale = tensor_scale<FORMAT, T>(a.tensor_scale);
  const int k = static_cast<int>(a.k), k32 = (k + 31) / 32 * 32, blocks = (k + B - 1) / B;
  const T* x = static_cast<const T*>(a.x);
  // rows of codes start on 8 bytes; an operand's always do
  const bool wide = PACKED || ((reinterpret_cast<uintptr_t>(a.codes) | static_cast<uintptr_t>(a.codes_pitch)) & 7) == 0;
  for (uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5); unit < units; unit += warps) {
    const uint32_t row = split == 1 ? unit : unit / split;
    const int part = static_cast<int>(unit - row * split);
    const long long src = a.row_index ? a.row_index[row] : row;
    const bool there = src >= 0 && src < a.x_rows;
    const T* from = x + (there ? src : 0) * a.x_stride;
    const int k_here = there ? k : 0;
    uint8_t* codes_row = a.codes + row * a.codes_pitch;
    int c = part * kChunk + lane * 16;
    const int step = split * kChunk, whole = k_here / kChunk;      // chunks with no column behind the row's end
    auto load = [&](int chunk, int at) {
      return VEC && chunk < whole ? load_whole(from + at) : load_16<T, VEC>(from, at, k_here, staging, lane);
    };
    Sixteen<T> t = load(part, c);
    uint8_t* tile = nullptr;
    long long tile_step = 0;
    if (PACKED) {       // this lane's word of its first chunk's scales; a chunk is two k-blocks
      const long long block = static_cast<long long>(a.scale_tiles) * (PER * kScaleTile);
      tile = packed_place<FORMAT>(a, row, lane);
      if (lane % (4 * LANES) != 0) tile = nullptr;
      if (tile) tile += (2 * part + lane / 16) * block + lane % 16 / (4 * LANES) * kScaleTile;
      tile_step = 2 * split * block;
    }
    for (int chunk = part; chunk < chunks; chunk += split) {
      Sixteen<T> next = t;
      if (chunk + split < chunks) next = load(chunk + split, c + step);
      uint32_t byte;
      const uint2 codes = quantize_16<FORMAT>(t, scale, byte, [&](int i) { return to_float(from[c + i]); });
      // k32 is a multiple of 32, c of 16: all sixteen codes lie inside the row or none; an operand's k is a multiple of 32
      if (chunk < whole || c < k32) {
        uint32_t* to = reinterpret_cast<uint32_t*>(codes_row + c / 2);
        if (wide) *reinterpret_cast<uint2*>(to) = codes;
        else { to[0] = codes.x; to[1] = codes.y; }
      }
      if (PACKED) {
        if (chunk >= whole && c >= k) byte = 0;
        const uint32_t word = scale_word<FORMAT>(byte);
        if (tile) {
          if (c / 256 * 256 < k) *reinterpret_cast<uint32_t*>(tile) = word;
          tile += tile_step;
        }
      } else if (lane % LANES == 0 && c / B < blocks) {
        a.scales[row * a.scales_pitch + c / B] = static_cast<uint8_t>(byte);
      }
      t = next;
      c += step;
    }
  }
}

// Rows that are quantized already, scales by rows, to a product's operand: row i is row row_index[i] (zeros where that is out of range).
// A warp copies a row: 16 bytes of codes a lane, then four scale bytes a lane.
template <int FORMAT>
__global__ void __launch_bounds__(kWarps * 32) gather_fp4_kernel(const QuantizeArgs a, const uint8_t* codes, const uint8_t* scales, long long scales_pitch) {
  constexpr int PER = scale_words_per_stage(FORMAT), B = fp4_block(FORMAT);
  pdl_wait();
  pdl_trigger();   // as above
  const int lane = threadIdx.x & 31, pieces = static_cast<int>(a.k / 32), blocks = static_cast<int>(a.k / B), words = static_cast<int>((a.k + 255) / 256) * PER;
  for (uint32_t row = blockIdx.x * kWarps + (threadIdx.x >> 5); row < a.rows; row += gridDim.x * kWarps) {
    const long long src = a.row_index[row];
    const bool there = src >= 0 && src < a.x_rows;
    const uint4* from = reinterpret_cast<const uint4*>(codes + (there ? src : 0) * a.codes_pitch);
    uint4* to = reinterpret_cast<uint4*>(a.codes + row * a.codes_pitch);
    for (int i = lane; i < pieces; i += 32) to[i] = there ? __ldg(from + i) : make_uint4(0, 0, 0, 0);
    const uint8_t* scale_row = scales + (there ? src : 0) * scales_pitch;
    uint8_t* tile = packed_place<FORMAT>(a, row, lane);
    if (!tile) continue;
    for (int w = lane; w < words; w += 32) {
      uint32_t word = 0;
      if (there && 4 * w + 4 <= blocks) word = __ldg(reinterpret_cast<const uint32_t*>(scale_row + 4 * w));
      else if (there) for (int b = 0; 4 * w + b < blocks; ++b) word |= static_cast<uint32_t>(scale_row[4 * w + b]) << (8 * b);
      *reinterpret_cast<uint32_t*>(tile + (static_cast<long long>(w / PER) * a.scale_tiles * PER + w % PER) * kScaleTile) = word;
    }
  }
}

// Rows of values: `split` warps share a row as above, eight columns a lane and step (whole 16-byte stores of 16-bit numbers side by side),
// four steps asked for at once.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* codes, long long codes_pitch, const uint8_t* scales, long long scales_pitch,
                                                                 const float* tensor_scale, uint32_t rows, int k, T* y, long long y_stride,
                                                                 int chunks, int split) {
  constexpr int B = fp4_block(FORMAT), U = 4, kStep = 256, W = sizeof(T) / 2, kPitch = 8 + 16 / sizeof(T);   // W: 16-byte pieces of eight numbers
  __shared__ uint4 all_staging[VEC ? 1 : kWarps * 32 * (W + 1)];
  uint4* staging = all_staging + (VEC ? 0 : (threadIdx.x >> 5) * 32 * (W + 1));
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const float g = FORMAT == B2VX_FP4_BLOCK16 ? __ldg(tensor_scale) : 1.0f;
  const uint32_t warps = gridDim.x * kWarps, units = rows * split;
  for (uint32_t unit = blockIdx.x * kWarps + (threadIdx.x >> 5); unit < units; unit += warps) {
    const uint32_t row = split == 1 ? unit : unit / split;
    const uint8_t *codes_row = codes + row * codes_pitch, *scales_row = scales + row * scales_pitch;
    T* to = y + row * y_stride;
    for (int chunk = static_cast<int>(unit - row * split); chunk < chunks; chunk += U * split) {
      uint32_t word[U], byte[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int c = (chunk + u * split) * kStep + lane * 8;
        word[u] = c < k ? __ldg(reinterpret_cast<const uint32_t*>(codes_row + c / 2)) : 0u;
        byte[u] = c < k ? __ldg(scales_row + c / B) : 0u;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int first = (chunk + u * split) * kStep, c = first + lane * 8;
        if (first >= k) break;
        const float s = scale_value<FORMAT>(byte[u]);
        float v[8];
        e2m1_values(word[u], v);
        struct alignas(16) {
          T v[8];
        } out;
        // v s has few bits and is exact.  Its product with g is rounded to float32 before the type's own rounding: one that looks at the product's rest as
        // well would cost each number three more instructions for a 2^-24 of it.
#pragma unroll
        for (int j = 0; j < 8; ++j) out.v[j] = from_float<T>(FORMAT == B2VX_FP4_BLOCK16 ? v[j] * s * g : v[j] * s);
        if (VEC && c + 8 <= k) {
#pragma unroll
          for (int i = 0; i < W; ++i) reinterpret_cast<uint4*>(to + c)[i] = reinterpret_cast<const uint4*>(&out)[i];
        } else if (VEC) {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (c + j < k) to[c + j] = out.v[j];
        } else {       // as load_16, the other way
          const T* values = reinterpret_cast<const T*>(staging);
          __syncwarp();
#pragma unroll
          for (int i = 0; i < W; ++i) staging[lane * (W + 1) + i] = reinterpret_cast<const uint4*>(&out)[i];
          __syncwarp();
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int at = i * 32 + lane;
            if (first + at < k) to[first + at] = values[(at >> 3) * kPitch + (at & 7)];
          }
        }
      }
    }
  }
}

// One thread per word (four blocks of a row) of the packed layout; per: words of a row and stage.
__global__ void __launch_bounds__(256) pack_scales_kernel(const uint8_t* scales, long long matrices, long long n, int gated, long long blocks,
                                                          long long words, int per, uint32_t* packed) {
  pdl_trigger();
  pdl_wait();
  const long long tiles = weight_tiles(n, gated), total = matrices * tiles * words * 128, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const int in = static_cast<int>(i & 127), r = (in & 3) * 32 + (in >> 2);
    const long long m = (i >> 7) / (words * tiles), in_matrix = (i >> 7) % (words * tiles);
    const long long t = in_matrix / per % tiles, w = in_matrix / (per * tiles) * per + in_matrix % per;
    const long long f = gated ? t * 64 + (r >> 4) * 8 + (r & 7) : t * 128 + r;
    uint32_t word = 0;
    if (f < n) {
      const long long row = gated ? (2 * m + ((r >> 3) & 1)) * n + f : m * n + f;
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (w * 4 + b < blocks) word |= static_cast<uint32_t>(scales[row * blocks + w * 4 + b]) << (8 * b);
    }
    packed[i] = word;
  }
}

__global__ void __launch_bounds__(256) gather_rows_kernel(const uint16_t* x, long long x_stride, long long x_rows, const int32_t* row_index,
                                                          long long rows, long long k, int pieces, uint4* y, int vec) {
  pdl_wait();
  pdl_trigger();   // as above
  const long long total = rows * pieces, step = static_cast<long long>(gridDim.x) * blockDim.x;
  for (long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x; i < total; i += step) {
    const long long row = i / pieces, c = (i - row * pieces) * 8;
    const long long src = row_index ? row_index[row] : row;
    uint4 v = make_uint4(0, 0, 0, 0);
    if (src >= 0 && src < x_rows) {
      const uint16_t* from = x + src * x_stride + c;
      if (vec) {
        v = __ldg(reinterpret_cast<const uint4*>(from));
      } else {
        alignas(16) uint16_t t[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) t[j] = from[j];
        v = *reinterpret_cast<const uint4*>(t);
      }
    }
    y[i] = v;
  }
}

int blocks_for(long long units, int per_block, int most) {
  return static_cast<int>(std::max<long long>(1, std::min<long long>((units + per_block - 1) / per_block, most)));
}

// Warps that share a row: up to as many as it has chunks, so that there are about four units of work for each warp that fits the GPU and an
// uneven last round costs little.
int split_of(long long rows, int chunks, int sm_count) {
  const long long fill = 4ll * sm_count * 40;
  return static_cast<int>(std::max<long long>(1, std::min<long long>(chunks, fill / std::max<long long>(1, rows))));
}
// The same for a product's operand, where a row's start costs about as much as a chunk (the place of its scales): rounds of `warps` units, each
// as long as its chunks and one more; of the splits that fill 1 to 8 rounds the one whose rounds together are shortest.  2048 x 8192 numbers
// and a product with 128 features: 27 us by the rule above, 24 by this one.
int operand_split_of(long long rows, int chunks, int warps) {
  long long best = 1, least = LLONG_MAX;
  for (int round = 1; round <= 8; ++round) {
    const long long split = std::max<long long>(1, std::min<long long>(chunks, static_cast<long long>(warps) * round / rows));
    const long long cost = (rows * split + warps - 1) / warps * ((chunks + split - 1) / split + 1);
    if (cost < least) {
      least = cost;
      best = split;
    }
  }
  return static_cast<int>(best);
}

template <typename T, int FORMAT, bool VEC>
cudaError_t quantize(const QuantizeArgs& a, cudaStream_t s) {
  const int chunks = static_cast<int>((a.k + kChunk - 1) / kChunk);
  const bool operand = a.scales_pitch == 0;
  const int kBlocks = quantize_blocks(FORMAT, sizeof(T), operand);
  const int split = operand ? operand_split_of(a.rows, chunks, a.sm_count * kBlocks * kWarps) : split_of(a.rows, chunks, a.sm_count);
  const int grid = blocks_for(a.rows * split, kWarps, a.sm_count * kBlocks);
  if (operand) return launch_pdl(quantize_kernel<T, FORMAT, VEC, true>, dim3(grid), dim3(kWarps * 32), 0, s, a, chunks, split);
  return launch_pdl(quantize_kernel<T, FORMAT, VEC, false>, dim3(grid), dim3(kWarps * 32), 0, s, a, chunks, split);
}
template <typename T, int FORMAT>
cudaError_t quantize_vec(const QuantizeArgs& a, cudaStream_t s) {
  const bool vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && (a.x_stride * sizeof(T)) % 16 == 0;
  return vec ? quantize<T, FORMAT, true>(a, s) : quantize<T, FORMAT, false>(a, s);
}
template <typename T>
cudaError_t quantize_format(const QuantizeArgs& a, cudaStream_t s) {
  return a.format == B2VX_FP4_BLOCK32 ? quantize_vec<T, B2VX_FP4_BLOCK32>(a, s) : quantize_vec<T, B2VX_FP4_BLOCK16>(a, s);
}
template <typename T>
cudaError_t dequantize(const uint8_t* codes, long long codes_pitch, const uint8_t* scales, long long scales_pitch, const float* tensor_scale, int format,
                       long long rows, long long k, void* y, long long y_stride, int sm_count, cudaStream_t s) {
  const int chunks = static_cast<int>((k + 255) / 256);
  const int split = split_of(rows, (chunks + 3) / 4, sm_count);
  const bool vec = reinterpret_cast<uintptr_t>(y) % 16 == 0 && (y_stride * sizeof(T)) % 16 == 0;
  auto* kernel = format == B2VX_FP4_BLOCK32 ? (vec ? dequantize_kernel<T, B2VX_FP4_BLOCK32, true> : dequantize_kernel<T, B2VX_FP4_BLOCK32, false>)
                                            : (vec ? dequantize_kernel<T, B2VX_FP4_BLOCK16, true> : dequantize_kernel<T, B2VX_FP4_BLOCK16, false>);
  return launch_pdl(kernel, dim3(blocks_for(rows * split, kWarps, sm_count * 6)), dim3(kWarps * 32), 0, s, codes, codes_pitch, scales, scales_pitch, tensor_scale,
                    static_cast<uint32_t>(rows), static_cast<int>(k), static_cast<T*>(y), y_stride, chunks, split);
}

}  // namespace

cudaError_t launch_fp4_quantize(const QuantizeArgs& a, cudaStream_t s) {
  if (a.x_dtype == B2VX_DT_FLOAT32) return quantize_format<float>(a, s);
  if (a.x_dtype == B2VX_DT_FLOAT16) return quantize_format<__half>(a, s);
  return quantize_format<__nv_bfloat16>(a, s);
}
size_t fp4_twice_bytes(const QuantizeArgs& a) {
  if (!a.row_index || a.rows < 2 * a.x_rows || a.rows * a.k < kTwiceElements) return 0;
  const size_t scales = (static_cast<size_t>(a.k) / fp4_block(a.format) + 15) / 16 * 16;
  return static_cast<size_t>(a.x_rows) * (a.k / 2 + scales);
}
cudaError_t launch_fp4_operand(const QuantizeArgs& a, void* between, cudaStream_t s) {
  if (fp4_twice_bytes(a) == 0) return launch_fp4_quantize(a, s);
  QuantizeArgs once = a;
  once.rows = a.x_rows;
  once.row_index = nullptr;
  once.offsets = nullptr;
  once.codes = static_cast<uint8_t*>(between);
  once.scales = once.codes + static_cast<size_t>(a.x_rows) * a.codes_pitch;
  once.scales_pitch = (a.k / fp4_block(a.format) + 15) / 16 * 16;
  cudaError_t e = launch_fp4_quantize(once, s);
  if (e != cudaSuccess) return e;
  auto* kernel = a.format == B2VX_FP4_BLOCK32 ? gather_fp4_kernel<B2VX_FP4_BLOCK32> : gather_fp4_kernel<B2VX_FP4_BLOCK16>;
  return launch_pdl(kernel, dim3(blocks_for(a.rows, kWarps, a.sm_count * 8)), dim3(kWarps * 32), 0, s, a, static_cast<const uint8_t*>(once.codes),
                    static_cast<const uint8_t*>(once.scales), once.scales_pitch);
}
cudaError_t launch_fp4_dequantize(const uint8_t* codes, long long codes_pitch, const uint8_t* scales, long long scales_pitch,
                                  const float* tensor_scale, int format, long long rows, long long k, void* y, int y_dtype,
                                  long long y_stride, int sm_count, cudaStream_t s) {
  if (y_dtype == B2VX_DT_FLOAT32) return dequantize<float>(codes, codes_pitch, scales, scales_pitch, tensor_scale, format, rows, k, y, y_stride, sm_count, s);
  if (y_dtype == B2VX_DT_FLOAT16) return dequantize<__half>(codes, codes_pitch, scales, scales_pitch, tensor_scale, format, rows, k, y, y_stride, sm_count, s);
  return dequantize<__nv_bfloat16>(codes, codes_pitch, scales, scales_pitch, tensor_scale, format, rows, k, y, y_stride, sm_count, s);
}
cudaError_t launch_fp4_pack_scales(const uint8_t* scales, int format, long long matrices, long long n, int gated, long long k, uint8_t* packed,
                                   int sm_count, cudaStream_t s) {
  const long long blocks = (k + fp4_block(format) - 1) / fp4_block(format), words = scale_words(k, format);
  const long long total = static_cast<long long>(packed_scale_bytes(matrices, n, gated, k, format) / 4);
  return launch_pdl(pack_scales_kernel, dim3(blocks_for(total, 256, sm_count * 8)), dim3(256), 0, s, scales, matrices, n, gated, blocks, words,
                    scale_words_per_stage(format), reinterpret_cast<uint32_t*>(packed));
}
cudaError_t launch_gather_rows(const void* x, long long x_stride, long long x_rows, const int32_t* row_index, long long rows, long long k, void* y,
                               int sm_count, cudaStream_t s) {
  const int pieces = static_cast<int>(k / 8);
  const int vec = reinterpret_cast<uintptr_t>(x) % 16 == 0 && x_stride % 8 == 0;
  return launch_pdl(gather_rows_kernel, dim3(blocks_for(rows * pieces, 256, sm_count * 8)), dim3(256), 0, s, static_cast<const uint16_t*>(x), x_stride, x_rows,
                    row_index, rows, k, pieces, static_cast<uint4*>(y), vec);
}

}  // namespace b2vx
