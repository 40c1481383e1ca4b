// Products y = x W^T on Blackwell tensor cores for operands in 4-bit block floating point or in 16 bits, for one matrix or for
// groups of rows that each have their own (experts).
//
//   y[m][f] = act( alpha_e * sum_k x[m][k] * W_e[f][k] + bias_e[f] ),   rows m in [offsets[e], offsets[e + 1])
//
// Features are the instruction's M (128 rows of W per tile) and rows of x its N: a few rows then cost a narrow N instead of
// an M tile of padding, the same kernel serves one row (where W streams from memory once) and many, and gate and up halves of a
// gated product meet in one thread of the epilogue, in two accumulators.
//
// One persistent CTA per SM, warp-specialised:
//   warp 0      producer   per stage of 128 bytes of K: TMA boxes of W (P tiles of 128 rows) and of x (32 rows each), bulk copies of
//                          the packed scales
//   warp 1      issuer     copies a stage's scales into tensor memory (tcgen05.cp, two slots in turn) and issues the stage's
//                          four K steps of 32 bytes for each of the P accumulators
//   warps 4-11  epilogue   out of tensor memory, scale and bias, activation, rounding, stores
// Every wait is bounded as in gemm_tc.cu: on a time-out the CTA records a code and leaves through its common exit.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>

#include "block_linear.cuh"
#include "pdl.cuh"
#include "tma.cuh"

namespace b2vx {
namespace {

constexpr int kThreads = 12 * 32;
constexpr int kFirstEpilogueWarp = 4;
constexpr int kEpilogueWarps = 8;
constexpr int kMaxStages = 10;
constexpr int kBoxRows = 32;
constexpr int kSmemBudget = 224 * 1024;
constexpr int kMaxDynSmem = 227 * 1024;
constexpr int kMaxDevices = 64;
constexpr int kMinDynSmem = 120 * 1024;   // keeps two CTAs from sharing an SM and its tensor memory

struct LinearParams {
  int n, rows, experts, gated;
  int bn;                     // most rows of x in a tile, a multiple of 64
  int feature_tiles;          // tiles along the features of one group
  int scale_tiles;            // packed scale tiles along the rows of one matrix of W
  int k_stages, stages, acc_bufs;
  int sfb_atoms;              // most scale tiles of x under one tile's rows
  int words;                  // scale words (tiles along K) of a row tile
  uint32_t stage_bytes, slab_bytes;
  uint32_t idesc;             // without N
  uint32_t acc_cols;          // TMEM columns of one accumulator buffer
  uint32_t sf_cols, sf_base;  // TMEM columns of a scale slot, first column of the slots
  const uint8_t* w_scales;
  const uint8_t* x_scales;
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  const int32_t* offsets;
  void* y;
  long long y_stride;
  int y_dtype;
  int y_vec;                  // rows of y start on 16 bytes
  int* status;
};

struct Header {
  unsigned long long full[kMaxStages], empty[kMaxStages];
  unsigned long long acc_full[2], acc_empty[2];
  uint32_t tmem_base;
  int abort_flag;
  int num_tiles;
};
// Behind the header: the groups' first rows lo[experts + 1] (group e ends where e + 1 begins) and first tiles start[experts + 1].

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar)
      : "memory");
}
// K-major operand rows of one 128-byte swizzle span: groups of eight rows 1024 bytes apart.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | (1ull << 16) | (64ull << 32) | (1ull << 46) | (2ull << 61);
}
// A scale tile: 32 rows of 16 bytes, not swizzled, groups of eight rows 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | (1ull << 16) | (8ull << 32) | (1ull << 46);
}
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
template <int KIND>
__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (KIND == 0) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
  } else if constexpr (KIND == B2VX_FP4_BLOCK32) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4nvf4.block_scale.scale_vec::4X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  }
}
// Lane t of the warp gets 16 columns of TMEM lane t.
__device__ __forceinline__ void load_lane_columns(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 16 lanes x 8 N columns, N = 2 or 4: of column group h, thread t gets columns 2 (t % 4), + 1 of lane t / 4 in r[4 h], r[4 h + 1] and of lane
// t / 4 + 8 in r[4 h + 2], r[4 h + 3].
__device__ __forceinline__ void load_16_lanes(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void load_16_lanes(uint32_t taddr, uint32_t (&r)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.16x256b.x2.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
               : "r"(taddr)
               : "memory");
}
// The registers of a load are valid after the wait; naming them there keeps their uses behind it.
__device__ __forceinline__ void loads_done(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                 "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void loads_done(uint32_t (&r)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7])
               :
               : "memory");
}
// Four 8 x 8 matrices of 16-bit numbers to shared memory, transposed: lane i gives the address of row i % 8 of matrix i / 8.
__device__ __forceinline__ void store_transposed(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// A barrier of the epilogue warps that also tells every one of them whether all came with ok.
__device__ __forceinline__ bool epilogue_all(bool ok) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, 1, %2, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"(static_cast<uint32_t>(ok)), "n"(kEpilogueWarps * 32) : "memory");
  return r != 0;
}
__device__ __forceinline__ void epilogue_barrier() { asm volatile("bar.sync 1, %0;" ::"n"(kEpilogueWarps * 32) : "memory"); }

// One tile of the schedule: group, first row inside it, rows (as the instruction's N and as they are), feature tile.
struct Tile {
  int e, r0, rows, n_mma, f, lo;
};
__device__ __forceinline__ Tile tile_of(const int* lo, const int* start, const LinearParams& p, int t) {
  int a = 0, b = p.experts;           // the last group whose first tile is not behind t
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (start[mid] <= t) a = mid; else b = mid;
  }
  const int count = lo[a + 1] - lo[a], row_tiles = (count + p.bn - 1) / p.bn;
  const int i = t - start[a];
  const int per = ((count + row_tiles - 1) / row_tiles + 63) & ~63;   // even shares, whole halves of a scale tile
  Tile r;
  r.e = a;
  r.f = i / row_tiles;
  r.r0 = (i % row_tiles) * per;
  r.rows = max(0, min(per, count - r.r0));
  r.n_mma = max(16, (r.rows + 15) & ~15);
  r.lo = lo[a];
  return r;
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same<T, __half>::value) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
__device__ __forceinline__ float gate(float g, float u) { return __fdividef(g, 1.0f + expf(-g)) * u; }

template <int KIND, int P, typename T>
__global__ void __launch_bounds__(kThreads, 1)
block_linear_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const LinearParams p) {
  constexpr int NW = KIND == 0 ? 0 : (KIND == B2VX_FP4_BLOCK32 ? 2 : 4);   // scale words per stage
  constexpr uint32_t kATile = 128 * kStageBytes;
  extern __shared__ uint8_t smem_raw[];
  pdl_trigger();
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  const uint32_t staging = ring + p.stages * p.stage_bytes;       // two slabs of the epilogue
  Header* h = reinterpret_cast<Header*>(smem_raw + (staging - raw) + 2 * p.slab_bytes);
  int* lo = reinterpret_cast<int*>(h + 1);
  int* start = lo + p.experts + 1;
  volatile int* abort_flag = &h->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // a stage: [P tiles of W | rows of x | scales of W | scales of x]
  const uint32_t x_off = P * kATile, sfa_off = x_off + static_cast<uint32_t>(p.bn) * kStageBytes;
  const uint32_t sfb_off = sfa_off + P * NW * kScaleTile;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&h->full[i]), 1);
      mbar_init(smem_u32(&h->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&h->acc_full[i]), 1);
      mbar_init(smem_u32(&h->acc_empty[i]), kEpilogueWarps);
    }
    h->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&h->tmem_base)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (threadIdx.x == 64) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_x)) : "memory");
  }
  pdl_wait();   // offsets, rows and scales are other kernels' outputs
  // The groups.  Offsets are device data that nobody has checked: they are cut to rising values among the rows that exist.
  if (warp == 0) {
    int high = 0, total = 0;
    for (int e0 = 0; e0 <= p.experts; e0 += 32) {
      const int e = e0 + lane;
      int v = e < p.experts ? 0 : p.rows;
      if (p.offsets) v = e <= p.experts ? min(max(p.offsets[e], 0), p.rows) : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v = max(v, up);
      }
      v = max(v, high);
      // this chunk's last value is the next chunk's first bound; tiles of group e - 1, which ends at v
      const int prev = __shfl_up_sync(0xffffffffu, v, 1);
      const int from = lane ? prev : high;
      high = __shfl_sync(0xffffffffu, v, 31);
      int sum = e >= 1 && e <= p.experts ? (v - from + p.bn - 1) / p.bn * p.feature_tiles : 0;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int up = __shfl_up_sync(0xffffffffu, sum, d);
        if (lane >= d) sum += up;
      }
      if (e <= p.experts) {
        lo[e] = v;
        start[e] = total + sum;
      }
      total += __shfl_sync(0xffffffffu, sum, 31);
    }
    if (lane == 0) h->num_tiles = total;
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = h->tmem_base;
  const int num_tiles = h->num_tiles;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x) {
      const Tile tile = tile_of(lo, start, p, t);
      const int boxes = (tile.n_mma + kBoxRows - 1) / kBoxRows;
      const int atoms = NW ? ((tile.r0 & 127) + tile.n_mma + 127) >> 7 : 0;
      const uint32_t tx = P * kATile + boxes * kBoxRows * kStageBytes + (P + atoms) * NW * kScaleTile;
      // scale tiles of W: rows that do not exist use the last tile that does (their outputs are not stored)
      const uint8_t* sfa[P];
#pragma unroll
      for (int q = 0; q < P; ++q) {
        const long long mat = p.gated ? 2ll * tile.e + q : tile.e;
        const int st = min(p.gated ? tile.f : tile.f * P + q, p.scale_tiles - 1);
        sfa[q] = p.w_scales + (mat * p.scale_tiles + st) * p.words * kScaleTile;
      }
      const uint8_t* sfb = p.x_scales + (expert_scale_row(tile.lo, tile.e) + tile.r0) / 128 * p.words * kScaleTile;
      for (int ks = 0; ks < p.k_stages; ++ks) {
        ok = mbar_wait(smem_u32(&h->empty[s]), ph ^ 1, abort_flag, p.status, 101);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (elect_one()) {
          const uint32_t full = smem_u32(&h->full[s]);
          const uint32_t dst = ring + s * p.stage_bytes;
          mbar_arrive_expect_tx(full, tx);
#pragma unroll
          for (int q = 0; q < P; ++q) {
            if (p.gated) tma_load_3d(dst + q * kATile, &map_w, ks * kStageBytes, tile.f * 128, 2 * tile.e + q, full);
            else tma_load_3d(dst + q * kATile, &map_w, ks * kStageBytes, (tile.f * P + q) * 128, tile.e, full);
          }
          for (int b = 0; b < boxes; ++b)
            tma_load_2d(dst + x_off + b * kBoxRows * kStageBytes, &map_x, ks * kStageBytes, tile.lo + tile.r0 + b * kBoxRows, full);
          if constexpr (NW > 0) {
#pragma unroll
            for (int q = 0; q < P; ++q) bulk_load(dst + sfa_off + q * NW * kScaleTile, sfa[q] + ks * NW * kScaleTile, NW * kScaleTile, full);
            for (int a = 0; a < atoms; ++a)
              bulk_load(dst + sfb_off + a * NW * kScaleTile, sfb + (static_cast<long long>(a) * p.words + ks * NW) * kScaleTile, NW * kScaleTile, full);
          }
        }
        __syncwarp();
        if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ issuer
    uint32_t s = 0, ph = 0, slot = 0;
    bool ok = true;
    int j = 0;
    for (int t = blockIdx.x; ok && t < num_tiles; t += gridDim.x, ++j) {
      const Tile tile = tile_of(lo, start, p, t);
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(tile.n_mma) >> 3) << 17;
      const int atoms = NW ? ((tile.r0 & 127) + tile.n_mma + 127) >> 7 : 0;
      const uint32_t sfb_col = (tile.r0 & 127) >> 5;
      const int buf = p.acc_bufs == 2 ? (j & 1) : 0;
      const uint32_t buf_ph = p.acc_bufs == 2 ? (j >> 1) & 1 : j & 1;
      ok = mbar_wait(smem_u32(&h->acc_empty[buf]), buf_ph ^ 1, abort_flag, p.status, 102);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      fence_after();
      const uint32_t d = tmem + buf * p.acc_cols;
      for (int ks = 0; ks < p.k_stages; ++ks) {
        ok = mbar_wait(smem_u32(&h->full[s]), ph, abort_flag, p.status, 103);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after();
        if (elect_one()) {
          const uint32_t base = ring + s * p.stage_bytes;
          const uint32_t sfa_t = tmem + p.sf_base + slot * p.sf_cols, sfb_t = sfa_t + P * NW * 4;
          if constexpr (NW > 0) {
            // The slot was last read by instructions two stages ago.  Copies and products of one thread execute in the order issued.
#pragma unroll
            for (int q = 0; q < P * NW; ++q) copy_scales(sfa_t + q * 4, scale_desc(base + sfa_off + q * kScaleTile));
            for (int a = 0; a < atoms; ++a)
#pragma unroll
              for (int w = 0; w < NW; ++w) copy_scales(sfb_t + (w * p.sfb_atoms + a) * 4, scale_desc(base + sfb_off + (a * NW + w) * kScaleTile));
          }
          const uint64_t da = operand_desc(base), db = operand_desc(base + x_off);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int w = KIND == B2VX_FP4_BLOCK32 ? k >> 1 : k;
            // the first of the word's bytes that this K step uses
            const uint32_t id = KIND == B2VX_FP4_BLOCK32 ? (k & 1) * 2u : 0u;
            const uint32_t desc = idesc | (id << 4) | (id << 29);
#pragma unroll
            for (int q = 0; q < P; ++q)
              mma<KIND>(d + q * p.bn, da + q * (kATile >> 4) + 2 * k, db + 2 * k, desc, sfa_t + (q * NW + w) * 4,
                        sfb_t + w * p.sfb_atoms * 4 + sfb_col, (ks | k) != 0);
          }
          commit(smem_u32(&h->empty[s]));
        }
        __syncwarp();
        slot ^= 1;
        if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1; }
      }
      if (ok && elect_one()) commit(smem_u32(&h->acc_full[buf]));
      __syncwarp();
    }
  } else if (warp >= kFirstEpilogueWarp) {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - kFirstEpilogueWarp, quarter = ew & 3, half = ew >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    T* y = static_cast<T*>(p.y);
    const bool gated = P == 2 && p.gated;
    int j = 0, slab = 0;
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x, ++j) {
      const Tile tile = tile_of(lo, start, p, t);
      const int buf = p.acc_bufs == 2 ? (j & 1) : 0;
      const uint32_t buf_ph = p.acc_bufs == 2 ? (j >> 1) & 1 : j & 1;
      float alpha = 1.0f;
      if (p.x_scale) alpha = __ldg(p.x_scale);
      if (p.w_scale) alpha *= __ldg(p.w_scale + tile.e);
      const uint32_t taddr = tmem + buf * p.acc_cols + lanes;
      const long long row0 = static_cast<long long>(tile.lo) + tile.r0;
      const int f0 = gated ? tile.f * 128 : tile.f * P * 128;             // first feature of the tile
      const float* bias = p.bias ? p.bias + static_cast<long long>(tile.e) * (p.gated ? 2 : 1) * p.n : nullptr;
      if constexpr (sizeof(T) == 4) {
        // A thread owns a feature; a warp stores 128 bytes of a row at a time.
        float b[P];
        int f[P];
#pragma unroll
        for (int q = 0; q < P; ++q) {
          f[q] = f0 + (gated ? 0 : q * 128) + quarter * 32 + lane;
          b[q] = bias && f[q] < p.n ? __ldg(bias + (gated && q ? p.n : 0) + f[q]) : 0.0f;
        }
        const bool ok = epilogue_all(mbar_wait(smem_u32(&h->acc_full[buf]), buf_ph, abort_flag, p.status, 104));
        if (!ok) break;
        fence_after();
        for (int c = half * 16; c < tile.rows; c += 32) {
          uint32_t v[P][16];
#pragma unroll
          for (int q = 0; q < P; ++q) load_lane_columns(taddr + q * p.bn + c, v[q]);
#pragma unroll
          for (int q = 0; q < P; ++q) loads_done(v[q]);
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float* to = reinterpret_cast<float*>(y) + (row0 + c + i) * p.y_stride;
            if (c + i >= tile.rows) break;
            if (gated) {
              if (f[0] < p.n) to[f[0]] = gate(fmaf(__uint_as_float(v[0][i]), alpha, b[0]), fmaf(__uint_as_float(v[P - 1][i]), alpha, b[P - 1]));
            } else {
#pragma unroll
              for (int q = 0; q < P; ++q)
                if (f[q] < p.n) to[f[q]] = fmaf(__uint_as_float(v[q][i]), alpha, b[q]);
            }
          }
          __syncwarp();
        }
        fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&h->acc_empty[buf]));
      } else {
        // Slabs of 32 rows: each warp turns its 32 features (of one accumulator, or of both of a gated product or half of the rows)
        // into 16-bit numbers, transposes them into the slab buffer [row][feature] (16-byte pieces exchanged by the row's number, so
        // that neither side meets bank conflicts), and after a barrier all warps store whole rows.  Two buffers in turn.
        float b[4], b2[4];         // of features 8 i + lane / 4 of the warp's 32; b2: of the up half
        const bool split = P == 1 || gated;                 // the two halves of the warps share rows, not accumulators
        const int fw = f0 + (split ? 0 : half * 128) + quarter * 32;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = fw + 8 * i + (lane >> 2);
          b[i] = bias && f < p.n ? __ldg(bias + f) : 0.0f;
          b2[i] = gated && bias && f < p.n ? __ldg(bias + p.n + f) : 0.0f;
        }
        const int pieces = split ? 16 : 32;                 // 16-byte pieces of a row
        const uint32_t pitch = pieces * 16;
        const uint32_t my_piece = (split ? 0 : half * 16) + quarter * 4 + (lane >> 3);
        const bool ok = epilogue_all(mbar_wait(smem_u32(&h->acc_full[buf]), buf_ph, abort_flag, p.status, 104));
        if (!ok) break;
        fence_after();
        for (int c0 = 0; c0 < tile.rows; c0 += 32, ++slab) {
          const uint32_t out = staging + (slab & 1) * p.slab_bytes;
          const uint32_t at = out + (lane & 7) * pitch + ((my_piece ^ (lane & 7)) << 4);
          if (!split) {
            uint32_t v[2][16];
            load_16_lanes(taddr + half * p.bn + c0, v[0]);
            load_16_lanes(taddr + half * p.bn + c0 + (16u << 16), v[1]);
            loads_done(v[0]);
            loads_done(v[1]);
#pragma unroll
            for (int g = 0; g < 4; ++g) {
              uint32_t m[4];
#pragma unroll
              for (int i = 0; i < 4; ++i)
                m[i] = pack2<T>(fmaf(__uint_as_float(v[i >> 1][4 * g + 2 * (i & 1)]), alpha, b[i]),
                                fmaf(__uint_as_float(v[i >> 1][4 * g + 2 * (i & 1) + 1]), alpha, b[i]));
              store_transposed(at + g * 8 * pitch, m[0], m[1], m[2], m[3]);
            }
          } else {
            const int c = half * 16;
            uint32_t v[2][8], u[2][8];
            load_16_lanes(taddr + c0 + c, v[0]);
            load_16_lanes(taddr + c0 + c + (16u << 16), v[1]);
            if (gated) {
              load_16_lanes(taddr + p.bn + c0 + c, u[0]);
              load_16_lanes(taddr + p.bn + c0 + c + (16u << 16), u[1]);
              loads_done(u[0]);
              loads_done(u[1]);
            }
            loads_done(v[0]);
            loads_done(v[1]);
#pragma unroll
            for (int g = 0; g < 2; ++g) {
              uint32_t m[4];
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const int r = 4 * g + 2 * (i & 1);
                float v0 = fmaf(__uint_as_float(v[i >> 1][r]), alpha, b[i]), v1 = fmaf(__uint_as_float(v[i >> 1][r + 1]), alpha, b[i]);
                if (gated) {
                  v0 = gate(v0, fmaf(__uint_as_float(u[i >> 1][r]), alpha, b2[i]));
                  v1 = gate(v1, fmaf(__uint_as_float(u[i >> 1][r + 1]), alpha, b2[i]));
                }
                m[i] = pack2<T>(v0, v1);
              }
              store_transposed(at + (c + g * 8) * pitch, m[0], m[1], m[2], m[3]);
            }
          }
          if (c0 + 32 >= tile.rows) {
            // everything of this accumulator has been read
            fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&h->acc_empty[buf]));
          }
          epilogue_barrier();
          const int rows = min(32, tile.rows - c0);
          for (int i = threadIdx.x - kFirstEpilogueWarp * 32; i < rows * pieces; i += kEpilogueWarps * 32) {
            const int r = split ? i >> 4 : i >> 5, q = i & (pieces - 1);
            const int f = f0 + q * 8;
            if (f >= p.n) continue;
            uint32_t w0, w1, w2, w3;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w0), "=r"(w1), "=r"(w2), "=r"(w3) : "r"(out + r * pitch + ((q ^ (r & 7)) << 4)));
            T* to = y + (row0 + c0 + r) * p.y_stride + f;
            if (p.y_vec && f + 8 <= p.n) {
              *reinterpret_cast<uint4*>(to) = make_uint4(w0, w1, w2, w3);
            } else {
              const uint32_t w[4] = {w0, w1, w2, w3};
#pragma unroll
              for (int k = 0; k < 8; ++k)
                if (f + k < p.n) reinterpret_cast<uint16_t*>(to)[k] = static_cast<uint16_t>(w[k >> 1] >> (16 * (k & 1)));
            }
          }
        }
      }
    }
  }

  // ---------------------------------------------------------------- common exit
  fence_before();
  __syncthreads();
  if (warp == 1) {
    __syncwarp();
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

bool encode_rows(CUtensorMap* map, const void* base, int rank, uint64_t kbytes, uint64_t pitch, uint64_t rows, uint64_t mats, uint32_t box_rows) {
  EncodeTiledFn fn = get_encode_fn();
  if (!fn) return false;
  const cuuint64_t dims[3] = {kbytes, rows, mats}, strides[2] = {pitch, pitch * rows};
  const cuuint32_t box[3] = {kStageBytes, box_rows, 1}, estr[3] = {1, 1, 1};
  return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, estr,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, int P, typename T>
cudaError_t start(const CUtensorMap& w, const CUtensorMap& x, const LinearParams& p, int grid, size_t smem, cudaStream_t s) {
  auto* kernel = block_linear_kernel<KIND, P, T>;
  // once per GPU (a repeated setting by racing first calls does no harm): the attribute costs a call a microsecond of the host's time
  static std::atomic<bool> ready[kMaxDevices];
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev >= kMaxDevices || !ready[dev].load(std::memory_order_acquire)) {
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxDynSmem);
    if (e != cudaSuccess) return e;
    if (dev < kMaxDevices) ready[dev].store(true, std::memory_order_release);
  }
  return launch_pdl(kernel, dim3(grid), dim3(kThreads), smem, s, w, x, p);
}
template <int KIND, int P>
cudaError_t start_typed(const CUtensorMap& w, const CUtensorMap& x, const LinearParams& p, int grid, size_t smem, cudaStream_t s) {
  if (p.y_dtype == B2VX_DT_FLOAT32) return start<KIND, P, float>(w, x, p, grid, smem, s);
  if (p.y_dtype == B2VX_DT_FLOAT16) return start<KIND, P, __half>(w, x, p, grid, smem, s);
  return start<KIND, P, __nv_bfloat16>(w, x, p, grid, smem, s);
}

}  // namespace

cudaError_t launch_linear(const LinearArgs& a, cudaStream_t s, const char** why) {
  *why = "";
  const bool fp4 = a.format != 0;
  const int nw = fp4 ? scale_words_per_stage(a.format) : 0;
  LinearParams p = {};
  p.n = static_cast<int>(a.n);
  p.rows = static_cast<int>(a.rows);
  p.experts = a.experts;
  p.gated = a.gated;
  const uint64_t kbytes = fp4 ? static_cast<uint64_t>(a.k) / 2 : static_cast<uint64_t>(a.k) * 2;
  p.k_stages = static_cast<int>((kbytes + kStageBytes - 1) / kStageBytes);
  p.words = p.k_stages * nw;
  p.scale_tiles = static_cast<int>((a.n + 127) / 128);

  const long long mean = (a.rows + a.experts - 1) / a.experts;
  p.bn = mean <= 64 ? 64 : (mean <= 128 ? 128 : 192);
  // Two tiles of W per CTA halve what x costs per product; one tile makes twice as many tiles.
  const int groups = static_cast<int>(std::min<long long>(a.experts, a.rows));
  const long long tiles2 = ((a.n + 255) / 256) * ((mean + p.bn - 1) / p.bn) * groups;
  const int P = a.gated || tiles2 >= 2 * a.sm_count ? 2 : 1;
  p.feature_tiles = a.gated ? p.scale_tiles : (p.scale_tiles + P - 1) / P;
  p.sfb_atoms = fp4 ? (p.bn + 127) / 128 + (p.bn % 128 ? 0 : 1) : 0;   // tiles start on multiples of 64 rows
  if (p.bn == 64) p.sfb_atoms = fp4 ? 1 : 0;
  p.acc_cols = P * p.bn;
  p.sf_cols = (P + p.sfb_atoms) * nw * 4;
  p.acc_bufs = 2 * p.acc_cols + 2 * p.sf_cols <= 512 ? 2 : 1;
  p.sf_base = p.acc_bufs * p.acc_cols;
  p.stage_bytes = (P * 128 + p.bn) * kStageBytes + (P + p.sfb_atoms) * nw * kScaleTile;
  p.stage_bytes = (p.stage_bytes + 1023u) & ~1023u;
  const int elem = a.y_dtype == B2VX_DT_FLOAT32 ? 4 : 2;
  p.y_vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_stride * elem % 16 == 0;
  p.slab_bytes = elem == 4 ? 0 : 32 * 256 * (P == 2 && !a.gated ? 2 : 1);
  const int header = 2 * p.slab_bytes + static_cast<int>(sizeof(Header)) + 8 * (a.experts + 1) + 1024;   // and the ring's alignment
  p.stages = std::min(kMaxStages, static_cast<int>((kSmemBudget - header) / p.stage_bytes));
  const size_t smem = std::max<size_t>(kMinDynSmem, p.stages * p.stage_bytes + header);
  if (fp4) {
    // a and b e2m1; scales e8m0 (block32) or e4m3
    p.idesc = (1u << 7) | (1u << 10) | (a.format == B2VX_FP4_BLOCK32 ? 1u << 23 : 0u) | (8u << 24);
  } else {
    const uint32_t t = a.x_dtype == B2VX_DT_FLOAT16 ? 0u : 1u;
    p.idesc = (1u << 4) | (t << 7) | (t << 10) | (8u << 24);
  }
  p.w_scales = a.w_scales;
  p.x_scales = a.x_scales;
  p.x_scale = a.x_scale;
  p.w_scale = a.w_scale;
  p.bias = a.bias;
  p.offsets = a.offsets;
  p.y = a.y;
  p.y_stride = a.y_stride;
  p.y_dtype = a.y_dtype;
  p.status = a.status;

  CUtensorMap map_w, map_x;
  const uint64_t mats = static_cast<uint64_t>(a.experts) * (a.gated ? 2 : 1);
  if (!encode_rows(&map_w, a.w, 3, kbytes, kbytes, a.n, mats, 128) ||
      !encode_rows(&map_x, a.x, 2, kbytes, static_cast<uint64_t>(a.x_pitch), a.rows, 1, kBoxRows)) {
    *why = "tensor map refused";
    return cudaErrorInvalidValue;
  }
  const long long most = (a.rows / p.bn + groups) * p.feature_tiles;
  const int grid = static_cast<int>(std::max<long long>(1, std::min<long long>(a.sm_count, most)));
  if (a.format == 0) return P == 2 ? start_typed<0, 2>(map_w, map_x, p, grid, smem, s) : start_typed<0, 1>(map_w, map_x, p, grid, smem, s);
  if (a.format == B2VX_FP4_BLOCK32)
    return P == 2 ? start_typed<B2VX_FP4_BLOCK32, 2>(map_w, map_x, p, grid, smem, s) : start_typed<B2VX_FP4_BLOCK32, 1>(map_w, map_x, p, grid, smem, s);
  return P == 2 ? start_typed<B2VX_FP4_BLOCK16, 2>(map_w, map_x, p, grid, smem, s) : start_typed<B2VX_FP4_BLOCK16, 1>(map_w, map_x, p, grid, smem, s);
}

}  // namespace b2vx
