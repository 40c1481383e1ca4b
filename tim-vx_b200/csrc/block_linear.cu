// Products y = x W^T on Blackwell tensor cores for operands in 4-bit block floating point or in 16 bits, for one matrix or for
// groups of rows that each have their own (experts).
//
//   y[m][f] = alpha_e * sum_k x[m][k] * W_e[f][k] + bias_e[f],   rows m in [offsets[e], offsets[e + 1])
//   gated:    silu(that with gate row f of W_e) * (that with up row f)
//
// Features are the instruction's M and rows of x its N: a few rows then cost a narrow N instead of an M tile of padding, and the same
// kernel serves one row (where W streams from memory once) and many.  A tile is 128 rows of W for each CTA.  The rows of a
// gated W come in alternating groups of eight gate and eight up rows (one five-dimensional TMA box fetches them so), so that a
// thread of the epilogue finds the gate and the up sum of a feature in its own registers.
//
// Persistent CTAs, one per SM, warp-specialised:
//   warps 0, 2  producers  of W and of x: per k-block of 128 bytes one TMA box each (small ones of few rows)
//   warp 3      producer   of the packed scales of both.  Three warps because a wait, an announcement and a copy take one thread about
//                          340 cycles and each further copy 55.
//   warp 1      issuer     copies a k-block's scales into tensor memory (tcgen05.cp, two slots in turn) and issues its four K steps
//   warps 4-11  epilogue   two sets of four warps take slabs of 32 rows of the tile in turn: out of tensor memory, scale and bias,
//                          activation, rounding, transposition through a buffer in shared memory, 16-byte stores
//
// CG = 2 (many rows): two CTAs of a cluster share a tile of 256 rows of W; each holds its 128 rows of W and half of the rows of x, and
// the first one's issuer issues for both.  An instruction then is twice the work for the same issue, and rows of x are fetched
// once for 256 features.  No load is multicast: every CTA fetches its own operands; the loads of both announce themselves on
// the first one's barrier.
//
// SPLIT (few tiles): the CTAs of a cluster share one tile's K.  Each writes its partial sums into the shared memory of the CTA that a share of
// the tile's features belongs to, and after a barrier of the cluster that one adds them up, in the order of the CTAs.  (One row through 4096 x 4096 has
// 32 tiles: 32 SMs draw their 128 rows of W at 65 bytes a clock, a fifth of what memory gives.)
//
// RAW (with SPLIT, up to 16 rows): x comes as it is, and the epilogue warps, idle until the sums are there, quantize the CTA's part of it
// into shared memory, where it stays; the ring then holds W alone.  Every tile's CTAs repeat that work, but it saves a launch
// and what the products wait for it.
//
// Every wait is bounded as in gemm_tc.cu: on a time-out the CTA records a code, tells the other CTA of its tiles, and both leave through their common
// exit: producers load nothing more, the issuer issues and announces nothing more.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cstdlib>

#include "block_linear.cuh"
#include "fp4.cuh"
#include "pdl.cuh"
#include "tma.cuh"

namespace b2vx {
namespace {

constexpr int kThreads = 12 * 32;
constexpr int kFirstEpilogueWarp = 4;
constexpr int kEpilogueWarps = 8;
constexpr int kMaxStages = 10;
constexpr uint32_t kBufferColumns = 256;                   // of tensor memory: an accumulator of up to 224 columns (256 without scales) and a slot of scales behind it
constexpr int kGroup = 2;                                  // k-blocks of a stage, and slots of scales in tensor memory
constexpr int kBoxRows = 32;
constexpr int kRawRows = 16;                               // rows of x that a product quantizes itself
constexpr int kSlabRows = 32;
constexpr int kSlabBytes = kSlabRows * 256;                // 128 features of 16 bits, two boxes of 64
constexpr int kStagingBytes = 2 * kSlabBytes;              // one for each set
constexpr uint32_t kWTile = 128 * kStageBytes;
constexpr int kSmemBudget = 226 * 1024;
constexpr int kMaxDynSmem = 227 * 1024;
constexpr int kMaxDevices = 64;
constexpr int kMinDynSmem = 120 * 1024;   // keeps two CTAs from sharing an SM and its tensor memory

struct LinearParams {
  int n, rows, experts;
  int bn;                     // most rows of x in a tile
  int feature_tiles;          // tiles along the features of one group
  int scale_tiles;            // 128-row tiles of one matrix of W (and of its packed scales)
  int k_blocks, stages;       // blocks of 128 bytes of K
  int x_box;                  // rows of x in the large box, bn / CG
  int sfb_atoms;              // scale tiles of x to a tile of bn rows
  int x_scale_tiles;          // packed scale tiles along the rows of x
  int split, split_blocks;    // CTAs that share a tile's K, k-blocks of each
  uint32_t staging_bytes, x_bytes;   // RAW: of the quantized part of x
  const void* x;              // RAW: rows, x_pitch bytes apart
  long long x_pitch;
  int x_dtype, x_vec, k;      // x_vec: rows of x start on 16 bytes
  int after_operand;
  uint32_t block_bytes, stage_bytes;
  uint32_t idesc;             // without N
  const float* x_scale;
  const float* w_scale;
  const float* bias;
  const int32_t* offsets;
  void* y;
  long long y_stride;
  int y_dtype;
  int y_vec;                  // rows of y start on 16 bytes
  int* status;
  long long wait_limit;       // cycles
  uint32_t tx_extra;          // bytes announced and never loaded (B2VX_TEST_STALL)
};

struct Maps {
  CUtensorMap w, x, x32, w_scales, x_scales;
};

struct alignas(16) Header {
  unsigned long long full[kMaxStages], empty[kMaxStages];
  unsigned long long acc_full[2], acc_empty[2];
  unsigned long long x_ready;
  uint32_t tmem_base;
  int abort_flag;
  int num_tiles;
  int scan[32];
};
// Behind the header, for each group and one more: first row, first tile, tiles along its rows, rows of each of them.
struct Group {
  int lo, start, tiles, per;
};

// ---- PTX wrappers (the rest: tma.cuh) ----------------------------------------

__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The address of the first CTA's copy of a shared variable.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
  return r;
}
// The same address in CTA `cta`.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int cta) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(cta));
  return r;
}
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// What it tells of is tensor memory that has been read (tcgen05 fences order that), so it need not order this thread's stores to global
// memory: with release at cluster scope it waited for the rows of y to arrive, 1.5 us a tile.
__device__ __forceinline__ void arrive_remote(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}
// A wait for arrivals that may come from the other CTA.
__device__ __forceinline__ bool wait_cluster(uint32_t bar, uint32_t parity, volatile int* abort_flag, int* status, int code, long long limit) {
  const long long began = clock64();
  while (true) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity), "r"(100u) : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    if (clock64() - began > limit) {
      *abort_flag = 1;
      atomicCAS(status, 0, code);
      return false;
    }
  }
}
// Sets the abort flag of the other CTA of a pair; ordered before this thread's arrival at the exit's barrier, until which that CTA stays.
__device__ __forceinline__ void abort_other(uint32_t flag) {
  asm volatile("st.relaxed.cluster.shared::cluster.u32 [%0], %1;\n\tfence.acq_rel.cluster;" ::"r"(in_cta(flag, static_cast<int>(cluster_rank() ^ 1u))), "r"(1u) : "memory");
}
// Arrives on the barrier (CG = 2: of both CTAs) when the instructions issued so far are done.
template <int CG>
__device__ __forceinline__ void commit(uint32_t bar) {
  if constexpr (CG == 1)
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(static_cast<uint16_t>(3)) : "memory");
}
// TMA loads into this CTA's memory; CG = 2: bar may be the first CTA's.
template <int CG>
__device__ __forceinline__ void load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  if constexpr (CG == 1) {
    tma_load_2d(dst, map, c0, c1, bar);
  } else {
    asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(bar) : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
  } else {
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c3, int c4, uint32_t bar) {
  if constexpr (CG == 1) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %6, %6, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c3), "r"(c4), "r"(bar), "r"(0) : "memory");
  } else {
    asm volatile("cp.async.bulk.tensor.5d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %6, %6, %3, %4}], [%5];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c3), "r"(c4), "r"(bar), "r"(0) : "memory");
  }
}
// Descriptors of shared-memory operands as their low halves, start address in 16-byte units (addresses stay below 256 KB, so
// additions do not leave that field), and constant high halves.
//   operand: K-major rows of one 128-byte swizzle span, groups of eight rows 1024 bytes apart
//   scales:  a tile of 32 rows of 16 bytes, not swizzled, groups of eight rows 128 bytes apart
constexpr uint32_t kDescLow = 1u << 16;
constexpr uint32_t kOperandHigh = 64u | (1u << 14) | (2u << 29), kScaleHigh = 8u | (1u << 14);
template <int CG>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t desc_low) {
  if constexpr (CG == 1)
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::1.32x128b.warpx4 [%0], d;\n\t}" ::"r"(taddr), "r"(desc_low), "n"(kScaleHigh) : "memory");
  else
    asm volatile("{\n\t.reg .b64 d;\n\tmov.b64 d, {%1, %2};\n\ttcgen05.cp.cta_group::2.32x128b.warpx4 [%0], d;\n\t}" ::"r"(taddr), "r"(desc_low), "n"(kScaleHigh) : "memory");
}
#define B2VX_MMA(group, kind, scales)                                                                                      \
  asm volatile("{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tmov.b64 da, {%1, %7};\n\tmov.b64 db, {%2, %7};\n\tsetp.ne.b32 p, %6, 0;\n\t" \
               "tcgen05.mma.cta_group::" group ".kind::" kind " [%0], da, db, %3" scales ", p;\n\t}"                         \
               ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate), "n"(kOperandHigh) : "memory")
template <int KIND, int CG>
__device__ __forceinline__ void mma(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if constexpr (KIND == 0 && CG == 1) B2VX_MMA("1", "f16", "");
  else if constexpr (KIND == 0) B2VX_MMA("2", "f16", "");
  else if constexpr (KIND == B2VX_FP4_BLOCK32 && CG == 1) B2VX_MMA("1", "mxf4.block_scale.scale_vec::2X", ", [%4], [%5]");
  else if constexpr (KIND == B2VX_FP4_BLOCK32) B2VX_MMA("2", "mxf4.block_scale.scale_vec::2X", ", [%4], [%5]");
  else if constexpr (CG == 1) B2VX_MMA("1", "mxf4nvf4.block_scale.scale_vec::4X", ", [%4], [%5]");
  else B2VX_MMA("2", "mxf4nvf4.block_scale.scale_vec::4X", ", [%4], [%5]");
}
#undef B2VX_MMA
// Lane t of the warp gets 16 columns of TMEM lane t.
__device__ __forceinline__ void load_lane_columns(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}
// 16 lanes x 32 columns: of column group h (eight columns), thread t gets columns 2 (t % 4), + 1 of lane t / 4 in r[4 h], r[4 h + 1] and of lane
// t / 4 + 8 in r[4 h + 2], r[4 h + 3].
__device__ __forceinline__ void load_16_lanes(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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
// Four 8 x 8 matrices of 16-bit numbers to shared memory, transposed: lane i gives the address of row i % 8 of matrix i / 8.
__device__ __forceinline__ void store_transposed(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// Barriers of a set of epilogue warps; the second also tells every one whether all came with ok.
__device__ __forceinline__ void set_barrier(int set) { asm volatile("bar.sync %0, 128;" ::"r"(1 + set) : "memory"); }
__device__ __forceinline__ bool set_all(int set, bool ok) {
  uint32_t r;
  asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.and.pred q, %2, 128, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
               : "=r"(r) : "r"(static_cast<uint32_t>(ok)), "r"(1 + set) : "memory");
  return r != 0;
}

// One tile of the schedule: group, its first row, the tile's number and first row inside it, rows (as they are and as the instruction's N),
// feature tile.
struct Tile {
  int e, lo, i, r0, rows, n_mma, f;
};
// `from`: a group at or before the tile's (that of an earlier tile of this CTA).  Kept short, in particular of divisions: between two
// tiles every role makes this computation.
template <int CG>
__device__ __forceinline__ Tile tile_of(const Group* groups, const LinearParams& p, int t, int from) {
  int a = from, b = p.experts;           // the last group whose first tile is not behind t
  while (b - a > 1) {
    const int mid = (a + b) >> 1;
    if (groups[mid].start <= t) a = mid; else b = mid;
  }
  const Group g = groups[a];
  const int in = t - g.start;
  int f = in;
  if (g.tiles > 1) {                     // in / g.tiles: the quotient of floats is off by one at most
    f = static_cast<int>(__fdividef(static_cast<float>(in), static_cast<float>(g.tiles)));
    const int r = in - f * g.tiles;
    f += r < 0 ? -1 : (r >= g.tiles ? 1 : 0);
  }
  constexpr int step = 16 * CG;
  Tile r;
  r.e = a;
  r.f = f;
  r.i = in - f * g.tiles;
  r.r0 = r.i * g.per;
  r.rows = max(0, min(g.per, groups[a + 1].lo - g.lo - r.r0));
  r.n_mma = max(step, (r.rows + step - 1) / step * step);
  r.lo = g.lo;
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
// The same 16-byte pieces one number at a time, where rows of y are not aligned or a piece is cut; out of line, it would only be in the way.
template <typename T>
__device__ __noinline__ void store_elements(T* to, long long step, uint32_t from, int row_step, int steps, int rows, int count) {
  for (int u = 0; u < steps && u * row_step < rows; ++u, to += step)
    for (int k = 0; k < count; ++k) {
      uint16_t v;
      asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(from + u * row_step * 128 + 2 * k));
      reinterpret_cast<uint16_t*>(to)[k] = v;
    }
}
// silu(g) u.  The exponential is at most 1, so the divisor lies in [1, 2]: that of -g leaves __fdividef's range from g = -87.4 on, where 0 came out
// for results that a large u makes ordinary numbers.
__device__ __forceinline__ float gate(float g, float u) {
  const float t = expf(-fabsf(g));
  return __fdividef(g < 0.0f ? g * t : g, 1.0f + t) * u;
}

// RAW: k-blocks kb .. kb + blocks - 1 of the rows of x into shared memory, as the loads of a quantized x would put them there (16-byte pieces
// exchanged by the row's number: the 128-byte swizzle).  A warp takes two k-blocks of a row at a time.  Rows up to 15 that do not
// exist keep what lies there; what comes of them is not stored.
template <int KIND, typename X>
__device__ __forceinline__ void quantize_part(const LinearParams& p, int kb, int blocks, uint32_t codes, uint32_t sf, int warp, int lane) {
  constexpr int NW = scale_words_per_stage(KIND), LANES = fp4_block(KIND) / 16;
  const TensorScale scale = tensor_scale<KIND, X>(p.x_scale);
  const int chunks = (blocks + 1) / 2;
  for (int u = warp; u < p.rows * chunks; u += kEpilogueWarps) {
    const int r = u / chunks, chunk = u - r * chunks, block = 2 * chunk + (lane >> 4), c = (kb + 2 * chunk) * 256 + lane * 16;
    const X* row = reinterpret_cast<const X*>(static_cast<const uint8_t*>(p.x) + r * p.x_pitch);
    Sixteen<X> t;
    if (p.x_vec) {
      t = load_16<X, true>(row, c, p.k, nullptr, lane);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) t.v[i] = c + i < p.k ? row[c + i] : from_float<X>(0.0f);
    }
    uint32_t byte;
    const uint2 code = quantize_16<KIND>(t, scale, byte, [&](int i) { return to_float(row[c + i]); });
    if (c >= p.k) byte = 0;
    const uint32_t word = scale_word<KIND>(byte);
    if (block >= blocks) continue;
    const int at = lane % 16 * 8;
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};"
                 ::"r"(codes + block * (kRawRows * kStageBytes) + (r >> 3) * 1024 + (r & 7) * 128 + (((at >> 4) ^ (r & 7)) << 4) + (at & 8)), "r"(code.x), "r"(code.y) : "memory");
    if (lane % (4 * LANES) == 0)
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(sf + (block * NW + lane % 16 / (4 * LANES)) * kScaleTile + r * 16), "r"(word) : "memory");
  }
}

template <int KIND, int CG, bool GATED, bool SPLIT, bool RAW, typename T>
__global__ void __launch_bounds__(kThreads, 1) block_linear_kernel(const __grid_constant__ Maps maps, const LinearParams p) {
  constexpr int NW = KIND == 0 ? 0 : (KIND == B2VX_FP4_BLOCK32 ? 2 : 4);   // scale words per stage
  extern __shared__ uint8_t smem_raw[];
  pdl_trigger();
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t ring = (raw + 1023u) & ~1023u;
  const uint32_t x_codes = ring + p.stages * p.stage_bytes;       // RAW: a k-block's 16 rows of 128 bytes after the other, then their scale tiles
  const uint32_t x_sf = x_codes + p.split_blocks * kRawRows * kStageBytes;
  const uint32_t staging = x_codes + (RAW ? p.x_bytes : 0u);
  Header* h = reinterpret_cast<Header*>(smem_raw + (staging - raw) + p.staging_bytes);
  Group* groups = reinterpret_cast<Group*>(h + 1);
  volatile int* abort_flag = &h->abort_flag;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = CG == 1 ? 0u : cluster_rank();
  const int sharing = SPLIT ? p.split : CG;
  const int first_tile = blockIdx.x / sharing, tile_step = gridDim.x / sharing;
  const int part = SPLIT ? static_cast<int>(cluster_rank()) : 0;
  const int kb_first = SPLIT ? part * p.split_blocks : 0, kb_end = SPLIT ? min(p.k_blocks, kb_first + p.split_blocks) : p.k_blocks;
  // a k-block: [128 rows of W | rows of x | scales of W | scales of x]
  const uint32_t x_off = kWTile, sfa_off = x_off + (RAW ? 0u : static_cast<uint32_t>(p.x_box) * kStageBytes), sfb_off = sfa_off + NW * kScaleTile;

  if (threadIdx.x == 0) {
    for (int i = 0; i < p.stages; ++i) {
      mbar_init(smem_u32(&h->full[i]), NW && !RAW ? 3 : 2);
      mbar_init(smem_u32(&h->empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&h->acc_full[i]), 1);
      mbar_init(smem_u32(&h->acc_empty[i]), CG * kEpilogueWarps);
    }
    mbar_init(smem_u32(&h->x_ready), kEpilogueWarps);
    h->abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {   // all of the SM's tensor memory, so column addresses start at 0
    if constexpr (CG == 1) {
      asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&h->tmem_base)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&h->tmem_base)), "r"(512u) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
  }
  if (threadIdx.x == 64) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w)) : "memory");
    if (NW) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.w_scales)) : "memory");
    if (!RAW) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.x)) : "memory");
    if (NW && !RAW) asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&maps.x_scales)) : "memory");
  }
  // Behind the kernel that made the operand x, which began its work after everything before it had ended, only the loads of x wait.
  if (!p.after_operand) pdl_wait();
  // The groups.  Offsets are device data that nobody has checked: they are cut to rising values among the rows that exist.  Up to three
  // neighbouring offsets a thread, a scan of maxima and one of tiles over the whole block: a decode step waits for this (a warp alone, chunk
  // by chunk, took 3 us for 128 experts).
  if (!p.offsets) {
    if (threadIdx.x == 0) {
      const int n = (p.rows + p.bn - 1) / p.bn;
      groups[0] = {0, 0, n, rows_of_tile(p.rows, p.bn)};
      groups[1] = {p.rows, n * p.feature_tiles, 0, 0};
      h->num_tiles = n * p.feature_tiles;
    }
  } else {
    constexpr int kEach = (kMaxExperts + kThreads) / kThreads;
    const int each = p.experts < kThreads ? 1 : kEach, first = static_cast<int>(threadIdx.x) * each;
    int v[kEach], high = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      v[i] = 0;
      if (i < each && first + i <= p.experts) v[i] = min(max(__ldg(p.offsets + first + i), 0), p.rows);
      high = v[i] = max(high, v[i]);
    }
    int all = high;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, all, d);
      if (lane >= d) all = max(all, up);
    }
    if (lane == 31) h->scan[warp] = all;
    int from = __shfl_up_sync(0xffffffffu, all, 1);
    if (lane == 0) from = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w)
      if (w < warp) from = max(from, h->scan[w]);
    // entry first + i: where group first + i begins and the one before it ends
    int tiles[kEach], sum = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      const int e = first + i, begin = from;
      from = max(from, v[i]);
      tiles[i] = 0;
      if (i >= each || e > p.experts) continue;
      v[i] = from;
      if (e == 0) continue;
      const int count = from - begin, n = count <= p.bn ? (count ? 1 : 0) : (count + p.bn - 1) / p.bn;
      groups[e - 1].tiles = n;
      groups[e - 1].per = n > 1 ? rows_of_tile(count, p.bn) : (count + 31) / 32 * 32;
      tiles[i] = n * p.feature_tiles;
      sum += tiles[i];
    }
    int before = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, d);
      if (lane >= d) before += up;
    }
    if (lane == 31) h->scan[16 + warp] = before;
    before -= sum;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w)
      if (w < warp) before += h->scan[16 + w];
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
      before += tiles[i];
      if (i < each && first + i <= p.experts) {
        groups[first + i].lo = v[i];
        groups[first + i].start = before;
        if (first + i == p.experts) h->num_tiles = before;
      }
    }
  }
  fence_before();
  if constexpr (CG == 1 && !SPLIT) __syncthreads();
  else cluster_barrier();       // the other CTAs have started and their barriers are ready, too
  fence_after();
  const int num_tiles = h->num_tiles;

  // A bounded wait; false: given up, here or elsewhere in the CTA or its pair.
  auto wait = [&](uint32_t bar, uint32_t parity, int code) {
    if (mbar_wait(bar, parity, abort_flag, p.status, code, p.wait_limit)) return true;
    if constexpr (CG == 2) abort_other(smem_u32(&h->abort_flag));
    return false;
  };
  // The control warps run their loops with all lanes, so that what feeds a copy or an instruction is the same in all of them and can live
  // in uniform registers, and elect one (always the same) for the issue.  What a stage costs the issuing thread besides
  // its instructions, some 300 cycles of waiting and bookkeeping, is why a stage holds two k-blocks, and why nothing votes on a wait
  // that gave up: the elected lane then does nothing more in its rounds, and the exit waits for copies in flight.
  const uint32_t full0 = smem_u32(h->full), empty0 = smem_u32(h->empty);
  uint32_t next_stage = 0, next_phase = 0;         // of the producer of W, at its end
  if (warp == 0) {
    // ------------------------------------------------------------ producer of W
    const uint32_t announce = CG == 1 ? full0 : in_first_cta(full0);
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int t = first_tile, e = 0; t < num_tiles; t += tile_step) {
      const Tile tile = tile_of<CG>(groups, p, t, e);
      e = tile.e;
      const int ft = tile.f * CG + static_cast<int>(rank);
      for (int kb = kb_first; kb < kb_end; kb += kGroup) {
        if (elect_one()) {
          ok = ok && wait(empty0 + 8 * s, ph ^ 1, 101);
          if (ok) {
            uint32_t dst = ring + s * p.stage_bytes;
            const uint32_t full = announce + 8 * s;
            const int end = min(kb + kGroup, kb_end);
            if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, (end - kb) * CG * kWTile + p.tx_extra);
            for (int k = kb; k < end; ++k, dst += p.block_bytes) {
              if (GATED) load_5d<CG>(dst, &maps.w, k * kStageBytes, ft * 8, tile.e, full);
              else load_3d<CG>(dst, &maps.w, k * kStageBytes, ft * 128, tile.e, full);
            }
          }
        }
        __syncwarp();
        if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1; }
      }
    }
    next_stage = s;
    next_phase = ph;
  } else if (!RAW && warp == 2) {
    // ------------------------------------------------------------ producer of x
    pdl_wait();
    const uint32_t announce = CG == 1 ? full0 : in_first_cta(full0);
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int t = first_tile, e = 0; t < num_tiles; t += tile_step) {
      const Tile tile = tile_of<CG>(groups, p, t, e);
      e = tile.e;
      const int need = tile.n_mma / CG, row = tile.lo + tile.r0 + static_cast<int>(rank) * need;
      // one large box where most of it is needed, else boxes of 32 rows
      const bool large = 2 * need > p.x_box;
      const int boxes = large ? 1 : (need + kBoxRows - 1) / kBoxRows;
      const uint32_t tx = CG * (large ? p.x_box : boxes * kBoxRows) * kStageBytes;
      for (int kb = kb_first; kb < kb_end; kb += kGroup) {
        if (elect_one()) {
          ok = ok && wait(empty0 + 8 * s, ph ^ 1, 105);
          if (ok) {
            uint32_t dst = ring + s * p.stage_bytes;
            const uint32_t full = announce + 8 * s;
            const int end = min(kb + kGroup, kb_end);
            if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, (end - kb) * tx);
            for (int k = kb; k < end; ++k, dst += p.block_bytes) {
              if (large) {
                load_2d<CG>(dst + x_off, &maps.x, k * kStageBytes, row, full);
              } else {
                for (int b = 0; b < boxes; ++b) load_2d<CG>(dst + x_off + b * kBoxRows * kStageBytes, &maps.x32, k * kStageBytes, row + b * kBoxRows, full);
              }
            }
          }
        }
        __syncwarp();
        if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1; }
      }
    }
  } else if (NW > 0 && warp == 3) {
    // ------------------------------------------------------------ producer of scales
    pdl_wait();
    const uint32_t announce = CG == 1 ? full0 : in_first_cta(full0);
    const uint32_t tx = CG * (1 + (RAW ? 0 : p.sfb_atoms)) * NW * kScaleTile;
    uint32_t s = 0, ph = 0;
    bool ok = true;
    for (int t = first_tile, e = 0; t < num_tiles; t += tile_step) {
      const Tile tile = tile_of<CG>(groups, p, t, e);
      e = tile.e;
      // of a tile of W whose rows do not exist those of the last that do (its outputs are not stored)
      int sfa = ((tile.e * p.k_blocks + kb_first) * p.scale_tiles + min(tile.f * CG + static_cast<int>(rank), p.scale_tiles - 1)) * NW;
      int sfb = (kb_first * p.x_scale_tiles + expert_scale_tile(tile.lo, tile.e, p.bn) + tile.i * p.sfb_atoms) * NW;
      for (int kb = kb_first; kb < kb_end; kb += kGroup) {
        const int blocks = min(kGroup, kb_end - kb);
        if (elect_one()) {
          ok = ok && wait(empty0 + 8 * s, ph ^ 1, 106);
          if (ok) {
            uint32_t dst = ring + s * p.stage_bytes;
            const uint32_t full = announce + 8 * s;
            if (rank == 0) mbar_arrive_expect_tx(full0 + 8 * s, blocks * tx);
            for (int b = 0; b < blocks; ++b, dst += p.block_bytes) {
              load_2d<CG>(dst + sfa_off, &maps.w_scales, 0, sfa + b * p.scale_tiles * NW, full);
              if (!RAW) load_2d<CG>(dst + sfb_off, &maps.x_scales, 0, sfb + b * p.x_scale_tiles * NW, full);
            }
          }
        }
        __syncwarp();
        sfa += kGroup * p.scale_tiles * NW;
        sfb += kGroup * p.x_scale_tiles * NW;
        if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1; }
      }
    }
  } else if (warp == 1 && rank == 0) {
    // ------------------------------------------------------------ issuer
    uint32_t s = 0, ph = 0;
    int j = 0;
    const uint32_t ring_low = (ring >> 4) | kDescLow, stage_low = p.stage_bytes >> 4, block_low = p.block_bytes >> 4;
    uint32_t low = ring_low;                               // of the stage's first operand
    bool ok = true;
    Tile tile = {};
    if (first_tile < num_tiles) tile = tile_of<CG>(groups, p, first_tile, 0);
    for (int t = first_tile; t < num_tiles; t += tile_step, ++j) {
      const uint32_t idesc = p.idesc | (static_cast<uint32_t>(tile.n_mma) >> 3) << 17;
      const int atoms = NW ? (tile.n_mma + 127) >> 7 : 0;
      const int buf = j & 1;
      const uint32_t buf_ph = (j >> 1) & 1;
      if constexpr (CG == 1) {
        ok &= wait(smem_u32(&h->acc_empty[buf]), buf_ph ^ 1, 102);
      } else if (!wait_cluster(smem_u32(&h->acc_empty[buf]), buf_ph ^ 1, abort_flag, p.status, 102, p.wait_limit)) {
        ok = false;
        abort_other(smem_u32(&h->abort_flag));
      }
      __syncwarp();
      fence_after();
      const uint32_t d = buf * kBufferColumns;
      // One k-block: its scales into slot `slot` of tensor memory, then four K steps.  The slot was last read by the instructions of
      // the stage before; copies and products of one thread execute in the order issued.
      auto k_block = [&](uint32_t at, int slot, int kb, bool first) {
        const uint32_t sfa = p.bn + slot * kBufferColumns, sfb = sfa + NW * 4;
        const uint32_t x_at = RAW ? ((x_codes >> 4) | kDescLow) + (kb - kb_first) * (kRawRows * kStageBytes >> 4) : at + (x_off >> 4);
        if constexpr (NW > 0) {
          const uint32_t sfa_low = at + (sfa_off >> 4);
          const uint32_t sfb_low = RAW ? ((x_sf >> 4) | kDescLow) + (kb - kb_first) * (NW * kScaleTile >> 4) : at + (sfb_off >> 4);
#pragma unroll
          for (int w = 0; w < NW; ++w) copy_scales<CG>(sfa + w * 4, sfa_low + w * (kScaleTile >> 4));
#pragma unroll
          for (int w = 0; w < NW; ++w) copy_scales<CG>(sfb + w * 8, sfb_low + w * (kScaleTile >> 4));
          if (atoms > 1) {
#pragma unroll
            for (int w = 0; w < NW; ++w) copy_scales<CG>(sfb + w * 8 + 4, sfb_low + (NW + w) * (kScaleTile >> 4));
          }
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int w = KIND == B2VX_FP4_BLOCK32 ? k >> 1 : k;
          // the first of the word's bytes that this K step uses
          const uint32_t id = KIND == B2VX_FP4_BLOCK32 ? (k & 1) * 2u : 0u;
          mma<KIND, CG>(d, at + 2 * k, x_at + 2 * k, idesc | (id << 4) | (id << 29), sfa + w * 4, sfb + w * 8, !(first && k == 0));
        }
      };
      for (int kb = kb_first; kb < kb_end; kb += kGroup) {
        // the next tile is worked out while the instructions of this one's last stages run
        if (kb + kGroup >= kb_end && t + tile_step < num_tiles) tile = tile_of<CG>(groups, p, t + tile_step, tile.e);
        // given up, the waits of the rounds that are left return at once; a branch around them would cost every round
        if (RAW && kb == kb_first) ok &= wait(smem_u32(&h->x_ready), 0, 107);
        ok &= wait(full0 + 8 * s, ph, 103);
        if (elect_one() & ok) {
          fence_after();
          k_block(low, 0, kb, kb == kb_first);
          if (kb + 1 < kb_end) k_block(low + block_low, 1, kb + 1, false);
          commit<CG>(empty0 + 8 * s);
        }
        __syncwarp();
        low += stage_low;
        if (++s == static_cast<uint32_t>(p.stages)) { s = 0; ph ^= 1; low = ring_low; }
      }
      if (elect_one() & ok) commit<CG>(smem_u32(&h->acc_full[buf]));
      __syncwarp();
    }
  } else if (SPLIT && warp >= kFirstEpilogueWarp) {
    // ------------------------------------------------------------ partial sums, to the CTA whose lanes they are: [CTA][row][its lanes]
    const int ew = warp - kFirstEpilogueWarp, quarter = ew & 3, set = ew >> 2;
    if constexpr (RAW) {
      if (p.x_dtype == B2VX_DT_FLOAT32) quantize_part<KIND, float>(p, kb_first, kb_end - kb_first, x_codes, x_sf, ew, lane);
      else if (p.x_dtype == B2VX_DT_FLOAT16) quantize_part<KIND, __half>(p, kb_first, kb_end - kb_first, x_codes, x_sf, ew, lane);
      else quantize_part<KIND, __nv_bfloat16>(p, kb_first, kb_end - kb_first, x_codes, x_sf, ew, lane);
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&h->x_ready));
    }
    if (first_tile < num_tiles) {
      const Tile tile = tile_of<CG>(groups, p, first_tile, 0);
      const int width = 128 / p.split, l = quarter * 32 + lane, owner = l / width;
      const uint32_t to = in_cta(staging + (part * tile.rows * width + l - owner * width) * 4, owner), step = width * 4;
      wait(smem_u32(&h->acc_full[0]), 0, 104);             // given up: the sums are of no use, y is incomplete
      __syncwarp();
      fence_after();
      for (int c0 = set * 16; c0 < tile.rows; c0 += 32) {
        uint32_t v[16];
        load_lane_columns((static_cast<uint32_t>(quarter * 32) << 16) + c0, v);
        loads_done(v);
#pragma unroll
        for (int c = 0; c < 16; ++c)
          if (c0 + c < tile.rows) asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(to + (c0 + c) * step), "r"(v[c]) : "memory");
      }
    }
  } else if (!SPLIT && warp >= kFirstEpilogueWarp) {
    // ------------------------------------------------------------ epilogue
    const int ew = warp - kFirstEpilogueWarp, quarter = ew & 3, set = ew >> 2;
    const uint32_t lanes = static_cast<uint32_t>(quarter * 32) << 16;
    T* y = static_cast<T*>(p.y);
    const int width = GATED ? 64 : 128;                 // features of a CTA's tile
    const int warp_width = GATED ? 16 : 32;             // of a warp
    const uint32_t out = staging + set * kSlabBytes;
    const float x_scale = p.x_scale ? __ldg(p.x_scale) : 1.0f;
    // What a tile needs of global memory is asked for while the tile before it is worked on.  Bias of the TMEM lanes 8 i + lane / 4 of
    // the warp: features, or alternating eight gate and eight up features.
    struct Ahead {
      Tile tile;
      float w_scale, bias[4];
    };
    auto ahead = [&](int t, int e) {
      Ahead a = {};
      a.w_scale = 1.0f;
      if (t >= num_tiles) return a;
      a.tile = tile_of<CG>(groups, p, t, e);
      if (p.w_scale) a.w_scale = __ldg(p.w_scale + a.tile.e);
      if (p.bias) {
        const float* bias = p.bias + static_cast<long long>(a.tile.e) * (GATED ? 2 : 1) * p.n;
        const int f0 = (a.tile.f * CG + static_cast<int>(rank)) * width + quarter * warp_width + (lane >> 2);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int f = f0 + (GATED ? 8 * (i >> 1) : 8 * i);
          if (f < p.n) a.bias[i] = __ldg(bias + (GATED && (i & 1) ? p.n : 0) + f);
        }
      }
      return a;
    };
    int j = 0;
    Ahead next = ahead(first_tile, 0);
    for (int t = first_tile; t < num_tiles; t += tile_step, ++j) {
      const Ahead now = next;
      const Tile& tile = now.tile;
      const float alpha = x_scale * now.w_scale;
      const float (&b)[4] = now.bias;
      next = ahead(t + tile_step, tile.e);
      const int buf = j & 1;
      const uint32_t buf_ph = (j >> 1) & 1;
      const uint32_t taddr = buf * kBufferColumns + lanes;
      const int row0 = tile.lo + tile.r0;
      const int f0 = (tile.f * CG + static_cast<int>(rank)) * width;       // first feature of the CTA's tile
      const bool ok = set_all(set, wait(smem_u32(&h->acc_full[buf]), buf_ph, 104));
      if (!ok) break;
      fence_after();
      // The accumulator is free for the tile after the next one once everything of it is in registers, before any row is stored.  Where there is no
      // such tile nobody waits for that, and an arrival at the first CTA could come when it has left.
      const bool again = t + 2 * tile_step < num_tiles;
      auto release = [&] {
        if (!again) return;
        fence_before();
        __syncwarp();
        if (lane == 0) {
          if (CG == 1) mbar_arrive(smem_u32(&h->acc_empty[buf]));
          else arrive_remote(in_first_cta(smem_u32(&h->acc_empty[buf])));
        }
      };
      if (set * kSlabRows >= tile.rows) release();
      // Slabs of 32 rows, the sets in turn.
      for (int c0 = set * kSlabRows; c0 < tile.rows; c0 += 2 * kSlabRows) {
        uint32_t v[2][16];
        load_16_lanes(taddr + c0, v[0]);
        load_16_lanes(taddr + c0 + (16u << 16), v[1]);
        loads_done(v[0]);
        loads_done(v[1]);
        if (c0 + 2 * kSlabRows >= tile.rows) release();
        const int rows = min(kSlabRows, tile.rows - c0);
        // value of lane group i (eight TMEM lanes), column group g, column 2 (lane % 4) + k
        auto value = [&](int i, int g, int k) { return fmaf(__uint_as_float(v[i >> 1][4 * g + 2 * (i & 1) + k]), alpha, b[i]); };
        if constexpr (sizeof(T) == 4) {
#pragma unroll
          for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int k = 0; k < 2; ++k) {
              const int r = 8 * g + 2 * (lane & 3) + k;
              if (r >= rows) continue;
              float* to = reinterpret_cast<float*>(y) + (row0 + c0 + r) * p.y_stride + f0 + quarter * warp_width + (lane >> 2);
              const int f = f0 + quarter * warp_width + (lane >> 2);
              if (GATED) {
#pragma unroll
                for (int i = 0; i < 2; ++i)
                  if (f + 8 * i < p.n) to[8 * i] = gate(value(2 * i, g, k), value(2 * i + 1, g, k));
              } else {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                  if (f + 8 * i < p.n) to[8 * i] = value(i, g, k);
              }
            }
          __syncwarp();
        } else {
          // 16-bit numbers, transposed into the set's slab buffer: [64 features][row][128 bytes], 16-byte pieces exchanged by the row's number
          // (neither side then meets bank conflicts), and stored by threads.  A TMA store of the slab waits behind the loads of the next
          // tiles that are already queued: with 1408 columns of K a slab then took 2500 cycles.
          uint32_t m[4][4];
          uint32_t at, step;                               // where matrices m[0] go, and from one m to the next
          if (GATED) {
            // two matrices (features 8 i) of two column groups at a time
            const uint32_t piece = quarter * 2 + ((lane >> 3) & 1);
            at = out + (lane & 7) * 128 + ((piece ^ (lane & 7)) << 4) + (lane >> 4) * 1024;
            step = 2048;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                const int i = q & 1, c = 2 * g + (q >> 1);
                m[g][q] = pack2<T>(gate(value(2 * i, c, 0), value(2 * i + 1, c, 0)), gate(value(2 * i, c, 1), value(2 * i + 1, c, 1)));
              }
          } else {
            const uint32_t piece = (quarter & 1) * 4 + (lane >> 3);
            at = out + (quarter >> 1) * 4096 + (lane & 7) * 128 + ((piece ^ (lane & 7)) << 4);
            step = 1024;
#pragma unroll
            for (int g = 0; g < 4; ++g)
#pragma unroll
              for (int i = 0; i < 4; ++i) m[g][i] = pack2<T>(value(i, g, 0), value(i, g, 1));
          }
          set_barrier(set);                                // every thread has read the last slab
          store_transposed(at, m[0][0], m[0][1], m[0][2], m[0][3]);
          store_transposed(at + step, m[1][0], m[1][1], m[1][2], m[1][3]);
          if (!GATED) {
            store_transposed(at + 2 * step, m[2][0], m[2][1], m[2][2], m[2][3]);
            store_transposed(at + 3 * step, m[3][0], m[3][1], m[3][2], m[3][3]);
          }
          set_barrier(set);
          // 16 bytes a thread and step: of 128 (gated: 64) features a row, eight (sixteen) rows at a time
          constexpr int kSteps = GATED ? 2 : 4, kRowStep = kSlabRows / kSteps;
          const int thread = quarter * 32 + lane;
          const int q = GATED ? thread & 7 : thread & 15, r0 = GATED ? thread >> 3 : thread >> 4, f = f0 + 8 * q;
          T* to = y + (row0 + c0 + r0) * p.y_stride + f;
          const uint32_t from = out + (q >> 3) * 4096 + r0 * 128 + (((q & 7) ^ (r0 & 7)) << 4);
          if (f < p.n) {
            uint32_t w[kSteps][4];
#pragma unroll
            for (int u = 0; u < kSteps; ++u)
              asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[u][0]), "=r"(w[u][1]), "=r"(w[u][2]), "=r"(w[u][3]) : "r"(from + u * kRowStep * 128));
            if (p.y_vec && f + 8 <= p.n) {
              const long long step = kRowStep * p.y_stride;
#pragma unroll
              for (int u = 0; u < kSteps; ++u, to += step)
                if (r0 + u * kRowStep < rows) *reinterpret_cast<uint4*>(to) = make_uint4(w[u][0], w[u][1], w[u][2], w[u][3]);
            } else {
              store_elements<T>(to, kRowStep * p.y_stride, from, kRowStep, kSteps, rows - r0, min(8, p.n - f));
            }
          }
        }
      }
    }
  }

  if constexpr (SPLIT) {
    // This CTA's share of the tile's lanes (features, or gate and up features eight by eight): four features a thread.
    constexpr int G = GATED ? 2 : 1;
    Tile tile = {};
    if (first_tile < num_tiles) tile = tile_of<CG>(groups, p, first_tile, 0);
    const int width = 128 / p.split, quads = width / (4 * G), n = tile.rows * quads;
    const int f_first = tile.f * (128 / G) + part * (width / G);
    const float* bias = p.bias ? p.bias + static_cast<long long>(tile.e) * G * p.n : nullptr;
    // what comes from global memory is asked for before the barrier
    const float alpha = (p.x_scale ? __ldg(p.x_scale) : 1.0f) * (p.w_scale ? __ldg(p.w_scale + tile.e) : 1.0f);
    float b[G][4];
#pragma unroll
    for (int g = 0; g < G; ++g)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int f = f_first + 4 * (static_cast<int>(threadIdx.x) % quads) + k;
        b[g][k] = bias && f < p.n ? __ldg(bias + g * p.n + f) : 0.0f;
      }
    __syncwarp();
    cluster_barrier();
    // kThreads is a multiple of quads (a power of two up to 32), so a thread keeps its features
    const int q = threadIdx.x % quads, f = f_first + 4 * q;
    for (int i = threadIdx.x; i < n; i += kThreads) {
      const int r = i / quads;
      // quads of a gated tile: two of gate, two of up in turn
      const uint32_t at = staging + (r * width + (GATED ? (q >> 1) * 16 + (q & 1) * 4 : 4 * q)) * 4;
      float sum[G][4];
#pragma unroll
      for (int g = 0; g < G; ++g)
#pragma unroll
        for (int k = 0; k < 4; ++k) sum[g][k] = 0.0f;
      for (int c = 0; c < p.split; ++c)
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float v[4];
          asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3])
                       : "r"(at + c * tile.rows * width * 4 + g * 32) : "memory");
#pragma unroll
          for (int k = 0; k < 4; ++k) sum[g][k] += v[k];
        }
      T* to = static_cast<T*>(p.y) + (static_cast<long long>(tile.lo) + tile.r0 + r) * p.y_stride + f;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (f + k >= p.n) break;
        float v = fmaf(sum[0][k], alpha, b[0][k]);
        if (GATED) v = gate(v, fmaf(sum[G - 1][k], alpha, b[G - 1][k]));
        if constexpr (sizeof(T) == 4) to[k] = v;
        else reinterpret_cast<uint16_t*>(to)[k] = static_cast<uint16_t>(pack2<T>(v, v));
      }
    }
  }

  // ---------------------------------------------------------------- common exit
  // What the other CTA's instructions still tell this one's barriers, the last use of each stage, has to arrive while it exists: a lane waits for each.
  // (Within a CTA the epilogue has seen a later word of the same issuer.  Waiting there too cost one row through 4096 x 4096 0.2 us.)
  if (CG == 2 && warp == 0 && lane < p.stages) wait(empty0 + 8 * lane, static_cast<uint32_t>(lane) < next_stage ? next_phase : next_phase ^ 1, 101);
  __syncwarp();
  fence_before();
  if constexpr (CG == 1) __syncthreads();
  else asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");   // the other CTA's instructions reach into this one's memory (its arrivals and loads have all been waited for); stores need not be waited for
  if (*abort_flag) {          // copies and instructions in flight end within microseconds; both CTAs of a pair wait for them
    const long long began = clock64();
    while (clock64() - began < 200000) {}
    __syncwarp();
  }
  if (warp == 1) {
    fence_after();
    if constexpr (CG == 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(h->tmem_base), "r"(512u) : "memory");
    else asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(h->tmem_base), "r"(512u) : "memory");
  }
}

// ---- host side ---------------------------------------------------------------

bool encode(CUtensorMap* map, CUtensorMapDataType type, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
            CUtensorMapSwizzle swizzle) {
  EncodeTiledFn fn = get_encode_fn();
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  return fn && fn(map, type, static_cast<cuuint32_t>(rank), const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}
// Rows of kbytes bytes, in boxes of one stage's bytes.
bool encode_rows(CUtensorMap* map, const void* base, uint64_t kbytes, uint64_t pitch, uint64_t rows, uint64_t mats, int rank, uint32_t box_rows) {
  const cuuint64_t dims[3] = {kbytes, rows, mats}, strides[2] = {pitch, pitch * rows};
  const cuuint32_t box[3] = {kStageBytes, box_rows, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, rank, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// A gated W [experts][gate, up][n][kbytes]: eight rows of gate and eight of up in turn, 64 of each to a box.
bool encode_gated(CUtensorMap* map, const void* base, uint64_t kbytes, uint64_t n, uint64_t experts) {
  const cuuint64_t dims[5] = {kbytes, 8, 2, n / 8, experts}, strides[4] = {kbytes, kbytes * n, kbytes * 8, kbytes * n * 2};
  const cuuint32_t box[5] = {kStageBytes, 8, 2, 8, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, base, 5, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
}
// Packed scales: tiles of 512 bytes.
bool encode_scales(CUtensorMap* map, const void* base, uint64_t tiles, uint32_t box_tiles) {
  const cuuint64_t dims[2] = {kScaleTile / 4, tiles}, strides[1] = {kScaleTile};
  const cuuint32_t box[2] = {kScaleTile / 4, box_tiles};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, base, 2, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE);
}
template <int KIND, int CG, bool GATED, bool SPLIT, bool RAW, typename T>
cudaError_t start(const Maps& maps, const LinearParams& p, int grid, size_t smem, cudaStream_t s) {
  auto* kernel = block_linear_kernel<KIND, CG, GATED, SPLIT, RAW, T>;
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
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (CG > 1 || SPLIT) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = SPLIT ? p.split : CG;
    attr[n].val.clusterDim.y = attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_enabled()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr;
  cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, kernel, maps, p);
}
template <int KIND, int CG, bool GATED, bool SPLIT, bool RAW>
cudaError_t start_typed(const Maps& m, const LinearParams& p, int grid, size_t smem, cudaStream_t s) {
  if (p.y_dtype == B2VX_DT_FLOAT32) return start<KIND, CG, GATED, SPLIT, RAW, float>(m, p, grid, smem, s);
  if (p.y_dtype == B2VX_DT_FLOAT16) return start<KIND, CG, GATED, SPLIT, RAW, __half>(m, p, grid, smem, s);
  return start<KIND, CG, GATED, SPLIT, RAW, __nv_bfloat16>(m, p, grid, smem, s);
}
template <int KIND, bool GATED>
cudaError_t start_kind(const Maps& m, const LinearParams& p, int cg, bool clusters, bool raw, int grid, size_t smem, cudaStream_t s) {
  if (cg == 2) return start_typed<KIND, 2, GATED, false, false>(m, p, grid, smem, s);
  if constexpr (KIND != 0)
    if (raw) return start_typed<KIND, 1, GATED, true, true>(m, p, grid, smem, s);
  if (clusters) return start_typed<KIND, 1, GATED, true, false>(m, p, grid, smem, s);
  return start_typed<KIND, 1, GATED, false, false>(m, p, grid, smem, s);
}

// CTAs to a tile's K: as many of 8, 4, 2 as leave every tile a cluster of its own in one round, every CTA a stage of K and none without;
// else 1.
struct Split {
  int ctas, blocks;
};
Split split_of(long long tiles, int k_blocks, int sm_count) {
  for (int c = 8; c > 1; c /= 2) {
    const int blocks = (k_blocks + c - 1) / c;
    if (tiles * c <= sm_count && blocks >= kGroup && (c - 1) * blocks < k_blocks) return {c, blocks};
  }
  return {1, k_blocks};
}

}  // namespace

bool linear_raw(int format, long long rows, long long n, long long k, int experts, int gated, int sm_count) {
  if (!format || experts != 1 || rows > kRawRows) return false;
  const long long tiles = weight_tiles(n, gated);
  if (tiles > sm_count) return false;
  // What a CTA quantizes: up to 32 k-blocks of a row, two rounds of its 8 warps.  4096 x 4096 (4 k-blocks a CTA) with 1 / 8 / 16 rows:
  // 7.7 / 7.6 / 7.7 us with a launch of its own for that, 6.3 / 6.8 / 8.2 without; 8192 x 8192 (16) with 1 / 4 rows 11.8 / 11.8 and 9.9 / 12.3.
  const Split split = split_of(tiles, static_cast<int>((k + 255) / 256), sm_count);
  return rows * split.blocks <= 32;
}

cudaError_t launch_linear(const LinearArgs& a, cudaStream_t s, const char** why) {
  *why = "";
  const bool fp4 = a.format != 0;
  const int nw = fp4 ? scale_words_per_stage(a.format) : 0;
  LinearParams p = {};
  p.n = static_cast<int>(a.n);
  p.rows = static_cast<int>(a.rows);
  p.experts = a.experts;
  const uint64_t kbytes = fp4 ? static_cast<uint64_t>(a.k) / 2 : static_cast<uint64_t>(a.k) * 2;
  p.k_blocks = static_cast<int>((kbytes + kStageBytes - 1) / kStageBytes);
  p.scale_tiles = static_cast<int>(weight_tiles(a.n, a.gated));

  const int groups = static_cast<int>(std::min<long long>(a.experts, a.rows));
  p.bn = tile_rows(a.rows, a.experts, a.format);
  const int cg = p.bn <= 64 ? 1 : 2;
  p.x_box = p.bn / cg;
  p.feature_tiles = (p.scale_tiles + cg - 1) / cg;
  p.sfb_atoms = fp4 ? (p.bn + 127) / 128 : 0;
  p.block_bytes = a.raw ? kWTile + nw * kScaleTile : (128 + p.x_box) * kStageBytes + (1 + p.sfb_atoms) * nw * kScaleTile;
  p.block_bytes = (p.block_bytes + 1023u) & ~1023u;
  const int elem = a.y_dtype == B2VX_DT_FLOAT32 ? 4 : 2;
  p.y_vec = reinterpret_cast<uintptr_t>(a.y) % 16 == 0 && a.y_stride * elem % 16 == 0;
  const long long most = (a.rows / p.bn + groups) * p.feature_tiles;
  const Split split = cg == 1 ? split_of(most, p.k_blocks, a.sm_count) : Split{1, p.k_blocks};
  p.split = split.ctas;
  p.split_blocks = split.blocks;
  const bool clusters = a.raw || p.split > 1;
  p.x = a.x;
  p.x_pitch = a.x_pitch;
  p.x_dtype = a.x_dtype;
  p.x_vec = reinterpret_cast<uintptr_t>(a.x) % 16 == 0 && a.x_pitch % 16 == 0;
  p.k = static_cast<int>(a.k);
  p.x_bytes = a.raw ? (p.split_blocks * (kRawRows * kStageBytes + nw * kScaleTile) + 1023u) & ~1023u : 0u;
  p.staging_bytes = clusters ? (a.raw ? kRawRows : p.bn) * 512 : kStagingBytes;
  const int behind = static_cast<int>(p.staging_bytes + p.x_bytes) + static_cast<int>(sizeof(Header)) + static_cast<int>(sizeof(Group)) * (a.experts + 1) + 1024;   // and the ring's alignment
  const int room = static_cast<int>((kSmemBudget - behind) / p.block_bytes);      // k-blocks that fit
  p.stages = std::min(kMaxStages, room / kGroup);
  p.stage_bytes = kGroup * p.block_bytes;
  const size_t smem = std::max<size_t>(kMinDynSmem, p.stages * p.stage_bytes + behind);
  const uint32_t m = 8u * cg << 24;
  if (fp4) {
    // a and b e2m1; scales e8m0 (block32) or e4m3
    p.idesc = (1u << 7) | (1u << 10) | (a.format == B2VX_FP4_BLOCK32 ? 1u << 23 : 0u) | m;
  } else {
    const uint32_t t = a.x_dtype == B2VX_DT_FLOAT16 ? 0u : 1u;
    p.idesc = (1u << 4) | (t << 7) | (t << 10) | m;
  }
  p.x_scale = a.x_scale;
  p.w_scale = a.w_scale;
  p.bias = a.bias;
  p.offsets = a.offsets;
  p.y = a.y;
  p.y_stride = a.y_stride;
  p.y_dtype = a.y_dtype;
  p.status = a.status;
  p.wait_limit = kWaitLimitCycles;
  // Test aid, as in gemm_tc.cu: B2VX_TEST_STALL=<n> makes the first n products of the process announce 16 bytes more than their loads deliver and give
  // up after about a millisecond.
  static std::atomic<int> stall_left([] { const char* v = std::getenv("B2VX_TEST_STALL"); return v ? std::atoi(v) : 0; }());
  if (stall_left.load(std::memory_order_relaxed) > 0 && stall_left.fetch_sub(1) > 0) {
    p.wait_limit = 2000000LL;
    p.tx_extra = 16;
  }
  p.x_scale_tiles = fp4 ? static_cast<int>(expert_scale_tiles(a.rows, a.experts, p.bn)) : 0;
  p.after_operand = a.after_operand;

  Maps maps = {};
  const uint64_t rows = static_cast<uint64_t>(a.rows), x_pitch = static_cast<uint64_t>(a.x_pitch);
  const uint64_t w_tiles = static_cast<uint64_t>(a.experts) * p.k_blocks * p.scale_tiles * nw, x_tiles = static_cast<uint64_t>(p.k_blocks) * p.x_scale_tiles * nw;
  bool ok = a.gated ? encode_gated(&maps.w, a.w, kbytes, a.n, a.experts) : encode_rows(&maps.w, a.w, kbytes, kbytes, a.n, a.experts, 3, 128);
  if (fp4) ok = ok && encode_scales(&maps.w_scales, a.w_scales, w_tiles, nw);
  if (!a.raw) {
    ok = ok && encode_rows(&maps.x, a.x, kbytes, x_pitch, rows, 1, 2, p.x_box) && encode_rows(&maps.x32, a.x, kbytes, x_pitch, rows, 1, 2, kBoxRows);
    if (fp4) ok = ok && encode_scales(&maps.x_scales, a.x_scales, x_tiles, nw * p.sfb_atoms);
  }
  if (!ok) {
    *why = "tensor map refused";
    return cudaErrorInvalidValue;
  }
  const int grid = clusters ? static_cast<int>(most) * p.split : static_cast<int>(std::max<long long>(1, std::min<long long>(a.sm_count / cg, most))) * cg;
  auto start_format = [&](auto kind) {
    constexpr int KIND = decltype(kind)::value;
    return a.gated ? start_kind<KIND, true>(maps, p, cg, clusters, a.raw, grid, smem, s) : start_kind<KIND, false>(maps, p, cg, clusters, a.raw, grid, smem, s);
  };
  if (a.format == 0) return start_format(std::integral_constant<int, 0>{});
  if (a.format == B2VX_FP4_BLOCK32) return start_format(std::integral_constant<int, B2VX_FP4_BLOCK32>{});
  return start_format(std::integral_constant<int, B2VX_FP4_BLOCK16>{});
}

}  // namespace b2vx
