// Projections of microscaled operands on the tensor cores:
//   y[m][n] = sum over blocks b of 2^(sx[m][b] + sw[n][b]) * sum over k in b of x[m][k] * w[n][k]
// with float32 accumulation, plain or as silu(gate) * up of two weights.  Both operands may be e4m3 or
// e2m1 (tcgen05.mma kind::mxf8f6f4 with block scales takes any pairing).
//
// The weight is the 128-row operand of the instruction and the rows of x are its columns, so one
// kernel serves one row of x as well as thousands: the accumulator is [128 features][NT rows of x] in
// tensor memory, and a thread of the epilogue owns a feature.  Both operands are staged by bulk tensor
// copies, 128 elements of K at a time; a copy of e2m1 codes spreads sixteen of them over sixteen bytes
// of shared memory, the form the instruction reads.  A step's scales are one 512-byte copy per 128 rows and
// go on to tensor memory with tcgen05.cp.  With few output tiles K is split over the CTAs of a cluster,
// which add their accumulators through distributed shared memory in rank order.
//
// Warp 0 issues the copies, warp 1 the matrix instructions, warps 2-5 run the epilogue.  Every wait
// is bounded: a wait that runs out raises a status word and the kernel runs to its end.
#include <cuda.h>

#include <algorithm>
#include <type_traits>

#include "fl_mx_common.cuh"

namespace fl {
namespace {

constexpr int kLinThreads = 192;
constexpr int kWaitTries = 1 << 15;
constexpr int kTileW = 128 * 128;  // bytes of a staged weight tile
constexpr int kMaxStages = 12;
constexpr int kSmemLimit = 232448;
constexpr int kSmemPerSm = 233472;
constexpr int kTailBytes = 512;  // barriers and the tensor memory base

__device__ int g_mx_status;

enum OutKind { kOutBf16 = FL_DTYPE_BF16, kOutF16 = FL_DTYPE_F16, kOutF32 = FL_DTYPE_F32, kOutFp8 = 3, kOutFp4 = 4 };

struct LinearParams {
  const uint8_t *x_scales, *w_scales[2];
  void* out;            // [rows][features], or the codes of a microscaled result
  uint8_t* out_scales;  // of a microscaled result
  int64_t rows;
  int features;
  int steps;   // of K
  int stages;  // of the shared-memory ring
  int w_tiles;
  uint32_t tile_bytes;  // that the copies of one step's element tiles report: a spread e2m1 tile counts as packed
  uint32_t idesc;
  uint32_t tmem_cols;
  int out_kind;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return uint32_t(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
template <bool CLUSTER>
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  if constexpr (CLUSTER) {  // the barrier is arrived at by the other CTA of a pair
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done) : "r"(bar), "r"(parity) : "memory");
  }
  return done != 0;
}
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < kWaitTries; ++i)
    if (mbar_try<CLUSTER>(bar, parity)) return true;
  atomicExch(&g_mx_status, 1);
  return false;
}
// Position in a ring of stages and the parity of its current round.
struct Ring {
  int stage = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void advance(int stages) {
    if (++stage == stages) {
      stage = 0;
      parity ^= 1;
    }
  }
};
__device__ __forceinline__ void copy_tile(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
               ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// Shared-memory descriptor of an operand tile: rows of 128 bytes in the 128-byte swizzle, eight-row
// groups 1024 bytes apart (K-major).
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3fff) | uint64_t(1) << 16 | uint64_t(1024 >> 4) << 32 | uint64_t(1) << 46 |
         uint64_t(2) << 61;
}
// ... and of 32 rows of 16 bytes without swizzle, eight-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t addr) {
  return uint64_t((addr >> 4) & 0x3fff) | uint64_t(1) << 16 | uint64_t(128 >> 4) << 32 | uint64_t(1) << 46;
}
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(scale_desc(smem)) : "memory");
}
__device__ __forceinline__ void mma_mx(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void commit_to(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_load16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
// One lane of the (converged) warp.  The roles that issue copies and matrix instructions run as whole
// warps and issue from one lane, so that addresses and descriptors stay in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ float peer_load(uint32_t addr, uint32_t rank) {
  float v;
  asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %1, %2;\n\tld.shared::cluster.f32 %0, [a];\n\t}"
               : "=f"(v) : "r"(addr), "r"(rank) : "memory");
  return v;
}

// silu(g) * u.  The exponential and the quotient are the hardware's approximations, a few units in the last place of
// float32: far below the rounding of the operands, and the exact forms cost the epilogue more than the
// products take (gated 16384 x 2048 -> 5632: 421 us with expf and a rounded division, 265 us with these and emit16).
__device__ __forceinline__ float gated(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Stores feature n (this thread's) of row m; the 32 lanes of a warp hold 32 consecutive features,
// which are one block of a microscaled result.  Called by whole warps.
__device__ __forceinline__ void emit(const LinearParams& p, int64_t m, int n, float v) {
  if (p.out_kind <= kOutF32) {
    if (n >= p.features) return;
    const int64_t at = m * p.features + n;
    if (p.out_kind == kOutBf16) {
      static_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    } else if (p.out_kind == kOutF16) {
      static_cast<__half*>(p.out)[at] = __float2half_rn(v);
    } else {
      static_cast<float*>(p.out)[at] = v;
    }
    return;
  }
  if (n >= p.features) v = 0.f;
  const uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(v) & 0x7fffffffu);
  const bool fp8 = p.out_kind == kOutFp8;
  const uint32_t byte = fp8 ? mx_scale_byte<FL_MX_FP8>(amax) : mx_scale_byte<FL_MX_FP4>(amax);
  v = byte == 255u ? 0.f : v * mx_inverse(byte);
  uint8_t* codes = static_cast<uint8_t*>(p.out) + m * (int64_t(p.w_tiles) * (fp8 ? kMxStep : kMxStep / 2));
  if (fp8) {
    codes[n] = uint8_t(cvt_e4m3x2(v, 0.f));
  } else {
    const float odd = __shfl_down_sync(0xffffffffu, v, 1);
    if ((n & 1) == 0) codes[n / 2] = uint8_t(cvt_e2m1x2(v, odd));
  }
  if ((n & 31) == 0) p.out_scales[mx_scale_offset(m, n / kMxStep, p.w_tiles) + n / kMxBlock % 4] = uint8_t(byte);
}

template <int NT, bool DUAL>
__global__ void __launch_bounds__(kLinThreads)
mx_linear_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                 const __grid_constant__ CUtensorMap map_w1, const LinearParams p) {
  constexpr int kWeights = DUAL ? 2 : 1;
  constexpr int kXTiles = NT > 128 ? NT / 128 : 1;  // scale tiles of the x rows of a step
  constexpr int kScalesAt = kWeights * kTileW + NT * 128;
  constexpr int kStageBytes = (kScalesAt + (kWeights + kXTiles) * kMxTileBytes + 1023) / 1024 * 1024;
  constexpr uint32_t kScaleCols = 4 * (kWeights + kXTiles);  // tensor memory columns of a stage's scales
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = raw_smem + (1024 - (smem_addr(raw_smem) & 1023)) % 1024;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.stages * kStageBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 1);
  const uint32_t ring = smem_addr(smem), full = smem_addr(bars), empty = full + 8 * kMaxStages,
                 done = empty + 8 * kMaxStages;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = threadIdx.x & 31;
  const uint32_t splits = cluster_size(), rank = cluster_rank();
  const int tile = blockIdx.x / splits;
  const int x_tile = tile / p.w_tiles, w_tile = tile - x_tile * p.w_tiles;
  const int64_t row0 = int64_t(x_tile) * NT;
  const int first = int(int64_t(p.steps) * rank / splits), last = int(int64_t(p.steps) * (rank + 1) / splits);

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    mbar_init(done, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t tmem_scales = tmem + NT * kWeights;

  if (warp == 0) {
    const int x_scale_tiles = int(min(int64_t(kXTiles), (p.rows - row0 + kMxTileRows - 1) / kMxTileRows));
    const uint32_t bytes = p.tile_bytes + (kWeights + x_scale_tiles) * kMxTileBytes;
    Ring ring_at;
    int issued = 0;
    for (int k = first; k < last; ++k, ++issued, ring_at.advance(p.stages)) {
      const int s = ring_at.stage;
      if (issued >= p.stages && !mbar_wait(empty + 8 * s, ring_at.parity ^ 1)) break;
      const uint32_t at = ring + s * kStageBytes, bar = full + 8 * s;
      if (elect_one()) {
        mbar_expect(bar, bytes);
        copy_tile(at, &map_w0, k * kMxStep, w_tile * 128, bar);
        if (DUAL) copy_tile(at + kTileW, &map_w1, k * kMxStep, w_tile * 128, bar);
        copy_tile(at + kWeights * kTileW, &map_x, k * kMxStep, int(row0), bar);
        uint32_t scales = at + kScalesAt;
        for (int i = 0; i < kWeights; ++i, scales += kMxTileBytes)
          copy_bytes(scales, p.w_scales[i] + (int64_t(w_tile) * p.steps + k) * kMxTileBytes, kMxTileBytes, bar);
        for (int i = 0; i < x_scale_tiles; ++i, scales += kMxTileBytes)
          copy_bytes(scales, p.x_scales + ((row0 / kMxTileRows + i) * p.steps + k) * kMxTileBytes, kMxTileBytes, bar);
      }
      __syncwarp();
    }
    // leave only when every copy has landed (the last round of the ring)
    for (int i = max(0, issued - p.stages); i < issued; ++i)
      if (!mbar_wait(full + 8 * (i % p.stages), uint32_t(i / p.stages) & 1)) break;
  } else if (warp == 1) {
    Ring ring_at;
    for (int k = first; k < last; ++k, ring_at.advance(p.stages)) {
      const int s = ring_at.stage;
      if (!mbar_wait(full + 8 * s, ring_at.parity)) break;
      const uint32_t at = ring + s * kStageBytes, scales = at + kScalesAt;
      const uint32_t sf = tmem_scales + s * kScaleCols;
      const uint64_t x_desc = tile_desc(at + kWeights * kTileW);
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < kWeights + kXTiles; ++t) scales_to_tmem(sf + 4 * t, scales + t * kMxTileBytes);
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
          const uint64_t w_desc = tile_desc(at + w * kTileW);
#pragma unroll
          for (int b = 0; b < 4; ++b)  // a block of 32 elements is 32 bytes along the swizzled row
            mma_mx(tmem + w * NT, w_desc + 2 * b, x_desc + 2 * b, p.idesc | uint32_t(b) << 29 | uint32_t(b) << 4,
                   sf + 4 * w, sf + 4 * kWeights, k > first || b > 0);
        }
        commit_to(empty + 8 * s);
      }
      __syncwarp();
    }
    if (elect_one()) commit_to(done);
  }
  __syncwarp();

  const int n = w_tile * 128 + (warp & 3) * 32 + lane;
  const int cols = int(min(int64_t(NT), p.rows - row0));
  if (warp >= 2) {
    mbar_wait(done, 0);
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t mine = tmem + (uint32_t(warp & 3) * 32 << 16);
    float* partial = reinterpret_cast<float*>(smem) + (warp & 3) * 32 + lane;  // [weight][column][feature]
    for (int c = 0; c < cols; c += 16) {
      uint32_t a[16], b[16];
      tmem_load16(mine + c, a);
      if (DUAL) tmem_load16(mine + NT + c, b);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        if (c + j >= cols) break;
        float v = __uint_as_float(a[j]);
        if (splits > 1) {
          partial[(c + j) * 128] = v;
          if (DUAL) partial[(NT + c + j) * 128] = __uint_as_float(b[j]);
        } else {
          if (DUAL) v = gated(v, __uint_as_float(b[j]));
          emit(p, row0 + c + j, n, v);
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  if (splits > 1) {
    cluster_sync();
    if (warp >= 2) {
      const uint32_t mine = ring + ((warp & 3) * 32 + lane) * 4;
      for (int c = rank; c < cols; c += splits) {
        float v = 0.f, u = 0.f;
        for (uint32_t r = 0; r < splits; ++r) {
          v += peer_load(mine + c * 512, r);
          if (DUAL) u += peer_load(mine + (NT + c) * 512, r);
        }
        if (DUAL) v = gated(v, u);
        emit(p, row0 + c, n, v);
      }
    }
    cluster_sync();
  } else {
    __syncthreads();
  }
  // rows of the result's last scale tile past the last row
  if (p.out_kind > kOutF32 && rank == 0 && row0 + NT >= p.rows) {
    const int64_t end = (p.rows + kMxTileRows - 1) / kMxTileRows * kMxTileRows;
    for (int64_t r = p.rows + threadIdx.x; r < end; r += kLinThreads)
      *reinterpret_cast<uint32_t*>(p.out_scales + mx_scale_offset(r, w_tile, p.w_tiles)) = 0u;
  }
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
  }
}

// ---------------------------------------------------------------------------------------
// Many rows of x: persistent CTA pairs (tcgen05 cta_group::2).  A pair computes 256 features by NT
// rows of x at a time: each CTA stages its 128 features and half of the rows, one thread of the first
// CTA issues the matrix instructions for both, and each CTA holds [128 features][NT] of the
// accumulator.  Two accumulators alternate, so the epilogue of one tile runs under the products of
// the next; beside their 2 * NT columns tensor memory holds the scales of every stage of the ring.
//
// silu(gate) * up: the gate tile and the up tile of the same features are two units one after the
// other; the epilogue moves the gate accumulator to registers while the up products run.

constexpr int kPairThreads = 320;  // copies, matrix instructions, eight epilogue warps
// NT: rows of x per tile.  A multiple of 64, as the scales of x start at an even column of tensor memory.
constexpr int kPairRows = 192;
constexpr int kPairStages = 7;
constexpr int kPairXTiles = 2;  // scale tiles that 192 rows starting at a multiple of 64 touch
constexpr int kPairXBytes = kPairRows / 2 * 128;
constexpr int kPairScalesAt = kTileW + kPairXBytes;
constexpr int kPairStageBytes = (kPairScalesAt + (1 + kPairXTiles) * kMxTileBytes + 1023) / 1024 * 1024;
constexpr uint32_t kPairScaleCols = 4 * (1 + kPairXTiles);
static_assert(kPairXBytes % 1024 == 0, "tiles need 1024-byte alignment");
static_assert(2 * kPairRows + kPairStages * kPairScaleCols <= 512, "tensor memory columns");
static_assert(1024 + kPairStages * kPairStageBytes + kTailBytes <= kSmemLimit, "shared memory");

struct PairMaps {
  CUtensorMap x, x_scales, w[2], w_scales[2];
};

struct PairParams {
  void* out;
  uint8_t* out_scales;
  int64_t rows;
  int features;
  int steps;
  int w_tiles;       // of 128 features
  int pair_tiles;    // of 256 features
  int64_t units;     // tiles times weights
  uint32_t step_bytes;  // that the copies of one step report, both CTAs
  uint32_t idesc;
};

__device__ __forceinline__ void copy_tile_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(scale_desc(smem)) : "memory");
}
__device__ __forceinline__ void mma_mx_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
}
// Arrives on the barrier at this offset in both CTAs once every matrix instruction issued so far is done.
__device__ __forceinline__ void commit_to_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// Stores sixteen rows of this thread's feature n, from row m on, of which `count` exist; whole warps call
// it.  WHOLE: all sixteen, and the feature exists.  That path has no branches: the epilogue is bound by
// the instructions of its eight warps.
template <int KIND, bool WHOLE>
__device__ __forceinline__ void emit16(const PairParams& p, int64_t m, int n, const float (&v)[16], int count) {
  const bool live = WHOLE || n < p.features;
  if constexpr (KIND <= kOutF32) {
    using T = std::conditional_t<KIND == kOutBf16, __nv_bfloat16, std::conditional_t<KIND == kOutF16, __half, float>>;
    T* dst = static_cast<T*>(p.out) + m * p.features + n;
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (WHOLE || (live && j < count)) dst[int64_t(j) * p.features] = round_to<T>(v[j]);
  } else {
    constexpr int kFormat = KIND == kOutFp8 ? FL_MX_FP8 : FL_MX_FP4;
    const int64_t row_bytes = int64_t(p.w_tiles) * (KIND == kOutFp8 ? kMxStep : kMxStep / 2);
    uint8_t* codes = static_cast<uint8_t*>(p.out) + m * row_bytes + (KIND == kOutFp8 ? n : n / 2);
    uint8_t* scale = p.out_scales + mx_scale_offset(m, n / kMxStep, p.w_tiles) + n / kMxBlock % 4;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      if (!WHOLE && j >= count) break;  // the same for the warp
      const float x = live ? v[j] : 0.f;
      const uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(x) & 0x7fffffffu);
      const uint32_t byte = mx_scale_byte<kFormat>(amax);
      const float q = byte == 255u ? 0.f : x * mx_inverse(byte);
      if constexpr (KIND == kOutFp8) {
        codes[j * row_bytes] = uint8_t(cvt_e4m3x2(q, 0.f));
      } else {
        const float odd = __shfl_down_sync(0xffffffffu, q, 1);
        if ((n & 1) == 0) codes[j * row_bytes] = uint8_t(cvt_e2m1x2(q, odd));
      }
      if ((n & 31) == 0) scale[j * 16] = uint8_t(byte);  // sixteen rows from a multiple of 16 on share a lane group
    }
  }
}

template <int KIND, bool DUAL>
__global__ void __launch_bounds__(kPairThreads)
mx_linear_pair_kernel(const __grid_constant__ PairMaps maps, const PairParams p) {
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = raw_smem + (1024 - (smem_addr(raw_smem) & 1023)) % 1024;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kPairStages * kPairStageBytes);
  const uint32_t ring = smem_addr(smem), full = smem_addr(bars), empty = full + 8 * kPairStages,
                 acc_full = empty + 8 * kPairStages, acc_empty = acc_full + 16, drained = acc_empty + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kPairStages + 5);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int64_t pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  constexpr int kWeights = DUAL ? 2 : 1;

  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < kPairStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + 8 * b, 1);
      mbar_init(acc_empty + 8 * b, 16);  // a lane of each epilogue warp of both CTAs
    }
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t tmem_scales = tmem + 2 * kPairRows;

  // unit u of this pair: tile t = pair + (u / kWeights) * pairs, weight u % kWeights, features fastest
  if (warp == 0) {
    const uint32_t leader_full = in_cta(full, 0);
    Ring ring_at;
    bool ok = true, again = false;  // again: the ring has been filled once
    for (int64_t unit = pair * kWeights; ok && unit < p.units;
         unit += (DUAL && (unit & 1) == 0) ? 1 : pairs * kWeights - (DUAL ? 1 : 0)) {
      const int64_t tile = unit / kWeights;
      const int which = int(unit % kWeights);
      const int w_tile = int(tile % p.pair_tiles) * 2 + int(rank);
      const int row0 = int(tile / p.pair_tiles) * kPairRows;
      for (int k = 0; k < p.steps; ++k) {
        const int s = ring_at.stage;
        if (again && !mbar_wait(empty + 8 * s, ring_at.parity ^ 1)) {
          ok = false;
          break;
        }
        const uint32_t at = ring + s * kPairStageBytes, bar = leader_full + 8 * s;
        if (elect_one()) {
          if (rank == 0) mbar_expect(full + 8 * s, p.step_bytes);
          copy_tile_pair(at, &maps.w[which], k * kMxStep, w_tile * 128, bar);
          copy_tile_pair(at + kTileW, &maps.x, k * kMxStep, row0 + int(rank) * (kPairRows / 2), bar);
          copy_tile_pair(at + kPairScalesAt, &maps.w_scales[which], 0, w_tile * p.steps + k, bar);
#pragma unroll
          for (int i = 0; i < kPairXTiles; ++i)
            copy_tile_pair(at + kPairScalesAt + (1 + i) * kMxTileBytes, &maps.x_scales, 0,
                           (row0 / kMxTileRows + i) * p.steps + k, bar);
        }
        __syncwarp();
        ring_at.advance(kPairStages);
        again |= ring_at.stage == 0;
      }
    }
    // leave only when every copy of the pair has landed: the stages of this round, then those of the last
    if (rank == 0) {
      for (int s = 0; ok && s < kPairStages; ++s) {
        const bool this_round = s < ring_at.stage;
        if (this_round || again) ok = mbar_wait(full + 8 * s, this_round ? ring_at.parity : ring_at.parity ^ 1);
      }
    }
  } else if (warp == 1 && rank == 0) {
    Ring ring_at, acc_at;
    bool ok = true, again = false;
    for (int64_t unit = pair * kWeights; ok && unit < p.units;
         unit += (DUAL && (unit & 1) == 0) ? 1 : pairs * kWeights - (DUAL ? 1 : 0)) {
      const int buffer = acc_at.stage;
      const int row0 = int(unit / kWeights / p.pair_tiles) * kPairRows;
      if (again && !mbar_wait<true>(acc_empty + 8 * buffer, acc_at.parity ^ 1)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + buffer * kPairRows;
      for (int k = 0; k < p.steps; ++k, ring_at.advance(kPairStages)) {
        const int s = ring_at.stage;
        if (!mbar_wait(full + 8 * s, ring_at.parity)) {
          ok = false;
          break;
        }
        const uint32_t at = ring + s * kPairStageBytes, scales = at + kPairScalesAt;
        const uint32_t sf = tmem_scales + uint32_t(s) * kPairScaleCols;
        const uint64_t w_desc = tile_desc(at), x_desc = tile_desc(at + kTileW);
        const uint32_t sfb = sf + 4 + (row0 % kMxTileRows) / 32;
        if (elect_one()) {
#pragma unroll
          for (int t = 0; t < 1 + kPairXTiles; ++t) scales_to_tmem_pair(sf + 4 * t, scales + t * kMxTileBytes);
#pragma unroll
          for (int b = 0; b < 4; ++b)
            mma_mx_pair(acc, w_desc + 2 * b, x_desc + 2 * b, p.idesc | uint32_t(b) << 29 | uint32_t(b) << 4, sf, sfb,
                        k > 0 || b > 0);
          commit_to_both(empty + 8 * s);
        }
        __syncwarp();
      }
      if (elect_one()) commit_to_both(acc_full + 8 * buffer);
      __syncwarp();
      acc_at.advance(2);
      again |= acc_at.stage == 0;
    }
    // every product is done before tensor memory is given back
    if (elect_one()) commit_to_both(drained);
    __syncwarp();
    mbar_wait(drained, 0);
  } else if (warp >= 2) {
    const uint32_t quarter = uint32_t(warp & 3) * 32, half = uint32_t(warp - 2) / 4;
    constexpr int kCols = kPairRows / 2;  // this warp's columns of a tile
    const uint32_t mine = tmem + (quarter << 16) + half * kCols;
    const uint32_t leader_empty = in_cta(acc_empty, 0);
    Ring acc_at;
    for (int64_t tile = pair; tile < p.units / kWeights; tile += pairs) {
      const int n0 = (int(tile % p.pair_tiles) * 2 + int(rank)) * 128;
      const int n = n0 + int(quarter) + lane;
      const int64_t m0 = tile / p.pair_tiles * kPairRows + half * kCols;
      const int cols = n0 < p.features ? int(max(int64_t(0), min(int64_t(kCols), p.rows - m0))) : 0;
      const bool whole = cols == kCols && n0 + 128 <= p.features;
      float gate[DUAL ? kCols : 1];
      if constexpr (DUAL) {
        const int buffer = acc_at.stage;
        if (!mbar_wait(acc_full + 8 * buffer, acc_at.parity)) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
        for (int c = 0; c < kCols; c += 16) {
          uint32_t a[16];
          tmem_load16(mine + buffer * kPairRows + c, a);
          asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
          for (int j = 0; j < 16; ++j) gate[c + j] = __uint_as_float(a[j]);
        }
        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
        __syncwarp();
        if (lane == 0) arrive_at(leader_empty + 8 * buffer);
        acc_at.advance(2);
      }
      const int buffer = acc_at.stage;
      if (!mbar_wait(acc_full + 8 * buffer, acc_at.parity)) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
      for (int c = 0; c < kCols; c += 16) {
        uint32_t a[16];
        tmem_load16(mine + buffer * kPairRows + c, a);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (c + 16 == kCols) {
          asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
          __syncwarp();
          if (lane == 0) arrive_at(leader_empty + 8 * buffer);
        }
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) v[j] = DUAL ? gated(gate[DUAL ? c + j : 0], __uint_as_float(a[j])) : __uint_as_float(a[j]);
        if (whole) {
          emit16<KIND, true>(p, m0 + c, n, v, 16);
        } else if (c < cols) {
          emit16<KIND, false>(p, m0 + c, n, v, cols - c);
        }
      }
      acc_at.advance(2);
      // rows of the result's last scale tile past the last row
      if (KIND > kOutF32 && n0 < p.features && m0 <= p.rows && p.rows <= m0 + kCols) {
        const int64_t end = (p.rows + kMxTileRows - 1) / kMxTileRows * kMxTileRows;
        for (int64_t r = p.rows + quarter + lane; r < end; r += 128)
          *reinterpret_cast<uint32_t*>(p.out_scales + mx_scale_offset(r, n0 / kMxStep, p.w_tiles)) = 0u;
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  __syncwarp();
  cluster_sync();
  if (warp == 0) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
}

// ------------------------------------------------------------------------------------ host

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return reinterpret_cast<EncodeTiled>(p);
  }();
  return fn;
}

// Codes [rows][steps * 128] as boxes of 128 elements by box_rows rows in the 128-byte swizzle; rows past
// the last read as zero.
bool make_map(CUtensorMap* map, const void* codes, int format, int64_t rows, int64_t steps, int box_rows) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const bool fp8 = format == FL_MX_FP8;
  const cuuint64_t dims[2] = {cuuint64_t(steps * kMxStep), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(steps * (fp8 ? kMxStep : kMxStep / 2))};
  const cuuint32_t box[2] = {kMxStep, cuuint32_t(box_rows)};
  const cuuint32_t unit[2] = {1, 1};
  return encode(map, fp8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2,
                const_cast<void*>(codes), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;

int sm_count(int device) {
  static int counts[kMaxDevices];  // written with the same value by whoever comes first
  if (device < 0 || device >= kMaxDevices) return 148;
  if (counts[device] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || n <= 0) n = 148;
    counts[device] = n;
  }
  return counts[device];
}

struct Operand {
  const void *codes, *scales;
  int format;
};

struct LinearCall {
  Operand x, w[2];
  int64_t rows;
  int32_t cols, features;
  int out_kind;
  void *out, *out_scales;
  cudaStream_t stream;
  const char* who;
};

template <int NT, bool DUAL>
int launch_linear(const LinearCall& call, int splits) {
  constexpr int kWeights = DUAL ? 2 : 1, kXTiles = NT > 128 ? NT / 128 : 1;
  constexpr int kStageBytes =
      (kWeights * kTileW + NT * 128 + (kWeights + kXTiles) * kMxTileBytes + 1023) / 1024 * 1024;
  constexpr int kScaleCols = 4 * (kWeights + kXTiles);
  constexpr int kPartialBytes = kWeights * NT * 512;
  const int steps = int(mx_steps(call.cols));
  LinearParams p;
  p.x_scales = static_cast<const uint8_t*>(call.x.scales);
  p.w_scales[0] = static_cast<const uint8_t*>(call.w[0].scales);
  p.w_scales[1] = static_cast<const uint8_t*>(call.w[1].scales);
  p.out = call.out;
  p.out_scales = static_cast<uint8_t*>(call.out_scales);
  p.rows = call.rows;
  p.features = call.features;
  p.steps = steps;
  p.w_tiles = (call.features + 127) / 128;
  p.out_kind = call.out_kind;
  p.tile_bytes = uint32_t((kWeights * kTileW >> (call.w[0].format == FL_MX_FP8 ? 0 : 1)) +
                          (NT * 128 >> (call.x.format == FL_MX_FP8 ? 0 : 1)));
  const int most = std::min(kMaxStages, (kSmemLimit - 1024 - kTailBytes) / kStageBytes);
  p.stages = std::min(most, (steps + splits - 1) / splits);
  const int need = NT * kWeights + p.stages * kScaleCols;
  p.tmem_cols = need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512;
  // Shared memory in proportion to the columns: CTAs of these kernels that fit an SM together
  // never want more than its 512 columns, so none waits for columns while its cluster waits for it.
  const int smem = std::max({1024 + kTailBytes + std::max(p.stages * kStageBytes, splits > 1 ? kPartialBytes : 0),
                             int(p.tmem_cols) * (kSmemPerSm / 512) - 1024});
  // instruction descriptor: element types (e4m3 0, e2m1 5), e8m0 scales, N, M = 128
  p.idesc = uint32_t(call.w[0].format == FL_MX_FP8 ? 0 : 5) << 7 | uint32_t(call.x.format == FL_MX_FP8 ? 0 : 5) << 10 |
            uint32_t(NT / 8) << 17 | 1u << 23 | uint32_t(128 / 16) << 24;
  CUtensorMap map_x, map_w0, map_w1;
  FL_REQUIRE(make_map(&map_x, call.x.codes, call.x.format, call.rows, steps, NT) &&
                 make_map(&map_w0, call.w[0].codes, call.w[0].format, call.features, steps, 128) &&
                 make_map(&map_w1, call.w[DUAL ? 1 : 0].codes, call.w[0].format, call.features, steps, 128),
             "%s: the operands cannot be described as tensor maps", call.who);
  const int64_t tiles = (call.rows + NT - 1) / NT * p.w_tiles;
  FL_REQUIRE(tiles * splits < (int64_t(1) << 31), "%s: too many elements", call.who);
  auto kernel = mx_linear_kernel<NT, DUAL>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(tiles * splits));
  config.blockDim = dim3(kLinThreads);
  config.dynamicSmemBytes = smem;
  config.stream = call.stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = splits;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&config, kernel, map_x, map_w0, map_w1, p);
  if (err != cudaSuccess) {
    cudaGetLastError();
    set_error("%s: %s", call.who, cudaGetErrorString(err));
    return FL_ERR_CUDA;
  }
  return FL_OK;
}

// Scale tiles as rows of 128 words; tiles past the last read as zero.
bool make_scale_map(CUtensorMap* map, const void* scales, int64_t rows, int64_t steps) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {kMxTileBytes / 4, cuuint64_t((rows + kMxTileRows - 1) / kMxTileRows * steps)};
  const cuuint64_t strides[1] = {kMxTileBytes};
  const cuuint32_t box[2] = {kMxTileBytes / 4, 1};
  const cuuint32_t unit[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<void*>(scales), dims, strides, box, unit,
                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int KIND, bool DUAL>
int launch_pairs(const LinearCall& call, int sms) {
  const int steps = int(mx_steps(call.cols));
  PairMaps maps;
  PairParams p;
  p.out = call.out;
  p.out_scales = static_cast<uint8_t*>(call.out_scales);
  p.rows = call.rows;
  p.features = call.features;
  p.steps = steps;
  p.w_tiles = (call.features + 127) / 128;
  p.pair_tiles = (call.features + 255) / 256;
  const int64_t tiles = (call.rows + kPairRows - 1) / kPairRows * p.pair_tiles;
  p.units = tiles * (DUAL ? 2 : 1);
  p.step_bytes = 2 * uint32_t((kTileW >> (call.w[0].format == FL_MX_FP8 ? 0 : 1)) +
                              (kPairXBytes >> (call.x.format == FL_MX_FP8 ? 0 : 1)) + (1 + kPairXTiles) * kMxTileBytes);
  p.idesc = uint32_t(call.w[0].format == FL_MX_FP8 ? 0 : 5) << 7 | uint32_t(call.x.format == FL_MX_FP8 ? 0 : 5) << 10 |
            uint32_t(kPairRows / 8) << 17 | 1u << 23 | uint32_t(256 / 16) << 24;
  bool ok = make_map(&maps.x, call.x.codes, call.x.format, call.rows, steps, kPairRows / 2) &&
            make_scale_map(&maps.x_scales, call.x.scales, call.rows, steps);
  for (int i = 0; i < 2; ++i) {
    const Operand& w = call.w[DUAL ? i : 0];
    ok = ok && make_map(&maps.w[i], w.codes, w.format, call.features, steps, 128) &&
         make_scale_map(&maps.w_scales[i], w.scales, call.features, steps);
  }
  FL_REQUIRE(ok, "%s: the operands cannot be described as tensor maps", call.who);
  FL_REQUIRE(int64_t(p.w_tiles + 2) * steps < (int64_t(1) << 31) &&
                 (call.rows / kMxTileRows + kPairXTiles + 1) * steps < (int64_t(1) << 31),
             "%s: too many elements", call.who);
  auto kernel = mx_linear_pair_kernel<KIND, DUAL>;
  cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(unsigned(2 * std::min<int64_t>(tiles, sms / 2)));
  config.blockDim = dim3(kPairThreads);
  config.dynamicSmemBytes = kSmemLimit;  // all of an SM's, as it takes all of its tensor memory (see above)
  config.stream = call.stream;
  cudaLaunchAttribute attribute;
  attribute.id = cudaLaunchAttributeClusterDimension;
  attribute.val.clusterDim.x = 2;
  attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
  config.attrs = &attribute;
  config.numAttrs = 1;
  if (err == cudaSuccess) err = cudaLaunchKernelEx(&config, kernel, maps, p);
  if (err != cudaSuccess) {
    cudaGetLastError();
    set_error("%s: %s", call.who, cudaGetErrorString(err));
    return FL_ERR_CUDA;
  }
  return FL_OK;
}

template <bool DUAL>
int launch_pairs_of_kind(const LinearCall& call, int sms) {
  switch (call.out_kind) {
    case kOutBf16: return launch_pairs<kOutBf16, DUAL>(call, sms);
    case kOutF16: return launch_pairs<kOutF16, DUAL>(call, sms);
    case kOutF32: return launch_pairs<kOutF32, DUAL>(call, sms);
    default: break;
  }
  if constexpr (DUAL) {
    return call.out_kind == kOutFp8 ? launch_pairs<kOutFp8, true>(call, sms) : launch_pairs<kOutFp4, true>(call, sms);
  } else {
    FL_REQUIRE(false, "%s: unknown output type", call.who);
  }
}

template <bool DUAL>
int choose_linear(const LinearCall& call) {
  int device = 0;
  cudaGetDevice(&device);
  const int sms = sm_count(device);
  const int steps = int(mx_steps(call.cols));
  const int64_t w_tiles = (call.features + 127) / 128;
  auto splits_for = [&](int nt) {
    const int64_t tiles = (call.rows + nt - 1) / nt * w_tiles;
    int splits = 1;
    while (splits < 8 && tiles * splits * 2 <= sms && splits * 2 <= steps) splits *= 2;
    return splits;
  };
  if (call.rows <= 16) return launch_linear<16, DUAL>(call, splits_for(16));
  if (call.rows <= 32) return launch_linear<32, DUAL>(call, splits_for(32));
  if (call.rows <= 64) return launch_linear<64, DUAL>(call, splits_for(64));
  if ((call.rows + kPairRows - 1) / kPairRows * ((call.features + 255) / 256) >= sms / 2)
    return launch_pairs_of_kind<DUAL>(call, sms);
  return launch_linear<128, DUAL>(call, splits_for(128));
}

int check_operand(const char* who, const char* name, const Operand& o) {
  FL_REQUIRE(mx_format_ok(o.format), "%s: unknown format of %s", who, name);
  FL_REQUIRE(o.codes && o.scales, "%s: null argument", who);
  FL_REQUIRE((reinterpret_cast<uintptr_t>(o.codes) & 31u) == 0 && aligned16(o.scales),
             "%s: codes of %s must be 32-byte aligned and its scales 16-byte aligned", who, name);
  return FL_OK;
}

}  // namespace
}  // namespace fl

using namespace fl;

extern "C" int fl_mx_linear(const void* x_codes, const void* x_scales, int32_t x_format, const void* w_codes,
                            const void* w_scales, int32_t w_format, int64_t rows, int32_t out_features,
                            int32_t in_features, void* out, int32_t out_dtype, fl_cuda_stream stream) {
  const char* who = "fl_mx_linear";
  FL_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && out_features > 0 && in_features > 0, "%s: bad sizes", who);
  FL_REQUIRE(out_dtype >= kOutBf16 && out_dtype <= kOutF32, "%s: unknown output type", who);
  if (rows == 0) return FL_OK;
  LinearCall call{{x_codes, x_scales, x_format}, {{w_codes, w_scales, w_format}, {w_codes, w_scales, w_format}}, rows,
                  in_features, out_features, out_dtype, out, nullptr, static_cast<cudaStream_t>(stream), who};
  if (int rc = check_operand(who, "x", call.x)) return rc;
  if (int rc = check_operand(who, "weight", call.w[0])) return rc;
  FL_REQUIRE(out && aligned16(out), "%s: out must be given, 16-byte aligned", who);
  return choose_linear<false>(call);
}

extern "C" int fl_mx_linear_swiglu(const void* x_codes, const void* x_scales, int32_t x_format, const void* gate_codes,
                                   const void* gate_scales, const void* up_codes, const void* up_scales,
                                   int32_t w_format, int64_t rows, int32_t out_features, int32_t in_features,
                                   void* out, int32_t out_dtype, int32_t out_format, void* out_scales,
                                   fl_cuda_stream stream) {
  const char* who = "fl_mx_linear_swiglu";
  FL_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && out_features > 0 && in_features > 0, "%s: bad sizes", who);
  FL_REQUIRE(out_scales == nullptr ? out_dtype >= kOutBf16 && out_dtype <= kOutF32 : mx_format_ok(out_format),
             "%s: unknown output type or format", who);
  if (rows == 0) return FL_OK;
  const int kind = out_scales == nullptr ? out_dtype : out_format == FL_MX_FP8 ? int(kOutFp8) : int(kOutFp4);
  LinearCall call{{x_codes, x_scales, x_format}, {{gate_codes, gate_scales, w_format}, {up_codes, up_scales, w_format}},
                  rows, in_features, out_features, kind, out, out_scales, static_cast<cudaStream_t>(stream), who};
  if (int rc = check_operand(who, "x", call.x)) return rc;
  if (int rc = check_operand(who, "gate", call.w[0])) return rc;
  if (int rc = check_operand(who, "up", call.w[1])) return rc;
  FL_REQUIRE(out && aligned16(out) && aligned16(out_scales), "%s: outputs must be given, 16-byte aligned", who);
  return choose_linear<true>(call);
}

extern "C" int fl_mx_status(int32_t* status, int32_t reset, fl_cuda_stream stream) {
  FL_REQUIRE(status != nullptr, "fl_mx_status: null status");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  cudaError_t err = cudaMemcpyFromSymbolAsync(status, g_mx_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, s);
  if (err == cudaSuccess) err = cudaStreamSynchronize(s);
  if (err == cudaSuccess && reset != 0) {
    static const int32_t zero = 0;
    err = cudaMemcpyToSymbolAsync(g_mx_status, &zero, sizeof(int32_t), 0, cudaMemcpyHostToDevice, s);
    if (err == cudaSuccess) err = cudaStreamSynchronize(s);
  }
  if (err != cudaSuccess) {
    set_error("fl_mx_status: %s", cudaGetErrorString(err));
    return FL_ERR_CUDA;
  }
  return FL_OK;
}
