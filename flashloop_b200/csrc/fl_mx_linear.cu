// Projections of microscaled operands on the tensor cores:
//   y[m][n] = sum over blocks b of 2^(sx[m][b] + sw[n][b]) * sum over k in b of x[m][k] * w[n][k]
// with float32 accumulation, plain or as silu(gate) * up of two weights.  Both operands may be e4m3 or
// e2m1 (tcgen05.mma kind::mxf8f6f4 with block scales takes any pairing; many rows of e2m1 by e2m1 use kind::mxf4).
//
// The weight is the 128-row operand of the instruction and the rows of x are its columns, so one
// kernel serves one row of x as well as thousands: the accumulator is [128 features][NT rows of x] in
// tensor memory, and a thread of the epilogue owns a feature.  Both operands are staged by bulk tensor
// copies, 128 elements of K at a time; a copy of e2m1 codes spreads sixteen of them over sixteen bytes
// of shared memory, the form the instruction reads.  A step's scales are one 512-byte copy per 128 rows and
// go on to tensor memory with tcgen05.cp.  With few output tiles K is split over the CTAs of a cluster,
// which add their accumulators through distributed shared memory in rank order.
//
// Every wait on a copy or another CTA's sums is bounded: one that runs out raises a status word and the kernel runs to its
// end.  The warp that issues the matrix instructions gives up first: the warps that copy wait several times as long
// for a stage that it frees, so that when one of them stops it has stopped long ago, and all stop at the same step, the ring's
// length after its last.  A CTA (or pair) ends only when every copy under way has landed and every matrix
// instruction is done.
//
// may_start_next() comes after a CTA has its tensor memory, so that a kernel let in early never holds columns
// that this one still needs.  The other way round, a kernel that waits for the one before it holds few columns (few
// rows: at most 256 to the half of an SM's shared memory) or allocates after the wait (many rows).
#include <cuda.h>

#include <algorithm>
#include <atomic>
#include <mutex>
#include <type_traits>

#include "fl_mx_common.cuh"

namespace fl {
namespace {

constexpr int kLinThreads = 192;
constexpr int kWaitTries = 1 << 15;  // of one wait, and for every step of K that it may have to sit through:
constexpr int kWaitTriesPerStep = 256;
constexpr int kCopierPatience = 4;  // times the tries of the waits between two stages that are freed
constexpr int kTileW = 128 * 128;  // bytes of a staged weight tile
constexpr int kMaxStages = 12;
constexpr int kMaxSplits = 8;
constexpr int kSmemLimit = 232448;
constexpr int kSmemPerSm = 233472;
constexpr int kSmemHalf = 112 * 1024;  // with the 1 KB that the system takes of each CTA, two fit an SM
constexpr int kTailBytes = 512;  // barriers and the tensor memory base

__device__ int g_mx_status;

enum OutKind { kOutBf16 = FL_DTYPE_BF16, kOutF16 = FL_DTYPE_F16, kOutF32 = FL_DTYPE_F32, kOutFp8 = 3, kOutFp4 = 4 };

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
// The tries of a wait that may sit through this many steps of K.
__device__ __forceinline__ int64_t tries_for(int steps) { return kWaitTries + int64_t(steps) * kWaitTriesPerStep; }
__device__ __forceinline__ void report_timeout() { atomicExch(&g_mx_status, 1); }
// Called by whole warps, whose lanes all get the same answer: what follows is uniform also where the tries ran out.
template <bool CLUSTER = false>
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int64_t tries = kWaitTries) {
  bool done = false;
  for (int64_t i = tries; i > 0 && !done; --i) done = mbar_try<CLUSTER>(bar, parity);
  if (__any_sync(0xffffffffu, done)) return true;
  report_timeout();
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
  // Waits for the last copies into every stage of a ring that stands here, the first round of which is over if `again`.
  __device__ __forceinline__ void drain(uint32_t full, int stages, bool again) const {
    for (int s = 0; s < stages; ++s) {
      const bool this_round = s < stage;
      if (this_round || again) mbar_wait(full + 8 * s, this_round ? parity : parity ^ 1);
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
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, uint32_t rank) {
  uint32_t a;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(addr), "r"(rank));
  return a;
}
// Four values into the shared memory of another CTA, counted by its barrier.
__device__ __forceinline__ void send16(uint32_t cluster_addr, const uint32_t* v, uint32_t cluster_bar) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%1, %2, %3, %4}, [%5];"
               ::"r"(cluster_addr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(cluster_bar) : "memory");
}
__device__ __forceinline__ void prefetch_l2(const void* p) {
  asm volatile("prefetch.global.L2 [%0];" ::"l"(p) : "memory");
}
__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// silu(g) * u.  The exponential and the quotient are the hardware's approximations: the exponential is documented to
// 2 + 1.17 |g| units in the last place, which is what one rounding of g does to it, so that the result is within
// (6 + 1.2 |g|) * 2^-23 of its formula, relative; where exp(-g) exceeds 2^126 (g below -87.3) the quotient is 0, of a
// true value below 1.1e-36.  The sums that g comes from are off by more, and the exact forms cost the epilogue more than
// the products take (gated 16384 x 2048 -> 5632: 421 us with expf and a rounded division, 265 us with these and without branches in the stores).
__device__ __forceinline__ float gated(float g, float u) { return __fdividef(g, 1.f + __expf(-g)) * u; }

// Where a product goes.
struct Output {
  void* data;       // [rows][features], or the codes of a microscaled result
  uint8_t* scales;  // of a microscaled result
  int features;
  int w_tiles;  // of 128 features
};

// Stores N rows of this thread's feature n, from row m on, of which `count` exist.  The 32 lanes of a
// warp hold 32 consecutive features, which are one block of a microscaled result; whole warps call it.
// WHOLE: all N rows exist.  That path has one branch at most: the epilogue of many rows is bound by the
// instructions of its warps.
template <int KIND, bool WHOLE, int N>
__device__ __forceinline__ void emit_rows(const Output& o, int64_t m, int n, const float (&v)[N], int count) {
  const bool live = n < o.features;
  if constexpr (KIND <= kOutF32) {
    using T = std::conditional_t<KIND == kOutBf16, __nv_bfloat16, std::conditional_t<KIND == kOutF16, __half, float>>;
    T* dst = static_cast<T*>(o.data) + m * o.features + n;
    if (live) {
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (WHOLE || j < count) dst[int64_t(j) * o.features] = round_to<T>(v[j]);
    }
  } else {
    // m is a multiple of N, a divisor of 32, so that the scales of these rows lie sixteen bytes apart
    static_assert(N % 4 == 0 && 32 % N == 0, "rows of one scale group, four to a word");
    constexpr int kFormat = KIND == kOutFp8 ? FL_MX_FP8 : FL_MX_FP4;
    const int lane = threadIdx.x & 31;
    const int64_t row_bytes = int64_t(o.w_tiles) * (KIND == kOutFp8 ? kMxStep : kMxStep / 2);
    float q[N];
    uint32_t mine = 0;  // the largest magnitude of row `lane`, which works out its scale for all
#pragma unroll
    for (int j = 0; j < N; ++j) {
      q[j] = live && (WHOLE || j < count) ? v[j] : 0.f;
      const uint32_t amax = __reduce_max_sync(0xffffffffu, __float_as_uint(q[j]) & 0x7fffffffu);
      mine = lane == j ? amax : mine;
    }
    const uint32_t byte = mx_scale_byte<kFormat>(mine);
    const float inv = mx_inverse(byte);
    const uint32_t bad = __ballot_sync(0xffffffffu, byte == 255u);
#pragma unroll
    for (int j = 0; j < N; ++j) q[j] *= __shfl_sync(0xffffffffu, inv, j);
    if (bad != 0) {  // a block that is not finite has codes 0
#pragma unroll
      for (int j = 0; j < N; ++j) q[j] = bad >> j & 1 ? 0.f : q[j];
    }
    if (lane < (WHOLE ? N : min(N, count)))
      o.scales[mx_scale_offset(m, n / kMxStep, o.w_tiles) + lane * 16 + n / kMxBlock % 4] = uint8_t(byte);
    if constexpr (KIND == kOutFp8) {
      // The codes of four rows in a word, then a 4 x 4 transposition of bytes within each four lanes: a lane
      // has four features of row (lane % 4) and stores them at once.
      uint8_t* codes = static_cast<uint8_t*>(o.data) + (m + (lane & 3)) * row_bytes + (n & ~3);
#pragma unroll
      for (int j = 0; j < N; j += 4) {
        uint32_t x = __byte_perm(cvt_e4m3x2(q[j], q[j + 1]), cvt_e4m3x2(q[j + 2], q[j + 3]), 0x5410);
        x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 1), lane & 1 ? 0x3715 : 0x6240);
        x = __byte_perm(x, __shfl_xor_sync(0xffffffffu, x, 2), lane & 2 ? 0x3276 : 0x5410);
        if (WHOLE || j + (lane & 3) < count) *reinterpret_cast<uint32_t*>(codes + j * row_bytes) = x;
      }
    } else {
      uint8_t* codes = static_cast<uint8_t*>(o.data) + m * row_bytes + n / 2;
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const float odd = __shfl_down_sync(0xffffffffu, q[j], 1);
        if ((n & 1) == 0 && (WHOLE || j < count)) codes[j * row_bytes] = uint8_t(cvt_e2m1x2(q[j], odd));
      }
    }
  }
}
// The scales of the result's last tile past its last row, for 128 features from n0 on: zero.
__device__ __forceinline__ void zero_scales(const Output& o, int64_t rows, int n0, int thread, int threads) {
  const int64_t end = (rows + kMxTileRows - 1) / kMxTileRows * kMxTileRows;
  for (int64_t r = rows + thread; r < end; r += threads)
    *reinterpret_cast<uint32_t*>(o.scales + mx_scale_offset(r, n0 / kMxStep, o.w_tiles)) = 0u;
}

struct LinearParams {
  const uint8_t *x_scales, *w_scales[2], *w_codes[2];
  int w_row_step;  // bytes of a row of the weight's codes per step
  Output out;
  int64_t rows;
  int steps;   // of K
  int stages;  // of the shared-memory ring
  uint32_t w_bytes, x_bytes;  // that the copies of one step's tiles report: a spread e2m1 tile counts as packed
  uint32_t idesc;
  uint32_t tmem_cols;
  int give_up;  // step of a CTA's share whose copies are taken not to come (tests; never in its share otherwise)
};

// Shared memory of the kernel for few rows.
template <int NT, bool DUAL>
struct FewRows {
  static constexpr int kWeights = DUAL ? 2 : 1;
  static constexpr int kXBytes = NT * 128;
  static constexpr int kScalesAt = kWeights * kTileW + kXBytes;
  static constexpr int kStageBytes = (kScalesAt + (kWeights + 1) * kMxTileBytes + 1023) / 1024 * 1024;
  static constexpr uint32_t kScaleCols = 4 * (kWeights + 1);  // tensor memory columns of a stage's scales
  // groups of four columns of the accumulator that a CTA of a split finishes, and the shared memory in which
  // it receives them from every CTA of its cluster: [source][weight][group][feature][column of the group]
  static constexpr __host__ __device__ int groups(int splits, int cols) {
    return ((cols + 3) / 4 + splits - 1) / splits;
  }
  static int exchange_bytes(int splits, int cols) {
    return splits > 1 ? splits * kWeights * groups(splits, cols) * 2048 : 0;
  }
};

// Few rows of x: a CTA computes 128 features by NT rows over its share of K.  What such a call
// takes is latency, so the copies start before anything else, issued by four warps, and a split sends
// its sums straight into the shared memory of the CTA that finishes them, which waits for their bytes.
template <int KIND, int NT, bool DUAL>
__global__ void __launch_bounds__(kLinThreads, 1)
mx_linear_kernel(const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w0,
                 const __grid_constant__ CUtensorMap map_w1, const LinearParams p) {
  using Shape = FewRows<NT, DUAL>;
  constexpr int kWeights = Shape::kWeights, kStageBytes = Shape::kStageBytes, kScalesAt = Shape::kScalesAt;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = raw_smem + (1024 - (smem_addr(raw_smem) & 1023)) % 1024;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + p.stages * kStageBytes);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kMaxStages + 2);
  float4* exchange = reinterpret_cast<float4*>(smem + p.stages * kStageBytes + kTailBytes);
  const uint32_t ring = smem_addr(smem), full = smem_addr(bars), empty = full + 8 * kMaxStages,
                 done = empty + 8 * kMaxStages, received = done + 8;
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = threadIdx.x & 31;
  const int splits = int(cluster_size()), rank = int(cluster_rank());
  const int tile = blockIdx.x / splits;
  const int x_tile = tile / p.out.w_tiles, w_tile = tile - x_tile * p.out.w_tiles;
  const int row0 = x_tile * NT;  // NT < 128 only where there is one tile of x or NT divides 128
  const int first = p.steps * rank / splits, last = p.steps * (rank + 1) / splits;

  const int cols = int(min(int64_t(NT), p.rows - row0));
  const int groups = Shape::groups(splits, cols);  // that each CTA of a split finishes
  const int my_groups = max(0, min(groups, (cols + 3) / 4 - rank * groups));

  if (warp == 0) {
    if (lane < p.stages) {
      mbar_init(full + 8 * lane, 4);  // the four warps that copy
      mbar_init(empty + 8 * lane, 1);
    } else if (lane == 30) {
      mbar_init(done, 1);
    } else if (lane == 31) {
      mbar_init(received, 1);
      if (splits > 1) mbar_expect(received, uint32_t(splits * kWeights * my_groups) * 2048);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  } else if (warp == 1) {
    if (lane == 0) {
      prefetch_map(&map_w0);
      prefetch_map(&map_x);
      if (DUAL) prefetch_map(&map_w1);
    }
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                 "r"(p.tmem_cols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // The weight on its way into the L2 cache, which is harmless whoever still writes it.
  {
    const int row_lines = ((last - first) * p.w_row_step + 127) / 128;
    for (int i = threadIdx.x; i < 128 * row_lines; i += kLinThreads) {
      const int row = w_tile * 128 + i / row_lines;
      const int64_t at = (int64_t(row) * p.steps + first) * p.w_row_step + i % row_lines * 128;
      if (row < p.out.features) {
        prefetch_l2(p.w_codes[0] + at);
        if (DUAL) prefetch_l2(p.w_codes[1] + at);
      }
    }
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  wait_for_inputs();
  may_start_next();
  if (splits > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");  // this CTA runs

  if (warp == 0 || (warp >= 2 && warp <= 4)) {
    // warp 0: weight tiles; 2: rows of x; 3: scales of x; 4: scales of the weights
    const uint8_t* x_scales = p.x_scales + int64_t(row0 / kMxTileRows) * p.steps * kMxTileBytes;
    const int64_t w_scales_at = int64_t(w_tile) * p.steps * kMxTileBytes;
    const int end = min(last, first + p.give_up + p.stages);
    Ring ring_at;
    int k = first;
    for (; k < end; ++k, ring_at.advance(p.stages)) {
      const int s = ring_at.stage;
      if (k - first >= p.stages && !mbar_wait(empty + 8 * s, ring_at.parity ^ 1, kCopierPatience * kWaitTries)) break;
      const uint32_t at = ring + s * kStageBytes, bar = full + 8 * s;
      if (elect_one()) {
        if (warp == 0) {
          mbar_expect(bar, kWeights * p.w_bytes);
          copy_tile(at, &map_w0, k * kMxStep, w_tile * 128, bar);
          if (DUAL) copy_tile(at + kTileW, &map_w1, k * kMxStep, w_tile * 128, bar);
        } else if (warp == 2) {
          mbar_expect(bar, p.x_bytes);
          copy_tile(at + kWeights * kTileW, &map_x, k * kMxStep, row0, bar);
        } else if (warp == 3) {
          mbar_expect(bar, kMxTileBytes);
          copy_bytes(at + kScalesAt + kWeights * kMxTileBytes, x_scales + int64_t(k) * kMxTileBytes, kMxTileBytes, bar);
        } else {
          mbar_expect(bar, kWeights * kMxTileBytes);
          for (int i = 0; i < kWeights; ++i)
            copy_bytes(at + kScalesAt + i * kMxTileBytes, p.w_scales[i] + w_scales_at + int64_t(k) * kMxTileBytes,
                       kMxTileBytes, bar);
        }
      }
      __syncwarp();
    }
    if (warp == 0) ring_at.drain(full, p.stages, k - first >= p.stages);  // a stage is full when all four have copied
  } else if (warp == 1) {
    const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
    const uint32_t tmem_scales = tmem + NT * kWeights;
    // scales of x: NT rows of a 128-row tile start at its column (row0 % 128) / 32, an even one
    const uint32_t x_col = 4 * kWeights + uint32_t(row0 % kMxTileRows) / 32;
    const int end = min(last, first + p.give_up);
    Ring ring_at;
    for (int k = first; k < end; ++k, ring_at.advance(p.stages)) {
      const int s = ring_at.stage;
      if (!mbar_wait(full + 8 * s, ring_at.parity)) break;
      const uint32_t at = ring + s * kStageBytes, scales = at + kScalesAt;
      const uint32_t sf = tmem_scales + s * Shape::kScaleCols;
      const uint64_t x_desc = tile_desc(at + kWeights * kTileW);
      if (elect_one()) {
#pragma unroll
        for (int t = 0; t < kWeights + 1; ++t) scales_to_tmem(sf + 4 * t, scales + t * kMxTileBytes);
#pragma unroll
        for (int w = 0; w < kWeights; ++w) {
          const uint64_t w_desc = tile_desc(at + w * kTileW);
#pragma unroll
          for (int b = 0; b < 4; ++b)  // a block of 32 elements is 32 bytes along the swizzled row
            mma_mx(tmem + w * NT, w_desc + 2 * b, x_desc + 2 * b, p.idesc | uint32_t(b) << 29 | uint32_t(b) << 4,
                   sf + 4 * w, sf + x_col, k > first || b > 0);
        }
        commit_to(empty + 8 * s);
      }
      __syncwarp();
    }
    if (end < last) report_timeout();
    if (elect_one()) commit_to(done);
    __syncwarp();
    mbar_wait(done, 0, tries_for(p.steps));  // every product is done before tensor memory is given back
  }
  __syncwarp();

  const int n = w_tile * 128 + (warp & 3) * 32 + lane;
  if (warp >= 2) {
    const uint32_t acc = __shfl_sync(0xffffffffu, *tmem_slot, 0) + (uint32_t(warp & 3) * 32 << 16);
    mbar_wait(done, 0, tries_for(p.steps));
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    if (splits > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");  // all of the cluster run
    const int feature = (warp & 3) * 32 + lane;
    const uint32_t slot = smem_addr(exchange) + uint32_t(rank * kWeights * groups * 128 + feature) * 16;
#pragma unroll
    for (int c = 0; c < NT; c += 16) {
      if (c >= cols) break;
      uint32_t a[16], b[16];
      tmem_load16(acc + c, a);
      if (DUAL) tmem_load16(acc + NT + c, b);
      asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
      if (splits > 1) {
#pragma unroll
        for (int j = 0; j < 16; j += 4) {
          if (c + j < cols) {
            const int group = (c + j) / 4, owner = group / groups, at = group - owner * groups;
            const uint32_t bar = in_cta(received, uint32_t(owner));
            const uint32_t dst = in_cta(slot + uint32_t(at) * 2048, uint32_t(owner));
            send16(dst, a + j, bar);
            if (DUAL) send16(dst + uint32_t(groups) * 2048, b + j, bar);
          }
        }
      } else {
        float v[16];
#pragma unroll
        for (int j = 0; j < 16; ++j)
          v[j] = DUAL ? gated(__uint_as_float(a[j]), __uint_as_float(b[j])) : __uint_as_float(a[j]);
        if (c + 16 <= cols) {
          emit_rows<KIND, true>(p.out, row0 + c, n, v, 16);
        } else {
          emit_rows<KIND, false>(p.out, row0 + c, n, v, cols - c);
        }
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    if (splits > 1 && my_groups > 0) {
      // The other CTAs always send, also after a wait of theirs has run out: wait as long as they may take.
      for (int i = 0; i < 16 && !mbar_wait<true>(received, 0, tries_for(p.steps)); ++i) {
      }
      for (int g = 0; g < my_groups; ++g) {
        const float4* src = exchange + g * 128 + feature;
        float v[4] = {}, u[4] = {};
#pragma unroll
        for (int r = 0; r < kMaxSplits; ++r) {  // in rank order
          if (r < splits) {
            const float4 t = src[r * kWeights * groups * 128];
            v[0] += t.x; v[1] += t.y; v[2] += t.z; v[3] += t.w;
            if (DUAL) {
              const float4 w = src[(r * kWeights + 1) * groups * 128];
              u[0] += w.x; u[1] += w.y; u[2] += w.z; u[3] += w.w;
            }
          }
        }
        if (DUAL) {
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] = gated(v[j], u[j]);
        }
        const int c = (rank * groups + g) * 4;
        if (c + 4 <= cols) {
          emit_rows<KIND, true>(p.out, row0 + c, n, v, 4);
        } else {
          emit_rows<KIND, false>(p.out, row0 + c, n, v, cols - c);
        }
      }
    }
  } else if (splits > 1) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  }
  if (KIND > kOutF32 && rank == 0 && row0 + NT >= p.rows) zero_scales(p.out, p.rows, w_tile * 128, threadIdx.x, kLinThreads);
  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(*tmem_slot), "r"(p.tmem_cols) : "memory");
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
//
// PACKED: both operands are e2m1.  They stay packed in shared memory, 256 elements to a stage, and go through
// kind::mxf4, 64 elements an instruction at twice the rate (32768 x 5632 -> 2048: 139 us = 5440 TFLOP/s against 257 us
// with x in mxfp8; gated 16384 x 2048 -> 5632: 164 against 266 us).

// Warps of the epilogue: with a gate to work out sixteen are faster than eight, without one slower (16384 x 2048 -> 5632
// to mxfp8: 275 us with sixteen, 288 with eight, of 4-bit operands 177 and 235; 32768 x 2048 -> 6144: 325 us with sixteen, 292
// with eight).
template <bool DUAL>
constexpr int kPairEpilogue = DUAL ? 16 : 8;
template <bool DUAL>
constexpr int kPairThreads = 64 + 32 * kPairEpilogue<DUAL>;  // and one each for copies and matrix instructions
// NT: rows of x per tile.  A multiple of 64, as the scales of x start at an even column of tensor memory.
constexpr int kPairRows = 192;
constexpr int kPairXTiles = 2;  // scale tiles that 192 rows starting at a multiple of 64 touch
constexpr int kPairXBytes = kPairRows / 2 * 128;
constexpr int kPairScalesAt = kTileW + kPairXBytes;

template <bool PACKED>
struct Pair {
  static constexpr int kSteps = PACKED ? 2 : 1;  // of K in a stage
  // scales of a stage, in shared memory and in tensor memory: those of the weight step by step, then those of x
  static constexpr int kScaleTiles = kSteps * (1 + kPairXTiles);
  static constexpr uint32_t kScaleCols = 4 * kScaleTiles;
  static constexpr int kStageBytes = (kPairScalesAt + kScaleTiles * kMxTileBytes + 1023) / 1024 * 1024;
  static constexpr int kStages = PACKED ? 5 : 7;
  static_assert(2 * kPairRows + kStages * kScaleCols <= 512, "tensor memory columns");
  static_assert(1024 + kStages * kStageBytes + kTailBytes <= kSmemLimit, "shared memory");
};
static_assert(kPairXBytes % 1024 == 0, "tiles need 1024-byte alignment");

struct PairMaps {
  CUtensorMap x, x_scales, w[2], w_scales[2];
};

struct PairParams {
  Output out;
  int64_t rows;
  int steps;
  int pair_tiles;    // of 256 features
  int64_t units;     // tiles times weights
  uint32_t stage_bytes;  // that the copies of one stage report, both CTAs
  uint32_t idesc;
  int give_up;  // use of a stage by a pair whose copies are taken not to come (tests)
};

__device__ __forceinline__ void copy_tile_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint32_t smem) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(scale_desc(smem)) : "memory");
}
template <bool PACKED>
__device__ __forceinline__ void mma_mx_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                            uint32_t accumulate) {
  if constexpr (PACKED) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X [%0], %1, %2, %3, [%4], [%5], p;\n\t}"
        ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate) : "memory");
  }
}
// Arrives on the barrier at this offset in both CTAs once every matrix instruction issued so far is done.
__device__ __forceinline__ void commit_to_both(uint32_t bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
      ::"r"(bar), "h"(uint16_t(3)) : "memory");
}
// ... and on that of this CTA alone: the other one may be gone when it comes.
__device__ __forceinline__ void commit_here(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

template <int KIND, bool DUAL, bool PACKED>
__global__ void __launch_bounds__(kPairThreads<DUAL>)
mx_linear_pair_kernel(const __grid_constant__ PairMaps maps, const PairParams p) {
  using Shape = Pair<PACKED>;
  constexpr int kStages = Shape::kStages, kStageBytes = Shape::kStageBytes, kSteps = Shape::kSteps;
  extern __shared__ uint8_t raw_smem[];
  uint8_t* smem = raw_smem + (1024 - (smem_addr(raw_smem) & 1023)) % 1024;
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + kStages * kStageBytes);
  const uint32_t ring = smem_addr(smem), full = smem_addr(bars), empty = full + 8 * kStages,
                 acc_full = empty + 8 * kStages, acc_empty = acc_full + 16, drained = acc_empty + 16;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * kStages + 5);
  const int warp = __shfl_sync(0xffffffffu, int(threadIdx.x) / 32, 0), lane = threadIdx.x & 31;
  const uint32_t rank = cluster_rank();
  const int64_t pairs = gridDim.x / 2, pair = blockIdx.x / 2;
  constexpr int kWeights = DUAL ? 2 : 1;

  wait_for_inputs();
  if (warp == 0) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)), "r"(512u)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
  if (threadIdx.x == 32) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full + 8 * b, 1);
      mbar_init(acc_empty + 8 * b, 2 * kPairEpilogue<DUAL>);  // a lane of each epilogue warp of both CTAs
    }
    mbar_init(drained, 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  cluster_sync();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  may_start_next();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);
  const uint32_t tmem_scales = tmem + 2 * kPairRows;

  // unit u of this pair: tile t = pair + (u / kWeights) * pairs, weight u % kWeights, features fastest
  if (warp == 0) {
    const uint32_t leader_full = in_cta(full, 0);
    Ring ring_at;
    bool ok = true, again = false;  // again: the ring has been filled once
    int64_t left = int64_t(p.give_up) + kStages;  // uses of stages
    for (int64_t unit = pair * kWeights; ok && unit < p.units;
         unit += (DUAL && (unit & 1) == 0) ? 1 : pairs * kWeights - (DUAL ? 1 : 0)) {
      const int64_t tile = unit / kWeights;
      const int which = int(unit % kWeights);
      const int w_tile = int(tile % p.pair_tiles) * 2 + int(rank);
      const int row0 = int(tile / p.pair_tiles) * kPairRows;
      const int end = int(min(int64_t(p.steps), left * kSteps));
      left -= (p.steps + kSteps - 1) / kSteps;
      ok = end == p.steps;
      for (int k = 0; k < end; k += kSteps) {
        const int s = ring_at.stage;
        if (again && !mbar_wait(empty + 8 * s, ring_at.parity ^ 1, kCopierPatience * tries_for(p.steps))) {
          ok = false;
          break;
        }
        const uint32_t at = ring + s * kStageBytes, bar = leader_full + 8 * s;
        if (elect_one()) {
          if (rank == 0) mbar_expect(full + 8 * s, p.stage_bytes);
          // packed codes are copied as bytes, two elements each
          const int at_k = PACKED ? k * (kMxStep / 2) : k * kMxStep;
          copy_tile_pair(at, &maps.w[which], at_k, w_tile * 128, bar);
          copy_tile_pair(at + kTileW, &maps.x, at_k, row0 + int(rank) * (kPairRows / 2), bar);
          uint32_t scales = at + kPairScalesAt;
#pragma unroll
          for (int j = 0; j < kSteps; ++j, scales += kMxTileBytes)
            copy_tile_pair(scales, &maps.w_scales[which], 0, w_tile * p.steps + k + j, bar);
#pragma unroll
          for (int j = 0; j < kSteps; ++j)
#pragma unroll
            for (int i = 0; i < kPairXTiles; ++i, scales += kMxTileBytes)
              copy_tile_pair(scales, &maps.x_scales, 0, (row0 / kMxTileRows + i) * p.steps + k + j, bar);
        }
        __syncwarp();
        ring_at.advance(kStages);
        again |= ring_at.stage == 0;
      }
    }
    // leave only when every copy of the pair has landed: the stages of this round, then those of the last
    if (rank == 0) ring_at.drain(full, kStages, again);
  } else if (warp == 1 && rank == 0) {
    Ring ring_at, acc_at;
    bool ok = true, again = false;
    int64_t left = p.give_up;
    for (int64_t unit = pair * kWeights; ok && unit < p.units;
         unit += (DUAL && (unit & 1) == 0) ? 1 : pairs * kWeights - (DUAL ? 1 : 0)) {
      const int buffer = acc_at.stage;
      const int row0 = int(unit / kWeights / p.pair_tiles) * kPairRows;
      if (again && !mbar_wait<true>(acc_empty + 8 * buffer, acc_at.parity ^ 1, tries_for(p.steps))) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t acc = tmem + buffer * kPairRows;
      const int end = int(min(int64_t(p.steps), left * kSteps));
      left -= (p.steps + kSteps - 1) / kSteps;
      ok = end == p.steps;
      if (!ok) report_timeout();
      for (int k = 0; k < end; k += kSteps, ring_at.advance(kStages)) {
        const int s = ring_at.stage;
        if (!mbar_wait(full + 8 * s, ring_at.parity)) {
          ok = false;
          break;
        }
        const uint32_t at = ring + s * kStageBytes, scales = at + kPairScalesAt;
        const uint32_t sf = tmem_scales + uint32_t(s) * Shape::kScaleCols;
        const uint64_t w_desc = tile_desc(at), x_desc = tile_desc(at + kTileW);
        const uint32_t sfb = sf + 4 * kSteps + (row0 % kMxTileRows) / 32;
        if (elect_one()) {
#pragma unroll
          for (int t = 0; t < Shape::kScaleTiles; ++t) scales_to_tmem_pair(sf + 4 * t, scales + t * kMxTileBytes);
          // Four instructions of 32 bytes along the swizzled row: a block each, or packed two blocks, of which a step
          // has two pairs.  What lies past the last step of a stage is not multiplied (its scales are another tile's).
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            const uint32_t step = PACKED ? b / 2 : 0, block = PACKED ? b % 2 * 2 : b;
            if (!PACKED || b < 2 || k + 1 < p.steps)
              mma_mx_pair<PACKED>(acc, w_desc + 2 * b, x_desc + 2 * b, p.idesc | block << 29 | block << 4, sf + 4 * step,
                                  sfb + 4 * kPairXTiles * step, k > 0 || b > 0);
          }
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
    if (elect_one()) commit_here(drained);
    __syncwarp();
    mbar_wait(drained, 0, tries_for(p.steps));
  } else if (warp >= 2) {
    const uint32_t quarter = uint32_t(warp & 3) * 32, part = uint32_t(warp - 2) / 4;
    constexpr int kCols = kPairRows / (kPairEpilogue<DUAL> / 4);  // this warp's columns of a tile
    const uint32_t mine = tmem + (quarter << 16) + part * kCols;
    const uint32_t leader_empty = in_cta(acc_empty, 0);
    Ring acc_at;
    for (int64_t tile = pair; tile < p.units / kWeights; tile += pairs) {
      const int n0 = (int(tile % p.pair_tiles) * 2 + int(rank)) * 128;
      const int n = n0 + int(quarter) + lane;
      const int64_t m0 = tile / p.pair_tiles * kPairRows + part * kCols;
      const int cols = n0 < p.out.features ? int(max(int64_t(0), min(int64_t(kCols), p.rows - m0))) : 0;
      const bool whole = cols == kCols;
      float gate[DUAL ? kCols : 1];
      if constexpr (DUAL) {
        const int buffer = acc_at.stage;
        if (!mbar_wait(acc_full + 8 * buffer, acc_at.parity, tries_for(2 * p.steps))) break;
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
      if (!mbar_wait(acc_full + 8 * buffer, acc_at.parity, tries_for(2 * p.steps))) break;
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
          emit_rows<KIND, true>(p.out, m0 + c, n, v, 16);
        } else if (c < cols) {
          emit_rows<KIND, false>(p.out, m0 + c, n, v, cols - c);
        }
      }
      acc_at.advance(2);
      if (KIND > kOutF32 && n0 < p.out.features && m0 <= p.rows && p.rows <= m0 + kCols)
        zero_scales(p.out, p.rows, n0, int(quarter) + lane, 128);
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

// Codes [rows][steps * 128] as boxes of 128 elements by box_rows rows in the 128-byte swizzle, or, packed, of 128
// bytes of e2m1; rows past the last and bytes past the end of a row read as zero.
bool make_map(CUtensorMap* map, const void* codes, int format, int64_t rows, int64_t steps, int box_rows,
              bool packed = false) {
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr) return false;
  const bool fp8 = format == FL_MX_FP8;
  const cuuint64_t dims[2] = {cuuint64_t(steps * (packed ? kMxStep / 2 : kMxStep)), cuuint64_t(rows)};
  const cuuint64_t strides[1] = {cuuint64_t(steps * (fp8 ? kMxStep : kMxStep / 2))};
  const cuuint32_t box[2] = {kMxStep, cuuint32_t(box_rows)};
  const cuuint32_t unit[2] = {1, 1};
  return encode(map, fp8 || packed ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B, 2,
                const_cast<void*>(codes), dims, strides, box, unit, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

constexpr int kMaxDevices = 64;

// Lets a kernel use all of an SM's shared memory, once per device.
template <typename K>
cudaError_t allow_shared_memory(K kernel, std::atomic<bool> (&done)[kMaxDevices], int device) {
  if (done[device].load(std::memory_order_acquire)) return cudaSuccess;
  const cudaError_t err = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
  if (err == cudaSuccess) done[device].store(true, std::memory_order_release);
  return err;
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
  int device;
};

// Step at which the kernels launched by this thread give up: none, but in tests.  More than any share has, and
// 32 bits hold it with a share's first step and a ring's stages added.
constexpr int kNever = 1 << 30;
thread_local int t_give_up = kNever;

template <int KIND, int NT, bool DUAL>
int launch_linear(const LinearCall& call, int splits, int smem_limit) {
  using Shape = FewRows<NT, DUAL>;
  const int steps = int(mx_steps(call.cols));
  LinearParams p;
  p.x_scales = static_cast<const uint8_t*>(call.x.scales);
  p.w_scales[0] = static_cast<const uint8_t*>(call.w[0].scales);
  p.w_scales[1] = static_cast<const uint8_t*>(call.w[1].scales);
  p.w_codes[0] = static_cast<const uint8_t*>(call.w[0].codes);
  p.w_codes[1] = static_cast<const uint8_t*>(call.w[1].codes);
  p.w_row_step = call.w[0].format == FL_MX_FP8 ? kMxStep : kMxStep / 2;
  p.out = Output{call.out, static_cast<uint8_t*>(call.out_scales), call.features, (call.features + 127) / 128};
  p.rows = call.rows;
  p.steps = steps;
  p.w_bytes = uint32_t(kTileW >> (call.w[0].format == FL_MX_FP8 ? 0 : 1));
  p.x_bytes = uint32_t(Shape::kXBytes >> (call.x.format == FL_MX_FP8 ? 0 : 1));
  const int exchange = Shape::exchange_bytes(splits, int(std::min<int64_t>(NT, call.rows)));
  const int room = (smem_limit - 1024 - kTailBytes - exchange) / Shape::kStageBytes;
  p.stages = std::min({kMaxStages, room, (steps + splits - 1) / splits});
  const int need = NT * Shape::kWeights + p.stages * int(Shape::kScaleCols);
  p.tmem_cols = need <= 32 ? 32 : need <= 64 ? 64 : need <= 128 ? 128 : need <= 256 ? 256 : 512;
  // Shared memory in proportion to the columns: CTAs of these kernels that fit an SM together never want more
  // than its 512 columns, so none waits for columns while its cluster waits for it.  Half of an SM's at least, which
  // keeps kernels that fill an SM (a library's matrix product before this one or on another stream, which may wait
  // for columns in the same way) from sharing it.
  const int smem = std::max({1024 + kTailBytes + p.stages * Shape::kStageBytes + exchange,
                             int(p.tmem_cols) * (kSmemPerSm / 512) - 1024, kSmemHalf});
  p.give_up = t_give_up;
  // instruction descriptor: element types (e4m3 0, e2m1 5), e8m0 scales, N, M = 128
  p.idesc = uint32_t(call.w[0].format == FL_MX_FP8 ? 0 : 5) << 7 | uint32_t(call.x.format == FL_MX_FP8 ? 0 : 5) << 10 |
            uint32_t(NT / 8) << 17 | 1u << 23 | uint32_t(128 / 16) << 24;
  CUtensorMap map_x, map_w0, map_w1;
  bool ok = make_map(&map_x, call.x.codes, call.x.format, call.rows, steps, NT) &&
            make_map(&map_w0, call.w[0].codes, call.w[0].format, call.features, steps, 128);
  if (DUAL) {
    ok = ok && make_map(&map_w1, call.w[1].codes, call.w[1].format, call.features, steps, 128);
  } else {
    map_w1 = map_w0;
  }
  FL_REQUIRE(ok, "%s: the operands cannot be described as tensor maps", call.who);
  const int64_t tiles = (call.rows + NT - 1) / NT * p.out.w_tiles;
  FL_REQUIRE(tiles * splits < (int64_t(1) << 31), "%s: too many elements", call.who);
  auto kernel = mx_linear_kernel<KIND, NT, DUAL>;
  static std::atomic<bool> allowed[kMaxDevices];
  cudaError_t err = allow_shared_memory(kernel, allowed, call.device);
  if (err == cudaSuccess)
    err = launch_overlapped(kernel, unsigned(tiles * splits), kLinThreads, smem, splits, call.stream, map_x, map_w0, map_w1, p);
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

template <int KIND, bool DUAL, bool PACKED>
int launch_pairs(const LinearCall& call, int sms) {
  using Shape = Pair<PACKED>;
  const int steps = int(mx_steps(call.cols));
  PairMaps maps;
  PairParams p;
  p.out = Output{call.out, static_cast<uint8_t*>(call.out_scales), call.features, (call.features + 127) / 128};
  p.rows = call.rows;
  p.steps = steps;
  p.pair_tiles = (call.features + 255) / 256;
  const int64_t tiles = (call.rows + kPairRows - 1) / kPairRows * p.pair_tiles;
  p.units = tiles * (DUAL ? 2 : 1);
  p.give_up = t_give_up;
  const bool w_spread = !PACKED && call.w[0].format == FL_MX_FP4, x_spread = !PACKED && call.x.format == FL_MX_FP4;
  p.stage_bytes = 2 * uint32_t((kTileW >> int(w_spread)) + (kPairXBytes >> int(x_spread)) + Shape::kScaleTiles * kMxTileBytes);
  // element types as in launch_linear, or e2m1 of kind::mxf4 (1)
  const uint32_t w_type = PACKED ? 1 : w_spread ? 5 : 0, x_type = PACKED ? 1 : x_spread ? 5 : 0;
  p.idesc = w_type << 7 | x_type << 10 | uint32_t(kPairRows / 8) << 17 | 1u << 23 | uint32_t(256 / 16) << 24;
  bool ok = make_map(&maps.x, call.x.codes, call.x.format, call.rows, steps, kPairRows / 2, PACKED) &&
            make_scale_map(&maps.x_scales, call.x.scales, call.rows, steps);
  for (int i = 0; i < (DUAL ? 2 : 1); ++i) {
    const Operand& w = call.w[i];
    ok = ok && make_map(&maps.w[i], w.codes, w.format, call.features, steps, 128, PACKED) &&
         make_scale_map(&maps.w_scales[i], w.scales, call.features, steps);
  }
  if (!DUAL) {
    maps.w[1] = maps.w[0];
    maps.w_scales[1] = maps.w_scales[0];
  }
  FL_REQUIRE(ok, "%s: the operands cannot be described as tensor maps", call.who);
  FL_REQUIRE(int64_t(p.out.w_tiles + 2) * steps < (int64_t(1) << 31) &&
                 (call.rows / kMxTileRows + kPairXTiles + 1) * steps < (int64_t(1) << 31),
             "%s: too many elements", call.who);
  auto kernel = mx_linear_pair_kernel<KIND, DUAL, PACKED>;
  static std::atomic<bool> allowed[kMaxDevices];
  cudaError_t err = allow_shared_memory(kernel, allowed, call.device);
  // all of an SM's shared memory, as it takes all of its tensor memory (see above)
  if (err == cudaSuccess)
    err = launch_overlapped(kernel, unsigned(2 * std::min<int64_t>(tiles, sms / 2)), kPairThreads<DUAL>, kSmemLimit, 2, call.stream,
                            maps, p);
  if (err != cudaSuccess) {
    cudaGetLastError();
    set_error("%s: %s", call.who, cudaGetErrorString(err));
    return FL_ERR_CUDA;
  }
  return FL_OK;
}

// Never launched: asked about for the kernels below, for which the driver counts one CTA to an SM
// whatever their shared memory, although two run there (as seen from %smid and %globaltimer).
__global__ void __launch_bounds__(kLinThreads) cluster_probe_kernel() {}

// Multiprocessors of a device and, for every cluster size, how many clusters run at once of CTAs that take
// all of an SM's shared memory and of CTAs that take half (the GPU's processor groups do not divide evenly).
struct Device {
  int sms;
  int clusters[2][kMaxSplits + 1];
};
const Device& device_limits(int device) {
  static Device limits[kMaxDevices];
  static std::once_flag once[kMaxDevices];
  std::call_once(once[device], [device] {
    Device& d = limits[device];
    d.sms = 0;
    if (cudaDeviceGetAttribute(&d.sms, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || d.sms <= 0) d.sms = 148;
    auto kernel = cluster_probe_kernel;
    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemLimit);
    for (int half = 0; half < 2; ++half) {
      for (int size = 1; size <= kMaxSplits; ++size) {
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(unsigned(size));
        config.blockDim = dim3(kLinThreads);
        config.dynamicSmemBytes = half ? kSmemHalf : kSmemLimit;
        cudaLaunchAttribute attribute;
        attribute.id = cudaLaunchAttributeClusterDimension;
        attribute.val.clusterDim.x = size;
        attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
        config.attrs = &attribute;
        config.numAttrs = 1;
        if (cudaOccupancyMaxActiveClusters(&d.clusters[half][size], kernel, &config) != cudaSuccess)
          d.clusters[half][size] = 0;
      }
    }
    cudaGetLastError();
  });
  return limits[device];
}

// How a call is cut, by its tiles of 128 features by NT rows and its steps of K:
// - up to 32 rows (16 of a gated product, whose stages are twice as large), CTAs take half of an SM's shared memory, so
//   that two fit an SM and the next kernel's can set up beside the last ones of this; K is split while that gives at most three CTAs to two SMs and three steps to a CTA
//   (16 rows, mxfp4, weights not in L2; 2048 -> 6144: split two ways with all of the shared memory 4.7 us, two ways
//   with half 4.8, three 4.4, four 4.1, five 4.5; 2048 -> 2048: four 3.4, six 3.3, eight 3.4; 5632 -> 2048: four
//   5.2, six 4.5, eight 4.3; gated 2048 -> 5632: two with all 7.0, three with all 6.7, five with half 6.5);
// - with more rows CTAs take all of an SM's shared memory, and K is split while that leaves a third of the SMs idle (none
//   up to 32 rows).  The exchange of the sums takes longer the more rows there are, so that it has to save some
//   rows / 8 steps, of which a two-way split saves only half (warm weights; 2048 -> 2048: 64 rows whole 5.7 us, six
//   ways 4.8, 96 rows 6.6 and 5.9, 128 rows 7.0 and 7.7, 128 rows of 4096 -> 2048 10.2 and 8.5; 2048 -> 6144: 40 rows
//   whole 5.9, two ways 5.5, 64 rows 5.8 and 6.3; gated 1000 -> 2048: 40 rows whole 6.9, five ways 5.3);
// - never more than run at once: a cluster that waits for another to end doubles the call (2048 -> 6144
//   split three ways with all of the shared memory: 7.8 us);
// - pairs of CTAs once tiles of 128 rows (64 of a gated product) no longer run at once (2048 -> 6144: 384 rows 8.5 us
//   either way, 512 rows 15.0 in tiles and 9.0 in pairs, 256 rows 7.8 and 8.8; gated 2048 -> 5632: 192 rows 13.0
//   and 18.3, 256 rows 24.2 and 18.2).
template <int KIND, bool DUAL>
int choose_linear(const LinearCall& call) {
  const Device& device = device_limits(call.device);
  const int sms = device.sms;
  const int steps = int(mx_steps(call.cols));
  const int64_t w_tiles = (call.features + 127) / 128;
  auto run = [&](auto nt, bool half) {
    constexpr int kRows = decltype(nt)::value;
    const int64_t tiles = (call.rows + kRows - 1) / kRows * w_tiles;
    const int64_t most = half ? sms * 3 / 2 : kRows <= 32 ? sms : sms * 2 / 3;
    int splits = std::max(1, std::min(kMaxSplits, (steps + 2) / 3));
    while (splits > 1 && (tiles * splits > most || tiles > device.clusters[half][splits])) --splits;
    if (!half && steps * (splits == 2 ? 3 : 8) <= std::min<int64_t>(call.rows, kRows)) splits = 1;
    return launch_linear<KIND, kRows, DUAL>(call, splits, half ? kSmemHalf : kSmemLimit);
  };
  if (call.rows <= 16) return run(std::integral_constant<int, 16>{}, true);
  if (call.rows <= 32) return run(std::integral_constant<int, 32>{}, !DUAL);
  if (call.rows <= 64) return run(std::integral_constant<int, 64>{}, false);
  constexpr int kTile = DUAL ? 64 : 128;
  if ((call.rows + kTile - 1) / kTile * w_tiles > sms) {
    const bool packed = call.x.format == FL_MX_FP4 && call.w[0].format == FL_MX_FP4;
    return packed ? launch_pairs<KIND, DUAL, true>(call, sms) : launch_pairs<KIND, DUAL, false>(call, sms);
  }
  return run(std::integral_constant<int, kTile>{}, false);
}

template <bool DUAL>
int run_linear(LinearCall call) {
  FL_REQUIRE(cudaGetDevice(&call.device) == cudaSuccess && call.device >= 0 && call.device < kMaxDevices,
             "%s: no current device", call.who);
  // Tensor maps are encoded by the driver, which wants the device's context current in this thread: the runtime
  // binds it at a thread's first launch, and this call may be the first thing that a thread does.  Once per thread
  // and change of device, as it takes 0.3 us.
  thread_local int bound = -1;
  if (bound != call.device) {
    FL_REQUIRE(cudaSetDevice(call.device) == cudaSuccess, "%s: device %d has no context", call.who, call.device);
    bound = call.device;
  }
  switch (call.out_kind) {
    case kOutBf16: return choose_linear<kOutBf16, DUAL>(call);
    case kOutF16: return choose_linear<kOutF16, DUAL>(call);
    case kOutF32: return choose_linear<kOutF32, DUAL>(call);
    default: break;
  }
  if constexpr (DUAL) {
    return call.out_kind == kOutFp8 ? choose_linear<kOutFp8, true>(call) : choose_linear<kOutFp4, true>(call);
  } else {
    FL_REQUIRE(false, "%s: unknown output type", call.who);
  }
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
                  in_features, out_features, out_dtype, out, nullptr, static_cast<cudaStream_t>(stream), who, 0};
  if (int rc = check_operand(who, "x", call.x)) return rc;
  if (int rc = check_operand(who, "weight", call.w[0])) return rc;
  FL_REQUIRE(out && aligned16(out), "%s: out must be given, 16-byte aligned", who);
  return run_linear<false>(call);
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
                  rows, in_features, out_features, kind, out, out_scales, static_cast<cudaStream_t>(stream), who, 0};
  if (int rc = check_operand(who, "x", call.x)) return rc;
  if (int rc = check_operand(who, "gate", call.w[0])) return rc;
  if (int rc = check_operand(who, "up", call.w[1])) return rc;
  FL_REQUIRE(out && aligned16(out) && aligned16(out_scales), "%s: outputs must be given, 16-byte aligned", who);
  return run_linear<true>(call);
}

extern "C" int fl_mx_give_up_at(int32_t step) {
  t_give_up = step < 0 ? kNever : std::min(step, kNever);
  return FL_OK;
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
