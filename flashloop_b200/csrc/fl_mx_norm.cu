// RMSNorm that leaves its rows in a microscaled format.
#include <algorithm>
#include <atomic>

#include "fl_mx_common.cuh"

namespace fl {
namespace {

// Rows up to 8192 wide: 256 threads of two chunks of sixteen elements.
constexpr int kMaxNormWidth = 8192;

template <typename T>
struct MxNormParams {
  const T* x;
  const T* addend;    // or null
  const T* residual;  // or null
  const T* weight;
  const T* weight2;  // or null: quantise the first norm
  float eps, eps2;
  int64_t rows;
  int width;
  uint32_t steps;
  T* sum_out;  // or null: addend + x as rounded
  T* hidden;   // with weight2: [residual +] norm(s)
  uint8_t* codes;
  uint8_t* scales;
};

// Sum over the LANES threads of a row; every one of them gets it.
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* part) {
#pragma unroll
  for (int o = (LANES < 32 ? LANES : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (LANES > 32) {
    constexpr int kWarps = LANES / 32;
    const int warp = threadIdx.x >> 5, first = warp / kWarps * kWarps;
    if ((threadIdx.x & 31) == 0) part[warp] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += part[first + w];
  }
  return v;
}

// In four chains: shorter, and each rounds to less.
__device__ __forceinline__ float sum_of_squares(const float (&v)[16]) {
  float s[4] = {};
#pragma unroll
  for (int k = 0; k < 16; ++k) s[k & 3] = fmaf(v[k], v[k], s[k & 3]);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// 1 / sqrt(mean + eps): the hardware's root and one Newton step, so that the float32 result carries the rounding
// of its products only.  The step is for a finite, positive mean: of an infinite one (an infinity in the row, or
// squares past float32's range) the factor is 0, of zero it is infinite, of a NaN a NaN.
__device__ __forceinline__ float inverse_root(float sum, int width, float eps) {
  const float m = sum / float(width) + eps;
  const float y = rsqrtf(m);
  const float r = fmaf(-m * y, y, 1.f);
  return y > 0.f && isfinite(y) ? fmaf(0.5f * y, r, y) : y;
}

// s = round(addend + x) or x;  n = weight * s * rsqrt(mean(s^2) + eps).  Without weight2 the codes are
// those of n; with it hidden = round([residual +] n) and the codes are those of weight2 * hidden *
// rsqrt(mean(hidden^2) + eps2).  Everything between two stored tensors stays in float32.
//
// LANES threads share a row and hold it in registers, CHUNKS times sixteen elements per thread; as few as hold it, eight
// (one scale word) at least.  CTAs take rows one after the other and ask for the next ones before they work on the
// present ones: bound by memory with many rows (bfloat16, residual and second norm: 32768 x
// 2048 79 us, 0.92 of the copy rate; 100000 x 192 36 us, 0.6; rows of 2047, which go through shared memory, 145 us), by
// latency with few (16 x 2048: 2.2 us).
template <int LANES>
constexpr int kNormThreads = LANES < 128 ? 128 : LANES;

template <typename T, int ALIGN, bool SECOND, int LANES, int CHUNKS>
struct NormRow {
  Load16<T, ALIGN> x[CHUNKS], a[CHUNKS], r[SECOND ? CHUNKS : 1];
  __device__ __forceinline__ void load(const MxNormParams<T>& p, int64_t row, int thread) {
    const int64_t base = row * p.width;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int e = (c * LANES + thread) * 16, n = row < p.rows ? p.width - e : 0;
      x[c].load(p.x + base + e, n);
      if (p.addend) a[c].load(p.addend + base + e, n);
      if constexpr (SECOND) {
        if (p.residual) r[c].load(p.residual + base + e, n);
      }
    }
  }
};

// SECOND: weight2 is given.
template <typename T, int FORMAT, int ALIGN, bool SECOND, int LANES, int CHUNKS>
__global__ void __launch_bounds__(kNormThreads<LANES>) norm_mx_kernel(const MxNormParams<T> p) {
  constexpr int kThreads = kNormThreads<LANES>, kRowThreads = LANES, kRows = kThreads / LANES;
  __shared__ float s_part[2][kThreads / 32];
  __shared__ __align__(16) WarpStage<T, ALIGN, kThreads> stage;
  const int thread = threadIdx.x % kRowThreads;
  const int64_t stride = int64_t(gridDim.x) * kRows;
  const bool one_group = p.rows <= 32;  // a row's word is then the only one of its sixteen bytes
  int64_t row = int64_t(blockIdx.x) * kRows + threadIdx.x / kRowThreads;
  wait_for_inputs();
  may_start_next();
  NormRow<T, ALIGN, SECOND, LANES, CHUNKS> next;
  next.load(p, row, thread);
  Raw16<T> raw_w[CHUNKS], raw_w2[SECOND ? CHUNKS : 1];
#pragma unroll
  for (int c = 0; c < CHUNKS; ++c) {
    const int e = (c * kRowThreads + thread) * 16;
    Load16<T, ALIGN> w, w2;
    w.load(p.weight + e, p.width - e);
    if constexpr (SECOND) w2.load(p.weight2 + e, p.width - e);
    raw_w[c] = w.get(stage.mine());
    if constexpr (SECOND) raw_w2[c] = w2.get(stage.mine());
  }
  // the same number of rounds for all threads of the CTA, which meet at barriers
  for (int64_t first = int64_t(blockIdx.x) * kRows; first < p.rows; first += stride, row += stride) {
    const bool live = row < p.rows;
    const int64_t base = row * p.width;
    Raw16<T> x[CHUNKS], a[CHUNKS], r[SECOND ? CHUNKS : 1];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      x[c] = next.x[c].get(stage.mine());
      if (p.addend) a[c] = next.a[c].get(stage.mine());
      if constexpr (SECOND) {
        if (p.residual) r[c] = next.r[c].get(stage.mine());
      }
    }
    if (first + stride < p.rows) next.load(p, row + stride, thread);
    float v[CHUNKS][16];
    float sq = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      x[c].unpack(v[c]);
      if (p.addend) {
        const int e = (c * kRowThreads + thread) * 16, n = live ? p.width - e : 0;
        float add[16];
        a[c].unpack(add);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[c][k] += add[k];
        store16<T, ALIGN>(p.sum_out + base + e, p.sum_out ? n : 0, v[c], stage.mine());
      }
      sq += sum_of_squares(v[c]);
    }
    float inv = inverse_root(row_sum<LANES>(sq, s_part[0]), p.width, p.eps);
    sq = 0.f;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      float res[16] = {}, w[16];
      raw_w[c].unpack(w);
      if constexpr (SECOND) {
        if (p.residual) r[c].unpack(res);
      }
#pragma unroll
      for (int k = 0; k < 16; ++k) v[c][k] = fmaf(w[k], v[c][k] * inv, res[k]);
      if constexpr (SECOND) {
        const int e = (c * kRowThreads + thread) * 16, n = live ? p.width - e : 0;
        store16<T, ALIGN>(p.hidden + base + e, n, v[c], stage.mine());
        sq += sum_of_squares(v[c]);
      }
    }
    // one barrier per round orders the reads of s_part[0] before its next writes, and the second sum's does s_part[1]
    if constexpr (SECOND) {
      inv = inverse_root(row_sum<LANES>(sq, s_part[1]), p.width, p.eps2);
    } else if (LANES > 32) {
      __syncthreads();
    }
    uint8_t* codes = p.codes + row * p.steps * (FORMAT == FL_MX_FP8 ? kMxStep : kMxStep / 2);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int e = (c * kRowThreads + thread) * 16;
      const uint32_t step = uint32_t(e) / kMxStep;
      if constexpr (SECOND) {
        float w[16];
        raw_w2[c].unpack(w);
#pragma unroll
        for (int k = 0; k < 16; ++k) v[c][k] = w[k] * (v[c][k] * inv);
      }
      if (e >= p.width) {  // padding is zero also where the row is not finite
#pragma unroll
        for (int k = 0; k < 16; ++k) v[c][k] = 0.f;
      }
      uint32_t out[4];
      const uint32_t word = mx_join_scales(mx_encode16<FORMAT>(v[c], out));
      if (live && step < p.steps) {
        store_codes<FORMAT>(codes, e, out);
        if ((threadIdx.x & 7) == 0) {
          uint8_t* at = p.scales + mx_scale_offset(row, step, p.steps);
          if (one_group) {
            *reinterpret_cast<uint4*>(at) = make_uint4(word, 0u, 0u, 0u);
          } else {
            *reinterpret_cast<uint32_t*>(at) = word;
          }
        }
      }
    }
  }
  // rows of the last scale tile past the last row, shared out over all threads
  const uint32_t threads = gridDim.x * kThreads, mine = blockIdx.x * kThreads + threadIdx.x;
  if (one_group) {
    const uint32_t empty = 32u - uint32_t(p.rows);  // sixteen-byte groups of a step that hold no row
    for (uint32_t i = mine; i < empty * p.steps; i += threads)
      *reinterpret_cast<uint4*>(p.scales + mx_scale_offset(p.rows + i / p.steps, i % p.steps, p.steps)) = make_uint4(0u, 0u, 0u, 0u);
  } else {
    const uint32_t empty = uint32_t(-p.rows & (kMxTileRows - 1));
    for (uint32_t i = mine; i < empty * p.steps; i += threads)
      *reinterpret_cast<uint32_t*>(p.scales + mx_scale_offset(p.rows + i / p.steps, i % p.steps, p.steps)) = 0u;
  }
}

struct NormArgs {
  const void *x, *addend, *residual, *weight, *weight2;
  float eps, eps2;
  int64_t rows;
  int32_t width;
  void *sum_out, *hidden, *codes, *scales;
};

template <typename T, int FORMAT, int ALIGN, bool SECOND, int LANES, int CHUNKS>
cudaError_t launch_norm_shape(const MxNormParams<T>& p, cudaStream_t stream) {
  constexpr int kThreads = kNormThreads<LANES>, kRows = kThreads / LANES;
  auto kernel = norm_mx_kernel<T, FORMAT, ALIGN, SECOND, LANES, CHUNKS>;
  static std::atomic<int> fit;  // CTAs that run on an SM at once, asked once
  int ctas = fit.load(std::memory_order_relaxed);
  if (ctas == 0) {
    const cudaError_t err = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&ctas, kernel, kThreads, 0);
    if (err != cudaSuccess) return err;
    fit.store(ctas, std::memory_order_relaxed);
  }
  return launch_overlapped(kernel, unsigned(std::min<int64_t>((p.rows + kRows - 1) / kRows, 148 * ctas)), kThreads, 0, 1, stream, p);
}

template <typename T, int FORMAT, int ALIGN, bool SECOND>
cudaError_t launch_norm_rows(const MxNormParams<T>& p, cudaStream_t stream) {
  if (p.width <= 128) return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 8, 1>(p, stream);
  if (p.width <= 256) return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 16, 1>(p, stream);
  if (p.width <= 512) return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 32, 1>(p, stream);
  if (p.width <= 1024) return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 64, 1>(p, stream);
  if (p.width <= 2048) return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 128, 1>(p, stream);
  if (p.width <= 4096) return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 256, 1>(p, stream);
  return launch_norm_shape<T, FORMAT, ALIGN, SECOND, 256, 2>(p, stream);
}

template <typename T, int FORMAT>
int launch_norm(const NormArgs& a, cudaStream_t stream) {
  MxNormParams<T> p;
  p.x = static_cast<const T*>(a.x);
  p.addend = static_cast<const T*>(a.addend);
  p.residual = static_cast<const T*>(a.residual);
  p.weight = static_cast<const T*>(a.weight);
  p.weight2 = static_cast<const T*>(a.weight2);
  p.eps = a.eps;
  p.eps2 = a.eps2;
  p.rows = a.rows;
  p.width = a.width;
  p.steps = uint32_t(mx_steps(a.width));
  p.sum_out = static_cast<T*>(a.sum_out);
  p.hidden = static_cast<T*>(a.hidden);
  p.codes = static_cast<uint8_t*>(a.codes);
  p.scales = static_cast<uint8_t*>(a.scales);
  uintptr_t at = uintptr_t(a.width) * sizeof(T);
  for (const void* q : {a.x, a.addend, a.residual, a.weight, a.weight2, static_cast<const void*>(a.sum_out),
                        static_cast<const void*>(a.hidden)})
    at |= reinterpret_cast<uintptr_t>(q);
  const cudaError_t err = by_alignment<T>(at, [&](auto align) {
    constexpr int kAlign = decltype(align)::value;
    return a.weight2 ? launch_norm_rows<T, FORMAT, kAlign, true>(p, stream) : launch_norm_rows<T, FORMAT, kAlign, false>(p, stream);
  });
  return launched(err, "fl_rmsnorm_mx");
}

struct NormCall {
  NormArgs args;
  cudaStream_t stream;
  template <typename T, int FORMAT>
  int run() const { return launch_norm<T, FORMAT>(args, stream); }
};

}  // namespace
}  // namespace fl

using namespace fl;

extern "C" int fl_rmsnorm_mx(const void* x, const void* addend, const void* residual, const void* weight, float eps,
                             const void* weight2, float eps2, int32_t dtype, int64_t rows, int32_t width,
                             int32_t format, void* sum_out, void* hidden, void* codes, void* scales,
                             fl_cuda_stream stream) {
  const char* who = "fl_rmsnorm_mx";
  FL_REQUIRE(dtype_ok(dtype) && mx_format_ok(format), "%s: unknown type or format", who);
  FL_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && width > 0 && width <= kMaxNormWidth,
             "%s: width must be 1 to %d, got %d", who, kMaxNormWidth, width);
  if (rows == 0) return FL_OK;  // an empty tensor has no address
  FL_REQUIRE((weight2 == nullptr) == (hidden == nullptr), "%s: weight2 and hidden go together", who);
  FL_REQUIRE(residual == nullptr || weight2 != nullptr, "%s: a residual needs weight2", who);
  FL_REQUIRE(sum_out == nullptr || addend != nullptr, "%s: sum_out needs an addend", who);
  FL_REQUIRE(x && weight && codes && scales, "%s: null argument", who);
  for (const void* p : {x, addend, residual, weight, weight2, static_cast<const void*>(sum_out), static_cast<const void*>(hidden)})
    FL_REQUIRE(aligned_to(p, dtype), "%s: tensors must be aligned to their elements", who);
  FL_REQUIRE(aligned16(codes) && aligned16(scales), "%s: codes and scales must be 16-byte aligned", who);
  return by_type_and_format(dtype, format,
                            NormCall{{x, addend, residual, weight, weight2, eps, eps2, rows, width, sum_out, hidden,
                                      codes, scales},
                                     static_cast<cudaStream_t>(stream)});
}
