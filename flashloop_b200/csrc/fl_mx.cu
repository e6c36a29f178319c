// Quantisation to the microscaled formats, its inverse, and the RMSNorm that leaves its rows in one.
#include <algorithm>
#include <atomic>
#include <cstring>
#include <type_traits>

#include "fl_mx_common.cuh"

namespace fl {
namespace {

constexpr int kMxThreads = 256;

// Eight lanes take one step (128 elements) of a row, sixteen elements each: two lanes share a block, and
// the four scale bytes of the step leave as one word.  A CTA takes UNROLL * 32 consecutive steps and asks for all of its elements before it uses any.
template <typename T, int FORMAT, int ALIGN, int UNROLL>
__global__ void __launch_bounds__(kMxThreads)
quantize_kernel(const T* __restrict__ x, uint32_t rows, int cols, int64_t row_stride, uint32_t steps, uint32_t units,
                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const uint32_t first = blockIdx.x * (UNROLL * kMxThreads / 8) + threadIdx.x / 8;
  const int lane = threadIdx.x & 7;
  __shared__ __align__(16) WarpStage<T, ALIGN, kMxThreads> stage;
  wait_for_inputs();
  may_start_next();
  Load16<T, ALIGN> raw[UNROLL];
  uint32_t row[UNROLL];
  int e[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    const uint32_t unit = first + i * (kMxThreads / 8);
    row[i] = unit / steps;
    e[i] = int(unit - row[i] * steps) * kMxStep + lane * 16;
    raw[i].load(x + int64_t(row[i]) * row_stride + e[i], unit < units && row[i] < rows ? cols - e[i] : 0);
  }
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    const uint32_t unit = first + i * (kMxThreads / 8);
    float v[16];
    raw[i].get(stage.mine()).unpack(v);
    uint32_t out[4];
    const uint32_t word = mx_join_scales(mx_encode16<FORMAT>(v, out));
    if (unit >= units) continue;
    if (row[i] < rows) {
      store_codes<FORMAT>(codes + int64_t(unit) * (FORMAT == FL_MX_FP8 ? kMxStep : kMxStep / 2), lane * 16, out);
    }
    // steps past the last row belong to the last scale tile: their values are zero, and so is the word
    if (lane == 0)
      *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(row[i], uint32_t(e[i]) / kMxStep, steps)) = word;
  }
}

// Sixteen elements of a row per thread and round.
template <typename T, int FORMAT, int ALIGN, int UNROLL>
__global__ void __launch_bounds__(kMxThreads)
dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int cols, uint32_t steps,
                  uint32_t units, T* __restrict__ out) {
  const uint32_t first = blockIdx.x * (UNROLL * kMxThreads / 8) + threadIdx.x / 8;
  const int lane = threadIdx.x & 7;
  __shared__ __align__(16) WarpStage<T, ALIGN, kMxThreads> stage;
  wait_for_inputs();
  may_start_next();
  uint4 word[UNROLL] = {};
  uint32_t byte[UNROLL] = {};
  uint32_t row[UNROLL];
  int e[UNROLL];
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    const uint32_t unit = first + i * (kMxThreads / 8);
    row[i] = unit / steps;
    const uint32_t step = unit - row[i] * steps;
    e[i] = unit < units ? int(step) * kMxStep + lane * 16 : cols;
    if (e[i] < cols) {
      const uint8_t* src = codes + int64_t(unit) * (FORMAT == FL_MX_FP8 ? kMxStep : kMxStep / 2);
      if (FORMAT == FL_MX_FP8) {
        word[i] = ldg128(src + lane * 16);
      } else {
        const uint2 half = ldg64(src + lane * 8);
        word[i].x = half.x;
        word[i].y = half.y;
      }
      byte[i] = __ldg(scales + mx_scale_offset(row[i], step, steps) + lane / 2);
    }
  }
#pragma unroll
  for (int i = 0; i < UNROLL; ++i) {
    if (ALIGN == 16 && e[i] >= cols) continue;
    const float scale = mx_scale_value(byte[i]);
    const uint32_t w[4] = {word[i].x, word[i].y, word[i].z, word[i].w};
    float v[16];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      uint32_t h;
      if (FORMAT == FL_MX_FP8) {
        const uint16_t pair = uint16_t(w[k / 2] >> (16 * (k & 1)));
        asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pair));
      } else {
        asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"((w[k / 4] >> (8 * (k & 3))) & 255u));
      }
      const float2 f = __half22float2(as_half2(h));
      v[2 * k] = f.x * scale;
      v[2 * k + 1] = f.y * scale;
    }
    store16<T, ALIGN>(out + int64_t(row[i]) * cols + e[i], cols - e[i], v, stage.mine());
  }
}

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
  if (LANES <= 32) return v;
  constexpr int kWarps = LANES / 32;
  const int warp = threadIdx.x >> 5, first = warp / kWarps * kWarps;
  if ((threadIdx.x & 31) == 0) part[warp] = v;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) total += part[first + w];
  return total;
}

// In four chains: shorter, and each rounds to less.
__device__ __forceinline__ float sum_of_squares(const float (&v)[16]) {
  float s[4] = {};
#pragma unroll
  for (int k = 0; k < 16; ++k) s[k & 3] = fmaf(v[k], v[k], s[k & 3]);
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// 1 / sqrt(mean + eps): the hardware's root and one Newton step, so that the float32 result carries the rounding
// of its products only.
__device__ __forceinline__ float inverse_root(float sum, int width, float eps) {
  const float m = sum / float(width) + eps;
  const float y = rsqrtf(m);
  const float r = fmaf(-m * y, y, 1.f);
  return isfinite(y) ? fmaf(0.5f * y, r, y) : y;
}

// s = round(addend + x) or x;  n = weight * s * rsqrt(mean(s^2) + eps).  Without weight2 the codes are
// those of n; with it hidden = round([residual +] n) and the codes are those of weight2 * hidden *
// rsqrt(mean(hidden^2) + eps2).  Everything between two stored tensors stays in float32.
//
// LANES threads share a row and hold it in registers, CHUNKS times sixteen elements per thread; as few as hold it, eight
// (one scale word) at least.  CTAs take rows one after the other and ask for the next ones before they work on the
// present ones: bound by memory with many rows (MEASURED), by latency with few.
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

// Rounds per thread: several where that still leaves several CTAs to an SM, one below.
constexpr int64_t kUnrollUnits = 148 * 8 * 64;

// Calls f with the largest of 16, 4 and 2 bytes at whose multiples the addresses or-ed into `at` all lie.
template <typename T, typename F>
auto by_alignment(uintptr_t at, F&& f) {
  if (at % 16 == 0) return f(std::integral_constant<int, 16>{});
  if constexpr (sizeof(T) == 2) {
    if (at % 4 != 0) return f(std::integral_constant<int, 2>{});
  }
  return f(std::integral_constant<int, 4>{});
}

int launched(cudaError_t err, const char* who) {
  if (err == cudaSuccess) return FL_OK;
  cudaGetLastError();
  set_error("%s: %s", who, cudaGetErrorString(err));
  return FL_ERR_CUDA;
}

template <typename T, int FORMAT>
int launch_quantize(const void* x, int64_t rows, int32_t cols, int64_t stride, void* codes, void* scales,
                    cudaStream_t stream) {
  const int64_t steps = mx_steps(cols);
  const int64_t units = (rows + kMxTileRows - 1) / kMxTileRows * kMxTileRows * steps;
  FL_REQUIRE(units < (int64_t(1) << 31), "fl_mx_quantize: too many elements");
  const uintptr_t at = reinterpret_cast<uintptr_t>(x) | (rows > 1 ? uintptr_t(stride) * sizeof(T) : 0);
  const bool many = units >= kUnrollUnits;
  auto kernel = by_alignment<T>(at % 16 == 0 ? 0 : at | uintptr_t(cols) * sizeof(T), [&](auto align) {
    constexpr int kAlign = decltype(align)::value;
    return many ? quantize_kernel<T, FORMAT, kAlign, 2> : quantize_kernel<T, FORMAT, kAlign, 1>;
  });
  const int64_t each = (many ? 2 : 1) * (kMxThreads / 8);
  return launched(launch_overlapped(kernel, unsigned((units + each - 1) / each), kMxThreads, 0, 1, stream,
                                    static_cast<const T*>(x), uint32_t(rows), cols, stride, uint32_t(steps), uint32_t(units),
                                    static_cast<uint8_t*>(codes), static_cast<uint8_t*>(scales)),
                  "fl_mx_quantize");
}

template <typename T, int FORMAT>
int launch_dequantize(const void* codes, const void* scales, int64_t rows, int32_t cols, void* out,
                      cudaStream_t stream) {
  const int64_t steps = mx_steps(cols), units = rows * steps;
  FL_REQUIRE(units < (int64_t(1) << 31), "fl_mx_dequantize: too many elements");
  constexpr int kUnits = kMxThreads / 8;
  const uint8_t* c = static_cast<const uint8_t*>(codes);
  const uint8_t* s = static_cast<const uint8_t*>(scales);
  const bool many = units >= kUnrollUnits;
  auto kernel = by_alignment<T>(uintptr_t(cols) * sizeof(T), [&](auto align) {
    constexpr int kAlign = decltype(align)::value;
    return many ? dequantize_kernel<T, FORMAT, kAlign, 4> : dequantize_kernel<T, FORMAT, kAlign, 1>;
  });
  const int64_t each = many ? 4 * kUnits : kUnits;
  return launched(launch_overlapped(kernel, unsigned((units + each - 1) / each), kMxThreads, 0, 1, stream, c, s, cols,
                                    uint32_t(steps), uint32_t(units), static_cast<T*>(out)),
                  "fl_mx_dequantize");
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

// Calls f.template run<T, FORMAT>() for the type and format codes (validated by the caller).
template <typename F>
int by_type_and_format(int dtype, int format, F&& f) {
  const bool fp8 = format == FL_MX_FP8;
  switch (dtype) {
    case FL_DTYPE_BF16:
      return fp8 ? f.template run<__nv_bfloat16, FL_MX_FP8>() : f.template run<__nv_bfloat16, FL_MX_FP4>();
    case FL_DTYPE_F16:
      return fp8 ? f.template run<__half, FL_MX_FP8>() : f.template run<__half, FL_MX_FP4>();
    default:
      return fp8 ? f.template run<float, FL_MX_FP8>() : f.template run<float, FL_MX_FP4>();
  }
}
bool dtype_ok(int dtype) { return dtype == FL_DTYPE_BF16 || dtype == FL_DTYPE_F16 || dtype == FL_DTYPE_F32; }

struct QuantizeCall {
  const void* x;
  int64_t rows;
  int32_t cols;
  int64_t stride;
  void *codes, *scales;
  cudaStream_t stream;
  template <typename T, int FORMAT>
  int run() const { return launch_quantize<T, FORMAT>(x, rows, cols, stride, codes, scales, stream); }
};
struct DequantizeCall {
  const void *codes, *scales;
  int64_t rows;
  int32_t cols;
  void* out;
  cudaStream_t stream;
  template <typename T, int FORMAT>
  int run() const { return launch_dequantize<T, FORMAT>(codes, scales, rows, cols, out, stream); }
};
struct NormCall {
  NormArgs args;
  cudaStream_t stream;
  template <typename T, int FORMAT>
  int run() const { return launch_norm<T, FORMAT>(args, stream); }
};

}  // namespace
}  // namespace fl

using namespace fl;

extern "C" int64_t fl_mx_codes_bytes(int64_t rows, int32_t cols, int32_t format) {
  return rows < 0 || cols <= 0 || !mx_format_ok(format) ? 0 : rows * mx_row_bytes(cols, format);
}

extern "C" int64_t fl_mx_scales_bytes(int64_t rows, int32_t cols) {
  return rows < 0 || cols <= 0 ? 0 : (rows + kMxTileRows - 1) / kMxTileRows * mx_steps(cols) * kMxTileBytes;
}

extern "C" int fl_mx_quantize(const void* x, int32_t x_dtype, int64_t rows, int32_t cols, int64_t row_stride,
                              int32_t format, void* codes, void* scales, fl_cuda_stream stream) {
  const char* who = "fl_mx_quantize";
  FL_REQUIRE(dtype_ok(x_dtype) && mx_format_ok(format), "%s: unknown type or format", who);
  FL_REQUIRE(rows >= 0 && cols > 0 && (row_stride >= cols || rows <= 1), "%s: bad sizes", who);
  if (rows == 0) return FL_OK;
  FL_REQUIRE(x && codes && scales, "%s: null argument", who);
  FL_REQUIRE(aligned16(codes) && aligned16(scales), "%s: codes and scales must be 16-byte aligned", who);
  return by_type_and_format(x_dtype, format, QuantizeCall{x, rows, cols, row_stride, codes, scales,
                                                          static_cast<cudaStream_t>(stream)});
}

extern "C" int fl_mx_dequantize(const void* codes, const void* scales, int32_t format, int64_t rows, int32_t cols,
                                void* out, int32_t out_dtype, fl_cuda_stream stream) {
  const char* who = "fl_mx_dequantize";
  FL_REQUIRE(dtype_ok(out_dtype) && mx_format_ok(format), "%s: unknown type or format", who);
  FL_REQUIRE(rows >= 0 && cols > 0, "%s: bad sizes", who);
  if (rows == 0) return FL_OK;
  FL_REQUIRE(out && codes && scales, "%s: null argument", who);
  FL_REQUIRE(aligned16(codes) && aligned16(scales) && aligned16(out), "%s: pointers must be 16-byte aligned", who);
  return by_type_and_format(out_dtype, format, DequantizeCall{codes, scales, rows, cols, out,
                                                              static_cast<cudaStream_t>(stream)});
}

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
  FL_REQUIRE(aligned16(codes) && aligned16(scales), "%s: codes and scales must be 16-byte aligned", who);
  return by_type_and_format(dtype, format,
                            NormCall{{x, addend, residual, weight, weight2, eps, eps2, rows, width, sum_out, hidden,
                                      codes, scales},
                                     static_cast<cudaStream_t>(stream)});
}
