// Quantisation to the microscaled formats, its inverse, and the RMSNorm that leaves its rows in one.
#include <cstring>
#include <type_traits>

#include "fl_mx_common.cuh"

namespace fl {
namespace {

constexpr int kMxThreads = 256;

// Sixteen lanes take one step (128 elements) of a row, eight elements each: four lanes share a block,
// whose largest magnitude takes two shuffles, and the four scale bytes of the step leave as one word.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kMxThreads)
quantize_kernel(const T* __restrict__ x, int64_t rows, int cols, int64_t row_stride, uint32_t steps, uint32_t units,
                uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  const uint32_t unit = blockIdx.x * (kMxThreads / 16) + threadIdx.x / 16;
  const int lane = threadIdx.x & 15;
  const uint32_t row = unit / steps, step = unit - row * steps;
  const bool live = unit < units && row < rows;
  float v[8] = {};
  const int e = int(step) * kMxStep + lane * 8;
  if (live) load8<T, VEC>(x + int64_t(row) * row_stride + e, cols - e, v);
  uint32_t out[2];
  const uint32_t word = mx_join_scales(mx_encode8<FORMAT>(v, out));
  if (live) store_codes<FORMAT>(codes + int64_t(row) * steps * (FORMAT == FL_MX_FP8 ? kMxStep : kMxStep / 2), e, out);
  // units past the last row belong to the last scale tile: their values are zero, and so is the word
  if (unit < units && lane == 0) *reinterpret_cast<uint32_t*>(scales + mx_scale_offset(row, step, steps)) = word;
}

// Eight elements of a row per thread.
template <typename T, int FORMAT>
__global__ void __launch_bounds__(kMxThreads)
dequantize_kernel(const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales, int cols, uint32_t steps,
                  uint32_t units, T* __restrict__ out) {
  const uint32_t unit = blockIdx.x * (kMxThreads / 16) + threadIdx.x / 16;
  if (unit >= units) return;
  const uint32_t row = unit / steps, step = unit - row * steps;
  const int lane = threadIdx.x & 15;
  const int e = int(step) * kMxStep + lane * 8;
  if (e >= cols) return;
  const float scale = mx_scale_value(__ldg(scales + mx_scale_offset(row, step, steps) + lane / 4));
  const uint8_t* src = codes + int64_t(unit) * (FORMAT == FL_MX_FP8 ? kMxStep : kMxStep / 2);
  float v[8];
  if (FORMAT == FL_MX_FP8) {
    const uint2 w = ldg64(src + lane * 8);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const uint16_t pair = uint16_t((k < 2 ? w.x : w.y) >> (16 * (k & 1)));
      uint32_t h;
      asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(pair));
      const float2 f = __half22float2(as_half2(h));
      v[2 * k] = f.x * scale;
      v[2 * k + 1] = f.y * scale;
    }
  } else {
    const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(src + lane * 4));
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t h;
      asm("{\n\t.reg .b8 t;\n\tcvt.u8.u32 t, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, t;\n\t}" : "=r"(h) : "r"((w >> (8 * k)) & 255u));
      const float2 f = __half22float2(as_half2(h));
      v[2 * k] = f.x * scale;
      v[2 * k + 1] = f.y * scale;
    }
  }
  T* dst = out + int64_t(row) * cols + e;
  if (cols % 8 == 0) {
    store8<T, true>(dst, cols - e, v);
  } else {
    store8<T, false>(dst, cols - e, v);
  }
}

constexpr int kNormChunks = 4;  // eight elements per thread and chunk: rows up to 8192 wide

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

__device__ __forceinline__ float cta_sum(float v, float* s_part) {
  v = warp_sum(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s_part[threadIdx.x >> 5] = v;
  __syncthreads();
  float total = 0.f;
#pragma unroll
  for (int w = 0; w < kMxThreads / 32; ++w) total += s_part[w];
  return total;
}

// s = round(addend + x) or x;  n = weight * s * rsqrt(mean(s^2) + eps).  Without weight2 the codes are
// those of n; with it hidden = round([residual +] n) and the codes are those of weight2 * hidden *
// rsqrt(mean(hidden^2) + eps2).  Everything between two stored tensors stays in float32.
template <typename T, int FORMAT, bool VEC>
__global__ void __launch_bounds__(kMxThreads) norm_mx_kernel(const MxNormParams<T> p) {
  __shared__ float s_part[kMxThreads / 32];
  const int64_t row = blockIdx.x;
  const int64_t base = row * p.width;
  float v[kNormChunks][8];
  float sq = 0.f;
#pragma unroll
  for (int c = 0; c < kNormChunks; ++c) {
    const int e = (c * kMxThreads + threadIdx.x) * 8;
    const int n = p.width - e;
    if (n <= 0) continue;
    load8<T, VEC>(p.x + base + e, n, v[c]);
    if (p.addend) {
      float a[8];
      load8<T, VEC>(p.addend + base + e, n, a);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] += a[k];
      store8<T, VEC>(p.sum_out ? p.sum_out + base + e : nullptr, n, v[c]);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) sq = fmaf(v[c][k], v[c][k], sq);
  }
  float inv = rsqrtf(cta_sum(sq, s_part) / float(p.width) + p.eps);
  sq = 0.f;
#pragma unroll
  for (int c = 0; c < kNormChunks; ++c) {
    const int e = (c * kMxThreads + threadIdx.x) * 8;
    const int n = p.width - e;
    if (n <= 0) continue;
    float w[8];
    load8<T, VEC>(p.weight + e, n, w);
#pragma unroll
    for (int k = 0; k < 8; ++k) v[c][k] = w[k] * (v[c][k] * inv);
    if (p.weight2) {
      if (p.residual) {
        float r[8];
        load8<T, VEC>(p.residual + base + e, n, r);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] += r[k];
      }
      store8<T, VEC>(p.hidden + base + e, n, v[c]);
#pragma unroll
      for (int k = 0; k < 8; ++k) sq = fmaf(v[c][k], v[c][k], sq);
    }
  }
  if (p.weight2) inv = rsqrtf(cta_sum(sq, s_part) / float(p.width) + p.eps2);
#pragma unroll
  for (int c = 0; c < kNormChunks; ++c) {
    const uint32_t step = (c * kMxThreads + threadIdx.x) / 16;
    if (c * (kMxThreads / 16) >= int(p.steps)) continue;  // the same for the whole CTA
    const int e = (c * kMxThreads + threadIdx.x) * 8;
    const int n = p.width - e;
    if (n <= 0) {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = 0.f;
    } else if (p.weight2) {
      float w[8];
      load8<T, VEC>(p.weight2 + e, n, w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = w[k] * (v[c][k] * inv);
    }
    uint32_t out[2];
    const uint32_t word = mx_join_scales(mx_encode8<FORMAT>(v[c], out));
    if (step < p.steps) {
      store_codes<FORMAT>(p.codes + row * p.steps * (FORMAT == FL_MX_FP8 ? kMxStep : kMxStep / 2), e, out);
      if ((threadIdx.x & 15) == 0) *reinterpret_cast<uint32_t*>(p.scales + mx_scale_offset(row, step, p.steps)) = word;
    }
  }
  // rows of the last scale tile past the last row
  const int64_t end = (p.rows + kMxTileRows - 1) / kMxTileRows * kMxTileRows;
  for (int64_t r = row + p.rows; r < end; r += p.rows)
    for (uint32_t step = threadIdx.x; step < p.steps; step += kMxThreads)
      *reinterpret_cast<uint32_t*>(p.scales + mx_scale_offset(r, step, p.steps)) = 0u;
}

template <typename T, int FORMAT>
int launch_quantize(const void* x, int64_t rows, int32_t cols, int64_t stride, void* codes, void* scales,
                    cudaStream_t stream) {
  const int64_t steps = mx_steps(cols);
  const int64_t units = (rows + kMxTileRows - 1) / kMxTileRows * kMxTileRows * steps;
  FL_REQUIRE(units < (int64_t(1) << 31), "fl_mx_quantize: too many elements");
  const unsigned grid = unsigned((units + kMxThreads / 16 - 1) / (kMxThreads / 16));
  const T* src = static_cast<const T*>(x);
  uint8_t* c = static_cast<uint8_t*>(codes);
  uint8_t* s = static_cast<uint8_t*>(scales);
  if (aligned16(x) && stride * sizeof(T) % 16 == 0) {
    quantize_kernel<T, FORMAT, true><<<grid, kMxThreads, 0, stream>>>(src, rows, cols, stride, uint32_t(steps), uint32_t(units), c, s);
  } else {
    quantize_kernel<T, FORMAT, false><<<grid, kMxThreads, 0, stream>>>(src, rows, cols, stride, uint32_t(steps), uint32_t(units), c, s);
  }
  FL_CHECK_LAUNCH("fl_mx_quantize");
  return FL_OK;
}

template <typename T, int FORMAT>
int launch_dequantize(const void* codes, const void* scales, int64_t rows, int32_t cols, void* out,
                      cudaStream_t stream) {
  const int64_t steps = mx_steps(cols), units = rows * steps;
  FL_REQUIRE(units < (int64_t(1) << 31), "fl_mx_dequantize: too many elements");
  const unsigned grid = unsigned((units + kMxThreads / 16 - 1) / (kMxThreads / 16));
  dequantize_kernel<T, FORMAT><<<grid, kMxThreads, 0, stream>>>(
      static_cast<const uint8_t*>(codes), static_cast<const uint8_t*>(scales), cols, uint32_t(steps), uint32_t(units),
      static_cast<T*>(out));
  FL_CHECK_LAUNCH("fl_mx_dequantize");
  return FL_OK;
}

struct NormArgs {
  const void *x, *addend, *residual, *weight, *weight2;
  float eps, eps2;
  int64_t rows;
  int32_t width;
  void *sum_out, *hidden, *codes, *scales;
};

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
  const bool vec = aligned16(a.x) && aligned16(a.addend) && aligned16(a.residual) && aligned16(a.weight) &&
                   aligned16(a.weight2) && aligned16(a.sum_out) && aligned16(a.hidden) &&
                   a.width * sizeof(T) % 16 == 0;
  if (vec) {
    norm_mx_kernel<T, FORMAT, true><<<unsigned(a.rows), kMxThreads, 0, stream>>>(p);
  } else {
    norm_mx_kernel<T, FORMAT, false><<<unsigned(a.rows), kMxThreads, 0, stream>>>(p);
  }
  FL_CHECK_LAUNCH("fl_rmsnorm_mx");
  return FL_OK;
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
  FL_REQUIRE(rows >= 0 && rows < (int64_t(1) << 31) && width > 0 && width <= kNormChunks * kMxThreads * 8,
             "%s: width must be 1 to %d, got %d", who, kNormChunks * kMxThreads * 8, width);
  FL_REQUIRE((weight2 == nullptr) == (hidden == nullptr), "%s: weight2 and hidden go together", who);
  FL_REQUIRE(residual == nullptr || weight2 != nullptr, "%s: a residual needs weight2", who);
  FL_REQUIRE(sum_out == nullptr || addend != nullptr, "%s: sum_out needs an addend", who);
  if (rows == 0) return FL_OK;
  FL_REQUIRE(x && weight && codes && scales, "%s: null argument", who);
  FL_REQUIRE(aligned16(codes) && aligned16(scales), "%s: codes and scales must be 16-byte aligned", who);
  return by_type_and_format(dtype, format,
                            NormCall{{x, addend, residual, weight, weight2, eps, eps2, rows, width, sum_out, hidden,
                                      codes, scales},
                                     static_cast<cudaStream_t>(stream)});
}
