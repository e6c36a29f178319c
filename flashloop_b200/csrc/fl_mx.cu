// Quantisation to the microscaled formats and its inverse.
#include <cstring>
#include <type_traits>

#include "fl_mx_common.cuh"

namespace fl {
namespace {

constexpr int kMxThreads = 256;

// Eight lanes take one step (128 elements) of a row, sixteen elements each: two lanes share a block, and
// the four scale bytes of the step leave as one word.  A CTA takes UNROLL * 32 consecutive steps and asks for all
// of its elements before it uses any.  Bound by memory: 16384 x 5632 bfloat16 to mxfp8 43 us, the copy rate; rows of
// 5631, which go through shared memory, 60 us.
template <typename T, int FORMAT, int ALIGN, int UNROLL>
__global__ void __launch_bounds__(kMxThreads)
quantize_kernel(const T* x, uint32_t rows, int cols, int64_t row_stride, uint32_t steps, uint32_t units,
                uint8_t* codes, uint8_t* scales) {
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
dequantize_kernel(const uint8_t* codes, const uint8_t* scales, int cols, uint32_t steps,
                  uint32_t units, T* out) {
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
        word[i] = load_uint4(src + lane * 16);
      } else {
        const uint2 half = load_uint2(src + lane * 8);
        word[i].x = half.x;
        word[i].y = half.y;
      }
      byte[i] = load_piece(scales + mx_scale_offset(row[i], step, steps) + lane / 2);
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

// Rounds per thread: several where that still leaves several CTAs to an SM, one below.
constexpr int64_t kUnrollUnits = 148 * 8 * 64;

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
  FL_REQUIRE(aligned_to(x, x_dtype), "%s: x must be aligned to its elements", who);
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
