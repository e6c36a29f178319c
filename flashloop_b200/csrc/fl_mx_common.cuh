// Microscaled formats shared by the quantiser and norm (fl_mx.cu) and the projections
// (fl_mx_linear.cu): blocks of 32 elements along a row, each with a power-of-two scale (e8m0: byte b
// stands for 2^(b - 127), 255 for NaN) and elements of eight bits (e4m3) or four (e2m1).
//
// Codes are stored row by row, every row padded with zeros to a multiple of 128 elements (the
// product's step along K); of two e2m1 codes in a byte the even element has the low nibble.  Scales
// are stored in tiles of 128 rows by 128 elements, 512 bytes each:
//   scales[row / 128][k / 128][row % 32][row / 32 % 4][k / 32 % 4]
// which is the order in which tcgen05.cp spreads scale factors over the 32 lanes of tensor memory, so
// a tile of scales is one bulk copy.  Rows of the last tile past the last row hold scale byte 0.
#pragma once

#include <cstring>
#include <type_traits>

#include "fl_common.cuh"

namespace fl {
namespace {

constexpr int kMxBlock = 32;
constexpr int kMxStep = 128;       // elements of a row per scale tile
constexpr int kMxTileRows = 128;   // rows per scale tile
constexpr int kMxTileBytes = 512;

constexpr int64_t mx_steps(int64_t cols) { return (cols + kMxStep - 1) / kMxStep; }
constexpr int64_t mx_row_bytes(int64_t cols, int format) {
  return mx_steps(cols) * (format == FL_MX_FP8 ? kMxStep : kMxStep / 2);
}
inline bool mx_format_ok(int format) { return format == FL_MX_FP8 || format == FL_MX_FP4; }

#ifdef __CUDACC__

// Byte offset of the scale of (row, step, block 0 of the step).
__device__ __forceinline__ int64_t mx_scale_offset(int64_t row, int64_t step, int64_t steps) {
  return ((row >> 7) * steps + step) * kMxTileBytes + (row & 31) * 16 + ((row >> 5) & 3) * 4;
}

// The scale byte of a block whose largest magnitude has the float32 bits `amax`: the smallest power
// of two that keeps the block in range.  With the largest element L = D * 2^T of the format (448 =
// 1.75 * 2^8, 6 = 1.5 * 2^2) and amax = m * 2^E that is 2^(E - T), or one more where m > D.
// Magnitudes compare as their bits, so a NaN or an infinity anywhere in the block shows here.
// Rounding the exponent up instead of down (which clips up to an eighth of the largest value) gives
// a smaller error on normal blocks at 8 bits (0.0264 against 0.0302 relative) and the same at 4
// (0.1165 against 0.1161), and none of the clipping on heavy tails.
template <int FORMAT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t amax) {
  constexpr int kTop = FORMAT == FL_MX_FP8 ? 8 : 2;
  constexpr uint32_t kDigits = FORMAT == FL_MX_FP8 ? 0x600000u : 0x400000u;
  if (amax >= 0x7f800000u) return 255u;
  const int e = int(amax >> 23) - kTop + ((amax & 0x7fffffu) > kDigits ? 1 : 0);
  return uint32_t(max(e, 0));
}
// 2^(127 - byte), exact in float32 for the bytes mx_scale_byte gives.
__device__ __forceinline__ float mx_inverse(uint32_t byte) {
  return byte == 255u ? 0.f : __uint_as_float((254u - byte) << 23);
}
// 2^(byte - 127); byte 0 is a subnormal.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  if (byte == 255u) return __uint_as_float(0x7fffffffu);
  return byte == 0 ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);
}

// Two scaled values -> two e4m3 bytes / two e2m1 nibbles, round to nearest even, the first in the low half.
__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e2m1x2(float lo, float hi) {
  uint32_t r;
  asm("{\n\t.reg .b8 t;\n\tcvt.rn.satfinite.e2m1x2.f32 t, %1, %2;\n\tcvt.u32.u8 %0, t;\n\t}"
      : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Eight values of one block, held by one of the four lanes that share it (lanes 4i .. 4i + 3).
// Returns the block's scale byte and writes the codes: e4m3 into codes[0..1], e2m1 into codes[0].
template <int FORMAT>
__device__ __forceinline__ uint32_t mx_encode8(const float (&v)[8], uint32_t (&codes)[2]) {
  uint32_t amax = 0;
#pragma unroll
  for (int k = 0; k < 8; ++k) amax = max(amax, __float_as_uint(v[k]) & 0x7fffffffu);
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
  const uint32_t byte = mx_scale_byte<FORMAT>(amax);
  const float inv = mx_inverse(byte);
  if (byte == 255u) {
    codes[0] = codes[1] = 0u;
  } else if (FORMAT == FL_MX_FP8) {
    codes[0] = cvt_e4m3x2(v[0] * inv, v[1] * inv) | cvt_e4m3x2(v[2] * inv, v[3] * inv) << 16;
    codes[1] = cvt_e4m3x2(v[4] * inv, v[5] * inv) | cvt_e4m3x2(v[6] * inv, v[7] * inv) << 16;
  } else {
    codes[0] = cvt_e2m1x2(v[0] * inv, v[1] * inv) | cvt_e2m1x2(v[2] * inv, v[3] * inv) << 8 |
               cvt_e2m1x2(v[4] * inv, v[5] * inv) << 16 | cvt_e2m1x2(v[6] * inv, v[7] * inv) << 24;
    codes[1] = 0u;
  }
  return byte;
}
// The four scale bytes of a step from the sixteen lanes that hold it, in every one of them.
__device__ __forceinline__ uint32_t mx_join_scales(uint32_t byte) {
  uint32_t word = byte << (8 * ((threadIdx.x >> 2) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 4);
  return word | __shfl_xor_sync(0xffffffffu, word, 8);
}

// Eight consecutive elements as they lie in memory, so that a load can be under way while others are
// used.  `count` of them exist (none if it is not positive), the others are zero.  VEC loads 16 bytes at a
// time (the caller has checked the alignment of the base and of the row stride).
template <typename T>
struct Raw8 {
  static constexpr int kWords = sizeof(T) / 2;  // of 16 bytes
  uint4 w[kWords];
  template <bool VEC>
  __device__ __forceinline__ void load(const T* p, int count) {
    if (VEC && count >= 8) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) w[i] = ldg128(reinterpret_cast<const uint4*>(p) + i);
      return;
    }
    T t[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) t[k] = k < count ? p[k] : T(0.f);
    memcpy(w, t, sizeof(t));
  }
  __device__ __forceinline__ void unpack(float (&v)[8]) const {
    const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[kWords - 1].x, w[kWords - 1].y, w[kWords - 1].z,
                                    w[kWords - 1].w};
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[k] = __uint_as_float(u[k]);
      } else if constexpr (std::is_same<T, __half>::value) {
        v[k] = k & 1 ? __high2float(as_half2(u[k / 2])) : __low2float(as_half2(u[k / 2]));
      } else {
        v[k] = k & 1 ? bf16_hi(u[k / 2]) : bf16_lo(u[k / 2]);
      }
    }
  }
};
template <typename T, bool VEC>
__device__ __forceinline__ void load8(const T* p, int count, float (&v)[8]) {
  Raw8<T> raw;
  raw.template load<VEC>(p, count);
  raw.unpack(v);
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }

// Eight values rounded to T, stored; `v` keeps what was stored.
template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, int count, float (&v)[8]) {
  T t[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
    t[k] = round_to<T>(v[k]);
    v[k] = load_as_float<T>(&t[k]);
  }
  if (p == nullptr) return;
  if (VEC && count >= 8) {
    uint4 w[sizeof(T) / 2];
    memcpy(w, t, sizeof(t));
#pragma unroll
    for (int k = 0; k < int(sizeof(T) / 2); ++k) reinterpret_cast<uint4*>(p)[k] = w[k];
    return;
  }
#pragma unroll
  for (int k = 0; k < 8; ++k)
    if (k < count) p[k] = t[k];
}

// Codes of eight elements starting at element `e` of a row (e a multiple of 8).
template <int FORMAT>
__device__ __forceinline__ void store_codes(uint8_t* row_codes, int64_t e, const uint32_t (&codes)[2]) {
  if (FORMAT == FL_MX_FP8) {
    *reinterpret_cast<uint2*>(row_codes + e) = make_uint2(codes[0], codes[1]);
  } else {
    *reinterpret_cast<uint32_t*>(row_codes + e / 2) = codes[0];
  }
}

#endif  // __CUDACC__

}  // namespace
}  // namespace fl
