// Microscaled formats shared by the quantiser (fl_mx.cu), the norm (fl_mx_norm.cu) and the projections
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
#include <utility>

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

// The kernels on microscaled tensors are launched so that they may start while the kernel before them
// in the stream is ending (programmatic dependent launch).  They read and write nothing of the caller's
// before wait_for_inputs(), which every thread passes and which returns when all earlier work of the stream is
// done and visible; what comes before it is their own set-up.  may_start_next() lets the next such
// kernel set up once all CTAs of this one run.
__device__ __forceinline__ void wait_for_inputs() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void may_start_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Loads of the caller's data in these kernels.  The kernel before may still be writing it when this one
// starts, so it is not constant for the kernel's life (no ld.global.nc, no __ldg), and nothing may
// move such a load in front of wait_for_inputs(): volatile, with a memory clobber as the wait has.
__device__ __forceinline__ void load_words(const void* p, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d, uint32_t& e,
                                           uint32_t& f, uint32_t& g, uint32_t& h) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(a), "=r"(b), "=r"(c), "=r"(d), "=r"(e), "=r"(f), "=r"(g), "=r"(h) : "l"(p) : "memory");
}
__device__ __forceinline__ uint4 load_uint4(const void* p) {
  uint4 q;
  asm volatile("ld.global.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(q.x), "=r"(q.y), "=r"(q.z), "=r"(q.w) : "l"(p) : "memory");
  return q;
}
__device__ __forceinline__ uint2 load_uint2(const void* p) {
  uint2 q;
  asm volatile("ld.global.v2.b32 {%0, %1}, [%2];" : "=r"(q.x), "=r"(q.y) : "l"(p) : "memory");
  return q;
}
__device__ __forceinline__ uint32_t load_piece(const uint32_t* p) {
  uint32_t v;
  asm volatile("ld.global.b32 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_piece(const uint16_t* p) {
  uint16_t v;
  asm volatile("ld.global.b16 %0, [%1];" : "=h"(v) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint32_t load_piece(const uint8_t* p) {
  uint32_t v;
  asm volatile("ld.global.u8 %0, [%1];" : "=r"(v) : "l"(p) : "memory");
  return v;
}

template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), unsigned grid, unsigned block, size_t smem, unsigned cluster,
                              cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(grid);
  config.blockDim = dim3(block);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute attributes[2];
  attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[0].val.programmaticStreamSerializationAllowed = 1;
  attributes[1].id = cudaLaunchAttributeClusterDimension;
  attributes[1].val.clusterDim.x = cluster;
  attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
  config.attrs = attributes;
  config.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&config, kernel, std::forward<Args>(args)...);
}

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

// Sixteen values of one block, held by one of the two lanes that share it (lanes 2i and 2i + 1).
// Returns the block's scale byte and writes the codes: e4m3 into codes[0..3], e2m1 into codes[0..1].
template <int FORMAT>
__device__ __forceinline__ uint32_t mx_encode16(const float (&v)[16], uint32_t (&codes)[4]) {
  float top = fabsf(v[0]);
#pragma unroll
  for (int k = 1; k < 15; k += 2)  // the largest of three in one instruction, a NaN if there is one
    asm("max.NaN.f32 %0, %0, %1, %2;" : "+f"(top) : "f"(fabsf(v[k])), "f"(fabsf(v[k + 1])));
  asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(v[15])));
  uint32_t amax = __float_as_uint(top) & 0x7fffffffu;
  amax = max(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
  const uint32_t byte = mx_scale_byte<FORMAT>(amax);
  const float inv = mx_inverse(byte);
  const uint32_t keep = byte == 255u ? 0u : 0xffffffffu;  // a block that is not finite has codes 0
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float a = v[4 * i] * inv, b = v[4 * i + 1] * inv, c = v[4 * i + 2] * inv, d = v[4 * i + 3] * inv;
    if (FORMAT == FL_MX_FP8) {
      codes[i] = __byte_perm(cvt_e4m3x2(a, b), cvt_e4m3x2(c, d), 0x5410) & keep;
    } else {
      const uint32_t w = __byte_perm(cvt_e2m1x2(a, b), cvt_e2m1x2(c, d), 0x3340) & keep;
      if (i % 2 == 0) {
        codes[i / 2] = w;
      } else {
        codes[i / 2] |= w << 16;
      }
    }
  }
  return byte;
}
// The four scale bytes of a step from the eight lanes that hold it, in every one of them.
__device__ __forceinline__ uint32_t mx_join_scales(uint32_t byte) {
  uint32_t word = byte << (8 * ((threadIdx.x >> 1) & 3));
  word |= __shfl_xor_sync(0xffffffffu, word, 2);
  return word | __shfl_xor_sync(0xffffffffu, word, 4);
}

// Sixteen consecutive elements as they lie in memory.
template <typename T>
struct Raw16 {
  static constexpr int kWords = 4 * sizeof(T);  // of four bytes
  uint32_t w[kWords];
  __device__ __forceinline__ void unpack(float (&v)[16]) const {
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      if constexpr (sizeof(T) == 4) {
        v[k] = __uint_as_float(w[k]);
      } else if constexpr (std::is_same<T, __half>::value) {
        v[k] = k & 1 ? __high2float(as_half2(w[k / 2])) : __low2float(as_half2(w[k / 2]));
      } else {
        v[k] = k & 1 ? bf16_hi(w[k / 2]) : bf16_lo(w[k / 2]);
      }
    }
  }
};

// A load of Raw16 that can be under way while others are used: load() asks, get() waits.  `count` of the elements
// exist (none if it is not positive), the others are zero.
// ALIGN: the bytes at whose multiples base and row stride are known to lie.  16: loads of 16 bytes, of 32
// where the address allows.  Less: the warp, whose groups of eight lanes each hold 128 consecutive elements, loads
// them ALIGN bytes (and the rows' lengths are multiples of that) lane by lane and passes them on through 512 elements of
// shared memory, `stage`; all of its lanes make both calls.
template <typename T, int ALIGN>
struct Load16 {
  using Piece = std::conditional_t<ALIGN == 2, uint16_t, uint32_t>;
  static constexpr int kOfPiece = ALIGN / sizeof(T);    // elements
  static constexpr int kPieces = 128 / 32 / kOfPiece;   // of a lane and group
  uint32_t t[4 * kPieces];
  __device__ __forceinline__ void load(const T* p, int count) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const Piece* q = reinterpret_cast<const Piece*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(p), g * 8));
      const int total = __shfl_sync(0xffffffffu, count, g * 8);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        t[g * kPieces + i] = (lane + 32 * i) * kOfPiece < total ? load_piece(q + lane + 32 * i) : 0u;
    }
  }
  __device__ __forceinline__ Raw16<T> get(T* stage) const {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4 * kPieces; ++i) reinterpret_cast<Piece*>(stage)[lane + 32 * i] = Piece(t[i]);
    __syncwarp();
    Raw16<T> raw;
#pragma unroll
    for (int i = 0; i < Raw16<T>::kWords; i += 4) {
      const uint4 q = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(stage) + lane * Raw16<T>::kWords + i);
      raw.w[i] = q.x, raw.w[i + 1] = q.y, raw.w[i + 2] = q.z, raw.w[i + 3] = q.w;
    }
    return raw;
  }
};
template <typename T>
struct Load16<T, 16> {
  Raw16<T> raw;
  __device__ __forceinline__ void load(const T* p, int count) {
    constexpr int kWords = Raw16<T>::kWords;
    uint32_t (&w)[kWords] = raw.w;
    if (count >= 16 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
      for (int i = 0; i < kWords; i += 8)
        load_words(reinterpret_cast<const uint32_t*>(p) + i, w[i], w[i + 1], w[i + 2], w[i + 3], w[i + 4], w[i + 5],
                   w[i + 6], w[i + 7]);
      return;
    }
    constexpr int kEach = 16 / sizeof(T);  // elements of 16 bytes
#pragma unroll
    for (int i = 0; i < kWords; i += 4) {
      const int at = i / 4 * kEach, left = count - at;
      uint4 q = make_uint4(0u, 0u, 0u, 0u);
      if (left >= kEach) {
        q = load_uint4(p + at);
      } else if (left > 0) {  // rows that end inside 16 bytes
        using Bits = std::conditional_t<sizeof(T) == 2, uint16_t, uint32_t>;
        Bits t[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k)
          t[k] = k < left ? Bits(load_piece(reinterpret_cast<const Bits*>(p) + at + k)) : Bits(0);
        memcpy(&q, t, sizeof(t));
      }
      w[i] = q.x, w[i + 1] = q.y, w[i + 2] = q.z, w[i + 3] = q.w;
    }
  }
  __device__ __forceinline__ Raw16<T> get(T*) const { return raw; }
};
template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }

// Sixteen values rounded to T.
template <typename T>
__device__ __forceinline__ Raw16<T> pack16(const float (&v)[16]) {
  Raw16<T> raw;
#pragma unroll
  for (int i = 0; i < Raw16<T>::kWords; ++i) {
    if constexpr (sizeof(T) == 4) {
      raw.w[i] = __float_as_uint(v[i]);
    } else if constexpr (std::is_same<T, __half>::value) {
      raw.w[i] = as_u32(__floats2half2_rn(v[2 * i], v[2 * i + 1]));
    } else {
      const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
      memcpy(&raw.w[i], &h, 4);
    }
  }
  return raw;
}

// The first `count` of sixteen values (none if it is not positive) rounded to T and stored; `v` becomes what
// they are rounded to.  ALIGN, `stage` and the call by whole warps as for the load.
template <typename T, int ALIGN>
__device__ __forceinline__ void store16(T* p, int count, float (&v)[16], T* stage) {
  const Raw16<T> raw = pack16<T>(v);
  raw.unpack(v);
  const uint32_t* w = raw.w;
  if constexpr (ALIGN == 16) {
    uint32_t* q = reinterpret_cast<uint32_t*>(p);
    if (count >= 16 && (reinterpret_cast<uintptr_t>(p) & 31) == 0) {
#pragma unroll
      for (int i = 0; i < Raw16<T>::kWords; i += 8)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                     ::"l"(q + i), "r"(w[i]), "r"(w[i + 1]), "r"(w[i + 2]), "r"(w[i + 3]), "r"(w[i + 4]), "r"(w[i + 5]),
                       "r"(w[i + 6]), "r"(w[i + 7]) : "memory");
    } else {
      constexpr int kEach = 16 / sizeof(T);
#pragma unroll
      for (int i = 0; i < Raw16<T>::kWords; i += 4) {
        const int at = i / 4 * kEach, left = count - at;
        if (left >= kEach) {
          *reinterpret_cast<uint4*>(q + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
        } else if (left > 0) {
          T t[kEach];
          memcpy(t, w + i, sizeof(t));
#pragma unroll
          for (int k = 0; k < kEach; ++k)
            if (k < left) p[at + k] = t[k];
        }
      }
    }
  } else {
    const int lane = threadIdx.x & 31;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < Raw16<T>::kWords; i += 4)
      *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(stage) + lane * Raw16<T>::kWords + i) =
          make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
    __syncwarp();
    using Piece = typename Load16<T, ALIGN>::Piece;
    constexpr int kOfPiece = Load16<T, ALIGN>::kOfPiece, kPieces = Load16<T, ALIGN>::kPieces;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      Piece* base = reinterpret_cast<Piece*>(__shfl_sync(0xffffffffu, reinterpret_cast<uintptr_t>(p), g * 8));
      const int total = __shfl_sync(0xffffffffu, count, g * 8);
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        if ((lane + 32 * i) * kOfPiece < total)
          base[lane + 32 * i] = reinterpret_cast<const Piece*>(stage)[(g * kPieces + i) * 32 + lane];
    }
  }
}
// Shared memory of the warps for loads and stores of less than 16 bytes.
template <typename T, int ALIGN, int THREADS>
struct WarpStage {
  T data[THREADS / 32][ALIGN == 16 ? 16 : 512];
  __device__ __forceinline__ T* mine() { return data[threadIdx.x >> 5]; }
};

// Codes of sixteen elements starting at element `e` of a row (e a multiple of 16).
template <int FORMAT>
__device__ __forceinline__ void store_codes(uint8_t* row_codes, int64_t e, const uint32_t (&codes)[4]) {
  if (FORMAT == FL_MX_FP8) {
    *reinterpret_cast<uint4*>(row_codes + e) = make_uint4(codes[0], codes[1], codes[2], codes[3]);
  } else {
    *reinterpret_cast<uint2*>(row_codes + e / 2) = make_uint2(codes[0], codes[1]);
  }
}

// ------------------------------------------------------------------------------ host side

// Calls f with the largest of 16, 4 and 2 bytes at whose multiples the addresses or-ed into `at` all lie.
template <typename T, typename F>
auto by_alignment(uintptr_t at, F&& f) {
  if (at % 16 == 0) return f(std::integral_constant<int, 16>{});
  if constexpr (sizeof(T) == 2) {
    if (at % 4 != 0) return f(std::integral_constant<int, 2>{});
  }
  return f(std::integral_constant<int, 4>{});
}

inline int launched(cudaError_t err, const char* who) {
  if (err == cudaSuccess) return FL_OK;
  cudaGetLastError();
  set_error("%s: %s", who, cudaGetErrorString(err));
  return FL_ERR_CUDA;
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
// Whether an address is one of an element of this type (null is).
inline bool aligned_to(const void* p, int dtype) {
  return (reinterpret_cast<uintptr_t>(p) & (dtype == FL_DTYPE_F32 ? 3u : 1u)) == 0;
}
inline bool dtype_ok(int dtype) { return dtype == FL_DTYPE_BF16 || dtype == FL_DTYPE_F16 || dtype == FL_DTYPE_F32; }

#endif  // __CUDACC__

}  // namespace
}  // namespace fl
