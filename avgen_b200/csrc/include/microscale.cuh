// Block-scaled ("microscaled") formats: element codes, scale bytes and where a
// scale byte lies. Shared by the kernels that make, read and multiply them.
//
//   mxfp8  e4m3 elements, one power-of-two scale (e8m0 byte) per 32 columns
//   mxfp4  e2m1 elements, one power-of-two scale (e8m0 byte) per 32 columns
//   nvfp4  e2m1 elements, one e4m3 scale per 16 columns times one fp32 scale g
//          for the whole tensor
//
// A value is code * block scale (* g). Codes are row-major, columns padded with
// zero codes to a multiple of 32 so that every row starts on 16 bytes; two 4-bit
// codes share a byte, the even column in the low half. Scale bytes lie in tiles of
// 128 rows x 4 blocks (512 bytes), the layout the tensor cores read them in.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <type_traits>

namespace avgen {

enum MxFormat : int { kMxFp8 = 0, kMxFp4 = 1, kNvFp4 = 2 };

__host__ __device__ constexpr int mx_block(int fmt) { return fmt == kNvFp4 ? 16 : 32; }
__host__ __device__ constexpr int mx_bits(int fmt) { return fmt == kMxFp8 ? 8 : 4; }
__host__ __device__ constexpr long mx_row_bytes(int fmt, long cols) {
  return (cols + 31) / 32 * 32 * mx_bits(fmt) / 8;
}
// Tiles of four blocks along a row, and scale bytes of a whole tensor.
__host__ __device__ constexpr long mx_scale_tiles(int fmt, long cols) {
  return (cols + 4 * mx_block(fmt) - 1) / (4 * mx_block(fmt));
}
__host__ __device__ constexpr long mx_scale_bytes(int fmt, long rows, long cols) {
  return (rows + 127) / 128 * mx_scale_tiles(fmt, cols) * 512;
}

#ifdef __CUDACC__
// Smallest tensor scale: below it 1 / (block scale * g) would leave fp32's range.
constexpr float kMxScaleFloor = 7.888609052210118e-31f;  // 2^-100

// Bits of |x|. As whole numbers they order like |x|, with infinities and NaNs above
// every finite value, so one integer maximum finds both a block's largest value and
// whether the block holds a value that no scale can represent.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
constexpr uint32_t kInfBits = 0x7f800000u;

struct MxScale {
  uint32_t byte;  // stored scale
  float inv;      // elements are multiplied by this before rounding
};

// The tensor scale that makes the largest block scale 448, the largest e4m3 number.
__device__ __forceinline__ float nvfp4_tensor_scale(uint32_t amax_bits) {
  return fmaxf(__uint_as_float(amax_bits) * (1.0f / 2688.0f), kMxScaleFloor);
}

__device__ __forceinline__ uint32_t cvt_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %2, %1;" : "=h"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ uint32_t cvt_e4m3x4(float a, float b, float c, float d) {
  return cvt_e4m3x2(a, b) | (cvt_e4m3x2(c, d) << 16);
}
// Eight e2m1 codes, v[0] in the lowest four bits.
__device__ __forceinline__ uint32_t cvt_e2m1x8(const float* v) {
  uint32_t r;
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
      "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
      : "=r"(r)
      : "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint32_t two) {
  uint32_t h;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(h) : "h"(static_cast<uint16_t>(two)));
  return __half22float2(*reinterpret_cast<__half2*>(&h));
}
__device__ __forceinline__ float e4m3_to_float(uint32_t byte) { return e4m3x2_to_float2(byte & 0xffu).x; }
// Values of the eight e2m1 codes of a word.
__device__ __forceinline__ void e2m1x8_to_float(uint32_t w, float* v) {
  uint32_t h[4];
  asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
      "mov.b32 {b0, b1, b2, b3}, %4;\n\t"
      "cvt.rn.f16x2.e2m1x2 %0, b0;\n\t"
      "cvt.rn.f16x2.e2m1x2 %1, b1;\n\t"
      "cvt.rn.f16x2.e2m1x2 %2, b2;\n\t"
      "cvt.rn.f16x2.e2m1x2 %3, b3;\n\t}"
      : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
      : "r"(w));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(*reinterpret_cast<__half2*>(&h[i]));
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

// Scale of a block whose |values| have the integer maximum `amax`.
//
// Power-of-two formats: the smallest 2^s with amax <= top * 2^s, so nothing in the
// block saturates (top = 448 = 1.75 * 2^8 or 6 = 1.5 * 2^2): s follows from the
// exponent and a compare of the fraction. s stays within [-126, 126], where 2^s and
// 2^-s are both normal fp32 numbers and scaling is exact.
//
// nvfp4: amax / (6 g) rounded to e4m3; six_g = 6 * g, inv_six_g its rounded reciprocal. A
// block so small that this rounds to zero has all codes zero. The quotient is the
// correctly rounded one (Markstein, IBM J. Res. Dev. 34, 1990): with y = 1 / b rounded,
// q = a y and the exact remainder r = a - b q, q + r y rounds to a / b; a tiny quotient
// whose remainder is not exact rounds to zero, one that overflows saturates.
//
// A block with an infinity or a NaN gets the NaN scale: whatever its codes, it reads
// back as NaN, and so does every product it enters.
template <int FMT>
__device__ __forceinline__ MxScale mx_scale_of(uint32_t amax, float g, float six_g, float inv_six_g) {
  MxScale r;
  if constexpr (FMT == kNvFp4) {
    if (amax >= kInfBits) return {0x7fu, 0.f};
    const float a = __uint_as_float(amax), q = a * inv_six_g;
    r.byte = cvt_e4m3x2(fminf(fmaf(fmaf(-six_g, q, a), inv_six_g, q), 448.f), 0.f) & 0xffu;
    const float s = e4m3_to_float(r.byte);
    r.inv = r.byte != 0u ? __frcp_rn(s * g) : 0.f;
  } else {
    if (amax >= kInfBits) return {0xffu, 0.f};
    constexpr int kTopExp = FMT == kMxFp8 ? 8 : 2;
    constexpr uint32_t kTopFraction = FMT == kMxFp8 ? 0x600000u : 0x400000u;
    int s = static_cast<int>(amax >> 23) - 127 - kTopExp + ((amax & 0x7fffffu) > kTopFraction ? 1 : 0);
    s = max(-126, min(126, s));
    r.byte = static_cast<uint32_t>(s + 127);
    r.inv = __uint_as_float(static_cast<uint32_t>(127 - s) << 23);
  }
  return r;
}

// fp32 value of a stored block scale (without the tensor scale).
template <int FMT>
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
  if constexpr (FMT == kNvFp4) return e4m3_to_float(byte);
  if (byte == 0xffu) return __uint_as_float(0x7fffffffu);
  return byte == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(byte << 23);  // byte 0: 2^-127
}

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float<float>(float v) { return v; }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
// Two 16-bit values of a word.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
}
template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    lo = __uint_as_float(w << 16), hi = __uint_as_float(w & 0xffff0000u);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x, hi = f.y;
  }
}
#endif  // __CUDACC__

}  // namespace avgen
