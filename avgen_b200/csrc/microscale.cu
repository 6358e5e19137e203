// Quantising rows to block-scaled formats, reading them back, and the residual
// RMSNorm that writes its output quantised.
#include <algorithm>

#include "include/host_utils.h"
#include "include/launchers.h"
#include "include/microscale.cuh"
#include "include/sm100.cuh"

namespace avgen {
namespace {

// ---------------------------------------------------------------- quantise
template <typename T>
__global__ void __launch_bounds__(256) mx_amax_kernel(MxQuantDesc d) {
  uint32_t m = 0;
  const long n = d.rows * d.cols;
  for (long i = blockIdx.x * 256L + threadIdx.x; i < n; i += gridDim.x * 256L) {
    const long r = i / d.cols;
    const uint32_t b = abs_bits(to_float(reinterpret_cast<const T*>(d.x)[r * d.ldx + (i - r * d.cols)]));
    if (b < kInfBits) m = max(m, b);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if ((threadIdx.x & 31) == 0) atomicMax(d.amax, m);
}

// One thread per block of columns, over the scale tiles' whole area: rows and
// blocks past the tensor only get their (zero) scale bytes.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) mx_quantize_kernel(MxQuantDesc d, long tiles, long row_bytes) {
  constexpr int B = mx_block(FMT);
  const long blk = blockIdx.x * 256L + threadIdx.x;
  const long row = blockIdx.y + 65535L * blockIdx.z;
  if (blk >= 4 * tiles || row >= (d.rows + 127) / 128 * 128) return;
  float g = 1.f;
  if constexpr (FMT == kNvFp4) {
    g = d.amax != nullptr ? nvfp4_tensor_scale(*d.amax) : (d.g != nullptr ? *d.g : 1.f);
    if (d.amax != nullptr && blk == 0 && row == 0) *d.g_out = g;
  }
  uint8_t* scale = d.scales + mx_scale_word(row, blk / 4, tiles) + blk % 4;
  const long c0 = blk * B;
  if (row >= d.rows || c0 >= d.cols) {
    *scale = 0;
    if (row < d.rows && c0 * mx_bits(FMT) / 8 < row_bytes)
      for (int i = 0; i < B * mx_bits(FMT) / 8; ++i) d.codes[row * row_bytes + c0 * mx_bits(FMT) / 8 + i] = 0;
    return;
  }
  const T* x = reinterpret_cast<const T*>(d.x) + row * d.ldx + c0;
  float v[B];
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < B; ++i) {
    v[i] = c0 + i < d.cols ? to_float(x[i]) : 0.f;
    m = max(m, abs_bits(v[i]));
  }
  const MxScale s = mx_scale_of<FMT>(m, g, 6.f * g);
  *scale = static_cast<uint8_t>(s.byte);
#pragma unroll
  for (int i = 0; i < B; ++i) v[i] *= s.inv;
  uint32_t* out = reinterpret_cast<uint32_t*>(d.codes + row * row_bytes + c0 * mx_bits(FMT) / 8);
  if constexpr (FMT == kMxFp8) {
#pragma unroll
    for (int i = 0; i < B / 4; ++i) out[i] = cvt_e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
  } else {
#pragma unroll
    for (int i = 0; i < B / 8; ++i) out[i] = cvt_e2m1x8(v + 8 * i);
  }
}

// ---------------------------------------------------------------- read back
template <typename T, int FMT>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(MxDequantDesc d, long tiles, long row_bytes) {
  const long c0 = (blockIdx.x * 256L + threadIdx.x) * 8;
  const long row = blockIdx.y + 65535L * blockIdx.z;
  if (c0 >= d.cols || row >= d.rows) return;
  const long blk = c0 / mx_block(FMT);
  const float s = mx_scale_value<FMT>(d.scales[mx_scale_word(row, blk / 4, tiles) + blk % 4]);
  const float g = FMT == kNvFp4 && d.g != nullptr ? *d.g : 1.f;
  const uint32_t* in = reinterpret_cast<const uint32_t*>(d.codes + row * row_bytes + c0 * mx_bits(FMT) / 8);
  float v[8];
  if constexpr (FMT == kMxFp8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float2 lo = e4m3x2_to_float2(in[i] & 0xffffu), hi = e4m3x2_to_float2(in[i] >> 16);
      v[4 * i] = lo.x, v[4 * i + 1] = lo.y, v[4 * i + 2] = hi.x, v[4 * i + 3] = hi.y;
    }
  } else {
    e2m1x8_to_float(in[0], v);
  }
  T* out = reinterpret_cast<T*>(d.out) + row * d.cols + c0;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    if (c0 + i < d.cols) out[i] = from_float<T>(v[i] * s * g);
}

// ---------------------------------------------------------------- residual RMSNorm
__device__ __forceinline__ float block_sum(float v, float* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.f;
  for (int i = 0; i < static_cast<int>(blockDim.x) / 32; ++i) v += smem[i];
  return v;
}

// One CTA per row. The norm takes the fp32 sum, not its rounding to T.
template <typename T, int FMT>
__global__ void __launch_bounds__(256) mx_add_rmsnorm_kernel(MxNormDesc d, long tiles, long row_bytes) {
  constexpr int B = mx_block(FMT);
  __shared__ float red[8];
  const long row = blockIdx.x;
  const long words = row < d.rows ? 0 : tiles;
  for (long t = threadIdx.x; t < words; t += 256) *reinterpret_cast<uint32_t*>(d.scales + mx_scale_word(row, t, tiles)) = 0;
  if (row >= d.rows) return;
  const T* x = reinterpret_cast<const T*>(d.x) + row * d.ldx;
  const T* u = d.update != nullptr ? reinterpret_cast<const T*>(d.update) + row * d.ldu : nullptr;
  const long b = mod_row(d.groups, d.num_groups, row, d.rows_per_batch);
  const float* gate = d.gate != nullptr ? d.gate + b * d.gate_stride : nullptr;
  auto sum_at = [&](long c) {
    float v = to_float(x[c]);
    if (u != nullptr) v += (gate != nullptr ? gate[c] : 1.f) * to_float(u[c]);
    return v;
  };
  float ss = 0.f;
  for (long c = threadIdx.x; c < d.W; c += 256) {
    const float v = sum_at(c);
    ss += v * v;
    if (d.x_out != nullptr) reinterpret_cast<T*>(d.x_out)[row * d.W + c] = from_float<T>(v);
  }
  const float r = rsqrtf(block_sum(ss, red) / static_cast<float>(d.W) + d.eps);
  const float g = FMT == kNvFp4 && d.g != nullptr ? *d.g : 1.f;
  for (long blk = threadIdx.x; blk < 4 * tiles; blk += 256) {
    uint8_t* scale = d.scales + mx_scale_word(row, blk / 4, tiles) + blk % 4;
    uint8_t* out = d.codes + row * row_bytes + blk * B * mx_bits(FMT) / 8;
    if (blk * B >= d.W) {
      *scale = 0;
      if (blk * B * mx_bits(FMT) / 8 < row_bytes)
        for (int i = 0; i < B * mx_bits(FMT) / 8; ++i) out[i] = 0;
      continue;
    }
    float v[B];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < B; ++i) {
      const long c = blk * B + i;
      v[i] = 0.f;
      if (c < d.W) {
        v[i] = sum_at(c) * r;
        if (d.w != nullptr) v[i] *= d.w[c];
        if (d.scale != nullptr) v[i] *= 1.f + d.scale[b * d.mod_stride + c];
        if (d.shift != nullptr) v[i] += d.shift[b * d.mod_stride + c];
      }
      m = max(m, abs_bits(v[i]));
    }
    const MxScale s = mx_scale_of<FMT>(m, g, 6.f * g);
    *scale = static_cast<uint8_t>(s.byte);
#pragma unroll
    for (int i = 0; i < B; ++i) v[i] *= s.inv;
    if constexpr (FMT == kMxFp8) {
#pragma unroll
      for (int i = 0; i < B / 4; ++i)
        reinterpret_cast<uint32_t*>(out)[i] = cvt_e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    } else {
#pragma unroll
      for (int i = 0; i < B / 8; ++i) reinterpret_cast<uint32_t*>(out)[i] = cvt_e2m1x8(v + 8 * i);
    }
  }
}

template <typename T, int FMT>
void quantize(const MxQuantDesc& d, cudaStream_t stream) {
  const long tiles = mx_scale_tiles(FMT, d.cols);
  if (d.amax != nullptr) {
    AVGEN_CUDA_CHECK(cudaMemsetAsync(d.amax, 0, sizeof(uint32_t), stream));
    const long blocks = std::min<long>((d.rows * d.cols + 2047) / 2048, 8L * num_sms(d.device));
    mx_amax_kernel<T><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(d);
  }
  const long rows = (d.rows + 127) / 128 * 128;
  const dim3 grid(static_cast<unsigned>((4 * tiles + 255) / 256), static_cast<unsigned>(std::min(rows, 65535L)),
                  static_cast<unsigned>((rows + 65534) / 65535));
  mx_quantize_kernel<T, FMT><<<grid, 256, 0, stream>>>(d, tiles, mx_row_bytes(FMT, d.cols));
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT>
void dequantize(const MxDequantDesc& d, cudaStream_t stream) {
  const dim3 grid(static_cast<unsigned>((d.cols + 2047) / 2048), static_cast<unsigned>(std::min(d.rows, 65535L)),
                  static_cast<unsigned>((d.rows + 65534) / 65535));
  mx_dequantize_kernel<T, FMT>
      <<<grid, 256, 0, stream>>>(d, mx_scale_tiles(FMT, d.cols), mx_row_bytes(FMT, d.cols));
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT>
void add_rmsnorm(const MxNormDesc& d, cudaStream_t stream) {
  mx_add_rmsnorm_kernel<T, FMT><<<static_cast<unsigned>((d.rows + 127) / 128 * 128), 256, 0, stream>>>(
      d, mx_scale_tiles(FMT, d.W), mx_row_bytes(FMT, d.W));
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

}  // namespace

#define AVGEN_MX_DISPATCH(what, d, stream)                                                      \
  do {                                                                                          \
    if ((d).dtype == kMxBf16 && (d).fmt == kMxFp8) return what<__nv_bfloat16, kMxFp8>(d, stream); \
    if ((d).dtype == kMxBf16 && (d).fmt == kMxFp4) return what<__nv_bfloat16, kMxFp4>(d, stream); \
    if ((d).dtype == kMxBf16 && (d).fmt == kNvFp4) return what<__nv_bfloat16, kNvFp4>(d, stream); \
    if ((d).dtype == kMxFp16 && (d).fmt == kMxFp8) return what<__half, kMxFp8>(d, stream);        \
    if ((d).dtype == kMxFp16 && (d).fmt == kMxFp4) return what<__half, kMxFp4>(d, stream);        \
    if ((d).dtype == kMxFp16 && (d).fmt == kNvFp4) return what<__half, kNvFp4>(d, stream);        \
    if ((d).dtype == kMxFp32 && (d).fmt == kMxFp8) return what<float, kMxFp8>(d, stream);         \
    if ((d).dtype == kMxFp32 && (d).fmt == kMxFp4) return what<float, kMxFp4>(d, stream);         \
    if ((d).dtype == kMxFp32 && (d).fmt == kNvFp4) return what<float, kNvFp4>(d, stream);         \
    AVGEN_CHECK(false, #what ": unsupported type ", (d).dtype, " or format ", (d).fmt);           \
  } while (0)

void mx_quantize_launch(const MxQuantDesc& d, cudaStream_t stream) { AVGEN_MX_DISPATCH(quantize, d, stream); }
void mx_dequantize_launch(const MxDequantDesc& d, cudaStream_t stream) { AVGEN_MX_DISPATCH(dequantize, d, stream); }
void mx_add_rmsnorm_launch(const MxNormDesc& d, cudaStream_t stream) { AVGEN_MX_DISPATCH(add_rmsnorm, d, stream); }

}  // namespace avgen
