// Quantising rows to block-scaled formats, reading them back, and the residual
// RMSNorm that writes its output quantised.
//
// All three are bound by memory. In each, a lane owns 16 consecutive columns of a row
// (one nvfp4 block, half an mx block) and a warp 512: inputs of aligned rows arrive in
// 32-byte loads, a block's largest value needs at most one shuffle, the four scales of
// a tile's row one or two more, and codes leave in 8- or 16-byte stores. Rows of any
// other alignment pass through shared memory, so that global memory still sees a
// warp's accesses side by side.
#include <algorithm>

#include "include/host_utils.h"
#include "include/launchers.h"
#include "include/microscale.cuh"
#include "include/sm100.cuh"

namespace avgen {
namespace {

constexpr int kLane = 16;         // columns of a lane
constexpr int kSpan = 32 * kLane; // columns of a warp

// ---------------------------------------------------------------- 16 columns per lane
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
               : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& lo, float& hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    lo = bf16_lo(w), hi = bf16_hi(w);
  } else {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    lo = f.x, hi = f.y;
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    return pack_bf16(lo, hi);
  } else {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}

// A lane's 16 values as loaded: 8 words of 16-bit values or 16 of fp32.
template <typename T>
struct Raw {
  static constexpr int WORDS = kLane * sizeof(T) / 4;
  uint32_t w[WORDS];

  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void unpack(float (&v)[kLane]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kLane / 2; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void pack(const float (&v)[kLane]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < kLane; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < kLane / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
};

// Columns [c0, c0 + 16) of a row of `cols`, zero past its end; `c0` = the warp's first
// column + 16 * lane, `stage` 16 * 32 values of shared memory of the warp's own.
// Called by whole warps.
template <typename T, bool ALIGNED>
__device__ __forceinline__ void load16(const T* row, long c0, long cols, uint32_t* stage, Raw<T>& r) {
  if constexpr (ALIGNED) {  // cols is a multiple of 16
    if (c0 < cols) {
#pragma unroll
      for (int i = 0; i < Raw<T>::WORDS; i += 8) load32(reinterpret_cast<const uint32_t*>(row + c0) + i, r.w + i);
    } else {
      r.zero();
    }
  } else {
    T* s = reinterpret_cast<T*>(stage);
    const int lane = lane_id();
    const long base = c0 - kLane * lane;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const long c = base + 32 * i + lane;
      s[32 * i + lane] = c < cols ? row[c] : from_float<T>(0.f);
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < Raw<T>::WORDS; i += 4)
      *reinterpret_cast<uint4*>(r.w + i) = *reinterpret_cast<const uint4*>(stage + lane * Raw<T>::WORDS + i);
  }
}
template <typename T, bool ALIGNED>
__device__ __forceinline__ void store16(T* row, long c0, long cols, uint32_t* stage, const Raw<T>& r) {
  if constexpr (ALIGNED) {
    if (c0 < cols) {
#pragma unroll
      for (int i = 0; i < Raw<T>::WORDS; i += 8) store32(reinterpret_cast<uint32_t*>(row + c0) + i, r.w + i);
    }
  } else {
    const T* s = reinterpret_cast<const T*>(stage);
    const int lane = lane_id();
    const long base = c0 - kLane * lane;
    __syncwarp();
#pragma unroll
    for (int i = 0; i < Raw<T>::WORDS; i += 4)
      *reinterpret_cast<uint4*>(stage + lane * Raw<T>::WORDS + i) = *reinterpret_cast<const uint4*>(r.w + i);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kLane; ++i) {
      const long c = base + 32 * i + lane;
      if (c < cols) row[c] = s[32 * i + lane];
    }
  }
}

// Where a packed row goes.
struct PackedRows {
  uint8_t* codes;
  uint8_t* scales;
  long row_bytes;
  long tiles;
  long cols;
};

// Quantises and stores a lane's 16 values (zero past the row's end). Called by whole warps.
template <int FMT>
__device__ __forceinline__ void store_packed(const PackedRows& p, long row, long c0, float (&v)[kLane], float g,
                                             float six_g) {
  constexpr int B = mx_block(FMT);
  constexpr int LANES = B / kLane;  // lanes of a block
  const int lane = lane_id();
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kLane; ++i) m = max(m, abs_bits(v[i]));
  if constexpr (LANES == 2) m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  const MxScale s = mx_scale_of<FMT>(m, g, six_g);
  uint32_t word = (c0 & ~static_cast<long>(B - 1)) < p.cols ? s.byte << (8 * (lane / LANES & 3)) : 0u;
  word |= __shfl_xor_sync(0xffffffffu, word, LANES);
  word |= __shfl_xor_sync(0xffffffffu, word, 2 * LANES);
  const long tile = c0 / (4 * B);
  if (lane % (4 * LANES) == 0 && tile < p.tiles)
    *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, tile, p.tiles)) = word;
  const long at = c0 * mx_bits(FMT) / 8;
  if (at >= p.row_bytes) return;
#pragma unroll
  for (int i = 0; i < kLane; ++i) v[i] *= s.inv;
  uint8_t* out = p.codes + row * p.row_bytes + at;
  if constexpr (FMT == kMxFp8) {
    *reinterpret_cast<uint4*>(out) =
        make_uint4(cvt_e4m3x4(v[0], v[1], v[2], v[3]), cvt_e4m3x4(v[4], v[5], v[6], v[7]),
                   cvt_e4m3x4(v[8], v[9], v[10], v[11]), cvt_e4m3x4(v[12], v[13], v[14], v[15]));
  } else {
    *reinterpret_cast<uint2*>(out) = make_uint2(cvt_e2m1x8(v), cvt_e2m1x8(v + 8));
  }
}
// The (zero) scales of a row past the tensor, inside its last 128-row group.
__device__ __forceinline__ void store_pad_scales(const PackedRows& p, long row, long first_tile, long end_tile, int lane,
                                                 int lanes) {
  for (long t = first_tile + lane; t < min(end_tile, p.tiles); t += lanes)
    *reinterpret_cast<uint32_t*>(p.scales + mx_scale_word(row, t, p.tiles)) = 0u;
}

// ---------------------------------------------------------------- quantise
// Largest finite |value| of a lane's 16, as bits.
template <typename T>
__device__ __forceinline__ uint32_t finite_amax(const Raw<T>& r) {
  float v[kLane];
  r.unpack(v);
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    const uint32_t b = abs_bits(v[i]);
    m = max(m, b < kInfBits ? b : 0u);
  }
  return m;
}

// The tensor scale's pass: atomicMax of whole numbers, so the order does not matter.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) mx_amax_kernel(MxQuantDesc d, int segments) {
  __shared__ __align__(16) uint32_t stage[ALIGNED ? 1 : 8][kSpan * sizeof(T) / 4];
  const int warp = warp_id(), lane = lane_id();
  const long units = d.rows * segments;  // of one row x 512 columns
  uint32_t m = 0;
  for (long u = blockIdx.x * 8L + warp; u < units; u += gridDim.x * 8L) {
    const long row = u / segments;
    Raw<T> r;
    load16<T, ALIGNED>(reinterpret_cast<const T*>(d.x) + row * d.ldx, (u - row * segments) * kSpan + lane * kLane, d.cols,
                       stage[ALIGNED ? 0 : warp], r);
    m = max(m, finite_amax(r));
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0 && m != 0u) atomicMax(d.amax, m);
}

// A CTA quantises `rows_per_cta` rows x 512 columns, a warp one row at a time.
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(256) mx_quantize_kernel(MxQuantDesc d, PackedRows p, int rows_per_cta) {
  __shared__ __align__(16) uint32_t stage[ALIGNED ? 1 : 8][kSpan * sizeof(T) / 4];
  constexpr int UNROLL = ALIGNED ? (sizeof(T) == 2 ? 4 : 2) : 1;
  const int warp = warp_id(), lane = lane_id();
  // nvfp4 has just read the whole tensor for its scale: from the end, where L2 still holds it
  const long group = FMT == kNvFp4 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const long c0 = static_cast<long>(blockIdx.y) * kSpan + lane * kLane;
  float g = 1.f;
  if constexpr (FMT == kNvFp4) {
    if (d.amax != nullptr) {
      g = nvfp4_tensor_scale(*d.amax);
      if (group == 0 && blockIdx.y == 0 && threadIdx.x == 0) *d.g_out = g;
    } else if (d.g != nullptr) {
      g = *d.g;
    }
  }
  const float six_g = 6.f * g;
  const long end = min((d.rows + 127) / 128 * 128, (group + 1) * rows_per_cta);
  for (long row = group * rows_per_cta + warp; row < end; row += 8 * UNROLL) {
    Raw<T> r[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long at = row + 8 * i;
      if (at < min(end, d.rows))
        load16<T, ALIGNED>(reinterpret_cast<const T*>(d.x) + at * d.ldx, c0, d.cols, stage[ALIGNED ? 0 : warp], r[i]);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long at = row + 8 * i;
      if (at >= end) break;
      if (at < d.rows) {
        float v[kLane];
        r[i].unpack(v);
        store_packed<FMT>(p, at, c0, v, g, six_g);
      } else {
        constexpr int TILES = kSpan / (4 * mx_block(FMT));
        store_pad_scales(p, at, static_cast<long>(blockIdx.y) * TILES, static_cast<long>(blockIdx.y + 1) * TILES, lane, 32);
      }
    }
  }
}

// ---------------------------------------------------------------- read back
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(MxDequantDesc d, PackedRows p, int rows_per_cta) {
  __shared__ __align__(16) uint32_t stage[ALIGNED ? 1 : 8][kSpan * sizeof(T) / 4];
  constexpr int B = mx_block(FMT);
  constexpr int WORDS = kLane * mx_bits(FMT) / 32;
  constexpr int UNROLL = 4;
  const int warp = warp_id(), lane = lane_id();
  const long c0 = static_cast<long>(blockIdx.y) * kSpan + lane * kLane;
  const float g = FMT == kNvFp4 && d.g != nullptr ? *d.g : 1.f;
  const long end = min(d.rows, (blockIdx.x + 1L) * rows_per_cta);
  const long at = c0 * mx_bits(FMT) / 8;
  const bool inside = c0 < d.cols;
  for (long row = static_cast<long>(blockIdx.x) * rows_per_cta + warp; row < end; row += 8 * UNROLL) {
    uint32_t w[UNROLL][WORDS], sb[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long r = row + 8 * i;
      if (r < end && inside) {
        const uint32_t* in = reinterpret_cast<const uint32_t*>(p.codes + r * p.row_bytes + at);
        if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(w[i]) = *reinterpret_cast<const uint4*>(in);
        else *reinterpret_cast<uint2*>(w[i]) = *reinterpret_cast<const uint2*>(in);
        sb[i] = p.scales[mx_scale_word(r, c0 / (4 * B), p.tiles) + c0 / B % 4];
      }
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long r = row + 8 * i;
      if (r >= end) break;
      float v[kLane];
      Raw<T> out;
      if (inside) {
        const float s = mx_scale_value<FMT>(sb[i]);
        if constexpr (FMT == kMxFp8) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float2 lo = e4m3x2_to_float2(w[i][j] & 0xffffu), hi = e4m3x2_to_float2(w[i][j] >> 16);
            v[4 * j] = lo.x * s, v[4 * j + 1] = lo.y * s, v[4 * j + 2] = hi.x * s, v[4 * j + 3] = hi.y * s;
          }
        } else {
          e2m1x8_to_float(w[i][0], v);
          e2m1x8_to_float(w[i][1], v + 8);
#pragma unroll
          for (int j = 0; j < kLane; ++j) v[j] = FMT == kNvFp4 ? v[j] * s * g : v[j] * s;
        }
        out.pack(v);
      }
      store16<T, ALIGNED>(reinterpret_cast<T*>(d.out) + r * d.cols, c0, d.cols, stage[ALIGNED ? 0 : warp], out);
    }
  }
}

// ---------------------------------------------------------------- residual RMSNorm
// A CTA takes one row at a time, CHUNKS pieces of 16 columns per lane held in
// registers between the sum of squares and the store: x and the update are read once.
// The norm takes the fp32 sum x + gate * update, not its rounding to T; statistics,
// modulation and scaling stay in fp32 until the codes.
template <typename T, int FMT, int CHUNKS, bool ALIGNED>
__global__ void __launch_bounds__(CHUNKS == 4 ? 1024 : 512) mx_add_rmsnorm_kernel(MxNormDesc d, PackedRows p) {
  extern __shared__ __align__(16) uint32_t stages[];  // 512 fp32 per warp where rows are not aligned
  __shared__ float red[2][32];
  const int warp = warp_id(), lane = lane_id(), warps = blockDim.x >> 5;
  uint32_t* stage = ALIGNED ? nullptr : stages + warp * kSpan;
  const float g = FMT == kNvFp4 && d.g != nullptr ? *d.g : 1.f;
  const float six_g = 6.f * g;
  const long padded = (d.rows + 127) / 128 * 128;
  int turn = 0;
  for (long row = blockIdx.x; row < padded; row += gridDim.x) {
    if (row >= d.rows) {
      store_pad_scales(p, row, 0, p.tiles, threadIdx.x, blockDim.x);
      continue;
    }
    float v[CHUNKS][kLane];
    const T* x = reinterpret_cast<const T*>(d.x) + row * d.ldx;
    const long b = d.num_groups > 0 ? mod_row(d.groups, d.num_groups, row, d.rows_per_batch) : 0;
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const long c0 = static_cast<long>(i * warps + warp) * kSpan + lane * kLane;
      Raw<T> rx, ru;
      load16<T, ALIGNED>(x, c0, d.W, stage, rx);
      if (d.update != nullptr)
        load16<T, ALIGNED>(reinterpret_cast<const T*>(d.update) + row * d.ldu, c0, d.W, stage, ru);
      rx.unpack(v[i]);
      if (d.update != nullptr) {
        float u[kLane];
        ru.unpack(u);
        if (d.gate != nullptr) {
          Raw<float> t;
          load16<float, ALIGNED>(d.gate + b * d.gate_stride, c0, d.W, stage, t);
#pragma unroll
          for (int e = 0; e < kLane; ++e) v[i][e] = fmaf(__uint_as_float(t.w[e]), u[e], v[i][e]);
        } else {
#pragma unroll
          for (int e = 0; e < kLane; ++e) v[i][e] += u[e];
        }
        rx.pack(v[i]);
        store16<T, ALIGNED>(reinterpret_cast<T*>(d.x_out) + row * d.W, c0, d.W, stage, rx);
      }
#pragma unroll
      for (int e = 0; e < kLane; ++e) ss = fmaf(v[i][e], v[i][e], ss);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (lane == 0) red[turn][warp] = ss;
    __syncthreads();  // one per row: the next row's sums go to the other buffer
    ss = 0.f;
    for (int i = 0; i < warps; ++i) ss += red[turn][i];
    turn ^= 1;
    const float r = rsqrtf(ss / static_cast<float>(d.W) + d.eps);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const long c0 = static_cast<long>(i * warps + warp) * kSpan + lane * kLane;
      Raw<float> t;
#pragma unroll
      for (int e = 0; e < kLane; ++e) v[i][e] *= r;
      if (d.w != nullptr) {
        load16<float, ALIGNED>(d.w, c0, d.W, stage, t);
#pragma unroll
        for (int e = 0; e < kLane; ++e) v[i][e] *= __uint_as_float(t.w[e]);
      }
      if (d.scale != nullptr) {
        load16<float, ALIGNED>(d.scale + b * d.mod_stride, c0, d.W, stage, t);
#pragma unroll
        for (int e = 0; e < kLane; ++e) v[i][e] *= 1.f + __uint_as_float(t.w[e]);
      }
      if (d.shift != nullptr) {
        load16<float, ALIGNED>(d.shift + b * d.mod_stride, c0, d.W, stage, t);
#pragma unroll
        for (int e = 0; e < kLane; ++e) v[i][e] += __uint_as_float(t.w[e]);
      }
      if (c0 >= d.W) {  // 0 * (a statistic that overflowed) is not 0
#pragma unroll
        for (int e = 0; e < kLane; ++e) v[i][e] = 0.f;
      } else if (!ALIGNED) {
#pragma unroll
        for (int e = 0; e < kLane; ++e) v[i][e] = c0 + e < d.W ? v[i][e] : 0.f;
      }
      store_packed<FMT>(p, row, c0, v[i], g, six_g);
    }
  }
}

// ---------------------------------------------------------------- launches
bool aligned32(const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 32 == 0; }
// Whether rows of `cols` values of `size` bytes, `ld` values apart, all start on 32 bytes and end on 16 values.
bool rows_aligned(const void* ptr, long rows, long ld, long cols, int size) {
  return aligned32(ptr) && cols % kLane == 0 && (rows <= 1 || ld * size % 32 == 0);
}

// Rows of a CTA: as many as leave four CTAs for every SM (fewer, larger CTAs keep the
// scale tiles' lines in one place), at least one per warp.
int rows_per_cta(long rows, long segments, int sms) {
  for (int r = 128; r > 8; r /= 2)
    if ((rows + r - 1) / r * segments >= 4L * sms) return r;
  return 8;
}

template <typename T, int FMT, bool ALIGNED>
void quantize_as(const MxQuantDesc& d, const PackedRows& p, cudaStream_t stream) {
  const long segments = (p.tiles * 4 * mx_block(FMT) + kSpan - 1) / kSpan;
  AVGEN_CHECK(segments <= 65535, "quantize: too many columns: ", d.cols);
  const int sms = num_sms(d.device);
  if (d.amax != nullptr) {
    AVGEN_CUDA_CHECK(cudaMemsetAsync(d.amax, 0, sizeof(uint32_t), stream));
    const long blocks = std::min<long>((d.rows * segments + 31) / 32, 8L * sms);
    mx_amax_kernel<T, ALIGNED><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(d, static_cast<int>(segments));
  }
  const long rows = (d.rows + 127) / 128 * 128;
  const int rpc = rows_per_cta(d.rows, segments, sms);
  mx_quantize_kernel<T, FMT, ALIGNED>
      <<<dim3(static_cast<unsigned>(rows / rpc), static_cast<unsigned>(segments)), 256, 0, stream>>>(d, p, rpc);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT>
void quantize(const MxQuantDesc& d, cudaStream_t stream) {
  const PackedRows p{d.codes, d.scales, mx_row_bytes(FMT, d.cols), mx_scale_tiles(FMT, d.cols), d.cols};
  if (rows_aligned(d.x, d.rows, d.ldx, d.cols, sizeof(T))) quantize_as<T, FMT, true>(d, p, stream);
  else quantize_as<T, FMT, false>(d, p, stream);
}

template <typename T, int FMT, bool ALIGNED>
void dequantize_as(const MxDequantDesc& d, const PackedRows& p, cudaStream_t stream) {
  const long segments = (d.cols + kSpan - 1) / kSpan;
  AVGEN_CHECK(segments <= 65535, "dequantize: too many columns: ", d.cols);
  const int rpc = rows_per_cta(d.rows, segments, num_sms(d.device));
  mx_dequantize_kernel<T, FMT, ALIGNED>
      <<<dim3(static_cast<unsigned>((d.rows + rpc - 1) / rpc), static_cast<unsigned>(segments)), 256, 0, stream>>>(d, p, rpc);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT>
void dequantize(const MxDequantDesc& d, cudaStream_t stream) {
  const PackedRows p{const_cast<uint8_t*>(d.codes), const_cast<uint8_t*>(d.scales), mx_row_bytes(FMT, d.cols),
                     mx_scale_tiles(FMT, d.cols), d.cols};
  if (rows_aligned(d.out, d.rows, d.cols, d.cols, sizeof(T))) dequantize_as<T, FMT, true>(d, p, stream);
  else dequantize_as<T, FMT, false>(d, p, stream);
}

template <typename T, int FMT, int CHUNKS, bool ALIGNED>
void add_rmsnorm_as(const MxNormDesc& d, const PackedRows& p, int warps, cudaStream_t stream) {
  auto kernel = mx_add_rmsnorm_kernel<T, FMT, CHUNKS, ALIGNED>;
  const int smem = ALIGNED ? 0 : warps * kSpan * 4;
  static PerDeviceOnce once;
  if (!ALIGNED) raise_smem_limit(once, kernel, 32 * kSpan * 4);
  const long padded = (d.rows + 127) / 128 * 128;
  const long ctas = static_cast<long>(std::max(1, 64 / warps)) * num_sms(d.device);
  kernel<<<static_cast<unsigned>(std::min(padded, ctas)), 32 * warps, smem, stream>>>(d, p);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT, bool ALIGNED>
void add_rmsnorm_aligned(const MxNormDesc& d, const PackedRows& p, cudaStream_t stream) {
  const int spans = static_cast<int>(std::max<long>((d.W + kSpan - 1) / kSpan, 1));
  if (spans <= 8) return add_rmsnorm_as<T, FMT, 1, ALIGNED>(d, p, spans, stream);
  if (spans <= 32) return add_rmsnorm_as<T, FMT, 2, ALIGNED>(d, p, (spans + 1) / 2, stream);
  add_rmsnorm_as<T, FMT, 4, ALIGNED>(d, p, (spans + 3) / 4, stream);
}

template <typename T, int FMT>
void add_rmsnorm(const MxNormDesc& d, cudaStream_t stream) {
  AVGEN_CHECK(d.W <= kMxNormMaxCols, "add_rmsnorm: at most ", kMxNormMaxCols, " columns, got ", d.W);
  const PackedRows p{d.codes, d.scales, mx_row_bytes(FMT, d.W), mx_scale_tiles(FMT, d.W), d.W};
  auto mod = [&](const float* t, long stride) { return t == nullptr || (aligned32(t) && stride % 8 == 0); };
  const bool aligned = rows_aligned(d.x, d.rows, d.ldx, d.W, sizeof(T)) &&
                       (d.update == nullptr || (rows_aligned(d.update, d.rows, d.ldu, d.W, sizeof(T)) &&
                                                rows_aligned(d.x_out, d.rows, d.W, d.W, sizeof(T)))) &&
                       mod(d.w, 0) && mod(d.scale, d.mod_stride) && mod(d.shift, d.mod_stride) &&
                       mod(d.gate, d.gate_stride);
  if (aligned) add_rmsnorm_aligned<T, FMT, true>(d, p, stream);
  else add_rmsnorm_aligned<T, FMT, false>(d, p, stream);
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
