// Quantising rows to block-scaled formats, reading them back, and the residual
// RMSNorm that writes its output quantised.
//
// All three are bound by memory, quantising to 4 bits also by instruction issue. A lane
// owns 16 (norm: 8) consecutive columns: a block's largest value takes at most two
// shuffles, the scales of a tile's row are joined by two, codes leave in one store.
// Aligned rows are read and written in 16- and 32-byte accesses. Rows of any other
// alignment are read and written by every 32nd column, so that a warp's accesses still
// lie side by side, and change layout in shared memory.
//
// Measured on a B200 whose plain copy runs at 6.56 TB/s; 65536 x 2560 bf16 where no size
// is given, bytes counted once each (us, TB/s):
//   quantise   mxfp8 83 (6.1), mxfp4 73 (5.8), nvfp4 with a given tensor scale 77 (5.6),
//              with its own 134; fp32 13824 x 5120 to mxfp4 54 (6.0); 20000 x 5001 to
//              mxfp4, rows not aligned, 69 (3.7)
//   read back  mxfp8 85 (6.0), 4 bits 74 (5.8); 20000 x 5001 from mxfp4 60 (4.2)
//   norm       to mxfp8 192 to 203 (6.1 to 5.8), with two modulation levels 203 to 221; to
//              mxfp4 173 (6.3) and 200, to nvfp4 186 (5.9) and 223; of fp32 rows to mxfp8 354
//              (6.2) and 365; 16387 x 5120 95 (6.2) and 111; 20000 x 5001, whose rows are not
//              aligned, 227 (3.1) and 309; 4096 x 40000 476 (2.4) and 793, of fp32 930 and 1089
#include <algorithm>
#include <limits>

#include "include/host_utils.h"
#include "include/launchers.h"
#include "include/microscale.cuh"
#include "include/sm100.cuh"

namespace avgen {
namespace {

constexpr uint32_t kAllLanes = 0xffffffffu;

// ---------------------------------------------------------------- global memory
// Inputs are never written by the kernel that reads them (ld.global.nc).
__device__ __forceinline__ void load32(const void* p, uint32_t* w) {
  asm("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
      : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
      : "l"(p));
}
__device__ __forceinline__ void load16(const void* p, uint32_t* w) {
  asm("ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "l"(p));
}
__device__ __forceinline__ void store32(void* p, const uint32_t* w) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
               "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void store16(void* p, const uint32_t* w) {
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

// abs_bits of the largest magnitude; a NaN among the values gives one (three-input
// maximum, two values an instruction).
template <int N>
__device__ __forceinline__ uint32_t amax_of(const float (&v)[N]) {
  float m = 0.f;
#pragma unroll
  for (int i = 0; i < N; i += 2)
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(m) : "f"(m), "f"(fabsf(v[i])), "f"(fabsf(v[i + 1])));
  return __float_as_uint(m);
}

// Two fp32 values in one 64-bit register: one instruction does both.
struct Pair {
  unsigned long long b;

  __device__ __forceinline__ Pair(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(b) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(b));
  }
  __device__ __forceinline__ Pair operator*(Pair o) const {
    Pair r = *this;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.b) : "l"(b), "l"(o.b));
    return r;
  }
  __device__ __forceinline__ Pair operator+(Pair o) const {
    Pair r = *this;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.b) : "l"(b), "l"(o.b));
    return r;
  }
  // this * o + c
  __device__ __forceinline__ Pair times_plus(Pair o, Pair c) const {
    Pair r = *this;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.b) : "l"(b), "l"(o.b), "l"(c.b));
    return r;
  }
};

// v[i] *= s
template <int N>
__device__ __forceinline__ void scale_all(float (&v)[N], float s) {
  const Pair ss(s, s);
#pragma unroll
  for (int i = 0; i < N; i += 2) (Pair(v[i], v[i + 1]) * ss).get(v[i], v[i + 1]);
}

// N values of type T as they lie in memory.
template <typename T, int N>
struct Raw {
  static constexpr int WORDS = N * sizeof(T) / 4;
  uint32_t w[WORDS];

  // From / to an address on 32 bytes (or on all of a shorter run).
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (WORDS == 4) {
      load16(p, w);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 8) load32(reinterpret_cast<const uint32_t*>(p) + i, w + i);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (WORDS == 4) {
      store16(p, w);
    } else {
#pragma unroll
      for (int i = 0; i < WORDS; i += 8) store32(reinterpret_cast<uint32_t*>(p) + i, w + i);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < WORDS; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void unpack(float (&v)[N]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = __uint_as_float(w[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void pack(const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < N; ++i) w[i] = __float_as_uint(v[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N / 2; ++i) w[i] = pack2<T>(v[2 * i], v[2 * i + 1]);
    }
  }
  // abs_bits of the largest magnitude. 16-bit values are compared two at a time by their
  // own bits, which order like theirs as fp32.
  __device__ __forceinline__ uint32_t amax() const {
    if constexpr (sizeof(T) == 4) {
      float v[N];
      unpack(v);
      return amax_of(v);
    } else {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < WORDS; i += 2)
        m = __vimax3_u16x2(m, w[i] & 0x7fff7fffu, w[i + 1] & 0x7fff7fffu);
      const uint32_t top = max(m & 0xffffu, m >> 16);
      if constexpr (std::is_same<T, __nv_bfloat16>::value) return top << 16;
      return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(top))));
    }
  }
};

// ---------------------------------------------------------------- packed rows
struct PackedRows {
  uint8_t* codes;
  uint8_t* scales;
  long row_bytes;
  long tiles;
  long cols;

  __device__ __forceinline__ uint8_t* codes_of(long row) const { return codes + row * row_bytes; }
  // The scales of a row's first tile.
  __device__ __forceinline__ uint8_t* scales_of(long row) const {
    const uint32_t r = static_cast<uint32_t>(row);
    return scales + static_cast<long>(r >> 7) * (tiles * 512) + (r & 31u) * 16 + (r >> 5 & 3u) * 4;
  }
};

// What a lane with the N columns from c0 (a multiple of N) stores in every row. Lanes of a
// warp lie side by side.
template <int FMT, int N>
struct LanePlace {
  static constexpr int B = mx_block(FMT);
  static constexpr int LANES = B / N;  // lanes of a block
  uint32_t code_at;   // offset of its codes, or past any row
  uint32_t scale_at;  // offset of the scale word it writes, or past any tile
  uint32_t byte_mask; // its block's place in that word, or none

  __device__ __forceinline__ LanePlace(const PackedRows& p, long c0) {
    const int lane = lane_id();
    const long at = c0 * mx_bits(FMT) / 8, tile = c0 / (4 * B);
    code_at = at < p.row_bytes ? static_cast<uint32_t>(at) : ~0u;
    scale_at = lane % (4 * LANES) == 0 && tile < p.tiles ? static_cast<uint32_t>(tile * 512) : ~0u;
    byte_mask = (c0 & ~static_cast<long>(B - 1)) < p.cols ? 0xffu << (8 * (lane / LANES & 3)) : 0u;
  }
};

// Quantises and stores a lane's N values (zero past the row's end), whose largest
// magnitude is `m`. Called by whole warps.
template <int FMT, int N>
__device__ __forceinline__ void store_packed(const LanePlace<FMT, N>& at, uint8_t* codes, uint8_t* scales,
                                             float (&v)[N], uint32_t m, float g, float six_g, float inv_six_g) {
  constexpr int LANES = LanePlace<FMT, N>::LANES;
  if constexpr (LANES >= 2) m = max(m, __shfl_xor_sync(kAllLanes, m, 1));
  if constexpr (LANES >= 4) m = max(m, __shfl_xor_sync(kAllLanes, m, 2));
  const MxScale s = mx_scale_of<FMT>(m, g, six_g, inv_six_g);
  uint32_t word = (s.byte * 0x01010101u) & at.byte_mask;
  word |= __shfl_xor_sync(kAllLanes, word, LANES);
  word |= __shfl_xor_sync(kAllLanes, word, 2 * LANES);
  if (at.scale_at != ~0u) *reinterpret_cast<uint32_t*>(scales + at.scale_at) = word;
  if (at.code_at == ~0u) return;
  scale_all(v, s.inv);
  constexpr int WORDS = N * mx_bits(FMT) / 32;
  uint32_t w[WORDS];
#pragma unroll
  for (int i = 0; i < WORDS; ++i) {
    if constexpr (FMT == kMxFp8) w[i] = cvt_e4m3x4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
    else w[i] = cvt_e2m1x8(v + 8 * i);
  }
  uint32_t* out = reinterpret_cast<uint32_t*>(codes + at.code_at);
  if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(out) = make_uint4(w[0], w[1], w[2], w[3]);
  else if constexpr (WORDS == 2) *reinterpret_cast<uint2*>(out) = make_uint2(w[0], w[1]);
  else *out = w[0];
}

// The (zero) scales of a row past the tensor, inside its last 128-row group.
__device__ __forceinline__ void store_pad_scales(const PackedRows& p, long row, long first_tile, long end_tile,
                                                 int lane, int lanes) {
  for (long t = first_tile + lane; t < min(end_tile, p.tiles); t += lanes)
    *reinterpret_cast<uint32_t*>(p.scales_of(row) + t * 512) = 0u;
}

// ---------------------------------------------------------------- quantise
constexpr int kLane = 16;          // columns of a lane
constexpr int kSpan = 32 * kLane;  // columns of a warp

// 512 columns of an unaligned row: read side by side, handed to the lanes that own them
// through the warp's `stage`, and back.
template <typename T>
struct Unaligned {
  T v[kLane];  // columns base + 32 j + lane

  __device__ __forceinline__ void load(const T* row, long base, long cols) {
    const T* at = row + base + lane_id();
    if (base + kSpan <= cols) {  // no bounds inside the row
#pragma unroll
      for (int j = 0; j < kLane; ++j) v[j] = at[32 * j];
    } else {
      const int end = static_cast<int>(cols - base) - lane_id();
#pragma unroll
      for (int j = 0; j < kLane; ++j) v[j] = 32 * j < end ? at[32 * j] : from_float<T>(0.f);
    }
  }
  __device__ __forceinline__ void to_lanes(T* stage, Raw<T, kLane>& r) const {
    __syncwarp();
#pragma unroll
    for (int j = 0; j < kLane; ++j) stage[32 * j + lane_id()] = v[j];
    __syncwarp();
#pragma unroll
    for (int i = 0; i < r.WORDS; i += 4)
      *reinterpret_cast<uint4*>(r.w + i) = reinterpret_cast<const uint4*>(stage + lane_id() * kLane)[i / 4];
  }
  static __device__ __forceinline__ void store(T* row, long base, long cols, T* stage, const Raw<T, kLane>& r) {
    __syncwarp();
#pragma unroll
    for (int i = 0; i < r.WORDS; i += 4)
      reinterpret_cast<uint4*>(stage + lane_id() * kLane)[i / 4] = *reinterpret_cast<const uint4*>(r.w + i);
    __syncwarp();
    T* at = row + base + lane_id();
    const T* from = stage + lane_id();
    if (base + kSpan <= cols) {
#pragma unroll
      for (int j = 0; j < kLane; ++j) at[32 * j] = from[32 * j];
    } else {
      const int end = static_cast<int>(cols - base) - lane_id();
#pragma unroll
      for (int j = 0; j < kLane; ++j)
        if (32 * j < end) at[32 * j] = from[32 * j];
    }
  }
};

__device__ __forceinline__ uint32_t finite_max(const float (&v)[kLane]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kLane; ++i) {
    const uint32_t b = abs_bits(v[i]);
    m = max(m, b < kInfBits ? b : 0u);
  }
  return m;
}
// The same, a few instructions where all values are finite.
template <typename T>
__device__ __forceinline__ uint32_t finite_max(const Raw<T, kLane>& r) {
  const uint32_t m = r.amax();
  if (m < kInfBits) return m;
  float v[kLane];
  r.unpack(v);
  return finite_max(v);
}

// The tensor scale's pass: each CTA writes the largest finite |value| it saw, and the
// quantising CTAs take the maximum of those words. The second read of x is what a scale of
// the whole tensor costs; the quantising pass runs from the tensor's end, which L2 holds.
template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(256) mx_amax_kernel(MxQuantDesc d) {
  constexpr int UNROLL = ALIGNED ? 4 : 1;
  const int lane = lane_id();
  const long base = static_cast<long>(blockIdx.y) * kSpan;
  const long c0 = base + lane * kLane;
  const long step = gridDim.x * 8L;
  __shared__ uint32_t warp_max[8];
  uint32_t m = 0;
  for (long row = blockIdx.x * 8L + warp_id(); row < d.rows; row += UNROLL * step) {
    if constexpr (ALIGNED) {
      Raw<T, kLane> r[UNROLL];
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) {
        const long at = row + i * step;
        if (at < d.rows && c0 < d.cols) r[i].load(reinterpret_cast<const T*>(d.x) + at * d.ldx + c0);
        else r[i].zero();
      }
#pragma unroll
      for (int i = 0; i < UNROLL; ++i) m = max(m, finite_max(r[i]));
    } else {
      Unaligned<T> u;
      u.load(reinterpret_cast<const T*>(d.x) + row * d.ldx, base, d.cols);
      float v[kLane];
#pragma unroll
      for (int i = 0; i < kLane; ++i) v[i] = to_float(u.v[i]);
      m = max(m, finite_max(v));
    }
  }
  m = __reduce_max_sync(kAllLanes, m);
  if (lane == 0) warp_max[warp_id()] = m;
  __syncthreads();
  if (warp_id() == 0) {
    m = __reduce_max_sync(kAllLanes, lane < 8 ? warp_max[lane] : 0u);
    if (lane == 0) d.amax[blockIdx.y * gridDim.x + blockIdx.x] = m;
  }
}

// A CTA quantises `rows_per_cta` rows x 512 columns, a warp one row at a time with the
// loads of four in flight. About seven instructions per value to 4 bits, which at the copy
// rate is most of what an SM issues: maxima are taken on the 16-bit values two at a time
// and scaling two at a time in fp32 (nvfp4 with a given tensor scale 94 -> 79 us).
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(256, 4)
    mx_quantize_kernel(MxQuantDesc d, PackedRows p, int rows_per_cta) {
  constexpr int UNROLL = !ALIGNED ? 1 : sizeof(T) == 2 ? 4 : 2;
  __shared__ __align__(16) T stage[ALIGNED ? 1 : 8][ALIGNED ? 8 : kSpan];
  const int warp = warp_id(), lane = lane_id();
  // nvfp4 has just read the whole tensor for its scale: from the end, where L2 still holds it
  const long group = FMT == kNvFp4 ? gridDim.x - 1 - blockIdx.x : blockIdx.x;
  const long base = static_cast<long>(blockIdx.y) * kSpan;
  const long c0 = base + lane * kLane;
  float g = 1.f;
  if constexpr (FMT == kNvFp4) {
    if (d.amax != nullptr) {
      __shared__ uint32_t warp_max[8];
      uint32_t m = 0;
      for (int i = threadIdx.x; i < d.parts; i += 256) m = max(m, d.amax[i]);
      m = __reduce_max_sync(kAllLanes, m);
      if (lane == 0) warp_max[warp] = m;
      __syncthreads();
      g = nvfp4_tensor_scale(__reduce_max_sync(kAllLanes, warp_max[lane & 7]));
      if (group == 0 && blockIdx.y == 0 && threadIdx.x == 0) *d.g_out = g;
    } else if (d.g != nullptr) {
      g = *d.g;
    }
  }
  const float six_g = 6.f * g, inv_six_g = __frcp_rn(six_g);
  const LanePlace<FMT, kLane> place(p, c0);
  const long end = min((d.rows + 127) / 128 * 128, (group + 1) * rows_per_cta);
  for (long row = group * rows_per_cta + warp; row < end; row += 8 * UNROLL) {
    Raw<T, kLane> r[UNROLL];
    Unaligned<T> u[ALIGNED ? 1 : UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long at = row + 8 * i;
      const T* x = reinterpret_cast<const T*>(d.x) + at * d.ldx;
      if constexpr (ALIGNED) {
        if (at < min(end, d.rows) && c0 < d.cols) r[i].load(x + c0);
        else r[i].zero();
      } else if (at < min(end, d.rows)) {
        u[i].load(x, base, d.cols);
      }
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long at = row + 8 * i;
      if (at >= end) break;
      if (at < d.rows) {
        float v[kLane];
        if constexpr (!ALIGNED) u[i].to_lanes(stage[warp], r[i]);
        r[i].unpack(v);
        store_packed<FMT>(place, p.codes_of(at), p.scales_of(at), v, r[i].amax(), g, six_g, inv_six_g);
      } else {
        constexpr int TILES = kSpan / (4 * mx_block(FMT));
        const long first_tile = static_cast<long>(blockIdx.y) * TILES;
        store_pad_scales(p, at, first_tile, first_tile + TILES, lane, 32);
      }
    }
  }
}

// Small nvfp4 tensors in one launch of one cluster: every warp holds one row x 512
// columns while the CTAs exchange their maxima (1 x 2560: 15 -> 8 us a call against
// clearing a word, measuring and quantising in three launches).
constexpr int kSmallWarps = 16, kSmallCtas = 8;

template <typename T, bool ALIGNED>
__global__ void __launch_bounds__(32 * kSmallWarps)
    mx_quantize_small_kernel(MxQuantDesc d, PackedRows p, int segments) {
  __shared__ __align__(16) T stage[ALIGNED ? 1 : kSmallWarps][ALIGNED ? 8 : kSpan];
  __shared__ uint32_t warp_max[kSmallWarps];
  __shared__ uint32_t cta_max[kSmallCtas];  // every CTA writes its word in every CTA
  const int warp = warp_id(), lane = lane_id(), ctas = gridDim.x;
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");  // waited for below: every CTA has started
  const int unit = blockIdx.x * kSmallWarps + warp;
  const long row = unit / segments, base = static_cast<long>(unit % segments) * kSpan, c0 = base + lane * kLane;
  const T* x = reinterpret_cast<const T*>(d.x) + row * d.ldx;
  Raw<T, kLane> r;
  r.zero();
  if (row < d.rows) {
    if constexpr (ALIGNED) {
      if (c0 < d.cols) r.load(x + c0);
    } else {
      Unaligned<T> u;
      u.load(x, base, d.cols);
      u.to_lanes(stage[warp], r);
    }
  }
  const uint32_t m = __reduce_max_sync(kAllLanes, finite_max(r));
  if (lane == 0) warp_max[warp] = m;
  __syncthreads();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  if (warp == 0) {
    const uint32_t all = __reduce_max_sync(kAllLanes, warp_max[lane % kSmallWarps]);
    if (lane < ctas) {
      uint32_t at;  // of this CTA's word in CTA `lane`
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(&cta_max[blockIdx.x])), "r"(lane));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(all) : "memory");
    }
  }
  // the scales past the tensor meanwhile
  const long pad = (p.tiles * ((d.rows + 127) / 128 * 128 - d.rows));
  for (long i = blockIdx.x * blockDim.x + threadIdx.x; i < pad; i += static_cast<long>(ctas) * blockDim.x)
    *reinterpret_cast<uint32_t*>(p.scales_of(d.rows + i / p.tiles) + i % p.tiles * 512) = 0u;
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  const float g = nvfp4_tensor_scale(__reduce_max_sync(kAllLanes, lane < ctas ? cta_max[lane % kSmallCtas] : 0u));
  if (blockIdx.x == 0 && threadIdx.x == 0) *d.g_out = g;
  if (row >= d.rows) return;
  float v[kLane];
  r.unpack(v);
  const float six_g = 6.f * g;
  store_packed<kNvFp4>(LanePlace<kNvFp4, kLane>(p, c0), p.codes_of(row), p.scales_of(row), v, r.amax(), g, six_g,
                       __frcp_rn(six_g));
}

// ---------------------------------------------------------------- read back
// code * block scale (* g), exact products of the first two, rounded once to T.
template <typename T, int FMT, bool ALIGNED>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(MxDequantDesc d, PackedRows p, int rows_per_cta) {
  constexpr int B = mx_block(FMT);
  constexpr int WORDS = kLane * mx_bits(FMT) / 32;
  constexpr int UNROLL = ALIGNED ? 4 : 1;
  __shared__ __align__(16) T stage[ALIGNED ? 1 : 8][ALIGNED ? 8 : kSpan];
  const int warp = warp_id(), lane = lane_id();
  const long base = static_cast<long>(blockIdx.y) * kSpan;
  const long c0 = base + lane * kLane;
  const float g = FMT == kNvFp4 && d.g != nullptr ? *d.g : 1.f;
  const long end = min(d.rows, (blockIdx.x + 1L) * rows_per_cta);
  const long at = c0 * mx_bits(FMT) / 8;
  const long scale_at = c0 / (4 * B) * 512 + c0 / B % 4;
  const bool inside = c0 < d.cols;
  for (long row = static_cast<long>(blockIdx.x) * rows_per_cta + warp; row < end; row += 8 * UNROLL) {
    uint32_t w[UNROLL][WORDS] = {}, sb[UNROLL] = {};
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long r = row + 8 * i;
      if (r < end && inside) {
        const uint32_t* in = reinterpret_cast<const uint32_t*>(p.codes_of(r) + at);
        if constexpr (WORDS == 4) *reinterpret_cast<uint4*>(w[i]) = __ldg(reinterpret_cast<const uint4*>(in));
        else *reinterpret_cast<uint2*>(w[i]) = __ldg(reinterpret_cast<const uint2*>(in));
        sb[i] = __ldg(p.scales_of(r) + scale_at);
      }
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long r = row + 8 * i;
      if (r >= end) break;
      if (ALIGNED && !inside) break;
      float v[kLane];
      const float s = mx_scale_value<FMT>(sb[i]);
      if constexpr (FMT == kMxFp8) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 lo = e4m3x2_to_float2(w[i][j] & 0xffffu), hi = e4m3x2_to_float2(w[i][j] >> 16);
          v[4 * j] = lo.x, v[4 * j + 1] = lo.y, v[4 * j + 2] = hi.x, v[4 * j + 3] = hi.y;
        }
      } else {
        e2m1x8_to_float(w[i][0], v);
        e2m1x8_to_float(w[i][1], v + 8);
      }
      scale_all(v, s);
      if constexpr (FMT == kNvFp4) scale_all(v, g);
      Raw<T, kLane> out;
      out.pack(v);
      T* dst = reinterpret_cast<T*>(d.out) + r * d.cols;
      if constexpr (ALIGNED) out.store(dst + c0);
      else Unaligned<T>::store(dst, base, d.cols, stage[warp], out);
    }
  }
}

// ---------------------------------------------------------------- residual RMSNorm
constexpr int kNormLane = 8;  // columns of a lane in one chunk: fp32 modulation rows in 32-byte loads side by side
constexpr int kNormSpan = 32 * kNormLane;

// What a missing row reads as, in the aligned layout (eight columns, the same for every lane).
__device__ const __align__(32) float kNormZeros[kNormLane] = {};
__device__ const __align__(32) float kNormOnes[kNormLane] = {1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f, 1.f};

// A row of the input or of a modulation, or `other` (0 or 1) in every column where there
// is none. An aligned row is read without conditions: lanes past its end read its first
// columns, a missing row is a short constant one.
template <typename T, bool ALIGNED>
struct NormRow {
  const T* row;
  int mask;  // of a lane's column
  float other;

  __device__ __forceinline__ NormRow(const T* base, long at, float other_) : other(other_) {
    mask = base != nullptr ? ~0 : 0;
    row = base != nullptr ? base + at : nullptr;
    if (ALIGNED && base == nullptr) row = reinterpret_cast<const T*>(other_ == 0.f ? kNormZeros : kNormOnes);
  }
};

// Eight columns per lane of the 256-column chunk at `base`: consecutive ones of an
// aligned row, every 32nd of any other.
template <typename T, bool ALIGNED>
struct Chunk {
  Raw<T, kNormLane> r;

  // `column`: the lane's first one in this chunk, or 0 where that lies past the row's end.
  __device__ __forceinline__ void load(const NormRow<T, ALIGNED>& from, int base, int column, int cols) {
    if constexpr (ALIGNED) {
      r.load(from.row + (column & from.mask));
    } else {
      const int lane = lane_id();
      const T* at = from.row + base + lane;
      T v[kNormLane];
      if (from.row != nullptr && base + kNormSpan <= cols) {  // a whole chunk: no bounds
#pragma unroll
        for (int e = 0; e < kNormLane; ++e) v[e] = at[32 * e];
      } else {
        const int end = from.row != nullptr ? cols - base - lane : 0;
#pragma unroll
        for (int e = 0; e < kNormLane; ++e) v[e] = 32 * e < end ? at[32 * e] : from_float<T>(from.other);
      }
      memcpy(r.w, v, sizeof(v));
    }
  }
  __device__ __forceinline__ void store(T* row, int base, int cols) const {
    const int lane = lane_id();
    if constexpr (ALIGNED) {
      const int c = base + lane * kNormLane;
      if (c < cols) r.store(row + c);
    } else {
      T* at = row + base + lane;
      T v[kNormLane];
      memcpy(v, r.w, sizeof(v));
      if (base + kNormSpan <= cols) {
#pragma unroll
        for (int e = 0; e < kNormLane; ++e) at[32 * e] = v[e];
      } else {
        const int end = cols - base - lane;
#pragma unroll
        for (int e = 0; e < kNormLane; ++e)
          if (32 * e < end) at[32 * e] = v[e];
      }
    }
  }
  __device__ __forceinline__ Pair pair(int e) const { return {__uint_as_float(r.w[e]), __uint_as_float(r.w[e + 1])}; }
};

// 1 / sqrt(x), the hardware's approximation improved by a Newton step: an error of a row's
// factor moves all of the row's values towards the same side of their roundings. Outside
// the step's range (0, infinity, NaN) the approximation stands.
__device__ __forceinline__ float inverse_root(float x) {
  const float r = rsqrtf(x);
  const float e = fmaf(-x * r, r, 1.f);
  return fabsf(e) < 0.5f ? fmaf(0.5f * r, e, r) : r;
}

// A row is held on its SM, CHUNKS x 8 columns per lane, between its sum of squares
// and its store: x and the update are read once. Rows of up to 768 columns take one
// warp each (WARP_ROWS) and no barrier; longer ones a CTA, with one barrier per row. The
// next row's x and update are requested before the reduction, so that loads stay in
// flight through it.
//
// Up to 16384 columns that is in registers, but for fp32 rows and modulated 16-bit ones of no
// alignment, which spill up to 450 bytes a thread (16-bit ones of 257 to 512 columns 64). Wider
// rows (8 chunks) take 1024 threads of 64 registers, as many as their own 64 values: they
// spill 0.7 to 1.5 KB a thread, of fp32 1.8 to 3.2 KB, and run at 1.4 to 2.4 TB/s.
//
// The norm takes the fp32 sum x + gate * update, not its rounding to T; statistics,
// modulation and scaling stay in fp32 until the codes.
//
// What bounds it: memory without modulation; with it, instruction issue and the three fp32
// rows per token from L1 (12 of the 19 bytes a value moves through it). Registers decide
// how many rows are in flight: rows of up to 8192 columns keep to 64 (two modulation
// levels 244 -> 228 us), and MODULATED = false leaves gate, scale and shift out, whose
// neutral values would cost 20 (235 -> 186 us). The row's factor to the last bit or so
// costs 4 us (187 -> 192) and keeps the share of values that round otherwise than in 64
// bits at that of the same formula in plain fp32.
template <typename T, int FMT, int CHUNKS, bool WARP_ROWS, bool ALIGNED, bool MODULATED>
__global__ void __launch_bounds__(CHUNKS == 8 ? 1024 : WARP_ROWS ? 128 : 512,
                                  WARP_ROWS ? (CHUNKS <= 2 ? 8 : 5) : CHUNKS <= 2 ? 2 : 1)
    mx_add_rmsnorm_kernel(MxNormDesc d, PackedRows p) {
  extern __shared__ __align__(16) float stages[];  // 256 per warp, unaligned rows only
  __shared__ float red[2][32];
  const int warp = warp_id(), lane = lane_id();
  const int warps = WARP_ROWS ? 1 : blockDim.x >> 5;  // of a row
  const int place = WARP_ROWS ? 0 : warp;
  const float g = FMT == kNvFp4 && d.g != nullptr ? *d.g : 1.f;
  const float six_g = 6.f * g, inv_six_g = __frcp_rn(six_g);
  const float width = static_cast<float>(d.W), inv_w = __frcp_rn(width);  // 1 / W = inv_w + inv_w_rest
  const float inv_w_rest = fmaf(-width, inv_w, 1.f) * inv_w;
  const int padded = static_cast<int>((d.rows + 127) / 128 * 128), rows = static_cast<int>(d.rows);
  const int step = WARP_ROWS ? gridDim.x * (blockDim.x >> 5) : gridDim.x;
  int row = WARP_ROWS ? blockIdx.x * (blockDim.x >> 5) + warp : blockIdx.x;
  const int base = place * kNormSpan, stride = warps * kNormSpan;  // of the warp's chunks

  int column[CHUNKS];  // of the lane's first value in each chunk, 0 past the end
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = base + i * stride + lane * kNormLane;
    column[i] = c < d.W ? c : 0;
  }
  Chunk<T, ALIGNED> rx[CHUNKS], ru[CHUNKS];
  int next_b = 0;
  auto request = [&](int at) {
    if (d.last_mod_row >= 0)
      next_b = d.groups != nullptr ? max(0, min(__ldg(d.groups + at), d.last_mod_row))
                                   : static_cast<int>(at / d.rows_per_batch);
    const NormRow<T, ALIGNED> x(reinterpret_cast<const T*>(d.x), at * d.ldx, 0.f);
    const NormRow<T, ALIGNED> u(reinterpret_cast<const T*>(d.update), at * d.ldu, 0.f);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      rx[i].load(x, base + i * stride, column[i], d.W);
      ru[i].load(u, base + i * stride, column[i], d.W);
    }
  };
  const NormRow<float, ALIGNED> weight(d.w, 0, 1.f);
  if (row < rows) request(row);
  int turn = 0;
  for (; row < rows; row += step) {
    __align__(16) float v[CHUNKS][kNormLane];
    const NormRow<float, ALIGNED> gate(d.gate, next_b * d.gate_stride, 1.f);
    const NormRow<float, ALIGNED> scale(d.scale, next_b * d.mod_stride, 0.f);
    const NormRow<float, ALIGNED> shift(d.shift, next_b * d.mod_stride, 0.f);
    T* x_out = reinterpret_cast<T*>(d.x_out) + static_cast<long>(row) * d.W;
    Pair ss(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      Chunk<float, ALIGNED> t;
      if constexpr (MODULATED) t.load(gate, base + i * stride, column[i], d.W);
      float u[kNormLane];
      rx[i].r.unpack(v[i]);
      ru[i].r.unpack(u);
      const bool past = ALIGNED && base + i * stride + lane * kNormLane >= d.W;
#pragma unroll
      for (int e = 0; e < kNormLane; e += 2) {
        Pair x2(v[i][e], v[i][e + 1]);
        const Pair u2(u[e], u[e + 1]);
        if constexpr (MODULATED) x2 = t.pair(e).times_plus(u2, x2);
        else x2 = x2 + u2;
        x2.get(v[i][e], v[i][e + 1]);
      }
      if (past) {
#pragma unroll
        for (int e = 0; e < kNormLane; ++e) v[i][e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < kNormLane; e += 2) {
        const Pair x2(v[i][e], v[i][e + 1]);
        ss = x2.times_plus(x2, ss);
      }
      if (d.x_out != nullptr) {
        rx[i].r.pack(v[i]);
        rx[i].store(x_out, base + i * stride, d.W);
      }
    }
    if (row + step < rows) request(row + step);
    float sum, other;
    ss.get(sum, other);
    sum += other;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, o);
    if constexpr (!WARP_ROWS) {
      if (lane == 0) red[turn][warp] = sum;
      __syncthreads();  // one per row: the next row's sums go to the other buffer
      constexpr int MOST = CHUNKS == 8 ? 32 : 16;  // warps; each run of as many lanes adds them up
      const int from = lane % MOST;
      sum = from < warps ? red[turn][from] : 0.f;
#pragma unroll
      for (int o = MOST / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(kAllLanes, sum, o);
      turn ^= 1;
    }
    const float r = inverse_root(fmaf(sum, inv_w, fmaf(sum, inv_w_rest, d.eps)));
    uint8_t* codes = p.codes_of(row);
    uint8_t* scales = p.scales_of(row);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int at = base + i * stride;
      Chunk<float, ALIGNED> w, sc, sh;
      w.load(weight, at, column[i], d.W);
      if constexpr (MODULATED) {
        sc.load(scale, at, column[i], d.W);
        sh.load(shift, at, column[i], d.W);
      }
      const Pair r2(r, r), one(1.f, 1.f);
#pragma unroll
      for (int e = 0; e < kNormLane; e += 2) {
        Pair y = Pair(v[i][e], v[i][e + 1]) * r2 * w.pair(e);
        if constexpr (MODULATED) y = y.times_plus(sc.pair(e) + one, sh.pair(e));
        y.get(v[i][e], v[i][e + 1]);
      }
      const int c0 = at + lane * kNormLane;
      if constexpr (!ALIGNED) {
        float* stage = stages + warp * kNormSpan;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < kNormLane; ++e) stage[32 * e + lane] = v[i][e];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < kNormLane; e += 4)
          *reinterpret_cast<float4*>(v[i] + e) = *reinterpret_cast<const float4*>(stage + lane * kNormLane + e);
        if (at + kNormSpan > d.W) {
#pragma unroll
          for (int e = 0; e < kNormLane; ++e) v[i][e] = c0 + e < d.W ? v[i][e] : 0.f;
        }
      } else if (c0 >= d.W) {  // 0 * (a statistic that overflowed) is not 0
#pragma unroll
        for (int e = 0; e < kNormLane; ++e) v[i][e] = 0.f;
      }
      store_packed<FMT>(LanePlace<FMT, kNormLane>(p, c0), codes, scales, v[i], amax_of(v[i]), g, six_g, inv_six_g);
    }
  }
  for (; row < padded; row += step)
    store_pad_scales(p, row, 0, p.tiles, WARP_ROWS ? lane : threadIdx.x, WARP_ROWS ? 32 : blockDim.x);
}

// ---------------------------------------------------------------- launches
bool aligned32(const void* ptr) { return reinterpret_cast<uintptr_t>(ptr) % 32 == 0; }
// Whether rows of `cols` values of `size` bytes, `ld` values apart, all start on 32 bytes
// and end on a lane's run of `lane` values.
bool rows_aligned(const void* ptr, long rows, long ld, long cols, int size, int lane) {
  return aligned32(ptr) && cols % lane == 0 && (rows <= 1 || ld * size % std::min(32, lane * size) == 0);
}

// Rows of a CTA: as many as leave four CTAs for every SM (fewer, larger CTAs keep the
// scale tiles' lines in one place), at least one per warp.
int rows_per_cta(long rows, long segments, int sms) {
  for (int r = 128; r > 8; r /= 2)
    if ((rows + r - 1) / r * segments >= 4L * sms) return r;
  return 8;
}

long segments_of(long cols) { return (cols + kSpan - 1) / kSpan; }

template <typename T, int FMT, bool ALIGNED>
void quantize_as(const MxQuantDesc& d, const PackedRows& p, cudaStream_t stream) {
  const long segments = segments_of(d.cols);
  AVGEN_CHECK(segments <= 65535, "quantize: too many columns: ", d.cols);
  if constexpr (FMT == kNvFp4) {
    if (d.g_out != nullptr && d.amax == nullptr) {
      cudaLaunchConfig_t cfg{};
      cfg.gridDim = dim3(static_cast<unsigned>((d.rows * segments + kSmallWarps - 1) / kSmallWarps));
      cfg.blockDim = dim3(32 * kSmallWarps);
      cfg.stream = stream;
      cudaLaunchAttribute attr{};
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = cfg.gridDim.x;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      auto kernel = mx_quantize_small_kernel<T, ALIGNED>;
      AVGEN_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, d, p, static_cast<int>(segments)));
      return;
    }
    if (d.amax != nullptr)
      mx_amax_kernel<T, ALIGNED>
          <<<dim3(static_cast<unsigned>(d.parts / segments), static_cast<unsigned>(segments)), 256, 0, stream>>>(d);
  }
  const long rows = (d.rows + 127) / 128 * 128;
  const int rpc = rows_per_cta(d.rows, segments, num_sms(d.device));
  mx_quantize_kernel<T, FMT, ALIGNED>
      <<<dim3(static_cast<unsigned>(rows / rpc), static_cast<unsigned>(segments)), 256, 0, stream>>>(d, p, rpc);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT>
void quantize(const MxQuantDesc& d, cudaStream_t stream) {
  const PackedRows p{d.codes, d.scales, mx_row_bytes(FMT, d.cols), mx_scale_tiles(FMT, d.cols), d.cols};
  if (rows_aligned(d.x, d.rows, d.ldx, d.cols, sizeof(T), kLane)) quantize_as<T, FMT, true>(d, p, stream);
  else quantize_as<T, FMT, false>(d, p, stream);
}

template <typename T, int FMT, bool ALIGNED>
void dequantize_as(const MxDequantDesc& d, const PackedRows& p, cudaStream_t stream) {
  const long segments = segments_of(d.cols);
  AVGEN_CHECK(segments <= 65535, "dequantize: too many columns: ", d.cols);
  const int rpc = rows_per_cta(d.rows, segments, num_sms(d.device));
  const dim3 grid(static_cast<unsigned>((d.rows + rpc - 1) / rpc), static_cast<unsigned>(segments));
  mx_dequantize_kernel<T, FMT, ALIGNED><<<grid, 256, 0, stream>>>(d, p, rpc);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT>
void dequantize(const MxDequantDesc& d, cudaStream_t stream) {
  const PackedRows p{const_cast<uint8_t*>(d.codes), const_cast<uint8_t*>(d.scales), mx_row_bytes(FMT, d.cols),
                     mx_scale_tiles(FMT, d.cols), d.cols};
  if (rows_aligned(d.out, d.rows, d.cols, d.cols, sizeof(T), kLane)) dequantize_as<T, FMT, true>(d, p, stream);
  else dequantize_as<T, FMT, false>(d, p, stream);
}

constexpr int kNormWarpsPerSm = 64;  // of a launch: the most rows one step of the norm's loop passes over, per SM

template <typename T, int FMT, int CHUNKS, bool WARP_ROWS, bool ALIGNED>
void add_rmsnorm_as(const MxNormDesc& d, const PackedRows& p, int warps, cudaStream_t stream) {
  auto kernel = d.gate != nullptr || d.scale != nullptr || d.shift != nullptr
                    ? mx_add_rmsnorm_kernel<T, FMT, CHUNKS, WARP_ROWS, ALIGNED, true>
                    : mx_add_rmsnorm_kernel<T, FMT, CHUNKS, WARP_ROWS, ALIGNED, false>;
  const long padded = (d.rows + 127) / 128 * 128;
  const long units = WARP_ROWS ? (padded + warps - 1) / warps : padded;
  const long ctas = static_cast<long>(std::max(1, kNormWarpsPerSm / warps)) * num_sms(d.device);
  const int smem = ALIGNED ? 0 : warps * kNormSpan * 4;  // at most 32 KB
  kernel<<<static_cast<unsigned>(std::min(units, ctas)), 32 * warps, smem, stream>>>(d, p);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

template <typename T, int FMT, bool ALIGNED>
void add_rmsnorm_aligned(const MxNormDesc& d, const PackedRows& p, cudaStream_t stream) {
  const int spans = static_cast<int>((d.W + kNormSpan - 1) / kNormSpan);
  if (spans == 1) return add_rmsnorm_as<T, FMT, 1, true, ALIGNED>(d, p, 4, stream);
  if (spans == 2) return add_rmsnorm_as<T, FMT, 2, true, ALIGNED>(d, p, 4, stream);
  if (spans == 3) return add_rmsnorm_as<T, FMT, 3, true, ALIGNED>(d, p, 4, stream);
  if (spans <= 32) return add_rmsnorm_as<T, FMT, 2, false, ALIGNED>(d, p, (spans + 1) / 2, stream);
  if (spans <= 64) return add_rmsnorm_as<T, FMT, 4, false, ALIGNED>(d, p, (spans + 3) / 4, stream);
  add_rmsnorm_as<T, FMT, 8, false, ALIGNED>(d, p, (spans + 7) / 8, stream);
}

template <typename T, int FMT>
void add_rmsnorm(const MxNormDesc& d, cudaStream_t stream) {
  AVGEN_CHECK(d.W <= kMxNormMaxCols, "add_rmsnorm: at most ", kMxNormMaxCols, " columns, got ", d.W);
  const PackedRows p{d.codes, d.scales, mx_row_bytes(FMT, d.W), mx_scale_tiles(FMT, d.W), d.W};
  auto mod = [&](const float* t, long stride) { return t == nullptr || (aligned32(t) && stride % 8 == 0); };
  auto rows = [&](const void* t, long ld) { return rows_aligned(t, d.rows, ld, d.W, sizeof(T), kNormLane); };
  const bool aligned = rows(d.x, d.ldx) && (d.update == nullptr || (rows(d.update, d.ldu) && rows(d.x_out, d.W))) &&
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

int mx_quantize_parts(const MxQuantDesc& d) {
  const long segments = segments_of(d.cols);
  if (d.rows * segments <= kSmallWarps * kSmallCtas) return 0;
  // CTAs of the measuring pass: up to eight for every SM, a row per warp at least
  const long blocks = std::min<long>((d.rows + 7) / 8, std::max<long>(1, 8L * num_sms(d.device) / segments));
  return static_cast<int>(blocks * segments);
}

// The norm counts rows in 32 signed bits; the last row of the last 128-row group plus one
// step has to stay within them.
long mx_norm_max_rows(int device) {
  return std::numeric_limits<int>::max() - 127L - static_cast<long>(kNormWarpsPerSm) * num_sms(device);
}

void mx_quantize_launch(const MxQuantDesc& d, cudaStream_t stream) { AVGEN_MX_DISPATCH(quantize, d, stream); }
void mx_dequantize_launch(const MxDequantDesc& d, cudaStream_t stream) { AVGEN_MX_DISPATCH(dequantize, d, stream); }
void mx_add_rmsnorm_launch(const MxNormDesc& d, cudaStream_t stream) { AVGEN_MX_DISPATCH(add_rmsnorm, d, stream); }

}  // namespace avgen
