// Block-scaled tcgen05 product for sm_100a.
//
//   D[M, N] = alpha * (A . B^T) (+ bias),  A [M, K], B [N, K] in mxfp8, mxfp4 or nvfp4
//
// The tensor cores multiply each block's products by both block scales while they
// accumulate in fp32 (kind::mxf8f6f4 / mxf4 / mxf4nvf4 with .block_scale), so the
// operands stay packed all the way; alpha = g_a * g_b is nvfp4's pair of tensor scales.
//
// Structure (one CTA per SM, persistent over output tiles):
//   warp 0      producer: per k-block (128 code bytes of each row) the A and B tiles
//               by TMA, their scale tiles by bulk copies, into a ring
//   warp 1      MMA issuer: copies a stage's scales to TMEM (tcgen05.cp), then issues
//               its products; the two kinds of instruction execute in issue order
//   warps 2..5  epilogue, one TMEM lane quadrant each
#include <algorithm>

#include "include/host_utils.h"
#include "include/launchers.h"
#include "include/microscale.cuh"
#include "include/sm100.cuh"

namespace avgen {
namespace {

struct MxArgs {
  int M, N, K;
  int row_bytes;  // of a row's codes
  int tiles_k;    // scale tiles along K
  const uint8_t* a_scales;
  const uint8_t* b_scales;
  const float* a_g;
  const float* b_g;
  const float* bias;
  void* out;
  int* err;
};

constexpr int kBM = 128;
constexpr int kRowBytes = 128;  // code bytes of a row in one k-block: one swizzle row
constexpr int kSteps = 4;       // products per k-block, 32 code bytes each

template <int FMT, int BN>
struct Cfg {
  static constexpr int SF_TILES = FMT == kNvFp4 ? 4 : FMT == kMxFp4 ? 2 : 1;  // scale tiles per k-block
  static constexpr int A_BYTES = kBM * kRowBytes;
  static constexpr int B_BYTES = BN * kRowBytes;
  static constexpr int SFA_BYTES = SF_TILES * 512;
  static constexpr int SFB_BYTES = BN / 128 * SF_TILES * 512;
  static constexpr int STAGE_BYTES = (A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES + 1023) / 1024 * 1024;
  static constexpr int STAGES = (232448 - 2048) / STAGE_BYTES;
  static constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + 1024 + 256;
  static constexpr int SF_COL = 2 * BN;  // TMEM columns of the scales, after both accumulators
  static constexpr int SFB_COL = SF_COL + SF_TILES * 4;
  static constexpr int TMEM_COLS = 512;
};

// Instruction descriptor of the block-scaled kinds: element types, scale type, shape.
// The positions of the scales inside a 32-bit TMEM cell (4, 29) vary by step.
template <int FMT>
constexpr uint32_t mx_idesc(int m, int n) {
  const uint32_t type = FMT == kMxFp8 ? 0u : 1u;    // e4m3 / e2m1
  const uint32_t scale = FMT == kNvFp4 ? 0u : 1u;   // e4m3 / e8m0
  return (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (scale << 23) |
         (static_cast<uint32_t>(m >> 7) << 27);
}

template <int FMT>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
#define AVGEN_MX_MMA(KIND)                                                                    \
  asm volatile(                                                                               \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                       \
      "tcgen05.mma.cta_group::1." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),     \
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                         \
      : "memory")
  if constexpr (FMT == kMxFp8) AVGEN_MX_MMA("kind::mxf8f6f4.block_scale.scale_vec::1X");
  if constexpr (FMT == kMxFp4) AVGEN_MX_MMA("kind::mxf4.block_scale.scale_vec::2X");
  if constexpr (FMT == kNvFp4) AVGEN_MX_MMA("kind::mxf4nvf4.block_scale.scale_vec::4X");
#undef AVGEN_MX_MMA
}

// One scale tile (512 bytes of shared memory: 32 rows of 16 bytes) to four TMEM
// columns, repeated in all four lane quadrants.
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint32_t smem_addr) {
  const uint64_t desc = static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 32) |
                        (1ull << 46);  // no swizzle, 8-row groups 128 bytes apart
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Bytes of 16-byte granularity from global to shared memory.
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
                   smem_u32(dst)),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ void drain_wait(uint64_t* bar, uint32_t parity) {
  const uint32_t a = smem_u32(bar);
  const uint64_t t0 = globaltimer();
  while (!mbar_try_wait(a, parity)) {
    if (globaltimer() - t0 > kWaitTimeoutNs) return;
  }
}

template <typename T, int FMT, int BN>
__global__ void __launch_bounds__(192, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB, const MxArgs args) {
  using C = Cfg<FMT, BN>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + C::STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = warp_id();
  const int lane = lane_id();
  const int num_m = (args.M + kBM - 1) / kBM;
  const int num_n = (args.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int num_kb = (args.row_bytes + kRowBytes - 1) / kRowBytes;
  const int last_steps = (args.row_bytes - (num_kb - 1) * kRowBytes + 31) / 32;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], 128);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, C::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 0;
      bool aborted = false;
      for (int t = blockIdx.x; t < num_tiles && !aborted; t += gridDim.x) {
        const int tm = t % num_m, tn = t / num_m;
        const int b_groups = min(BN, args.N - tn * BN + 127) / 128;  // 128-row scale groups this tile has
        for (int kb = 0; kb < num_kb; ++kb) {
          if (!mbar_wait(&empty[stage], phase ^ 1, abort_flag, args.err, kErrTimeoutProducer)) {
            aborted = true;
            break;
          }
          uint8_t* sa = smem + stage * C::STAGE_BYTES;
          uint8_t* sb = sa + C::A_BYTES;
          uint8_t* sfa = sb + C::B_BYTES;
          uint8_t* sfb = sfa + C::SFA_BYTES;
          const int tile0 = kb * C::SF_TILES;
          const uint32_t sf_bytes = static_cast<uint32_t>(min(C::SF_TILES, args.tiles_k - tile0)) * 512u;
          mbar_arrive_expect_tx(&full[stage], C::A_BYTES + C::B_BYTES + sf_bytes * (1 + b_groups));
          tma_load_2d(sa, &tmA, &full[stage], kb * kRowBytes, tm * kBM);
          tma_load_2d(sb, &tmB, &full[stage], kb * kRowBytes, tn * BN);
          bulk_load(sfa, args.a_scales + (static_cast<long>(tm) * args.tiles_k + tile0) * 512, sf_bytes, &full[stage]);
          for (int j = 0; j < b_groups; ++j)
            bulk_load(sfb + j * C::SFA_BYTES,
                      args.b_scales + (static_cast<long>(tn * (BN / 128) + j) * args.tiles_k + tile0) * 512, sf_bytes,
                      &full[stage]);
          ++issued;
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
      }
      if (aborted) {  // copies in flight land before the CTA's shared memory goes away
        for (int i = 0; i < min(issued, C::STAGES); ++i) {
          if (--stage < 0) {
            stage = C::STAGES - 1;
            phase ^= 1;
          }
          drain_wait(&full[stage], phase);
        }
      }
    }
  } else if (warp == 1) {
    constexpr uint32_t idesc = mx_idesc<FMT>(kBM, BN);
    int stage = 0, acc = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool aborted = false;
    for (int t = blockIdx.x; t < num_tiles && !aborted; t += gridDim.x) {
      if (!mbar_wait(&tempty[acc], acc_phase ^ 1, abort_flag, args.err, kErrTimeoutMma)) break;
      tc_fence_after();
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(&full[stage], phase, abort_flag, args.err, kErrTimeoutMma)) {
          aborted = true;
          break;
        }
        tc_fence_after();
        if (elect_one()) {
          const uint32_t sa = smem_u32(smem + stage * C::STAGE_BYTES);
          const uint32_t sb = sa + C::A_BYTES;
          const uint32_t sfa = sb + C::B_BYTES;
          const uint32_t sfb = sfa + C::SFA_BYTES;
#pragma unroll
          for (int i = 0; i < C::SF_TILES; ++i) {
            copy_scales(tmem + C::SF_COL + 4 * i, sfa + 512 * i);
#pragma unroll
            for (int j = 0; j < BN / 128; ++j)
              copy_scales(tmem + C::SFB_COL + (i * (BN / 128) + j) * 4, sfb + j * C::SFA_BYTES + 512 * i);
          }
          const int steps = kb == num_kb - 1 ? last_steps : kSteps;
#pragma unroll
          for (int k = 0; k < kSteps; ++k) {
            if (k < steps) {
              constexpr int PER = kSteps / C::SF_TILES;                        // steps per scale tile
              const uint32_t id = static_cast<uint32_t>(k % PER * (4 / PER));  // byte of the first scale
              const int i = k / PER;
              mx_mma<FMT>(tmem + acc * BN, umma_desc_sw128(sa + 32 * k, 16, 1024), umma_desc_sw128(sb + 32 * k, 16, 1024),
                          idesc | (id << 4) | (id << 29), tmem + C::SF_COL + 4 * i,
                          tmem + C::SFB_COL + i * (BN / 128) * 4, (kb > 0 || k > 0) ? 1u : 0u);
            }
          }
          mma_commit(&empty[stage]);
        }
        __syncwarp();
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
      if (aborted) break;
      if (elect_one()) mma_commit(&tfull[acc]);
      __syncwarp();
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  } else {
    const int q = warp & 3;
    int acc = 0;
    uint32_t acc_phase = 0;
    const float alpha = (args.a_g != nullptr ? *args.a_g : 1.f) * (args.b_g != nullptr ? *args.b_g : 1.f);
    for (int t = blockIdx.x; t < num_tiles; t += gridDim.x) {
      const int tm = t % num_m, tn = t / num_m;
      if (!mbar_wait(&tfull[acc], acc_phase, abort_flag, args.err, kErrTimeoutEpilogue)) break;
      tc_fence_after();
      const int row = tm * kBM + q * 32 + lane;
      T* out = reinterpret_cast<T*>(args.out) + static_cast<long>(row) * args.N;
      for (int c = 0; c < BN / 32; ++c) {
        uint32_t r[32];
        tmem_ld32(tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * BN + 32 * c, r);
        tmem_wait_ld();
        if (row < args.M) {
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int n = tn * BN + 32 * c + i;
            if (n < args.N)
              out[n] = from_float<T>(fmaf(__uint_as_float(r[i]), alpha, args.bias != nullptr ? args.bias[n] : 0.f));
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty[acc]);
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1;
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, C::TMEM_COLS);
  }
}

// Codes as a byte matrix [rows, row_bytes], boxes of `box_rows` x 128 bytes.
CUtensorMap make_codes_map(const void* ptr, long row_bytes, long rows, int box_rows) {
  CUtensorMap map;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  const cuuint32_t box[2] = {kRowBytes, static_cast<cuuint32_t>(box_rows)};
  const cuuint32_t estr[2] = {1, 1};
  const CUresult r = tensor_map_encoder()(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides,
                                          box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AVGEN_CHECK(r == CUDA_SUCCESS, "mx_gemm: cuTensorMapEncodeTiled failed (", static_cast<int>(r), ")");
  return map;
}

template <typename T, int FMT>
void launch(const MxGemmDesc& d, cudaStream_t stream) {
  constexpr int BN = 128;
  using C = Cfg<FMT, BN>;
  MxArgs args{};
  args.M = d.M, args.N = d.N, args.K = d.K;
  args.row_bytes = static_cast<int>(mx_row_bytes(FMT, d.K));
  args.tiles_k = static_cast<int>(mx_scale_tiles(FMT, d.K));
  args.a_scales = d.a_scales, args.b_scales = d.b_scales;
  args.a_g = d.a_g, args.b_g = d.b_g;
  args.bias = d.bias, args.out = d.out, args.err = d.err;
  const CUtensorMap ta = make_codes_map(d.a_codes, args.row_bytes, d.M, kBM);
  const CUtensorMap tb = make_codes_map(d.b_codes, args.row_bytes, d.N, BN);
  auto kernel = mx_gemm_kernel<T, FMT, BN>;
  static PerDeviceOnce once;
  raise_smem_limit(once, kernel, C::SMEM_BYTES);
  const int tiles = (d.M + kBM - 1) / kBM * ((d.N + BN - 1) / BN);
  kernel<<<std::min(tiles, num_sms(d.device)), 192, C::SMEM_BYTES, stream>>>(ta, tb, args);
  AVGEN_CUDA_CHECK(cudaGetLastError());
}

}  // namespace

void mx_gemm_launch(const MxGemmDesc& d, cudaStream_t stream) {
  AVGEN_CHECK(d.M > 0 && d.N > 0 && d.K > 0, "mx_gemm: empty problem");
#define AVGEN_MX_CASE(TYPE, T, FMT) \
  if (d.dtype == TYPE && d.fmt == FMT) return launch<T, FMT>(d, stream);
  AVGEN_MX_CASE(kMxBf16, __nv_bfloat16, kMxFp8)
  AVGEN_MX_CASE(kMxBf16, __nv_bfloat16, kMxFp4)
  AVGEN_MX_CASE(kMxBf16, __nv_bfloat16, kNvFp4)
  AVGEN_MX_CASE(kMxFp16, __half, kMxFp8)
  AVGEN_MX_CASE(kMxFp16, __half, kMxFp4)
  AVGEN_MX_CASE(kMxFp16, __half, kNvFp4)
  AVGEN_MX_CASE(kMxFp32, float, kMxFp8)
  AVGEN_MX_CASE(kMxFp32, float, kMxFp4)
  AVGEN_MX_CASE(kMxFp32, float, kNvFp4)
#undef AVGEN_MX_CASE
  AVGEN_CHECK(false, "mx_gemm: unsupported type ", d.dtype, " or format ", d.fmt);
}

}  // namespace avgen
