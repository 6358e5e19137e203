// Block-scaled tcgen05 product for sm_100a.
//
//   D[M, N] = (A . B^T) * g_a * g_b (+ bias),  A [M, K], B [N, K] in mxfp8, mxfp4 or nvfp4
//
// The tensor cores multiply each block's products by both block scales while they
// accumulate in fp32 (kind::mxf8f6f4 / mxf4 / mxf4nvf4 with .block_scale), so the
// operands stay packed all the way; g_a and g_b are nvfp4's tensor scales, else 1.
//
// Structure (persistent over output tiles; CTAS = 2 pairs the two SMs of a TPC on one
// 256 x 256 tile, CTAS = 1 gives each SM a 128 x 128 tile):
//   warp 0      producer: per k-block (128 code bytes of each row) this CTA's A and B
//               rows and the scale tiles by TMA into a ring
//   warp 1      MMA issuer (the pair's first CTA): copies a stage's scales to TMEM
//               (tcgen05.cp), then issues its products; both kinds of instruction
//               execute in issue order
//   warps 2..9  epilogue, two per TMEM lane quadrant (32 rows), half the columns each:
//               TMEM -> registers -> shared memory -> TMA store, 128 bytes of a row at a time
// Outputs too small to fill the SMs with such tiles take the split form below it: a
// cluster of CTAs shares one tile, each with a part of K, and adds up over distributed
// shared memory in rank order, so results repeat bitwise.
//
// In a pair each CTA stages its own 128 rows of A and half of B's 256 rows: the same
// operand bytes from L2 and shared memory per product as one SM would need for half
// the work.
//
// What bounds it, as far as it was taken apart (mxfp8, 40 k-blocks): an SM takes in about 52
// bytes a clock through TMA here, so a k-block of 34 to 38 KB takes some 650 clocks, against
// 512 for its products; with both at once it measured 750 to 780 whatever the ring's depth
// beyond four stages. Short K adds the store of the output (19 % at K = 2560 in nvfp4, ten
// k-blocks, where the roles' waits were not measured). Times on a B200 at its 1 kW power limit:
//   65536 x 20480 x 2560 nvfp4   1.75 to 1.84 ms, 3.9 to 3.7 PFLOP/s (4.7 before the limit sets in)
//   16384 x 2560 x 10240 mxfp4   165 to 172 us, 5.2 to 5.0 PFLOP/s (6.1)
//   32768 x 5120 x 5120 mxfp8    686 to 731 us, 2.5 to 2.4 PFLOP/s (2.9)
#include <algorithm>
#include <cfloat>

#include "include/host_utils.h"
#include "include/launchers.h"
#include "include/microscale.cuh"
#include "include/sm100.cuh"

namespace avgen {
namespace {

struct MxArgs {
  int M, N;
  int num_kb;      // k-blocks
  int last_steps;  // products in the last one
  const float* a_g;
  const float* b_g;
  const float* bias;
  void* out;
  int* err;
};

constexpr int kBM = 128;        // rows of A per CTA
constexpr int kRowBytes = 128;  // code bytes of a row in one k-block: one swizzle row
constexpr int kSteps = 4;       // products per k-block, 32 code bytes each
constexpr int kBoxBytes = 32 * 128;  // one warp's store: 32 rows x 128 bytes
constexpr int kSmemLimit = 232448;
// Two epilogue warps per quadrant: with one, a 256 x 256 tile took 4.6 us to store, longer
// than the products of K = 2560 in 4 bits.
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;

// One staged k-block and the TMEM columns of its scales.
template <int FMT, int BN, int CTAS>
struct StageCfg {
  static constexpr int SF_TILES = FMT == kNvFp4 ? 4 : FMT == kMxFp4 ? 2 : 1;  // scale tiles per k-block
  static constexpr int B_ROWS = BN / CTAS;
  static constexpr int A_BYTES = kBM * kRowBytes;
  static constexpr int B_BYTES = B_ROWS * kRowBytes;
  static constexpr int SFA_BYTES = SF_TILES * 512;
  static constexpr int SFB_GROUPS = (BN + 127) / 128;
  static constexpr int SFB_BYTES = SFB_GROUPS * SFA_BYTES;  // of all BN rows, in both CTAs
  static constexpr int TX_BYTES = A_BYTES + B_BYTES + SFA_BYTES + SFB_BYTES;
  static constexpr int STAGE_BYTES = (TX_BYTES + 1023) / 1024 * 1024;
  static constexpr int SF_COLS = (SF_TILES * 4 * (1 + SFB_GROUPS) + 31) / 32 * 32;
};

template <int FMT, int BN, int CTAS>
struct Cfg : StageCfg<FMT, BN, CTAS> {
  using S = StageCfg<FMT, BN, CTAS>;
  static constexpr int OUT_BYTES = kEpiWarps * kBoxBytes;
  static constexpr int STAGES = std::min(8, (kSmemLimit - 2048 - OUT_BYTES) / S::STAGE_BYTES);
  static constexpr int SMEM_BYTES = STAGES * S::STAGE_BYTES + OUT_BYTES + 1024 + 256;
  // TMEM: two accumulators and the scales of one k-block. Two 256-column accumulators
  // leave no room for scales, so the second starts inside the first: the epilogue reads
  // the shared columns first and hands them over, and the next tile's products wait for
  // that instead of for a free accumulator.
  static constexpr bool OVERLAP = 2 * BN + S::SF_COLS > 512;
  static constexpr int ACC1 = OVERLAP ? 512 - S::SF_COLS - BN : BN;
  static constexpr int SF_COL = ACC1 + BN;
};

// Instruction descriptor of the block-scaled kinds: element types, scale type, shape.
// The positions of the scales inside a 32-bit TMEM cell (bits 4 and 29) vary by step.
template <int FMT>
constexpr uint32_t mx_idesc(int m, int n) {
  const uint32_t type = FMT == kMxFp8 ? 0u : 1u;   // e4m3 / e2m1
  const uint32_t scale = FMT == kNvFp4 ? 0u : 1u;  // e4m3 / e8m0
  return (type << 7) | (type << 10) | (static_cast<uint32_t>(n >> 3) << 17) | (scale << 23) |
         (static_cast<uint32_t>(m >> 7) << 27);
}

template <int FMT, int CTAS>
__device__ __forceinline__ void mx_mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                       uint32_t accumulate) {
#define AVGEN_MX_MMA(CG, KIND)                                                            \
  asm volatile(                                                                           \
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %6, 0;\n\t"                                   \
      "tcgen05.mma.cta_group::" CG "." KIND " [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d), \
      "l"(a), "l"(b), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                     \
      : "memory")
  if constexpr (CTAS == 1) {
    if constexpr (FMT == kMxFp8) AVGEN_MX_MMA("1", "kind::mxf8f6f4.block_scale.scale_vec::1X");
    if constexpr (FMT == kMxFp4) AVGEN_MX_MMA("1", "kind::mxf4.block_scale.scale_vec::2X");
    if constexpr (FMT == kNvFp4) AVGEN_MX_MMA("1", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  } else {
    if constexpr (FMT == kMxFp8) AVGEN_MX_MMA("2", "kind::mxf8f6f4.block_scale.scale_vec::1X");
    if constexpr (FMT == kMxFp4) AVGEN_MX_MMA("2", "kind::mxf4.block_scale.scale_vec::2X");
    if constexpr (FMT == kNvFp4) AVGEN_MX_MMA("2", "kind::mxf4nvf4.block_scale.scale_vec::4X");
  }
#undef AVGEN_MX_MMA
}

// A scale tile in shared memory: 32 rows of 16 bytes, no swizzle, 8-row groups 128 bytes apart.
__device__ __forceinline__ uint64_t scale_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr >> 4) & 0x3FFFu) | (static_cast<uint64_t>(128 >> 4) << 32) | (1ull << 46);
}
// One scale tile to four TMEM columns, repeated in all four lane quadrants; in a pair, in
// each CTA from its own shared memory.
template <int CTAS>
__device__ __forceinline__ void copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (CTAS == 1)
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// Descriptors of stage 0 and the tensor-memory places, from which a stage's follow by one
// addition (addresses are below 2^18 bytes, so the 14-bit field does not carry).
template <int FMT, int BN, int CTAS>
struct Issuer {
  using C = StageCfg<FMT, BN, CTAS>;
  static constexpr int SFB_TILES = C::SFB_GROUPS;
  static constexpr int PER = kSteps / C::SF_TILES;  // products per scale tile
  uint64_t a, b, sfa, sfb;
  uint32_t t_sfa, t_sfb;

  // `sf`: TMEM address of the scales.
  __device__ __forceinline__ Issuer(uint32_t smem_addr, uint32_t sf) {
    a = umma_desc_sw128(smem_addr, 16, 1024);
    b = umma_desc_sw128(smem_addr + C::A_BYTES, 16, 1024);
    sfa = scale_desc(smem_addr + C::A_BYTES + C::B_BYTES);
    sfb = scale_desc(smem_addr + C::A_BYTES + C::B_BYTES + C::SFA_BYTES);
    t_sfa = sf;
    t_sfb = sf + C::SF_TILES * 4;
  }
  // The scales and products of one staged k-block.
  __device__ __forceinline__ void block(int stage, uint32_t tmem_acc, uint32_t idesc, int steps, bool first) const {
    const uint32_t at = static_cast<uint32_t>(stage) * (C::STAGE_BYTES / 16);
#pragma unroll
    for (int i = 0; i < C::SF_TILES; ++i) {
      copy_scales<CTAS>(t_sfa + 4 * i, sfa + at + 32 * i);
#pragma unroll
      for (int j = 0; j < SFB_TILES; ++j)
        copy_scales<CTAS>(t_sfb + (i * SFB_TILES + j) * 4, sfb + at + j * (C::SFA_BYTES / 16) + 32 * i);
    }
#pragma unroll
    for (int k = 0; k < kSteps; ++k) {
      if (k < steps) {
        const uint32_t id = static_cast<uint32_t>(k % PER * (4 / PER));  // the step's first scale in its 4-byte cell
        mx_mma<FMT, CTAS>(tmem_acc, a + at + 2 * k, b + at + 2 * k, idesc | (id << 4) | (id << 29),
                          t_sfa + 4 * (k / PER), t_sfb + (k / PER) * SFB_TILES * 4, (!first || k > 0) ? 1u : 0u);
      }
    }
  }
};

// ---------------------------------------------------------------- pair plumbing
// The warp's number as a value the compiler knows to be uniform.
__device__ __forceinline__ int uniform_warp_id() { return __shfl_sync(0xffffffffu, warp_id(), 0); }

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}

// TMA loads whose completion is counted at `bar`, a shared::cluster address (in a pair:
// of the first CTA).
template <int CTAS>
__device__ __forceinline__ void load_2d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  if constexpr (CTAS == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void load_3d(void* dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  if constexpr (CTAS == 1)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::
            "r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, "
        "%5}], [%2];" ::"r"(smem_u32(dst)),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}
__device__ __forceinline__ void store_2d(const CUtensorMap* map, const void* src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(x), "r"(y)
               : "memory");
}

// Arrive at `bar` (in a pair: at this offset in both CTAs) when every tcgen05 operation
// this thread issued so far is done.
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if constexpr (CTAS == 1)
    mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
}
template <int CTAS>
__device__ __forceinline__ void alloc_tmem(uint32_t* slot) {
  if constexpr (CTAS == 1) {
    tmem_alloc(slot, 512);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(slot)));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CTAS>
__device__ __forceinline__ void free_tmem(uint32_t taddr) {
  if constexpr (CTAS == 1)
    tmem_dealloc(taddr, 512);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, 512;" ::"r"(taddr));
}

// mbar_wait with one answer for the whole warp.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* err,
                                          int code) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, err, code));
}

// nvfp4's two tensor scales as factors that a sum takes one after the other. Their product
// alone may leave fp32's range where the result does not (sums reach 2688^2 * K): then the
// larger one goes first if it is too small, the smaller one if it is too large.
struct TensorScales {
  float first, last;

  __device__ __forceinline__ explicit TensorScales(const MxArgs& args) {
    const float a = args.a_g != nullptr ? *args.a_g : 1.f, b = args.b_g != nullptr ? *args.b_g : 1.f;
    const float both = a * b;
    const bool swap = (fabsf(both) < 1.f) != (fabsf(a) > fabsf(b));
    first = swap ? b : a;
    last = swap ? a : b;
    if (fabsf(both) >= FLT_MIN && fabsf(both) <= FLT_MAX) first = 1.f, last = both;
  }
  __device__ __forceinline__ float operator()(float sum) const { return sum * first * last; }
  __device__ __forceinline__ float operator()(float sum, float bias) const { return fmaf(sum * first, last, bias); }
};

// After an abort: copies still in flight land well within a millisecond.
__device__ __forceinline__ void let_copies_land() {
  const uint64_t t0 = globaltimer();
  while (globaltimer() - t0 < 1000000ull) __nanosleep(1000);
}

// Grouped raster: 8 row tiles share each sweep over the columns, so that the tiles in
// flight together re-read few operand rows from L2.
__device__ __forceinline__ void tile_at(int t, int num_m, int num_n, int& tm, int& tn) {
  constexpr int G = 8;
  const int group = t / (G * num_n);
  const int rows = min(G, num_m - group * G);
  const int r = t - group * G * num_n;
  tm = group * G + r % rows;
  tn = r / rows;
}

// Stages one row's 128 bytes (64 16-bit or 32 fp32 values) of a 32-row store box in
// the 128-byte swizzle: 16-byte chunk j of row r at chunk j ^ (r % 8).
template <typename T>
__device__ __forceinline__ void stage_row(uint8_t* box, int lane, const float* v) {
  uint4* row = reinterpret_cast<uint4*>(box + lane * 128);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    uint4 w;
    if constexpr (sizeof(T) == 2) {
      w = make_uint4(pack2<T>(v[8 * j], v[8 * j + 1]), pack2<T>(v[8 * j + 2], v[8 * j + 3]),
                     pack2<T>(v[8 * j + 4], v[8 * j + 5]), pack2<T>(v[8 * j + 6], v[8 * j + 7]));
    } else {
      w = make_uint4(__float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]), __float_as_uint(v[4 * j + 2]),
                     __float_as_uint(v[4 * j + 3]));
    }
    row[j ^ (lane & 7)] = w;
  }
}

// A staged box to rows of no 16-byte pitch: a word of the row per lane, eight rows in flight.
template <typename T>
__device__ __forceinline__ void store_box_words(const MxArgs& args, const uint8_t* box, int lane, int row0, int col) {
  constexpr int WORD = 4 / static_cast<int>(sizeof(T));  // values of a word
  const int c = col + lane * WORD;
  const bool first = c < args.N, second = c + 1 < args.N, words = WORD == 1 || args.N % 2 == 0;
  T* out = reinterpret_cast<T*>(args.out) + static_cast<long>(row0) * args.N + c;
  for (int r0 = 0; r0 < min(32, args.M - row0); r0 += 8) {
    uint32_t w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
      w[i] = *reinterpret_cast<const uint32_t*>(box + (r0 + i) * 128 + ((lane / 4) ^ i) * 16 + lane % 4 * 4);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (row0 + r0 + i < args.M) {
        if (words) {
          if (first) *reinterpret_cast<uint32_t*>(out) = w[i];
        } else {
          if (first) reinterpret_cast<uint16_t*>(out)[0] = static_cast<uint16_t>(w[i]);
          if (second) reinterpret_cast<uint16_t*>(out)[1] = static_cast<uint16_t>(w[i] >> 16);
        }
      }
      out += args.N;
    }
  }
}

template <typename T, int FMT, int BN, int CTAS>
__global__ void __launch_bounds__(kThreads, 1)
    mx_gemm_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmB,
                   const __grid_constant__ CUtensorMap tmSFA, const __grid_constant__ CUtensorMap tmSFB,
                   const __grid_constant__ CUtensorMap tmOut, const bool tma_out, const MxArgs args) {
  using C = Cfg<FMT, BN, CTAS>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (1024u - smem_u32(smem_raw) % 1024u) % 1024u;
  uint8_t* smem_out = smem + C::STAGES * C::STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem_out + C::OUT_BYTES);
  uint64_t* empty = full + C::STAGES;
  uint64_t* tfull = empty + C::STAGES;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform_warp_id();
  const int lane = lane_id();
  const int rank = CTAS == 2 ? static_cast<int>(cluster_rank()) : 0;
  const int num_m = (args.M + CTAS * kBM - 1) / (CTAS * kBM);
  const int num_n = (args.N + BN - 1) / BN;
  const int num_tiles = num_m * num_n;
  const int first = blockIdx.x / CTAS, step = gridDim.x / CTAS;

  if (threadIdx.x == 0) {
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&tfull[b], 1);
      mbar_init(&tempty[b], kEpiWarps * CTAS);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    prefetch_tmap(&tmA);
    prefetch_tmap(&tmB);
    prefetch_tmap(&tmSFA);
    prefetch_tmap(&tmSFB);
    if (tma_out) prefetch_tmap(&tmOut);
  }
  if (warp == 1) alloc_tmem<CTAS>(tmem_slot);
  tc_fence_before();
  if constexpr (CTAS == 2) cluster_sync();
  else __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // Both issuing roles run warp-uniform with one elected thread: from a divergent branch
  // each TMA or tcgen05 instruction takes several times as long to issue (mxfp8 16384 x
  // 5120 x 5120: products issued by `if (lane == 0)` ran at 2.2 instead of 2.8 PFLOP/s).
  // A wait that runs out may do so for some lanes only, so no lane leaves its loop early:
  // an aborted one goes on without waiting or issuing.
  if (warp == 0) {
    int stage = 0;
    uint32_t phase = 0;
    bool aborted = false;
    const uint32_t bar0 = CTAS == 2 ? map_to_rank(smem_u32(full), 0) : smem_u32(full);
    for (int t = first; t < num_tiles; t += step) {
      int tm, tn;
      tile_at(t, num_m, num_n, tm, tn);
      for (int kb = 0; kb < args.num_kb; ++kb) {
        if (!aborted) aborted = !mbar_wait(&empty[stage], phase ^ 1, abort_flag, args.err, kErrTimeoutProducer);
        if (elect_one() && !aborted) {
          uint8_t* sa = smem + stage * C::STAGE_BYTES;
          uint8_t* sb = sa + C::A_BYTES;
          uint8_t* sfa = sb + C::B_BYTES;
          uint8_t* sfb = sfa + C::SFA_BYTES;
          if (rank == 0) mbar_arrive_expect_tx(&full[stage], CTAS * C::TX_BYTES);
          const uint32_t bar = bar0 + stage * 8;
          load_2d<CTAS>(sa, &tmA, bar, kb * kRowBytes, (tm * CTAS + rank) * kBM);
          load_2d<CTAS>(sb, &tmB, bar, kb * kRowBytes, tn * BN + rank * C::B_ROWS);
          load_3d<CTAS>(sfa, &tmSFA, bar, 0, kb * C::SF_TILES, tm * CTAS + rank);
          load_3d<CTAS>(sfb, &tmSFB, bar, 0, kb * C::SF_TILES, tn * (BN / 128));
        }
        __syncwarp();
        if (++stage == C::STAGES) {
          stage = 0;
          phase ^= 1;
        }
      }
    }
    if (aborted) let_copies_land();
  } else if (warp == 1) {
    if (rank == 0) {
      constexpr uint32_t idesc = mx_idesc<FMT>(CTAS * kBM, BN);
      const Issuer<FMT, BN, CTAS> issue(smem_u32(smem), tmem + C::SF_COL);
      int stage = 0;
      uint32_t phase = 0;
      bool aborted = false;
      int i = 0;  // tiles done by this CTA
      for (int t = first; t < num_tiles; t += step, ++i) {
        const int acc = i & 1;
        // the tile that must have been read (its shared columns, or all of it) before this one
        const int before = C::OVERLAP ? i - 1 : i - 2;
        if (before >= 0 && !aborted)
          aborted = !mbar_wait(&tempty[before & 1], (before >> 1) & 1, abort_flag, args.err, kErrTimeoutMma);
        tc_fence_after();
        for (int kb = 0; kb < args.num_kb; ++kb) {
          if (!aborted) aborted = !mbar_wait(&full[stage], phase, abort_flag, args.err, kErrTimeoutMma);
          tc_fence_after();
          if (elect_one() && !aborted) {
            issue.block(stage, tmem + acc * C::ACC1, idesc, kb == args.num_kb - 1 ? args.last_steps : kSteps, kb == 0);
            commit<CTAS>(&empty[stage]);
          }
          __syncwarp();
          if (++stage == C::STAGES) {
            stage = 0;
            phase ^= 1;
          }
        }
        if (elect_one() && !aborted) commit<CTAS>(&tfull[acc]);
        __syncwarp();
      }
    }
  } else {
    constexpr int GROUPS = BN / 64 / 2;                     // groups of 64 columns of this warp's half
    constexpr int BOX = 128 / static_cast<int>(sizeof(T));  // columns of a store box
    const int q = warp & 3, half = (warp - 2) >> 2;
    uint8_t* box = smem_out + (warp - 2) * kBoxBytes;
    const TensorScales scaled(args);
    uint32_t release[2];
    for (int b = 0; b < 2; ++b)
      release[b] = CTAS == 2 ? map_to_rank(smem_u32(&tempty[b]), 0) : smem_u32(&tempty[b]);
    int i = 0;
    for (int t = first; t < num_tiles; t += step, ++i) {
      int tm, tn;
      tile_at(t, num_m, num_n, tm, tn);
      const int acc = i & 1;
      if (!warp_wait(&tfull[acc], (i >> 1) & 1, abort_flag, args.err, kErrTimeoutEpilogue)) break;
      tc_fence_after();
      // What this warp has to have read before the next tile's products may start: with
      // overlapping accumulators the shared columns (the first one's last, the second one's
      // first group) if they are in its half, else nothing of this tile (its arrival says
      // that it is done with the tile before); without overlap all of its half.
      const bool holds_shared = C::OVERLAP && half == 1 - acc;
      if (C::OVERLAP && !holds_shared) {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) arrive_at(release[acc]);
      }
      const int row0 = (tm * CTAS + rank) * kBM + q * 32;
#pragma unroll
      for (int step_g = 0; step_g < GROUPS; ++step_g) {
        const int g = half * GROUPS + (C::OVERLAP && acc == 0 ? GROUPS - 1 - step_g : step_g);  // shared columns first
        uint32_t r[2][32];
        const uint32_t taddr = tmem + (static_cast<uint32_t>(q * 32) << 16) + acc * C::ACC1 + 64 * g;
        tmem_ld32(taddr, r[0]);
        tmem_ld32(taddr + 32, r[1]);
        tmem_wait_ld();
        static_assert(!C::OVERLAP || BN - C::ACC1 <= 64, "shared columns lie in one group");
        if (C::OVERLAP ? holds_shared && step_g == 0 : step_g == GROUPS - 1) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) arrive_at(release[acc]);
        }
        const int col0 = tn * BN + 64 * g;
        if (row0 >= args.M || col0 >= args.N) continue;
        float v[64];
#pragma unroll
        for (int j = 0; j < 64; ++j) v[j] = scaled(__uint_as_float(r[j / 32][j % 32]));
        if (args.bias != nullptr) {
#pragma unroll
          for (int j = 0; j < 64; ++j) v[j] += col0 + j < args.N ? __ldg(args.bias + col0 + j) : 0.f;
        }
#pragma unroll
        for (int h = 0; h < 64 / BOX; ++h) {
          const int col = col0 + BOX * h;
          if (lane == 0) bulk_wait_group_read0();
          __syncwarp();
          stage_row<T>(box, lane, v + BOX * h);
          if (tma_out) {
            fence_proxy_async();
            __syncwarp();
            if (lane == 0 && col < args.N) {
              store_2d(&tmOut, box, col, row0);
              bulk_commit_group();
            }
          } else {
            __syncwarp();
            store_box_words<T>(args, box, lane, row0, col);
          }
        }
      }
    }
    if (lane == 0) bulk_wait_group_read0();
  }

  tc_fence_before();
  if constexpr (CTAS == 2) cluster_sync();
  else __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    free_tmem<CTAS>(tmem);
  }
}

// ---------------------------------------------------------------- few rows
// out[m, n] of 128 weight rows (B's, which take the tensor core's 128 lanes) by MT rows
// of A, over a part of K per CTA of the cluster. What bounds it is the time to stream the
// weights, so a CTA's whole part is requested at once as far as shared memory goes; a
// launch that does next to nothing takes 3.6 us here. Measured, in a graph, weights from
// memory: 1 x 15360 x 2560 nvfp4 7.5 us (2.9 TB/s; 5.9 where L2 holds them), 32 x 20480 x 2560
// mxfp8 13 us (4.1 TB/s; 9.3).
constexpr int kMaxSplits = 8;  // CTAs of a portable cluster

// The 32-row form's ring leaves room for two CTAs on an SM, which share one where there are more
// tiles than SMs (above 148 x 128 outputs); with fewer, half of the shared memory stays unused.
template <int FMT, int MT>
struct SplitCfg {
  using C = StageCfg<FMT, MT, 1>;
  static constexpr int CTAS_PER_SM = MT <= 32 ? 2 : 1;
  static constexpr int STAGES = std::min(8, (kSmemLimit / CTAS_PER_SM - 2048) / C::STAGE_BYTES);
  static constexpr int SMEM_BYTES = STAGES * C::STAGE_BYTES + 1024 + 256;
  static constexpr int TMEM_COLS = MT + C::SF_COLS <= 64 ? 64 : MT + C::SF_COLS <= 128 ? 128 : 256;
  static_assert(MT * 128 * 4 <= STAGES * C::STAGE_BYTES, "the partial sums reuse the ring");
};

template <typename T, int FMT, int MT>
__global__ void __launch_bounds__(192, 1)
    mx_gemm_split_kernel(const __grid_constant__ CUtensorMap tmW, const __grid_constant__ CUtensorMap tmX,
                         const __grid_constant__ CUtensorMap tmSFW, const __grid_constant__ CUtensorMap tmSFX,
                         const int splits, const int kb_per_split, const MxArgs args) {
  using S = SplitCfg<FMT, MT>;
  using C = typename S::C;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = smem_raw + (1024u - smem_u32(smem_raw) % 1024u) % 1024u;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + S::STAGES * C::STAGE_BYTES);
  uint64_t* empty = full + S::STAGES;
  uint64_t* tfull = empty + S::STAGES;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tfull + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = uniform_warp_id();
  const int lane = lane_id();
  const int rank = blockIdx.x % splits;  // clusters lie along x
  const int n0 = blockIdx.x / splits * 128, m0 = blockIdx.y * MT;
  const int kb0 = rank * kb_per_split, kb1 = min(args.num_kb, kb0 + kb_per_split);

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    mbar_init(tfull, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, S::TMEM_COLS);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 0) {
    bool aborted = false;
    for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
      const int stage = i % S::STAGES;
      if (i >= S::STAGES && !aborted)
        aborted = !mbar_wait(&empty[stage], (i / S::STAGES - 1) & 1, abort_flag, args.err, kErrTimeoutProducer);
      if (elect_one() && !aborted) {
        uint8_t* sw = smem + stage * C::STAGE_BYTES;
        uint8_t* sx = sw + C::A_BYTES;
        uint8_t* sfw = sx + C::B_BYTES;
        mbar_arrive_expect_tx(&full[stage], C::TX_BYTES);
        const uint32_t bar = smem_u32(&full[stage]);
        load_2d<1>(sw, &tmW, bar, kb * kRowBytes, n0);
        load_2d<1>(sx, &tmX, bar, kb * kRowBytes, m0);
        load_3d<1>(sfw, &tmSFW, bar, 0, kb * C::SF_TILES, n0 / 128);
        load_3d<1>(sfw + C::SFA_BYTES, &tmSFX, bar, 0, kb * C::SF_TILES, m0 / 128);
      }
      __syncwarp();
    }
    if (aborted) let_copies_land();
  } else if (warp == 1) {
    constexpr uint32_t idesc = mx_idesc<FMT>(128, MT);
    const Issuer<FMT, MT, 1> issue(smem_u32(smem), tmem + MT);
    bool aborted = false;
    for (int kb = kb0, i = 0; kb < kb1; ++kb, ++i) {
      const int stage = i % S::STAGES;
      if (!aborted) aborted = !mbar_wait(&full[stage], (i / S::STAGES) & 1, abort_flag, args.err, kErrTimeoutMma);
      tc_fence_after();
      if (elect_one() && !aborted) {
        issue.block(stage, tmem, idesc, kb == args.num_kb - 1 ? args.last_steps : kSteps, kb == kb0);
        mma_commit(&empty[stage]);
      }
      __syncwarp();
    }
    if (elect_one() && !aborted) mma_commit(tfull);
    __syncwarp();
  } else if (warp_wait(tfull, 0, abort_flag, args.err, kErrTimeoutEpilogue)) {
    tc_fence_after();
    const int q = warp & 3;
    const int lane_n = q * 32 + lane, n = n0 + lane_n;
    const int rows = min(MT, args.M - m0);
    const TensorScales scaled(args);
    const float bias = args.bias != nullptr && n < args.N ? args.bias[n] : 0.f;
    float* partial = reinterpret_cast<float*>(smem);  // [row][128 weight rows]: every staged block has been multiplied
#pragma unroll
    for (int c = 0; c < MT / 32; ++c) {
      if (32 * c >= rows) break;
      uint32_t r[32];
      tmem_ld32(tmem + (static_cast<uint32_t>(q * 32) << 16) + 32 * c, r);
      tmem_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const int m = 32 * c + i;
        if (m >= rows) break;
        if (splits > 1)
          partial[m * 128 + lane_n] = __uint_as_float(r[i]);
        else if (n < args.N)
          reinterpret_cast<T*>(args.out)[static_cast<long>(m0 + m) * args.N + n] =
              from_float<T>(scaled(__uint_as_float(r[i]), bias));
      }
    }
  }
  tc_fence_before();
  if (splits > 1) {
    cluster_sync();
    if (warp >= 2) {  // a warp per row, four columns per lane, every CTA's part requested before the first is added
      const int n = n0 + 4 * lane;
      const int rows = min(MT, args.M - m0);
      const TensorScales scaled(args);
      float bias[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bias[j] = args.bias != nullptr && n + j < args.N ? args.bias[n + j] : 0.f;
      const bool whole = args.N % 4 == 0 && n < args.N;
      uint32_t part_at[kMaxSplits];
#pragma unroll
      for (int s = 0; s < kMaxSplits; ++s) part_at[s] = map_to_rank(smem_u32(smem) + lane * 16u, min(s, splits - 1));
#pragma unroll 2
      for (int m = rank + splits * (warp & 3); m < rows; m += 4 * splits) {
        float4 part[kMaxSplits];
#pragma unroll
        for (int s = 0; s < kMaxSplits; ++s) {
          part[s] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (s < splits)
            asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                         : "=f"(part[s].x), "=f"(part[s].y), "=f"(part[s].z), "=f"(part[s].w)
                         : "r"(part_at[s] + m * 512u)
                         : "memory");
        }
        float4 sum = part[0];
#pragma unroll
        for (int s = 1; s < kMaxSplits; ++s)
          sum.x += part[s].x, sum.y += part[s].y, sum.z += part[s].z, sum.w += part[s].w;
        T* out = reinterpret_cast<T*>(args.out) + static_cast<long>(m0 + m) * args.N + n;
        alignas(16) T v[4] = {from_float<T>(scaled(sum.x, bias[0])), from_float<T>(scaled(sum.y, bias[1])),
                              from_float<T>(scaled(sum.z, bias[2])), from_float<T>(scaled(sum.w, bias[3]))};
        if (whole) {  // rows on 4 values
          if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(v);
          else *reinterpret_cast<uint4*>(out) = *reinterpret_cast<const uint4*>(v);
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (n + j < args.N) out[j] = v[j];
        }
      }
    }
    cluster_sync();  // no CTA leaves while another reads its sums
  } else {
    __syncthreads();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem, S::TMEM_COLS);
  }
}

CUtensorMap encode(CUtensorMapDataType type, int rank, const void* ptr, const cuuint64_t* dims,
                   const cuuint64_t* strides, const cuuint32_t* box, CUtensorMapSwizzle swizzle, const char* what) {
  CUtensorMap map;
  const cuuint32_t estr[3] = {1, 1, 1};
  const CUresult r = tensor_map_encoder()(&map, type, rank, const_cast<void*>(ptr), dims, strides, box, estr,
                                          CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  AVGEN_CHECK(r == CUDA_SUCCESS, "mx_gemm: cuTensorMapEncodeTiled failed for ", what, " (", static_cast<int>(r), ")");
  return map;
}

// Codes as a byte matrix [rows, row_bytes], boxes of `box_rows` x 128 bytes.
CUtensorMap codes_map(const void* ptr, long row_bytes, long rows, int box_rows) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(row_bytes), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(row_bytes)};
  const cuuint32_t box[2] = {kRowBytes, static_cast<cuuint32_t>(box_rows)};
  return encode(CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "codes");
}

// Scale tiles as [row groups, tiles, 128 words], boxes of `tiles` tiles of `groups` row groups.
CUtensorMap scales_map(const void* ptr, long tiles_k, long rows, int tiles, int groups) {
  const cuuint64_t dims[3] = {128, static_cast<cuuint64_t>(tiles_k), static_cast<cuuint64_t>((rows + 127) / 128)};
  const cuuint64_t strides[2] = {512, static_cast<cuuint64_t>(tiles_k * 512)};
  const cuuint32_t box[3] = {128, static_cast<cuuint32_t>(tiles), static_cast<cuuint32_t>(groups)};
  return encode(CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_NONE, "scales");
}

template <typename T>
CUtensorMap out_map(void* ptr, long rows, long cols) {
  constexpr auto type = sizeof(T) == 4                           ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                        : std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(cols) * sizeof(T)};
  const cuuint32_t box[2] = {128 / sizeof(T), 32};
  return encode(type, 2, ptr, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B, "the output");
}

template <typename T, int FMT, int BN, int CTAS>
void launch_tiles(const MxGemmDesc& d, const MxArgs& args, cudaStream_t stream) {
  using C = Cfg<FMT, BN, CTAS>;
  const long row_bytes = mx_row_bytes(FMT, d.K), tiles_k = mx_scale_tiles(FMT, d.K);
  const CUtensorMap ta = codes_map(d.a_codes, row_bytes, d.M, kBM);
  const CUtensorMap tb = codes_map(d.b_codes, row_bytes, d.N, C::B_ROWS);
  const CUtensorMap tsa = scales_map(d.a_scales, tiles_k, d.M, C::SF_TILES, 1);
  const CUtensorMap tsb = scales_map(d.b_scales, tiles_k, d.N, C::SF_TILES, BN / 128);
  const bool tma_out = static_cast<long>(d.N) * sizeof(T) % 16 == 0;
  const CUtensorMap to = tma_out ? out_map<T>(d.out, d.M, d.N) : ta;
  auto kernel = mx_gemm_kernel<T, FMT, BN, CTAS>;
  static PerDeviceOnce once;
  raise_smem_limit(once, kernel, C::SMEM_BYTES);
  const long tiles = static_cast<long>((d.M + CTAS * kBM - 1) / (CTAS * kBM)) * ((d.N + BN - 1) / BN);
  AVGEN_CHECK(tiles < (1L << 30), "mx_gemm: too many output tiles");
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(CTAS * std::min<long>(tiles, num_sms(d.device) / CTAS)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = C::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = CTAS;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = CTAS == 2 ? 1 : 0;
  AVGEN_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, ta, tb, tsa, tsb, to, tma_out, args));
}

// Clusters of 1..kMaxSplits CTAs, a CTA per SM, that the device holds at once: a cluster
// stays within one GPC, so larger ones leave SMs idle (148, 74, 45, 33, 26, 22, 15, 15).
struct ClusterRoom {
  int clusters[kMaxSplits + 1] = {};
};

// As many parts as leave every tile its cluster at once. More would put two CTAs on some
// SMs, which then share what an SM takes in (1 x 15360 x 2560 nvfp4, 120 tiles: one part 5.8
// us, two 7.3), or wait for a second round (77 x 2560 x 4096 mxfp8, 20 tiles: six parts 7.5
// us, seven 13).
inline int choose_splits(const ClusterRoom& room, long tiles, int num_kb) {
  int s = std::min(kMaxSplits, num_kb);
  while (s > 1 && room.clusters[s] < tiles) --s;
  return s;
}

template <typename T, int FMT, int MT>
void launch_split(const MxGemmDesc& d, const MxArgs& args, cudaStream_t stream) {
  using S = SplitCfg<FMT, MT>;
  using C = typename S::C;
  const long row_bytes = mx_row_bytes(FMT, d.K), tiles_k = mx_scale_tiles(FMT, d.K);
  const CUtensorMap tw = codes_map(d.b_codes, row_bytes, d.N, 128);
  const CUtensorMap tx = codes_map(d.a_codes, row_bytes, d.M, MT);
  const CUtensorMap tsw = scales_map(d.b_scales, tiles_k, d.N, C::SF_TILES, 1);
  const CUtensorMap tsx = scales_map(d.a_scales, tiles_k, d.M, C::SF_TILES, 1);
  auto kernel = mx_gemm_split_kernel<T, FMT, MT>;
  static PerDeviceOnce once, asked;
  raise_smem_limit(once, kernel, S::SMEM_BYTES);
  const unsigned tiles_n = static_cast<unsigned>((d.N + 127) / 128);
  const unsigned tiles_m = static_cast<unsigned>((d.M + MT - 1) / MT);
  cudaLaunchConfig_t cfg{};
  cfg.blockDim = dim3(192);
  cfg.dynamicSmemBytes = S::SMEM_BYTES;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  static ClusterRoom rooms[kMaxDevices];
  ClusterRoom& room = rooms[d.device];
  asked.run(d.device, [&] {
    for (int s = 1; s <= kMaxSplits; ++s) {
      cfg.gridDim = dim3(static_cast<unsigned>(s));
      attr.val.clusterDim.x = static_cast<unsigned>(s);
      AVGEN_CUDA_CHECK(cudaOccupancyMaxActiveClusters(&room.clusters[s], kernel, &cfg));
    }
  });
  int splits = choose_splits(room, static_cast<long>(tiles_n) * tiles_m, args.num_kb);
  const int per = (args.num_kb + splits - 1) / splits;
  splits = (args.num_kb + per - 1) / per;  // every CTA has a part
  cfg.gridDim = dim3(tiles_n * splits, tiles_m);
  attr.val.clusterDim.x = static_cast<unsigned>(splits);
  AVGEN_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, tw, tx, tsw, tsx, splits, per, args));
}

template <typename T, int FMT>
void launch(const MxGemmDesc& d, cudaStream_t stream) {
  MxArgs args{};
  args.M = d.M, args.N = d.N;
  const long row_bytes = mx_row_bytes(FMT, d.K);
  args.num_kb = static_cast<int>((row_bytes + kRowBytes - 1) / kRowBytes);
  args.last_steps = static_cast<int>((row_bytes - static_cast<long>(args.num_kb - 1) * kRowBytes + 31) / 32);
  args.a_g = d.a_g, args.b_g = d.b_g;
  args.bias = d.bias, args.out = d.out, args.err = d.err;
  // A k-block costs a CTA about as much in every form: its operand bytes from L2 (32 to 38
  // KB at some 45 bytes a clock). So the form with the fewest rounds of k-blocks wins: split
  // ones take 1 / splits of a round, 256 x 256 tiles one round for every SMs / 2 of them,
  // 128 x 128 tiles one for every SMs.
  const int sms = num_sms(d.device);
  const long tiles = static_cast<long>((d.M + 127) / 128) * ((d.N + 127) / 128);
  const long pairs = static_cast<long>((d.M + 255) / 256) * ((d.N + 255) / 256);
  if (d.M <= 32) return launch_split<T, FMT, 32>(d, args, stream);
  if (2 * tiles <= sms && args.num_kb > 1) return launch_split<T, FMT, 128>(d, args, stream);
  if ((pairs + sms / 2 - 1) / (sms / 2) <= (tiles + sms - 1) / sms)
    return launch_tiles<T, FMT, 256, 2>(d, args, stream);
  launch_tiles<T, FMT, 128, 1>(d, args, stream);
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
