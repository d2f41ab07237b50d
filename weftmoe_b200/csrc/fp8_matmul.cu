// FP8 matrix product  out[M, N] (+)= A[M, K] B[N, K]^T  with an FP32 scale for each block of 128 along K
// (per row, or per 128 rows, of either operand).
//
//   out[m, n] = sum over K blocks b of  sa[m, b] * sb[n, b] * ( sum over k in b of  a[m, k] * b[n, k] )
//
// The inner sum runs on the tensor cores (tcgen05.mma kind::f8f6f4, FP32 accumulator in TMEM, a fresh one for each
// block of 128); the outer sum runs in FP32 registers of the adding warps, which read each block's accumulator
// once and add it times the block's scales.  So any FP32 scales are applied as they are, to operands as they are
// stored, and the accumulation across blocks is plain FP32.
//
// "P" is the operand whose rows lie on the TMEM lanes (128 a CTA), "Q" the one whose rows are its columns (BN a tile).
// P = A, Q = B in general; for few rows of A (rides_in_columns) the roles are swapped (SWAP): the weights' rows fill the lanes and the
// tokens are BN = 16, 32 or 64 columns, so that no lane is idle and the weights stream through once.
//
// Warps of a CTA: 0 TMA, 1 MMA and TMEM, 2 and 3 fetch the scales, the others add up the blocks.  A stage's `done`
// barrier, one commit per block, both frees the stage and hands its accumulator to the adding warps.
// PAIR: two CTAs compute one 256 x 256 tile with cta_group::2, each fetching its own 128 rows of P and half of Q's 256,
// so a byte of either operand feeds twice the arithmetic of a 128 x 128 tile.
// PAIR, scales all powers of two (what this library's quantisers give): the tensor cores apply the scales themselves
// (kind::mxf8f6f4.block_scale, scales as UE8M0 in TMEM) and accumulate up to 32 blocks before the adding warps take them
// over.  The accumulator cuts what it cannot hold, so its error grows with the number of blocks (normal operands: 4.9e-7
// of the result at K = 8192 and 3.0e-6 at 32768 in one go); with 32 it stays at 2.2e-7 from K = 4096 up (general form: 0.7
// to 2.3e-7 from 4096 to 32768), at 5.4e-7 where the products of scales vary by 2^6 from block to block (general form
// 1.3e-7, K = 8190), and at 1.4e-6 where all products are positive and every cut goes the same way (general form 0.9 to
// 2.5e-7).  E4M3 itself is off by up to 2^-4 an operand.  A kernel in front packs the scales and notes whether one is no
// power of two; the product then takes the general form above.
// Otherwise `split` CTAs of a cluster may share one tile, each a range of the blocks; their sums are joined through
// distributed shared memory in a fixed order.
//
// What bounds it.  Few rows (64 x 4096 x 4096: 9.3 us back to back; its 17 MB of weights take 2.7 us to read): the start of
// the kernel, 8 blocks a CTA one after the other, and the join of four sums.  Large products with packed scales (8192 x
// 4096 x 4096: 94 us on its own with the packing in front, 2.9 PFLOP/s, tensor pipe 76 % busy): operands from shared
// memory and L2; back to back the power limit makes it 116 us.  Long K on few tiles (4096 x 2048, K = 8190: 58 us replayed,
// 60 % busy): 128 tiles on 74 pairs, a second wave that is three quarters full, and the packing.  General scales on pairs
// (137 and 148 us for these two): the adding warps, 128 accumulators a thread read, scaled and added for every block.
#include <limits.h>

#include <algorithm>
#include <atomic>

#include "../../include/weftmoe_b200.h"
#include "gemm.cuh"
#include "kernels.h"

using namespace wm;

namespace {

__device__ int g_matmul_status;   // a bounded wait that ran out (read by wm_fp8_matmul_status)

constexpr int kScaleChunk = 8;    // blocks of scales held at a time
constexpr int kGroupBlocks = 32;  // blocks that the tensor cores accumulate when they apply the scales
constexpr int kPackBlocks = 32;   // blocks of K that one CTA of the packing kernel takes

struct MatmulArgs {
  const float* p_scales;
  const float* q_scales;
  int p_rows, q_rows;             // M, N or N, M
  int p_shift, q_shift;           // log2 of the rows of a scale: 0 or 7
  int kblocks;                    // stride of the scales
  int p_tiles, q_tiles, split;
  void* out;
  long long ld;
  int out_is_f32, accumulate;
  int vector_store;               // rows of out are 16-byte aligned
  int tma_store;                  // ... and tmap_out describes them
  const int* findings;            // of the packing kernel: non-zero where a scale is no power of two; null = not packed
  int num_findings;
};

// ---------------------------------------------------------------- instructions
__device__ __forceinline__ void tmem_ld_32x8(uint32_t taddr, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
        "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15])
      : "r"(taddr)
      : "memory");
}
template <int N>
__device__ __forceinline__ void tmem_ld_cols(uint32_t taddr, uint32_t (&v)[N]) {
  static_assert(N == 8 || N == 16 || N == 32, "columns of one load");
  if constexpr (N == 8) tmem_ld_32x8(taddr, v);
  else if constexpr (N == 16) tmem_ld_32x16(taddr, v);
  else tmem_ld_32x32(taddr, v);
}
// Waits for this thread's TMEM loads.  The registers pass through empty statements behind the wait, so that
// nothing that reads them is moved before it.
template <int N>
__device__ __forceinline__ void tmem_ld_wait_for(uint32_t (&v)[N]) {
  tmem_ld_wait();
#pragma unroll
  for (int j = 0; j < N; ++j) asm volatile("" : "+r"(v[j]));
}
// 4 bytes global -> shared, or zero.
__device__ __forceinline__ void copy_async_4(float* dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0)
               : "memory");
}
// One arrival of this thread on `bar` when its copies so far have landed.
__device__ __forceinline__ void copy_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_all;" ::: "memory"); }
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Two FP32 multiply-adds in one instruction, on register pairs.
__device__ __forceinline__ uint64_t pair_of(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 halves_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul_pair(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// CTA-pair MMA of 8-bit operands (M = 256: 128 rows in each CTA's TMEM).
__device__ __forceinline__ void umma_f8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                             uint32_t accumulate) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// One commit that arrives on the barrier at this offset in both CTAs of the pair.
__device__ __forceinline__ void umma_commit_both(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
          smem_u32(bar)),
      "h"(static_cast<uint16_t>(3))
      : "memory");
}
// Arrives on an mbarrier of the cluster without a fence over global memory: what the arrival orders are TMEM reads,
// and those are complete (tcgen05.wait::ld).  With .release.cluster here, once per block, the product of
// 8192 x 4096 x 4096 took 278 us instead of 171, the difference in the fence.
__device__ __forceinline__ void arrive_in_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Block-scaled MMA on a CTA pair (one UE8M0 scale per row and 32 elements of K, in TMEM), and the copy that brings a
// 512-byte chunk of scales from each CTA's shared memory to its TMEM.
__device__ __forceinline__ void umma_mxf8_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                               uint32_t accumulate, uint32_t tmem_sfa, uint32_t tmem_sfb) {
  asm volatile(
      "{\n"
      ".reg .pred p;\n"
      "setp.ne.b32 p, %4, 0;\n"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n"
      "}\n" ::"r"(tmem_d),
      "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate), "r"(tmem_sfa), "r"(tmem_sfb)
      : "memory");
}
__device__ __forceinline__ void tmem_cp_pair(uint32_t taddr, uint64_t smem_desc) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(smem_desc) : "memory");
}
template <int REGS>
__device__ __forceinline__ void registers_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS>
__device__ __forceinline__ void registers_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }

// ---------------------------------------------------------------- layout
template <int BN, int EPI, bool SWAP, bool Q_COLS, bool PAIR>
struct Matmul {
  static constexpr int kThreads = 128 + 32 * EPI;
  static constexpr int kCols = BN / (EPI / 4);                   // columns of one adding warp
  static constexpr int kLoad = kCols / 2 < 32 ? kCols / 2 : 32;  // ... of one TMEM load
  static constexpr int kRowsP = PAIR ? 256 : 128;                // of a tile
  static constexpr int kPBytes = 128 * 128;
  static constexpr int kQBytes = (PAIR ? BN / 2 : BN) * 128;     // this CTA's
  static constexpr int kStageBytes = kPBytes + kQBytes;
  static constexpr int kBuffers = BN == 256 ? 2 : 4;             // accumulators in TMEM
  static constexpr int kColumns = BN * kBuffers < 32 ? 32 : BN * kBuffers;
  static constexpr int kStages = PAIR ? 5 : BN == 128 ? 5 : 8;
  static_assert(kStages >= kBuffers, "an adding warp is never a whole round of stages behind the MMA");
  // Scales: [2][kScaleChunk][pitch] of P, then of Q.  Eight lanes copy the eight blocks of one row (one 32-byte
  // sector); the pitch of 4 (mod 32) words keeps those eight and the next three rows in different banks.
  static constexpr int kPitchP = 128 + 4;
  static constexpr int kPitchQ = Q_COLS ? BN + 4 : 4;
  static constexpr int kScaleBytes = 2 * kScaleChunk * (kPitchP + kPitchQ) * 4;
  static constexpr int kStoreBytes = SWAP ? 0 : 4096;            // staging of one adding warp: a box of 32 rows x 128 bytes
  static constexpr int kScalesAt = kStages * kStageBytes + EPI * kStoreBytes;
  static constexpr int kBarriersAt = kScalesAt + kScaleBytes;
  static constexpr int kTotal = kBarriersAt + 256 + 1024;
  static_assert(kScalesAt % 16 == 0 && kTotal <= 227 * 1024, "shared memory");
  static_assert(PAIR || BN * 128 * 4 <= kStages * kStageBytes, "the joined sums fit in the stages");
  // PAIR with packed scales: chunks of 128 rows' scales of four blocks, one of P and two of Q, come with every fourth
  // stage, in place of the table; in TMEM twice behind the one accumulator, 16 columns each.  (A chunk for every block, the
  // same byte four times, took 131 us for 8192 x 4096 x 4096 where four blocks a chunk took 117, repeated without a pause.)
  static constexpr int kPackedBytes = 3 * 512;
  static constexpr uint32_t kTmemScales = BN;
  static_assert(!PAIR || kStages * kPackedBytes <= kScaleBytes, "packed scales fit where the table is");
  // PAIR: the four service warps give registers to the eight adding warps: 128 x 56 + 256 x 224 = 384 x 168, what
  // the block is launched with (pair_kernels_fit looks before a launch is planned).
  static constexpr int kRegisters = 168, kLow = 56, kHigh = 224;
  static_assert(!PAIR || 128 * kLow + 256 * kHigh <= kThreads * kRegisters, "registers of the block");
};

struct Tile {
  int p0, q0;   // first rows of this CTA's P, of the tile's Q
};
// Tiles are walked in groups of eight rows of tiles, so that the CTAs in flight share both operands in L2.
template <int ROWS_P, int BN>
__device__ __forceinline__ Tile tile_at(const MatmulArgs& a, int tile) {
  const int per_group = 8 * a.q_tiles;
  const int group = tile / per_group, rem = tile - group * per_group;
  const int rows = min(8, a.p_tiles - group * 8);
  return Tile{(group * 8 + rem % rows) * ROWS_P, rem / rows * BN};
}

// ---------------------------------------------------------------- results
template <bool SWAP>
__device__ __forceinline__ void store_one(const MatmulArgs& a, int p, int q, float v) {
  const long long at = SWAP ? static_cast<long long>(q) * a.ld + p : static_cast<long long>(p) * a.ld + q;
  if (a.out_is_f32) {
    float* o = static_cast<float*>(a.out) + at;
    *o = a.accumulate ? *o + v : v;
  } else {
    static_cast<__nv_bfloat16*>(a.out)[at] = __float2bfloat16_rn(v);
  }
}
// COLS consecutive columns of row p (not swapped): 16-byte stores where the rows are aligned and whole.
template <int COLS>
__device__ __forceinline__ void store_row(const MatmulArgs& a, int p, int q, const float (&v)[COLS]) {
  if (a.vector_store && q + COLS <= a.q_rows) {
    if (a.out_is_f32) {
      float4* o = reinterpret_cast<float4*>(static_cast<float*>(a.out) + static_cast<long long>(p) * a.ld + q);
#pragma unroll
      for (int j = 0; j < COLS / 4; ++j) {
        float4 w = make_float4(v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
        if (a.accumulate) {
          const float4 old = o[j];
          w.x += old.x; w.y += old.y; w.z += old.z; w.w += old.w;
        }
        o[j] = w;
      }
    } else {
      uint4* o = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + static_cast<long long>(p) * a.ld + q);
#pragma unroll
      for (int j = 0; j < COLS / 8; ++j)
        o[j] = make_uint4(pack_bf16x2(v[8 * j], v[8 * j + 1]), pack_bf16x2(v[8 * j + 2], v[8 * j + 3]),
                          pack_bf16x2(v[8 * j + 4], v[8 * j + 5]), pack_bf16x2(v[8 * j + 6], v[8 * j + 7]));
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < COLS; ++j)
    if (q + j < a.q_rows) store_one<false>(a, p, q + j, v[j]);
}
// A warp's 32 rows x 2 * PAIRS columns by way of shared memory: boxes of 32 rows x 128 bytes, 16-byte pieces swizzled by
// the row.  From there TMA writes them (tma_store; the map clips what lies outside the matrix), or, where the rows of out do
// not start and end on 16 bytes or are added to, the warp does, row by row: 64 or 128 neighbouring bytes an instruction.
template <int PAIRS>
__device__ __forceinline__ void store_boxes(const MatmulArgs& a, const CUtensorMap* tmap, uint8_t* staging, int p, int q,
                                            int lane, const uint64_t (&sum)[PAIRS]) {
  uint8_t* line = staging + lane * 128;
  const int boxes = a.out_is_f32 ? PAIRS / 16 : PAIRS / 32;
#pragma unroll
  for (int b = 0; b < PAIRS / 16; ++b) {
    if (b == boxes) break;
    if (a.tma_store && lane == 0) bulk_wait_group_read<0>();   // the box before this one has left the staging
    __syncwarp();
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      uint4 w;
      if (a.out_is_f32) {
        const int from = b * 16 + c * 2;
        const float2 x = halves_of(sum[from]), y = halves_of(sum[from + 1]);
        w = make_uint4(__float_as_uint(x.x), __float_as_uint(x.y), __float_as_uint(y.x), __float_as_uint(y.y));
      } else {
        const int from = (b * 32 + c * 4) % PAIRS;       // (boxes behind the last are not reached)
        const float2 x = halves_of(sum[from]), y = halves_of(sum[from + 1]), z = halves_of(sum[from + 2]),
                     t = halves_of(sum[from + 3]);
        w = make_uint4(pack_bf16x2(x.x, x.y), pack_bf16x2(y.x, y.y), pack_bf16x2(z.x, z.y), pack_bf16x2(t.x, t.y));
      }
      *reinterpret_cast<uint4*>(line + ((c ^ (lane & 7)) << 4)) = w;
    }
    const int x = q + b * (a.out_is_f32 ? 32 : 64);
    if (a.tma_store) {
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) {
        if (p < a.p_rows && x < a.q_rows) tma_store_2d(tmap, staging, x, p);
        bulk_commit_group();
      }
    } else {
      __syncwarp();
      const int rows = min(32, a.p_rows - p);
#pragma unroll 4
      for (int r = 0; r < rows; ++r) {
        const long long at = static_cast<long long>(p + r) * a.ld + x + lane;
        if (a.out_is_f32) {
          const float w = *reinterpret_cast<const float*>(staging + r * 128 + (((lane >> 2) ^ (r & 7)) << 4) + (lane & 3) * 4);
          float* o = static_cast<float*>(a.out) + at;
          if (x + lane < a.q_rows) *o = a.accumulate ? *o + w : w;
        } else {
          __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.out) + at;
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int col = lane + 32 * h;
            const uint8_t* from = staging + r * 128 + (((col >> 3) ^ (r & 7)) << 4) + (col & 7) * 2;
            if (x + col < a.q_rows) o[32 * h] = *reinterpret_cast<const __nv_bfloat16*>(from);
          }
        }
      }
      __syncwarp();
    }
  }
}

// ---------------------------------------------------------------- the kernel
template <int BN, int EPI, bool SWAP, bool Q_COLS, bool PAIR>
__global__ void __launch_bounds__(128 + 32 * EPI, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                  const __grid_constant__ CUtensorMap tmap_out, const __grid_constant__ CUtensorMap tmap_sp,
                  const __grid_constant__ CUtensorMap tmap_sq, const MatmulArgs a) {
  using S = Matmul<BN, EPI, SWAP, Q_COLS, PAIR>;
  constexpr int kCols = S::kCols, kLoad = S::kLoad;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* scales_p = reinterpret_cast<float*>(smem + S::kScalesAt);
  float* scales_q = scales_p + 2 * kScaleChunk * S::kPitchP;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::kBarriersAt);   // PAIR: the leader's is used
  uint64_t* done_bar = full_bar + S::kStages;                                // in both CTAs
  uint64_t* tmem_empty = done_bar + S::kStages;                              // the leader's
  uint64_t* scale_full = tmem_empty + S::kBuffers;
  uint64_t* scale_empty = scale_full + 2;
  uint64_t* group_full = scale_empty + 2;                                    // packed scales: accumulator ready, in both
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(group_full + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int cta = PAIR ? static_cast<int>(cluster_ctarank()) : 0;            // 0 = leader
  const int part = !PAIR && a.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full_bar + s, 1);
      mbar_init(done_bar + s, 1);
    }
    for (int s = 0; s < S::kBuffers; ++s) mbar_init(tmem_empty + s, PAIR ? 2 * EPI : EPI);
    for (int s = 0; s < 2; ++s) {
      mbar_init(scale_full + s, 64);
      mbar_init(scale_empty + s, EPI);
    }
    mbar_init(group_full, 1);
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
  }
  if (warp == 1) {
    tmem_alloc<PAIR ? 2 : 1>(tmem_holder, S::kColumns);   // PAIR: warp 1 of both CTAs, as all of the kernel's group
    tmem_relinquish<PAIR ? 2 : 1>();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the peer's barriers are initialised before anything arrives on them
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  cudaGridDependencySynchronize();   // launched while the kernel before still runs: nothing is read or written until here
  bool packed = false;
  if constexpr (PAIR) {
    if (a.findings != nullptr) {
      int found = 0;
      for (int i = threadIdx.x; i < a.num_findings; i += S::kThreads) found |= __ldcg(a.findings + i);
      packed = __syncthreads_or(found) == 0;
    }
  }

  const int group = PAIR ? 2 : a.split;    // CTAs of a tile
  const int kb0 = static_cast<int>(static_cast<long long>(a.kblocks) * part / a.split);
  const int kb1 = static_cast<int>(static_cast<long long>(a.kblocks) * (part + 1) / a.split);
  const int tiles = a.p_tiles * a.q_tiles;
  const int first = blockIdx.x / group, step = gridDim.x / group;

  if (warp < 4) {
    if constexpr (PAIR) registers_down<S::kLow>();
    if (warp == 0 && lane == 0) {
      // ------------------------------------------------------------ TMA
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < tiles; tile += step) {
        const Tile t = tile_at<S::kRowsP, BN>(a, tile);
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(done_bar + stage, phase ^ 1, abort_flag, &g_matmul_status, kStatusTimeoutSmemEmpty);
          if (!ok) break;
          uint8_t* sp = smem + stage * S::kStageBytes;
          if constexpr (PAIR) {
            const uint32_t bar = map_to_cta(smem_u32(full_bar + stage), 0);
            const bool scales_too = packed && kb % 4 == 0;
            if (cta == 0) mbar_expect_tx(full_bar + stage, 2 * (S::kStageBytes + (scales_too ? S::kPackedBytes : 0)));
            tma_load_2d_pair(sp, &tmap_p, bar, kb * 128, t.p0 + cta * 128);
            tma_load_2d_pair(sp + S::kPBytes, &tmap_q, bar, kb * 128, t.q0 + cta * (BN / 2));
            if (scales_too) {   // a chunk is four rows of 128 bytes; each CTA holds the scales of all 256 columns
              uint8_t* sf = smem + S::kScalesAt + stage * S::kPackedBytes;
              const int chunks = (a.kblocks + 3) / 4;
              tma_load_2d_pair(sf, &tmap_sp, bar, 0, ((t.p0 >> 7) + cta) * chunks * 4 + kb);
              tma_load_2d_pair(sf + 512, &tmap_sq, bar, 0, (t.q0 >> 7) * chunks * 4 + kb);
              tma_load_2d_pair(sf + 1024, &tmap_sq, bar, 0, ((t.q0 >> 7) + 1) * chunks * 4 + kb);
            }
          } else {
            mbar_expect_tx(full_bar + stage, S::kStageBytes);
            tma_load_2d(sp, &tmap_p, full_bar + stage, kb * 128, t.p0);
            tma_load_2d(sp + S::kPBytes, &tmap_q, full_bar + stage, kb * 128, t.q0);
          }
          if (++stage == S::kStages) { stage = 0; phase ^= 1; }
        }
      }
    } else if (warp == 1 && cta == 0) {
      // ------------------------------------------------------------ MMA
      // The whole warp walks the blocks and one elected lane issues, so that descriptors and addresses stay in uniform
      // registers: issued by a lane on its own, a block's four MMAs and commit took 462 cycles, more than the MMAs run.
      const uint64_t d0 = umma_desc_sw128(smem_u32(smem), 0, 1024);
      int stage = 0, buffer = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool ok = true;
      if constexpr (PAIR) {
        if (packed) {
          for (int tile = first; ok && tile < tiles; tile += step) {
            for (int kb = 0; kb < a.kblocks; ++kb) {
              const bool opens = kb % kGroupBlocks == 0;
              if (opens) {
                ok = mbar_wait(tmem_empty, buffer_phase ^ 1, abort_flag, &g_matmul_status, kStatusTimeoutTmemEmpty);
                buffer_phase ^= 1;
              }
              ok = ok && mbar_wait(full_bar + stage, phase, abort_flag, &g_matmul_status, kStatusTimeoutSmemFull);
              ok = __all_sync(0xffffffffu, ok);
              if (!ok) break;
              tc_fence_after();
              const uint64_t dp = d0 + static_cast<uint32_t>(stage * (S::kStageBytes >> 4)), dq = dp + (S::kPBytes >> 4);
              const uint32_t sfp = tmem_base + S::kTmemScales + (kb / 4 % 2) * 16, sfq = sfp + 4;
              const uint32_t idesc_kb = umma_idesc_block_scaled(0u, 1u, 256, BN, kb & 3, kb & 3);   // byte of the chunk
              const bool closes = kb + 1 == a.kblocks || (kb + 1) % kGroupBlocks == 0;
              if (elect_one()) {
                if (kb % 4 == 0) {
                  const uint64_t sf = umma_desc_noswizzle(smem_u32(smem + S::kScalesAt + stage * S::kPackedBytes), 128);
                  tmem_cp_pair(sfp, sf);
                  tmem_cp_pair(sfq, sf + 32);
                  tmem_cp_pair(sfq + 4, sf + 64);
                }
#pragma unroll
                for (int k = 0; k < 4; ++k)
                  umma_mxf8_pair(tmem_base, dp + 2 * k, dq + 2 * k, idesc_kb, opens && k == 0 ? 0u : 1u, sfp, sfq);
                umma_commit_both(done_bar + stage);
                if (closes) umma_commit_both(group_full);
              }
              __syncwarp();
              if (++stage == S::kStages) { stage = 0; phase ^= 1; }
            }
          }
          ok = false;   // the loop below is the other form's
        }
      }
      constexpr uint32_t idesc = umma_idesc(0u, S::kRowsP, BN, 0u, 0u);
      for (int tile = first; ok && tile < tiles; tile += step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(tmem_empty + buffer, buffer_phase ^ 1, abort_flag, &g_matmul_status, kStatusTimeoutTmemEmpty) &&
               mbar_wait(full_bar + stage, phase, abort_flag, &g_matmul_status, kStatusTimeoutSmemFull);
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          tc_fence_after();
          const uint64_t dp = d0 + static_cast<uint32_t>(stage * (S::kStageBytes >> 4)), dq = dp + (S::kPBytes >> 4);
          if (elect_one()) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if constexpr (PAIR) umma_f8_pair(tmem_base + buffer * BN, dp + 2 * k, dq + 2 * k, idesc, k != 0 ? 1u : 0u);
              else umma_f8(tmem_base + buffer * BN, dp + 2 * k, dq + 2 * k, idesc, k != 0 ? 1u : 0u);
            }
            if constexpr (PAIR) umma_commit_both(done_bar + stage);
            else umma_commit(done_bar + stage);
          }
          __syncwarp();
          if (++stage == S::kStages) { stage = 0; phase ^= 1; }
          if (++buffer == S::kBuffers) { buffer = 0; buffer_phase ^= 1; }
        }
      }
    } else if (warp >= 2 && !packed) {
      // ------------------------------------------------------------ scales
      const int kb = lane & 7, row = (threadIdx.x - 64) >> 3;
      int held = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < tiles; tile += step) {
        const Tile t = tile_at<S::kRowsP, BN>(a, tile);
        const int p0 = t.p0 + cta * 128;
        for (int chunk = kb0; chunk < kb1; chunk += kScaleChunk) {
          ok = mbar_wait(scale_empty + held, phase ^ 1, abort_flag, &g_matmul_status, kStatusTimeoutSmemEmpty);
          if (!ok) break;
          float* to = scales_p + (held * kScaleChunk + kb) * S::kPitchP;
          const bool in = chunk + kb < kb1;
#pragma unroll 4
          for (int r = row; r < 128; r += 8) {
            const bool there = in && p0 + r < a.p_rows;
            copy_async_4(to + r, a.p_scales + (there ? static_cast<long long>((p0 + r) >> a.p_shift) * a.kblocks + chunk + kb : 0),
                         there);
          }
          to = scales_q + (held * kScaleChunk + kb) * S::kPitchQ;
          constexpr int kEntries = Q_COLS ? BN : BN / 128;
#pragma unroll 4
          for (int c = row; c < kEntries; c += 8) {
            const int r = t.q0 + (Q_COLS ? c : c * 128);
            const bool there = in && r < a.q_rows;
            copy_async_4(to + c, a.q_scales + (there ? static_cast<long long>(r >> a.q_shift) * a.kblocks + chunk + kb : 0),
                         there);
          }
          copy_async_arrive(scale_full + held);
          if (++held == 2) { held = 0; phase ^= 1; }
        }
      }
      copy_async_wait();
    }
  } else {
    // ------------------------------------------------------------ sums
    if constexpr (PAIR) registers_up<S::kHigh>();
    const int q = warp & 3, col0 = ((warp - 4) >> 2) * kCols;
    const int row = q * 32 + lane;
    const uint32_t from = tmem_base + (static_cast<uint32_t>(q * 32) << 16) + col0;
    int stage = 0, buffer = 0, held = 0;
    uint32_t phase = 0, held_phase = 0;
    bool ok = true;
    for (int tile = first; ok && tile < tiles; tile += step) {
      const Tile t = tile_at<S::kRowsP, BN>(a, tile);
      const int p0 = t.p0 + cta * 128;
      uint64_t sum[kCols / 2];
#pragma unroll
      for (int j = 0; j < kCols / 2; ++j) sum[j] = 0;
      // Loads run ahead of the additions by kLoad columns, across blocks too.
      uint32_t v[2][kLoad];
      if (PAIR && packed) {
        for (int kb = 0; kb < a.kblocks; kb += kGroupBlocks) {
          ok = mbar_wait(group_full, phase, abort_flag, &g_matmul_status, kStatusTimeoutTmemFull);
          if (!ok) break;
          phase ^= 1;
          tc_fence_after();
          tmem_ld_cols<kLoad>(from, v[0]);
#pragma unroll
          for (int c = 0; c < kCols / kLoad; ++c) {
            tmem_ld_wait_for<kLoad>(v[c & 1]);
            if (c + 1 < kCols / kLoad) {
              tmem_ld_cols<kLoad>(from + (c + 1) * kLoad, v[(c + 1) & 1]);
            } else {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) arrive_in_cluster(map_to_cta(smem_u32(tmem_empty), 0));
            }
#pragma unroll
            for (int j = 0; j < kLoad / 2; ++j) {
              const float2 w = halves_of(sum[c * (kLoad / 2) + j]);
              sum[c * (kLoad / 2) + j] = pair_of(w.x + __uint_as_float(v[c & 1][2 * j]), w.y + __uint_as_float(v[c & 1][2 * j + 1]));
            }
          }
        }
      } else {
        ok = mbar_wait(done_bar + stage, phase, abort_flag, &g_matmul_status, kStatusTimeoutTmemFull);
        if (!ok) break;
        tc_fence_after();
        tmem_ld_cols<kLoad>(from + buffer * BN, v[0]);
      }
      for (int kb = PAIR && packed ? kb1 : kb0; kb < kb1; ++kb) {
        const int in_chunk = (kb - kb0) & (kScaleChunk - 1);
        if (in_chunk == 0) {
          ok = mbar_wait(scale_full + held, held_phase, abort_flag, &g_matmul_status, kStatusTimeoutTmemFull);
          if (!ok) break;
        }
        const float* tq = scales_q + (held * kScaleChunk + in_chunk) * S::kPitchQ + (Q_COLS ? col0 : col0 / 128);
        float factor = scales_p[(held * kScaleChunk + in_chunk) * S::kPitchP + row];
        if constexpr (!Q_COLS) factor *= *tq;
        const uint64_t factors = pair_of(factor, factor);
#pragma unroll
        for (int c = 0; c < kCols / kLoad; ++c) {
          tmem_ld_wait_for<kLoad>(v[c & 1]);
          if (c + 1 < kCols / kLoad) {
            tmem_ld_cols<kLoad>(from + buffer * BN + (c + 1) * kLoad, v[(c + 1) & 1]);
          } else {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
              if constexpr (PAIR) arrive_in_cluster(map_to_cta(smem_u32(tmem_empty + buffer), 0));
              else mbar_arrive(tmem_empty + buffer);
            }
            if (++stage == S::kStages) { stage = 0; phase ^= 1; }
            if (++buffer == S::kBuffers) buffer = 0;
            if (kb + 1 < kb1) {
              ok = mbar_wait(done_bar + stage, phase, abort_flag, &g_matmul_status, kStatusTimeoutTmemFull);
              tc_fence_after();
              tmem_ld_cols<kLoad>(from + buffer * BN, v[(c + 1) & 1]);
            }
          }
#pragma unroll
          for (int j = 0; j < kLoad / 2; ++j) {
            const uint64_t x = pair_of(__uint_as_float(v[c & 1][2 * j]), __uint_as_float(v[c & 1][2 * j + 1]));
            uint64_t f = factors;
            if constexpr (Q_COLS) {
              const float2 w = *reinterpret_cast<const float2*>(tq + c * kLoad + 2 * j);
              f = mul_pair(f, pair_of(w.x, w.y));
            }
            sum[c * (kLoad / 2) + j] = fma_pair(f, x, sum[c * (kLoad / 2) + j]);
          }
        }
        if (in_chunk == kScaleChunk - 1 || kb + 1 == kb1) {
          __syncwarp();
          if (lane == 0) mbar_arrive(scale_empty + held);
          if (++held == 2) { held = 0; held_phase ^= 1; }
        }
        if (!ok) break;
      }
      tmem_ld_wait();
      if (!ok) break;
      if (!PAIR && a.split > 1) {   // one tile per CTA: its stages are read and no longer written
        float* mine = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j) {
          const float2 w = halves_of(sum[j]);
          mine[(col0 + 2 * j) * 128 + row] = w.x;
          mine[(col0 + 2 * j + 1) * 128 + row] = w.y;
        }
      } else if constexpr (SWAP) {
#pragma unroll
        for (int j = 0; j < kCols / 2; ++j) {
          const float2 w = halves_of(sum[j]);
          if (p0 + row < a.p_rows && t.q0 + col0 + 2 * j < a.q_rows) store_one<true>(a, p0 + row, t.q0 + col0 + 2 * j, w.x);
          if (p0 + row < a.p_rows && t.q0 + col0 + 2 * j + 1 < a.q_rows)
            store_one<true>(a, p0 + row, t.q0 + col0 + 2 * j + 1, w.y);
        }
      } else {
        store_boxes<kCols / 2>(a, &tmap_out, smem + S::kStages * S::kStageBytes + (warp - 4) * S::kStoreBytes,
                               p0 + q * 32, t.q0 + col0, lane, sum);
      }
    }
    if (!SWAP && lane == 0) bulk_wait_group_read<0>();   // the staging stays until it is read
  }
  __syncwarp();
  if (!PAIR && a.split > 1) {
    cluster_sync_all();
    if (warp >= 4 && first < tiles && !*abort_flag) {
      const Tile t = tile_at<S::kRowsP, BN>(a, first);
      const int row = (warp & 3) * 32 + lane;
      const int cols = BN / a.split;                                        // this CTA's columns of the tile
      const uint32_t base = smem_u32(smem) + row * 4;
      constexpr int kAtOnce = BN / 4 < 8 ? BN / 4 : 8;                      // columns of a thread at a time (split <= 4)
      for (int c = (warp - 4) / 4 * kAtOnce; c < cols; c += EPI / 4 * kAtOnce) {
        const int col = part * cols + c;
        float v[kAtOnce], w[4][kAtOnce];                                      // all loads before the first addition
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          if (s >= a.split) break;
          const uint32_t from = map_to_cta(base + col * 512, s);
#pragma unroll
          for (int j = 0; j < kAtOnce; ++j) w[s][j] = load_cluster(from + j * 512);
        }
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          v[j] = w[0][j] + w[1][j];                                           // split is 2 or 4
          if (a.split == 4) v[j] = (v[j] + w[2][j]) + w[3][j];
        }
        if (t.p0 + row < a.p_rows) {
          if constexpr (SWAP) {
#pragma unroll
            for (int j = 0; j < kAtOnce; ++j)
              if (t.q0 + col + j < a.q_rows) store_one<true>(a, t.p0 + row, t.q0 + col + j, v[j]);
          } else {
            store_row<kAtOnce>(a, t.p0 + row, t.q0 + col, v);
          }
        }
      }
    }
    __syncwarp();
    cluster_arrive();
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (PAIR) cluster_sync_all();  // the peer's shared memory and barriers stay valid until both are done
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc<PAIR ? 2 : 1>(tmem_base, S::kColumns);
  }
  if (!PAIR && a.split > 1) cluster_wait();   // this CTA's sums stay until the others have read them
}

// FP32 scales -> UE8M0 chunks [ceil(rows / 128)][ceil(kblocks / 4)][512 bytes] in the 4 x 32 order of tcgen05.cp (word
// (r % 32) * 4 + r / 32 holds row r, byte i the block 4 c + i), of P and then of Q.  Rows and blocks behind the last get
// scale 1.  Each CTA, one of 128 rows x 32 blocks, notes whether it met a scale that is no power of two.  5.5 us alone,
// nearly all of it latency (1 MB in, 0.3 MB out for 8192 x 4096 scaled by rows); behind a quantiser its start is hidden.
__global__ void __launch_bounds__(256)
pack_scales_kernel(const float* p_scales, int p_rows, int p_shift, uint32_t* p_out, const float* q_scales, int q_rows,
                   int q_shift, uint32_t* q_out, int kblocks, int* findings) {
  __shared__ unsigned char codes[kPackBlocks][128 + 4];
  cudaTriggerProgrammaticLaunchCompletion();   // the product may take its place; it waits for these before it reads
  // As this kernel does for the one that quantised the operands.  That one may still write the scales while this one runs,
  // so they are read by ordinary loads: no __ldg and no __restrict__ here.
  cudaGridDependencySynchronize();
  const int p_tiles = (p_rows + 127) / 128;
  const bool of_p = static_cast<int>(blockIdx.x) < p_tiles;
  const int tile = of_p ? blockIdx.x : blockIdx.x - p_tiles;
  const float* scales = of_p ? p_scales : q_scales;
  const int rows = of_p ? p_rows : q_rows, shift = of_p ? p_shift : q_shift;
  const int kb0 = blockIdx.y * kPackBlocks, count = min(kPackBlocks, kblocks - kb0);
  int found = 0;
  constexpr int kEach = 128 * kPackBlocks / 256;
  const int kb = threadIdx.x % kPackBlocks, r0 = threadIdx.x / kPackBlocks;
  unsigned bits[kEach];   // all loads before the first use: one after the other they took 10 us
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const int row = tile * 128 + r0 + i * (256 / kPackBlocks);
    bits[i] = kb < count && row < rows
                  ? __float_as_uint(scales[static_cast<long long>(row >> shift) * kblocks + kb0 + kb]) : 0x3f800000u;
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i) {
    const unsigned code = bits[i] >> 23;   // the biased exponent is the UE8M0 code
    found |= (bits[i] & 0x7fffffu) != 0 || code == 0 || code >= 255;   // mantissa, zero, infinite, negative
    codes[kb][r0 + i * (256 / kPackBlocks)] = static_cast<unsigned char>(code);
  }
  found = __syncthreads_or(found);
  if (threadIdx.x == 0) findings[blockIdx.y * gridDim.x + blockIdx.x] = found;
  const int chunks = (kblocks + 3) / 4, here = (count + 3) / 4;
  uint32_t* out = (of_p ? p_out : q_out) + (static_cast<long long>(tile) * chunks + kb0 / 4) * 128;
  for (int i = threadIdx.x; i < 128 * here; i += 256) {
    const int c = i / 128 * 4, word = i % 128, r = (word >> 2) + 32 * (word & 3);
    out[i] = codes[c][r] | codes[c + 1][r] << 8 | codes[c + 2][r] << 16 | static_cast<unsigned>(codes[c + 3][r]) << 24;
  }
}

// What a product on CTA pairs with packed scales needs besides its operands.
struct Packing {
  int p_tiles, q_tiles, parts, chunks;
  long long q_at, findings_at, bytes;
};
Packing packing_of(int m, int n, int kblocks) {
  Packing k{};
  k.p_tiles = (m + 127) / 128;
  k.q_tiles = (n + 127) / 128;
  k.parts = (kblocks + kPackBlocks - 1) / kPackBlocks;
  k.chunks = (kblocks + 3) / 4;
  k.q_at = static_cast<long long>(k.p_tiles) * k.chunks * 512;
  k.findings_at = k.q_at + static_cast<long long>(k.q_tiles) * k.chunks * 512;
  k.bytes = k.findings_at + static_cast<long long>(k.p_tiles + k.q_tiles) * k.parts * 4;
  return k;
}

// Whether A's rows ride in the columns.  Up to 32 they do; beyond 64 they fill the lanes; between, the narrow tile pays
// where four CTAs share it, each with 4 to 16 blocks.  64 rows, in the columns / in the lanes, us: 4096 columns of out, K =
// 1024: 7.0 / 5.9, 2048: 7.8 / 8.4, 4096: 9.3 / 9.9, 16384: 18.1 / 17.3; 16384 columns (one CTA a tile), K = 512: 7.4 / 5.6,
// 4096: 17.7 / 13.9.
bool rides_in_columns(int m, int n, int kblocks, int sms) {
  return m <= 32 || (m <= 64 && (static_cast<long long>(n) + 127) / 128 * 4 <= sms && kblocks >= 16 && kblocks <= 64);
}

// Beyond 64 rows of A: CTA pairs take less time a block and wave but start about 2.6 us later (the packing kernel, a
// pair's set-up), so they pay where they save at least 8 blocks of a wave.  One CTA a tile / pairs, us: 1024 x 4096, K =
// 512: 8.0 / 8.7, K = 1024: 10.4 / 10.1, K = 4096: 25.4 / 18.2; 2048 x 4096, K = 512: 12.1 / 10.7, K = 4096: 46.6 / 28.8;
// 2048 x 1024, K = 4096: 14.9 / 17.2.
bool pays_for_pairs(int m, int n, int kblocks, int sms) {
  if (m <= 64) return false;
  const long long single = static_cast<long long>((m + 127) / 128) * ((n + 127) / 128);
  const long long paired = static_cast<long long>((m + 255) / 256) * ((n + 255) / 256);
  const long long waves = (single + sms - 1) / sms - (paired + sms / 2 - 1) / (sms / 2);
  return waves * kblocks >= 8;
}

// Whether both pair kernels were built with the registers that their warps share out: the launch bounds are only a
// limit from above, and warps that asked for more than the block has would wait for good.
std::atomic<int> g_most_registers{INT_MAX};   // wm_debug_matmul_pair_registers
int pair_kernels_fit(bool* fit) {
  using S = Matmul<256, 8, false, true, true>;
  static std::atomic<int> built{0};   // the lower of the two; 0 = not asked yet
  int registers = built.load(std::memory_order_relaxed);
  if (registers == 0) {
    cudaFuncAttributes by_column{}, by_block{};
    WM_CUDA(cudaFuncGetAttributes(&by_column, fp8_matmul_kernel<256, 8, false, true, true>));
    WM_CUDA(cudaFuncGetAttributes(&by_block, fp8_matmul_kernel<256, 8, false, false, true>));
    registers = std::min(by_column.numRegs, by_block.numRegs);
    built.store(registers, std::memory_order_relaxed);
  }
  *fit = std::min(registers, g_most_registers.load(std::memory_order_relaxed)) >= S::kRegisters;
  return WM_OK;
}

int sm_count(int* sms) {
  int dev = 0;
  WM_CUDA(cudaGetDevice(&dev));
  WM_CUDA(cudaDeviceGetAttribute(sms, cudaDevAttrMultiProcessorCount, dev));
  return WM_OK;
}

int takes_pairs(int m, int n, int kblocks, int sms, bool* pairs) {
  *pairs = pays_for_pairs(m, n, kblocks, sms);
  return *pairs ? pair_kernels_fit(pairs) : WM_OK;
}

template <int BN, int EPI, bool SWAP, bool Q_COLS, bool PAIR>
int launch_matmul(const CUtensorMap& tp, const CUtensorMap& tq, const CUtensorMap& tout, const CUtensorMap& tsp,
                  const CUtensorMap& tsq, MatmulArgs a, int sms, cudaStream_t stream) {
  using S = Matmul<BN, EPI, SWAP, Q_COLS, PAIR>;
  auto kernel = fp8_matmul_kernel<BN, EPI, SWAP, Q_COLS, PAIR>;
  static PerDeviceOnce configured;  // one table per template instantiation
  if (int rc = opt_in_dynamic_smem(kernel, S::kTotal, configured)) return rc;
  a.p_tiles = (a.p_rows + S::kRowsP - 1) / S::kRowsP;
  a.q_tiles = (a.q_rows + BN - 1) / BN;
  const long long tiles = static_cast<long long>(a.p_tiles) * a.q_tiles;
  if (tiles > 0x3fffffff) {
    set_error("wm_fp8_matmul: more than 2^30 tiles");
    return WM_ERR_INVALID;
  }
  // Few tiles: 2 or 4 CTAs take a share of the blocks each, while every SM still gets at most one CTA and every CTA
  // two blocks.  The join costs as much as some blocks: 100 x 1024, K = 1024: 6.0 us alone, 7.5 shared; 2048: 8.3 / 8.1;
  // 4096: 12.9 / 9.2; one row, K = 512: 4.5 / 4.9, 1024: 5.5 / 4.8.  (Clusters of 8 start 2 us later: 1 x 2048 x 4096 took
  // 10.0 us with them, 7.4 us with 4.)
  a.split = 1;
  if (!PAIR && a.kblocks >= (SWAP ? 8 : 16))
    while (a.split < 4 && tiles * a.split * 2 <= sms && a.kblocks / (a.split * 2) >= 2) a.split *= 2;
  const int group = PAIR ? 2 : a.split;
  const long long groups = tiles * group <= sms ? tiles : sms / group;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(groups * group));
  config.blockDim = dim3(S::kThreads);
  config.dynamicSmemBytes = S::kTotal;
  config.stream = stream;
  cudaLaunchAttribute attributes[2] = {};
  attributes[0].id = cudaLaunchAttributeClusterDimension;
  attributes[0].val.clusterDim.x = group;
  attributes[0].val.clusterDim.y = attributes[0].val.clusterDim.z = 1;
  attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attributes[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attributes;
  config.numAttrs = 2;
  WM_CUDA(cudaLaunchKernelEx(&config, kernel, tp, tq, tout, tsp, tsq, a));
  count_launch();
  return WM_OK;
}

}  // namespace

extern "C" int wm_fp8_matmul(const void* aq, const float* as, const void* bq, const float* bs, void* out, int64_t ld,
                             int32_t m, int32_t n, int32_t k, int32_t a_block_rows, int32_t b_block_rows,
                             int32_t out_is_f32, int32_t accumulate, void* workspace, int64_t workspace_bytes,
                             void* stream_) {
  if (m < 0 || n < 0 || k < 0 || (a_block_rows != 1 && a_block_rows != 128) ||
      (b_block_rows != 1 && b_block_rows != 128) || ld < n || (accumulate && !out_is_f32)) {
    set_error("wm_fp8_matmul: [M,K] x [N,K], block rows 1 or 128, rows of out at least N apart; accumulation needs an "
              "FP32 output");
    return WM_ERR_INVALID;
  }
  if (m == 0 || n == 0) return WM_OK;
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  const int element = out_is_f32 ? 4 : 2;
  if (!out || reinterpret_cast<uintptr_t>(out) % element) {
    set_error("wm_fp8_matmul: null or misaligned output");
    return WM_ERR_INVALID;
  }
  if (k == 0) {
    if (!accumulate)
      WM_CUDA(cudaMemset2DAsync(out, static_cast<size_t>(ld) * element, 0, static_cast<size_t>(n) * element, m, stream));
    return WM_OK;
  }
  if (!aq || !as || !bq || !bs || reinterpret_cast<uintptr_t>(aq) % 16 || reinterpret_cast<uintptr_t>(bq) % 16 ||
      reinterpret_cast<uintptr_t>(as) % 4 || reinterpret_cast<uintptr_t>(bs) % 4) {
    set_error("wm_fp8_matmul: null or misaligned operand (16-byte alignment required)");
    return WM_ERR_INVALID;
  }
  const int kblocks = static_cast<int>((static_cast<long long>(k) + 127) / 128);
  const uint64_t pitch = static_cast<uint64_t>(kblocks) * 128;
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const bool swap = rides_in_columns(m, n, kblocks, sms);
  bool pairs = false;
  if (int rc = takes_pairs(m, n, kblocks, sms, &pairs)) return rc;
  const int bn = swap ? (m <= 16 ? 16 : m <= 32 ? 32 : 64) : 128;
  const Packing packing = packing_of(m, n, kblocks);
  const bool packed = workspace && pairs;
  if (packed && (workspace_bytes < packing.bytes || reinterpret_cast<uintptr_t>(workspace) % 128)) {
    set_error("wm_fp8_matmul: small or misaligned workspace (wm_fp8_matmul_workspace, 128-byte aligned)");
    return WM_ERR_INVALID;
  }
  MatmulArgs a{};
  a.p_scales = swap ? bs : as;
  a.q_scales = swap ? as : bs;
  a.p_rows = swap ? n : m;
  a.q_rows = swap ? m : n;
  a.p_shift = (swap ? b_block_rows : a_block_rows) == 128 ? 7 : 0;
  a.q_shift = (swap ? a_block_rows : b_block_rows) == 128 ? 7 : 0;
  a.kblocks = kblocks;
  a.out = out;
  a.ld = ld;
  a.out_is_f32 = out_is_f32;
  a.accumulate = accumulate;
  a.vector_store = reinterpret_cast<uintptr_t>(out) % 16 == 0 && ld * element % 16 == 0;
  // The maps end at k, not at the padded row: what the padding bytes hold is never read.
  CUtensorMap tp, tq;
  if (int rc = make_tmap_2d(&tp, swap ? bq : aq, 1, k, a.p_rows, pitch, 128, 128)) return rc;
  if (int rc = make_tmap_2d(&tq, swap ? aq : bq, 1, k, a.q_rows, pitch, 128, bn)) return rc;
  CUtensorMap tout = tp;   // not read without tma_store
  // A TMA store writes 16 bytes at a time, also where the map's rows end between: those would reach behind column n.
  a.tma_store = !swap && a.vector_store && !accumulate && static_cast<long long>(n) * element % 16 == 0;
  if (a.tma_store)
    if (int rc = make_tmap_2d(&tout, out, element, n, m, static_cast<uint64_t>(ld) * element, 128 / element, 32)) return rc;
  CUtensorMap tsp = tp, tsq = tp;   // not read without packed scales
  if (packed) {
    uint8_t* room = static_cast<uint8_t*>(workspace);
    int* findings = reinterpret_cast<int*>(room + packing.findings_at);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(packing.p_tiles + packing.q_tiles, packing.parts);
    config.blockDim = dim3(256);
    config.stream = stream;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    WM_CUDA(cudaLaunchKernelEx(&config, pack_scales_kernel, as, m, a.p_shift, reinterpret_cast<uint32_t*>(room), bs, n,
                               a.q_shift, reinterpret_cast<uint32_t*>(room + packing.q_at), kblocks, findings));
    count_launch();
    a.findings = findings;
    a.num_findings = (packing.p_tiles + packing.q_tiles) * packing.parts;
    const uint64_t rows_p = static_cast<uint64_t>(packing.p_tiles) * packing.chunks * 4;
    const uint64_t rows_q = static_cast<uint64_t>(packing.q_tiles) * packing.chunks * 4;
    if (int rc = make_tmap_2d(&tsp, room, 1, 128, rows_p, 128, 128, 4, false)) return rc;
    if (int rc = make_tmap_2d(&tsq, room + packing.q_at, 1, 128, rows_q, 128, 128, 4, false)) return rc;
  }
  const bool by_column = a.q_shift == 0;
  if (bn == 16) return launch_matmul<16, 4, true, true, false>(tp, tq, tout, tsp, tsq, a, sms, stream);
  if (bn == 32) return launch_matmul<32, 8, true, true, false>(tp, tq, tout, tsp, tsq, a, sms, stream);
  if (bn == 64) return launch_matmul<64, 8, true, true, false>(tp, tq, tout, tsp, tsq, a, sms, stream);
  if (pairs)
    return by_column ? launch_matmul<256, 8, false, true, true>(tp, tq, tout, tsp, tsq, a, sms, stream)
                     : launch_matmul<256, 8, false, false, true>(tp, tq, tout, tsp, tsq, a, sms, stream);
  return by_column ? launch_matmul<128, 8, false, true, false>(tp, tq, tout, tsp, tsq, a, sms, stream)
                   : launch_matmul<128, 8, false, false, false>(tp, tq, tout, tsp, tsq, a, sms, stream);
}

extern "C" int wm_fp8_linear(const void* x, int32_t x_is_f32, int32_t rows, int32_t k, const void* wq, const float* ws,
                             int32_t n, void* out, void* workspace, int64_t workspace_bytes, void* stream) {
  if (rows < 0 || k < 0 || n < 0) {
    set_error("wm_fp8_linear: negative size");
    return WM_ERR_INVALID;
  }
  if (rows == 0 || n == 0) return WM_OK;
  const long long kblocks = (static_cast<long long>(k) + 127) / 128;
  // the quantised x, its scales, the product's own workspace
  const long long scales_at = static_cast<long long>(rows) * kblocks * 128;
  const long long rest_at = (scales_at + static_cast<long long>(rows) * kblocks * 4 + 127) / 128 * 128;
  int64_t rest = 0;
  if (int rc = wm_fp8_matmul_workspace(rows, n, k, &rest)) return rc;
  if ((!workspace && rest_at + rest > 0) || workspace_bytes < rest_at + rest || reinterpret_cast<uintptr_t>(workspace) % 128) {
    set_error("wm_fp8_linear: missing, small or misaligned workspace (wm_fp8_linear_workspace, 128-byte aligned)");
    return WM_ERR_INVALID;
  }
  char* room = static_cast<char*>(workspace);
  float* xs = reinterpret_cast<float*>(room + scales_at);
  if (int rc = wm_fp8_quantize(x, x_is_f32, 1, rows, k, 1, 0, room, xs, stream)) return rc;
  return wm_fp8_matmul(room, xs, wq, ws, out, n, rows, n, k, 1, 128, x_is_f32, 0, rest ? room + rest_at : nullptr, rest,
                       stream);
}

extern "C" int wm_fp8_linear_workspace(int32_t rows, int32_t n, int32_t k, int64_t* bytes) {
  if (int rc = wm_fp8_matmul_workspace(rows, n, k, bytes)) return rc;
  const long long kblocks = (static_cast<long long>(k) + 127) / 128;
  *bytes += (static_cast<long long>(rows) * kblocks * 132 + 127) / 128 * 128;
  return WM_OK;
}

extern "C" int wm_fp8_matmul_workspace(int32_t m, int32_t n, int32_t k, int64_t* bytes) {
  if (m < 0 || n < 0 || k < 0 || !bytes) {
    set_error("wm_fp8_matmul_workspace: negative size or null result");
    return WM_ERR_INVALID;
  }
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int kblocks = static_cast<int>((static_cast<long long>(k) + 127) / 128);
  bool pairs = false;
  if (int rc = takes_pairs(m, n, kblocks, sms, &pairs)) return rc;
  *bytes = pairs ? packing_of(m, n, kblocks).bytes : 0;
  return WM_OK;
}

extern "C" void wm_debug_matmul_pair_registers(int most) {
  g_most_registers.store(most > 0 ? most : INT_MAX, std::memory_order_relaxed);
}

extern "C" int wm_fp8_matmul_status(int32_t* code, void* stream_) {
  if (!code) { set_error("wm_fp8_matmul_status: null result"); return WM_ERR_INVALID; }
  cudaStream_t stream = static_cast<cudaStream_t>(stream_);
  void* word = nullptr;
  int status = 0;
  WM_CUDA(cudaGetSymbolAddress(&word, g_matmul_status));
  WM_CUDA(cudaMemcpyAsync(&status, word, sizeof(int), cudaMemcpyDeviceToHost, stream));
  WM_CUDA(cudaMemsetAsync(word, 0, sizeof(int), stream));
  WM_CUDA(cudaStreamSynchronize(stream));
  *code = status ? WM_ERR_TIMEOUT : WM_OK;
  return WM_OK;
}
