// FP8 matrix product  out[M, N] (+)= A[M, K] B[N, K]^T  with an FP32 scale for each block of 128 along K
// (per row, or per 128 rows, of either operand).
//
//   out[m, n] = sum over K blocks b of  sa[m, b] * sb[n, b] * ( sum over k in b of  a[m, k] * b[n, k] )
//
// The inner sum runs on the tensor cores (tcgen05.mma kind::f8f6f4, FP32 accumulator in TMEM, a fresh one for each
// block of 128); the outer sum runs in FP32 registers of the epilogue warps, which read each block's accumulator
// once and add it times the block's scales.  So any FP32 scales are applied as they are, to operands as they are
// stored, and the accumulation across blocks is plain FP32.
//
// "P" is the operand whose rows lie on the TMEM lanes (128 a tile), "Q" the one whose rows are its columns (BN a tile).
// P = A, Q = B in general; for few rows of A the roles are swapped (SWAP): the weights' rows fill the lanes and the
// tokens are BN = 16, 32 or 64 columns, so that no lane is idle and the weights stream through once.
//
// Roles of a CTA: warp 0 TMA, warp 1 MMA and TMEM, the others add up the blocks.  S CTAs of a cluster may share one
// tile, each a range of the blocks; their sums are joined through distributed shared memory in a fixed order.
#include "../../include/weftmoe_b200.h"
#include "gemm.cuh"
#include "kernels.h"

using namespace wm;

namespace {

__device__ int g_matmul_status;   // a bounded wait that ran out (read by wm_fp8_matmul_status)

constexpr int kScaleChunk = 8;    // blocks of scales held at a time

struct MatmulArgs {
  const float* p_scales;
  const float* q_scales;
  int p_rows, q_rows;             // M, N or N, M
  int p_block_rows, q_block_rows; // 1 or 128
  int kblocks;                    // stride of the scales
  int p_tiles, q_tiles, split;
  void* out;
  long long ld;
  int out_is_f32, accumulate, vector_store;
};

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
  static_assert(N == 16 || N == 32, "columns of one load");
  if constexpr (N == 16) tmem_ld_32x16(taddr, v);
  else tmem_ld_32x32(taddr, v);
}
// 4 bytes global -> shared, or zero.
__device__ __forceinline__ void copy_async_4(float* dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(there ? 4 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
__device__ __forceinline__ void copy_async_wait() { asm volatile("cp.async.wait_group 0;" ::: "memory"); }
template <int THREADS>
__device__ __forceinline__ void adders_sync() { asm volatile("bar.sync 1, %0;" ::"n"(THREADS) : "memory"); }
__device__ __forceinline__ float load_cluster(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}

// Shared memory of the scales: [2][kScaleChunk][pitch].  Eight lanes copy the eight blocks of one row (one 32-byte
// sector); the pitch of 4 (mod 32) words keeps those eight and the next three rows in different banks.
template <int BN, bool Q_COLS>
struct ScaleTable {
  static constexpr int kPitchP = 128 + 4;
  static constexpr int kPitchQ = Q_COLS ? BN + 4 : 4;
  static constexpr int kWords = 2 * kScaleChunk * (kPitchP + kPitchQ);
};

template <int BN, int EPI, bool Q_COLS>
__device__ __forceinline__ void fetch_scales(const MatmulArgs& a, float* table, int buffer, int p0, int q0, int kb0,
                                             int kb1, int thread) {
  using T = ScaleTable<BN, Q_COLS>;
  float* tp = table + buffer * kScaleChunk * T::kPitchP;
  float* tq = table + 2 * kScaleChunk * T::kPitchP + buffer * kScaleChunk * T::kPitchQ;
  const int kb = thread & 7;
  const bool in = kb0 + kb < kb1;
  for (int r = thread >> 3; r < 128; r += EPI * 4) {
    const bool there = in && p0 + r < a.p_rows;
    const float* src = a.p_scales + (there ? static_cast<long long>((p0 + r) / a.p_block_rows) * a.kblocks + kb0 + kb : 0);
    copy_async_4(tp + kb * T::kPitchP + r, src, there);
  }
  constexpr int kEntries = Q_COLS ? BN : BN / 128;
  for (int c = thread >> 3; c < kEntries; c += EPI * 4) {
    const int row = q0 + (Q_COLS ? c : c * 128);
    const bool there = in && row < a.q_rows;
    const float* src = a.q_scales + (there ? static_cast<long long>(row / a.q_block_rows) * a.kblocks + kb0 + kb : 0);
    copy_async_4(tq + kb * T::kPitchQ + c, src, there);
  }
  copy_async_commit();
}

template <int BN, int EPI, bool Q_COLS>
struct MatmulSmem {
  static constexpr int kPBytes = 128 * 128;
  static constexpr int kQBytes = BN * 128;
  static constexpr int kStageBytes = kPBytes + kQBytes;
  static constexpr int kBuffers = BN == 256 ? 2 : 4;       // accumulators in TMEM
  static constexpr int kColumns = BN * kBuffers < 32 ? 32 : BN * kBuffers;
  static constexpr int kStages = BN >= 128 ? 5 : 8;
  static constexpr int kScaleBytes = ScaleTable<BN, Q_COLS>::kWords * 4;
  static constexpr int kTotal = kStages * kStageBytes + kScaleBytes + 256 + 1024;
  static_assert(BN * 128 * 4 <= kStages * kStageBytes, "the joined sums fit in the stages");
};

// One column of a finished tile.
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

template <int BN, int EPI, bool SWAP, bool Q_COLS>
__global__ void __launch_bounds__(64 + 32 * EPI, 1)
fp8_matmul_kernel(const __grid_constant__ CUtensorMap tmap_p, const __grid_constant__ CUtensorMap tmap_q,
                  const MatmulArgs a) {
  using S = MatmulSmem<BN, EPI, Q_COLS>;
  using T = ScaleTable<BN, Q_COLS>;
  constexpr int kCols = BN / (EPI / 4);                   // columns of one adding warp
  constexpr int kLoad = kCols < 32 ? kCols : 32;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) &
                                             ~static_cast<uintptr_t>(1023));
  float* scales = reinterpret_cast<float*>(smem + S::kStages * S::kStageBytes);
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + S::kStages * S::kStageBytes + S::kScaleBytes);
  uint64_t* empty_bar = full_bar + S::kStages;
  uint64_t* tmem_full = empty_bar + S::kStages;
  uint64_t* tmem_empty = tmem_full + S::kBuffers;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(tmem_empty + S::kBuffers);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_holder + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int s = 0; s < S::kStages; ++s) {
      mbar_init(full_bar + s, 1);
      mbar_init(empty_bar + s, 1);
    }
    for (int s = 0; s < S::kBuffers; ++s) {
      mbar_init(tmem_full + s, 1);
      mbar_init(tmem_empty + s, EPI);
    }
    *abort_flag = 0;
    mbar_fence_init();
    tma_prefetch_desc(&tmap_p);
    tma_prefetch_desc(&tmap_q);
  }
  if (warp == 1) {
    tmem_alloc(tmem_holder, S::kColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;

  const int part = a.split > 1 ? static_cast<int>(cluster_ctarank()) : 0;
  const int kb0 = static_cast<int>(static_cast<long long>(a.kblocks) * part / a.split);
  const int kb1 = static_cast<int>(static_cast<long long>(a.kblocks) * (part + 1) / a.split);
  const int tiles = a.p_tiles * a.q_tiles;
  const int first = blockIdx.x / a.split, step = gridDim.x / a.split;

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < tiles; tile += step) {
        const int p0 = tile % a.p_tiles * 128, q0 = tile / a.p_tiles * BN;
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(empty_bar + stage, phase ^ 1, abort_flag, &g_matmul_status, kStatusTimeoutSmemEmpty);
          if (!ok) break;
          uint8_t* sp = smem + stage * S::kStageBytes;
          mbar_expect_tx(full_bar + stage, S::kStageBytes);
          tma_load_2d(sp, &tmap_p, full_bar + stage, kb * 128, p0);
          tma_load_2d(sp + S::kPBytes, &tmap_q, full_bar + stage, kb * 128, q0);
          if (++stage == S::kStages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = umma_idesc(0u, 128, BN, 0u, 0u);
      int stage = 0, buffer = 0;
      uint32_t phase = 0, buffer_phase = 0;
      bool ok = true;
      for (int tile = first; ok && tile < tiles; tile += step) {
        for (int kb = kb0; kb < kb1; ++kb) {
          ok = mbar_wait(tmem_empty + buffer, buffer_phase ^ 1, abort_flag, &g_matmul_status, kStatusTimeoutTmemEmpty) &&
               mbar_wait(full_bar + stage, phase, abort_flag, &g_matmul_status, kStatusTimeoutSmemFull);
          if (!ok) break;
          tc_fence_after();
          const uint32_t sp = smem_u32(smem + stage * S::kStageBytes);
          const uint64_t dp = umma_desc_sw128(sp, 0, 1024), dq = umma_desc_sw128(sp + S::kPBytes, 0, 1024);
#pragma unroll
          for (int k = 0; k < 4; ++k)
            umma_f8(tmem_base + buffer * BN, dp + 2 * k, dq + 2 * k, idesc, k != 0 ? 1u : 0u);
          umma_commit(empty_bar + stage);
          umma_commit(tmem_full + buffer);
          if (++stage == S::kStages) { stage = 0; phase ^= 1; }
          if (++buffer == S::kBuffers) { buffer = 0; buffer_phase ^= 1; }
        }
      }
    }
  } else {
    const int thread = threadIdx.x - 64;
    const int q = warp & 3, half = (warp - 2) >> 2;
    const int row = q * 32 + lane, col0 = half * kCols;
    int buffer = 0, held = 0;
    uint32_t buffer_phase = 0;
    bool ok = true;   // a wait that runs out skips the arithmetic; the barriers below are still met by every warp
    if (first < tiles)
      fetch_scales<BN, EPI, Q_COLS>(a, scales, 0, first % a.p_tiles * 128, first / a.p_tiles * BN, kb0, kb1, thread);
    for (int tile = first; tile < tiles; tile += step) {
      const int p0 = tile % a.p_tiles * 128, q0 = tile / a.p_tiles * BN;
      float sum[kCols];
#pragma unroll
      for (int j = 0; j < kCols; ++j) sum[j] = 0.0f;
      for (int chunk = kb0; chunk < kb1; chunk += kScaleChunk) {
        copy_async_wait();
        adders_sync<EPI * 32>();   // this chunk is here, and the other buffer is no longer read
        if (chunk + kScaleChunk < kb1)
          fetch_scales<BN, EPI, Q_COLS>(a, scales, held ^ 1, p0, q0, chunk + kScaleChunk, kb1, thread);
        else if (tile + step < tiles)
          fetch_scales<BN, EPI, Q_COLS>(a, scales, held ^ 1, (tile + step) % a.p_tiles * 128,
                                        (tile + step) / a.p_tiles * BN, kb0, kb1, thread);
        const float* tp = scales + held * kScaleChunk * T::kPitchP + row;
        const float* tq = scales + 2 * kScaleChunk * T::kPitchP + held * kScaleChunk * T::kPitchQ;
        const int last = min(kScaleChunk, kb1 - chunk);
        for (int kb = 0; kb < last; ++kb) {
          ok = ok && mbar_wait(tmem_full + buffer, buffer_phase, abort_flag, &g_matmul_status, kStatusTimeoutTmemFull);
          if (!ok) continue;
          tc_fence_after();
          float factor = tp[kb * T::kPitchP];
          if constexpr (!Q_COLS) factor *= tq[kb * T::kPitchQ + col0 / 128];
#pragma unroll
          for (int c = 0; c < kCols / kLoad; ++c) {
            uint32_t v[kLoad];
            tmem_ld_cols<kLoad>(tmem_base + (static_cast<uint32_t>(q * 32) << 16) + buffer * BN + col0 + c * kLoad, v);
            tmem_ld_wait();
            if (c == kCols / kLoad - 1) {
              tc_fence_before();
              __syncwarp();
              if (lane == 0) mbar_arrive(tmem_empty + buffer);
            }
#pragma unroll
            for (int j = 0; j < kLoad; ++j) {
              float f = factor;
              if constexpr (Q_COLS) f *= tq[kb * T::kPitchQ + col0 + c * kLoad + j];
              sum[c * kLoad + j] = fmaf(f, __uint_as_float(v[j]), sum[c * kLoad + j]);
            }
          }
          if (++buffer == S::kBuffers) { buffer = 0; buffer_phase ^= 1; }
        }
        held ^= 1;
      }
      if (a.split > 1) {   // one tile per CTA: the stages are no longer written
        float* mine = reinterpret_cast<float*>(smem);
#pragma unroll
        for (int j = 0; j < kCols; ++j) mine[(col0 + j) * 128 + row] = sum[j];
      } else if (ok && p0 + row < a.p_rows) {
        if constexpr (SWAP) {
#pragma unroll
          for (int j = 0; j < kCols; ++j)
            if (q0 + col0 + j < a.q_rows) store_one<true>(a, p0 + row, q0 + col0 + j, sum[j]);
        } else {
          store_row<kCols>(a, p0 + row, q0 + col0, sum);
        }
      }
    }
  }
  if (a.split > 1) {
    __syncwarp();
    cluster_sync_all();
    if (warp >= 2 && first < tiles && !*abort_flag) {
      const int p0 = first % a.p_tiles * 128, q0 = first / a.p_tiles * BN;
      const int row = (warp & 3) * 32 + lane;
      const int cols = BN / a.split;                                        // this CTA's columns of the tile
      const uint32_t base = smem_u32(smem);
      for (int c = (warp - 2) >> 2; c < cols; c += EPI / 4) {
        const int col = part * cols + c;
        float v = 0.0f;
        for (int s = 0; s < a.split; ++s) v += load_cluster(map_to_cta(base + (col * 128 + row) * 4, s));
        if (p0 + row < a.p_rows && q0 + col < a.q_rows) store_one<SWAP>(a, p0 + row, q0 + col, v);
      }
    }
    __syncwarp();
    cluster_sync_all();   // the others' shared memory stays until it is read
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, S::kColumns);
  }
}

template <int BN, int EPI, bool SWAP, bool Q_COLS>
int launch_matmul(const CUtensorMap& tp, const CUtensorMap& tq, MatmulArgs a, int sms, cudaStream_t stream) {
  auto kernel = fp8_matmul_kernel<BN, EPI, SWAP, Q_COLS>;
  constexpr int smem = MatmulSmem<BN, EPI, Q_COLS>::kTotal;
  static PerDeviceOnce configured;  // one table per template instantiation
  if (int rc = opt_in_dynamic_smem(kernel, smem, configured)) return rc;
  a.p_tiles = (a.p_rows + 127) / 128;
  a.q_tiles = (a.q_rows + BN - 1) / BN;
  const long long tiles = static_cast<long long>(a.p_tiles) * a.q_tiles;
  // Few tiles: 2, 4 or 8 CTAs take a share of the blocks each, while every SM still gets at most one CTA
  // and every CTA two blocks.
  a.split = 1;
  while (a.split < 8 && tiles * a.split * 2 <= sms && a.kblocks / (a.split * 2) >= 2) a.split *= 2;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(a.split > 1 ? tiles * a.split : tiles < sms ? tiles : sms));
  config.blockDim = dim3(64 + 32 * EPI);
  config.dynamicSmemBytes = smem;
  config.stream = stream;
  cudaLaunchAttribute cluster{};
  cluster.id = cudaLaunchAttributeClusterDimension;
  cluster.val.clusterDim.x = a.split;
  cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
  config.attrs = &cluster;
  config.numAttrs = 1;
  WM_CUDA(cudaLaunchKernelEx(&config, kernel, tp, tq, a));
  count_launch();
  return WM_OK;
}

}  // namespace

extern "C" int wm_fp8_matmul(const void* aq, const float* as, const void* bq, const float* bs, void* out, int64_t ld,
                             int32_t m, int32_t n, int32_t k, int32_t a_block_rows, int32_t b_block_rows,
                             int32_t out_is_f32, int32_t accumulate, void* stream_) {
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
  int sms = 0, dev = 0;
  WM_CUDA(cudaGetDevice(&dev));
  WM_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
  // Up to 64 rows of A ride in the columns; beyond that its rows fill the lanes.
  const bool swap = m <= 64;
  const int bn = swap ? (m <= 16 ? 16 : m <= 32 ? 32 : 64) : 128;
  MatmulArgs a{};
  a.p_scales = swap ? bs : as;
  a.q_scales = swap ? as : bs;
  a.p_rows = swap ? n : m;
  a.q_rows = swap ? m : n;
  a.p_block_rows = swap ? b_block_rows : a_block_rows;
  a.q_block_rows = swap ? a_block_rows : b_block_rows;
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
  if (swap) {
    if (bn == 16) return launch_matmul<16, 4, true, true>(tp, tq, a, sms, stream);
    if (bn == 32) return launch_matmul<32, 4, true, true>(tp, tq, a, sms, stream);
    return launch_matmul<64, 4, true, true>(tp, tq, a, sms, stream);
  }
  return a.q_block_rows == 128 ? launch_matmul<128, 8, false, false>(tp, tq, a, sms, stream)
                               : launch_matmul<128, 8, false, true>(tp, tq, a, sms, stream);
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
