// Projections on the tensor cores (bf16, fp16; fp32 accumulation in TMEM).
//
// gemm_kernel: a CTA takes tiles of 128 activation rows by up to 256 weight
// rows (output features). One thread of warp 4 copies 64-feature slices of
// both operands into a ring of shared-memory stages by TMA (128-byte swizzle),
// one thread of warp 5 issues the tcgen05.mma, and warps 0-3 turn a finished
// accumulator into outputs while the next tile accumulates in the other half
// of TMEM. A thread of warps 0-3 owns one activation row of the tile (its TMEM
// lane) and walks the row's columns, so the vocabulary head's maximum and sum
// need no exchange between threads.
//
// Weights may have either dimension contiguous: with the input features
// contiguous a stage holds them K-major (128-byte rows of 64 input features),
// else MN-major (blocks of 64 output features by 64 input features). Rows and
// features outside the operands arrive as zeros.
//
// stream_kernel: few activation rows. The weights are what has to be read, so
// here they are the 128-row operand and the activations the narrow one (16 to
// 64 columns): a CTA streams 128 output features over its share of the input
// features, a cluster of up to 8 CTAs shares a feature tile, and their partial
// sums meet in distributed shared memory.
#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "proj_common.cuh"
#include "tc_ptx.cuh"

namespace rlt {
namespace proj {
namespace {

constexpr long long kWaitLimit = 100000000LL;  // cycles (~50 ms)
constexpr int kBlockK = 64;                    // input features per stage (128 bytes)
constexpr int kTileM = 128;                    // activation rows per CTA
constexpr int kMaxStages = 8;
constexpr int kThreads = 192;
constexpr int kBytesA = kTileM * kBlockK * 2;
constexpr int kSmemBudget = 200 * 1024;

struct GemmParams {
  CUtensorMap map_x, map_w, map_up;
  Problem p;
  int stages;
  int stage_bytes;
  int box_m;      // activation rows copied per stage (the rest of the tile is never stored)
  int tile_n;     // accumulator columns: output features, or gate then up features
  int load_n;     // weight rows this CTA copies per operand
  int set_n;      // output features per tile
  int w_mn;       // weights MN-major in shared memory
  int row_tiles;
  int col_tiles;
  int vec;        // out (and bias, residual) allow 16-byte access
};

template <typename T>
struct Fmt;
template <>
struct Fmt<__half> {
  static constexpr uint32_t value = 0;
};
template <>
struct Fmt<__nv_bfloat16> {
  static constexpr uint32_t value = 1;
};

// 32 outputs of one row from column n on, up to column `end`: y = act(acc + bias) + residual, or
// act(acc) * up.
template <typename T, Kind kKind, int kAct>
__device__ __forceinline__ void finish32(const Problem& p, int vec, int row, int n, int end,
                                         const uint32_t (&acc)[32], const uint32_t (&up)[32]) {
  const T* bias = static_cast<const T*>(p.bias);
  const T* res = static_cast<const T*>(p.residual);
  T* out = static_cast<T*>(p.out) + row * p.o_rs + n;
  if (res != nullptr) res += row * p.r_rs + n;
  const bool in_row = row < p.rows;
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    float y[8], b[8], r[8];
    const bool whole = vec && n + g * 8 + 8 <= end;
    if (kKind == kLinear && bias != nullptr) {
      if (whole) {
        unpack16<T>(ld_vec(bias + n + g * 8), b);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) b[e] = n + g * 8 + e < end ? to_f32<T>(bias[n + g * 8 + e]) : 0.f;
      }
    }
    if (kKind == kLinear && res != nullptr && in_row) {
      if (whole) {
        unpack16<T>(ld_vec(res + g * 8), r);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] = n + g * 8 + e < end ? to_f32<T>(res[g * 8 + e]) : 0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = __uint_as_float(acc[g * 8 + e]);
      if (kKind == kGated) {
        y[e] = activate<false, kAct>(y[e]) * __uint_as_float(up[g * 8 + e]);
      } else {
        if (bias != nullptr) y[e] += b[e];
        y[e] = activate<false, kAct>(y[e]);
        if (res != nullptr && in_row) y[e] += r[e];
      }
    }
    if (!in_row) continue;
    if (whole) {
      st_vec(out + g * 8, pack16<T>(y));
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (n + g * 8 + e < end) out[g * 8 + e] = from_f32<T>(y[e]);
    }
  }
}

// A row's record of one vocabulary tile, from the accumulator's columns. The
// running maximum and sum move chunk by chunk (32 logits in registers).
__device__ __forceinline__ void vocab_tile_part(const GemmParams& g, uint32_t taddr, int row,
                                                int n0, int tile) {
  const Problem& p = g.p;
  const int cols = min(g.tile_n, p.outer - n0);
  const bool in_row = row < p.rows;
  const int64_t want64 = in_row && p.tokens != nullptr ? p.tokens[row] : -1;
  const int want = want64 >= n0 && want64 < n0 + cols ? static_cast<int>(want64) - n0 : -1;
  VocabPart part{-INFINITY, 0.f, n0, 0.f};
  for (int c = 0; c < cols; c += 32) {
    uint32_t v[32];
    __syncwarp();
    tc::tmem_ld32(taddr + c, v);
    tc::tmem_ld_wait(v);
    const int left = cols - c;
    if (left < 32) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (j >= left) v[j] = __float_as_uint(-INFINITY);
    }
    float m = __uint_as_float(v[0]);
#pragma unroll
    for (int j = 1; j < 32; ++j) m = fmaxf(m, __uint_as_float(v[j]));
    if (m > part.most) {
      if (p.tokens == nullptr) {
        int at = 0;
#pragma unroll
        for (int j = 31; j >= 0; --j)
          if (__uint_as_float(v[j]) == m) at = j;
        part.at = n0 + c + at;
      }
      part.sum *= ex2((part.most - m) * kLog2e);
      part.most = m;
    }
    const float base = part.most == -INFINITY ? 0.f : part.most;
    float s0 = 0.f, s1 = 0.f;
#pragma unroll
    for (int j = 0; j < 32; j += 2) {
      s0 += ex2((__uint_as_float(v[j]) - base) * kLog2e);
      s1 += ex2((__uint_as_float(v[j + 1]) - base) * kLog2e);
    }
    part.sum += s0 + s1;
    if (__any_sync(kFullMask, want >= c && want < c + 32)) {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (want == c + j) part.chosen = __uint_as_float(v[j]);
    }
  }
  // a NaN among the logits counts as the largest: find the first
  if (p.tokens == nullptr && __any_sync(kFullMask, part.sum != part.sum)) {
    for (int c = (cols - 1) / 32 * 32; c >= 0; c -= 32) {
      uint32_t v[32];
      __syncwarp();
      tc::tmem_ld32(taddr + c, v);
      tc::tmem_ld_wait(v);
#pragma unroll
      for (int j = 31; j >= 0; --j) {
        const float l = __uint_as_float(v[j]);
        if (c + j < cols && l != l) {
          part.most = l;
          part.at = n0 + c + j;
        }
      }
    }
  }
  if (in_row) p.parts[static_cast<int64_t>(row) * p.tiles + tile] = part;
}

template <typename T, Kind kKind, int kAct>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmParams g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  const Problem& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));

  if (threadIdx.x == 0) {
    for (int i = 0; i < g.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 4);
    }
    aborted = 0;
    tc::fence_mbar_init();
  }
  if (warp == 5) tc::tmem_alloc(&tmem_slot, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;

  const int kblocks = (p.inner + kBlockK - 1) / kBlockK;
  const int tiles = g.row_tiles * g.col_tiles;
  bool ok = true;

  if (warp == 4) {
    if (lane == 0) {
      const uint32_t bytes = g.box_m * 128 + g.load_n * 128 * (kKind == kGated ? 2 : 1);
      uint32_t it = 0;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x) {
        const int m0 = tile % g.row_tiles * kTileM;
        const int n0 = tile / g.row_tiles * g.set_n;
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % g.stages;
          if (it >= static_cast<uint32_t>(g.stages) &&
              !tc::mbar_wait(&empty[s], (it / g.stages - 1) & 1, kWaitLimit)) {
            ok = false;
            break;
          }
          uint8_t* a = smem + s * g.stage_bytes;
          uint8_t* b = a + kBytesA;
          tc::mbar_expect_tx(&full[s], bytes);
          tc::tma_load_2d(a, &g.map_x, &full[s], kb * kBlockK, m0);
          for (int half = 0; half < (kKind == kGated ? 2 : 1); ++half) {
            const CUtensorMap* map = half ? &g.map_up : &g.map_w;
            uint8_t* dst = b + half * g.load_n * 128;
            if (g.w_mn) {
              for (int n = 0; n < g.load_n; n += 64)
                tc::tma_load_2d(dst + n * 128, map, &full[s], n0 + n, kb * kBlockK);
            } else {
              tc::tma_load_2d(dst, map, &full[s], kb * kBlockK, n0);
            }
          }
        }
      }
    }
  } else if (warp == 5) {
    if (lane == 0) {
      const uint32_t idesc = tc::idesc_f16(Fmt<T>::value, kTileM, g.tile_n, g.w_mn);
      const uint32_t kstep_b = g.w_mn ? 2048 : 32;
      const uint32_t lbo_b = g.w_mn ? 8192 : 16;
      uint32_t it = 0, n = 0;
      for (int tile = blockIdx.x; ok && tile < tiles; tile += gridDim.x, ++n) {
        const uint32_t buf = n & 1;
        if (n >= 2 && !tc::mbar_wait(&acc_empty[buf], (n / 2 - 1) & 1, kWaitLimit)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        for (int kb = 0; kb < kblocks; ++kb, ++it) {
          const int s = it % g.stages;
          if (!tc::mbar_wait(&full[s], (it / g.stages) & 1, kWaitLimit)) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t a = tc::smem_u32(smem + s * g.stage_bytes);
          const uint32_t b = a + kBytesA;
#pragma unroll
          for (int ks = 0; ks < kBlockK / 16; ++ks)
            tc::mma_f16_ss(tmem + buf * 256, tc::smem_desc_sw128(a + ks * 32, 16, 1024),
                           tc::smem_desc_sw128(b + ks * kstep_b, lbo_b, 1024), idesc,
                           kb > 0 || ks > 0);
          tc::mma_commit(&empty[s]);
        }
        if (ok) tc::mma_commit(&acc_full[buf]);
      }
    }
  } else {
    uint32_t n = 0;
    for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x, ++n) {
      const uint32_t buf = n & 1;
      ok = __all_sync(kFullMask, tc::mbar_wait(&acc_full[buf], (n / 2) & 1, kWaitLimit));
      if (!ok) break;
      tc::tc_fence_after();
      const int col_tile = tile / g.row_tiles;
      const int row = tile % g.row_tiles * kTileM + threadIdx.x;
      const int n0 = col_tile * g.set_n;
      const uint32_t taddr = tmem + buf * 256 + (static_cast<uint32_t>(warp) << 21);
      if constexpr (kKind == kVocab) {
        vocab_tile_part(g, taddr, row, n0, col_tile);
      } else {
        const int cols = min(g.set_n, p.outer - n0);
        for (int c = 0; c < cols; c += 32) {
          uint32_t v[32], up[32];
          __syncwarp();
          tc::tmem_ld32(taddr + c, v);
          if constexpr (kKind == kGated) tc::tmem_ld32(taddr + g.set_n + c, up);
          tc::tmem_ld_wait(v);
          if constexpr (kKind == kGated) tc::tmem_ld_wait(up);
          finish32<T, kKind, kAct>(p, g.vec, row, n0 + c, n0 + cols, v, up);
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&acc_empty[buf]);
    }
  }
  if (!ok) {  // a wait ran out: let copies in flight land before the memory goes
    aborted = 1;
    const long long start = clock64();
    while (clock64() - start < 4000000LL) {
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (aborted && threadIdx.x == 0) raise_status(p.status, kStatusTimeout);
  if (warp == 5) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

// ---- few rows -----------------------------------------------------------------

constexpr int kStreamRows = 64;     // activation rows that stream_kernel takes
constexpr int kStreamStages = 12;
constexpr int kStreamFeatures = 128;
constexpr int kMaxSplits = 8;       // CTAs of a cluster (the portable limit)

struct StreamParams {
  CUtensorMap map_x, map_w, map_up;
  Problem p;
  int stages;
  int stage_bytes;
  int cols;    // activation rows rounded up to the instruction's 16
  int w_mn;
  int splits;  // CTAs per feature tile
  int vec;     // four neighbouring outputs are one 8-byte store
};

template <typename T, Kind kKind, int kAct>
__global__ void __launch_bounds__(kThreads) stream_kernel(const __grid_constant__ StreamParams g) {
  constexpr int kOps = kKind == kGated ? 2 : 1;
  constexpr int kBytesW = kStreamFeatures * kBlockK * 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStreamStages], empty[kStreamStages], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  const Problem& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const int rank = g.splits > 1 ? static_cast<int>(tc::cluster_rank()) : 0;
  const int n0 = blockIdx.x / g.splits * kStreamFeatures;
  const int kblocks = (p.inner + kBlockK - 1) / kBlockK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(kblocks) * rank / g.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(kblocks) * (rank + 1) / g.splits);
  constexpr uint32_t kTmemCols = kOps * kStreamRows;  // 64 or 128, powers of two

  if (threadIdx.x == 128) {
    tc::prefetch_tensormap(&g.map_w);
    tc::prefetch_tensormap(&g.map_x);
    if (kOps == 2) tc::prefetch_tensormap(&g.map_up);
    for (int i = 0; i < g.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    tc::mbar_init(&acc_full, 1);
    aborted = 0;
    tc::fence_mbar_init();
  }
  if (warp == 5) tc::tmem_alloc(&tmem_slot, kTmemCols);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp == 4) {
    if (lane == 0) {
      const uint32_t bytes = kOps * kBytesW + g.cols * 128;
      for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
        const int s = it % g.stages;
        if (it >= g.stages && !tc::mbar_wait(&empty[s], (it / g.stages - 1) & 1, kWaitLimit)) {
          ok = false;
          break;
        }
        uint8_t* w = smem + s * g.stage_bytes;
        tc::mbar_expect_tx(&full[s], bytes);
        for (int op = 0; op < kOps; ++op) {
          const CUtensorMap* map = op ? &g.map_up : &g.map_w;
          uint8_t* dst = w + op * kBytesW;
          if (g.w_mn) {
            tc::tma_load_2d(dst, map, &full[s], n0, kb * kBlockK);
            tc::tma_load_2d(dst + 8192, map, &full[s], n0 + 64, kb * kBlockK);
          } else {
            tc::tma_load_2d(dst, map, &full[s], kb * kBlockK, n0);
          }
        }
        tc::tma_load_2d(w + kOps * kBytesW, &g.map_x, &full[s], kb * kBlockK, 0);
      }
    }
  } else if (warp == 5) {
    if (lane == 0) {
      const uint32_t idesc = tc::idesc_f16(Fmt<T>::value, kStreamFeatures, g.cols, 0, g.w_mn);
      const uint32_t kstep_w = g.w_mn ? 2048 : 32;
      const uint32_t lbo_w = g.w_mn ? 8192 : 16;
      for (int kb = kb0, it = 0; kb < kb1; ++kb, ++it) {
        const int s = it % g.stages;
        if (!tc::mbar_wait(&full[s], (it / g.stages) & 1, kWaitLimit)) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t w = tc::smem_u32(smem + s * g.stage_bytes);
        const uint32_t x = w + kOps * kBytesW;
#pragma unroll
        for (int ks = 0; ks < kBlockK / 16; ++ks)
#pragma unroll
          for (int op = 0; op < kOps; ++op)
            tc::mma_f16_ss(tmem + op * kStreamRows,
                           tc::smem_desc_sw128(w + op * kBytesW + ks * kstep_w, lbo_w, 1024),
                           tc::smem_desc_sw128(x + ks * 32, 16, 1024), idesc, it > 0 || ks > 0);
        tc::mma_commit(&empty[s]);
      }
      if (ok) tc::mma_commit(&acc_full);
    }
  }
  __syncwarp();
  float* sums = reinterpret_cast<float*>(smem);  // [op][row][feature], where the stages were
  if (warp < 4) {
    ok = __all_sync(kFullMask, tc::mbar_wait(&acc_full, 0, kWaitLimit));
    tc::tc_fence_after();
    const uint32_t taddr = tmem + (static_cast<uint32_t>(warp) << 21);
    for (int c = 0; ok && c < p.rows; c += 16) {
      float* at = sums + c * kStreamFeatures + threadIdx.x;
#pragma unroll
      for (int op = 0; op < kOps; ++op) {
        uint32_t v[16];
        __syncwarp();
        tc::tmem_ld16(taddr + op * kStreamRows + c, v);
        tc::tmem_ld_wait(v);
#pragma unroll
        for (int j = 0; j < 16; ++j)
          at[(op * g.cols + j) * kStreamFeatures] = __uint_as_float(v[j]);
      }
    }
  }
  if (!ok) {  // a wait ran out: let copies in flight land before the memory goes
    aborted = 1;
    const long long start = clock64();
    while (clock64() - start < 4000000LL) {
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  if (g.splits > 1)
    tc::cluster_sync();
  else
    __syncthreads();
  if (aborted && threadIdx.x == 0) raise_status(p.status, kStatusTimeout);
  if (warp == 5) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, kTmemCols);
  }
  // Each CTA of the cluster finishes every splits-th row, adding in rank order:
  // a warp per row, four neighbouring features per lane.
  const int f0 = lane * 4;
  const int n = n0 + f0;
  if (n < p.outer) {
    const T* res = static_cast<const T*>(p.residual);
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    if (kKind == kLinear && p.bias != nullptr)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < p.outer) b[e] = to_f32<T>(static_cast<const T*>(p.bias)[n + e]);
#pragma unroll 2
    for (int row = rank + warp * g.splits; row < p.rows; row += kThreads / 32 * g.splits) {
      float r[4] = {0.f, 0.f, 0.f, 0.f};
      if (kKind == kLinear && res != nullptr)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.outer) r[e] = to_f32<T>(res[row * p.r_rs + n + e]);
      float y[kOps][4];
#pragma unroll
      for (int op = 0; op < kOps; ++op) {
        const float* mine = sums + (op * g.cols + row) * kStreamFeatures + f0;
        float4 v[kMaxSplits];
#pragma unroll
        for (int s = 0; s < kMaxSplits; ++s)
          if (s < g.splits) v[s] = g.splits > 1 ? tc::ld_peer4(tc::peer_smem(mine, s))
                                                : *reinterpret_cast<const float4*>(mine);
        float4 t = v[0];
#pragma unroll
        for (int s = 1; s < kMaxSplits; ++s)
          if (s < g.splits) {
            t.x += v[s].x;
            t.y += v[s].y;
            t.z += v[s].z;
            t.w += v[s].w;
          }
        y[op][0] = t.x;
        y[op][1] = t.y;
        y[op][2] = t.z;
        y[op][3] = t.w;
      }
      T o[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if constexpr (kKind == kGated)
          o[e] = from_f32<T>(activate<false, kAct>(y[0][e]) * y[1][e]);
        else
          o[e] = from_f32<T>(activate<false, kAct>(y[0][e] + b[e]) + r[e]);
      }
      T* out = static_cast<T*>(p.out) + row * p.o_rs + n;
      if (g.vec) {
        *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(o);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (n + e < p.outer) out[e] = o[e];
      }
    }
  }
  if (g.splits > 1) {
    __syncwarp();
    tc::cluster_sync();  // a peer may still be reading this CTA's sums
  }
}

// ---- host side --------------------------------------------------------------

PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static std::atomic<void*> known{nullptr};
  void* fn = known.load();
  if (fn == nullptr) {
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) !=
            cudaSuccess ||
        q != cudaDriverEntryPointSuccess)
      return nullptr;
    known.store(fn);
  }
  return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
}

// A [lines x line] matrix of 16-bit elements, `stride` elements between lines,
// copied in boxes of 64 elements by `box_lines` lines.
bool encode2d(CUtensorMap* map, int32_t dtype, const void* base, int line, int lines,
              int64_t stride, int box_lines) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(line), static_cast<cuuint64_t>(lines)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * 2};
  const cuuint32_t box[2] = {64, static_cast<cuuint32_t>(box_lines)};
  const cuuint32_t elem[2] = {1, 1};
  return fn(map,
            dtype == RLT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
            2, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Dynamic shared memory of kKernel raised once per device.
template <auto kKernel>
cudaError_t allow_smem(int bytes) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev >= 0 && dev < 64 && done[dev].load()) return cudaSuccess;
  const cudaError_t e =
      cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true);
  return e;
}

template <typename T, Kind kKind, int kAct>
int launch(const GemmParams& g, int ctas, cudaStream_t stream) {
  constexpr auto kernel = gemm_kernel<T, kKind, kAct>;
  if (const cudaError_t e = allow_smem<kernel>(kSmemBudget + 1024)) return static_cast<int>(e);
  kernel<<<ctas, kThreads, g.stages * g.stage_bytes + 1024, stream>>>(g);
  return launch_status(cudaGetLastError());
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Output features per tile: the width whose tiles waste least of the last
// wave of CTAs, the widest among equals. `step`: what the weights' layout asks.
int choose_set(int outer, int row_tiles, int widest, int step, int ctas) {
  int best = widest;
  double least = 1e300;
  for (int n = widest; n >= step; n -= step) {
    const int64_t tiles = static_cast<int64_t>(ceil_div(outer, n)) * row_tiles;
    const int64_t waves = (tiles + ctas - 1) / ctas;
    // a tile's time: its columns plus what every tile pays
    const double cost = static_cast<double>(waves) * (n + 32);
    if (cost < least * 0.999) {
      least = cost;
      best = n;
    }
  }
  return best;
}

template <typename T, Kind kKind, int kAct>
int launch(const StreamParams& g, int tiles, cudaStream_t stream) {
  constexpr auto kernel = stream_kernel<T, kKind, kAct>;
  if (const cudaError_t e = allow_smem<kernel>(kSmemBudget + 1024)) return static_cast<int>(e);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * g.splits));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = g.stages * g.stage_bytes + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = g.splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return launch_status(cudaLaunchKernelEx(&cfg, kernel, g));
}

// The kernel for a launch's type and activation.
template <Kind kKind, typename T, typename Params>
int by_activation(const Params& g, int ctas, cudaStream_t stream) {
  if constexpr (kKind == kVocab) return launch<T, kKind, RLT_ACT_NONE>(g, ctas, stream);
  switch (g.p.act) {
    case RLT_ACT_SILU: return launch<T, kKind, RLT_ACT_SILU>(g, ctas, stream);
    case RLT_ACT_GELU: return launch<T, kKind, RLT_ACT_GELU>(g, ctas, stream);
    case RLT_ACT_GELU_TANH: return launch<T, kKind, RLT_ACT_GELU_TANH>(g, ctas, stream);
    case RLT_ACT_RELU: return launch<T, kKind, RLT_ACT_RELU>(g, ctas, stream);
    case RLT_ACT_SIGMOID: return launch<T, kKind, RLT_ACT_SIGMOID>(g, ctas, stream);
    default: return launch<T, kKind, RLT_ACT_NONE>(g, ctas, stream);
  }
}
template <Kind kKind, typename Params>
int by_type(const Params& g, int32_t dtype, int ctas, cudaStream_t stream) {
  return dtype == RLT_BF16 ? by_activation<kKind, __nv_bfloat16>(g, ctas, stream)
                           : by_activation<kKind, __half>(g, ctas, stream);
}

int run_stream(Kind kind, const Problem& p, int32_t dtype, int ctas, cudaStream_t stream) {
  StreamParams g{};
  const int ops = kind == kGated ? 2 : 1;
  g.p = p;
  g.w_mn = p.w_ks != 1;
  g.cols = ceil_div(p.rows, 16) * 16;
  g.vec = p.outer % 4 == 0 && p.o_rs % 4 == 0 && reinterpret_cast<uintptr_t>(p.out) % 8 == 0;
  g.stage_bytes = ops * kStreamFeatures * kBlockK * 2 + g.cols * 128;
  const int tiles = ceil_div(p.outer, kStreamFeatures);
  const int kblocks = ceil_div(p.inner, kBlockK);
  // a cluster wide enough that the CTAs fill the SMs about twice
  g.splits = 1;
  while (g.splits < kMaxSplits && g.splits < kblocks && tiles * (g.splits + 1) <= 2 * ctas) ++g.splits;
  const int share = ceil_div(kblocks, g.splits);
  // two CTAs fit an SM, so that a cluster finds room whatever the number of
  // SMs its part of the die has
  g.stages = 110 * 1024 / g.stage_bytes;
  if (g.stages > kStreamStages) g.stages = kStreamStages;
  if (g.stages > share) g.stages = share;
  const int sums = ops * g.cols * kStreamFeatures * 4;  // partial sums lie where the stages were
  while (g.stages * g.stage_bytes < sums) ++g.stages;
  bool ok = encode2d(&g.map_x, dtype, p.x, p.inner, p.rows, p.x_rs, g.cols);
  for (int op = 0; op < ops; ++op) {
    CUtensorMap* map = op ? &g.map_up : &g.map_w;
    const void* base = op ? p.w_up : p.w;
    ok = ok && (g.w_mn ? encode2d(map, dtype, base, p.outer, p.inner, p.w_ks, 64)
                       : encode2d(map, dtype, base, p.inner, p.outer, p.w_ns, kStreamFeatures));
  }
  if (!ok) return RLT_E_DEVICE;
  return kind == kGated ? by_type<kGated>(g, dtype, tiles, stream)
                        : by_type<kLinear>(g, dtype, tiles, stream);
}

}  // namespace

int tc_vocab_tile(const Problem& p, int ctas) {
  const bool mn = p.w_ks != 1;
  return choose_set(p.outer, ceil_div(p.rows, kTileM), 256, mn ? 64 : 16, ctas);
}

int run_tc(Kind kind, const Problem& p, int32_t dtype, int ctas, cudaStream_t stream) {
  if (kind != kVocab && p.rows <= kStreamRows) return run_stream(kind, p, dtype, ctas, stream);
  GemmParams g{};
  g.p = p;
  g.w_mn = p.w_ks != 1;
  g.row_tiles = ceil_div(p.rows, kTileM);
  g.box_m = p.rows >= kTileM ? kTileM : ceil_div(p.rows, 8) * 8;
  g.set_n = kind == kVocab ? tc_vocab_tile(p, ctas)
                           : choose_set(p.outer, g.row_tiles, kind == kGated ? 128 : 256,
                                        g.w_mn ? 64 : 16, ctas);
  g.load_n = g.set_n;
  g.tile_n = kind == kGated ? 2 * g.set_n : g.set_n;
  g.col_tiles = ceil_div(p.outer, g.set_n);
  g.stage_bytes = kBytesA + g.tile_n * 128;
  g.stages = kSmemBudget / g.stage_bytes < kMaxStages ? kSmemBudget / g.stage_bytes : kMaxStages;
  g.vec = aligned16(p.out) && p.o_rs % 8 == 0 && (p.bias == nullptr || aligned16(p.bias)) &&
          (p.residual == nullptr || (aligned16(p.residual) && p.r_rs % 8 == 0));
  if (static_cast<int64_t>(g.row_tiles) * g.col_tiles > INT32_MAX) return RLT_E_SHAPE;
  bool ok = encode2d(&g.map_x, dtype, p.x, p.inner, p.rows, p.x_rs, g.box_m);
  for (int half = 0; half < (kind == kGated ? 2 : 1); ++half) {
    CUtensorMap* map = half ? &g.map_up : &g.map_w;
    const void* base = half ? p.w_up : p.w;
    ok = ok && (g.w_mn ? encode2d(map, dtype, base, p.outer, p.inner, p.w_ks, 64)
                       : encode2d(map, dtype, base, p.inner, p.outer, p.w_ns, g.load_n));
  }
  if (!ok) return RLT_E_DEVICE;
  const int tiles = g.row_tiles * g.col_tiles;
  if (tiles < ctas) ctas = tiles;
  switch (kind) {
    case kLinear: return by_type<kLinear>(g, dtype, ctas, stream);
    case kGated: return by_type<kGated>(g, dtype, ctas, stream);
    default: return by_type<kVocab>(g, dtype, ctas, stream);
  }
}

}  // namespace proj
}  // namespace rlt
