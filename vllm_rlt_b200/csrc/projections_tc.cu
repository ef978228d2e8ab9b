// Projections on the tensor cores (bf16, fp16; fp32 accumulation in TMEM).
//
// gemm_kernel: tiles of 128 activation rows by up to 256 weight rows (output
// features), or of 256 by 256 on a pair of CTAs (cta_group::2). A thread of
// warp 8 copies 64-feature slices of both operands into a ring of
// shared-memory stages by TMA (128-byte swizzle), one of warp 9 issues the
// tcgen05.mma, and warps 0-7 turn a finished accumulator into outputs while
// the next one fills the other half of TMEM.
//
// What bounds a tile: 64 input features take 2 N cycles of arithmetic, and an
// SM takes in about 60 bytes a cycle from L2, (128 + N) x 128 bytes for a CTA
// by itself, (128 + N / 2) x 128 for one of a pair (each holds half of the
// weights' slice). At N = 256 that is 819 and 546 cycles against 512, so wide
// tiles on pairs are the ones near the tensor cores' rate: 4096 x 2048 -> 2 x 5632
// takes 127 us, 1,490 TFLOP/s.
//
// A thread of warps 0-7 holds one activation row of the tile (its TMEM lane)
// and half of its columns, so the vocabulary head's maximum and sum need no
// exchange between threads. The tensor core truncates as it accumulates, an
// error of one sign that grows with the number of steps: over 16384 features of
// one sign a sum in TMEM came out 1.07e-4 too small (fp16; bf16 8.2e-5). So at
// most 768 input features are accumulated there (512 for the head, whose outputs
// are fp32), and those sums are added in registers, rounded to nearest: 4e-6 at
// any length. Of 4096 x 5632 -> 2048 in bf16, 5.0e-4 of the outputs then differ
// from the rounded exact ones, as with fp32 products rounded to nearest (4.5e-4),
// and 3.2e-3 did before.
//
// Weights may have either dimension contiguous: with the input features
// contiguous a stage holds them K-major (128-byte rows of 64 input features),
// else MN-major (blocks of 64 output features by 64 input features). Rows and
// features outside the operands arrive as zeros.
//
// stream_kernel: few activation rows. The weights are what has to be read, so
// here they are the 128-row operand and the activations the narrow one (16 to
// 64 columns): a CTA streams 128 output features over its share of the input
// features in TMEM accumulators of some hundred each, a cluster of up to 8 CTAs
// shares a feature tile, and their partial sums meet in distributed shared memory:
// each CTA reads the others' for the rows that it finishes (stored there by the
// others with st.async instead, 64 rows took 9.4 us where reading takes 7.9). While
// the stream's previous kernel still runs, the first weights are brought into L2.
#include <type_traits>

#include "proj_tc.cuh"

namespace rlt {
namespace proj {
namespace {

constexpr int kBlockK = 64;                    // input features per stage (128 bytes)
constexpr int kTileM = 128;                    // activation rows per CTA
constexpr int kMaxStages = 10;
constexpr int kEpilogueWarps = 8;
// Warps 8 and 9 copy and multiply; 10 and 11 complete their warpgroup. The
// epilogue threads hold 128 sums each and take registers from it.
constexpr int kThreads = (kEpilogueWarps + 4) * 32;
constexpr int kLaunchRegs = 168, kSumRegs = 232, kOtherRegs = 40;  // per thread
static_assert(256 * kSumRegs + 128 * kOtherRegs <= kThreads * kLaunchRegs,
              "the increase draws on what the launch allocated");
constexpr int kStagingBytes = kEpilogueWarps * 4096;  // 32 rows x 32 fp32 columns per warp
// 64-feature blocks accumulated in TMEM at a time, by the head and by the others.
// With 8 these would wait for the two accumulators while a tile's outputs are
// stored: 4096 x 5632 -> 2048 takes 78.9 us, the gated product
// 4096 x 2048 -> 2 x 5632 136; with 12, 75.8 and 127; with 16, 73.9 and 124.
constexpr int kSumBlocks = 8, kTileSumBlocks = 12;

struct GemmParams {
  CUtensorMap map_x, map_w, map_up;
  Problem p;
  int stages;
  int stage_bytes;
  int ring_bytes;
  int box_m;      // activation rows copied per stage (the rest of the tile is never stored)
  int tile_n;     // accumulator columns: output features, or gate then up features
  int load_n;     // weight rows this CTA copies per operand
  int set_n;      // output features per tile
  int w_mn;       // weights MN-major in shared memory
  int row_tiles;
  int col_tiles;
  int vec;        // out (and bias, residual) allow 8-byte access
  int pair;       // tiles of 256 rows on pairs of CTAs
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

// Columns n .. n + 31 of a warp's 32 rows, from the threads' registers (one row
// each) to `out`: the values go through shared memory so that neighbouring
// lanes hold neighbouring columns, then y = act(v + bias) + residual. 16-byte
// units are swizzled by row, which keeps both directions free of bank
// conflicts. `end`: columns that exist.
template <typename T, int kAct>
__device__ __forceinline__ void finish32(const Problem& p, int vec, uint8_t* staging, int row0,
                                         int n, int end, const float (&v)[32]) {
  const int lane = threadIdx.x & 31;
  const T* bias = static_cast<const T*>(p.bias);
  const T* res = static_cast<const T*>(p.residual);
  T* out = static_cast<T*>(p.out);
  const int rows = min(32, p.rows - row0);
#pragma unroll
  for (int c = 0; c < 8; ++c)
    *reinterpret_cast<float4*>(staging + lane * 128 + ((c ^ (lane & 7)) << 4)) =
        make_float4(v[c * 4], v[c * 4 + 1], v[c * 4 + 2], v[c * 4 + 3]);
  if (vec && n + 32 <= end) {  // 8 lanes per row, four columns each
    const int c = lane & 7, at = n + c * 4;
    float b[4] = {0.f, 0.f, 0.f, 0.f};
    uint2 r[8];  // the residuals, on their way together
    if (bias != nullptr) load4<T>(bias + at, b);
    if (res != nullptr)  // past the last row, that one's again: a test per load would part them
#pragma unroll
      for (int i = 0; i < 8; ++i)
        r[i] = *reinterpret_cast<const uint2*>(
            res + (row0 + min(i * 4 + (lane >> 3), rows - 1)) * p.r_rs + at);
    __syncwarp();
#pragma unroll
    for (int i0 = 0; i0 < 8; i0 += 4) {
      float4 f[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = (i0 + i) * 4 + (lane >> 3);
        f[i] = *reinterpret_cast<const float4*>(staging + row * 128 + ((c ^ (row & 7)) << 4));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = (i0 + i) * 4 + (lane >> 3);
        float y[4] = {f[i].x, f[i].y, f[i].z, f[i].w};
        float add[4] = {0.f, 0.f, 0.f, 0.f};
        if (res != nullptr) widen4<T>(r[i0 + i], add);
        T o[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[e] = from_f32<T>(activate<false, kAct>(y[e] + b[e]) + add[e]);
        if (row < rows)
          *reinterpret_cast<uint2*>(out + (row0 + row) * p.o_rs + at) = *reinterpret_cast<uint2*>(o);
      }
    }
  } else {  // one column per lane
    __syncwarp();
    if (n + lane < end) {
      const int at = n + lane;
      const float b = bias != nullptr ? to_f32<T>(bias[at]) : 0.f;
      for (int row = 0; row < rows; row += 16) {
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
          y[i] = res != nullptr && row + i < rows ? to_f32<T>(res[(row0 + row + i) * p.r_rs + at])
                                                  : 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float f = *reinterpret_cast<const float*>(
              staging + (row + i) * 128 + (((lane >> 2) ^ (i & 7)) << 4) + (lane & 3) * 4);
          y[i] += activate<false, kAct>(f + b);
        }
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (row + i < rows) out[(row0 + row + i) * p.o_rs + at] = from_f32<T>(y[i]);
      }
    }
  }
  __syncwarp();
}

template <typename T, Kind kKind, int kAct, bool kPair>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ GemmParams g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  constexpr int kCtas = kPair ? 2 : 1;
  const Problem& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = kPair ? static_cast<int>(tc::cluster_rank()) : 0;
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* ring = smem + kStagingBytes;

  if (threadIdx.x == 0) {
    tc::prefetch_tensormap(&g.map_x);
    tc::prefetch_tensormap(&g.map_w);
    if (kKind == kGated) tc::prefetch_tensormap(&g.map_up);
    for (int i = 0; i < g.stages; ++i) {
      tc::mbar_init(&full[i], 1);
      tc::mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], kEpilogueWarps * kCtas);
    }
    aborted = 0;
    tc::fence_mbar_init();
  }
  __syncwarp();  // the cluster's barrier wants whole warps
  if (warp == kEpilogueWarps + 1) {
    if (kPair)
      tc::tmem_alloc_pair(&tmem_slot, 512);
    else
      tc::tmem_alloc(&tmem_slot, 512);
  }
  tc::tc_fence_before();
  if (kPair)
    tc::cluster_sync();
  else
    __syncthreads();
  tc::tc_fence_after();
  tc::pdl_launch_dependents();
  tc::pdl_wait();
  const uint32_t tmem = tmem_slot;

  const int kblocks = (p.inner + kBlockK - 1) / kBlockK;
  const int tiles = g.row_tiles * g.col_tiles;
  constexpr int kPerAcc = kKind == kVocab ? kSumBlocks : kTileSumBlocks;
  const int first = blockIdx.x / kCtas, step = gridDim.x / kCtas;
  bool ok = true;

  if (warp >= kEpilogueWarps) {
    tc::setmaxnreg_dec<kOtherRegs>();
    if (warp == kEpilogueWarps) {
      const bool both = kKind == kGated && !kPair;  // this CTA copies gate and up rows
      const uint32_t bytes = (g.box_m + g.load_n * (both ? 2 : 1)) * 128 * kCtas;
      const int shift = kPair && kKind != kGated ? rank * g.load_n : 0;
      const CUtensorMap* map_b = kPair && kKind == kGated && rank == 1 ? &g.map_up : &g.map_w;
      auto load = [&](uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
        if (kPair)
          tc::tma_load_2d_pair(dst, map, bar, c0, c1);
        else
          tc::tma_load_2d(dst, map, bar, c0, c1);
      };
      Ring at;
      for (int tile = first; ok && tile < tiles; tile += step) {
        const int m0 = (tile % g.row_tiles * kCtas + rank) * kTileM;
        const int n0 = tile / g.row_tiles * g.set_n + shift;
        for (int k0 = 0; k0 < p.inner; k0 += kBlockK, at.next(g.stages)) {
          // a fresh barrier's earlier phase counts as complete
          if (!__all_sync(kFullMask, tc::mbar_wait(&empty[at.slot], at.parity ^ 1, kWaitLimit))) {
            ok = false;
            break;
          }
          if (tc::elect_one()) {
            uint64_t* bar = &full[at.slot];
            uint8_t* a = ring + at.slot * g.stage_bytes;
            uint8_t* b = a + g.box_m * 128;
            // the pair's copies all complete on the first CTA's barrier
            if (rank == 0) tc::mbar_expect_tx(bar, bytes);
            load(a, &g.map_x, bar, k0, m0);
            if (g.w_mn) {
              for (int n = 0; n < g.load_n; n += 64) load(b + n * 128, map_b, bar, n0 + n, k0);
              if (both)
                for (int n = 0; n < g.load_n; n += 64)
                  load(b + (g.load_n + n) * 128, &g.map_up, bar, n0 + n, k0);
            } else {
              load(b, map_b, bar, k0, n0);
              if (both) load(b + g.load_n * 128, &g.map_up, bar, k0, n0);
            }
          }
          __syncwarp();
        }
      }
    }
    if (warp == kEpilogueWarps + 1 && rank == 0) {
      const uint32_t idesc = tc::idesc_f16(Fmt<T>::value, kTileM * kCtas, g.tile_n, g.w_mn);
      const uint32_t kstep_b = (g.w_mn ? 2048 : 32) >> 4;  // in the descriptors' 16-byte units
      const uint64_t a_desc = tc::smem_desc_sw128(tc::smem_u32(ring), 16, 1024);
      const uint64_t b_desc =
          tc::smem_desc_sw128(tc::smem_u32(ring) + g.box_m * 128, g.w_mn ? 8192 : 16, 1024);
      const uint32_t a_hi = static_cast<uint32_t>(a_desc >> 32);
      const uint32_t b_hi = static_cast<uint32_t>(b_desc >> 32);
      const uint32_t stage_units = g.stage_bytes >> 4;
      Ring at, acc;
      for (int tile = first; ok && tile < tiles; tile += step) {
        for (int kb = 0; ok && kb < kblocks; acc.next(2)) {
          if (!__all_sync(kFullMask,
                          tc::mbar_poll(&acc_empty[acc.slot], acc.parity ^ 1, kWaitLimit))) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          const uint32_t d = tmem + acc.slot * 256;
          const int kb_end = min(kb + kPerAcc, kblocks);
          for (uint32_t more = 0; kb < kb_end; ++kb, at.next(g.stages)) {
            if (!__all_sync(kFullMask, tc::mbar_poll(&full[at.slot], at.parity, kWaitLimit))) {
              ok = false;
              break;
            }
            tc::tc_fence_after();
            if (tc::elect_one()) {
              const uint32_t a_lo = static_cast<uint32_t>(a_desc) + at.slot * stage_units;
              const uint32_t b_lo = static_cast<uint32_t>(b_desc) + at.slot * stage_units;
#pragma unroll
              for (int ks = 0; ks < kBlockK / 16; ++ks) {
                const uint64_t ad = tc::desc64(a_lo + ks * 2, a_hi);
                const uint64_t bd = tc::desc64(b_lo + ks * kstep_b, b_hi);
                if (kPair)
                  tc::mma_f16_ss_pair(d, ad, bd, idesc, ks > 0 ? 1 : more);
                else
                  tc::mma_f16_ss(d, ad, bd, idesc, ks > 0 ? 1 : more);
              }
              if (kPair)
                tc::mma_commit_pair(&empty[at.slot]);
              else
                tc::mma_commit(&empty[at.slot]);
              if (kb == kb_end - 1) {
                if (kPair)
                  tc::mma_commit_pair(&acc_full[acc.slot]);
                else
                  tc::mma_commit(&acc_full[acc.slot]);
              }
            }
            more = 1;
            __syncwarp();
          }
        }
      }
    }
  } else {
    tc::setmaxnreg_inc<kSumRegs>();
    uint8_t* staging = smem + warp * 4096;
    const int half = warp >> 2;  // this thread's columns
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;
    uint32_t n = 0;
    auto wait_acc = [&]() {
      ok = __all_sync(kFullMask,
                      tc::mbar_wait(&acc_full[n & 1], (n / 2) & 1, whole_sum_limit(kPerAcc)));
      tc::tc_fence_after();
      return ok;
    };
    auto release_acc = [&]() {
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (kPair)
          tc::mbar_arrive_at(&acc_empty[n & 1], 0);
        else
          tc::mbar_arrive(&acc_empty[n & 1]);
      }
      ++n;
    };
    for (int tile = first; ok && tile < tiles; tile += step) {
      const int col_tile = tile / g.row_tiles;
      const int row0 = (tile % g.row_tiles * kCtas + rank) * kTileM + (warp & 3) * 32;
      const int n0 = col_tile * g.set_n;
      if constexpr (kKind == kVocab) {
        const int mine = g.tile_n / 2;  // a multiple of 16, at most 128
        float v[128];
        for (int kb = 0; kb < kblocks; kb += kSumBlocks) {
          if (!wait_acc()) break;
          const uint32_t taddr = tmem + (n & 1) * 256 + lanes + half * mine;
#pragma unroll
          for (int c = 0; c < 128; c += 16) {
            if (c < mine) {
              uint32_t t[16];
              tc::tmem_ld16(taddr + c, t);
              tc::tmem_ld_wait(t);
#pragma unroll
              for (int j = 0; j < 16; ++j)
                v[c + j] = kb == 0 ? __uint_as_float(t[j]) : v[c + j] + __uint_as_float(t[j]);
            }
          }
          release_acc();
        }
        if (!ok) break;
        const int row = row0 + lane, at = n0 + half * mine;
        const int64_t want = p.tokens != nullptr && row < p.rows ? p.tokens[row] : -1;
        const VocabPart part = vocab_part(p, v, at, min(mine, p.outer - at), want);
        if (row < p.rows)
          *reinterpret_cast<float4*>(
              &p.parts[static_cast<int64_t>(row) * p.tiles + col_tile * 2 + half]) =
              make_float4(part.most, part.sum, __int_as_float(part.at), part.chosen);
      } else {
        // chunks of 32 features 64 apart: four of them, or two of gate and two of up
        constexpr int kChunks = kKind == kGated ? 2 : 4;
        const int end = min(p.outer, n0 + g.set_n);
        const int cols = row0 < p.rows ? end - n0 : 0;
        float v[4][32];
        for (int kb = 0; kb < kblocks; kb += kPerAcc) {
          if (!wait_acc()) break;
          const uint32_t taddr = tmem + (n & 1) * 256 + lanes;
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const int c = half * 32 + j % kChunks * 64;
            if (c < cols) {
              __syncwarp();
#pragma unroll
              for (int i0 = 0; i0 < 32; i0 += 16) {
                uint32_t t[16];
                tc::tmem_ld16(taddr + j / kChunks * g.set_n + c + i0, t);
                tc::tmem_ld_wait(t);
#pragma unroll
                for (int i = 0; i < 16; ++i)
                  v[j][i0 + i] =
                      kb == 0 ? __uint_as_float(t[i]) : v[j][i0 + i] + __uint_as_float(t[i]);
              }
            }
          }
          release_acc();
        }
        if (!ok) break;
        // one copy of the code that finishes a chunk (unrolled, its instructions
        // take longer to arrive than to run): the sums move up instead
#pragma unroll 1
        for (int c = half * 32; c < cols; c += 64) {
          if constexpr (kKind == kGated) {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              v[0][i] = activate<false, kAct>(v[0][i]) * v[kChunks][i];
            finish32<T, RLT_ACT_NONE>(p, g.vec, staging, row0, n0 + c, end, v[0]);
          } else {
            finish32<T, kAct>(p, g.vec, staging, row0, n0 + c, end, v[0]);
          }
#pragma unroll
          for (int j = 0; j < 3; ++j)
#pragma unroll
            for (int i = 0; i < 32; ++i) v[j][i] = v[j + 1][i];
        }
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
  if (kPair)
    tc::cluster_sync();
  else
    __syncthreads();
  if (aborted && threadIdx.x == 0) raise_status(p.status, kStatusTimeout);
  if (warp == kEpilogueWarps + 1) {
    tc::tc_fence_after();
    if (kPair)
      tc::tmem_dealloc_pair(tmem, 512);
    else
      tc::tmem_dealloc(tmem, 512);
  }
}

// ---- few rows -----------------------------------------------------------------

// Warps 0-3 move sums out of TMEM, 4 copies, 5 multiplies, and all finish rows:
// twelve, so that at 64 rows and a cluster of six or more each has one row.
constexpr int kStreamThreads = 384;
constexpr int kStreamRows = 64;     // activation rows that stream_kernel takes
constexpr int kStreamStages = 12;
constexpr int kStreamFeatures = 128;
constexpr int kStreamTmem = 256;    // columns of a CTA: its accumulators

constexpr int kStreamAhead = 16;  // blocks of weights brought into L2 ahead of time

struct StreamParams {
  CUtensorMap map_x, map_w, map_up;
  Problem p;
  int stages;
  int stage_bytes;
  int cols;    // activation rows rounded up to the instruction's 16
  int w_mn;
  int splits;  // CTAs per feature tile
  int smem_bytes;
  int vec;     // four neighbouring outputs (biases, residuals) are 8 aligned bytes
  int several;     // whether a CTA's share takes more than one accumulator
  int acc_blocks;  // blocks per accumulator
  int acc_cols;    // TMEM columns between a product's accumulators
};

// kSums: a CTA's share takes more than one accumulator. (As a test within one
// kernel it cost 64 rows with a single one 6 %.)
template <typename T, Kind kKind, int kAct, bool kSums>
__global__ void __launch_bounds__(kStreamThreads) stream_kernel(const __grid_constant__ StreamParams g) {
  constexpr int kOps = kKind == kGated ? 2 : 1;
  constexpr int kBytesW = kStreamFeatures * kBlockK * 2;
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[kStreamStages], empty[kStreamStages], acc_full;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  const Problem& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = align_1024(smem_raw);
  const int rank = g.splits > 1 ? static_cast<int>(tc::cluster_rank()) : 0;
  const int n0 = blockIdx.x / g.splits * kStreamFeatures;
  const int kblocks = (p.inner + kBlockK - 1) / kBlockK;
  const int kb0 = static_cast<int>(static_cast<int64_t>(kblocks) * rank / g.splits);
  const int kb1 = static_cast<int>(static_cast<int64_t>(kblocks) * (rank + 1) / g.splits);

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
  __syncwarp();
  if (warp == 5) tc::tmem_alloc(&tmem_slot, kStreamTmem);
  if (warp == 4 && tc::elect_one()) {
    for (int kb = kb0; kb < min(kb1, kb0 + kStreamAhead); ++kb)
#pragma unroll
      for (int op = 0; op < kOps; ++op) {
        const CUtensorMap* map = op ? &g.map_up : &g.map_w;
        if (g.w_mn) {
          tc::tma_prefetch_2d(map, n0, kb * kBlockK);
          tc::tma_prefetch_2d(map, n0 + 64, kb * kBlockK);
        } else {
          tc::tma_prefetch_2d(map, kb * kBlockK, n0);
        }
      }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  tc::pdl_launch_dependents();
  tc::pdl_wait();
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp == 4) {
    const uint32_t bytes = kOps * kBytesW + g.cols * 128;
    Ring at;
    for (int kb = kb0; kb < kb1; ++kb, at.next(g.stages)) {
      if (!__all_sync(kFullMask, tc::mbar_wait(&empty[at.slot], at.parity ^ 1, kWaitLimit))) {
        ok = false;
        break;
      }
      if (tc::elect_one()) {
        uint64_t* bar = &full[at.slot];
        uint8_t* w = smem + at.slot * g.stage_bytes;
        tc::mbar_expect_tx(bar, bytes);
#pragma unroll
        for (int op = 0; op < kOps; ++op) {
          const CUtensorMap* map = op ? &g.map_up : &g.map_w;
          uint8_t* dst = w + op * kBytesW;
          if (g.w_mn) {
            tc::tma_load_2d(dst, map, bar, n0, kb * kBlockK);
            tc::tma_load_2d(dst + 8192, map, bar, n0 + 64, kb * kBlockK);
          } else {
            tc::tma_load_2d(dst, map, bar, kb * kBlockK, n0);
          }
        }
        tc::tma_load_2d(w + kOps * kBytesW, &g.map_x, bar, kb * kBlockK, 0);
      }
      __syncwarp();
    }
  } else if (warp == 5) {
    const uint32_t idesc = tc::idesc_f16(Fmt<T>::value, kStreamFeatures, g.cols, 0, g.w_mn);
    const uint32_t kstep_w = (g.w_mn ? 2048 : 32) >> 4;  // in 16-byte units
    const uint64_t w_desc = tc::smem_desc_sw128(tc::smem_u32(smem), g.w_mn ? 8192 : 16, 1024);
    const uint64_t x_desc = tc::smem_desc_sw128(tc::smem_u32(smem) + kOps * kBytesW, 16, 1024);
    const uint32_t w_hi = static_cast<uint32_t>(w_desc >> 32);
    const uint32_t x_hi = static_cast<uint32_t>(x_desc >> 32);
    Ring at;
    uint32_t d = tmem, more = 0;
    int next_acc = kb0 + g.acc_blocks;
    for (int kb = kb0; kb < kb1; ++kb, at.next(g.stages)) {
      if (!__all_sync(kFullMask, tc::mbar_poll(&full[at.slot], at.parity, kWaitLimit))) {
        ok = false;
        break;
      }
      if (kSums && kb == next_acc) {
        next_acc += g.acc_blocks;
        d += g.acc_cols;
        more = 0;
      }
      tc::tc_fence_after();
      if (tc::elect_one()) {
        const uint32_t w_lo = static_cast<uint32_t>(w_desc) + at.slot * (g.stage_bytes >> 4);
        const uint32_t x_lo = static_cast<uint32_t>(x_desc) + at.slot * (g.stage_bytes >> 4);
#pragma unroll
        for (int ks = 0; ks < kBlockK / 16; ++ks)
#pragma unroll
          for (int op = 0; op < kOps; ++op)
            tc::mma_f16_ss(d + op * (kStreamTmem / kOps),
                           tc::desc64(w_lo + op * (kBytesW >> 4) + ks * kstep_w, w_hi),
                           tc::desc64(x_lo + ks * 2, x_hi), idesc, ks > 0 ? 1 : more);
        tc::mma_commit(&empty[at.slot]);
        if (kb == kb1 - 1) tc::mma_commit(&acc_full);
      }
      more = 1;
      __syncwarp();
    }
  }
  __syncwarp();
  // What this thread's first row is finished with is on its way meanwhile.
  const int n = n0 + lane * 4;
  const int row_first = rank + warp * g.splits, row_step = kStreamThreads / 32 * g.splits;
  const T* res = static_cast<const T*>(p.residual);
  const T* bias = static_cast<const T*>(p.bias);
  auto residual = [&](int row, float (&r)[4]) {
    read4<T>(res != nullptr && n < p.outer && row < p.rows ? res + row * p.r_rs + n : nullptr,
             g.vec, p.outer - n, r);
  };
  float b[4], r[4];
  read4<T>(bias != nullptr && n < p.outer ? bias + n : nullptr, g.vec, p.outer - n, b);
  residual(row_first, r);
  float* sums = reinterpret_cast<float*>(smem);  // [op][row][feature], where the stages were
  if (warp < 4) {
    ok = __all_sync(kFullMask, tc::mbar_wait(&acc_full, 0, whole_sum_limit(kb1 - kb0)));
    tc::tc_fence_after();
    const uint32_t taddr = tmem + (static_cast<uint32_t>(warp) << 21);
    auto gather = [&](uint32_t from, auto add) {
      for (int c = 0; ok && c < p.rows; c += 16) {
        float* at = sums + c * kStreamFeatures + threadIdx.x;
#pragma unroll
        for (int op = 0; op < kOps; ++op) {
          uint32_t v[16];
          __syncwarp();
          tc::tmem_ld16(from + op * (kStreamTmem / kOps) + c, v);
          tc::tmem_ld_wait(v);
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            float* to = at + (op * g.cols + j) * kStreamFeatures;
            *to = add() ? *to + __uint_as_float(v[j]) : __uint_as_float(v[j]);
          }
        }
      }
    };
    gather(taddr, std::false_type());
    if constexpr (kSums)
      for (int a = 1; a * g.acc_blocks < kb1 - kb0; ++a)
        gather(taddr + a * g.acc_cols, std::true_type());
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
    tc::tmem_dealloc(tmem, kStreamTmem);
  }
  // Each CTA of the cluster finishes every splits-th row, adding in rank order:
  // a warp per row, four neighbouring features per lane. A warp that has read
  // its last row lets the peers go before it turns the sums into outputs.
  bool arrived = false;
  for (int row = row_first; row < p.rows; row += row_step) {
    float y[kOps][4];
#pragma unroll
    for (int op = 0; op < kOps; ++op) {
      const float* mine = sums + (op * g.cols + row) * kStreamFeatures + lane * 4;
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
    if (g.splits > 1 && row + row_step >= p.rows) {
      float all = y[0][0] + y[0][1] + y[0][2] + y[0][3];
      if (kOps == 2) all += y[kOps - 1][0] + y[kOps - 1][1] + y[kOps - 1][2] + y[kOps - 1][3];
      __syncwarp();
      tc::cluster_arrive(all);
      arrived = true;
    }
    if constexpr (kKind == kVocab) {
      vocab_row(p, y[0], row, n, n0 / kStreamFeatures);
    } else {
      float next[4];
      residual(row + row_step, next);
      if (n < p.outer) finish4<T, kKind, kAct>(p, g.vec, row, n, y[0], y[kOps - 1], b, r);
#pragma unroll
      for (int e = 0; e < 4; ++e) r[e] = next[e];
    }
  }
  __syncwarp();
  if (g.splits > 1) {
    if (!arrived) tc::cluster_arrive(0.f);
    tc::cluster_wait();  // a peer may still be reading this CTA's sums
  }
}

// ---- host side --------------------------------------------------------------

template <typename T, Kind kKind, int kAct>
int launch(const GemmParams& g, int ctas, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = kStagingBytes + g.ring_bytes + 1024;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  cfg.attrs = attrs;
  cfg.numAttrs = launch_attributes(attrs, g.pair ? 2 : 1);
  if (g.pair) {
    constexpr auto kernel = gemm_kernel<T, kKind, kAct, true>;
    if (const cudaError_t e = allow_smem<kernel>(kSmemBudget, kLaunchRegs)) return static_cast<int>(e);
    return launch_status(cudaLaunchKernelEx(&cfg, kernel, g));
  }
  constexpr auto kernel = gemm_kernel<T, kKind, kAct, false>;
  if (const cudaError_t e = allow_smem<kernel>(kSmemBudget, kLaunchRegs)) return static_cast<int>(e);
  return launch_status(cudaLaunchKernelEx(&cfg, kernel, g));
}

// How gemm_kernel tiles a problem: output features per tile, and whether a
// tile is a pair of CTAs' (256 rows) or one CTA's (128).
struct Tiling {
  int set_n;
  bool pair;
};

// The tiling that a model of a tile's cycles says is fastest. Per 64 input
// features a tile of N columns takes 2 N cycles of arithmetic, and its copies
// arrive at about 60 bytes a cycle from L2, or 35 where all SMs stream weights
// that are read once (one row tile). Tiles run in waves; each pays a start, and
// the last wave's epilogue is exposed.
Tiling choose_tiling(Kind kind, const Problem& p, int ctas) {
  const int per = kind == kGated ? 2 : 1;
  const bool mn = p.w_ks != 1;
  const double kblocks = ceil_div(p.inner, kBlockK);
  Tiling best{256 / per, false};
  double least = 1e300;
  for (int pair = p.rows > kTileM ? 1 : 0; pair >= 0; --pair) {
    const int64_t row_tiles = ceil_div(p.rows, pair ? 2 * kTileM : kTileM);
    // a pair's CTAs copy half of B each: whole 64-feature blocks MN-major
    const int finest = mn ? (pair && per == 1 ? 128 : 64) : 32 / per;
    const int workers = pair ? ctas / 2 : ctas;
    for (int set = 256 / per; set >= finest; set -= finest) {
      const int n = set * per;
      const int64_t tiles = row_tiles * ceil_div(p.outer, set);
      const double waves = static_cast<double>((tiles + workers - 1) / workers);
      const int box = p.rows < kTileM ? p.rows : kTileM;
      const double rate = row_tiles == 1 && tiles > workers / 2 ? 35.0 : 60.0;
      const double copies = (box + (pair ? n / 2 : n)) * 128 / rate;
      const double cycles = copies > 2.0 * n ? copies : 2.0 * n;
      // a warp finishes every other chunk of 32 columns
      const double cost = waves * (kblocks * cycles + 600) + ceil_div(n, 64) * 1500;
      if (cost < least * 0.999) {
        least = cost;
        best = Tiling{set, pair == 1};
      }
    }
  }
  return best;
}

template <typename T, Kind kKind, int kAct>
int launch(const StreamParams& g, int tiles, cudaStream_t stream) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * g.splits));
  cfg.blockDim = dim3(kStreamThreads);
  cfg.dynamicSmemBytes = g.smem_bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  cfg.attrs = attrs;
  cfg.numAttrs = launch_attributes(attrs, g.splits);
  if (g.several) {
    constexpr auto kernel = stream_kernel<T, kKind, kAct, true>;
    if (const cudaError_t e = allow_smem<kernel>(kSmemBudget)) return static_cast<int>(e);
    return launch_status(cudaLaunchKernelEx(&cfg, kernel, g));
  }
  constexpr auto kernel = stream_kernel<T, kKind, kAct, false>;
  if (const cudaError_t e = allow_smem<kernel>(kSmemBudget)) return static_cast<int>(e);
  return launch_status(cudaLaunchKernelEx(&cfg, kernel, g));
}

template <Kind kKind, typename Params>
int by_type(const Params& g, int32_t dtype, int ctas, cudaStream_t stream) {
  return dtype == RLT_BF16 ? by_activation<kKind, __nv_bfloat16>(g, ctas, stream)
                           : by_activation<kKind, __half>(g, ctas, stream);
}

struct StreamPlan {
  int splits;  // CTAs per tile
  int budget;  // shared memory of a CTA's stages
};

StreamPlan stream_plan(const Problem& p, int ctas) {
  const int tiles = ceil_div(p.outer, kStreamFeatures);
  const int kblocks = ceil_div(p.inner, kBlockK);
  StreamPlan plan{1, 110 * 1024};
  // CTAs per tile and shared memory per CTA: the least weights per SM, where
  // either one CTA of 200 KB runs on an SM (its clusters then have to fit the
  // die's parts) or two of 110 KB. The partial sums of many rows cost more to
  // exchange in wide clusters: at 64 rows 3 x 200 KB takes 14.1 us for the gated
  // product and 6 x 110 KB 15.9, while one row takes 11.6 and 10.9; 64 rows of
  // 2048 x 2048 take 6.9 us with 6 x 200 KB and 7.6 with 8 x 110 KB. The border at
  // 16 rows lies between those sizes.
  const bool many = p.rows > 16;
  constexpr int kBig = 200 * 1024, kSmall = 110 * 1024;
  double least = 1e300;
  for (int s = 1; s <= kMaxSplits && s <= kblocks; ++s) {
    for (int big = 0; big < 2; ++big) {
      constexpr auto kernel = stream_kernel<__half, kLinear, RLT_ACT_NONE, false>;
      int waves;
      if (big) {
        if (s > 6) continue;
        const int at_once = s == 1 ? ctas : resident_clusters<kernel>(s, kStreamThreads, kBig);
        if (s > 1 && tiles > at_once) continue;
        waves = ceil_div(tiles, at_once);
      } else {
        if (s > 1 && tiles * s > 2 * ctas) continue;
        waves = ceil_div(tiles * s, ctas);
      }
      const double cost = static_cast<double>(waves) / s * (big == many ? 1.0 : 1.5);
      if (cost < least * (many ? 0.999 : 1.001)) {
        least = cost;
        plan.splits = s;
        plan.budget = big ? kBig : kSmall;
      }
    }
  }
  return plan;
}

// Blocks that an accumulator takes, and the columns between accumulators.
int stream_acc_blocks(Kind kind) { return kind == kVocab ? kSumBlocks : kTileSumBlocks; }
int stream_acc_cols(const Problem& p) { return p.rows <= 16 ? 16 : p.rows <= 32 ? 32 : 64; }

// Whether few rows stream. Their CTA's share of the input features has to fit
// its accumulators; the vocabulary head, whose tiles are many, streams where a
// share is at most half as many again as one holds.
bool streams(Kind kind, const Problem& p, int ctas) {
  if (p.rows > kStreamRows) return false;
  const int share = ceil_div(ceil_div(p.inner, kBlockK), stream_plan(p, ctas).splits);
  if (kind == kVocab) return share <= kSumBlocks + kSumBlocks / 2;
  const int accs = kStreamTmem / (kind == kGated ? 2 : 1) / stream_acc_cols(p);
  return share <= accs * stream_acc_blocks(kind);
}

int run_stream(Kind kind, const Problem& p, int32_t dtype, int ctas, cudaStream_t stream) {
  StreamParams g{};
  const int ops = kind == kGated ? 2 : 1;
  g.p = p;
  g.w_mn = p.w_ks != 1;
  g.cols = ceil_div(p.rows, 16) * 16;
  g.vec = p.outer % 4 == 0 && p.o_rs % 4 == 0 && p.r_rs % 4 == 0 && aligned_to(p.out, 8) &&
          aligned_to(p.bias, 8) && aligned_to(p.residual, 8);
  g.stage_bytes = ops * kStreamFeatures * kBlockK * 2 + g.cols * 128;
  const int tiles = ceil_div(p.outer, kStreamFeatures);
  const StreamPlan plan = stream_plan(p, ctas);
  g.splits = plan.splits;
  const int kblocks = ceil_div(p.inner, kBlockK);
  const int per_cta = ceil_div(kblocks, g.splits);
  const int accs = ceil_div(per_cta, stream_acc_blocks(kind));
  g.several = accs > 1;
  g.acc_blocks = ceil_div(per_cta, accs);
  g.acc_cols = stream_acc_cols(p);
  g.stages = plan.budget / g.stage_bytes;
  // The whole class even where less is used. CTAs of a cluster wait for one
  // another, and TMEM is handed out as it comes: were more CTAs on an SM than its
  // TMEM has room for, two clusters could each hold what the other waits for.
  // With 110 KB two of these CTAs fit (256 columns each), and none beside a
  // cluster that takes all of TMEM, which asks for more than the other half.
  g.smem_bytes = plan.budget + 1024;
  if (g.stages > kStreamStages) g.stages = kStreamStages;
  if (g.stages > per_cta) g.stages = per_cta;
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
  switch (kind) {
    case kLinear: return by_type<kLinear>(g, dtype, tiles, stream);
    case kGated: return by_type<kGated>(g, dtype, tiles, stream);
    default: return by_type<kVocab>(g, dtype, tiles, stream);
  }
}

}  // namespace

int tc_vocab_parts(const Problem& p, int ctas) {
  if (streams(kVocab, p, ctas)) return ceil_div(p.outer, kStreamFeatures);
  return 2 * ceil_div(p.outer, choose_tiling(kVocab, p, ctas).set_n);
}

int run_tc(Kind kind, const Problem& p, int32_t dtype, int ctas, cudaStream_t stream) {
  if (streams(kind, p, ctas))
    return run_stream(kind, p, dtype, ctas, stream);
  GemmParams g{};
  g.p = p;
  const Tiling tiling = choose_tiling(kind, p, ctas);
  g.pair = tiling.pair;
  g.set_n = tiling.set_n;
  g.w_mn = p.w_ks != 1;
  g.row_tiles = ceil_div(p.rows, g.pair ? 2 * kTileM : kTileM);
  g.box_m = p.rows >= kTileM ? kTileM : ceil_div(p.rows, 8) * 8;
  g.tile_n = kind == kGated ? 2 * g.set_n : g.set_n;
  g.load_n = g.pair ? g.tile_n / 2 : g.set_n;
  g.col_tiles = ceil_div(p.outer, g.set_n);
  g.stage_bytes = (g.box_m + (g.pair ? g.load_n : g.tile_n)) * 128;
  // the tensor core reads 128 rows of A whatever was copied: past the last
  // stage's end that is still inside the ring
  g.stages = (kSmemBudget - kStagingBytes - 1024 - (kTileM - g.box_m) * 128) / g.stage_bytes;
  if (g.stages > kMaxStages) g.stages = kMaxStages;
  g.ring_bytes = g.stages * g.stage_bytes + (kTileM - g.box_m) * 128;
  g.vec = aligned_to(p.out, 8) && p.o_rs % 4 == 0 && aligned_to(p.bias, 8) && aligned_to(p.residual, 8) &&
          p.r_rs % 4 == 0;
  // a CTA's count of tiles steps past the last
  if (static_cast<int64_t>(g.row_tiles) * g.col_tiles > RLT_PROJ_MAX_SIZE) return RLT_E_SHAPE;
  bool ok = encode2d(&g.map_x, dtype, p.x, p.inner, p.rows, p.x_rs, g.box_m);
  for (int half = 0; half < (kind == kGated ? 2 : 1); ++half) {
    CUtensorMap* map = half ? &g.map_up : &g.map_w;
    const void* base = half ? p.w_up : p.w;
    ok = ok && (g.w_mn ? encode2d(map, dtype, base, p.outer, p.inner, p.w_ks, 64)
                       : encode2d(map, dtype, base, p.inner, p.outer, p.w_ns, g.load_n));
  }
  if (!ok) return RLT_E_DEVICE;
  const int tiles = g.row_tiles * g.col_tiles;
  if (g.pair) ctas = ctas / 2 < tiles ? ctas / 2 * 2 : tiles * 2;
  if (tiles < ctas) ctas = g.pair ? ctas : tiles;
  switch (kind) {
    case kLinear: return by_type<kLinear>(g, dtype, ctas, stream);
    case kGated: return by_type<kGated>(g, dtype, ctas, stream);
    default: return by_type<kVocab>(g, dtype, ctas, stream);
  }
}

}  // namespace proj
}  // namespace rlt
