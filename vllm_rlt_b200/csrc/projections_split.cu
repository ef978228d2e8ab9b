// Projections of fp32 tensors on the tensor cores.
//
// An fp32 number is the sum of three bf16 numbers: itself rounded to nearest, h,
// what that leaves rounded to nearest, m, and the rest, l, which has 8 bits or
// fewer. With the number in [1, 2) times a power of two, |m| <= 2^-8 and |l| <=
// 2^-17 of that power. A product of two numbers is then the nine products of
// their parts, each exact in fp32; the six largest are formed (h h; h m, m h, m m,
// h l, l h), and what is left out (m l, l m, l l) is at most 2^-24 (1 + 2^-10) of
// the product, of either sign. (Split by truncation it reaches 2^-21, always of
// the product's sign: sums of positive numbers came out 4e-8 too small.) bf16
// products run 32 times as fast as fp32 multiply-adds here, so six of them still
// are five times faster.
//
// Bits of a number below 2^-133, bf16's smallest, are not counted: a number under
// 2^-110 has fewer than its 24.
//
// The tensor core truncates as it accumulates, an error of one sign that grows
// with the number of steps. h h and the five small products therefore have an
// accumulator each (the small one's truncations are 2^-8 smaller), at most 512
// input features go into them, and those sums are added in registers, rounded
// to nearest.
//
// Infinities, and numbers that round up to one, leave NaN parts, so their row or
// column comes out as NaN; a product within 2^-7 of the largest number may
// overflow in h h. Whatever comes out as NaN or infinite is recomputed by fp32
// multiply-adds from the operands, and ends up as it would there.
//
// A CTA (20 warps) takes a tile of 128 rows by 128 weight rows over its share of
// the input features; a cluster of up to 8 CTAs shares a tile when there are few.
// Warp 16 copies slices of 32 input features (fp32, 128 bytes) by TMA, warps
// 8-15 split them into parts in shared memory (two groups that take every other
// slice, so that one's waits and fences lie under the other's work), warp 17
// issues the products, and warps 0-7 gather the sums and finish the outputs. Per
// slice of 128 x 128 shared memory moves 32 KB
// in, 80 KB through the split and 96 KB into the tensor core, about 1660
// cycles against 768 of arithmetic: that traffic bounds the kernel (300 x 2048 -> 2048 in
// 37 us, 4096 x 2048 -> 2048 in 233 us, 147 TFLOP/s of fp32 products).
#include "proj_tc.cuh"

namespace rlt {
namespace proj {
namespace {

constexpr int kSplitThreads = 20 * 32;
constexpr int kSlice = 32;                   // input features per slice
constexpr int kTile = 128;                   // rows, and weight rows, of a tile
constexpr int kRawBytes = kTile * 128;       // one operand's slice as it arrives
constexpr int kPartBytes = kTile * kSlice * 2;
constexpr int kRawStages = 3, kPartStages = 2;
constexpr int kRawStage = 2 * kRawBytes, kPartStage = 6 * kPartBytes;
// All of an SM's: this kernel takes all of TMEM, and its clusters must not meet
// another kernel's on an SM where each would wait for what the other holds.
constexpr int kSplitSmem = kSmemBudget;
static_assert(kRawStages * kRawStage + kPartStages * kPartStage + 1024 <= kSplitSmem, "");
constexpr int kSumSlices = 512 / kSlice;     // slices accumulated in TMEM at a time
constexpr int kGatherWarps = 8, kGroupWarps = 4, kCopyWarp = 16, kIssueWarp = 17;
// Registers per thread: at launch, and as the warpgroups share them out.
constexpr int kSplitLaunchRegs = 96, kGatherRegs = 136, kConvertRegs = 80, kIssueRegs = 40;
static_assert(256 * (kGatherRegs + kConvertRegs) + 128 * kIssueRegs <=
                  kSplitThreads * kSplitLaunchRegs,
              "the increase draws on what the launch allocated");

struct SplitParams {
  CUtensorMap map_x, map_w, map_up;
  Problem p;
  int box_m;   // activation rows copied and split per slice
  int w_mn;    // weights with the output features contiguous
  int splits;  // CTAs per tile
  int row_tiles;
  int vec;     // four neighbouring outputs (biases, residuals) are 16 aligned bytes
};

// Eight fp32 numbers as 3 x 8 bf16, packed in 16 bytes each.
__device__ __forceinline__ void split8(const float4& a, const float4& b, uint4 (&part)[3]) {
  const float x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t h[4], m[4], l[4];
  auto nearest = [](float lo, float hi) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&t);
  };
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float r0 = x[2 * e], r1 = x[2 * e + 1];
    h[e] = nearest(r0, r1);
    r0 -= __uint_as_float(h[e] << 16);
    r1 -= __uint_as_float(h[e] & 0xffff0000u);
    m[e] = nearest(r0, r1);
    r0 -= __uint_as_float(m[e] << 16);
    r1 -= __uint_as_float(m[e] & 0xffff0000u);
    l[e] = __byte_perm(__float_as_uint(r0), __float_as_uint(r1), 0x7632);  // their upper halves
  }
  part[0] = make_uint4(h[0], h[1], h[2], h[3]);
  part[1] = make_uint4(m[0], m[1], m[2], m[3]);
  part[2] = make_uint4(l[0], l[1], l[2], l[3]);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) < INFINITY; }

// 64-byte-swizzled K-major tile: rows of 32 bf16, atoms of 8 rows.
__device__ __forceinline__ uint64_t smem_desc_sw64(uint32_t addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((addr >> 4) & 0x3fff);
  d |= static_cast<uint64_t>(1) << 16;            // leading dimension: not used K-major
  d |= static_cast<uint64_t>(512 >> 4) << 32;     // between atoms
  d |= static_cast<uint64_t>(1) << 46;            // version: sm_100
  d |= static_cast<uint64_t>(4) << 61;            // 64-byte swizzle
  return d;
}

// A wait ran out: let copies in flight land before the memory goes.
__device__ __forceinline__ void drain(volatile int* aborted) {
  *aborted = 1;
  const long long start = clock64();
  while (clock64() - start < 4000000LL) {
  }
}

// x[row] . w[n] in fp32 multiply-adds.
__device__ __forceinline__ float plain_dot(const Problem& p, const float* w, int row, int n) {
  const float* x = static_cast<const float*>(p.x) + row * p.x_rs;
  w += n * p.w_ns;
  float y = 0.f;
  // a NaN stays one: a row of them ends at once
  for (int k0 = 0; k0 < p.inner && y == y; k0 += 16)
    for (int k = k0; k < min(k0 + 16, p.inner); ++k) y = fmaf(x[k], w[k * p.w_ks], y);
  return y;
}

template <typename T, Kind kKind, int kAct>
__global__ void __launch_bounds__(kSplitThreads, 1)
    split_kernel(const __grid_constant__ SplitParams g) {
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t raw_full[kRawStages], raw_empty[kRawStages];
  __shared__ uint64_t part_full[kPartStages], part_empty[kPartStages];
  __shared__ uint64_t acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int aborted;
  constexpr int kSet = kKind == kGated ? kTile / 2 : kTile;  // output features per tile
  const Problem& p = g.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint8_t* smem = align_1024(smem_raw);
  uint8_t* raw = smem;
  uint8_t* parts = smem + kRawStages * kRawStage;
  const int rank = g.splits > 1 ? static_cast<int>(tc::cluster_rank()) : 0;
  const int tile = blockIdx.x / g.splits;
  const int m0 = tile % g.row_tiles * kTile;
  const int n0 = tile / g.row_tiles * kSet;
  const int slices = (p.inner + kSlice - 1) / kSlice;
  const int first = static_cast<int>(static_cast<int64_t>(slices) * rank / g.splits);
  const int count = static_cast<int>(static_cast<int64_t>(slices) * (rank + 1) / g.splits) - first;

  if (threadIdx.x == 0) {
    tc::prefetch_tensormap(&g.map_x);
    tc::prefetch_tensormap(&g.map_w);
    if (kKind == kGated) tc::prefetch_tensormap(&g.map_up);
    for (int i = 0; i < kRawStages; ++i) {
      tc::mbar_init(&raw_full[i], 1);
      tc::mbar_init(&raw_empty[i], kGroupWarps);
    }
    for (int i = 0; i < kPartStages; ++i) {
      tc::mbar_init(&part_full[i], kGroupWarps);
      tc::mbar_init(&part_empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&acc_full[i], 1);
      tc::mbar_init(&acc_empty[i], 8);
    }
    aborted = 0;
    tc::fence_mbar_init();
  }
  __syncwarp();
  if (warp == kIssueWarp) tc::tmem_alloc(&tmem_slot, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  tc::pdl_launch_dependents();
  tc::pdl_wait();
  const uint32_t tmem = tmem_slot;
  bool ok = true;

  if (warp >= kCopyWarp) {
    tc::setmaxnreg_dec<kIssueRegs>();
    if (warp == kCopyWarp) {
      const uint32_t bytes = kRawBytes + g.box_m * 128;
      Ring at;
      for (int i = 0; i < count; ++i, at.next(kRawStages)) {
        if (!__all_sync(kFullMask, tc::mbar_wait(&raw_empty[at.slot], at.parity ^ 1, kWaitLimit))) {
          ok = false;
          break;
        }
        if (tc::elect_one()) {
          uint64_t* bar = &raw_full[at.slot];
          uint8_t* x = raw + at.slot * kRawStage;
          uint8_t* w = x + kRawBytes;
          const int k0 = (first + i) * kSlice;
          tc::mbar_expect_tx(bar, bytes);
          tc::tma_load_2d(x, &g.map_x, bar, k0, m0);
          if (g.w_mn) {  // boxes of 32 output features by 32 input features
#pragma unroll
            for (int b = 0; b < 4; ++b) {
              const bool second = kKind == kGated && b >= 2;
              tc::tma_load_2d(w + b * 4096, second ? &g.map_up : &g.map_w, bar,
                              n0 + b * 32 - (second ? kSet : 0), k0);
            }
          } else {
            tc::tma_load_2d(w, &g.map_w, bar, k0, n0);
            if (kKind == kGated) tc::tma_load_2d(w + kRawBytes / 2, &g.map_up, bar, k0, n0);
          }
        }
        __syncwarp();
      }
    } else if (warp == kIssueWarp) {
      const uint32_t idesc = tc::idesc_f16(1, kTile, kTile, g.w_mn);
      const uint64_t x_desc = smem_desc_sw64(tc::smem_u32(parts));
      const uint64_t w_desc =
          g.w_mn ? tc::smem_desc_sw128(tc::smem_u32(parts) + 3 * kPartBytes, 4096, 1024)
                 : smem_desc_sw64(tc::smem_u32(parts) + 3 * kPartBytes);
      const uint32_t x_hi = static_cast<uint32_t>(x_desc >> 32);
      const uint32_t w_hi = static_cast<uint32_t>(w_desc >> 32);
      const uint32_t kstep_w = (g.w_mn ? 2048 : 32) >> 4;
      Ring at, acc;
      for (int i = 0; ok && i < count; acc.next(2)) {
        if (!__all_sync(kFullMask,
                        tc::mbar_poll(&acc_empty[acc.slot], acc.parity ^ 1, kWaitLimit))) {
          ok = false;
          break;
        }
        tc::tc_fence_after();
        const uint32_t d = tmem + acc.slot * 256;
        const int end = min(i + kSumSlices, count);
        for (uint32_t more = 0; i < end; ++i, at.next(kPartStages)) {
          if (!__all_sync(kFullMask, tc::mbar_poll(&part_full[at.slot], at.parity, kWaitLimit))) {
            ok = false;
            break;
          }
          tc::tc_fence_after();
          if (tc::elect_one()) {
            const uint32_t x_lo = static_cast<uint32_t>(x_desc) + at.slot * (kPartStage >> 4);
            const uint32_t w_lo = static_cast<uint32_t>(w_desc) + at.slot * (kPartStage >> 4);
            auto product = [&](uint32_t acc_at, int xp, int wp, int ks, uint32_t accumulate) {
              tc::mma_f16_ss(acc_at, tc::desc64(x_lo + xp * (kPartBytes >> 4) + ks * 2, x_hi),
                             tc::desc64(w_lo + wp * (kPartBytes >> 4) + ks * kstep_w, w_hi), idesc,
                             accumulate);
            };
#pragma unroll
            for (int ks = 0; ks < kSlice / 16; ++ks) {
              const uint32_t go = ks > 0 ? 1 : more;
              product(d, 0, 0, ks, go);
              product(d + kTile, 0, 2, ks, go);
              product(d + kTile, 2, 0, ks, 1);
              product(d + kTile, 1, 1, ks, 1);
              product(d + kTile, 0, 1, ks, 1);
              product(d + kTile, 1, 0, ks, 1);
            }
            tc::mma_commit(&part_empty[at.slot]);
            if (i == end - 1) tc::mma_commit(&acc_full[acc.slot]);
          }
          more = 1;
          __syncwarp();
        }
      }
    }
    if (!ok) drain(&aborted);
    __syncwarp();
    if (g.splits > 1) {
      tc::cluster_sync();
      tc::cluster_sync();
    }
  } else if (warp >= kGatherWarps) {
    tc::setmaxnreg_dec<kConvertRegs>();
    // A warp takes one 32-byte column of the slice's 128-byte lines: 8 elements
    // of 32 lines at a time. Neighbouring lanes have neighbouring lines (rows, or
    // input features of an MN-major slice), which keeps reads and writes free of
    // bank conflicts, and every address is a constant away from the lane's first.
    const int group = (warp - kGatherWarps) / kGroupWarps, c = warp % kGroupWarps;
    const uint32_t from = lane * 128 + (((2 * c) ^ (lane & 7)) << 4);
    const uint32_t to_k = lane * 64 + ((c ^ ((lane >> 1) & 3)) << 4);
    const uint32_t to_mn = lane * 128 + ((c ^ (lane & 7)) << 4);
    auto convert = [&](const uint8_t* line, uint32_t at, uint8_t* to) {
      uint4 part[3];
      split8(*reinterpret_cast<const float4*>(line + at),
             *reinterpret_cast<const float4*>(line + (at ^ 16)), part);
#pragma unroll
      for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(to + k * kPartBytes) = part[k];
    };
    Ring at;
    if (group) at.next(kRawStages);
    uint32_t parity = 1;
    for (int i = group; i < count; i += 2) {
      ok = __all_sync(kFullMask, tc::mbar_wait(&raw_full[at.slot], at.parity, kWaitLimit) &&
                                     tc::mbar_wait(&part_empty[group], parity, kWaitLimit));
      if (!ok) break;
      const uint8_t* src = raw + at.slot * kRawStage;
      uint8_t* dst = parts + group * kPartStage;
      if (g.w_mn) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          convert(src + kRawBytes + j * 4096, from,
                  dst + 3 * kPartBytes + (j >> 1) * 4096 + (to_mn ^ ((j & 1) << 6)));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          convert(src + kRawBytes + j * 4096, from, dst + 3 * kPartBytes + j * 2048 + to_k);
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j * 32 + lane < g.box_m) convert(src + j * 4096, from, dst + j * 2048 + to_k);
      tc::fence_proxy_async_smem();  // the parts are read by the tensor core
      __syncwarp();
      if (lane == 0) {
        tc::mbar_arrive(&part_full[group]);
        tc::mbar_arrive(&raw_empty[at.slot]);
      }
      parity ^= 1;
      at.next(kRawStages);
      at.next(kRawStages);
    }
    if (!ok) drain(&aborted);
    __syncwarp();
    if (g.splits > 1) {
      tc::cluster_sync();
      tc::cluster_sync();
    }
  } else {
    tc::setmaxnreg_inc<kGatherRegs>();
    float v[64];  // this thread's row, half of the columns
    const int half = warp >> 2;
    const uint32_t taddr = tmem + (static_cast<uint32_t>(warp & 3) << 21) + half * 64;
    Ring acc;
    for (int i = 0; i < count; i += kSumSlices, acc.next(2)) {
      ok = __all_sync(kFullMask, tc::mbar_wait(&acc_full[acc.slot], acc.parity, kWaitLimit));
      if (!ok) break;
      tc::tc_fence_after();
#pragma unroll
      for (int c = 0; c < 64; c += 16) {
        uint32_t big[16], small[16];
        tc::tmem_ld16(taddr + acc.slot * 256 + c, big);
        tc::tmem_ld16(taddr + acc.slot * 256 + kTile + c, small);
        tc::tmem_ld_wait(big);
        tc::tmem_ld_wait(small);
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          const float t = __uint_as_float(big[j]) + __uint_as_float(small[j]);
          v[c + j] = i == 0 ? t : v[c + j] + t;
        }
      }
      tc::tc_fence_before();
      __syncwarp();
      if (lane == 0) tc::mbar_arrive(&acc_empty[acc.slot]);
    }
    if (!ok) drain(&aborted);
    __syncwarp();
    if (kKind == kVocab && g.splits == 1) {
      // the logits are all here: a thread's record of its row's half needs no
      // exchange (600 rows against 15776 entries: 201 us, through shared memory 284)
      const int row = m0 + (warp & 3) * 32 + lane, at = n0 + half * 64;
      const int cols = min(64, p.outer - at);
      uint64_t odd = 0;
#pragma unroll
      for (int j = 0; j < 64; ++j)
        if (j < cols && !finite(v[j])) odd |= 1ull << j;
      if (row >= p.rows) odd = 0;
      while (odd != 0) {
        const int i = __ffsll(static_cast<long long>(odd)) - 1;
        odd &= odd - 1;
        const float y = plain_dot(p, static_cast<const float*>(p.w), row, at + i);
#pragma unroll
        for (int j = 0; j < 64; ++j)
          if (j == i) v[j] = y;
      }
      __syncwarp();
      const int64_t want = p.tokens != nullptr && row < p.rows ? p.tokens[row] : -1;
      const VocabPart part = vocab_part<64>(p, v, at, cols, want);
      if (row < p.rows)
        *reinterpret_cast<float4*>(
            &p.parts[static_cast<int64_t>(row) * p.tiles + tile / g.row_tiles * 2 + half]) =
            make_float4(part.most, part.sum, __int_as_float(part.at), part.chosen);
    } else {
      // Every product is done, so the stages are free: the sums take their place,
      // rows of 128 columns (gate then up) in 16-byte units swizzled by row.
      const int r0 = (warp & 3) * 32 + lane;
#pragma unroll
      for (int c = 0; c < 16; ++c)
        *reinterpret_cast<float4*>(smem + r0 * 512 + (((half * 16 + c) ^ (r0 & 7)) << 4)) =
            make_float4(v[c * 4], v[c * 4 + 1], v[c * 4 + 2], v[c * 4 + 3]);
      // Each CTA of the cluster finishes every splits-th row, adding in rank order.
      constexpr int kLanes = kSet / 4;  // lanes per row, four features each
      const int c = lane % kLanes, n = n0 + c * 4;
      const int rows = min(kTile, p.rows - m0);
      const int row_first = rank + (warp * (32 / kLanes) + lane / kLanes) * g.splits;
      const int row_step = kGatherWarps * (32 / kLanes) * g.splits;
      const float* bias_at = static_cast<const float*>(p.bias);
      const float* res_at = static_cast<const float*>(p.residual);
      auto residual = [&](int r, float (&add)[4]) {
        read4<float>(res_at != nullptr && n < p.outer && r < rows ? res_at + (m0 + r) * p.r_rs + n
                                                                  : nullptr,
                     g.vec, p.outer - n, add);
      };
      float bias[4], add[4];
      read4<float>(bias_at != nullptr && n < p.outer ? bias_at + n : nullptr, g.vec, p.outer - n,
                   bias);
      residual(row_first, add);
      __syncwarp();  // its reads differ by lane; the barrier wants whole warps
      if (g.splits > 1)
        tc::cluster_sync();
      else
        asm volatile("bar.sync 1, %0;" ::"n"(kGatherWarps * 32) : "memory");
      if (kKind == kVocab || n < p.outer) {  // the head's rows are whole warps'
        for (int r = row_first; r < rows; r += row_step) {
          float y[2][4];
#pragma unroll
          for (int op = 0; op < (kKind == kGated ? 2 : 1); ++op) {
            const uint8_t* at = smem + r * 512 + (((op * 16 + c) ^ (r & 7)) << 4);
            float4 t[kMaxSplits];
#pragma unroll
            for (int s = 0; s < kMaxSplits; ++s)
              if (s < g.splits)
                t[s] = g.splits > 1 ? tc::ld_peer4(tc::peer_smem(at, s))
                                    : *reinterpret_cast<const float4*>(at);
#pragma unroll
            for (int s = 1; s < kMaxSplits; ++s)
              if (s < g.splits) {
                t[0].x += t[s].x;
                t[0].y += t[s].y;
                t[0].z += t[s].z;
                t[0].w += t[s].w;
              }
            y[op][0] = t[0].x;
            y[op][1] = t[0].y;
            y[op][2] = t[0].z;
            y[op][3] = t[0].w;
            const float any = y[op][0] + y[op][1] + y[op][2] + y[op][3];
            if (!finite(any)) {
              const float* w = static_cast<const float*>(op == 0 ? p.w : p.w_up);
#pragma unroll 1
              for (int i = 0; i < 4 && n + i < p.outer; ++i) {
                float mine = y[op][0];
#pragma unroll
                for (int e = 1; e < 4; ++e)
                  if (e == i) mine = y[op][e];
                if (finite(mine)) continue;
                mine = plain_dot(p, w, m0 + r, n + i);
#pragma unroll
                for (int e = 0; e < 4; ++e)
                  if (e == i) y[op][e] = mine;
              }
            }
          }
          if constexpr (kKind == kVocab) {
            __syncwarp();
            const int at = tile / g.row_tiles * 2;  // two records a tile
            vocab_row(p, y[0], m0 + r, n, at);
            if (lane == 0)
              *reinterpret_cast<float4*>(&p.parts[static_cast<int64_t>(m0 + r) * p.tiles + at + 1]) =
                  make_float4(-INFINITY, 0.f, __int_as_float(INT32_MAX), 0.f);
          } else {
            float next[4];
            residual(r + row_step, next);
            finish4<float, kKind, kAct>(p, g.vec, m0 + r, n, y[0], y[kKind == kGated ? 1 : 0],
                                        bias, add);
#pragma unroll
            for (int e = 0; e < 4; ++e) add[e] = next[e];
          }
        }
      }
      __syncwarp();
      if (g.splits > 1) tc::cluster_sync();  // a peer may still be reading this CTA's sums
    }
  }
  __syncwarp();
  tc::tc_fence_before();
  __syncthreads();
  if (aborted && threadIdx.x == 0) raise_status(p.status, kStatusTimeout);
  if (warp == kIssueWarp) {
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem, 512);
  }
}

template <typename T, Kind kKind, int kAct>
int launch(const SplitParams& g, int ctas, cudaStream_t stream) {
  constexpr auto kernel = split_kernel<T, kKind, kAct>;
  if (const cudaError_t e = allow_smem<kernel>(kSplitSmem, kSplitLaunchRegs)) return static_cast<int>(e);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas));
  cfg.blockDim = dim3(kSplitThreads);
  cfg.dynamicSmemBytes = kSplitSmem;
  cfg.stream = stream;
  cudaLaunchAttribute attrs[2];
  cfg.attrs = attrs;
  cfg.numAttrs = launch_attributes(attrs, g.splits);
  return launch_status(cudaLaunchKernelEx(&cfg, kernel, g));
}

}  // namespace

int split_vocab_parts(const Problem& p) { return 2 * ceil_div(p.outer, kTile); }

int run_split(Kind kind, const Problem& p, int ctas, cudaStream_t stream) {
  SplitParams g{};
  const int set = kind == kGated ? kTile / 2 : kTile;
  g.p = p;
  g.w_mn = p.w_ks != 1;
  g.row_tiles = ceil_div(p.rows, kTile);
  g.box_m = p.rows >= kTile ? kTile : ceil_div(p.rows, 8) * 8;
  const int64_t tiles = static_cast<int64_t>(g.row_tiles) * ceil_div(p.outer, set);
  const int slices = ceil_div(p.inner, kSlice);
  // CTAs per tile: one CTA fits an SM, so what counts is how many clusters run
  // at once. In slices' times; a CTA pays about eight for its start and end. The
  // head, whose rows need no exchange in one CTA, has to gain half as much again
  // (600 rows of 2112 against 16496 entries: 269 us, in pairs 366).
  g.splits = 1;
  double least = 1e300;
  for (int s = 1; s <= kMaxSplits && slices >= 4 * s; ++s) {
    constexpr auto kernel = split_kernel<float, kLinear, RLT_ACT_NONE>;
    const int64_t at_once = s == 1 ? ctas : resident_clusters<kernel>(s, kSplitThreads, kSplitSmem);
    const double cost = static_cast<double>((tiles + at_once - 1) / at_once) *
                        (ceil_div(slices, s) + 8) * (kind == kVocab && s > 1 ? 1.5 : 1.0);
    if (cost < least) {
      least = cost;
      g.splits = s;
    }
  }
  if (tiles * g.splits > INT32_MAX) return RLT_E_SHAPE;
  g.vec = p.outer % 4 == 0 && p.o_rs % 4 == 0 && p.r_rs % 4 == 0 && aligned_to(p.out, 16) &&
          aligned_to(p.bias, 16) && aligned_to(p.residual, 16);
  bool ok = encode2d(&g.map_x, RLT_F32, p.x, p.inner, p.rows, p.x_rs, g.box_m);
  for (int op = 0; op < (kind == kGated ? 2 : 1); ++op) {
    CUtensorMap* map = op ? &g.map_up : &g.map_w;
    const void* base = op ? p.w_up : p.w;
    ok = ok && (g.w_mn ? encode2d(map, RLT_F32, base, p.outer, p.inner, p.w_ks, kSlice)
                       : encode2d(map, RLT_F32, base, p.inner, p.outer, p.w_ns, set));
  }
  if (!ok) return RLT_E_DEVICE;
  const int grid = static_cast<int>(tiles * g.splits);
  switch (kind) {
    case kLinear: return by_activation<kLinear, float>(g, grid, stream);
    case kGated: return by_activation<kGated, float>(g, grid, stream);
    default: return by_activation<kVocab, float>(g, grid, stream);
  }
}

}  // namespace proj
}  // namespace rlt
