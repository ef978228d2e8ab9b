// What the tensor-core projection kernels share.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <atomic>

#include "proj_common.cuh"
#include "tc_ptx.cuh"

namespace rlt {
namespace proj {
namespace {

constexpr long long kWaitLimit = 100000000LL;  // cycles (~50 ms)
// For a wait that covers `blocks` blocks of input features.
__device__ __forceinline__ long long whole_sum_limit(int blocks) {
  return kWaitLimit + blocks * 20000LL;
}
constexpr int kMaxSplits = 8;                  // CTAs of a cluster (the portable limit)
constexpr int kSmemBudget = 224 * 1024;        // dynamic shared memory of a CTA

// The first 1024-byte boundary in dynamic shared memory, as an offset from it:
// a pointer rounded up as a number would lose its address space, and every
// access through it would be a generic one.
__device__ __forceinline__ uint8_t* align_1024(uint8_t* smem) {
  return smem + ((1024u - (tc::smem_u32(smem) & 1023u)) & 1023u);
}

// Position in a ring of barriers: a slot, and the parity its next use has. The
// issuing threads step it without divisions (with them a 64-feature block took
// them 570 and 740 cycles, more than its 512 of arithmetic).
struct Ring {
  int slot = 0;
  uint32_t parity = 0;
  __device__ __forceinline__ void next(int size) {
    if (++slot == size) {
      slot = 0;
      parity ^= 1;
    }
  }
};

// Four neighbouring 16-bit values (8-byte aligned in memory).
template <typename T>
__device__ __forceinline__ void widen4(const uint2& r, float (&v)[4]) {
  T t[4];
  *reinterpret_cast<uint2*>(t) = r;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = to_f32<T>(t[e]);
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  widen4<T>(*reinterpret_cast<const uint2*>(p), v);
}

template <typename T>
struct alignas(sizeof(T) * 4) Four {
  T v[4];
};

// Four neighbouring outputs of a row from column n on: act(y + bias) +
// residual, or act(y) * up. `vec`: they are one store (and all four exist).
template <typename T, Kind kKind, int kAct>
__device__ __forceinline__ void finish4(const Problem& p, bool vec, int row, int n,
                                        const float (&y)[4], const float (&up)[4],
                                        const float (&bias)[4], const float (&add)[4]) {
  constexpr bool kPrecise = sizeof(T) == 4;
  Four<T> o;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (kKind == kGated)
      o.v[e] = from_f32<T>(activate<kPrecise, kAct>(y[e]) * up[e]);
    else
      o.v[e] = from_f32<T>(activate<kPrecise, kAct>(y[e] + bias[e]) + add[e]);
  }
  T* out = static_cast<T*>(p.out) + row * p.o_rs + n;
  if (vec) {
    *reinterpret_cast<Four<T>*>(out) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < p.outer) out[e] = o.v[e];
  }
}

// Four neighbouring values of a vector or a row (in one load where `vec`),
// zeros past `left` and without one.
template <typename T>
__device__ __forceinline__ void read4(const T* at, bool vec, int left, float (&v)[4]) {
  if (at != nullptr && vec) {
    const Four<T> f = *reinterpret_cast<const Four<T>*>(at);
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = to_f32<T>(f.v[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = at != nullptr && e < left ? to_f32<T>(at[e]) : 0.f;
  }
}

// A thread's record of its columns v[0 .. cols) of one vocabulary tile, the
// first of them vocabulary entry n0.
template <int kN>
__device__ __forceinline__ VocabPart vocab_part(const Problem& p, const float (&v)[kN], int n0,
                                                int cols, int64_t want) {
  VocabPart part{-INFINITY, 0.f, INT32_MAX, 0.f};
  if (cols <= 0) return part;
  // Sum of 2^(l log2e - b) with b = most * log2e rounded: one multiply-add and
  // one exponential per logit. b's rounding is the same in every term, and taken
  // back as a factor at the end.
  if (cols == kN) {  // the whole of a full tile: no test per column
#pragma unroll
    for (int j = 0; j < kN; ++j) part.most = fmaxf(part.most, v[j]);
  } else {
#pragma unroll
    for (int c = 0; c < kN; c += 16)
      if (c < cols)
#pragma unroll
        for (int j = 0; j < 16; ++j)
          part.most = fmaxf(part.most, c + j < cols ? v[c + j] : -INFINITY);
  }
  const float base = part.most == -INFINITY ? 0.f : part.most;
  const float b = base * kLog2e;
  float s0 = 0.f, s1 = 0.f;
  if (cols == kN) {
#pragma unroll
    for (int j = 0; j < kN; j += 2) {
      s0 += ex2(fmaf(v[j], kLog2e, -b));
      s1 += ex2(fmaf(v[j + 1], kLog2e, -b));
    }
  } else {
#pragma unroll
    for (int c = 0; c < kN; c += 16)
      if (c < cols)
#pragma unroll
        for (int j = 0; j < 16; j += 2) {
          s0 += c + j < cols ? ex2(fmaf(v[c + j], kLog2e, -b)) : 0.f;
          s1 += c + j + 1 < cols ? ex2(fmaf(v[c + j + 1], kLog2e, -b)) : 0.f;
        }
  }
  part.sum = (s0 + s1) * ex2(-fmaf(base, kLog2e, -b));
  // b's rounding reaches 2^-24 of it, which as an exponent has to stay small
  const bool far = !(fabsf(b) < 268435456.f);
  if (__any_sync(kFullMask, far)) {
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < kN; ++j) s += j < cols ? ex2((v[j] - base) * kLog2e) : 0.f;
    if (far) part.sum = s;
  }
  if (p.tokens != nullptr) {
    const bool here = want >= n0 && want < n0 + cols;
    if (__any_sync(kFullMask, here)) {
      const int at = here ? static_cast<int>(want - n0) : -1;
#pragma unroll
      for (int j = 0; j < kN; ++j)
        if (j == at) part.chosen = v[j];
    }
    return part;
  }
#pragma unroll
  for (int j = kN - 1; j >= 0; --j)
    if (j < cols && v[j] == part.most) part.at = n0 + j;
  if (__any_sync(kFullMask, part.sum != part.sum)) {  // a NaN counts as the largest: the first
#pragma unroll
    for (int j = kN - 1; j >= 0; --j)
      if (j < cols && v[j] != v[j]) {
        part.most = v[j];
        part.at = n0 + j;
      }
  }
  return part;
}

// The record of a row's 128 logits in one vocabulary tile, four to a lane from
// entry n on, written as the row's record `tile`. For a whole warp.
__device__ __forceinline__ void vocab_row(const Problem& p, const float (&l)[4], int row, int n,
                                          int tile) {
  VocabPart part{-INFINITY, 0.f, INT32_MAX, 0.f};
  const int64_t want = p.tokens != nullptr ? p.tokens[row] : -1;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (n + e >= p.outer) continue;
    if (beats(l[e], n + e, part.most, part.at)) {
      part.most = l[e];
      part.at = n + e;
    }
    if (n + e == want) part.chosen = l[e];
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float m = __shfl_xor_sync(kFullMask, part.most, o);
    const int at = __shfl_xor_sync(kFullMask, part.at, o);
    if (beats(m, at, part.most, part.at)) {
      part.most = m;
      part.at = at;
    }
    part.chosen += __shfl_xor_sync(kFullMask, part.chosen, o);
  }
  const float base = part.most == -INFINITY ? 0.f : part.most;
#pragma unroll
  for (int e = 0; e < 4; ++e)
    if (n + e < p.outer) part.sum += ex2((l[e] - base) * kLog2e);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) part.sum += __shfl_xor_sync(kFullMask, part.sum, o);
  if ((threadIdx.x & 31) == 0)
    *reinterpret_cast<float4*>(&p.parts[static_cast<int64_t>(row) * p.tiles + tile]) =
        make_float4(part.most, part.sum, __int_as_float(part.at), part.chosen);
}

// ---- host side ----

inline PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
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

// A [lines x line] matrix, `stride` elements between lines, copied in boxes of
// 128 bytes (64 elements of 16 bits, 32 of fp32) by `box_lines` lines.
inline bool encode2d(CUtensorMap* map, int32_t dtype, const void* base, int line, int lines,
              int64_t stride, int box_lines) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(line), static_cast<cuuint64_t>(lines)};
  const cuuint64_t es = dtype == RLT_F32 ? 4 : 2;
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(stride) * es};
  const cuuint32_t box[2] = {static_cast<cuuint32_t>(128 / es), static_cast<cuuint32_t>(box_lines)};
  const cuuint32_t elem[2] = {1, 1};
  const CUtensorMapDataType type = dtype == RLT_F32    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                   : dtype == RLT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16
                                                       : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return fn(map, type, 2, const_cast<void*>(base), dims, strides, box, elem,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Dynamic shared memory of kKernel raised (and its register count checked) once
// per device.
template <auto kKernel>
cudaError_t allow_smem(int bytes, int least_regs = 0) {
  static std::atomic<bool> done[64];
  int dev = 0;
  if (const cudaError_t e = cudaGetDevice(&dev)) return e;
  if (dev >= 0 && dev < 64 && done[dev].load()) return cudaSuccess;
  cudaError_t e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && least_regs > 0) {
    // with fewer registers at launch a warpgroup's increase could never be granted
    cudaFuncAttributes attr{};
    e = cudaFuncGetAttributes(&attr, kKernel);
    if (e == cudaSuccess && attr.numRegs < least_regs) e = cudaErrorInvalidConfiguration;
  }
  if (e == cudaSuccess && dev >= 0 && dev < 64) done[dev].store(true);
  return e;
}

// Clusters of `size` CTAs of kKernel that the device runs at once, each CTA
// with `smem` bytes of dynamic shared memory. An SM group of the die need not
// hold a whole number of clusters, so this can be well below CTAs / size.
template <auto kKernel>
int resident_clusters(int size, int threads, int smem) {
  static std::atomic<int> known[64][kMaxSplits + 1];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 1;
  if (dev >= 0 && dev < 64)
    if (const int n = known[dev][size].load()) return n;
  if (cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmemBudget) !=
      cudaSuccess)
    return 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(size);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = size;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  int n = 0;
  if (cudaOccupancyMaxActiveClusters(&n, kKernel, &cfg) != cudaSuccess || n < 1) {
    (void)cudaGetLastError();
    return 1;
  }
  if (dev >= 0 && dev < 64) known[dev][size].store(n);
  return n;
}

// The kernel for a launch's activation.
template <typename T, Kind kKind, int kAct, typename Params>
int launch(const Params& g, int ctas, cudaStream_t stream);
template <Kind kKind, typename T, typename Params>
int by_activation(const Params& g, int ctas, cudaStream_t stream) {
  if constexpr (kKind == kVocab) {
    return launch<T, kKind, RLT_ACT_NONE>(g, ctas, stream);
  } else {
    switch (g.p.act) {
      case RLT_ACT_SILU: return launch<T, kKind, RLT_ACT_SILU>(g, ctas, stream);
      case RLT_ACT_GELU: return launch<T, kKind, RLT_ACT_GELU>(g, ctas, stream);
      case RLT_ACT_GELU_TANH: return launch<T, kKind, RLT_ACT_GELU_TANH>(g, ctas, stream);
      case RLT_ACT_RELU: return launch<T, kKind, RLT_ACT_RELU>(g, ctas, stream);
      case RLT_ACT_SIGMOID: return launch<T, kKind, RLT_ACT_SIGMOID>(g, ctas, stream);
      default: return launch<T, kKind, RLT_ACT_NONE>(g, ctas, stream);
    }
  }
}

inline bool aligned_to(const void* p, int bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes == 0;
}

}  // namespace
}  // namespace proj
}  // namespace rlt
