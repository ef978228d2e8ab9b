// Projections with what follows them (sm_100a): the matrix product with bias,
// activation and residual in its epilogue, the gated product, and the
// vocabulary head that reduces its logits tile by tile.
//
// This file holds the C entries, the multiply-add kernel and the join of the
// vocabulary tiles.
#include <cooperative_groups.h>

#include "proj_common.cuh"

namespace rlt {
namespace proj {
namespace {

namespace cg = cooperative_groups;

constexpr int kBK = 16;  // input features per shared-memory tile

__device__ __forceinline__ void fma2(uint64_t& acc, uint64_t a, uint64_t b) {
  asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(acc) : "l"(a), "l"(b));
}
__device__ __forceinline__ uint64_t dup2(float a) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %1};" : "=l"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ void split2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}

// Four elements of a [lines x inner] operand, zeros outside it: along the
// input features (kAlongK: `line` fixed) or along the lines.
template <typename T>
__device__ __forceinline__ void load4(float (&v)[4], const T* base, int line, int k, int lines,
                                      int k_end, int64_t ls, int64_t ks, bool along_k) {
  const T* p = base + line * ls + k * ks;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = along_k ? (line < lines && k + j < k_end) : (line + j < lines && k < k_end);
    v[j] = in ? to_f32<T>(p[along_k ? j * ks : j * ls]) : 0.f;
  }
}

// A CTA's tile of BM = 16 TM rows and BN = 16 TN output columns, 256 threads
// in a 16 x 16 grid, each with TM rows and two groups of TN / 2 columns, one
// in each half of the tile. In a gated product the halves are gate and up
// columns of the same features, so a thread holds both of what it multiplies.
//
// With few tiles the input features are split over a cluster of CTAs; their
// partial sums are read through distributed shared memory and added in rank
// order, so the result repeats bit for bit.
template <typename T, int TM, int TN, Kind kKind>
__global__ void __launch_bounds__(256) fma_kernel(const Problem p) {
  constexpr int BM = 16 * TM, BN = 16 * TN;
  constexpr int MG = TM < 4 ? TM : 4, NG = TN / 2;
  constexpr int kSets = kKind == kGated ? BN / 2 : BN;  // output features per tile
  constexpr bool kPrecise = sizeof(T) == 4;
  constexpr int kTile = 2 * kBK * (BM + BN + 8);
  constexpr bool kSplits = kKind != kVocab && BM * BN <= 4096;  // partials fit where the tiles were
  __shared__ __align__(16) float smem[kSplits && BM * BN > kTile ? BM * BN : kTile];
  float(*xs)[kBK][BM + 4] = reinterpret_cast<float(*)[kBK][BM + 4]>(smem);
  float(*ws)[kBK][BN + 4] = reinterpret_cast<float(*)[kBK][BN + 4]>(smem + 2 * kBK * (BM + 4));

  cg::cluster_group cluster = cg::this_cluster();
  const int splits = kSplits ? cluster.num_blocks() : 1;
  const int rank = kSplits ? cluster.block_rank() : 0;
  const int item = blockIdx.x / splits;
  const int row_tiles = (p.rows + BM - 1) / BM;
  const int row0 = item % row_tiles * BM;
  const int col0 = item / row_tiles * kSets;
  const int ksteps = (p.inner + kBK - 1) / kBK;
  const int step0 = static_cast<int>(static_cast<int64_t>(ksteps) * rank / splits);
  const int step1 = static_cast<int>(static_cast<int64_t>(ksteps) * (rank + 1) / splits);
  const int tid = threadIdx.x, tx = tid & 15, ty = tid >> 4;

  const T* x = static_cast<const T*>(p.x);
  const T* w = static_cast<const T*>(p.w);
  const bool along_k = p.w_ks == 1;
  constexpr int XU = (BM * kBK / 4 + 255) / 256, WU = (BN * kBK / 4 + 255) / 256;
  float xr[XU][4], wr[WU][4];
  auto fetch = [&](int step) {
    const int k0 = step * kBK;
#pragma unroll
    for (int i = 0; i < XU; ++i) {
      const int u = tid + i * 256;
      if (u < BM * kBK / 4)
        load4<T>(xr[i], x, row0 + u / 4, k0 + u % 4 * 4, p.rows, p.inner, p.x_rs, 1, true);
    }
#pragma unroll
    for (int i = 0; i < WU; ++i) {
      const int u = tid + i * 256;
      if (u < BN * kBK / 4) {
        const int c = along_k ? u / 4 : u % (BN / 4) * 4;
        const int k = k0 + (along_k ? u % 4 * 4 : u / (BN / 4));
        const bool second = kKind == kGated && c >= BN / 2;
        load4<T>(wr[i], second ? static_cast<const T*>(p.w_up) : w,
                 col0 + c - (second ? BN / 2 : 0), k, p.outer, p.inner, p.w_ns, p.w_ks, along_k);
      }
    }
  };
  auto keep = [&](int buf) {
#pragma unroll
    for (int i = 0; i < XU; ++i) {
      const int u = tid + i * 256;
      if (u < BM * kBK / 4)
#pragma unroll
        for (int j = 0; j < 4; ++j) xs[buf][u % 4 * 4 + j][u / 4] = xr[i][j];
    }
#pragma unroll
    for (int i = 0; i < WU; ++i) {
      const int u = tid + i * 256;
      if (u < BN * kBK / 4) {
        if (along_k) {
#pragma unroll
          for (int j = 0; j < 4; ++j) ws[buf][u % 4 * 4 + j][u / 4] = wr[i][j];
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j) ws[buf][u / (BN / 4)][u % (BN / 4) * 4 + j] = wr[i][j];
        }
      }
    }
  };

  uint64_t acc[TM][NG];  // pairs of neighbouring columns; [.., NG / 2) in the first half
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < NG; ++j) acc[i][j] = 0;
  fetch(step0);
  keep(0);
  __syncthreads();
  for (int step = step0; step < step1; ++step) {
    const int buf = (step - step0) & 1;
    if (step + 1 < step1) fetch(step + 1);
#pragma unroll
    for (int k = 0; k < kBK; ++k) {
      float a[TM];
      uint64_t b[NG];
#pragma unroll
      for (int i = 0; i < TM; ++i) a[i] = xs[buf][k][i / MG * (16 * MG) + ty * MG + i % MG];
#pragma unroll
      for (int j = 0; j < NG; ++j)
        b[j] = *reinterpret_cast<const uint64_t*>(
            &ws[buf][k][j / (NG / 2) * (BN / 2) + tx * NG + j % (NG / 2) * 2]);
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const uint64_t aa = dup2(a[i]);
#pragma unroll
        for (int j = 0; j < NG; ++j) fma2(acc[i][j], aa, b[j]);
      }
    }
    if (step + 1 < step1) keep(buf ^ 1);
    __syncthreads();
  }

  auto row_of = [&](int i) { return i / MG * (16 * MG) + ty * MG + i % MG; };
  auto col_of = [&](int j) { return j / NG * (BN / 2) + tx * NG + j % NG; };
  auto value = [&](int i, int j) {
    float lo, hi;
    split2(acc[i][j / 2], lo, hi);
    return j & 1 ? hi : lo;
  };

  if constexpr (kKind == kVocab) {
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int row = row0 + row_of(i);
      const bool in = row < p.rows;
      const int64_t want = in && p.tokens != nullptr ? p.tokens[row] : -1;
      VocabPart part{-INFINITY, 0.f, INT32_MAX, 0.f};
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int v = col0 + col_of(j);
        if (v >= p.outer) continue;
        const float l = value(i, j);
        if (beats(l, v, part.most, part.at)) {
          part.most = l;
          part.at = v;
        }
        if (v == want) part.chosen = l;
      }
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) {
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
      for (int j = 0; j < TN; ++j)
        if (col0 + col_of(j) < p.outer) part.sum += expf(value(i, j) - base);
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) part.sum += __shfl_xor_sync(kFullMask, part.sum, o);
      if (in && tx == 0) p.parts[static_cast<int64_t>(row) * p.tiles + item / row_tiles] = part;
    }
    return;
  } else {
    const T* bias = static_cast<const T*>(p.bias);
    auto finish = [&](int row, int n, float y, float up) {  // one output element
      if (row >= p.rows || n >= p.outer) return;
      if (kKind == kGated) {
        y = activate<kPrecise>(p.act, y) * up;
      } else {
        if (bias != nullptr) y += to_f32<T>(bias[n]);
        y = activate<kPrecise>(p.act, y);
        if (p.residual != nullptr)
          y += to_f32<T>(static_cast<const T*>(p.residual)[row * p.r_rs + n]);
      }
      static_cast<T*>(p.out)[row * p.o_rs + n] = from_f32<T>(y);
    };
    if (splits == 1) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < (kKind == kGated ? NG : TN); ++j)
          finish(row0 + row_of(i), col0 + col_of(j), value(i, j),
                 kKind == kGated ? value(i, (j + NG) % TN) : 0.f);
      return;
    }
    if constexpr (kSplits) {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) smem[row_of(i) * BN + col_of(j)] = value(i, j);
      cluster.sync();
      constexpr int kOuts = BM * kSets;
      for (int e = rank * 256 + tid; e < kOuts; e += splits * 256) {
        const int r = e / kSets, c = e % kSets;
        float y = 0.f, up = 0.f;
        for (int s = 0; s < splits; ++s) {
          const float* peer = cluster.map_shared_rank(smem, s);
          y += peer[r * BN + c];
          if (kKind == kGated) up += peer[r * BN + (c + BN / 2) % BN];
        }
        finish(row0 + r, col0 + c, y, up);
      }
      cluster.sync();  // a peer may still be reading this CTA's sums
    }
  }
}

// Joins the vocabulary tiles of a row, one warp per row.
__global__ void __launch_bounds__(256) vocab_join_kernel(const VocabPart* parts,
                                                         const int64_t* tokens,
                                                         int64_t* out_tokens, float* logprobs,
                                                         int32_t* status, int rows, int tiles,
                                                         int vocab) {
  const int row = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (row >= rows) return;
  VocabPart a{-INFINITY, 0.f, INT32_MAX, 0.f};
  for (int t = lane; t < tiles; t += 32) fold(a, parts[static_cast<int64_t>(row) * tiles + t]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    VocabPart b;
    b.most = __shfl_xor_sync(kFullMask, a.most, o);
    b.sum = __shfl_xor_sync(kFullMask, a.sum, o);
    b.at = __shfl_xor_sync(kFullMask, a.at, o);
    b.chosen = __shfl_xor_sync(kFullMask, a.chosen, o);
    fold(a, b);
  }
  if (lane != 0) return;
  const float normaliser = a.most == -INFINITY ? NAN : logf(a.sum);
  if (tokens == nullptr) {
    out_tokens[row] = a.at;
    logprobs[row] = -normaliser;
    return;
  }
  const int64_t want = tokens[row];
  if (want >= vocab) raise_status(status, kStatusBadToken);
  logprobs[row] = want < 0 ? 0.f : want >= vocab ? NAN : a.chosen - a.most - normaliser;
}

int sm_count() {
  static int count[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  if (count[dev] == 0) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    count[dev] = n;
  }
  return count[dev];
}

template <typename T, int TM, int TN, Kind kKind>
int launch_fma(Problem p, cudaStream_t stream) {
  constexpr int BM = 16 * TM, kSets = kKind == kGated ? 8 * TN : 16 * TN;
  const int64_t items = static_cast<int64_t>(ceil_div(p.rows, BM)) * ceil_div(p.outer, kSets);
  int splits = 1;
  if (kKind != kVocab && BM * 16 * TN <= 4096)
    while (splits < 8 && items * splits < 2 * sm_count() && p.inner >= splits * 2 * 4 * kBK)
      splits *= 2;
  if (items * splits > INT32_MAX) return RLT_E_SHAPE;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(items * splits));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = splits;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return launch_status(cudaLaunchKernelEx(&cfg, fma_kernel<T, TM, TN, kKind>, p));
}

// Output columns of a multiply-add tile, by row count: few rows take a tile of
// 16 rows; a 128 x 128 tile needs enough of them to fill the SMs.
int fma_tile(int rows, int features) {
  if (rows <= 16) return 0;
  return static_cast<int64_t>(ceil_div(rows, 128)) * ceil_div(features, 128) >= sm_count() ? 2 : 1;
}

template <typename T, Kind kKind>
int run_fma(const Problem& p, cudaStream_t stream) {
  const int features = kKind == kGated ? 2 * p.outer : p.outer;
  switch (fma_tile(p.rows, features)) {
    case 0: return launch_fma<T, 1, 4, kKind>(p, stream);
    case 1: return launch_fma<T, 4, 4, kKind>(p, stream);
    default: return launch_fma<T, 8, 8, kKind>(p, stream);
  }
}

// ---- 16-bit operands for the tensor cores -------------------------------------

int64_t round8(int64_t n) { return (n + 7) / 8 * 8; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// What TMA asks of an operand of `lines` lines of `line` elements: a 16-byte
// aligned start and a stride of whole 16-byte units. A stride shorter than a
// line (a broadcast operand) is copied too.
bool tma_ready(const void* base, int line, int lines, int64_t stride) {
  return aligned16(base) && (lines == 1 || (stride % 8 == 0 && stride >= line));
}

struct Layout {  // of the weights: lines along the contiguous dimension
  int line, lines;
  int64_t stride;
};
Layout weight_layout(const Problem& p) {
  return p.w_ks == 1 ? Layout{p.inner, p.outer, p.w_ns} : Layout{p.outer, p.inner, p.w_ks};
}

bool x_ready(const Problem& p) { return tma_ready(p.x, p.inner, p.rows, p.x_rs); }
bool w_ready(const Problem& p) {
  const Layout l = weight_layout(p);
  return tma_ready(p.w, l.line, l.lines, l.stride) &&
         (p.w_up == nullptr || tma_ready(p.w_up, l.line, l.lines, l.stride));
}

size_t copies_bytes(const Problem& p, int32_t dtype) {
  if (dtype == RLT_F32) return 0;
  const Layout l = weight_layout(p);
  size_t bytes = 0;
  if (!x_ready(p)) bytes += static_cast<size_t>(round8(p.inner)) * p.rows * 2;
  if (!w_ready(p)) bytes += static_cast<size_t>(round8(l.line)) * l.lines * (p.w_up ? 4 : 2);
  return bytes;
}

// dst[line][0 .. pitch) = src[line * stride ..][0 .. length), 16-bit elements;
// what lies past `length` is never read.
__global__ void __launch_bounds__(256) align_kernel(const uint16_t* __restrict__ src,
                                                    uint16_t* __restrict__ dst, int length,
                                                    int lines, int64_t stride, int pitch) {
  const int units = pitch / 8;
  const int64_t total = static_cast<int64_t>(units) * lines;
  for (int64_t i = blockIdx.x * 256LL + threadIdx.x; i < total; i += gridDim.x * 256LL) {
    const int64_t line = i / units;
    const int c = static_cast<int>(i - line * units) * 8;
    const uint16_t* s = src + line * stride + c;
    uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < length) v[e / 2] |= static_cast<uint32_t>(s[e]) << (e % 2 * 16);
    st_vec(dst + line * pitch + c, make_uint4(v[0], v[1], v[2], v[3]));
  }
}

int align_copy(const void*& base, int64_t& stride, int length, int lines, char*& at,
               cudaStream_t stream) {
  const int64_t pitch = round8(length);
  if (pitch > INT32_MAX) return RLT_E_SHAPE;
  const int64_t blocks = (pitch / 8 * lines + 255) / 256;
  align_kernel<<<static_cast<unsigned>(blocks < 16 * sm_count() ? blocks : 16 * sm_count()), 256, 0,
                 stream>>>(static_cast<const uint16_t*>(base), reinterpret_cast<uint16_t*>(at),
                           length, lines, stride, static_cast<int>(pitch));
  base = at;
  stride = pitch;
  at += pitch * lines * 2;
  return launch_status(cudaGetLastError());
}

template <Kind kKind>
int dispatch(Problem p, int32_t dtype, char* copies, cudaStream_t stream) {
  if (dtype == RLT_F32) return run_fma<float, kKind>(p, stream);
  if (!x_ready(p))
    if (const int rc = align_copy(p.x, p.x_rs, p.inner, p.rows, copies, stream)) return rc;
  if (!w_ready(p)) {
    const Layout l = weight_layout(p);
    int64_t stride = l.stride;
    if (p.w_up != nullptr) {
      stride = l.stride;
      if (const int rc = align_copy(p.w_up, stride, l.line, l.lines, copies, stream)) return rc;
      stride = l.stride;
    }
    if (const int rc = align_copy(p.w, stride, l.line, l.lines, copies, stream)) return rc;
    (p.w_ks == 1 ? p.w_ns : p.w_ks) = stride;
  }
  // one line: its stride is never used, but has to be one that TMA accepts
  if (p.rows == 1) p.x_rs = round8(p.inner);
  if (p.w_ks == 1 && p.outer == 1) p.w_ns = round8(p.inner);
  if (p.w_ks != 1 && p.inner == 1) p.w_ks = round8(p.outer);
  return run_tc(kKind, p, dtype, sm_count(), stream);
}

// Vocabulary records per row that the call's kernel leaves.
int vocab_parts(const Problem& p, int32_t dtype) {
  if (dtype != RLT_F32) return tc_vocab_parts(p, sm_count());
  return ceil_div(p.outer, fma_tile(p.rows, p.outer) == 2 ? 128 : 64);
}

bool known(int32_t dtype) { return dtype == RLT_F32 || dtype == RLT_F16 || dtype == RLT_BF16; }

int check(int32_t dtype, int32_t rows, int32_t inner, int32_t outer, int32_t act, int64_t w_ns,
          int64_t w_ks) {
  if (!known(dtype)) return RLT_E_DTYPE;
  if (rows < 0 || inner < 1 || outer < 0 || act < RLT_ACT_NONE || act > RLT_ACT_SIGMOID)
    return RLT_E_SHAPE;
  if (w_ns != 1 && w_ks != 1) return RLT_E_SHAPE;
  return RLT_OK;
}

Problem problem(const void* x, const void* w, int32_t rows, int32_t inner, int32_t outer,
                int64_t x_rs, int64_t w_ns, int64_t w_ks) {
  Problem p{};
  p.x = x;
  p.w = w;
  p.rows = rows;
  p.inner = inner;
  p.outer = outer;
  p.x_rs = x_rs;
  p.w_ns = w_ns;
  p.w_ks = w_ks;
  return p;
}

const void* up_rows(const void* weight, int32_t dtype, int32_t out_features, int64_t w_ns) {
  return static_cast<const char*>(weight) + w_ns * out_features * (dtype == RLT_F32 ? 4 : 2);
}

size_t parts_bytes(const Problem& p, int32_t dtype) {
  return static_cast<size_t>(p.rows) * vocab_parts(p, dtype) * sizeof(VocabPart);
}

}  // namespace
}  // namespace proj
}  // namespace rlt

using namespace rlt;
using namespace rlt::proj;

extern "C" size_t rlt_linear_workspace_bytes(const void* x, const void* weight, int32_t dtype,
                                             int32_t rows, int32_t in_features,
                                             int32_t out_features, int32_t gated,
                                             int64_t x_row_stride, int64_t weight_out_stride,
                                             int64_t weight_in_stride) {
  if (check(dtype, rows, in_features, out_features, RLT_ACT_NONE, weight_out_stride,
            weight_in_stride) ||
      rows == 0 || out_features == 0)
    return 0;
  Problem p = problem(x, weight, rows, in_features, out_features, x_row_stride, weight_out_stride,
                      weight_in_stride);
  if (gated) p.w_up = up_rows(weight, dtype, out_features, weight_out_stride);
  return copies_bytes(p, dtype);
}

extern "C" int rlt_linear(const void* x, const void* weight, const void* bias,
                          const void* residual, void* out, void* workspace,
                          size_t workspace_bytes, int32_t* status, int32_t dtype, int32_t rows,
                          int32_t in_features, int32_t out_features, int32_t activation,
                          int64_t x_row_stride, int64_t weight_out_stride,
                          int64_t weight_in_stride, int64_t residual_row_stride,
                          int64_t out_row_stride, void* stream) {
  if (const int rc = check(dtype, rows, in_features, out_features, activation, weight_out_stride,
                           weight_in_stride))
    return rc;
  if (rows == 0 || out_features == 0) return RLT_OK;
  Problem p = problem(x, weight, rows, in_features, out_features, x_row_stride, weight_out_stride,
                      weight_in_stride);
  p.bias = bias;
  p.residual = residual;
  p.out = out;
  p.status = status;
  p.act = activation;
  p.r_rs = residual_row_stride;
  p.o_rs = out_row_stride;
  const size_t need = copies_bytes(p, dtype);
  if (need > 0 && (!aligned16(workspace) || workspace == nullptr || workspace_bytes < need))
    return RLT_E_WORKSPACE;
  return dispatch<kLinear>(p, dtype, static_cast<char*>(workspace),
                           static_cast<cudaStream_t>(stream));
}

extern "C" int rlt_gated_linear(const void* x, const void* weight, void* out, void* workspace,
                                size_t workspace_bytes, int32_t* status, int32_t dtype,
                                int32_t rows, int32_t in_features, int32_t out_features,
                                int32_t activation, int64_t x_row_stride,
                                int64_t weight_out_stride, int64_t weight_in_stride,
                                int64_t out_row_stride, void* stream) {
  if (const int rc = check(dtype, rows, in_features, out_features, activation, weight_out_stride,
                           weight_in_stride))
    return rc;
  if (rows == 0 || out_features == 0) return RLT_OK;
  Problem p = problem(x, weight, rows, in_features, out_features, x_row_stride, weight_out_stride,
                      weight_in_stride);
  p.w_up = up_rows(weight, dtype, out_features, weight_out_stride);
  p.out = out;
  p.status = status;
  p.act = activation;
  p.o_rs = out_row_stride;
  const size_t need = copies_bytes(p, dtype);
  if (need > 0 && (!aligned16(workspace) || workspace == nullptr || workspace_bytes < need))
    return RLT_E_WORKSPACE;
  return dispatch<kGated>(p, dtype, static_cast<char*>(workspace),
                          static_cast<cudaStream_t>(stream));
}

extern "C" size_t rlt_vocab_head_workspace_bytes(const void* hidden, const void* weight,
                                                 int32_t dtype, int32_t rows, int32_t in_features,
                                                 int32_t vocab, int64_t hidden_row_stride,
                                                 int64_t weight_out_stride,
                                                 int64_t weight_in_stride) {
  if (check(dtype, rows, in_features, vocab, RLT_ACT_NONE, weight_out_stride, weight_in_stride) ||
      rows == 0 || vocab == 0)
    return 0;
  const Problem p = problem(hidden, weight, rows, in_features, vocab, hidden_row_stride,
                            weight_out_stride, weight_in_stride);
  return parts_bytes(p, dtype) + copies_bytes(p, dtype);
}

extern "C" int rlt_vocab_head(const void* hidden, const void* weight, const int64_t* tokens,
                              int64_t* out_tokens, float* logprobs, void* workspace,
                              size_t workspace_bytes, int32_t* status, int32_t dtype, int32_t rows,
                              int32_t in_features, int32_t vocab, int64_t hidden_row_stride,
                              int64_t weight_out_stride, int64_t weight_in_stride, void* stream) {
  if (const int rc = check(dtype, rows, in_features, vocab, RLT_ACT_NONE, weight_out_stride,
                           weight_in_stride))
    return rc;
  if (vocab == 0) return RLT_E_SHAPE;
  if (rows == 0) return RLT_OK;
  Problem p = problem(hidden, weight, rows, in_features, vocab, hidden_row_stride,
                      weight_out_stride, weight_in_stride);
  const size_t parts = parts_bytes(p, dtype);
  if (workspace == nullptr || !aligned16(workspace) ||
      workspace_bytes < parts + copies_bytes(p, dtype))
    return RLT_E_WORKSPACE;
  p.status = status;
  p.tokens = tokens;
  p.parts = static_cast<VocabPart*>(workspace);
  p.tiles = vocab_parts(p, dtype);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (const int rc = dispatch<kVocab>(p, dtype, static_cast<char*>(workspace) + parts, s))
    return rc;
  vocab_join_kernel<<<ceil_div(rows, 8), 256, 0, s>>>(p.parts, tokens, out_tokens, logprobs,
                                                      status, rows, p.tiles, vocab);
  return launch_status(cudaGetLastError());
}
