// Projections with what follows them (sm_100a): the matrix product with bias,
// activation and residual in its epilogue, the gated product, and the
// vocabulary head that reduces its logits tile by tile.
//
// This file holds the C entries, the copies of operands that TMA cannot address
// as they are, and the join of the vocabulary tiles.
#include <atomic>

#include "proj_common.cuh"
#include "tc_ptx.cuh"

namespace rlt {
namespace proj {
namespace {

// Joins a row's vocabulary tiles, one CTA per row. A thread's records are all
// on their way before it folds the first (a warp per row with one record at a
// time took 11.5 us for 512 records, most of it waiting).
constexpr int kJoinThreads = 128, kJoinBatch = 4;

__global__ void __launch_bounds__(kJoinThreads) vocab_join_kernel(
    const VocabPart* parts, const int64_t* tokens, int64_t* out_tokens, float* logprobs,
    int32_t* status, int tiles, int vocab) {
  __shared__ VocabPart warps[kJoinThreads / 32];
  tc::pdl_launch_dependents();
  tc::pdl_wait();
  const int row = blockIdx.x, lane = threadIdx.x & 31;
  const float4* mine = reinterpret_cast<const float4*>(parts + static_cast<int64_t>(row) * tiles);
  const int64_t want = tokens != nullptr ? tokens[row] : -1;
  VocabPart a{-INFINITY, 0.f, INT32_MAX, 0.f};
  for (int first = threadIdx.x; first < tiles; first += kJoinThreads * kJoinBatch) {
    float4 r[kJoinBatch];
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i) {
      const int t = first + i * kJoinThreads;
      if (t < tiles) r[i] = mine[t];
    }
#pragma unroll
    for (int i = 0; i < kJoinBatch; ++i)
      if (first + i * kJoinThreads < tiles)
        fold(a, VocabPart{r[i].x, r[i].y, __float_as_int(r[i].z), r[i].w});
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    VocabPart b;
    b.most = __shfl_xor_sync(kFullMask, a.most, o);
    b.sum = __shfl_xor_sync(kFullMask, a.sum, o);
    b.at = __shfl_xor_sync(kFullMask, a.at, o);
    b.chosen = __shfl_xor_sync(kFullMask, a.chosen, o);
    fold(a, b);
  }
  if (lane == 0) warps[threadIdx.x >> 5] = a;
  __syncthreads();
  if (threadIdx.x != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinThreads / 32; ++w) fold(a, warps[w]);
  // the largest logit's own term is 1, however its sum was rounded; NaN stays
  const float normaliser = a.most == -INFINITY ? NAN : logf(a.sum < 1.f ? 1.f : a.sum);
  if (tokens == nullptr) {
    out_tokens[row] = a.at;
    logprobs[row] = -normaliser;
    return;
  }
  if (want >= vocab) raise_status(status, kStatusBadToken);
  logprobs[row] = want < 0 ? 0.f : want >= vocab ? NAN : a.chosen - a.most - normaliser;
}

int sm_count() {
  static std::atomic<int> count[64];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 148;
  int n = count[dev].load();
  if (n == 0) {
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
      n = 148;
    count[dev].store(n);
  }
  return n;
}

// ---- operands for TMA ----------------------------------------------------------

int elem_bytes(int32_t dtype) { return dtype == RLT_F32 ? 4 : 2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Elements rounded up to whole 16-byte units.
int64_t padded(int64_t n, int32_t dtype) {
  const int unit = 16 / elem_bytes(dtype);
  return (n + unit - 1) / unit * unit;
}

// What TMA asks of an operand of `lines` lines of `line` elements: a 16-byte
// aligned start and a stride of whole 16-byte units. A stride shorter than a
// line (a broadcast operand) is copied too.
bool tma_ready(const void* base, int line, int lines, int64_t stride, int32_t dtype) {
  return aligned16(base) &&
         (lines == 1 || (stride * elem_bytes(dtype) % 16 == 0 && stride >= line));
}

struct Layout {  // of the weights: lines along the contiguous dimension
  int line, lines;
  int64_t stride;
};
Layout weight_layout(const Problem& p) {
  return p.w_ks == 1 ? Layout{p.inner, p.outer, p.w_ns} : Layout{p.outer, p.inner, p.w_ks};
}

bool x_ready(const Problem& p, int32_t dtype) {
  return tma_ready(p.x, p.inner, p.rows, p.x_rs, dtype);
}
bool w_ready(const Problem& p, int32_t dtype) {
  const Layout l = weight_layout(p);
  return tma_ready(p.w, l.line, l.lines, l.stride, dtype) &&
         (p.w_up == nullptr || tma_ready(p.w_up, l.line, l.lines, l.stride, dtype));
}

size_t copies_bytes(const Problem& p, int32_t dtype) {
  const Layout l = weight_layout(p);
  const size_t es = elem_bytes(dtype);
  size_t bytes = 0;
  if (!x_ready(p, dtype)) bytes += padded(p.inner, dtype) * p.rows * es;
  if (!w_ready(p, dtype)) bytes += padded(l.line, dtype) * l.lines * es * (p.w_up ? 2 : 1);
  return bytes;
}

// dst[line][0 .. pitch) = src[line * stride ..][0 .. length); what lies past
// `length` is never read. U: an unsigned integer of the elements' size.
template <typename U>
__global__ void __launch_bounds__(256) align_kernel(const U* __restrict__ src,
                                                    U* __restrict__ dst, int length, int lines,
                                                    int64_t stride, int pitch) {
  constexpr int kUnit = 16 / sizeof(U);
  const int units = pitch / kUnit;
  // a warp takes 128 units of a line at a time
  const uint32_t chunks = (units + 127) / 128, lane = threadIdx.x & 31;
  const int64_t items = static_cast<int64_t>(chunks) * lines;
  for (int64_t item = blockIdx.x * 8LL + (threadIdx.x >> 5); item < items; item += gridDim.x * 8LL) {
    const int64_t line = items <= UINT32_MAX ? static_cast<uint32_t>(item) / chunks : item / chunks;
    const int first = static_cast<int>(item - line * chunks) * 128 + lane;
    const U* s = src + line * stride;
    U* d = dst + line * pitch;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int c = (first + q * 32) * kUnit;
      if (c >= pitch) continue;
      union {
        U v[kUnit];
        uint4 all;
      } t;
#pragma unroll
      for (int e = 0; e < kUnit; ++e) t.v[e] = c + e < length ? s[c + e] : static_cast<U>(0);
      st_vec(d + c, t.all);
    }
  }
}

int align_copy(const void*& base, int64_t& stride, int length, int lines, int32_t dtype, char*& at,
               cudaStream_t stream) {
  const int64_t pitch = padded(length, dtype);
  if (pitch > INT32_MAX) return RLT_E_SHAPE;
  const int64_t blocks = ((pitch * elem_bytes(dtype) / 16 + 127) / 128 * lines + 7) / 8;
  const unsigned grid =
      static_cast<unsigned>(blocks < 16 * sm_count() ? blocks : 16 * sm_count());
  if (dtype == RLT_F32)
    align_kernel<<<grid, 256, 0, stream>>>(static_cast<const uint32_t*>(base),
                                           reinterpret_cast<uint32_t*>(at), length, lines, stride,
                                           static_cast<int>(pitch));
  else
    align_kernel<<<grid, 256, 0, stream>>>(static_cast<const uint16_t*>(base),
                                           reinterpret_cast<uint16_t*>(at), length, lines, stride,
                                           static_cast<int>(pitch));
  base = at;
  stride = pitch;
  at += pitch * lines * elem_bytes(dtype);
  return launch_status(cudaGetLastError());
}

int dispatch(Kind kind, Problem p, int32_t dtype, char* copies, cudaStream_t stream) {
  if (!x_ready(p, dtype))
    if (const int rc = align_copy(p.x, p.x_rs, p.inner, p.rows, dtype, copies, stream)) return rc;
  if (!w_ready(p, dtype)) {
    const Layout l = weight_layout(p);
    int64_t stride = l.stride;
    if (p.w_up != nullptr) {
      if (const int rc = align_copy(p.w_up, stride, l.line, l.lines, dtype, copies, stream))
        return rc;
      stride = l.stride;
    }
    if (const int rc = align_copy(p.w, stride, l.line, l.lines, dtype, copies, stream)) return rc;
    (p.w_ks == 1 ? p.w_ns : p.w_ks) = stride;
  }
  // one line: its stride is never used, but has to be one that TMA accepts
  if (p.rows == 1) p.x_rs = padded(p.inner, dtype);
  if (p.w_ks == 1 && p.outer == 1) p.w_ns = padded(p.inner, dtype);
  if (p.w_ks != 1 && p.inner == 1) p.w_ks = padded(p.outer, dtype);
  return dtype == RLT_F32 ? run_split(kind, p, sm_count(), stream)
                          : run_tc(kind, p, dtype, sm_count(), stream);
}

// Vocabulary records per row that the call's kernel leaves.
int vocab_parts(const Problem& p, int32_t dtype) {
  return dtype == RLT_F32 ? split_vocab_parts(p) : tc_vocab_parts(p, sm_count());
}

bool known(int32_t dtype) { return dtype == RLT_F32 || dtype == RLT_F16 || dtype == RLT_BF16; }

int check(int32_t dtype, int32_t rows, int32_t inner, int32_t outer, int32_t act, int64_t w_ns,
          int64_t w_ks) {
  if (!known(dtype)) return RLT_E_DTYPE;
  if (rows < 0 || inner < 1 || outer < 0 || act < RLT_ACT_NONE || act > RLT_ACT_SIGMOID)
    return RLT_E_SHAPE;
  if (rows > RLT_PROJ_MAX_SIZE || inner > RLT_PROJ_MAX_SIZE || outer > RLT_PROJ_MAX_SIZE)
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
  return dispatch(kLinear, p, dtype, static_cast<char*>(workspace),
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
  return dispatch(kGated, p, dtype, static_cast<char*>(workspace),
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
  if (const int rc = dispatch(kVocab, p, dtype, static_cast<char*>(workspace) + parts, s))
    return rc;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(rows));
  cfg.blockDim = dim3(kJoinThreads);
  cfg.stream = s;
  cudaLaunchAttribute attrs[2];
  cfg.attrs = attrs;
  cfg.numAttrs = launch_attributes(attrs, 1);
  return launch_status(cudaLaunchKernelEx(&cfg, vocab_join_kernel,
                                          static_cast<const VocabPart*>(p.parts), tokens,
                                          out_tokens, logprobs, status, p.tiles,
                                          static_cast<int>(vocab)));
}
