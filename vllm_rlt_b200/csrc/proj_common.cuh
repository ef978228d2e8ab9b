// What the projection kernels share: the problem as the host hands it to
// them, the activations, and the per-tile record of the vocabulary head.
#pragma once

#include "common.cuh"

namespace rlt {
namespace proj {

struct VocabPart;

// out[r, n] = act(x[r] . w[n] + bias[n]) + residual[r, n], or with kGated
// act(x[r] . w[n]) * (x[r] . w_up[n]). Strides in elements.
struct Problem {
  const void* x;
  const void* w;
  const void* w_up;  // gated: the rows of the up projection
  const void* bias;
  const void* residual;
  void* out;
  int32_t* status;
  int rows;
  int inner;
  int outer;  // output features (gated: of each half)
  int act;
  int64_t x_rs;
  int64_t w_ns;  // between output features
  int64_t w_ks;  // between input features
  int64_t r_rs;
  int64_t o_rs;
  // vocabulary head
  const int64_t* tokens;   // tokens to score, or NULL for the likeliest one
  VocabPart* parts;  // [rows, tiles]
  int tiles;
};

// One vocabulary tile's contribution to a row: the largest logit, where it is
// first reached, sum of exp(logit - largest), and the scored token's logit if
// it lies in the tile (0 otherwise).
struct VocabPart {
  float most;
  float sum;
  int32_t at;
  float chosen;
};

enum Kind { kLinear = 0, kGated = 1, kVocab = 2 };

constexpr float kLog2e = 1.4426950408889634f;

// Activations in fp32. For fp32 tensors through expf and a division; for
// 16-bit ones through the hardware exponential and reciprocal, whose relative
// error of about 2^-22 is far below the output's rounding (2^-8 for bf16,
// 2^-11 for fp16); a sigmoid below 2^-126 counts as 0. Gelu takes the
// complementary error function, since 1 + erf cancels for negative x (at -5 it
// has 4 bits left). NaN stays NaN in each; exp overflowing to infinity gives the
// limit (0), as the formulas do.
template <bool kPrecise>
__device__ __forceinline__ float sigmoid_times(float x, float z) {  // x / (1 + exp(-z))
  if constexpr (kPrecise) return __fdiv_rn(x, 1.f + expf(-z));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + ex2(-z * kLog2e)));
  return x * r;
}

template <bool kPrecise, int kAct>
__device__ __forceinline__ float activate(float x) {
  if constexpr (kAct == RLT_ACT_SILU) return sigmoid_times<kPrecise>(x, x);
  if constexpr (kAct == RLT_ACT_GELU) return 0.5f * x * erfcf(-x * 0.70710678f);
  if constexpr (kAct == RLT_ACT_GELU_TANH)  // (1 + tanh u) / 2 = 1 / (1 + exp(-2u))
    return sigmoid_times<kPrecise>(x, 1.5957691216f * (x + 0.044715f * x * x * x));
  if constexpr (kAct == RLT_ACT_RELU) return x < 0.f ? 0.f : x;
  if constexpr (kAct == RLT_ACT_SIGMOID) return sigmoid_times<kPrecise>(1.f, x);
  return x;
}

// Whether logit b at vocabulary entry j beats a at i: larger, or NaN as torch's
// argmax orders it (above every number), the lower entry on a tie.
__device__ __forceinline__ bool beats(float b, int j, float a, int i) {
  const bool an = a != a, bn = b != b;
  if (an || bn) return bn && (!an || j < i);
  return b > a || (b == a && j < i);
}

// Folds part b of a row into a. The sums are relative to their own part's
// largest logit; a part whose largest is -infinity has a sum of 0.
__device__ __forceinline__ void fold(VocabPart& a, const VocabPart& b) {
  const float m = fmaxf(a.most, b.most);  // drops a NaN; its sum is NaN already
  const float base = m == -INFINITY ? 0.f : m;
  a.sum = a.sum * expf(a.most - base) + b.sum * expf(b.most - base);
  if (beats(b.most, b.at, a.most, a.at)) {
    a.most = b.most;
    a.at = b.at;
  }
  a.chosen += b.chosen;
}

// Launch attributes of these kernels: the cluster, and leave to start before
// the stream's previous kernel has ended (they wait for it themselves).
inline unsigned launch_attributes(cudaLaunchAttribute (&attrs)[2], int cluster) {
  attrs[0] = {};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  if (cluster == 1) return 1;
  attrs[1] = {};
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  return 2;
}

// 16-bit operands, and fp32 ones, whose pointers and strides TMA accepts.
int run_tc(Kind kind, const Problem& p, int32_t dtype, int ctas, cudaStream_t stream);
int run_split(Kind kind, const Problem& p, int ctas, cudaStream_t stream);
// Vocabulary records per row that they leave.
int tc_vocab_parts(const Problem& p, int ctas);
int split_vocab_parts(const Problem& p);

}  // namespace proj
}  // namespace rlt
