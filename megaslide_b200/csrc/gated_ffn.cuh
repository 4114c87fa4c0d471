// Parameters and launch functions of the gated feed-forward block's products (gated_ffn.cu dispatches).
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "msl_abi.cuh"
#include "msl_common.cuh"

namespace msl {
namespace ffn {

// What a product does with its result.
enum Epilogue : int {
  kPlain = 0,  // out = acc + bias
  kGate = 1,   // out = act(g) * u of the two accumulators g, u (bias added); gu receives g and u
  kDgate = 2,  // acc is the gradient of h: dgu = [acc * u * act'(g), acc * act(g)] of the kept g, u
};

// C[M, N] = sum_k A(m, k) B(n, k).  a_major / b_major: the contiguous axis is m / n instead of k (the operand
// is stored [K, M] / [K, N]).  kGate: B holds 2N rows, row n for g and row N + n for u.
struct Product {
  const void* a;
  const void* b;
  long long lda, ldb, ldo;
  void* out;
  const void* bias;  // [N] (kGate: [2N]) or NULL
  const void* gu;    // kDgate: kept g and u, [M, 2N]
  void* gu_out;      // kGate: [M, 2N] or NULL
  long long M, N, K;
  int dtype, act, epilogue;
  bool a_major, b_major;
  uint32_t* status;
};

// act(g) and its derivative, in float32.  FAST: the exponential by __expf, whose error (about 2^-22 of the
// result for the sizes that matter) is far below the rounding of a bf16 result.
template <bool FAST>
__device__ __forceinline__ float act_exp(float x) { return FAST ? __expf(x) : expf(x); }
template <bool FAST>
__device__ __forceinline__ float act_value(float g, int act) {
  if (act == MSL_ACT_SILU) return g / (1.f + act_exp<FAST>(-g));
  return 0.5f * g * (1.f + erff(g * 0.7071067811865476f));
}
template <bool FAST>
__device__ __forceinline__ float act_value_grad(float g, int act, float& da) {
  if (act == MSL_ACT_SILU) {
    const float s = 1.f / (1.f + act_exp<FAST>(-g));
    da = s * (1.f + g * (1.f - s));
    return g * s;
  }
  const float c = 0.5f * (1.f + erff(g * 0.7071067811865476f));
  da = fmaf(g * 0.3989422804014327f, act_exp<FAST>(-0.5f * g * g), c);
  return g * c;
}

cudaError_t launch_product_simt(const Product& p, cudaStream_t s);
// Tensor-core form (gated_ffn_tc.cu), and whether the operands allow it.
bool tc_applies(const Product& p);
cudaError_t launch_product_tc(const Product& p, cudaStream_t s);

}  // namespace ffn
}  // namespace msl
