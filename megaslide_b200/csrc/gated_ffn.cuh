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
  kGate = 1,   // out = act(g) * u of the two accumulators g, u (bias added); kept_out receives u act'(g) and act(g)
  kDgate = 2,  // acc is the gradient of h: dgu = acc times each of the two kept values
};

// C[M, N] = sum_k A(m, k) B(n, k).  a_major / b_major: the contiguous axis is m / n instead of k (the operand
// is stored [K, M] / [K, N]).  kGate: B holds 2N rows, row n for g and row N + n for u.
struct Product {
  const void* a;
  const void* b;
  long long lda, ldb, ldo;
  void* out;
  const void* bias;  // [N] (kGate: [2N]) or NULL
  const void* kept;  // kDgate: u act'(g), then act(g), [M, 2N]
  void* kept_out;    // kGate: [M, 2N] or NULL
  uint8_t* low;      // bf16: the next 8 bits of the kept factors (read or written), [M, 2, low_width(N)]
  long long M, N, K;
  int dtype, act, epilogue;
  bool a_major, b_major;
  uint32_t* status;
  float* partial;  // workspace of tiles that are cut along k
  size_t partial_bytes;
};

// The factors that the forward keeps for the backward.  float32: as they are.  bf16: 24 bits of float32's 32, the upper 16
// in `kept`, the next 8 in `low`, the rest cut off.  They are no operand of the tensor cores, and rounded to bf16 they put a
// third rounding into the gradients, beside those of the gradients of g and u (an operand) and of the result: 0.0029
// of the result in the 2-norm, where the two leave 0.0024.  All 32 bits would be another quarter of their bytes for nothing
// that a bf16 result shows.  Reading puts the low byte into the last 8 bits as well: on average the middle of what was
// cut off, and infinities, NaN and short numbers stay what they were.
__host__ __device__ __forceinline__ long long low_width(long long N) { return (N + 15) / 16 * 16; }

// one factor of one row, by the element; `which`: 0 u act'(g), 1 act(g)
template <typename T>
struct KeptRow {
  T* at;
  uint8_t* low;
  long long N, W;

  __device__ __forceinline__ KeptRow(const void* kept, const uint8_t* low_rows, long long row, long long n, long long N_)
      : at(static_cast<T*>(const_cast<void*>(kept)) + row * 2 * N_ + n), low(nullptr), N(N_), W(0) {
    if constexpr (sizeof(T) == 2) {
      W = low_width(N_);
      low = const_cast<uint8_t*>(low_rows) + row * 2 * W + n;
    }
  }
  __device__ __forceinline__ void put(int which, float v) const {
    if constexpr (sizeof(T) == 4) {
      at[which * N] = v;
    } else {
      const uint32_t b = __float_as_uint(v);
      reinterpret_cast<uint16_t*>(at)[which * N] = static_cast<uint16_t>(b >> 16);
      low[which * W] = static_cast<uint8_t>(b >> 8);
    }
  }
  __device__ __forceinline__ float get(int which) const {
    if constexpr (sizeof(T) == 4) {
      return at[which * N];
    } else {
      const uint32_t b = low[which * W];
      return __uint_as_float(static_cast<uint32_t>(reinterpret_cast<const uint16_t*>(at)[which * N]) << 16 | b << 8 | b);
    }
  }
};

// the same by words: the upper halves of two factors, the low bytes of four, and element j of both
__device__ __forceinline__ uint32_t kept_high(float a, float b) { return __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x7632); }
__device__ __forceinline__ uint32_t kept_low(float a, float b, float c, float d) {
  return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0051), __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0051), 0x5410);
}
template <int J>
__device__ __forceinline__ float kept_at(uint32_t high, uint32_t low) {  // J: place in the low word; its parity, that in the high word
  constexpr unsigned h = J & 1 ? 0x3200 : 0x1000, l = (4 + J) * 0x11;
  return __uint_as_float(__byte_perm(high, low, h | l));
}

// act(g) and its derivative, in float32, for results in float32.
__device__ __forceinline__ float act_value_grad(float g, int act, float& da) {
  if (act == MSL_ACT_SILU) {
    const float s = 1.f / (1.f + expf(-g));
    da = s * (1.f + g * (1.f - s));
    return g * s;
  }
  const float c = 0.5f * (1.f + erff(g * 0.7071067811865476f));
  da = fmaf(g * 0.3989422804014327f, expf(-0.5f * g * g), c);
  return g * c;
}

// The same for results in bf16, in a third of the instructions: the epilogues of the tensor-core products have
// about 150 clocks for a row of 32 elements before they hold up the multiplications.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float sigmoid_fast(float g) { return __fdividef(1.f, 1.f + fast_exp2(-1.4426950408889634f * g)); }
// Normal distribution function and, by e, exp(-g^2/2): for x = |g| the tail is exp(-x^2/2) q(t), t = 1/(1 + 0.38 x),
// where q is a minimax polynomial (least largest relative error on [0, 14], by linear programming) of
// exp(x^2/2) erfc(x/sqrt 2)/2: within 3.6e-5 of the tail, 2^-15.
__device__ __forceinline__ float normal_cdf_fast(float g, float& e) {
  const float x = fabsf(g);
  const float t = __fdividef(1.f, fmaf(0.38f, x, 1.f));
  e = fast_exp2(-0.7213475204444817f * g * g);
  float q = fmaf(t, -0.08992771633985343f, 0.18887508919166987f);
  q = fmaf(t, q, 0.09198074100439507f);
  q = fmaf(t, q, 0.15782920020547297f);
  q = fmaf(t, q, 0.15122516174542605f);
  const float tail = q * t * e;
  return g < 0.f ? tail : 1.f - tail;
}
template <int ACT>
__device__ __forceinline__ float act_fast(float g) {
  if (ACT == MSL_ACT_SILU) return g * sigmoid_fast(g);
  float e;
  return g * normal_cdf_fast(g, e);
}
template <int ACT>
__device__ __forceinline__ float act_grad_fast(float g, float& da) {
  if (ACT == MSL_ACT_SILU) {
    const float s = sigmoid_fast(g), a = g * s;
    da = fmaf(a, 1.f - s, s);
    return a;
  }
  float e;
  const float c = normal_cdf_fast(g, e);
  da = fmaf(g * 0.3989422804014327f, e, c);
  return g * c;
}

// Tensor-core form (gated_ffn_tc.cu), and whether the operands allow it.
bool tc_applies(const Product& p);
size_t tc_partial_bytes(long long M, long long N, long long K, int epilogue, bool b_major);
cudaError_t launch_product_tc(const Product& p, cudaStream_t s);

// Form for a few rows (gated_ffn_rows.cu): the forward's two products, launched one after the other.
constexpr int kMostRows = 16, kMostRowsF32 = 8;
long long rows_most(int dtype, long long weights);  // rows up to which it is taken, by the elements of the first product's weights
bool rows_apply(const Product& p);
cudaError_t launch_product_rows(const Product& p, cudaStream_t s);
// CUDA-core form for float32, few rows or small products (gated_ffn_skinny.cu).
size_t skinny_bytes(long long M, long long N, long long K, int epilogue, bool a_major);
cudaError_t launch_product_skinny(const Product& p, cudaStream_t s);
cudaError_t launch_skinny_join(const Product& p, int shares, cudaStream_t s);  // shares of k in p.partial, and the epilogue
// Tensor-core form for few rows of float32 (gated_ffn_few.cu), and the shapes it takes where the operands lie on 16 bytes.
constexpr int kMostRowsFew = 64;
bool few_shape(long long M, long long cols, long long K, bool a_major, bool b_major);
bool few_apply(const Product& p);
size_t few_bytes(long long M, long long N, long long K, int epilogue);
cudaError_t launch_product_few(const Product& p, cudaStream_t s);
// Tensor-core form for float32 and for widths that are no multiple of 8 (gated_ffn_planes.cu): the operands as
// planes [planes][rows][cols padded to 8] of planes_bytes, written by launch_planes from rows as they are stored.
bool planes_apply(const Product& p);
size_t planes_bytes(int dtype, long long rows, long long cols);
size_t planes_partial_bytes(int dtype, long long M, long long N, long long K, int epilogue);
struct PlaneJob {
  const void* x;
  long long ld, rows, cols;
  void* out;
};
cudaError_t launch_planes(int dtype, const PlaneJob* jobs, int count, cudaStream_t s);  // one or two
// dh: float32 [M, N] for the gradient of h of a kDgate product in bf16
cudaError_t launch_product_planes(const Product& p, const void* pa, const void* pb, float* dh, cudaStream_t s);

}  // namespace ffn
}  // namespace msl
