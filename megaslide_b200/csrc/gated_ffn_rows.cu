// The gated feed-forward block's forward products for a few rows (single tokens up to kMostRows): the weights are
// read once, at the speed of the memory, and the rows of x stay in the caches.
//
// One row of bf16, or up to 8 of float32 (rows_most): a warp takes two rows of the weights (the gate's and the other
// projection's of one hidden element, or two of the second projection) and all rows of x; its lanes split k in
// 16-byte loads, four of each weight row in flight before the first is used.  More rows of bf16: mma.sync, below.
// Where there are fewer pairs of rows than warps the GPU holds, several warps share a pair's k.  Sums are float32,
// joined in a fixed order.  The second projection is launched so that it may start while the first still
// runs: it loads weights first and waits for h only then.
//
// h is rounded to bf16 here too, though one row's second projection could read it unrounded: a token's result then is the
// same whether it comes alone or among others, and what the backward reads is what the forward used.
//
// What bounds it: 1 x 1152 x 4608 in bf16 (32 MB of weights, which the L2 cache holds) 10.3 us, 8 rows 12.3, 16 rows 16.4,
// both projections from a CUDA graph: the launches and one trip to the cache; 1 x 7168 x 28672 (1.23 GB) the memory, 249 us
// (by mma.sync 260, so one row does without; at the small size they are even).  The tensor cores' own form takes 28.7
// and 302 us for 17 rows.

#include "gated_ffn.cuh"

namespace msl {
namespace ffn {
namespace rows {

constexpr int kWarps = 8;

struct Args {
  const void* a;
  const void* b;
  const void* bias;
  void* out;
  void* kept_out;
  uint8_t* low;
  long long lda, ldb, ldo, N;
  int M, K, act, share;  // warps that share a pair of weight rows
};

template <typename T, int V>
__device__ __forceinline__ void dot(float& acc, const uint4& w, const uint4& x) {
  const T* const a = reinterpret_cast<const T*>(&w);
  const T* const b = reinterpret_cast<const T*>(&x);
#pragma unroll
  for (int i = 0; i < V; ++i) acc = fmaf(to_f32<T>(a[i]), to_f32<T>(b[i]), acc);
}

// Pairs of weight rows a warp takes: with more rows of x, more, so that a word of x serves several of them.
constexpr int pairs_of(int mr) { return mr >= 8 ? 4 : mr >= 4 ? 2 : 1; }

template <typename T, int MR, int EPI>
__global__ void __launch_bounds__(32 * kWarps) rows_kernel(const __grid_constant__ Args P) {
  constexpr int V = 16 / static_cast<int>(sizeof(T)), NP = pairs_of(MR), U = MR >= 8 ? 1 : MR >= 4 ? 2 : 4;
  __shared__ float part[kWarps][2 * NP * MR];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slot = warp % P.share;
  const long long group = static_cast<long long>(blockIdx.x) * (kWarps / P.share) + warp / P.share;
  long long n[NP][2];
  bool in[NP][2];
  const uint4* w_at[NP][2];
#pragma unroll
  for (int p = 0; p < NP; ++p) {
    const long long pair = group * NP + p;
    n[p][0] = EPI == kGate ? pair : 2 * pair;
    n[p][1] = EPI == kGate ? P.N + pair : 2 * pair + 1;
    in[p][0] = n[p][0] < P.N;
    in[p][1] = EPI == kGate ? in[p][0] : n[p][1] < P.N;
#pragma unroll
    for (int i = 0; i < 2; ++i) w_at[p][i] = reinterpret_cast<const uint4*>(static_cast<const T*>(P.b) + (in[p][i] ? n[p][i] : 0) * P.ldb);
  }
  const int words = P.K / V, step = 32 * P.share;
  float acc[NP][2][MR];
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int m = 0; m < MR; ++m) acc[p][0][m] = acc[p][1][m] = 0.f;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  bool waited = EPI == kGate;
  for (int c = slot * 32 + lane; c - lane < words; c += U * step) {
    uint4 w[U][NP][2];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int i = 0; i < 2; ++i) w[u][p][i] = in[p][i] && c + u * step < words ? __ldg(w_at[p][i] + c + u * step) : zero;
    if (!waited) {  // h is the kernel's before
      cudaGridDependencySynchronize();
      waited = true;
    }
#pragma unroll
    for (int m = 0; m < MR; ++m) {
      if (m >= P.M) break;
      const uint4* const x = reinterpret_cast<const uint4*>(static_cast<const T*>(P.a) + m * P.lda);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (c + u * step >= words) continue;
        const uint4 v = x[c + u * step];
#pragma unroll
        for (int p = 0; p < NP; ++p) {
          dot<T, V>(acc[p][0][m], w[u][p][0], v);
          dot<T, V>(acc[p][1][m], w[u][p][1], v);
        }
      }
    }
  }
  if (EPI == kGate) cudaTriggerProgrammaticLaunchCompletion();
  else if (!waited) cudaGridDependencySynchronize();
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int m = 0; m < MR; ++m) {
        float t = acc[p][i][m];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(kFull, t, o);
        if (lane == 0) part[warp][(p * 2 + i) * MR + m] = t;
      }
  __syncthreads();
  // lane: a pair and a row of x
  const int p = lane / MR, m = lane - p * MR;
  if (slot != 0 || p >= NP || m >= P.M) return;
  const long long pair = group * NP + p, n0 = EPI == kGate ? pair : 2 * pair, n1 = EPI == kGate ? P.N + pair : 2 * pair + 1;
  if (n0 >= P.N) return;
  const bool in1 = EPI == kGate || n1 < P.N;
  float s[2] = {0.f, 0.f};
  for (int k = 0; k < P.share; ++k) {
    s[0] += part[warp + k][p * 2 * MR + m];
    s[1] += part[warp + k][(p * 2 + 1) * MR + m];
  }
  const T* const bias = static_cast<const T*>(P.bias);
  if (bias) {
    s[0] += to_f32<T>(bias[n0]);
    if (in1) s[1] += to_f32<T>(bias[n1]);
  }
  T* const out = static_cast<T*>(P.out) + m * P.ldo;
  if (EPI == kGate) {
    float da;
    const float a = act_value_grad(s[0], P.act, da);
    out[n0] = from_f32<T>(a * s[1]);
    if (P.kept_out) {
      const KeptRow<T> kept(P.kept_out, P.low, m, n0, P.N);
      kept.put(0, s[1] * da);
      kept.put(1, a);
    }
  } else {
    out[n0] = from_f32<T>(s[0]);
    if (in1) out[n1] = from_f32<T>(s[1]);
  }
}

template <typename T, int MR, int EPI>
cudaError_t launch(Args a, cudaStream_t s) {
  const long long pairs = EPI == kGate ? a.N : (a.N + 1) / 2, groups = (pairs + pairs_of(MR) - 1) / pairs_of(MR);
  // warps enough for every SM to hold two dozen, as long as each still has a few loads of its own
  a.share = 1;
  while (a.share < kWarps && groups * a.share < 24LL * sm_count() && a.K * static_cast<long long>(sizeof(T)) / 16 > 64LL * a.share) a.share *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((groups + kWarps / a.share - 1) / (kWarps / a.share)));
  cfg.blockDim = dim3(32 * kWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = EPI == kGate ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, rows_kernel<T, MR, EPI>, a);
}

template <typename T, int EPI>
cudaError_t by_rows(const Args& a, cudaStream_t s) {
  if (a.M == 1) return launch<T, 1, EPI>(a, s);
  if (a.M == 2) return launch<T, 2, EPI>(a, s);
  return a.M <= 4 ? launch<T, 4, EPI>(a, s) : launch<T, 8, EPI>(a, s);
}

// bf16, up to 8 * NT rows: 16 rows of the weights a warp (the gate: 8 hidden elements, rows 0-7 the gate's and 8-15
// the other projection's, so both end in one thread) against the rows of x, by mma.sync.  A thread's fragments
// are 16 adjacent bytes of a row: the same 8 k of the weights and of x, in whatever place the instruction's own
// order of k has them, so nothing is shuffled or converted.  (tcgen05 would need 128 rows of operands in shared
// memory for this; here the memory is the limit.)
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

constexpr int kMmaWarps = 16;

template <int NT, int EPI>
__global__ void __launch_bounds__(32 * kMmaWarps) rows_mma_kernel(const __grid_constant__ Args P) {
  using T = __nv_bfloat16;
  constexpr int U = 4;
  __shared__ float part[kMmaWarps][NT * 4][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int slot = warp % P.share;
  const long long group = static_cast<long long>(blockIdx.x) * (kMmaWarps / P.share) + warp / P.share;
  const long long n0 = EPI == kGate ? group * 8 + g : group * 16 + g, n1 = EPI == kGate ? P.N + n0 : n0 + 8;
  const bool in0 = n0 < P.N, in1 = EPI == kGate ? in0 : n1 < P.N;
  const T* const w0 = static_cast<const T*>(P.b) + (in0 ? n0 : 0) * P.ldb + t * 8;
  const T* const w1 = static_cast<const T*>(P.b) + (in1 ? n1 : 0) * P.ldb + t * 8;
  const T* const x = static_cast<const T*>(P.a) + t * 8;
  float acc[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = 0.f;
  const uint4 zero = make_uint4(0, 0, 0, 0);
  bool waited = EPI == kGate;
  const int hop = 32 * P.share;
  for (int k = slot * 32; k < P.K; k += U * hop) {
    uint4 a[2][U], b[NT][U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = k + u * hop;
      const bool have = at + t * 8 < P.K;
      a[0][u] = have && in0 ? __ldg(reinterpret_cast<const uint4*>(w0 + at)) : zero;
      a[1][u] = have && in1 ? __ldg(reinterpret_cast<const uint4*>(w1 + at)) : zero;
    }
    if (!waited) {  // h is the kernel's before
      cudaGridDependencySynchronize();
      waited = true;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const int at = k + u * hop;
        b[i][u] = at + t * 8 < P.K && i * 8 + g < P.M ? *reinterpret_cast<const uint4*>(x + (i * 8 + g) * P.lda + at) : zero;
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        mma16816(acc[i], a[0][u].x, a[1][u].x, a[0][u].y, a[1][u].y, b[i][u].x, b[i][u].y);
        mma16816(acc[i], a[0][u].z, a[1][u].z, a[0][u].w, a[1][u].w, b[i][u].z, b[i][u].w);
      }
  }
  if (EPI == kGate) cudaTriggerProgrammaticLaunchCompletion();
  else if (!waited) cudaGridDependencySynchronize();
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) part[warp][i * 4 + j][lane] = acc[i][j];
  __syncthreads();
  if (slot != 0) return;
  const T* const bias = static_cast<const T*>(P.bias);
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int m = i * 8 + t * 2 + j;
      if (m >= P.M) continue;
      float v0 = 0.f, v1 = 0.f;  // weight rows g and g + 8
      for (int k = 0; k < P.share; ++k) {
        v0 += part[warp + k][i * 4 + j][lane];
        v1 += part[warp + k][i * 4 + 2 + j][lane];
      }
      if (bias) {
        v0 += in0 ? to_f32<T>(bias[n0]) : 0.f;
        v1 += in1 ? to_f32<T>(bias[n1]) : 0.f;
      }
      T* const out = static_cast<T*>(P.out) + m * P.ldo;
      if (EPI == kGate) {
        if (!in0) continue;
        float da;
        const float a = P.act == MSL_ACT_SILU ? act_grad_fast<MSL_ACT_SILU>(v0, da) : act_grad_fast<MSL_ACT_GELU>(v0, da);
        out[n0] = from_f32<T>(a * v1);
        if (P.kept_out) {
          const KeptRow<T> kept(P.kept_out, P.low, m, n0, P.N);
          kept.put(0, v1 * da);
          kept.put(1, a);
        }
      } else {
        if (in0) out[n0] = from_f32<T>(v0);
        if (in1) out[n1] = from_f32<T>(v1);
      }
    }
}

template <int NT, int EPI>
cudaError_t launch_mma(Args a, cudaStream_t s) {
  const long long per = EPI == kGate ? 8 : 16, groups = (a.N + per - 1) / per;
  a.share = 1;
  while (a.share < kMmaWarps && groups * a.share < 24LL * sm_count() && a.K > 64 * a.share) a.share *= 2;
  const int each = kMmaWarps / a.share;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>((groups + each - 1) / each));
  cfg.blockDim = dim3(32 * kMmaWarps);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = EPI == kGate ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, rows_mma_kernel<NT, EPI>, a);
}

}  // namespace rows

// More rows only while the caches hold the weights.  bf16, 7168 x 28672, 8, 9 and 16 rows: 281, 345 and 371 us, on the tensor
// cores 337, 329 and 299; 1152 x 4608 12.3, 14.4 and 16.4 against 28.7.  float32, 2, 3, 4 and 8 rows of 7168 x 28672: 449,
// 760, 1063 and 1556 us, by few_kernel 733, 737, 741 and 764; 1152 x 4608 16.5, 18.5, 22.5 and 36.8, by skinny_kernel 38.9.
long long rows_most(int dtype, long long weights) {
  const bool cached = weights < (1LL << 25);
  return dtype == MSL_DTYPE_F32 ? (cached ? kMostRowsF32 : 2) : cached ? kMostRows : kMostRows / 2;
}

bool rows_apply(const Product& p) {
  const long long es = p.dtype == MSL_DTYPE_BF16 ? 2 : 4;
  return p.M <= rows_most(p.dtype, p.N * p.K * (p.epilogue == kGate ? 2 : 1)) && !p.a_major && !p.b_major && p.epilogue != kDgate &&
         p.K * es % 16 == 0 && p.lda * es % 16 == 0 && p.ldb * es % 16 == 0 && multiple_of(p.a, 16) && multiple_of(p.b, 16) &&
         p.K <= (1 << 30) && p.N <= (1 << 30);
}

cudaError_t launch_product_rows(const Product& p, cudaStream_t s) {
  rows::Args a{};
  a.a = p.a; a.lda = p.lda;
  a.b = p.b; a.ldb = p.ldb;
  a.bias = p.bias;
  a.out = p.out; a.ldo = p.ldo;
  a.kept_out = p.kept_out;
  a.low = p.low;
  a.N = p.N;
  a.M = static_cast<int>(p.M);
  a.K = static_cast<int>(p.K);
  a.act = p.act;
  if (p.dtype == MSL_DTYPE_BF16 && a.M > 1) {
    if (a.M <= 8) return p.epilogue == kGate ? rows::launch_mma<1, kGate>(a, s) : rows::launch_mma<1, kPlain>(a, s);
    return p.epilogue == kGate ? rows::launch_mma<2, kGate>(a, s) : rows::launch_mma<2, kPlain>(a, s);
  }
  if (p.dtype == MSL_DTYPE_BF16)
    return p.epilogue == kGate ? rows::launch<__nv_bfloat16, 1, kGate>(a, s) : rows::launch<__nv_bfloat16, 1, kPlain>(a, s);
  return p.epilogue == kGate ? rows::by_rows<float, kGate>(a, s) : rows::by_rows<float, kPlain>(a, s);
}

}  // namespace ffn
}  // namespace msl
