// The gated feed-forward block's float32 products on the CUDA cores, where making planes for the tensor cores
// (10 bytes an element of each operand, gated_ffn_planes.cu) would cost more than it saves: up to about a hundred
// rows, and small products (few rows of wide weights on 16 bytes: gated_ffn_few.cu).
//
// A block has 128 columns and 8 to 64 rows of the result and a share of k; the operands come through registers
// into shared memory ([k][row], [k][column]) while the last tile is multiplied, two columns an instruction
// (fma.rn.f32x2).  Up to 16 rows a warp takes 8 rows x 128 columns and its own k of the tile (the weights are then
// read from shared memory once or twice, not by every warp), joined at the end; with more rows a thread has 2 x 8
// or 4 x 8 results of all k.  Shares of k leave their sums in the workspace; a second kernel joins them in
// order and does the epilogue.
//
// What bounds it: the weights' bytes up to about 16 rows, beyond that the multiplications.

#include "gated_ffn.cuh"

namespace msl {
namespace ffn {
namespace skinny {

constexpr int kTN = 128, kTK = 32;
constexpr int kPitchB = kTN + 4;

struct Args {
  const float* a;
  const float* b;
  float* out;  // [shares][M][N], or the result itself (share 0 alone)
  long long lda, ldb, ldo, M, N, K, kper, share_stride;
  int va, vb;  // operands in 16-byte loads
};

// four elements at p, of which `have` exist
__device__ __forceinline__ float4 load4(const float* p, long long have, int vec) {
  if (have >= 4 && vec) return __ldg(reinterpret_cast<const float4*>(p));
  float4 v;
  v.x = have > 0 ? __ldg(p) : 0.f;
  v.y = have > 1 ? __ldg(p + 1) : 0.f;
  v.z = have > 2 ? __ldg(p + 2) : 0.f;
  v.w = have > 3 ? __ldg(p + 3) : 0.f;
  return v;
}

__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}

// One operand's tile of W rows (of the result's rows or columns) x kTK, on its way through registers: NQ float4 a
// thread.  MAJOR: stored [k][row].
template <int W, bool MAJOR>
struct Side {
  static constexpr int NQ = W * kTK / 4 / 256 > 0 ? W * kTK / 4 / 256 : 1;
  float4 q[NQ];

  __device__ __forceinline__ void fetch(const float* p, long long ld, long long row0, long long rows, long long k0, long long k1, int vec) {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int e = i * 256 + threadIdx.x;
      if (W * kTK / 4 < 256 && e >= W * kTK / 4) continue;
      if (MAJOR) {
        const int k = e / (W / 4), r = e % (W / 4) * 4;
        q[i] = k0 + k < k1 ? load4(p + (k0 + k) * ld + row0 + r, rows - row0 - r, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
      } else {
        const int r = e / (kTK / 4), k = e % (kTK / 4) * 4;
        q[i] = row0 + r < rows ? load4(p + (row0 + r) * ld + k0 + k, k1 - k0 - k, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
    }
  }
  template <int PITCH>
  __device__ __forceinline__ void put(float* tile) const {
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
      const int e = i * 256 + threadIdx.x;
      if (W * kTK / 4 < 256 && e >= W * kTK / 4) continue;
      if (MAJOR) {
        const int k = e / (W / 4), r = e % (W / 4) * 4;
        *reinterpret_cast<float4*>(tile + k * PITCH + r) = q[i];
      } else {
        const int r = e / (kTK / 4), k = e % (kTK / 4) * 4;
        tile[k * PITCH + r] = q[i].x;
        tile[(k + 1) * PITCH + r] = q[i].y;
        tile[(k + 2) * PITCH + r] = q[i].z;
        tile[(k + 3) * PITCH + r] = q[i].w;
      }
    }
  }
};

__device__ __forceinline__ void put_row4(const Args& P, float* out, long long row, long long col, float4 v) {
  if (row >= P.M || col >= P.N) return;
  float* const to = out + row * P.ldo + col;
  if (col + 4 <= P.N && ((reinterpret_cast<uintptr_t>(to) & 15) == 0)) {
    *reinterpret_cast<float4*>(to) = v;
    return;
  }
  to[0] = v.x;
  if (col + 1 < P.N) to[1] = v.y;
  if (col + 2 < P.N) to[2] = v.z;
  if (col + 3 < P.N) to[3] = v.w;
}

template <int TM, bool AM, bool BM>
__global__ void __launch_bounds__(256, TM == 64 ? 2 : 3) skinny_kernel(const __grid_constant__ Args P) {
  constexpr int kPitchA = TM + 4;
  constexpr int kTile = kTK * (kPitchA + kPitchB);
  extern __shared__ __align__(16) float sm[];
  const long long m0 = static_cast<long long>(blockIdx.x) * TM, n0 = static_cast<long long>(blockIdx.y) * kTN;
  const long long k0 = blockIdx.z * P.kper, k1 = min(P.K, k0 + P.kper);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  constexpr bool FEW = TM <= 16;
  constexpr int R = FEW ? 8 : TM / 16, Q = FEW ? 2 : 4;  // a thread's rows, column pairs
  constexpr int KW = FEW ? 64 / TM : 1;                 // warps that share the k of a tile's 8 rows
  float2 acc[R][Q];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < Q; ++j) acc[i][j] = make_float2(0.f, 0.f);
  Side<TM, AM> sa;
  Side<kTN, BM> sb;
  sa.fetch(P.a, P.lda, m0, P.M, k0, k1, P.va);
  sb.fetch(P.b, P.ldb, n0, P.N, k0, k1, P.vb);
  int buf = 0;
  for (long long k = k0; k < k1; k += kTK, buf ^= 1) {
    float* const ta = sm + buf * kTile;
    float* const tb = ta + kTK * kPitchA;
    sa.template put<kPitchA>(ta);
    sb.template put<kPitchB>(tb);
    __syncthreads();
    if (k + kTK < k1) {
      sa.fetch(P.a, P.lda, m0, P.M, k + kTK, k1, P.va);
      sb.fetch(P.b, P.ldb, n0, P.N, k + kTK, k1, P.vb);
    }
    if constexpr (FEW) {
      const int first = warp / KW * 8;
#pragma unroll
      for (int i = 0; i < kTK / KW; ++i) {
        const int kk = i * KW + warp % KW;
        const float4 b = *reinterpret_cast<const float4*>(tb + kk * kPitchB + lane * 4);
        const float2 b0 = make_float2(b.x, b.y), b1 = make_float2(b.z, b.w);
#pragma unroll
        for (int r = 0; r < 8; r += 4) {
          const float4 a = *reinterpret_cast<const float4*>(ta + kk * kPitchA + first + r);
          const float av[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            acc[r + q][0] = fma2(make_float2(av[q], av[q]), b0, acc[r + q][0]);
            acc[r + q][1] = fma2(make_float2(av[q], av[q]), b1, acc[r + q][1]);
          }
        }
      }
    } else {
#pragma unroll 8
      for (int kk = 0; kk < kTK; ++kk) {
        float av[R];
        if constexpr (TM == 64) {
          const float4 a = *reinterpret_cast<const float4*>(ta + kk * kPitchA + ty * 4);
          av[0] = a.x; av[1] = a.y; av[2] = a.z; av[3] = a.w;
        } else {
          const float2 a = *reinterpret_cast<const float2*>(ta + kk * kPitchA + ty * 2);
          av[0] = a.x; av[1] = a.y;
        }
        const float4 b = *reinterpret_cast<const float4*>(tb + kk * kPitchB + tx * 4);
        const float4 c = *reinterpret_cast<const float4*>(tb + kk * kPitchB + 64 + tx * 4);
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float2 s = make_float2(av[r], av[r]);
          acc[r][0] = fma2(s, make_float2(b.x, b.y), acc[r][0]);
          acc[r][1] = fma2(s, make_float2(b.z, b.w), acc[r][1]);
          acc[r][2] = fma2(s, make_float2(c.x, c.y), acc[r][2]);
          acc[r][3] = fma2(s, make_float2(c.z, c.w), acc[r][3]);
        }
      }
    }
    // two tiles: the next put goes to the other, which every warp left before this iteration's barrier
  }
  float* const out = P.out + blockIdx.z * P.share_stride;
  if constexpr (FEW) {
    // the sums of the warps that share rows, through shared memory ([8 warps][8 rows][128]), in their order
    __syncthreads();
#pragma unroll
    for (int r = 0; r < 8; ++r)
      *reinterpret_cast<float4*>(sm + (warp * 8 + r) * kTN + lane * 4) = make_float4(acc[r][0].x, acc[r][0].y, acc[r][1].x, acc[r][1].y);
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TM / 8; ++i) {
      const int r = warp + 8 * i;  // of the tile
      float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int w = 0; w < KW; ++w) {
        const float4 v = *reinterpret_cast<const float4*>(sm + ((r / 8 * KW + w) * 8 + r % 8) * kTN + lane * 4);
        t.x += v.x; t.y += v.y; t.z += v.z; t.w += v.w;
      }
      put_row4(P, out, m0 + r, n0 + lane * 4, t);
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      put_row4(P, out, m0 + ty * R + r, n0 + tx * 4, make_float4(acc[r][0].x, acc[r][0].y, acc[r][1].x, acc[r][1].y));
      put_row4(P, out, m0 + ty * R + r, n0 + 64 + tx * 4, make_float4(acc[r][2].x, acc[r][2].y, acc[r][3].x, acc[r][3].y));
    }
  }
}

// Joins the shares of k in order and does the epilogue: a thread an element of the result (of h for the gate).
template <int EPI>
__global__ void __launch_bounds__(256) skinny_join_kernel(const float* __restrict__ partial, int shares, long long M, long long N, const float* bias,
                                                          const float* kept, float* kept_out, float* out, long long ldo, int act) {
  const long long cols = EPI == kGate ? 2 * N : N, stride = M * cols;
  const long long i = blockIdx.x * 256LL + threadIdx.x;
  if (i >= M * N) return;
  const long long m = i / N, n = i - m * N;
  float v = 0.f, u = 0.f;
#pragma unroll 4
  for (int s = 0; s < shares; ++s) {
    v += partial[s * stride + m * cols + n];
    if (EPI == kGate) u += partial[s * stride + m * cols + N + n];
  }
  if (EPI == kPlain) {
    out[m * ldo + n] = v + (bias ? bias[n] : 0.f);
  } else if (EPI == kGate) {
    v += bias ? bias[n] : 0.f;
    u += bias ? bias[N + n] : 0.f;
    float da;
    const float a = act_value_grad(v, act, da);
    if (kept_out) {
      kept_out[m * 2 * N + n] = u * da;
      kept_out[m * 2 * N + N + n] = a;
    }
    out[m * ldo + n] = a * u;
  } else {
    out[m * 2 * N + n] = v * kept[m * 2 * N + n];
    out[m * 2 * N + N + n] = v * kept[m * 2 * N + N + n];
  }
}

// The weights' gradients of up to KM rows, out[m][n] = sum_k a[k][m] b[k][n]: bound by the bytes of the result.  A thread
// has 4 columns, whose b stays in registers, and writes them for kOuterRows rows; a comes through shared memory.
// dw_out of 7168 x 25088 (0.72 GB), 1, 4 and 13 rows: 109, 111 and 159 us (6.6 TB/s of writes with one row), by
// skinny_kernel 280, 283 and 293; 1152 x 4608 6.2, 6.2 and 8.2, 12.3, 12.3 and 12.4.  With 30 rows it was 326 and 16.4 against
// 314 and 14.3, so beyond 16 skinny_kernel has them.
constexpr int kOuterRows = 32;

template <int KM>
__global__ void __launch_bounds__(256) outer_kernel(const __grid_constant__ Args P) {
  __shared__ __align__(16) float as[kOuterRows][KM];
  const long long m0 = static_cast<long long>(blockIdx.x) * kOuterRows, n = (blockIdx.y * 256LL + threadIdx.x) * 4;
  const int K = static_cast<int>(P.K);
  for (int e = threadIdx.x; e < kOuterRows * KM; e += 256) {
    const int k = e / kOuterRows, m = e % kOuterRows;
    as[m][k] = k < K && m0 + m < P.M ? __ldg(P.a + k * P.lda + m0 + m) : 0.f;
  }
  const bool in = n < P.N;
  float2 b[KM][2];
#pragma unroll
  for (int k = 0; k < KM; ++k) {
    const float4 v = in && k < K ? __ldg(reinterpret_cast<const float4*>(P.b + k * P.ldb + n)) : make_float4(0.f, 0.f, 0.f, 0.f);
    b[k][0] = make_float2(v.x, v.y);
    b[k][1] = make_float2(v.z, v.w);
  }
  __syncthreads();
  if (!in) return;
  const int rows = static_cast<int>(min(static_cast<long long>(kOuterRows), P.M - m0));
  float* out = P.out + m0 * P.ldo + n;
#pragma unroll 4
  for (int m = 0; m < rows; ++m, out += P.ldo) {
    float2 s = make_float2(0.f, 0.f), t = s;
#pragma unroll
    for (int k = 0; k < KM; ++k) {
      const float2 v = make_float2(as[m][k], as[m][k]);
      s = fma2(v, b[k][0], s);
      t = fma2(v, b[k][1], t);
    }
    *reinterpret_cast<float4*>(out) = make_float4(s.x, s.y, t.x, t.y);
  }
}

struct Plan {
  int tm, shares;
  long long kper;
  size_t bytes;
};

// Rows of a tile by the result's rows; k is shared until every SM has about two blocks, 128 k apiece at least.  The
// weights' gradients (rows the summed axis) have tiles enough and go straight to their result.
Plan plan(long long M, long long cols, long long K, bool direct) {
  Plan p{};
  p.tm = M <= 8 ? 8 : M <= 16 ? 16 : M <= 32 || (M > 64 && M <= 96) ? 32 : 64;
  const long long tiles = (M + p.tm - 1) / p.tm * ((cols + kTN - 1) / kTN);
  long long shares = direct ? 1 : (2LL * sm_count() + tiles - 1) / tiles;
  const long long most = (K + 127) / 128;
  if (shares > most) shares = most;
  if (shares > 64) shares = 64;
  p.kper = ((K + shares - 1) / shares + kTK - 1) / kTK * kTK;
  p.shares = static_cast<int>((K + p.kper - 1) / p.kper);
  p.bytes = direct ? 0 : sizeof(float) * static_cast<size_t>(p.shares) * static_cast<size_t>(M) * static_cast<size_t>(cols);
  return p;
}

template <int TM, bool AM, bool BM>
cudaError_t launch(const Args& a, int shares, cudaStream_t s) {
  constexpr size_t tiles = sizeof(float) * 2 * kTK * (TM + 4 + kPitchB), box = TM <= 16 ? sizeof(float) * 64 * kTN : 0;
  constexpr int smem = static_cast<int>(tiles > box ? tiles : box);
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(skinny_kernel<TM, AM, BM>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
  }
  const dim3 grid(static_cast<unsigned>((a.M + TM - 1) / TM), static_cast<unsigned>((a.N + kTN - 1) / kTN), static_cast<unsigned>(shares));
  skinny_kernel<TM, AM, BM><<<grid, 256, smem, s>>>(a);
  return cudaGetLastError();
}

template <int TM>
cudaError_t by_order(const Product& p, const Args& a, int shares, cudaStream_t s) {
  if (p.a_major) return launch<TM, true, true>(a, shares, s);
  return p.b_major ? launch<TM, false, true>(a, shares, s) : launch<TM, false, false>(a, shares, s);
}

}  // namespace skinny

size_t skinny_bytes(long long M, long long N, long long K, int epilogue, bool a_major) {
  return skinny::plan(M, epilogue == kGate ? 2 * N : N, K, a_major).bytes;
}

cudaError_t launch_skinny_join(const Product& p, int shares, cudaStream_t s) {
  const unsigned blocks = static_cast<unsigned>((p.M * p.N + 255) / 256);
  const float* const bias = static_cast<const float*>(p.bias);
  const float* const kept = static_cast<const float*>(p.kept);
  float* const kept_out = static_cast<float*>(p.kept_out);
  float* const out = static_cast<float*>(p.out);
  if (p.epilogue == kGate)
    skinny::skinny_join_kernel<kGate><<<blocks, 256, 0, s>>>(p.partial, shares, p.M, p.N, bias, kept, kept_out, out, p.ldo, p.act);
  else if (p.epilogue == kDgate)
    skinny::skinny_join_kernel<kDgate><<<blocks, 256, 0, s>>>(p.partial, shares, p.M, p.N, bias, kept, kept_out, out, p.ldo, p.act);
  else
    skinny::skinny_join_kernel<kPlain><<<blocks, 256, 0, s>>>(p.partial, shares, p.M, p.N, bias, kept, kept_out, out, p.ldo, p.act);
  count_launches(1);
  return cudaGetLastError();
}

cudaError_t launch_product_skinny(const Product& p, cudaStream_t s) {
  const long long cols = p.epilogue == kGate ? 2 * p.N : p.N;
  const bool direct = p.a_major;
  const skinny::Plan cut = skinny::plan(p.M, cols, p.K, direct);
  if (cut.bytes > p.partial_bytes) return cudaErrorInvalidValue;
  skinny::Args a{};
  a.a = static_cast<const float*>(p.a);
  a.b = static_cast<const float*>(p.b);
  a.out = direct ? static_cast<float*>(p.out) : p.partial;
  a.lda = p.lda;
  a.ldb = p.ldb;
  a.ldo = direct ? p.ldo : cols;
  a.M = p.M;
  a.N = cols;
  a.K = p.K;
  a.kper = cut.kper;
  a.share_stride = p.M * cols;
  a.va = multiple_of(p.a, 16) && p.lda % 4 == 0;
  a.vb = multiple_of(p.b, 16) && p.ldb % 4 == 0;
  cudaError_t e;
  if (direct && p.K <= 16 && p.N % 4 == 0 && a.vb && multiple_of(p.out, 16) && p.ldo % 4 == 0) {
    const dim3 grid(static_cast<unsigned>((p.M + skinny::kOuterRows - 1) / skinny::kOuterRows), static_cast<unsigned>((p.N + 1023) / 1024));
    if (p.K <= 4) skinny::outer_kernel<4><<<grid, 256, 0, s>>>(a);
    else if (p.K <= 8) skinny::outer_kernel<8><<<grid, 256, 0, s>>>(a);
    else skinny::outer_kernel<16><<<grid, 256, 0, s>>>(a);
    return cudaGetLastError();
  }
  // rows on the grid's x, the axis that may be long (columns: at most 2^21 / 128)
  switch (cut.tm) {
    case 8: e = skinny::by_order<8>(p, a, cut.shares, s); break;
    case 16: e = skinny::by_order<16>(p, a, cut.shares, s); break;
    case 32: e = skinny::by_order<32>(p, a, cut.shares, s); break;
    default: e = skinny::by_order<64>(p, a, cut.shares, s); break;
  }
  return e != cudaSuccess || direct ? e : launch_skinny_join(p, cut.shares, s);
}

}  // namespace ffn
}  // namespace msl
