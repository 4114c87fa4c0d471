// The gated feed-forward block's float32 products for up to 64 rows (forward, and from 9 rows on the gradients of h and
// x): the weights are read once, split into bf16 planes in registers and multiplied on the tensor cores by mma.sync.
//
// An element is hi + mid + lo, eight bits each: hi its upper half, cut off (so no finite value becomes infinite), the
// others rounded to nearest; the six products that reach 2^-24 of a product, the small ones of 32 k first.  Sums of 32 k
// stay in the instruction's accumulators, which cut off what does not fit, two full-sized additions that way; then they
// go into sums of their own, rounded.  Error of the whole block, 2560 to 7168 x 4108 to 25088, in the 2-norm: 2.7e-7
// to 4.4e-7, plain float32 products 3.7e-7 to 3.7e-6; with 64 k that were not small ones first 1.2e-6, in the same time to
// 10%.  Sums of 16 k 3.1e-7 to 6e-7 and, from 9 rows on, 5 to 10% slower.  An operand that is infinite gives NaN.
//
// A warp has 32 columns of the result (rows or columns of the weights) and all rows of x, a block 8 warps and a share
// of k.  A lane copies its own 8 x 16 bytes of 32 k of the weights to its own place in shared memory, two such stages
// ahead (cp.async); both storage orders give it 4 columns x 8 adjacent k, which are its place in the instruction's
// operand whatever order that has k and columns in, as long as x uses the same.  x goes through registers
// into planes in shared memory, kChunk k at a time, once for the block.  Shares of k are joined by skinny_join_kernel.
//
// Measured: at few_shape below.  What bounds it: up to 8 rows the splitting and the weights' bytes (7168 x 25088 forward, 2.16
// GB: 620 us, 3.5 TB/s), then the multiplications, 50 us for every 8 rows of 1.08 GB (2.4 clocks an instruction).  12 or
// 16 warps a block are as fast; x by 64 k at a time and five stages 5% slower than by 128 and three.

#include "gated_ffn.cuh"

namespace msl {
namespace ffn {
namespace few {

constexpr int kWarps = 8, kStages = 3, kColumns = 32 * kWarps, kChunk = 128;
constexpr int kStageBytes = 8 * 32 * 16;  // of a warp

struct Args {
  const float* a;
  const float* b;
  float* out;  // [shares][M][N]
  long long lda, ldb, N, K, kper;
  int M;
};

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3},{%4,%5,%6,%7},{%8,%9},{%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return reinterpret_cast<const uint32_t&>(t);
}

// The three planes of two neighbours, as words of two.
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& mid, uint32_t& lo) {
  hi = __byte_perm(__float_as_uint(x), __float_as_uint(y), 0x7632);
  const float rx = x - bf16_lo(hi), ry = y - bf16_hi(hi);
  mid = pack(rx, ry);
  lo = pack(rx - bf16_lo(mid), ry - bf16_hi(mid));
}

// 16 bytes of the weights, or zeros
__device__ __forceinline__ void copy16(uint32_t to, const float* from, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(in ? 16 : 0) : "memory");
}

// NT: groups of 8 rows of x.  NMAJOR: the weights are stored [K, N], else [N, K].
template <int NT, bool NMAJOR>
__global__ void __launch_bounds__(32 * kWarps, 1) few_kernel(const __grid_constant__ Args P) {
  constexpr int kRows = 8 * NT, kParts = kChunk / 32, kItems = kRows * kChunk / 4, kPer = (kItems + 32 * kWarps - 1) / (32 * kWarps);
  constexpr int kPlane = kRows * kChunk * 2;  // bytes: [groups of 32 k][rows][32]
  extern __shared__ __align__(128) uint8_t sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const long long n0 = static_cast<long long>(blockIdx.x) * kColumns + warp * 32;
  const long long k0 = blockIdx.y * P.kper, k1 = min(P.K, k0 + P.kper);
  uint8_t* const ring = sm + warp * kStages * kStageBytes + lane * 16;
  uint8_t* const xs = sm + kWarps * kStages * kStageBytes;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const int groups = static_cast<int>((k1 - k0 + 31) / 32);

  const float* src[NMAJOR ? 1 : 4];
  bool in[NMAJOR ? 1 : 4];
  if (NMAJOR) {
    in[0] = n0 + 4 * g < P.N;
    src[0] = P.b + (k0 + 8 * t) * P.ldb + (in[0] ? n0 + 4 * g : 0);
  } else {
#pragma unroll
    for (int r = 0; r < (NMAJOR ? 1 : 4); ++r) {
      in[r] = n0 + g + 8 * r < P.N;
      src[r] = P.b + (in[r] ? n0 + g + 8 * r : 0) * P.ldb + k0 + 8 * t;
    }
  }
  auto issue = [&](int group, int slot) {
    if (group < groups) {
      const long long k = k0 + group * 32LL + 8 * t;
      const uint32_t to = ring_at + slot * kStageBytes;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i >> 1, h = i & 1;
        if (NMAJOR) {
          const bool ok = in[0] && k + i < k1;
          copy16(to + i * 512, ok ? src[0] + (group * 32LL + i) * P.ldb : P.b, ok);
        } else {
          const bool ok = in[r % (NMAJOR ? 1 : 4)] && k + 4 * h < k1;
          copy16(to + i * 512, ok ? src[r % (NMAJOR ? 1 : 4)] + group * 32 + 4 * h : P.b, ok);
        }
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue(i, i);

  float4 xr[kPer];
  auto fetch = [&](long long k) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * 32 * kWarps + threadIdx.x, row = e / (kChunk / 4);
      const long long at = k + e % (kChunk / 4) * 4;
      xr[i] = e < kItems && row < P.M && at < k1 ? __ldg(reinterpret_cast<const float4*>(P.a + row * P.lda + at)) : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  };
  fetch(k0);

  float sum[2][NT][4];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int c = 0; c < 4; ++c) sum[i][j][c] = 0.f;
  int slot = 0, buf = 0;
  for (int first = 0; first < groups; first += kParts, buf ^= 1) {
    uint8_t* const planes = xs + buf * 3 * kPlane;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int e = i * 32 * kWarps + threadIdx.x, row = e / (kChunk / 4), k = e % (kChunk / 4) * 4;
      if (e >= kItems) continue;
      uint2 hi, mid, lo;
      split2(xr[i].x, xr[i].y, hi.x, mid.x, lo.x);
      split2(xr[i].z, xr[i].w, hi.y, mid.y, lo.y);
      uint8_t* const to = planes + ((k >> 5) * kRows + row) * 64 + (k & 31) * 2;
      *reinterpret_cast<uint2*>(to) = hi;
      *reinterpret_cast<uint2*>(to + kPlane) = mid;
      *reinterpret_cast<uint2*>(to + 2 * kPlane) = lo;
    }
    __syncthreads();  // the other buffer was left by all before they came here
    if (first + kParts < groups) fetch(k0 + (first + kParts) * 32LL);
#pragma unroll 1
    for (int part = 0; part < kParts && first + part < groups; ++part) {
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 2) : "memory");
      issue(first + part + kStages - 1, slot == 0 ? kStages - 1 : slot - 1);
      float w[4][8];  // 4 columns x 8 k
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 v = *reinterpret_cast<const float4*>(ring + slot * kStageBytes + i * 512);
        if (NMAJOR) {
          w[0][i] = v.x; w[1][i] = v.y; w[2][i] = v.z; w[3][i] = v.w;
        } else {
          float* const to = &w[i >> 1][(i & 1) * 4];
          to[0] = v.x; to[1] = v.y; to[2] = v.z; to[3] = v.w;
        }
      }
      slot = slot == kStages - 1 ? 0 : slot + 1;
      uint32_t wp[2][2][3][4];  // [half of the 8 k][16 columns][plane]
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float* const v = &w[2 * i + (q & 1)][4 * s + (q >> 1) * 2];
            split2(v[0], v[1], wp[s][i][0][q], wp[s][i][1][q], wp[s][i][2][q]);
          }
      constexpr int kOf[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};  // planes of w and x
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint4 x[3];
#pragma unroll
        for (int p = 0; p < 3; ++p) x[p] = *reinterpret_cast<const uint4*>(planes + p * kPlane + (part * kRows + j * 8 + g) * 64 + t * 16);
        float acc[2][4] = {};
#pragma unroll
        for (int c = 0; c < 6; ++c)
#pragma unroll
          for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int i = 0; i < 2; ++i) mma16816(acc[i], wp[s][i][kOf[c][0]], s ? x[kOf[c][1]].z : x[kOf[c][1]].x, s ? x[kOf[c][1]].w : x[kOf[c][1]].y);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) sum[i][j][c] += acc[i][c];
      }
    }
  }
  float* const out = P.out + static_cast<long long>(blockIdx.y) * P.M * P.N;
#pragma unroll
  for (int j = 0; j < NT; ++j)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int m = j * 8 + 2 * t + c;
      if (m >= P.M) continue;
      if (NMAJOR) {
        if (n0 + 4 * g < P.N)
          *reinterpret_cast<float4*>(out + m * P.N + n0 + 4 * g) = make_float4(sum[0][j][c], sum[0][j][2 + c], sum[1][j][c], sum[1][j][2 + c]);
      } else {
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (n0 + g + 8 * q < P.N) out[m * P.N + n0 + g + 8 * q] = sum[q >> 1][j][(q & 1) * 2 + c];
      }
    }
}

struct Plan {
  int shares;
  long long kper;
};

// One block a SM; shares of k for the least rounds of all SMs, each with 256 k's worth of start and end.
Plan plan(long long N, long long K) {
  const long long blocks = (N + kColumns - 1) / kColumns, sms = sm_count();
  Plan best{1, (K + kChunk - 1) / kChunk * kChunk};
  double least = 0;
  for (long long s = 1; s <= 64; ++s) {
    const long long kper = ((K + s - 1) / s + kChunk - 1) / kChunk * kChunk, shares = (K + kper - 1) / kper;
    if (shares != s) continue;
    const double cost = static_cast<double>((blocks * s + sms - 1) / sms) * (kper + 256.0);
    if (least != 0 && cost >= least) continue;
    least = cost;
    best = Plan{static_cast<int>(s), kper};
  }
  return best;
}

template <int NT, bool NMAJOR>
cudaError_t launch(const Args& a, int shares, cudaStream_t s) {
  constexpr int smem = kWarps * kStages * kStageBytes + 2 * 3 * 8 * NT * kChunk * 2;
  const cudaError_t e = cudaFuncSetAttribute(few_kernel<NT, NMAJOR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const dim3 grid(static_cast<unsigned>((a.N + kColumns - 1) / kColumns), static_cast<unsigned>(shares));
  few_kernel<NT, NMAJOR><<<grid, 32 * kWarps, smem, s>>>(a);
  return cudaGetLastError();
}

}  // namespace few

// Weights of 64 MB at least, and more than 8 rows where the weights are stored [K, N] (the gradients of h and x).  Forward of 5,
// 13, 30 and 60 rows of 2560 x 8960: 100, 113, 141 and 192 us, by skinny_kernel 170, 133, 242 and 282; 7168 x 25088: 628,
// 751, 961 and 1325, 1193, 913, 1758 and 2136.  Gradients of h and x, 5, 13, 30 and 60 rows of 7168 x 25088: 728, 835, 902 and
// 1389, 630, 823, 1658 and 2041; 2560 x 8960: 107, 120, 131 and 197, 105, 132, 253 and 292.  1152 x 4608 (21 and 42 MB),
// 13, 30 and 60 rows forward 45, 57 and 76, 43, 72 and 78; gradients 47, 54 and 76, 37, 59 and 72.
bool few_shape(long long M, long long cols, long long K, bool a_major, bool b_major) {
  return !a_major && M <= kMostRowsFew && cols * K >= (1LL << 24) && (b_major ? M > 8 && cols % 4 == 0 : K % 4 == 0);
}
size_t few_bytes(long long M, long long N, long long K, int epilogue) {
  const long long cols = epilogue == kGate ? 2 * N : N;
  return sizeof(float) * static_cast<size_t>(few::plan(cols, K).shares) * static_cast<size_t>(M) * static_cast<size_t>(cols);
}
bool few_apply(const Product& p) {
  return p.dtype == MSL_DTYPE_F32 && few_shape(p.M, p.epilogue == kGate ? 2 * p.N : p.N, p.K, p.a_major, p.b_major) && multiple_of(p.a, 16) && multiple_of(p.b, 16) && p.lda % 4 == 0 &&
         p.ldb % 4 == 0 && p.K % 4 == 0;
}

cudaError_t launch_product_few(const Product& p, cudaStream_t s) {
  const long long cols = p.epilogue == kGate ? 2 * p.N : p.N;
  const few::Plan cut = few::plan(cols, p.K);
  if (few_bytes(p.M, p.N, p.K, p.epilogue) > p.partial_bytes) return cudaErrorInvalidValue;
  few::Args a{};
  a.a = static_cast<const float*>(p.a);
  a.b = static_cast<const float*>(p.b);
  a.out = p.partial;
  a.lda = p.lda;
  a.ldb = p.ldb;
  a.N = cols;
  a.K = p.K;
  a.kper = cut.kper;
  a.M = static_cast<int>(p.M);
  cudaError_t e;
  if (p.M <= 8) e = few::launch<1, false>(a, cut.shares, s);
  else if (p.M <= 16) e = p.b_major ? few::launch<2, true>(a, cut.shares, s) : few::launch<2, false>(a, cut.shares, s);
  else if (p.M <= 32) e = p.b_major ? few::launch<4, true>(a, cut.shares, s) : few::launch<4, false>(a, cut.shares, s);
  else e = p.b_major ? few::launch<8, true>(a, cut.shares, s) : few::launch<8, false>(a, cut.shares, s);
  return e != cudaSuccess ? e : launch_skinny_join(p, cut.shares, s);
}

}  // namespace ffn
}  // namespace msl
