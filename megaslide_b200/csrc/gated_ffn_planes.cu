// The gated feed-forward block's products on the tensor cores for float32 operands, and for bf16 operands whose
// rows no TMA can address (widths that are no multiple of 8).
//
// float32: an operand is split into three bf16 planes, x = hi + mid + lo (8 bits of the significand each, every
// part rounded to nearest, so the sum is x to 2^-25), and a product is the six products of planes that reach
// 2^-24 of it:  lo hi', hi lo', mid mid', mid hi', hi mid', hi hi', the small ones first.  The tensor cores add
// into 32 bits but cut off what does not fit, so their sums run over 64 k only (24 multiplications); then the
// epilogue warps add them to sums in registers, rounding to nearest.  An operand that is infinite gives NaN.
// bf16: one plane, copied to rows of a multiple of 8 elements; sums stay in the tensor cores.
//
// The roles, pairs of CTAs and cuts along k are those of gated_ffn_tc.cu.  A stage holds the planes of 64 k
// (96 KB for three planes and 256 columns, two stages); results go through a transposing tile of shared memory, a
// row of 32 at a time, whatever their alignment.
//
// What bounds it: six times the multiplications, so about 220 TFLOP/s of float32 products (4096 x 4096 x 4096 forward 214,
// backward 219; 16384 x 2048 x 8192 219 and 214); the CUDA cores' limit is 75.

#include <algorithm>

#include "gated_ffn.cuh"
#include "tcgen05.cuh"

namespace msl {
namespace ffn {
namespace planes {

using namespace msl::t5;

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kBox = kBM * kBK * 2;  // bytes of a plane of A in a stage
constexpr int kRing = 12 * kBox;
constexpr int kMaxStages = 8;
constexpr int kPitch = 33;  // floats of a row of the transposing tile
constexpr int kTileBytes = 32 * kPitch * 4;

struct Maps {
  CUtensorMap a, b;
};

struct Args {
  const void* bias;
  void* out;
  void* kept_out;
  uint8_t* low;
  long long M, N, ldo;
  int np, act;
  int kblocks, mt, nt, gm;
  int bn, stages, stage_bytes, b_bytes;  // b_bytes: a plane of B in a stage
  int full, items, parts, kper;
  float* partial;  // [items - full][2 CTAs][4 x 32 rows][bn / 32][32 rows][32 columns]
  uint32_t* status;
};

// ------------------------------------------------------------------------------------------ planes

template <typename T>
__device__ __forceinline__ void split3(T, __nv_bfloat16 (&)[3]);
template <>
__device__ __forceinline__ void split3<float>(float x, __nv_bfloat16 (&p)[3]) {
  p[0] = __float2bfloat16_rn(x);
  float r = x - __bfloat162float(p[0]);
  if (!isfinite(__bfloat162float(p[0])) && isfinite(x)) {  // the last half ulp below infinity: round down
    p[0] = __float2bfloat16_rz(x);
    r = x - __bfloat162float(p[0]);
  }
  p[1] = __float2bfloat16_rn(r);
  p[2] = __float2bfloat16_rn(r - __bfloat162float(p[1]));
}

// out[plane][row][ldp] of x [rows, cols]; a thread does 8 columns, those beyond cols are zero.
struct Job {
  const void* x;
  __nv_bfloat16* out;
  long long ld, rows;
  int cols, ldp;
};
// One or two operands, each by half of the blocks (a small product's launches cost as much as their work).
struct Jobs {
  Job of[2];
};

template <typename T, int NP>
__global__ void __launch_bounds__(256) split_kernel(const __grid_constant__ Jobs jobs) {
  const Job& J = jobs.of[blockIdx.y];
  const T* const x = static_cast<const T*>(J.x);
  const int per = J.ldp / 8;
  const long long n = J.rows * per, plane = J.rows * J.ldp;
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    const long long r = i / per;
    const int c = static_cast<int>(i - r * per) * 8;
    const T* const p = x + r * J.ld + c;
    __nv_bfloat16 o[NP][8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const T v = c + j < J.cols ? p[j] : from_f32<T>(0.f);
      if constexpr (NP == 3) {
        __nv_bfloat16 s[3];
        split3<T>(v, s);
        o[0][j] = s[0];
        o[1][j] = s[1];
        o[2][j] = s[2];
      } else {
        o[0][j] = __float2bfloat16_rn(to_f32<T>(v));
      }
    }
#pragma unroll
    for (int k = 0; k < NP; ++k) *reinterpret_cast<uint4*>(J.out + k * plane + r * J.ldp + c) = *reinterpret_cast<const uint4*>(o[k]);
  }
}

// ------------------------------------------------------------------------------------------ kernel

__device__ __forceinline__ void tile_at(const Args& P, int t, int& m, int& n) {
  const int per = P.gm * P.nt, g = t / per, r = t - g * per;
  const int first = g * P.gm, rows = min(P.gm, P.mt - first);
  n = r / rows;
  m = first + r - n * rows;
}
struct Item {
  int m, n, k0, k1, part;
};
__device__ __forceinline__ Item item_at(const Args& P, int i) {
  Item w;
  w.k0 = 0;
  w.k1 = P.kblocks;
  w.part = -1;
  int t = i;
  if (i >= P.full) {
    w.part = i - P.full;
    t = P.full + w.part / P.parts;
    w.k0 = w.part % P.parts * P.kper;
    w.k1 = min(P.kblocks, w.k0 + P.kper);
  }
  tile_at(P, t, w.m, w.n);
  return w;
}

// An element's epilogue.
template <typename T>
__device__ __forceinline__ float bias_at(const void* bias, long long i) { return bias ? to_f32<T>(static_cast<const T*>(bias)[i]) : 0.f; }

// 32 rows x 32 columns from the lanes' rows in registers to the matrix: through the tile, a row of 32 at a time, `add`
// to a lane's column.
template <typename T>
__device__ __forceinline__ void put_block(float* tile, int lane, const float (&v)[32], float add, T* out, long long ld, long long row0, long long x,
                                          long long M, long long N) {
  __syncwarp();
#pragma unroll
  for (int j = 0; j < 32; ++j) tile[lane * kPitch + j] = v[j];
  __syncwarp();
  if (x + lane < N)
#pragma unroll 8
    for (int r = 0; r < 32; ++r)
      if (row0 + r < M) out[(row0 + r) * ld + x + lane] = from_f32<T>(tile[r * kPitch + lane] + add);
}

// The gate's epilogue of 32 rows x 32 columns: g and u of 16 rows at a time in the tile, a lane a column.  These loops,
// and those over a tile's blocks, stay rolled: a small product runs its epilogue once, and what it runs is fetched
// from the L2 cache (2048 x 256 x 2 x 1024 in float32: 27 us; 45 with the blocks and passes written out).
template <typename T>
__device__ __forceinline__ void gate_block(const Args& P, float* tile, int lane, const float (&g)[32], const float (&u)[32], long long row0, long long x) {
  const bool in = x + lane < P.N;
  const float bg = in ? bias_at<T>(P.bias, x + lane) : 0.f, bu = in ? bias_at<T>(P.bias, P.N + x + lane) : 0.f;
#pragma unroll 1
  for (int part = 0; part < 2; ++part, row0 += 16) {
    __syncwarp();
    if (lane >> 4 == part) {
#pragma unroll
      for (int j = 0; j < 32; ++j) {
        tile[(lane & 15) * kPitch + j] = g[j];
        tile[(16 + (lane & 15)) * kPitch + j] = u[j];
      }
    }
    __syncwarp();
    if (!in || row0 >= P.M) continue;
    const int rows = static_cast<int>(min(16LL, P.M - row0));
    T* const h = static_cast<T*>(P.out) + row0 * P.ldo + x + lane;
    KeptRow<T> kept(P.kept_out, P.low, row0, x + lane, P.N);
#pragma unroll 2
    for (int r = 0; r < rows; ++r) {
      const float ur = tile[(16 + r) * kPitch + lane] + bu;
      float da;
      const float a = act_value_grad(tile[r * kPitch + lane] + bg, P.act, da);
      h[r * P.ldo] = from_f32<T>(a * ur);
      if (P.kept_out) {
        kept.put(0, ur * da);
        kept.put(1, a);
        kept.at += 2 * kept.N;
        kept.low += 2 * kept.W;
      }
    }
  }
}

template <typename T, int EPI, bool AM, bool BM>
__global__ void __launch_bounds__(kThreads, 1) planes_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args P) {
  constexpr int kAcc = 256;
  const int half = P.bn / 2, width = EPI == kGate ? half : P.bn, stages = P.stages;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t tiles = base + kRing;
  const uint32_t bars = tiles + kEpiWarps * kTileBytes;
  const uint32_t full = bars, empty = bars + 8 * kMaxStages, peer = empty + 8 * kMaxStages, tfull = peer + 8 * kMaxStages, tempty = tfull + 16;
  const uint32_t tmem_slot = tempty + 16, last = tmem_slot + 8;
  volatile int* const dead = reinterpret_cast<volatile int*>(raw + (tmem_slot + 4 - smem_u32(raw)));
  volatile uint32_t* const slot = reinterpret_cast<volatile uint32_t*>(raw + (tmem_slot - smem_u32(raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = static_cast<int>(cluster_rank());
  const int t0 = blockIdx.x >> 1, tstep = gridDim.x >> 1;

  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
      mbar_init(peer + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + 8 * i, 1);
      mbar_init(tempty + 8 * i, 2 * kEpiWarps);
    }
    mbar_init(last, 1);
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(2 * kAcc) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  cluster_sync();
  fence_after();
  const uint32_t tmem = *slot;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool alive = true;
      for (int t = t0; t < P.items && alive; t += tstep) {
        const Item w = item_at(P, t);
        const int arow = (2 * w.m + rank) * kBM;
        const int brow = EPI == kGate ? w.n * width + (rank ? static_cast<int>(P.N) : 0) : w.n * width + rank * half;
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!wait(empty + 8 * st, ph ^ 1, dead, P.status)) { alive = false; break; }
          uint32_t to = base + st * P.stage_bytes;
          const uint32_t bar = full + 8 * st;
          mbar_expect(bar, P.stage_bytes);
          for (int p = 0; p < P.np; ++p, to += kBox) {
            if (AM) {
              tma_load_3d(to, &maps.a, bar, arow, kb * kBK, p);
              tma_load_3d(to + 8192, &maps.a, bar, arow + 64, kb * kBK, p);
            } else {
              tma_load_3d(to, &maps.a, bar, kb * kBK, arow, p);
            }
          }
          for (int p = 0; p < P.np; ++p, to += P.b_bytes) {
            if (BM) {
              for (int i = 0; i < half / 64; ++i) tma_load_3d(to + i * 8192, &maps.b, bar, brow + i * 64, kb * kBK, p);
            } else {
              tma_load_3d(to, &maps.b, bar, kb * kBK, brow, p);
            }
          }
          if (++st == stages) { st = 0; ph ^= 1; }
        }
      }
      const long long since = clock64();
      if (!alive)
        for (int i = 0; i < stages; ++i)
          while (!mbar_try(full + 8 * i, (i < st ? ph : ph ^ 1)) && clock64() - since < kWaitClocks) {
          }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (AM ? 1u << 15 : 0u) | (BM ? 1u << 16 : 0u) |
                             (static_cast<uint32_t>(P.bn >> 3) << 17) | (static_cast<uint32_t>(2 * kBM >> 4) << 24);
      constexpr uint64_t a_step = (AM ? 2048 : 32) >> 4, b_step = (BM ? 2048 : 32) >> 4;
      int st = 0, buf = 0;
      uint32_t ph = 0, tph = 0;
      bool alive = true;
      for (int t = t0; t < P.items && alive; t += tstep) {
        const Item w = item_at(P, t);
        for (int kb = w.k0; kb < w.k1; ++kb) {
          const bool begin = P.np == 3 || kb == w.k0, end = P.np == 3 || kb == w.k1 - 1;  // of a sum in the tensor cores
          if (begin && !wait(tempty + 8 * buf, tph ^ 1, dead, P.status)) { alive = false; break; }
          if (!wait(full + 8 * st, ph, dead, P.status) || !wait(peer + 8 * st, ph, dead, P.status)) { alive = false; break; }
          fence_after();
          const uint32_t a = base + st * P.stage_bytes, b = a + P.np * kBox;
          bool more = !begin;
          for (int q = P.np == 3 ? 0 : 5; q < 6; ++q) {
            // plane 0 is hi: (2,0) (0,2) (1,1) (1,0) (0,1) (0,0)
            const int pa = (0x001102 >> (4 * q)) & 0xf, pb = (0x010120 >> (4 * q)) & 0xf;
            const uint64_t da = operand<AM>(a + pa * kBox), db = operand<BM>(b + pb * P.b_bytes);
#pragma unroll
            for (int k = 0; k < kBK / 16; ++k) {
              mma(tmem + buf * kAcc, da + k * a_step, db + k * b_step, idesc, more);
              more = true;
            }
          }
          mma_commit(empty + 8 * st);
          if (++st == stages) { st = 0; ph ^= 1; }
          if (end) {
            mma_commit(tfull + 8 * buf);
            buf ^= 1;
            if (buf == 0) tph ^= 1;
          }
        }
      }
      if (!alive) mma_drain(last);
    } else if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool alive = true;
      for (int t = t0; t < P.items && alive; t += tstep) {
        const Item w = item_at(P, t);
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!wait(full + 8 * st, ph, dead, P.status)) { alive = false; break; }
          arrive_first(peer + 8 * st);
          if (++st == stages) { st = 0; ph ^= 1; }
        }
      }
    }
    __syncwarp();
  } else {
    const int ew = warp - 2, quad = warp & 3, set = ew >> 2;
    float* const tile = reinterpret_cast<float*>(raw + (tiles - smem_u32(raw))) + ew * 32 * kPitch;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    int buf = 0;
    uint32_t tph = 0;
    // blocks of 32 columns that the thread sums: plain, a half of the tile; gate, a half of the gate's columns
    // and the same ones of the other projection (blocks nb and up)
    const int nb = EPI == kGate ? P.bn / 128 : P.bn / 64;
    for (int t = t0; t < P.items; t += tstep) {
      const Item w = item_at(P, t);
      const long long row0 = (2LL * w.m + rank) * kBM + quad * 32;
      float acc[4][32];
#pragma unroll
      for (int b = 0; b < 4; ++b)
#pragma unroll
        for (int j = 0; j < 32; ++j) acc[b][j] = 0.f;
      const int sums = P.np == 3 ? w.k1 - w.k0 : 1;
      bool alive = true;
      for (int i = 0; i < sums; ++i) {
        if (!wait_warp(tfull + 8 * buf, tph, dead, P.status)) { alive = false; break; }
        fence_after();
        const uint32_t from = tmem + buf * kAcc + lanes;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          if (EPI == kGate ? b % 2 >= nb : b >= nb) continue;
          const int c = EPI == kGate ? (b / 2) * half + (set * nb + b % 2) * 32 : (set * nb + b) * 32;
          float v[32];
          tmem_ld32(from + c, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) acc[b][j] += v[j];
        }
        fence_before();
        __syncwarp();
        if (lane == 0) arrive_first(tempty + 8 * buf);
        buf ^= 1;
        if (buf == 0) tph ^= 1;
      }
      if (!alive) break;
      const long long col0 = static_cast<long long>(w.n) * width;
      const int blocks = P.bn / 32;
      float* const part = w.part < 0 ? nullptr : P.partial + static_cast<size_t>((w.part * 2 + rank) * 4 + quad) * blocks * 1024;
#pragma unroll 1
      for (int b = 0; b < nb; ++b) {  // the first block's registers, then the next's moved there
        const int block = set * nb + b;
        const long long x = col0 + block * 32;
        if (part) {
          put_block<float>(tile, lane, acc[0], 0.f, part + block * 1024, 32, 0, 0, 32, 32);
          if (EPI == kGate) put_block<float>(tile, lane, acc[2], 0.f, part + (half / 32 + block) * 1024, 32, 0, 0, 32, 32);
        } else if (EPI == kPlain) {
          put_block<T>(tile, lane, acc[0], x + lane < P.N ? bias_at<T>(P.bias, x + lane) : 0.f, static_cast<T*>(P.out), P.ldo, row0, x, P.M, P.N);
        } else {
          gate_block<T>(P, tile, lane, acc[0], acc[2], row0, x);
        }
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          acc[0][j] = acc[1][j];
          if (EPI == kPlain) acc[1][j] = acc[2][j];
          acc[2][j] = acc[3][j];
        }
      }
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kAcc));
  }
}

// Epilogue of the tiles that were cut along k: a warp does 4 rows x 32 columns, parts in their order.
template <typename T, int EPI>
__global__ void __launch_bounds__(256) planes_join_kernel(const __grid_constant__ Args P) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = P.bn / 2, width = EPI == kGate ? half : P.bn, steps = width / 32;
  const int rank = blockIdx.y, quad = blockIdx.z, tail = blockIdx.x / steps, i = blockIdx.x - tail * steps;
  int m, n;
  tile_at(P, P.full + tail, m, n);
  const long long x = static_cast<long long>(n) * width + i * 32 + lane;
  const int blocks = P.bn / 32;
  const size_t hop = static_cast<size_t>(8) * blocks * 1024;
  const float* const from = P.partial + static_cast<size_t>((tail * P.parts * 2 + rank) * 4 + quad) * blocks * 1024 + lane;
  if (x >= P.N) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const int r = warp * 4 + k;
    const long long row = (2LL * m + rank) * kBM + quad * 32 + r;
    if (row >= P.M) return;
    float v = 0.f, u = 0.f;
    for (int s = 0; s < P.parts; ++s) {
      v += from[s * hop + i * 1024 + r * 32];
      if (EPI == kGate) u += from[s * hop + (steps + i) * 1024 + r * 32];
    }
    if (EPI == kPlain) {
      static_cast<T*>(P.out)[row * P.ldo + x] = from_f32<T>(v + bias_at<T>(P.bias, x));
    } else {
      v += bias_at<T>(P.bias, x);
      u += bias_at<T>(P.bias, P.N + x);
      float da;
      const float a = act_value_grad(v, P.act, da);
      if (P.kept_out) {
        const KeptRow<T> kept(P.kept_out, P.low, row, x, P.N);
        kept.put(0, u * da);
        kept.put(1, a);
      }
      static_cast<T*>(P.out)[row * P.ldo + x] = from_f32<T>(a * u);
    }
  }
}

// The gradients of g and u, dgu [M, 2N], from that of h, which the product has left in float32 (rows of `ld`), and the
// factors, kept likewise: one rounding to the result's type.  float32 has the gradient of h in the place of that of u.  A kernel
// of its own: in the product's epilogue it would hold up the sums that run through there (float32), and the factors' loads
// would hold up the next tile (bf16, dx of 20001 x 1149 x 4605: 2410 us instead of 1180).
template <typename T>
__global__ void __launch_bounds__(256) dgate_kernel(const void* kept, const uint8_t* low, const float* dh, long long ld, T* dgu, long long M, long long N) {
  const long long row = blockIdx.x;
  const float* const from = dh + row * ld;
  T* const out = dgu + row * 2 * N;
#pragma unroll 4
  for (long long c = blockIdx.y * 256LL + threadIdx.x; c < N; c += gridDim.y * 256LL) {
    const float v = from[c];
    const KeptRow<T> by(kept, low, row, c, N);
    const float g = by.get(0), u = by.get(1);
    out[c] = from_f32<T>(v * g);
    out[N + c] = from_f32<T>(v * u);
  }
}

// ------------------------------------------------------------------------------------------ host

int planes_of(int dtype) { return dtype == MSL_DTYPE_F32 ? 3 : 1; }
long long padded(long long cols) { return (cols + 7) / 8 * 8; }

// Map of planes [np, rows, cols] (rows of `ld`): boxes of 64 columns x `box` rows of one plane, 128-byte swizzle.
bool plane_map(CUtensorMap* map, const void* p, int np, long long rows, long long cols, long long ld, int box) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows), static_cast<cuuint64_t>(np)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(ld) * 2, static_cast<cuuint64_t>(ld) * rows * 2};
  const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(box), 1}, steps[3] = {1, 1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Plan {
  int bn, parts, kper;
  long long mt, nt, full, items;
  size_t bytes;
};

// The cheapest cut (microseconds, as in gated_ffn_tc.cu): a block of 64 k takes 1.7 for three planes and 256 columns
// (24 multiplications), 1.0 for 128; one plane 0.45 and 0.35.
Plan plan(long long M, long long N, long long K, bool gate, int np) {
  const long long pairs = sm_count() / 2, kblocks = (K + kBK - 1) / kBK;
  Plan best{};
  double least = 0;
  for (int bn = 256; bn >= 128; bn -= 128) {
    Plan p{};
    const long long width = gate ? bn / 2 : bn;
    p.bn = bn;
    p.mt = (M + 2 * kBM - 1) / (2 * kBM);
    p.nt = (N + width - 1) / width;
    const long long tiles = p.mt * p.nt, tail = tiles % pairs;
    const double block = np == 3 ? (bn == 256 ? 1.7 : 1.0) : (bn == 256 ? 0.45 : 0.35);
    for (long long parts = 1; parts == 1 || (tail > 0 && parts <= pairs / tail && parts <= 32); ++parts) {
      const long long kper = (kblocks + parts - 1) / parts;
      if (parts > 1 && (kper < 2 || (kblocks + kper - 1) / kper != parts)) continue;
      const double rounds = static_cast<double>(tiles / pairs) + (tail == 0 ? 0.0 : parts == 1 ? 1.0 : static_cast<double>(kper) / kblocks);
      const double cost = rounds * kblocks * block + 3.0 + (parts > 1 ? 6.0 + 0.3 * parts : 0.0);
      if (least != 0 && cost >= least) continue;
      least = cost;
      p.parts = static_cast<int>(parts);
      p.kper = static_cast<int>(kper);
      p.full = parts == 1 ? tiles : tiles - tail;
      p.items = p.full + (parts == 1 ? 0 : tail * parts);
      p.bytes = sizeof(float) * static_cast<size_t>(p.items - p.full) * 2 * kBM * bn;
      best = p;
    }
  }
  return best;
}

template <typename T, int EPI, bool AM, bool BM>
cudaError_t launch(const Product& p, const void* pa, const void* pb, cudaStream_t s) {
  const int np = planes_of(p.dtype);
  const Plan cut = plan(p.M, p.N, p.K, EPI == kGate, np);
  if (cut.bytes > p.partial_bytes) return cudaErrorInvalidValue;
  Args a{};
  a.bias = p.bias;
  a.out = p.out;
  a.kept_out = p.kept_out;
  a.low = p.low;
  a.M = p.M;
  a.N = p.N;
  a.ldo = p.ldo;
  a.np = np;
  a.act = p.act;
  a.kblocks = static_cast<int>((p.K + kBK - 1) / kBK);
  a.mt = static_cast<int>(cut.mt);
  a.nt = static_cast<int>(cut.nt);
  a.gm = a.mt <= 16 ? a.mt : 8;
  a.bn = cut.bn;
  a.b_bytes = cut.bn / 2 * kBK * 2;
  a.stage_bytes = np * (kBox + a.b_bytes);
  a.stages = kRing / a.stage_bytes < kMaxStages ? kRing / a.stage_bytes : kMaxStages;
  a.full = static_cast<int>(cut.full);
  a.items = static_cast<int>(cut.items);
  a.parts = cut.parts;
  a.kper = cut.kper;
  a.partial = p.partial;
  a.status = p.status;
  cudaError_t e = bind_context();
  if (e != cudaSuccess) return e;
  Maps maps;
  const long long brows = EPI == kGate ? 2 * p.N : p.N;
  const bool ok = (AM ? plane_map(&maps.a, pa, np, p.K, p.M, padded(p.M), kBK) : plane_map(&maps.a, pa, np, p.M, p.K, padded(p.K), kBM)) &&
                  (BM ? plane_map(&maps.b, pb, np, p.K, p.N, padded(p.N), kBK) : plane_map(&maps.b, pb, np, brows, p.K, padded(p.K), cut.bn / 2));
  if (!ok) return cudaErrorInvalidValue;
  constexpr int smem = 1024 + kRing + kEpiWarps * kTileBytes + 24 * kMaxStages + 64;
  static_assert(smem <= 232448, "shared memory of a block");
  auto* const kernel = planes_kernel<T, EPI, AM, BM>;
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int pairs = sm_count() / 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(2 * (a.items < pairs ? a.items : pairs)));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kernel, maps, a);
  if (e != cudaSuccess || a.items == a.full) return e;
  const int steps = (EPI == kGate ? a.bn / 2 : a.bn) / 32;
  planes_join_kernel<T, EPI><<<dim3((a.mt * a.nt - a.full) * steps, 2, 4), 256, 0, s>>>(a);
  count_launches(1);
  return cudaGetLastError();
}

template <typename T>
cudaError_t by_epilogue(const Product& p, const void* pa, const void* pb, cudaStream_t s) {
  switch (p.epilogue) {
    case kGate: return launch<T, kGate, false, false>(p, pa, pb, s);
    default:
      if (p.a_major) return launch<T, kPlain, true, true>(p, pa, pb, s);
      return p.b_major ? launch<T, kPlain, false, true>(p, pa, pb, s) : launch<T, kPlain, false, false>(p, pa, pb, s);
  }
}

}  // namespace planes

size_t planes_bytes(int dtype, long long rows, long long cols) {
  const size_t n = sizeof(__nv_bfloat16) * planes::planes_of(dtype) * static_cast<size_t>(rows) * static_cast<size_t>(planes::padded(cols));
  return (n + 255) / 256 * 256;
}

cudaError_t launch_planes(int dtype, const PlaneJob* jobs, int count, cudaStream_t s) {
  planes::Jobs all{};
  long long n = 0;
  for (int i = 0; i < count; ++i) {
    planes::Job& j = all.of[i];
    j.x = jobs[i].x;
    j.out = static_cast<__nv_bfloat16*>(jobs[i].out);
    j.ld = jobs[i].ld;
    j.rows = jobs[i].rows;
    j.cols = static_cast<int>(jobs[i].cols);
    j.ldp = static_cast<int>(planes::padded(jobs[i].cols));
    n = std::max(n, j.rows * (j.ldp / 8));
  }
  const long long most = static_cast<long long>(sm_count()) * 16 / count, blocks = (n + 255) / 256;
  const dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most), static_cast<unsigned>(count));
  if (dtype == MSL_DTYPE_F32) planes::split_kernel<float, 3><<<grid, 256, 0, s>>>(all);
  else planes::split_kernel<__nv_bfloat16, 1><<<grid, 256, 0, s>>>(all);
  count_launches(1);
  return cudaGetLastError();
}

bool planes_apply(const Product& p) {
  if (!t5::encoder() || p.M > (1LL << 31) - 256 || p.N > (1LL << 30) || p.K > (1LL << 31) - 256 ||
      (p.M + 255) / 256 * ((p.N + 63) / 64) > (1LL << 30))
    return false;
  if (p.dtype != MSL_DTYPE_F32) return true;
  const double cols = p.epilogue == kGate ? 2.0 * p.N : p.N;
  // microseconds.  Planes: 10 bytes an element of both operands at 5 TB/s, rows in tiles of 256 and k in blocks of 64,
  // 95 G multiplications a millisecond, 7 for every round of tiles, some launches.  CUDA cores: rows in their tiles, 15 G multiplications
  // a millisecond (7.5 up to 16 rows, where the operands bound them), operands and result once.
  const double elements = 1.0 * p.M * p.K + cols * p.K;
  const double rows = (p.M + 255) / 256 * 256.0, rounds = rows * cols / 65536.0 / 74.0;
  const double tile = p.M <= 8 ? 8 : p.M <= 16 ? 16 : p.M <= 32 ? 32 : (p.M + 63) / 64 * 64.0;
  const double planes = elements * 10 / 5e6 + rows * cols * ((p.K + 63) / 64 * 64.0) / 95e6 + 7 * rounds + 12;
  const double cores = std::max(tile * cols * p.K / (p.M <= 16 ? 7.5e6 : 15e6), (elements + p.M * cols) * 4 / 4e6) + 6;
  return planes < cores;
}

size_t planes_partial_bytes(int dtype, long long M, long long N, long long K, int epilogue) {
  return planes::plan(M, N, K, epilogue == kGate, planes::planes_of(dtype)).bytes;
}

cudaError_t launch_product_planes(const Product& p, const void* pa, const void* pb, float* dh, cudaStream_t s) {
  const bool f32 = p.dtype == MSL_DTYPE_F32;
  if (p.epilogue != kDgate) return f32 ? planes::by_epilogue<float>(p, pa, pb, s) : planes::by_epilogue<__nv_bfloat16>(p, pa, pb, s);
  Product q = p;
  q.epilogue = kPlain;
  q.ldo = f32 ? 2 * p.N : p.N;
  q.out = dh = f32 ? static_cast<float*>(p.out) + p.N : dh;
  const cudaError_t e = planes::by_epilogue<float>(q, pa, pb, s);
  if (e != cudaSuccess) return e;
  const long long cols = (p.N + 1023) / 1024;
  const dim3 grid(static_cast<unsigned>(p.M), static_cast<unsigned>(cols < 64 ? cols : 64));
  if (f32)
    planes::dgate_kernel<float><<<grid, 256, 0, s>>>(p.kept, p.low, dh, q.ldo, static_cast<float*>(p.out), p.M, p.N);
  else
    planes::dgate_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(p.kept, p.low, dh, q.ldo, static_cast<__nv_bfloat16*>(p.out), p.M, p.N);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace ffn
}  // namespace msl
