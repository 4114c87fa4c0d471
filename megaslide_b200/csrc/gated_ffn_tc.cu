// The gated feed-forward block's products on the 5th-generation tensor cores (bf16 operands, float32 sums in
// tensor memory).
//
// C[M, N] = sum_k A(m, k) B(n, k), A and B each with k or its own axis contiguous, so one kernel serves the
// forward (x w_in^T, h w_out^T: both k-major), the input gradients (dy w_out, [dg du] w_in: B n-major) and the
// weight gradients ([dg du]^T x, dy^T h: both with the summed axis, the tokens, outermost).  Operand tiles come
// by TMA with the 128-byte swizzle that tcgen05.mma reads in either orientation; ragged edges are the TMA's zero
// fill and clipping, no element is handled apart.
//
// One CTA per SM walks over 128 x BN tiles: one thread loads (a ring of stages), one thread issues the
// multiplications (128 x BN x 16 each), eight warps turn finished accumulators into results while the next
// tile is multiplied into the other half of the tensor memory.
//   gate:  the tile's columns are 128 gate columns and the same 128 columns of the other projection, so g and u of an
//          element meet in one epilogue thread: bias, activation, product, and the kept g, u leave from there
//   dgate: the accumulator is the gradient of h; the epilogue reads the kept g, u and writes both their gradients

#include <cuda.h>
#include <cudaTypedefs.h>

#include "gated_ffn.cuh"

namespace msl {
namespace ffn {
namespace tc {

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kStageA = kBM * kBK * 2;
constexpr int kStaging = 32 * 128;  // of an epilogue warp: 32 rows x 64 bf16
constexpr unsigned long long kWaitNs = 2000000000ull;

struct Maps {
  CUtensorMap a, b, out, gu;
};

struct Args {
  const __nv_bfloat16* bias;
  const __nv_bfloat16* gu;
  long long M, N;
  int kblocks, mt, nt, gm, act, keep;
  uint32_t* status;
};

// ------------------------------------------------------------------------------------------ PTX

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile("{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}"
               : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for phase `parity` of a barrier, at most kWaitNs: then the CTA is marked dead and every role leaves.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* dead, uint32_t* status) {
  if (mbar_try(bar, parity)) return true;
  const unsigned long long t0 = now_ns();
  while (!mbar_try(bar, parity)) {
    if (*dead) return false;
    if (now_ns() - t0 > kWaitNs) {
      *dead = 1;
      if (status) atomicOr(status, MSL_STATUS_TIMEOUT);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tma_store_3d(const CUtensorMap* map, uint32_t src, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(reinterpret_cast<uint64_t>(map)),
               "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
               "l"(b), "r"(idesc), "r"(accumulate ? 1 : 0) : "memory");
}
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 columns of this warp's 32 lanes of tensor memory
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]),
        "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// Shared-memory operand descriptor of a tile with the 128-byte swizzle.  k-major: rows of 64 k (128 bytes), groups
// of 8 rows 1024 bytes apart.  Own axis contiguous: rows of 64 elements of it, one k each; groups of 8 k 1024 bytes
// apart, the next 64 elements after all 64 k of the stage (8192 bytes).
template <bool MAJOR>
__device__ __forceinline__ uint64_t operand(uint32_t addr) {
  const uint64_t lead = MAJOR ? 8192 >> 4 : 1, stride = 1024 >> 4;
  return static_cast<uint64_t>((addr & 0x3ffff) >> 4) | (lead << 16) | (stride << 32) | (1ull << 46) | (2ull << 61);
}

// ------------------------------------------------------------------------------------------ kernel

__device__ __forceinline__ void tile_at(const Args& P, int t, int& m, int& n) {
  const int per = P.gm * P.nt, g = t / per, r = t - g * per;
  const int first = g * P.gm, rows = min(P.gm, P.mt - first);
  n = r / rows;
  m = first + r - n * rows;
}

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}

// Half a row (32 columns) of a warp's staging tile: 16-byte chunk c of row r lies at c ^ (r & 7), as the TMA's
// 128-byte swizzle has it (and no two lanes of a quarter meet in a bank).
__device__ __forceinline__ void stage_half(uint32_t base, int row, int half, const uint32_t (&w)[16]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t at = base + row * 128 + (((half * 4 + c) ^ (row & 7)) << 4);
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[c * 4]), "r"(w[c * 4 + 1]), "r"(w[c * 4 + 2]), "r"(w[c * 4 + 3])
                 : "memory");
  }
}

// adds bias[n .. n+32) to v (columns at or beyond N are clipped by the store)
__device__ __forceinline__ void add_bias(float (&v)[32], const __nv_bfloat16* bias, long long n, long long N) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    if (n + c * 8 + 8 > N) continue;  // N is a multiple of 8
    const uint4 b = __ldg(reinterpret_cast<const uint4*>(bias + n) + c);
    const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[c * 8 + 2 * i] += bf16_lo(w[i]);
      v[c * 8 + 2 * i + 1] += bf16_hi(w[i]);
    }
  }
}

__device__ __forceinline__ void load_half(uint4 (&w)[4], const __nv_bfloat16* p, bool row_in, long long n, long long N) {
#pragma unroll
  for (int c = 0; c < 4; ++c)
    w[c] = row_in && n + c * 8 + 8 <= N ? __ldg(reinterpret_cast<const uint4*>(p + n) + c) : make_uint4(0, 0, 0, 0);
}

template <int EPI, int BN, int STAGES, bool AM, bool BM>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args P) {
  constexpr int kStageB = BN * kBK * 2, kStage = kStageA + kStageB;
  constexpr int kBoxN = EPI == kGate ? BN / 2 : BN;      // columns of N that a tile covers
  constexpr int kAcc = BN <= 128 ? 128 : 256;            // tensor memory columns of an accumulator
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t staging = base + STAGES * kStage;
  const uint32_t bars = staging + kEpiWarps * kStaging;
  const uint32_t full = bars, empty = bars + 8 * STAGES, tfull = empty + 8 * STAGES, tempty = tfull + 16;
  const uint32_t tmem_slot = tempty + 16;
  volatile int* const dead = reinterpret_cast<volatile int*>(raw + (tmem_slot + 4 - smem_u32(raw)));
  volatile uint32_t* const slot = reinterpret_cast<volatile uint32_t*>(raw + (tmem_slot - smem_u32(raw)));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int tiles = P.mt * P.nt;

  if (threadIdx.x == 0) {
    for (int i = 0; i < STAGES; ++i) {
      mbar_init(full + 8 * i, 1);
      mbar_init(empty + 8 * i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + 8 * i, 1);
      mbar_init(tempty + 8 * i, kEpiWarps);
    }
    *dead = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(2 * kAcc) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    fence_before();
  }
  __syncthreads();
  fence_after();
  const uint32_t tmem = *slot;

  if (warp == 0) {
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      bool alive = true;
      for (int t = blockIdx.x; t < tiles && alive; t += gridDim.x) {
        int m, n;
        tile_at(P, t, m, n);
        for (int kb = 0; kb < P.kblocks; ++kb) {
          if (!wait(empty + 8 * st, ph ^ 1, dead, P.status)) { alive = false; break; }
          const uint32_t a = base + st * kStage, b = a + kStageA, bar = full + 8 * st;
          mbar_expect(bar, kStage);
          if (AM) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i) tma_load_2d(a + i * 8192, &maps.a, bar, m * kBM + i * 64, kb * kBK);
          } else {
            tma_load_2d(a, &maps.a, bar, kb * kBK, m * kBM);
          }
          if (BM) {
#pragma unroll
            for (int i = 0; i < BN / 64; ++i) tma_load_2d(b + i * 8192, &maps.b, bar, n * BN + i * 64, kb * kBK);
          } else {
            tma_load_2d(b, &maps.b, bar, kb * kBK, n * kBoxN);
            if (EPI == kGate) tma_load_2d(b + kStageB / 2, &maps.b, bar, kb * kBK, static_cast<int>(P.N) + n * kBoxN);
          }
          if (++st == STAGES) { st = 0; ph ^= 1; }
        }
      }
      // the copies still in flight land before the CTA leaves
      const unsigned long long t0 = now_ns();
      if (!alive)
        for (int i = 0; i < STAGES; ++i)
          while (!mbar_try(full + 8 * i, (i < st ? ph : ph ^ 1)) && now_ns() - t0 < kWaitNs) {
          }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0) {
      // bf16 x bf16 -> float32, transpose bits where an operand's own axis is contiguous
      constexpr uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (AM ? 1u << 15 : 0u) | (BM ? 1u << 16 : 0u) |
                                 (static_cast<uint32_t>(BN >> 3) << 17) | (static_cast<uint32_t>(kBM >> 4) << 24);
      constexpr uint64_t a_step = (AM ? 2048 : 32) >> 4, b_step = (BM ? 2048 : 32) >> 4;
      int st = 0, buf = 0;
      uint32_t ph = 0, tph = 0;
      bool alive = true;
      for (int t = blockIdx.x; t < tiles && alive; t += gridDim.x) {
        if (!wait(tempty + 8 * buf, tph ^ 1, dead, P.status)) break;
        fence_after();
        for (int kb = 0; kb < P.kblocks; ++kb) {
          if (!wait(full + 8 * st, ph, dead, P.status)) { alive = false; break; }
          fence_after();
          const uint32_t a = base + st * kStage;
          const uint64_t da = operand<AM>(a), db = operand<BM>(a + kStageA);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) mma(tmem + buf * kAcc, da + k * a_step, db + k * b_step, idesc, kb > 0 || k > 0);
          mma_commit(empty + 8 * st);
          if (++st == STAGES) { st = 0; ph ^= 1; }
        }
        if (alive) mma_commit(tfull + 8 * buf);
        buf ^= 1;
        if (buf == 0) tph ^= 1;
      }
    }
    __syncwarp();
  } else {
    const int ew = warp - 2, quad = warp & 3, set = ew >> 2;
    const uint32_t mine = staging + ew * kStaging;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    int buf = 0;
    uint32_t tph = 0;
    for (int t = blockIdx.x; t < tiles; t += gridDim.x) {
      int m, n;
      tile_at(P, t, m, n);
      const long long row = static_cast<long long>(m) * kBM + quad * 32 + lane;
      const int row0 = m * kBM + quad * 32;
      const long long col0 = static_cast<long long>(n) * kBoxN;
      const uint32_t acc = tmem + buf * kAcc + lanes;
      uint4 kg[4], ku[4];
      if (EPI == kDgate)  // the first kept values come while the tile is still multiplied
      {
        const __nv_bfloat16* const p = P.gu + row * 2 * P.N;
        load_half(kg, p, row < P.M, col0 + set * 64, P.N);
        load_half(ku, p + P.N, row < P.M, col0 + set * 64, P.N);
      }
      if (!wait(tfull + 8 * buf, tph, dead, P.status)) break;
      fence_after();
      if (EPI == kGate) {
        // 64 columns a set: h, then (kept) g and u, each a 32 x 64 tile through the staging buffer
        if (set * 64 < kBoxN) {
#pragma unroll
          for (int what = 0; what < 3; ++what) {
            if (what > 0 && !P.keep) break;
            if (lane == 0) bulk_wait_read();
            __syncwarp();
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const int c = set * 64 + half * 32;
              uint32_t w[16];
              float g[32], u[32];
              if (what != 2) {
                tmem_ld32(acc + c, g);
                if (P.bias) add_bias(g, P.bias, col0 + c, P.N);
              }
              if (what != 1) {
                tmem_ld32(acc + kBoxN + c, u);
                if (P.bias) add_bias(u, P.bias + P.N, col0 + c, P.N);
              }
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                if (what == 0) w[i] = pack(act_value<true>(g[2 * i], P.act) * u[2 * i], act_value<true>(g[2 * i + 1], P.act) * u[2 * i + 1]);
                if (what == 1) w[i] = pack(g[2 * i], g[2 * i + 1]);
                if (what == 2) w[i] = pack(u[2 * i], u[2 * i + 1]);
              }
              stage_half(mine, lane, half, w);
            }
            fence_async();
            __syncwarp();
            const int x = static_cast<int>(col0) + set * 64;
            if (lane == 0 && x < P.N && row0 < P.M) {
              if (what == 0) tma_store_2d(&maps.out, mine, x, row0);
              else tma_store_3d(&maps.gu, mine, x, what - 1, row0);
              bulk_commit();
            }
          }
        }
      } else {
#pragma unroll 1
        for (int c0 = set * 64; c0 < BN; c0 += 128) {
          if (lane == 0) bulk_wait_read();
          __syncwarp();
          uint32_t later[2][16];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int c = c0 + half * 32;
            float v[32];
            uint32_t w[16];
            tmem_ld32(acc + c, v);
            if (EPI == kPlain) {
              if (P.bias) add_bias(v, P.bias, col0 + c, P.N);
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i] = pack(v[2 * i], v[2 * i + 1]);
            } else {
              const uint4 cg[4] = {kg[0], kg[1], kg[2], kg[3]}, cu[4] = {ku[0], ku[1], ku[2], ku[3]};
              const int next = half == 0 ? c + 32 : c0 + 128;
              if (next < BN) {
                const __nv_bfloat16* const p = P.gu + row * 2 * P.N;
                load_half(kg, p, row < P.M, col0 + next, P.N);
                load_half(ku, p + P.N, row < P.M, col0 + next, P.N);
              }
              const uint32_t* const gw = reinterpret_cast<const uint32_t*>(cg);
              const uint32_t* const uw = reinterpret_cast<const uint32_t*>(cu);
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                float d0, d1;
                const float a0 = act_value_grad<true>(bf16_lo(gw[i]), P.act, d0), a1 = act_value_grad<true>(bf16_hi(gw[i]), P.act, d1);
                w[i] = pack(v[2 * i] * bf16_lo(uw[i]) * d0, v[2 * i + 1] * bf16_hi(uw[i]) * d1);
                later[half][i] = pack(v[2 * i] * a0, v[2 * i + 1] * a1);
              }
            }
            stage_half(mine, lane, half, w);
          }
          fence_async();
          __syncwarp();
          const int x = static_cast<int>(col0) + c0;
          const bool store = lane == 0 && x < P.N && row0 < P.M;  // a box wholly outside is not started
          if (store) {
            if (EPI == kPlain) tma_store_2d(&maps.out, mine, x, row0);
            else tma_store_3d(&maps.out, mine, x, 0, row0);
            bulk_commit();
          }
          if (EPI == kDgate) {
            if (lane == 0) bulk_wait_read();
            __syncwarp();
            stage_half(mine, lane, 0, later[0]);
            stage_half(mine, lane, 1, later[1]);
            fence_async();
            __syncwarp();
            if (store) {
              tma_store_3d(&maps.out, mine, x, 1, row0);
              bulk_commit();
            }
          }
        }
      }
      fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(tempty + 8 * buf);
      buf ^= 1;
      if (buf == 0) tph ^= 1;
    }
    if (lane == 0) bulk_wait_all();
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kAcc));
  }
}

// ------------------------------------------------------------------------------------------ host

using Encode = PFN_cuTensorMapEncodeTiled_v12000;

Encode encoder() {
  static const Encode encode = []() -> Encode {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  return encode;
}

// Map of a bf16 matrix [rows, cols] with row stride ld: boxes of 64 columns x `box` rows, 128-byte swizzle.
bool matrix_map(CUtensorMap* map, const void* p, long long rows, long long cols, long long ld, int box) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t boxes[2] = {64, static_cast<cuuint32_t>(box)}, steps[2] = {1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Map of two matrices side by side, [rows, 2, cols] contiguous, that clips each at its own columns.
bool pair_map(CUtensorMap* map, const void* p, long long rows, long long cols, int box) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), 2, static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, static_cast<cuuint64_t>(cols) * 4};
  const cuuint32_t boxes[3] = {64, 1, static_cast<cuuint32_t>(box)}, steps[3] = {1, 1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int EPI, int BN, int STAGES, bool AM, bool BM>
cudaError_t launch(const Product& p, cudaStream_t s) {
  constexpr int kBoxN = EPI == kGate ? BN / 2 : BN;
  Maps maps;
  bool ok = AM ? matrix_map(&maps.a, p.a, p.K, p.M, p.lda, kBK) : matrix_map(&maps.a, p.a, p.M, p.K, p.lda, kBM);
  const long long brows = EPI == kGate ? 2 * p.N : p.N;
  ok = ok && (BM ? matrix_map(&maps.b, p.b, p.K, p.N, p.ldb, kBK) : matrix_map(&maps.b, p.b, brows, p.K, p.ldb, kBoxN));
  if (EPI == kDgate) ok = ok && pair_map(&maps.out, p.out, p.M, p.N, 32);
  else ok = ok && matrix_map(&maps.out, p.out, p.M, p.N, p.ldo, 32);
  maps.gu = maps.out;
  if (EPI == kGate && p.gu_out) ok = ok && pair_map(&maps.gu, p.gu_out, p.M, p.N, 32);
  if (!ok) return cudaErrorInvalidValue;
  Args a{};
  a.bias = static_cast<const __nv_bfloat16*>(p.bias);
  a.gu = static_cast<const __nv_bfloat16*>(p.gu);
  a.M = p.M;
  a.N = p.N;
  a.kblocks = static_cast<int>((p.K + kBK - 1) / kBK);
  a.mt = static_cast<int>((p.M + kBM - 1) / kBM);
  a.nt = static_cast<int>((p.N + kBoxN - 1) / kBoxN);
  a.gm = a.mt <= 32 ? a.mt : 16;  // rows of tiles that go together: their operands stay in the L2 cache
  a.act = p.act;
  a.keep = p.gu_out != nullptr;
  a.status = p.status;
  constexpr int smem = 1024 + STAGES * (kStageA + BN * kBK * 2) + kEpiWarps * kStaging + 16 * STAGES + 64;
  static_assert(smem <= 232448, "shared memory of a block");
  auto* const kernel = product_kernel<EPI, BN, STAGES, AM, BM>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const long long tiles = static_cast<long long>(a.mt) * a.nt;
  const int grid = static_cast<int>(tiles < sm_count() ? tiles : sm_count());
  kernel<<<grid, kThreads, smem, s>>>(maps, a);
  return cudaGetLastError();
}

// Width of the tiles: the one whose rounds of all SMs cover the result with the least columns (a tile's time
// goes by its columns, plus about 32 for what does not).
int choose_bn(long long M, long long N, bool gate, std::initializer_list<int> widths) {
  int best = 0;
  double least = 0;
  for (int bn : widths) {
    const long long box = gate ? bn / 2 : bn;
    const long long tiles = (M + kBM - 1) / kBM * ((N + box - 1) / box);
    const double cost = static_cast<double>((tiles + sm_count() - 1) / sm_count()) * (bn + 32);
    if (best == 0 || cost < least) {
      best = bn;
      least = cost;
    }
  }
  return best;
}

template <int EPI, bool AM, bool BM>
cudaError_t by_width(const Product& p, cudaStream_t s) {
  if constexpr (EPI == kGate) {
    if (choose_bn(p.M, p.N, true, {256, 128}) == 256) return launch<EPI, 256, 4, AM, BM>(p, s);
    return launch<EPI, 128, 6, AM, BM>(p, s);
  } else {
    switch (choose_bn(p.M, p.N, false, {256, 192, 128})) {
      case 256: return launch<EPI, 256, 4, AM, BM>(p, s);
      case 192: return launch<EPI, 192, 4, AM, BM>(p, s);
      default: return launch<EPI, 128, 6, AM, BM>(p, s);
    }
  }
}

}  // namespace tc

// TMA wants 16-byte aligned operands and rows; the kernel's tile counts fit 32 bits.
bool tc_applies(const Product& p) {
  if (p.dtype != MSL_DTYPE_BF16 || !tc::encoder()) return false;
  if (!multiple_of(p.a, 16) || !multiple_of(p.b, 16) || !multiple_of(p.out, 16) || p.lda % 8 || p.ldb % 8 || p.ldo % 8 || p.N % 8) return false;
  if (p.bias && !multiple_of(p.bias, 16)) return false;
  if ((p.gu && !multiple_of(p.gu, 16)) || (p.gu_out && !multiple_of(p.gu_out, 16))) return false;
  if (p.M > (1LL << 31) - 256 || p.N > (1LL << 30) || p.K > (1LL << 31) - 256) return false;
  if ((p.M + 127) / 128 * ((p.N + 63) / 64) > (1LL << 30)) return false;
  return true;
}

cudaError_t launch_product_tc(const Product& p, cudaStream_t s) {
  switch (p.epilogue) {
    case kGate: return tc::by_width<kGate, false, false>(p, s);
    case kDgate: return tc::by_width<kDgate, false, true>(p, s);
    default:
      if (p.a_major) return tc::by_width<kPlain, true, true>(p, s);
      return p.b_major ? tc::by_width<kPlain, false, true>(p, s) : tc::by_width<kPlain, false, false>(p, s);
  }
}

}  // namespace ffn
}  // namespace msl
