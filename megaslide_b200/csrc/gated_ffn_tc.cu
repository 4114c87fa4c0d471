// The gated feed-forward block's products on the 5th-generation tensor cores (bf16 operands, float32 sums in
// tensor memory).
//
// C[M, N] = sum_k A(m, k) B(n, k), A and B each with k or its own axis contiguous, so one kernel serves the
// forward (x w_in^T, h w_out^T: both k-major), the input gradients (dy w_out, [dg du] w_in: B n-major) and the
// weight gradients ([dg du]^T x, dy^T h: both with the summed axis, the tokens, outermost).  Operand tiles come
// by TMA with the 128-byte swizzle that tcgen05.mma reads in either orientation; ragged edges are the TMA's zero
// fill and clipping, no element is handled apart.
//
// Two CTAs (a cluster) share a 256 x BN tile: each holds 128 rows of A, half of B and the sums of its 128 rows,
// and every multiplication (256 x BN x 16) reads both halves of B, which each SM loads and stores only once.  In a
// CTA one thread loads (a ring of stages), one thread of the first CTA issues the multiplications, eight warps turn
// finished sums into results while the next tile is multiplied into the other half of the tensor memory.  The
// pairs walk over the tiles, one pair per two SMs.
//   gate:  the tile's columns are BN/2 gate columns (the first CTA's half of B) and the same columns of the other
//          projection, so g and u of an element meet in one epilogue thread: bias, activation and product; for
//          the backward it also keeps u act'(g) and act(g), 24 bits each (g and u themselves, in bf16, would
//          be rounded before the activation's derivative, and cost the backward the activation again): the upper 16 by
//          TMA, the lower 8 from the registers, 32 bytes a row
//   dgate: the sums are the gradient of h; the epilogue fetches the two kept factors a step ahead, by TMA and into
//          registers, and writes the gradients of g and u over the former in shared memory, from where they leave
//
// Tiles that do not fill a last round of all pairs are cut along k among the pairs left over: their parts' sums
// go to the workspace in float32 and a small kernel joins them, in order, and does the epilogue.
//
// What bounds it: an SM takes in about 63 bytes a clock, 520 clocks for the 32 KB of a stage, whose multiplications
// take 512; with both that near, a stage takes 620 to 680 clocks (82% of the tensor cores; 128 x 256 tiles of one CTA
// alone need 48 KB).  Where k is short the epilogue's bytes share that path: with 18 stages a tile (k = 1152) the gate's
// results are 17% more and its stage takes 900 clocks, dgate's kept factors and results 44% more.  16 epilogue warps
// instead of 8, or a second loading thread, change nothing.  In long runs the power limit holds the clock near
// 1.4 to 1.6 GHz.  16384 x 1152 x 4608: gate with kept factors 334 us (1.04 PFLOP/s), dgate 202 (0.86), the others 1.26 to
// 1.32 PFLOP/s.  In a hot loop 4096 x 7168 x 28672 forward 1.23 (with kept factors 1.18) and backward 1.18, the same
// products by cuBLAS 1.22 to 1.41 without the activations; 32768 x 1152 x 4608 1.20 (0.99) and 0.99, cuBLAS 1.20 to 1.30.

#include "gated_ffn.cuh"
#include "tcgen05.cuh"

namespace msl {
namespace ffn {
namespace tc {

using namespace msl::t5;

constexpr int kBM = 128, kBK = 64;  // of a CTA; a pair has 2 kBM rows
constexpr int kEpiWarps = 8;
constexpr int kThreads = 64 + 32 * kEpiWarps;
constexpr int kStageA = kBM * kBK * 2;
constexpr int kTile = 2048;           // a staging tile: 32 rows x 32 bf16
constexpr int kStaging = 4 * kTile;   // of an epilogue warp
constexpr int kRing = 5 * 2 * kStageA;  // shared memory of the stages
constexpr int kMaxStages = 8;

struct Maps {
  CUtensorMap a, b, out, kept;
};

struct Args {
  const __nv_bfloat16* bias;
  long long M, N;
  int kblocks, mt, nt, gm, keep;  // mt: tiles of 256 rows
  int bn, stages, stage_bytes, boxes;  // width of a tile, the ring, boxes of 64 that a CTA's half of B takes
  int full, items, parts, kper;        // tiles done whole; with the parts of the others; parts of a tile, their k-blocks
  float* partial;                      // [items - full][2 CTAs][4 x 32 rows][bn / 32][32 columns][32 rows]
  uint8_t* low;                        // low bytes of the kept factors
  uint32_t* status;
};

// ------------------------------------------------------------------------------------------ kernel

__device__ __forceinline__ void tile_at(const Args& P, int t, int& m, int& n) {
  const int per = P.gm * P.nt, g = t / per, r = t - g * per;
  const int first = g * P.gm, rows = min(P.gm, P.mt - first);
  n = r / rows;
  m = first + r - n * rows;
}

// What a pair does in a turn: a tile, its k-blocks [k0, k1), and its place in `partial` (-1: the whole tile).
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

__device__ __forceinline__ uint32_t pack(float lo, float hi) {
  __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&t);
}

// Chunk c (16 bytes) of row r of a staging tile lies at c ^ (r / 2 & 3), as the TMA's 64-byte swizzle has it (and no
// two lanes of a quarter meet in a bank).
__device__ __forceinline__ uint32_t chunk32(uint32_t base, int row, int c) { return base + row * 64 + ((c ^ ((row >> 1) & 3)) << 4); }
__device__ __forceinline__ uint4 lds(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ void sts(uint32_t at, const uint32_t (&w)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
}

__device__ __forceinline__ void stage(uint32_t base, int row, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t w[4] = {pack(v[c * 8], v[c * 8 + 1]), pack(v[c * 8 + 2], v[c * 8 + 3]), pack(v[c * 8 + 4], v[c * 8 + 5]), pack(v[c * 8 + 6], v[c * 8 + 7])};
    sts(chunk32(base, row, c), w);
  }
}

// Kept factors: upper halves to a staging tile, low bytes to 32 bytes of a row of their own (columns from N to low_width(N)
// are room for what is not read).
__device__ __forceinline__ void stage_high(uint32_t base, int row, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const uint32_t w[4] = {kept_high(v[c * 8], v[c * 8 + 1]), kept_high(v[c * 8 + 2], v[c * 8 + 3]), kept_high(v[c * 8 + 4], v[c * 8 + 5]), kept_high(v[c * 8 + 6], v[c * 8 + 7])};
    sts(chunk32(base, row, c), w);
  }
}
__device__ __forceinline__ void put_low(uint8_t* to, int cols, const float (&v)[32]) {
#pragma unroll
  for (int c = 0; c < 2; ++c)
    if (c * 16 < cols)
      reinterpret_cast<uint4*>(to)[c] = make_uint4(kept_low(v[c * 16], v[c * 16 + 1], v[c * 16 + 2], v[c * 16 + 3]), kept_low(v[c * 16 + 4], v[c * 16 + 5], v[c * 16 + 6], v[c * 16 + 7]),
                                                   kept_low(v[c * 16 + 8], v[c * 16 + 9], v[c * 16 + 10], v[c * 16 + 11]), kept_low(v[c * 16 + 12], v[c * 16 + 13], v[c * 16 + 14], v[c * 16 + 15]));
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

template <int EPI, bool AM, bool BM, int ACT>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args P) {
  constexpr int kAcc = 256;  // tensor memory columns of a tile's sums
  const int half = P.bn / 2;                              // rows of B that a CTA holds
  const int width = EPI == kGate ? half : P.bn;           // columns of the result that a tile covers
  const int stages = P.stages;
  extern __shared__ uint8_t raw[];
  const uint32_t base = (smem_u32(raw) + 1023) & ~1023u;
  const uint32_t staging = base + kRing;
  const uint32_t bars = staging + kEpiWarps * kStaging;
  const uint32_t full = bars, empty = bars + 8 * kMaxStages, peer = empty + 8 * kMaxStages, tfull = peer + 8 * kMaxStages, tempty = tfull + 16;
  const uint32_t kept = tempty + 16, tmem_slot = kept + 16 * kEpiWarps, last = tmem_slot + 8;
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
    for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(kept + 8 * i, 1);
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
        const int m = w.m, n = w.n;
        const int arow = (2 * m + rank) * kBM;
        // rows of B: halves of the tile's columns; for the gate the first CTA has the gate's, the second the others
        const int brow = EPI == kGate ? n * width + (rank ? static_cast<int>(P.N) : 0) : n * width + rank * half;
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!wait(empty + 8 * st, ph ^ 1, dead, P.status)) { alive = false; break; }
          const uint32_t a = base + st * P.stage_bytes, b = a + kStageA, bar = full + 8 * st;
          mbar_expect(bar, P.stage_bytes);
          if (AM) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i) tma_load_2d(a + i * 8192, &maps.a, bar, arow + i * 64, kb * kBK);
          } else {
            tma_load_2d(a, &maps.a, bar, kb * kBK, arow);
          }
          if (BM) {
            for (int i = 0; i < P.boxes; ++i) tma_load_2d(b + i * 8192, &maps.b, bar, brow + i * 64, kb * kBK);
          } else {
            tma_load_2d(b, &maps.b, bar, kb * kBK, brow);
          }
          if (++st == stages) { st = 0; ph ^= 1; }
        }
      }
      // the copies still in flight land before the CTA leaves
      const long long since = clock64();
      if (!alive)
        for (int i = 0; i < stages; ++i)
          while (!mbar_try(full + 8 * i, (i < st ? ph : ph ^ 1)) && clock64() - since < kWaitClocks) {
          }
    }
    __syncwarp();
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      // bf16 x bf16 -> float32, transpose bits where an operand's own axis is contiguous
      const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | (AM ? 1u << 15 : 0u) | (BM ? 1u << 16 : 0u) |
                             (static_cast<uint32_t>(P.bn >> 3) << 17) | (static_cast<uint32_t>(2 * kBM >> 4) << 24);
      constexpr uint64_t a_step = (AM ? 2048 : 32) >> 4, b_step = (BM ? 2048 : 32) >> 4;
      int st = 0, buf = 0;
      uint32_t ph = 0, tph = 0;
      bool alive = true;
      for (int t = t0; t < P.items && alive; t += tstep) {
        if (!wait(tempty + 8 * buf, tph ^ 1, dead, P.status)) { alive = false; break; }
        fence_after();
        const Item w = item_at(P, t);
        for (int kb = w.k0; kb < w.k1; ++kb) {
          if (!wait(full + 8 * st, ph, dead, P.status) || !wait(peer + 8 * st, ph, dead, P.status)) { alive = false; break; }
          fence_after();
          const uint32_t a = base + st * P.stage_bytes;
          const uint64_t da = operand<AM>(a), db = operand<BM>(a + kStageA);
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k) mma(tmem + buf * kAcc, da + k * a_step, db + k * b_step, idesc, kb > w.k0 || k > 0);
          mma_commit(empty + 8 * st);
          if (++st == stages) { st = 0; ph ^= 1; }
        }
        if (alive) mma_commit(tfull + 8 * buf);
        buf ^= 1;
        if (buf == 0) tph ^= 1;
      }
      if (!alive) mma_drain(last);
    } else if (lane == 0) {
      // the second CTA tells the first when its operands have landed
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
    const uint32_t mine = staging + ew * kStaging;
    const uint32_t lanes = static_cast<uint32_t>(quad * 32) << 16;
    const uint32_t mykept = kept + 16 * ew;
    int buf = 0;
    uint32_t tph = 0;
    uint32_t turn = 0;  // steps so far
    // a tile goes in steps of 32 columns, the first half of them to set 0
    const int steps = width / 32, first = set ? (steps + 1) / 2 : 0, last = set ? steps : (steps + 1) / 2;
    for (int t = t0; t < P.items; t += tstep) {
      const Item w = item_at(P, t);
      const int m = w.m, n = w.n;
      const int row0 = (2 * m + rank) * kBM + quad * 32;
      const int col0 = n * width;
      const uint32_t acc = tmem + buf * kAcc + lanes;
      const bool rows_in = row0 < P.M;  // a box wholly outside is not started
      // dgate: the staging buffer holds the kept factors of two steps
      auto fetch = [&](uint32_t at, int i) {
        const uint32_t to = mine + (at & 1) * 2 * kTile, bar = mykept + 8 * (at & 1);
        mbar_expect(bar, 2 * kTile);
        tma_load_3d(to, &maps.kept, bar, col0 + i * 32, 0, row0);
        tma_load_3d(to + kTile, &maps.kept, bar, col0 + i * 32, 1, row0);
      };
      uint4 low[4];  // of the step to come: 32 low bytes of either factor
      auto fetch_low = [&](int i) {
        const long long W = low_width(P.N), x = col0 + i * 32;
        const uint4* const from = reinterpret_cast<const uint4*>(P.low + 2 * W * (row0 + lane) + x);
        const bool in = row0 + lane < P.M;
#pragma unroll
        for (int f = 0; f < 2; ++f)
#pragma unroll
          for (int c = 0; c < 2; ++c) low[f * 2 + c] = in && x + c * 16 < P.N ? __ldg(from + f * (W / 16) + c) : make_uint4(0, 0, 0, 0);
      };
      if (EPI == kDgate && first < last && w.part < 0) fetch_low(first);
      if (EPI == kDgate && lane == 0 && first < last && w.part < 0) {  // on their way while the tile is still multiplied
        bulk_wait_read<0>();                             // the last tile's results have left
        fetch(turn, first);
        if (first + 1 < last) fetch(turn + 1, first + 1);
      }
      __syncwarp();
      if (!wait_warp(tfull + 8 * buf, tph, dead, P.status)) break;
      fence_after();
      bool alive = true;
      if (w.part >= 0) {
        const int blocks = P.bn / 32;
        float* const to = P.partial + static_cast<size_t>((w.part * 2 + rank) * 4 + quad) * blocks * 1024 + lane;
#pragma unroll 1
        for (int i = set; i < blocks; i += 2) {
          float v[32];
          tmem_ld32(acc + i * 32, v);
#pragma unroll
          for (int j = 0; j < 32; ++j) to[i * 1024 + j * 32] = v[j];
        }
      }
#pragma unroll 1
      for (int i = w.part < 0 ? first : last; i < last; ++i, ++turn) {
        const int c = i * 32, x = col0 + c;
        const bool store = lane == 0 && rows_in && x < P.N;
        float v[32];
        tmem_ld32(acc + c, v);
        if (EPI == kDgate) {
          const uint32_t g0 = mine + (turn & 1) * 2 * kTile, u0 = g0 + kTile;
          const uint4 now[4] = {low[0], low[1], low[2], low[3]};
          if (i + 1 < last) fetch_low(i + 1);
          if (!wait_warp(mykept + 8 * (turn & 1), (turn >> 1) & 1, dead, P.status)) { alive = false; break; }
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const uint4 gv = lds(chunk32(g0, lane, q)), uv = lds(chunk32(u0, lane, q));
            const uint4 gl = now[q / 2], ul = now[2 + q / 2];
            const uint32_t g01 = q & 1 ? gl.z : gl.x, g23 = q & 1 ? gl.w : gl.y, u01 = q & 1 ? ul.z : ul.x, u23 = q & 1 ? ul.w : ul.y;
            const float* const h = v + q * 8;
            const uint32_t dg[4] = {pack(h[0] * kept_at<0>(gv.x, g01), h[1] * kept_at<1>(gv.x, g01)), pack(h[2] * kept_at<2>(gv.y, g01), h[3] * kept_at<3>(gv.y, g01)),
                                    pack(h[4] * kept_at<0>(gv.z, g23), h[5] * kept_at<1>(gv.z, g23)), pack(h[6] * kept_at<2>(gv.w, g23), h[7] * kept_at<3>(gv.w, g23))};
            const uint32_t du[4] = {pack(h[0] * kept_at<0>(uv.x, u01), h[1] * kept_at<1>(uv.x, u01)), pack(h[2] * kept_at<2>(uv.y, u01), h[3] * kept_at<3>(uv.y, u01)),
                                    pack(h[4] * kept_at<0>(uv.z, u23), h[5] * kept_at<1>(uv.z, u23)), pack(h[6] * kept_at<2>(uv.w, u23), h[7] * kept_at<3>(uv.w, u23))};
            sts(chunk32(g0, lane, q), dg);
            sts(chunk32(u0, lane, q), du);
          }
          fence_async();
          __syncwarp();
          if (store) {
            tma_store_3d(&maps.out, g0, x, 0, row0);
            tma_store_3d(&maps.out, u0, x, 1, row0);
            bulk_commit();
          }
          if (i + 2 < last && lane == 0) {
            bulk_wait_read<0>();
            fetch(turn + 2, i + 2);
          }
        } else if (EPI == kGate) {
          // staging tiles: the two kept factors, and h in turn in the two others
          float u[32];
          tmem_ld32(acc + half + c, u);
          if (P.bias) {
            add_bias(v, P.bias, x, P.N);
            add_bias(u, P.bias + P.N, x, P.N);
          }
          if (P.keep) {
            float d[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) {
              float da;
              v[j] = act_grad_fast<ACT>(v[j], da);
              d[j] = u[j] * da;
            }
            if (lane == 0) bulk_wait_read<0>();
            __syncwarp();
            stage_high(mine, lane, d);
            stage_high(mine + kTile, lane, v);
            if (row0 + lane < P.M) {
              const long long W = low_width(P.N);
              uint8_t* const to = P.low + 2 * W * (row0 + lane) + x;
              const int cols = static_cast<int>(min(32LL, P.N - x));  // under 1 where the tile's columns are none of the matrix'
              put_low(to, cols, d);
              put_low(to + W, cols, v);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] *= u[j];
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) v[j] = act_fast<ACT>(v[j]) * u[j];
            if (lane == 0) bulk_wait_read<1>();
            __syncwarp();
          }
          const uint32_t to = mine + (2 + (turn & 1)) * kTile;
          stage(to, lane, v);
          fence_async();
          __syncwarp();
          if (store) {
            if (P.keep) {
              tma_store_3d(&maps.kept, mine, x, 0, row0);
              tma_store_3d(&maps.kept, mine + kTile, x, 1, row0);
            }
            tma_store_2d(&maps.out, to, x, row0);
          }
          if (lane == 0) bulk_commit();
        } else {
          if (P.bias) add_bias(v, P.bias, x, P.N);
          if (lane == 0) bulk_wait_read<3>();
          __syncwarp();
          const uint32_t to = mine + (turn & 3) * kTile;
          stage(to, lane, v);
          fence_async();
          __syncwarp();
          if (store) tma_store_2d(&maps.out, to, x, row0);
          if (lane == 0) bulk_commit();
        }
      }
      if (!alive) break;
      fence_before();
      __syncwarp();
      if (lane == 0) arrive_first(tempty + 8 * buf);
      buf ^= 1;
      if (buf == 0) tph ^= 1;
    }
    if (lane == 0) {
      if (EPI == kDgate && *dead) {  // fetches may still be in flight: those of the next two steps
        const long long since = clock64();
        for (uint32_t i = turn; i < turn + 2; ++i)
          while (!mbar_try(mykept + 8 * (i & 1), (i >> 1) & 1) && clock64() - since < kWaitClocks / 4) {
          }
      }
      bulk_wait_all();
    }
    __syncwarp();
  }
  fence_before();
  __syncthreads();
  cluster_sync();  // neither CTA leaves while the other may still read its operands or arrive at its barriers
  if (warp == 1) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * kAcc));
  }
}

// ------------------------------------------------------------------------------------------ join

// Epilogue of the tiles that were cut along k: a warp adds up the parts of 32 rows x 8 columns, four parts' loads
// in flight, always in their order.
struct JoinArgs {
  Args tc;
  __nv_bfloat16* out;
  const __nv_bfloat16* kept;
  __nv_bfloat16* kept_out;
  long long ldo;
};

__device__ __forceinline__ void add_parts(const Args& P, int tail, int rank, int quad, int block, int col, int lane, float (&v)[8]) {
  const size_t hop = static_cast<size_t>(8) * (P.bn / 32) * 1024;  // from a part to the next
  const float* from = P.partial + (static_cast<size_t>((tail * P.parts * 2 + rank) * 4 + quad) * (P.bn / 32) + block) * 1024 + col * 32 + lane;
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = 0.f;
  for (int s = 0; s < P.parts; s += 4) {
    float t[4][8];
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) t[u][j] = s + u < P.parts ? __ldg(from + (s + u) * hop + j * 32) : 0.f;
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] += t[u][j];
  }
}
__device__ __forceinline__ void add_bias8(float (&v)[8], const __nv_bfloat16* bias) {
  const uint4 b = __ldg(reinterpret_cast<const uint4*>(bias));
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] += bf16_lo(w[i]);
    v[2 * i + 1] += bf16_hi(w[i]);
  }
}
__device__ __forceinline__ void put8(__nv_bfloat16* to, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = make_uint4(pack(v[0], v[1]), pack(v[2], v[3]), pack(v[4], v[5]), pack(v[6], v[7]));
}

__device__ __forceinline__ void keep8(__nv_bfloat16* to, uint8_t* low, const float (&v)[8]) {
  *reinterpret_cast<uint4*>(to) = make_uint4(kept_high(v[0], v[1]), kept_high(v[2], v[3]), kept_high(v[4], v[5]), kept_high(v[6], v[7]));
  *reinterpret_cast<uint2*>(low) = make_uint2(kept_low(v[0], v[1], v[2], v[3]), kept_low(v[4], v[5], v[6], v[7]));
}
__device__ __forceinline__ void kept8(const __nv_bfloat16* from, const uint8_t* low, float (&v)[8]) {
  const uint4 w = __ldg(reinterpret_cast<const uint4*>(from));
  const uint2 l = __ldg(reinterpret_cast<const uint2*>(low));
  v[0] = kept_at<0>(w.x, l.x); v[1] = kept_at<1>(w.x, l.x); v[2] = kept_at<2>(w.y, l.x); v[3] = kept_at<3>(w.y, l.x);
  v[4] = kept_at<0>(w.z, l.y); v[5] = kept_at<1>(w.z, l.y); v[6] = kept_at<2>(w.w, l.y); v[7] = kept_at<3>(w.w, l.y);
}

template <int EPI, int ACT>
__global__ void __launch_bounds__(512) join_kernel(const __grid_constant__ JoinArgs J) {
  const Args& P = J.tc;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, half = P.bn / 2, width = EPI == kGate ? half : P.bn, steps = width / 32;
  const int quad = warp & 3, col = (warp >> 2) * 8, rank = blockIdx.y, tail = blockIdx.x / steps, i = blockIdx.x - tail * steps;
  int m, n;
  tile_at(P, P.full + tail, m, n);
  const long long row = (2LL * m + rank) * kBM + quad * 32 + lane;
  const int x = n * width + i * 32 + col;
  if (x >= P.N || (2LL * m + rank) * kBM + quad * 32 >= P.M) return;  // N is a multiple of 8
  float v[8], u[8];
  add_parts(P, tail, rank, quad, i, col, lane, v);
  if (EPI == kGate) add_parts(P, tail, rank, quad, steps + i, col, lane, u);
  if (EPI != kDgate && P.bias) add_bias8(v, P.bias + x);
  if (EPI == kGate && P.bias) add_bias8(u, P.bias + P.N + x);
  if (row >= P.M) return;
  if (EPI == kGate) {
    float d[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float da;
      v[j] = act_grad_fast<ACT>(v[j], da);
      d[j] = u[j] * da;
    }
    if (J.kept_out) {
      uint8_t* const low = P.low + row * 2 * low_width(P.N) + x;
      keep8(J.kept_out + row * 2 * P.N + x, low, d);
      keep8(J.kept_out + row * 2 * P.N + P.N + x, low + low_width(P.N), v);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= u[j];
  }
  if (EPI == kDgate) {
    const __nv_bfloat16* const kept = J.kept + row * 2 * P.N + x;
    const uint8_t* const low = P.low + row * 2 * low_width(P.N) + x;
    float g[8], a[8];
    kept8(kept, low, g);
    kept8(kept + P.N, low + low_width(P.N), a);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      u[j] = v[j] * a[j];
      v[j] *= g[j];
    }
    put8(J.out + row * 2 * P.N + x, v);
    put8(J.out + row * 2 * P.N + P.N + x, u);
  } else {
    put8(J.out + row * J.ldo + x, v);
  }
}

// ------------------------------------------------------------------------------------------ host

// Map of a bf16 matrix [rows, cols] with row stride ld: boxes of `box` rows x 64 columns (128-byte swizzle) or 32 (64).
bool matrix_map(CUtensorMap* map, const void* p, long long rows, long long cols, long long ld, int box, int width = 64) {
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(ld) * 2};
  const cuuint32_t boxes[2] = {static_cast<cuuint32_t>(width), static_cast<cuuint32_t>(box)}, steps[2] = {1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   width == 64 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Map of two matrices side by side, [rows, 2, cols] contiguous, that clips each at its own columns: boxes of 32 rows
// x 32 columns (64-byte swizzle).
bool pair_map(CUtensorMap* map, const void* p, long long rows, long long cols) {
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(cols), 2, static_cast<cuuint64_t>(rows)};
  const cuuint64_t strides[2] = {static_cast<cuuint64_t>(cols) * 2, static_cast<cuuint64_t>(cols) * 4};
  const cuuint32_t boxes[3] = {32, 1, 32}, steps[3] = {1, 1, 1};
  return encoder()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(p), dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                   CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a product is cut: tiles of bn columns, `full` of them whole, the others in `parts` along k.
struct Plan {
  int bn, parts, kper;
  long long mt, nt, full, items;
  size_t bytes;
};

// The cheapest cut by what was measured (microseconds): a block of 64 k of a 256 x bn tile takes 0.23 + 0.00066
// bn (B by boxes of 64 where its own axis is contiguous) whatever its neighbours do, the end of a round about 3
// more, joining parts 7; a part has at least 4 blocks.
Plan plan(long long M, long long N, long long K, bool gate, bool boxed) {
  const long long pairs = sm_count() / 2, kblocks = (K + kBK - 1) / kBK;
  Plan best{};
  double least = 0;
  for (int bn = 256; bn >= 64; bn -= gate ? 64 : 32) {
    Plan p{};
    const long long width = gate ? bn / 2 : bn;
    p.bn = bn;
    p.mt = (M + 2 * kBM - 1) / (2 * kBM);
    p.nt = (N + width - 1) / width;
    const long long tiles = p.mt * p.nt, tail = tiles % pairs;
    const double block = 0.23 + 0.00066 * (boxed ? (bn / 2 + 63) / 64 * 128 : bn) + 0.0001 * bn;
    for (long long parts = 1; parts == 1 || (tail > 0 && parts <= pairs / tail && parts <= 32); ++parts) {
      const long long kper = (kblocks + parts - 1) / parts;
      if (parts > 1 && (kper < 4 || (kblocks + kper - 1) / kper != parts)) continue;
      const double rounds = static_cast<double>(tiles / pairs) + (tail == 0 ? 0.0 : parts == 1 ? 1.0 : static_cast<double>(kper) / kblocks);
      const double cost = rounds * kblocks * block + 3.0 + (parts > 1 ? 7.0 : 0.0);
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

template <int EPI, bool AM, bool BM, int ACT>
cudaError_t launch(const Product& p, cudaStream_t s) {
  const Plan cut = plan(p.M, p.N, p.K, EPI == kGate, BM);
  if (cut.bytes > p.partial_bytes) return cudaErrorInvalidValue;
  Args a{};
  a.bn = cut.bn;
  a.full = static_cast<int>(cut.full);
  a.items = static_cast<int>(cut.items);
  a.parts = cut.parts;
  a.kper = cut.kper;
  a.partial = p.partial;
  a.boxes = (a.bn / 2 + 63) / 64;
  a.stage_bytes = kStageA + (BM ? a.boxes * 8192 : a.bn / 2 * kBK * 2);
  // stages start on the swizzle's 1024 bytes: half of B is a multiple of 16 rows of 128 bytes
  a.stages = kRing / a.stage_bytes < kMaxStages ? kRing / a.stage_bytes : kMaxStages;
  cudaError_t e = bind_context();
  if (e != cudaSuccess) return e;
  Maps maps;
  bool ok = AM ? matrix_map(&maps.a, p.a, p.K, p.M, p.lda, kBK) : matrix_map(&maps.a, p.a, p.M, p.K, p.lda, kBM);
  const long long brows = EPI == kGate ? 2 * p.N : p.N;
  ok = ok && (BM ? matrix_map(&maps.b, p.b, p.K, p.N, p.ldb, kBK) : matrix_map(&maps.b, p.b, brows, p.K, p.ldb, a.bn / 2));
  if (EPI == kDgate) ok = ok && pair_map(&maps.out, p.out, p.M, p.N) && pair_map(&maps.kept, p.kept, p.M, p.N);
  else ok = ok && matrix_map(&maps.out, p.out, p.M, p.N, p.ldo, 32, 32);
  if (EPI == kGate && p.kept_out) ok = ok && pair_map(&maps.kept, p.kept_out, p.M, p.N);
  else if (EPI != kDgate) maps.kept = maps.out;
  if (!ok) return cudaErrorInvalidValue;
  a.bias = static_cast<const __nv_bfloat16*>(p.bias);
  a.M = p.M;
  a.N = p.N;
  a.kblocks = static_cast<int>((p.K + kBK - 1) / kBK);
  a.mt = static_cast<int>(cut.mt);
  a.nt = static_cast<int>(cut.nt);
  a.gm = a.mt <= 16 ? a.mt : 8;  // rows of tiles that go together: their operands stay in the L2 cache
  a.keep = p.kept_out != nullptr;
  a.low = p.low;
  a.status = p.status;
  constexpr int smem = 1024 + kRing + kEpiWarps * kStaging + 24 * kMaxStages + 16 * kEpiWarps + 64;
  static_assert(smem <= 232448, "shared memory of a block");
  auto* const kernel = product_kernel<EPI, AM, BM, ACT>;
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
  JoinArgs j{a, static_cast<__nv_bfloat16*>(p.out), static_cast<const __nv_bfloat16*>(p.kept), static_cast<__nv_bfloat16*>(p.kept_out), p.ldo};
  const int steps = (EPI == kGate ? a.bn / 2 : a.bn) / 32;
  join_kernel<EPI, ACT><<<dim3((a.mt * a.nt - a.full) * steps, 2), 512, 0, s>>>(j);
  count_launches(1);
  return cudaGetLastError();
}

}  // namespace tc

// TMA wants 16-byte aligned operands and rows; the kernel's tile counts fit 32 bits.
bool tc_applies(const Product& p) {
  if (p.dtype != MSL_DTYPE_BF16 || !t5::encoder()) return false;
  if (!multiple_of(p.a, 16) || !multiple_of(p.b, 16) || !multiple_of(p.out, 16) || p.lda % 8 || p.ldb % 8 || p.ldo % 8 || p.N % 8) return false;
  if (p.bias && !multiple_of(p.bias, 16)) return false;
  if ((p.kept && !multiple_of(p.kept, 16)) || (p.kept_out && !multiple_of(p.kept_out, 16)) || ((p.kept || p.kept_out) && !multiple_of(p.low, 16))) return false;
  if (p.M > (1LL << 31) - 256 || p.N > (1LL << 30) || p.K > (1LL << 31) - 256) return false;
  if ((p.M + 127) / 128 * ((p.N + 63) / 64) > (1LL << 30)) return false;
  return true;
}

size_t tc_partial_bytes(long long M, long long N, long long K, int epilogue, bool b_major) {
  return tc::plan(M, N, K, epilogue == kGate, b_major).bytes;
}

cudaError_t launch_product_tc(const Product& p, cudaStream_t s) {
  const bool silu = p.act == MSL_ACT_SILU;
  switch (p.epilogue) {
    case kGate:
      return silu ? tc::launch<kGate, false, false, MSL_ACT_SILU>(p, s) : tc::launch<kGate, false, false, MSL_ACT_GELU>(p, s);
    case kDgate:
      return tc::launch<kDgate, false, true, 0>(p, s);
    default:
      if (p.a_major) return tc::launch<kPlain, true, true, 0>(p, s);
      return p.b_major ? tc::launch<kPlain, false, true, 0>(p, s) : tc::launch<kPlain, false, false, 0>(p, s);
  }
}

}  // namespace ffn
}  // namespace msl
