// Rotary positions with several axes, alone (msl_rope3d) and in one pass with the RMS norm of queries and
// keys for each head (msl_qk_norm_rope_fwd / _bwd).
//
//   r = 1 / sqrt(mean_i x_i^2 + eps),  n_i = x_i r g_i,  (y_a, y_b) = (n_a c - n_b s, n_b c + n_a s)
//   backward: dn = the inverse rotation of dy,  dg_i = sum over tokens and heads of dn_i x_i r,
//             a_i = dn_i g_i,  dx_i = r (a_i - x_i r^2 mean_j(a_j x_j))
//
// Bound by bytes: every element is read once and written once (the backward reads x again instead of
// keeping r, which costs nothing, as the norm's gradient needs x anyway).
//
// Layout: a block works on the queries or on the keys; a warp takes a few consecutive tokens, one after the
// other, and goes through a token's heads.  A head is cut into slots of 2V channels, V pairs; a lane keeps one
// slot (SL of them where V is small) for the whole call, so the cosines and sines of a token are loaded once and
// serve all its heads, and the gradients of the weights add up in registers.  32 / (lanes of a head) heads go
// through together, whole rows of adjacent loads; the sums of a head are shuffles among its lanes.
// The loads run three stages ahead through shared memory, each lane copying its own bytes to its own place
// (cp.async: no registers hold them and no lane waits for another), over a warp's tokens.  The arithmetic goes
// two pairs at a time (fma.rn.f32x2), the weights are multiplied into the cosines and sines once per token, and
// lanes without a head load a neighbour's instead of branching (they only never store).
//
// Measured, bf16 (of the measured copy bandwidth): rotation of 131072 x 16 x 72, 604 MB, 113 us, 5.4 TB/s (82%); norm and
// rotation of 262144 x 24 x 64 queries and keys, 3.2 GB, 545 us, 5.9 TB/s (90%); their backward, 4.8 GB, 758 us, 6.4 TB/s
// (97%); in a long loop 593 and 859.  At these rates the GPU comes to its 1000 W (a plain copy takes 770) and the clock
// falls to 1.7 GHz, so instructions count beside bytes.  131072 x 16 x 72 queries and keys, whose 9 lanes a head sum by
// the loop and leave 5 of 32 idle: 297 and 505 us, 4.1 and 3.6 TB/s.  With loads straight to registers 145, 740 and
// 1035 us.

#include "msl_abi.cuh"
#include "msl_common.cuh"

namespace msl {
namespace rot {

struct Params {
  const void* x[2];
  const void* dy[2];
  void* y[2];
  long long x_ld[2], dy_ld[2], y_ld[2];
  const void* weight[2];
  float* partial;  // [blocks][d] sums of the weights' gradients
  int blocks0;     // blocks of the queries; the others are the keys'
  int heads[2];
  int w_bf16;
  const float2* table;
  const int* index;
  long long index_rows;
  uint32_t* status;
  long long rows, tokens;
  int splits;     // warps that share a token's heads
  int group;      // consecutive tokens of a warp
  int table_vec;  // the table's entries of a slot are one axis' and 16-byte aligned
  int size[3], npair[3];
  int frame0, HW, W;
  int d, R;
  int lanes;  // of a head
  float eps, inv_d, sign;
};

// ------------------------------------------------------------------------------------------ two at a time

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(reinterpret_cast<uint64_t&>(d)) : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;"
      : "=l"(reinterpret_cast<uint64_t&>(d))
      : "l"(reinterpret_cast<uint64_t&>(a)), "l"(reinterpret_cast<uint64_t&>(b)), "l"(reinterpret_cast<uint64_t&>(c)));
  return d;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
__device__ __forceinline__ float2 neg(float2 v) { return make_float2(-v.x, -v.y); }

template <int BYTES>
struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// N elements between p and registers, in words of their size or 16 bytes, whichever is less
template <typename T, int N>
__device__ __forceinline__ void load(const T* p, T* o) {
  constexpr int kBytes = N * static_cast<int>(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16;
  using W = typename Word<kWord>::type;
#pragma unroll
  for (int i = 0; i < kBytes / kWord; ++i) reinterpret_cast<W*>(o)[i] = reinterpret_cast<const W*>(p)[i];
}
template <typename T, int N>
__device__ __forceinline__ void store(T* p, const T* o) {
  constexpr int kBytes = N * static_cast<int>(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16;
  using W = typename Word<kWord>::type;
#pragma unroll
  for (int i = 0; i < kBytes / kWord; ++i) reinterpret_cast<W*>(p)[i] = reinterpret_cast<const W*>(o)[i];
}

// A lane's V * SL pairs of one head, as they lie in memory.
template <typename T, int V, int SL, bool INTER>
struct alignas(16) Raw {
  T e[SL][2 * V];

  // `hi` elements after the slot's first half lies its second
  __device__ __forceinline__ void get(const T* const (&slot)[SL], const int (&hi)[SL]) {
#pragma unroll
    for (int s = 0; s < SL; ++s) {
      if constexpr (INTER && V > 1) {
        load<T, 2 * V>(slot[s], e[s]);
      } else {
        load<T, V>(slot[s], e[s]);
        load<T, V>(slot[s] + hi[s], e[s] + V);
      }
    }
  }
  __device__ __forceinline__ void put(T* const (&slot)[SL], const int (&hi)[SL], const bool (&valid)[SL]) const {
#pragma unroll
    for (int s = 0; s < SL; ++s) {
      if (!valid[s]) continue;
      if constexpr (INTER && V > 1) {
        store<T, 2 * V>(slot[s], e[s]);
      } else {
        store<T, V>(slot[s], e[s]);
        store<T, V>(slot[s] + hi[s], e[s] + V);
      }
    }
  }
  // pair j = (first, second); two pairs a float2.  bf16 goes by words of two elements: a shift or a mask each way out, one
  // conversion for both on the way back.
  static constexpr bool kWords = sizeof(T) == 2 && V > 1;
  __device__ __forceinline__ void split(float2 (&a)[V * SL / 2], float2 (&b)[V * SL / 2]) const {
#pragma unroll
    for (int j = 0; j < V * SL; ++j) {
      const int s = j / V, i = j % V;
      float x, y;
      if constexpr (kWords) {
        const uint32_t* const w = reinterpret_cast<const uint32_t*>(e[s]);
        x = INTER ? bf16_lo(w[i]) : i & 1 ? bf16_hi(w[i / 2]) : bf16_lo(w[i / 2]);
        y = INTER ? bf16_hi(w[i]) : i & 1 ? bf16_hi(w[(V + i) / 2]) : bf16_lo(w[(V + i) / 2]);
      } else {
        x = to_f32<T>(e[s][INTER ? 2 * i : i]);
        y = to_f32<T>(e[s][INTER ? 2 * i + 1 : V + i]);
      }
      (j & 1 ? a[j / 2].y : a[j / 2].x) = x;
      (j & 1 ? b[j / 2].y : b[j / 2].x) = y;
    }
  }
  __device__ __forceinline__ void join(const float2 (&a)[V * SL / 2], const float2 (&b)[V * SL / 2]) {
    if constexpr (kWords) {
#pragma unroll
      for (int j = 0; j < V * SL; j += 2) {
        const int s = j / V, i = j % V;
        uint32_t* const w = reinterpret_cast<uint32_t*>(e[s]);
        const float2 p = a[j / 2], q = b[j / 2];
        w[INTER ? i : i / 2] = INTER ? pack(p.x, q.x) : pack(p.x, p.y);
        w[INTER ? i + 1 : (V + i) / 2] = INTER ? pack(p.y, q.y) : pack(q.x, q.y);
      }
    } else {
#pragma unroll
      for (int j = 0; j < V * SL; ++j) {
        const int s = j / V, i = j % V;
        e[s][INTER ? 2 * i : i] = from_f32<T>(j & 1 ? a[j / 2].y : a[j / 2].x);
        e[s][INTER ? 2 * i + 1 : V + i] = from_f32<T>(j & 1 ? b[j / 2].y : b[j / 2].x);
      }
    }
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __nv_bfloat162 t = __floats2bfloat162_rn(lo, hi);
    return reinterpret_cast<const uint32_t&>(t);
  }
};

// Sum over the adjacent lanes of a head, on each of them, always in the same order.  LC: their number where
// it is a power of two known to the compiler, else 0.
template <int LC>
__device__ __forceinline__ float head_sum(float v, int lanes, int in_head, int first) {
  if constexpr (LC > 0) {
#pragma unroll
    for (int o = LC >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
  } else {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      if (o >= lanes) break;
      const float t = __shfl_down_sync(kFull, v, o);
      if (in_head + o < lanes) v += t;
    }
    return __shfl_sync(kFull, v, first);
  }
}

// Copies of a lane's own bytes to its own place in shared memory: the loads ahead, without registers to hold them.
template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void* from) {
  if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copy_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

// Stages of a warp's ring and units (steps of 32 / lanes heads) of a stage, where a lane's unit is whole 16- or two
// 8-byte words (V = 4).  Stages 6: as fast; one unit a stage and 8 stages: forward 671 us instead of 598.
constexpr int kStages = 4;
constexpr int units_of(bool bwd, int element) { return bwd && element == 4 ? 1 : 2; }

enum Mode : int { kRotate = 0, kForward = 1, kBackward = 2 };

template <typename T, int V, int SL, bool INTER, int MODE, int LC>
__global__ void __launch_bounds__(256, V == 4 ? (MODE == kBackward ? 2 : 3) : 1) rotary_kernel(const __grid_constant__ Params P) {
  constexpr int NP = V * SL, N2 = NP / 2;         // pairs of a lane
  constexpr int UU = units_of(MODE == kBackward, sizeof(T)), OPS = MODE == kBackward ? 2 : 1;
  // pieces of a lane's unit: 16 bytes of adjacent pairs, or the two halves of split ones
  constexpr int kPiece = INTER ? 16 : V * static_cast<int>(sizeof(T)), kPieces = 2 * V * static_cast<int>(sizeof(T)) / kPiece;
  extern __shared__ __align__(16) uint8_t ring[];  // [warps][stages][units][operands][pieces][32 lanes]
  constexpr bool NORM = MODE != kRotate, BWD = MODE == kBackward;
  using R = Raw<T, V, SL, INTER>;
  const int lane = threadIdx.x & 31;
  const int L = LC > 0 ? LC : P.lanes;
  const int seg = lane / L, in_head = lane - seg * L;
  const int per_warp = 32 / L;  // heads of one step
  const int nslots = P.d / (2 * V), turning = P.R / (2 * V);
  const bool mine = seg < per_warp;
  const uint32_t ring_at = static_cast<uint32_t>(__cvta_generic_to_shared(ring));
  const uint32_t mine_at = ring_at + (threadIdx.x >> 5) * (kStages * UU * OPS * kPieces * 32 * kPiece) + lane * kPiece;
  const int first = min(seg, per_warp - 1) * L;
  // queries or keys
  const int o = static_cast<int>(blockIdx.x) >= P.blocks0 ? 1 : 0;
  const unsigned block = blockIdx.x - (o ? P.blocks0 : 0), nblocks = o ? gridDim.x - P.blocks0 : P.blocks0;
  const int nh = P.heads[o];
  const int units = (nh + per_warp - 1) / per_warp;
  const bool ragged = units * per_warp != nh;

  int lo[SL], hi[SL];  // the slot's first channel, and from there to its second half
  bool valid[SL];
#pragma unroll
  for (int s = 0; s < SL; ++s) {
    const int slot = in_head + s * L;
    valid[s] = mine && slot < nslots;
    const bool turns = valid[s] && slot < turning;
    lo[s] = !valid[s] ? 0 : !INTER && turns ? slot * V : slot * 2 * V;
    hi[s] = !INTER && turns ? P.R / 2 : V;
  }
  // channel of a pair's first (k = 0) or second (k = 1) element
  auto channel = [&](int j, int k) {
    const int s = j / V, i = j % V;
    return INTER ? lo[s] + 2 * i + k : lo[s] + (k ? hi[s] : 0) + i;
  };
  float2 wa[NORM ? N2 : 1], wb[NORM ? N2 : 1];  // weights of the pairs' first and second channels
  float2 ga[BWD ? N2 : 1], gb[BWD ? N2 : 1];    // sums of their gradients
  if (NORM) {
    const void* const weight = P.weight[o];
#pragma unroll
    for (int j = 0; j < NP; ++j) {
      float w[2] = {1.f, 1.f};
      if (weight) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
          w[k] = P.w_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(weight)[channel(j, k)]) : static_cast<const float*>(weight)[channel(j, k)];
      }
      (j & 1 ? wa[j / 2].y : wa[j / 2].x) = w[0];
      (j & 1 ? wb[j / 2].y : wb[j / 2].x) = w[1];
    }
    if (BWD) {
#pragma unroll
      for (int j = 0; j < N2; ++j) ga[j] = gb[j] = both(0.f);
    }
  }
  // where the lane's pairs lie in the table: axis and entry of position 0
  const int start1 = P.npair[0], start2 = P.npair[0] + P.npair[1];
  const int off1 = P.size[0] * P.npair[0], off2 = off1 + P.size[1] * P.npair[1];
  int entry[NP];
  unsigned axes = 0;  // 2 bits a pair: the axis, 3 where the pair does not turn
#pragma unroll
  for (int j = 0; j < NP; ++j) {
    const int slot = in_head + j / V * L, p = slot * V + j % V;
    const bool turns = valid[j / V] && slot < turning;
    const int a = p < start1 ? 0 : p < start2 ? 1 : 2;
    entry[j] = a == 0 ? p : a == 1 ? off1 + p - start1 : off2 + p - start2;
    axes |= (turns ? a : 3u) << (2 * j);
  }
  const int chunk = (units + P.splits - 1) / P.splits;
  const long long nitems = (P.rows + P.group - 1) / P.group * P.splits;
  const long long step = static_cast<long long>(nblocks) * (blockDim.x >> 5);
  for (long long item = static_cast<long long>(block) * (blockDim.x >> 5) + (threadIdx.x >> 5); item < nitems; item += step) {
    const long long grp = P.splits == 1 ? item : item / P.splits;
    const int b0 = P.splits == 1 ? 0 : static_cast<int>(item - grp * P.splits) * chunk;
    const int b1 = min(units, b0 + chunk);
    if (b0 >= b1) continue;
    const long long row0 = grp * P.group;
    const long long row1 = min(P.rows, row0 + P.group);
    long long n = 0;  // token of its sample
    int pos[3] = {0, 0, 0};
    if (turning > 0 && !P.index) {
      int f, rest;
      if (P.tokens <= 0x7fffffffLL && P.rows <= 0x7fffffffLL) {
        const unsigned t = static_cast<unsigned>(row0) % static_cast<unsigned>(P.tokens);
        n = t;
        f = t / static_cast<unsigned>(P.HW);
        rest = t - f * P.HW;
      } else {
        n = row0 % P.tokens;
        f = static_cast<int>(n / P.HW);
        rest = static_cast<int>(n - static_cast<long long>(f) * P.HW);
      }
      pos[0] = P.frame0 + f;
      pos[1] = rest / P.W;
      pos[2] = rest - pos[1] * P.W;
    }
    // The item's units in their order, a few stages ahead.  A unit's place in its row is min(unit's first, last head's)
    // + lo, kept up from unit to unit.
    const int step_at = per_warp * P.d, last_at = (nh - 1) * P.d, first_at = (b0 * per_warp + seg) * P.d;
    long long ahead = row0;
    int ahead_unit = b0, ahead_at = first_at, slot = 0;
    const T* src[OPS];
    src[0] = static_cast<const T*>(P.x[o]) + row0 * P.x_ld[o] + lo[0];
    if (BWD) src[OPS - 1] = static_cast<const T*>(P.dy[o]) + row0 * P.dy_ld[o] + lo[0];
    auto issue = [&](int to) {
      if (ahead < row1) {
#pragma unroll
        for (int u = 0; u < UU; ++u) {  // units beyond b1 (another warp's, or the last head again) only fill the stage
          const int at = min(ahead_at, last_at);
          ahead_at += step_at;
#pragma unroll
          for (int k = 0; k < OPS; ++k)
#pragma unroll
            for (int i = 0; i < kPieces; ++i)
              copy_async<kPiece>(mine_at + (((to * UU + u) * OPS + k) * kPieces + i) * 32 * kPiece, src[k] + (at + i * (INTER ? kPiece / static_cast<int>(sizeof(T)) : hi[0])));
        }
        ahead_unit += UU;
        if (ahead_unit >= b1) {
          ahead_unit = b0;
          ahead_at = first_at;
          ++ahead;
#pragma unroll
          for (int k = 0; k < OPS; ++k) src[k] += k ? P.dy_ld[o] : P.x_ld[o];
        }
      }
      copy_commit();
    };
    auto take = [&](int from, int u, int k, R& r) {
#pragma unroll
      for (int i = 0; i < kPieces; ++i)
        load<T, kPiece / static_cast<int>(sizeof(T))>(
            reinterpret_cast<const T*>(ring + (mine_at - ring_at) + (((from * UU + u) * OPS + k) * kPieces + i) * 32 * kPiece), &r.e[0][i * (kPiece / static_cast<int>(sizeof(T)))]);
    };
    if constexpr (V == 4) {
#pragma unroll
      for (int i = 0; i < kStages - 1; ++i) issue(i);
    }
    for (long long row = row0; row < row1; ++row) {
      float2 cs[N2], sn[N2];
#pragma unroll
      for (int j = 0; j < N2; ++j) { cs[j] = both(1.f); sn[j] = both(0.f); }
      if (turning > 0) {
        if (P.index) {
          const int* ix = P.index + (row % P.index_rows) * 3;
          bool out = false;
#pragma unroll
          for (int a = 0; a < 3; ++a) {
            pos[a] = ix[a];
            if (P.npair[a] > 0 && static_cast<unsigned>(pos[a]) >= static_cast<unsigned>(P.size[a])) { pos[a] = -1; out = true; }
          }
          if (out && lane == 0 && P.status) atomicOr(P.status, MSL_STATUS_ROTARY_INDEX);
        }
        if (P.table_vec) {  // every axis has whole slots, on 16-byte boundaries
          const int a = axes & 3u;
          const int at = a == 0 ? pos[0] : a == 1 ? pos[1] : pos[2];
          if (a < 3 && at >= 0) {
            const float4* const c = reinterpret_cast<const float4*>(P.table + entry[0] + at * (a == 0 ? P.npair[0] : a == 1 ? P.npair[1] : P.npair[2]));
#pragma unroll
            for (int j = 0; j < N2; ++j) {
              const float4 v = __ldg(c + j);
              cs[j] = make_float2(v.x, v.z);
              sn[j] = make_float2(v.y, v.w);
            }
          }
        } else {
#pragma unroll
          for (int j = 0; j < NP; ++j) {
            const int a = (axes >> (2 * j)) & 3u;
            const int at = a == 0 ? pos[0] : a == 1 ? pos[1] : pos[2];
            if (a < 3 && at >= 0) {
              const float2 c = __ldg(P.table + entry[j] + at * (a == 0 ? P.npair[0] : a == 1 ? P.npair[1] : P.npair[2]));
              (j & 1 ? cs[j / 2].y : cs[j / 2].x) = c.x;
              (j & 1 ? sn[j / 2].y : sn[j / 2].x) = c.y;
            }
          }
        }
        if (!P.index) {  // the next token's place
          if (++pos[2] == P.W) {
            pos[2] = 0;
            if (++pos[1] == P.size[1]) { pos[1] = 0; ++pos[0]; }
          }
          if (++n == P.tokens) { n = 0; pos[0] = P.frame0; pos[1] = pos[2] = 0; }
        }
      }
      // forward: y_a = r (x_a A + x_b B), y_b = r (x_b C + x_a D), the weights inside; a rotation alone: r = 1.
      // backward: n_a = dy_a A + dy_b B, n_b = dy_b A + dy_a D, the inverse rotation
      float2 A[N2], B[N2], C[N2], D[N2];
#pragma unroll
      for (int j = 0; j < N2; ++j) {
        const float2 s = P.sign < 0.f ? neg(sn[j]) : sn[j];
        A[j] = MODE == kForward ? mul2(cs[j], wa[j]) : cs[j];
        B[j] = neg(MODE == kForward ? mul2(s, wb[j]) : s);
        C[j] = MODE == kForward ? mul2(cs[j], wb[j]) : cs[j];
        D[j] = MODE == kForward ? mul2(s, wa[j]) : s;
      }
      T* const yr = static_cast<T*>(P.y[o]) + row * P.y_ld[o];
      auto finish = [&](R& raw, const R& rdy, int b) {
        const int at = first_at + (b - b0) * step_at;
        const bool on = at <= last_at;
        float2 xa[N2], xb[N2];
        raw.split(xa, xb);
        float r = 1.f;
        if (NORM) {
          float2 ss = both(0.f);
          if (SL > 1) {  // slots beyond the head were loaded from its first
#pragma unroll
            for (int j = 0; j < NP; ++j)
              if (!valid[j / V]) {
                (j & 1 ? xa[j / 2].y : xa[j / 2].x) = 0.f;
                (j & 1 ? xb[j / 2].y : xb[j / 2].x) = 0.f;
              }
          }
#pragma unroll
          for (int j = 0; j < N2; ++j) ss = fma2(xb[j], xb[j], fma2(xa[j], xa[j], ss));
          r = rsqrtf(fmaf(head_sum<LC>(ss.x + ss.y, L, in_head, first), P.inv_d, P.eps));
        }
        if (!BWD) {
#pragma unroll
          for (int j = 0; j < N2; ++j) {
            float2 ya = fma2(xb[j], B[j], mul2(xa[j], A[j])), yb = fma2(xa[j], D[j], mul2(xb[j], C[j]));
            if (NORM) { ya = mul2(ya, both(r)); yb = mul2(yb, both(r)); }
            xa[j] = ya;
            xb[j] = yb;
          }
        } else {
          float2 da[N2], db[N2], dot = both(0.f);
          const float2 rr = both(on ? r : 0.f);  // a head loaded twice counts once
          rdy.split(da, db);
          if (ragged && b == units - 1) {  // what a lane without a head has loaded may be another's result by now (dx over dy)
#pragma unroll
            for (int j = 0; j < N2; ++j)
              if (!on) xa[j] = xb[j] = da[j] = db[j] = both(0.f);
          }
#pragma unroll
          for (int j = 0; j < N2; ++j) {
            const float2 na = fma2(db[j], B[j], mul2(da[j], A[j])), nb = fma2(da[j], D[j], mul2(db[j], A[j]));
            ga[j] = fma2(na, mul2(xa[j], rr), ga[j]);
            gb[j] = fma2(nb, mul2(xb[j], rr), gb[j]);
            da[j] = mul2(na, wa[j]);
            db[j] = mul2(nb, wb[j]);
            dot = fma2(db[j], xb[j], fma2(da[j], xa[j], dot));
          }
          const float m = -head_sum<LC>(dot.x + dot.y, L, in_head, first) * P.inv_d * r * r;
#pragma unroll
          for (int j = 0; j < N2; ++j) {
            xa[j] = mul2(fma2(xa[j], both(m), da[j]), both(r));
            xb[j] = mul2(fma2(xb[j], both(m), db[j]), both(r));
          }
        }
        raw.join(xa, xb);
        if (on) {
          T* to[SL];
#pragma unroll
          for (int s = 0; s < SL; ++s) to[s] = yr + (at + lo[s]);
          raw.put(to, hi, valid);
        }
      };
      if constexpr (V == 4) {
        for (int b = b0; b < b1; b += UU) {
          copy_wait<kStages - 2>();
          issue(slot == 0 ? kStages - 1 : slot - 1);  // the stage that was used last
          R raw[UU], rdy[UU];
#pragma unroll
          for (int u = 0; u < UU; ++u) {
            take(slot, u, 0, raw[u]);
            if (BWD) take(slot, u, 1, rdy[u]);
          }
          slot = slot == kStages - 1 ? 0 : slot + 1;
#pragma unroll
          for (int u = 0; u < UU; ++u)
            if (u == 0 || b + u < b1) finish(raw[u], rdy[u], b + u);
        }
      } else {
        const T* const xr = static_cast<const T*>(P.x[o]) + row * P.x_ld[o];
        const T* const gr = BWD ? static_cast<const T*>(P.dy[o]) + row * P.dy_ld[o] : nullptr;
        for (int b = b0; b < b1; ++b) {
          R raw, rdy;
          const int at = min(first_at + (b - b0) * step_at, last_at);
          const T* from[SL];
#pragma unroll
          for (int s = 0; s < SL; ++s) from[s] = xr + at + lo[s];
          raw.get(from, hi);
          if (BWD) {
#pragma unroll
            for (int s = 0; s < SL; ++s) from[s] = gr + at + lo[s];
            rdy.get(from, hi);
          }
          finish(raw, rdy, b);
        }
      }
    }
  }

  if (BWD && P.partial) {
    // the block's sums: every warp and head position of a warp writes its channels, then one thread per
    // channel adds them in order
    float* const sums = reinterpret_cast<float*>(ring);  // [warps * per_warp][d]
    const int nw = blockDim.x >> 5, warp = threadIdx.x >> 5;
    __syncthreads();
    if (mine) {
      float* const to = sums + static_cast<size_t>(warp * per_warp + seg) * P.d;
#pragma unroll
      for (int j = 0; j < NP; ++j) {
        if (!valid[j / V]) continue;
        to[channel(j, 0)] = j & 1 ? ga[BWD ? j / 2 : 0].y : ga[BWD ? j / 2 : 0].x;
        to[channel(j, 1)] = j & 1 ? gb[BWD ? j / 2 : 0].y : gb[BWD ? j / 2 : 0].x;
      }
    }
    __syncthreads();
    for (int c = threadIdx.x; c < P.d; c += blockDim.x) {
      float t = 0.f;
      for (int k = 0; k < nw * per_warp; ++k) t += sums[static_cast<size_t>(k) * P.d + c];
      P.partial[static_cast<size_t>(blockIdx.x) * P.d + c] = t;
    }
  }
}

// dg[c] = sum over the queries' or the keys' blocks of partial[block][c]: 32 columns a block, 32 threads a
// column, joined in order
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int blocks0, int blocks, int d,
                                                           void* dq_weight, void* dk_weight, int bf16) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), k0 = threadIdx.x >> 5;
  const int first = blockIdx.y ? blocks0 : 0, last = blockIdx.y ? blocks : blocks0;
  float t = 0.f;
  if (c < d)
    for (int b = first + k0; b < last; b += 32) t += partial[static_cast<size_t>(b) * d + c];
  part[k0][threadIdx.x & 31] = t;
  __syncthreads();
  void* const out = blockIdx.y ? dk_weight : dq_weight;
  if (k0 == 0 && c < d && out) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += part[k][threadIdx.x];
    if (bf16) static_cast<__nv_bfloat16*>(out)[c] = __float2bfloat16_rn(t);
    else static_cast<float*>(out)[c] = t;
  }
}

// ------------------------------------------------------------------------------------------ host

constexpr int kWarps = 8;
constexpr int kBwdBlocksPerSm = 4;

int fill(const msl_rotary_geometry* g, Params& P) {
  if (!g) return failf(MSL_ERR_INVALID, "geometry is NULL");
  if (g->rows < 0 || g->tokens < 1 || g->frames < 1 || g->height < 1 || g->width < 1)
    return failf(MSL_ERR_INVALID, "rows must be >= 0; tokens, frames, height and width >= 1");
  if (g->head_dim < 2 || g->head_dim % 2) return failf(MSL_ERR_INVALID, "head_dim %d must be even", g->head_dim);
  if (g->head_dim > 256) return failf(MSL_ERR_UNSUPPORTED, "head_dim %d is over 256", g->head_dim);
  if (g->axis_t < 0 || g->axis_h < 0 || g->axis_w < 0 || g->axis_t % 2 || g->axis_h % 2 || g->axis_w % 2)
    return failf(MSL_ERR_INVALID, "axes (%d, %d, %d) must be even", g->axis_t, g->axis_h, g->axis_w);
  const long long R = static_cast<long long>(g->axis_t) + g->axis_h + g->axis_w;
  if (R > g->head_dim)
    return failf(MSL_ERR_INVALID, "axes (%d, %d, %d) take more than head_dim %d channels", g->axis_t, g->axis_h, g->axis_w, g->head_dim);
  if (g->dtype != MSL_DTYPE_F32 && g->dtype != MSL_DTYPE_BF16) return failf(MSL_ERR_INVALID, "unknown dtype %d", g->dtype);
  if (g->frame0 < 0) return failf(MSL_ERR_INVALID, "frame0 must be >= 0");
  if (static_cast<long long>(g->height) * g->width > 0x7fffffffLL) return failf(MSL_ERR_UNSUPPORTED, "height * width is over 2^31");
  P = Params{};
  P.rows = g->rows;
  P.tokens = g->tokens;
  P.size[0] = g->frames; P.size[1] = g->height; P.size[2] = g->width;
  P.npair[0] = g->axis_t / 2; P.npair[1] = g->axis_h / 2; P.npair[2] = g->axis_w / 2;
  P.frame0 = g->frame0;
  P.HW = g->height * g->width;
  P.W = g->width;
  P.d = g->head_dim;
  P.R = static_cast<int>(R);
  P.inv_d = 1.f / static_cast<float>(g->head_dim);
  P.sign = 1.f;
  return MSL_OK;
}

// Table and index of a rotating call.
int fill_positions(const msl_rotary_geometry* g, Params& P, const float* table, const int32_t* index, int64_t index_rows,
                   uint32_t* status) {
  if (!table || P.R == 0) {
    P.R = 0;
    P.npair[0] = P.npair[1] = P.npair[2] = 0;
    return MSL_OK;
  }
  if (!multiple_of(table, 8)) return failf(MSL_ERR_INVALID, "table must be 8-byte aligned");
  if (static_cast<long long>(g->frames) * P.npair[0] + static_cast<long long>(g->height) * P.npair[1] + static_cast<long long>(g->width) * P.npair[2] > (1LL << 30))
    return failf(MSL_ERR_UNSUPPORTED, "the table has over 2^30 entries");
  P.table = reinterpret_cast<const float2*>(table);
  P.index = index;
  P.index_rows = index_rows;
  P.status = status;
  if (g->rows == 0) return MSL_OK;
  if (index) {
    if (index_rows < 1) return failf(MSL_ERR_INVALID, "index needs index_rows >= 1");
  } else {
    if (g->tokens % P.HW) return failf(MSL_ERR_INVALID, "tokens %lld are no whole frames of %d", static_cast<long long>(g->tokens), P.HW);
    if (g->frame0 + g->tokens / P.HW > g->frames)
      return failf(MSL_ERR_INVALID, "frames [%d, %lld) are outside the table's [0, %d)", g->frame0,
                   static_cast<long long>(g->frame0 + g->tokens / P.HW), g->frames);
  }
  return MSL_OK;
}

// The widest slot that head_dim, the turning channels and the alignment of every row operand allow (V = 1 goes
// element by element).  SL (slots of a lane)
// follows from it: V = 4 needs at most 32 lanes for 256 channels, V = 2 two slots, V = 1 four.
int choose_v(const Params& P, bool inter, int dtype, bool bwd, int nops) {
  const int es = dtype == MSL_DTYPE_BF16 ? 2 : 4;
  for (int v = 4; v > 1; v /= 2) {
    if (P.d % (2 * v) || P.R % (2 * v)) continue;
    const int bytes = min((inter ? 2 * v : v) * es, 16);
    bool ok = true;
    for (int o = 0; o < nops; ++o) {
      if (P.heads[o] == 0) continue;
      ok = ok && multiple_of(P.x[o], bytes) && multiple_of(P.y[o], bytes) && P.x_ld[o] * es % bytes == 0 && P.y_ld[o] * es % bytes == 0;
      if (bwd) ok = ok && multiple_of(P.dy[o], bytes) && P.dy_ld[o] * es % bytes == 0;
    }
    if (ok) return v;
  }
  return 1;
}

// Blocks of a backward whose weights' gradients are wanted: each keeps its sums, so at most four a SM, in two rounds (two
// or eight a SM take the same time).  The queries' share goes by the heads.
int bwd_blocks(const msl_rotary_geometry* g, const msl_qk_norm_io* io, int* blocks0) {
  const long long most = static_cast<long long>(sm_count()) * kBwdBlocksPerSm;
  const long long need = (g->rows * io->heads + kWarps - 1) / kWarps, need1 = (g->rows * io->kv_heads + kWarps - 1) / kWarps;
  if (need + need1 <= most) {
    *blocks0 = static_cast<int>(need > 0 ? need : 1);
    return *blocks0 + static_cast<int>(need1);
  }
  long long b0 = io->kv_heads ? most * io->heads / (io->heads + io->kv_heads) : most;
  if (b0 < 1) b0 = 1;
  if (io->kv_heads && b0 == most) b0 = most - 1;
  *blocks0 = static_cast<int>(b0);
  return static_cast<int>(most);
}

template <typename T, int V, int SL, bool INTER, int MODE, int LC>
cudaError_t launch(Params P, cudaStream_t s, int blocks) {
  P.lanes = (P.d / (2 * V) + SL - 1) / SL;
  const int per_warp = 32 / P.lanes;
  const int units0 = (P.heads[0] + per_warp - 1) / per_warp, units1 = (P.heads[1] + per_warp - 1) / per_warp;
  // few tokens: several warps share a token's heads, until every SM has some
  const long long want = static_cast<long long>(sm_count()) * kWarps;
  long long splits = P.rows >= want ? 1 : (want + P.rows - 1) / P.rows;
  if (splits > (units0 > units1 ? units0 : units1)) splits = units0 > units1 ? units0 : units1;
  P.splits = static_cast<int>(splits);
  // Several tokens a warp once every SM has its warps: their loads run ahead over them, their places follow.  Up to 8,
  // and more where the GPU has its blocks four times over all the same (norm and rotation of 262144 x 24 x 64 queries
  // and keys: 8 600 us, 37 582, 148 586; rotation of 131072 x 16 x 72: 8 114 us, 10 115, 37 122).
  const long long resident = 3 * want, tokens = P.rows * (P.heads[1] ? 2 : 1);
  const long long few = (P.rows + resident - 1) / resident, four = (tokens + 4 * resident - 1) / (4 * resident);
  P.group = static_cast<int>(splits > 1 ? 1 : few <= 8 ? few : four > 8 ? four : 8);
  P.table_vec = SL == 1 && V % 2 == 0 && multiple_of(P.table, 16);
  for (int a = 0; a < 3; ++a) P.table_vec = P.table_vec && P.npair[a] % V == 0;
  if (blocks == 0) {
    long long each = ((P.rows + P.group - 1) / P.group * splits + kWarps - 1) / kWarps;
    if (each > 0x3fffffffLL) each = 0x3fffffffLL;  // the kernel strides over the rest
    P.blocks0 = static_cast<int>(each);
    blocks = static_cast<int>(P.heads[1] ? 2 * each : each);
  }
  constexpr size_t kRing = V == 4 ? kWarps * kStages * units_of(MODE == kBackward, sizeof(T)) * (MODE == kBackward ? 2 : 1) * 32 * 2 * V * sizeof(T) : 0;
  const size_t sums = MODE == kBackward && P.partial ? sizeof(float) * kWarps * per_warp * P.d : 0;
  const size_t smem = sums > kRing ? sums : kRing;
  if (smem > 48 * 1024) {
    const cudaError_t e = cudaFuncSetAttribute(rotary_kernel<T, V, SL, INTER, MODE, LC>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  rotary_kernel<T, V, SL, INTER, MODE, LC><<<static_cast<unsigned>(blocks), kWarps * 32, smem, s>>>(P);
  return cudaGetLastError();
}

template <typename T, bool INTER, int MODE>
cudaError_t by_v(const Params& P, int v, cudaStream_t s, int blocks) {
  switch (v) {
    case 4:
      // A head's sums: where its lanes are a power of two, shuffles of a number that the compiler knows, else a loop with
      // a broadcast.  Norm and rotation of 131072 tokens of about 1536 channels in bf16, forward and backward: 4 lanes
      // (head 32) 261 and 385 us, by the loop 268 and 429; 8 lanes 260 and 389, 277 and 459; 16 lanes 258 and 403, 290 and
      // 495; 32 lanes 275 and 386, 302 and 527.  float32 within 6% either way.
      if (MODE != kRotate) {
        switch (P.d / 8) {
          case 4: return launch<T, 4, 1, INTER, MODE, 4>(P, s, blocks);
          case 8: return launch<T, 4, 1, INTER, MODE, 8>(P, s, blocks);
          case 16: return launch<T, 4, 1, INTER, MODE, 16>(P, s, blocks);
          case 32: return launch<T, 4, 1, INTER, MODE, 32>(P, s, blocks);
          default: break;  // any other number; 1 and 2 lanes (heads of 8 and 16) are no or one step of the loop
        }
      }
      return launch<T, 4, 1, INTER, MODE, 0>(P, s, blocks);
    case 2: return launch<T, 2, 2, INTER, MODE, 0>(P, s, blocks);
    default: return launch<T, 1, 4, INTER, MODE, 0>(P, s, blocks);
  }
}

template <int MODE>
cudaError_t dispatch(const Params& P, bool inter, int dtype, cudaStream_t s, int blocks) {
  const int v = choose_v(P, inter, dtype, MODE == kBackward, 2);
  if (dtype == MSL_DTYPE_BF16)
    return inter ? by_v<__nv_bfloat16, true, MODE>(P, v, s, blocks) : by_v<__nv_bfloat16, false, MODE>(P, v, s, blocks);
  return inter ? by_v<float, true, MODE>(P, v, s, blocks) : by_v<float, false, MODE>(P, v, s, blocks);
}

int fill_norm(const msl_rotary_geometry* g, const msl_qk_norm_io* io, Params& P) {
  int rc = fill(g, P);
  if (rc) return rc;
  if (!io) return failf(MSL_ERR_INVALID, "io is NULL");
  if (io->heads < 1 || io->kv_heads < 0) return failf(MSL_ERR_INVALID, "heads must be >= 1 and kv_heads >= 0");
  if (io->weight_dtype != MSL_DTYPE_F32 && io->weight_dtype != MSL_DTYPE_BF16)
    return failf(MSL_ERR_INVALID, "unknown weight_dtype %d", io->weight_dtype);
  if (!(io->eps >= 0.f)) return failf(MSL_ERR_INVALID, "eps must be >= 0");
  P.heads[0] = io->heads;
  P.heads[1] = io->kv_heads;
  P.eps = io->eps;
  P.x[0] = io->q; P.x_ld[0] = io->q_ld;
  P.x[1] = io->k; P.x_ld[1] = io->k_ld;
  P.weight[0] = io->q_weight;
  P.weight[1] = io->k_weight;
  P.w_bf16 = io->weight_dtype == MSL_DTYPE_BF16;
  return fill_positions(g, P, io->table, io->index, io->index_rows, io->status);
}

int check_rows(const char* what, const void* p, long long ld, long long heads, int d, int dtype) {
  if (!p) return failf(MSL_ERR_INVALID, "%s is required", what);
  if (heads > (1 << 20)) return failf(MSL_ERR_UNSUPPORTED, "%s: over 2^20 heads", what);
  if (!multiple_of(p, dtype == MSL_DTYPE_BF16 ? 2 : 4)) return failf(MSL_ERR_INVALID, "%s is not aligned to its elements", what);
  if (ld < heads * d) return failf(MSL_ERR_INVALID, "%s: row stride %lld is under heads * head_dim = %lld", what, ld, heads * d);
  return MSL_OK;
}

}  // namespace rot
}  // namespace msl

using namespace msl;

extern "C" {

int msl_rope3d(const msl_rotary_geometry* geom, int32_t heads, const void* x, int64_t x_ld, const float* table,
               const int32_t* index, int64_t index_rows, int32_t inverse, void* y, int64_t y_ld, uint32_t* status,
               void* stream) {
  rot::Params P;
  int rc = rot::fill(geom, P);
  if (rc) return rc;
  if (heads < 1) return failf(MSL_ERR_INVALID, "heads must be >= 1");
  if (!table) return failf(MSL_ERR_INVALID, "table is required");
  rc = rot::fill_positions(geom, P, table, index, index_rows, status);
  if (rc) return rc;
  if (geom->rows == 0) return MSL_OK;
  rc = rot::check_rows("x", x, x_ld, heads, P.d, geom->dtype);
  if (!rc) rc = rot::check_rows("y", y, y_ld, heads, P.d, geom->dtype);
  if (rc) return rc;
  P.heads[0] = heads;
  P.x[0] = x; P.x_ld[0] = x_ld;
  P.y[0] = y; P.y_ld[0] = y_ld;
  P.sign = inverse ? -1.f : 1.f;
  const cudaError_t e = rot::dispatch<rot::kRotate>(P, geom->interleaved != 0, geom->dtype, static_cast<cudaStream_t>(stream), 0);
  if (e != cudaSuccess) return cuda_failf(e, "rotary_kernel launch");
  count_launches(1);
  return MSL_OK;
}

int msl_qk_norm_rope_fwd(const msl_rotary_geometry* geom, const msl_qk_norm_io* io, void* stream) {
  rot::Params P;
  int rc = rot::fill_norm(geom, io, P);
  if (rc) return rc;
  if (geom->rows == 0) return MSL_OK;
  rc = rot::check_rows("q", io->q, io->q_ld, io->heads, P.d, geom->dtype);
  if (!rc) rc = rot::check_rows("q_out", io->q_out, io->q_out_ld, io->heads, P.d, geom->dtype);
  if (!rc && io->kv_heads) rc = rot::check_rows("k", io->k, io->k_ld, io->kv_heads, P.d, geom->dtype);
  if (!rc && io->kv_heads) rc = rot::check_rows("k_out", io->k_out, io->k_out_ld, io->kv_heads, P.d, geom->dtype);
  if (rc) return rc;
  P.y[0] = io->q_out; P.y_ld[0] = io->q_out_ld;
  P.y[1] = io->k_out; P.y_ld[1] = io->k_out_ld;
  const cudaError_t e = rot::dispatch<rot::kForward>(P, geom->interleaved != 0, geom->dtype, static_cast<cudaStream_t>(stream), 0);
  if (e != cudaSuccess) return cuda_failf(e, "rotary_kernel launch");
  count_launches(1);
  return MSL_OK;
}

size_t msl_qk_norm_rope_bwd_workspace_bytes(const msl_rotary_geometry* geom, const msl_qk_norm_io* io) {
  rot::Params P;
  if (rot::fill_norm(geom, io, P)) return 0;
  if (!io->dq_weight && !io->dk_weight) return 0;
  int blocks0 = 0;
  return sizeof(float) * P.d * rot::bwd_blocks(geom, io, &blocks0);
}

int msl_qk_norm_rope_bwd(const msl_rotary_geometry* geom, const msl_qk_norm_io* io, void* workspace,
                         size_t workspace_bytes, void* stream) {
  rot::Params P;
  int rc = rot::fill_norm(geom, io, P);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool dw = io->dq_weight || io->dk_weight;
  const size_t es = io->weight_dtype == MSL_DTYPE_BF16 ? 2 : 4;
  if (geom->rows == 0) {
    cudaError_t e = cudaSuccess;
    if (io->dq_weight) e = cudaMemsetAsync(io->dq_weight, 0, es * P.d, s);
    if (e == cudaSuccess && io->dk_weight) e = cudaMemsetAsync(io->dk_weight, 0, es * P.d, s);
    return e == cudaSuccess ? MSL_OK : cuda_failf(e, "clearing the weights' gradients");
  }
  rc = rot::check_rows("q", io->q, io->q_ld, io->heads, P.d, geom->dtype);
  if (!rc) rc = rot::check_rows("dq_out", io->dq_out, io->dq_out_ld, io->heads, P.d, geom->dtype);
  if (!rc) rc = rot::check_rows("dq", io->dq, io->dq_ld, io->heads, P.d, geom->dtype);
  if (!rc && io->kv_heads) {
    rc = rot::check_rows("k", io->k, io->k_ld, io->kv_heads, P.d, geom->dtype);
    if (!rc) rc = rot::check_rows("dk_out", io->dk_out, io->dk_out_ld, io->kv_heads, P.d, geom->dtype);
    if (!rc) rc = rot::check_rows("dk", io->dk, io->dk_ld, io->kv_heads, P.d, geom->dtype);
  }
  if (rc) return rc;
  P.dy[0] = io->dq_out; P.dy_ld[0] = io->dq_out_ld;
  P.dy[1] = io->dk_out; P.dy_ld[1] = io->dk_out_ld;
  P.y[0] = io->dq; P.y_ld[0] = io->dq_ld;
  P.y[1] = io->dk; P.y_ld[1] = io->dk_ld;
  P.sign = -1.f;
  int blocks0 = 0;
  const int blocks = rot::bwd_blocks(geom, io, &blocks0);
  if (dw) {
    P.blocks0 = blocks0;
    const size_t need = sizeof(float) * P.d * blocks;
    if (!workspace || workspace_bytes < need)
      return failf(MSL_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : 0);
    if (!multiple_of(workspace, 4)) return failf(MSL_ERR_INVALID, "workspace must be 4-byte aligned");
    P.partial = static_cast<float*>(workspace);
  }
  cudaError_t e = rot::dispatch<rot::kBackward>(P, geom->interleaved != 0, geom->dtype, s, dw ? blocks : 0);
  if (e != cudaSuccess) return cuda_failf(e, "rotary_kernel launch");
  if (dw) {
    rot::weight_grad_kernel<<<dim3((P.d + 31) / 32, io->kv_heads ? 2 : 1), 1024, 0, s>>>(P.partial, blocks0, blocks, P.d, io->dq_weight, io->dk_weight,
                                                                                        io->weight_dtype == MSL_DTYPE_BF16);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_failf(e, "weight_grad_kernel launch");
  }
  count_launches(dw ? 2 : 1);
  return MSL_OK;
}

}  // extern "C"
