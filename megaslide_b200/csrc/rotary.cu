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
// Layout: a warp takes one token and goes through its heads, first the queries', then the keys'.  A head
// is cut into slots of 2V channels, V pairs; a lane keeps one slot (SL of them where V is small) for the
// whole call, so the cosines and sines of a token are loaded once and serve all its heads, and the
// gradients of the weights add up in registers.  32 / (lanes of a head) heads go through together, whole
// rows of adjacent 16-byte loads; the sums of a head are shuffles among its lanes.

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
  float* partial;  // [blocks][2][d] sums of the weights' gradients
  int heads[2];
  int w_bf16;
  const float2* table;
  const int* index;
  long long index_rows;
  uint32_t* status;
  long long rows, tokens;
  int splits;  // warps that share a token's heads
  int size[3], npair[3];
  int frame0, HW, W;
  int d, R;
  int lanes;  // of a head
  float eps, inv_d, sign;
};

template <int BYTES>
struct Word;
template <> struct Word<2> { using type = uint16_t; };
template <> struct Word<4> { using type = uint32_t; };
template <> struct Word<8> { using type = uint2; };
template <> struct Word<16> { using type = uint4; };

// N elements at p, aligned to their size or 16 bytes, whichever is less
template <typename T, int N>
__device__ __forceinline__ void load(const T* p, float* o) {
  constexpr int kBytes = N * static_cast<int>(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16;
  constexpr int kPer = kWord / static_cast<int>(sizeof(T));
  using W = typename Word<kWord>::type;
#pragma unroll
  for (int i = 0; i < N / kPer; ++i) {
    const W w = reinterpret_cast<const W*>(p)[i];
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < kPer; ++j) o[i * kPer + j] = to_f32<T>(e[j]);
  }
}

template <typename T, int N>
__device__ __forceinline__ void store(T* p, const float* o) {
  constexpr int kBytes = N * static_cast<int>(sizeof(T)), kWord = kBytes < 16 ? kBytes : 16;
  constexpr int kPer = kWord / static_cast<int>(sizeof(T));
  using W = typename Word<kWord>::type;
#pragma unroll
  for (int i = 0; i < N / kPer; ++i) {
    W w;
    T* e = reinterpret_cast<T*>(&w);
#pragma unroll
    for (int j = 0; j < kPer; ++j) e[j] = from_f32<T>(o[i * kPer + j]);
    reinterpret_cast<W*>(p)[i] = w;
  }
}

// Sum over the `lanes` adjacent lanes of a head, on each of them, always in the same order.
__device__ __forceinline__ float head_sum(float v, int lanes, int in_head, int first) {
  if ((lanes & (lanes - 1)) == 0) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const float t = __shfl_down_sync(kFull, v, o);
    if (in_head + o < lanes) v += t;
  }
  return __shfl_sync(kFull, v, first);
}

template <typename T, int V, int SL, bool INTER, bool NORM, bool BWD>
__global__ void __launch_bounds__(256) rotary_kernel(const Params P) {
  constexpr int U = BWD ? (SL == 1 && V <= 4 ? 2 : 1) : (SL == 1 ? (V <= 4 ? 4 : 2) : 1);  // heads in flight
  const int lane = threadIdx.x & 31;
  const int L = P.lanes;
  const int seg = lane / L, in_head = lane - seg * L;
  const int per_warp = 32 / L;  // heads of one step
  const int nslots = P.d / (2 * V), turning = P.R / (2 * V);
  const bool mine = seg < per_warp;
  const int first = min(seg, per_warp - 1) * L;

  int lo[SL], hi[SL];
  bool valid[SL];
  float w[2][SL][2 * V];
  float acc[2][SL][2 * V];
#pragma unroll
  for (int s = 0; s < SL; ++s) {
    const int slot = in_head + s * L;
    valid[s] = mine && slot < nslots;
    const bool turns = slot < turning;
    lo[s] = !INTER && turns ? slot * V : slot * 2 * V;
    hi[s] = !INTER && turns ? P.R / 2 + slot * V : slot * 2 * V + V;
    if (NORM) {
#pragma unroll
      for (int o = 0; o < 2; ++o) {
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) {
          const int ch = (i < V ? lo[s] : hi[s] - V) + i;
          w[o][s][i] = 1.f;
          if (P.weight[o] && valid[s])
            w[o][s][i] = P.w_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(P.weight[o])[ch])
                                  : static_cast<const float*>(P.weight[o])[ch];
          acc[o][s][i] = 0.f;
        }
      }
    }
  }
  const int start1 = P.npair[0], start2 = P.npair[0] + P.npair[1];
  const long long off1 = static_cast<long long>(P.size[0]) * P.npair[0];
  const long long off2 = off1 + static_cast<long long>(P.size[1]) * P.npair[1];
  const int units0 = (P.heads[0] + per_warp - 1) / per_warp, units1 = (P.heads[1] + per_warp - 1) / per_warp;
  const int units = units0 + units1;
  const int chunk = (units + P.splits - 1) / P.splits;

  const long long nitems = P.rows * P.splits;
  const long long step = static_cast<long long>(gridDim.x) * (blockDim.x >> 5);
  for (long long item = static_cast<long long>(blockIdx.x) * (blockDim.x >> 5) + (threadIdx.x >> 5); item < nitems;
       item += step) {
    const long long row = P.splits == 1 ? item : item / P.splits;
    const int u0 = P.splits == 1 ? 0 : static_cast<int>(item - row * P.splits) * chunk;
    const int u1 = min(units, u0 + chunk);
    float cs[SL][V], sn[SL][V];
#pragma unroll
    for (int s = 0; s < SL; ++s)
#pragma unroll
      for (int i = 0; i < V; ++i) { cs[s][i] = 1.f; sn[s][i] = 0.f; }
    if (turning > 0) {
      int pos[3];
      bool out = false;
      if (P.index) {
        const int* ix = P.index + (row % P.index_rows) * 3;
#pragma unroll
        for (int a = 0; a < 3; ++a) {
          pos[a] = ix[a];
          if (P.npair[a] > 0 && static_cast<unsigned>(pos[a]) >= static_cast<unsigned>(P.size[a])) { pos[a] = -1; out = true; }
        }
        if (out && lane == 0 && P.status) atomicOr(P.status, MSL_STATUS_ROTARY_INDEX);
      } else {
        const long long n = row % P.tokens;
        const int f = static_cast<int>(n / P.HW), rest = static_cast<int>(n - static_cast<long long>(f) * P.HW);
        pos[0] = P.frame0 + f;
        pos[1] = rest / P.W;
        pos[2] = rest - pos[1] * P.W;
      }
#pragma unroll
      for (int s = 0; s < SL; ++s) {
        const int slot = in_head + s * L;
        if (valid[s] && slot < turning) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const int p = slot * V + i;
            const int a = p < start1 ? 0 : p < start2 ? 1 : 2;
            const int at = a == 0 ? pos[0] : a == 1 ? pos[1] : pos[2];
            const long long base = a == 0 ? p : a == 1 ? off1 + p - start1 : off2 + p - start2;
            if (at >= 0) {
              const float2 c = __ldg(P.table + base + static_cast<long long>(at) * P.npair[a]);
              cs[s][i] = c.x;
              sn[s][i] = c.y * P.sign;
            }
          }
        }
      }
    }
#pragma unroll
    for (int o = 0; o < 2; ++o) {
      const int nh = P.heads[o];
      const int b0 = o == 0 ? u0 : max(u0 - units0, 0), b1 = o == 0 ? min(u1, units0) : u1 - units0;
      const T* const xr = static_cast<const T*>(P.x[o]) + row * P.x_ld[o];
      const T* const gr = BWD ? static_cast<const T*>(P.dy[o]) + row * P.dy_ld[o] : nullptr;
      T* const yr = static_cast<T*>(P.y[o]) + row * P.y_ld[o];
      for (int b = b0; b < b1; b += U) {
        float e[U][SL][2 * V], g[BWD ? U : 1][SL][2 * V];
        bool on[U][SL];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int h = (b + u) * per_warp + seg;
#pragma unroll
          for (int s = 0; s < SL; ++s) {
            on[u][s] = valid[s] && b + u < b1 && h < nh;
            const T* const p = xr + static_cast<long long>(h) * P.d;
            const T* const q = BWD ? gr + static_cast<long long>(h) * P.d : nullptr;
            if (on[u][s]) {
              if (INTER && V > 1) {
                load<T, 2 * V>(p + lo[s], e[u][s]);
                if (BWD) load<T, 2 * V>(q + lo[s], g[u][s]);
              } else {
                load<T, V>(p + lo[s], e[u][s]);
                load<T, V>(p + hi[s], e[u][s] + V);
                if (BWD) {
                  load<T, V>(q + lo[s], g[u][s]);
                  load<T, V>(q + hi[s], g[u][s] + V);
                }
              }
            } else {
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) {
                e[u][s][i] = 0.f;
                if (BWD) g[u][s][i] = 0.f;
              }
            }
          }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float r = 1.f;
          if (NORM) {
            float ss = 0.f;
#pragma unroll
            for (int s = 0; s < SL; ++s)
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) ss = fmaf(e[u][s][i], e[u][s][i], ss);
            r = rsqrtf(fmaf(head_sum(ss, L, in_head, first), P.inv_d, P.eps));
          }
          if (!BWD) {
#pragma unroll
            for (int s = 0; s < SL; ++s) {
              float* const v = e[u][s];
              if (NORM)
#pragma unroll
                for (int i = 0; i < 2 * V; ++i) v[i] = v[i] * r * w[o][s][i];
#pragma unroll
              for (int i = 0; i < V; ++i) {
                float& a = v[INTER ? 2 * i : i];
                float& c = v[INTER ? 2 * i + 1 : V + i];
                const float ya = a * cs[s][i] - c * sn[s][i], yc = c * cs[s][i] + a * sn[s][i];
                a = ya;
                c = yc;
              }
            }
          } else {
            float dot = 0.f;
#pragma unroll
            for (int s = 0; s < SL; ++s) {
              float* const v = g[u][s];
#pragma unroll
              for (int i = 0; i < V; ++i) {
                float& a = v[INTER ? 2 * i : i];
                float& c = v[INTER ? 2 * i + 1 : V + i];
                const float ya = a * cs[s][i] - c * sn[s][i], yc = c * cs[s][i] + a * sn[s][i];
                a = ya;
                c = yc;
              }
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) {
                acc[o][s][i] = fmaf(v[i], e[u][s][i] * r, acc[o][s][i]);
                v[i] *= w[o][s][i];
                dot = fmaf(v[i], e[u][s][i], dot);
              }
            }
            const float m = head_sum(dot, L, in_head, first) * P.inv_d * r * r;
#pragma unroll
            for (int s = 0; s < SL; ++s)
#pragma unroll
              for (int i = 0; i < 2 * V; ++i) e[u][s][i] = r * (g[u][s][i] - e[u][s][i] * m);
          }
          const int h = (b + u) * per_warp + seg;
          T* const q = yr + static_cast<long long>(h) * P.d;
#pragma unroll
          for (int s = 0; s < SL; ++s) {
            if (!on[u][s]) continue;
            if (INTER && V > 1) {
              store<T, 2 * V>(q + lo[s], e[u][s]);
            } else {
              store<T, V>(q + lo[s], e[u][s]);
              store<T, V>(q + hi[s], e[u][s] + V);
            }
          }
        }
      }
    }
  }

  if (BWD && P.partial) {
    // the block's sums: every warp and head position of a warp writes its channels, then one thread per
    // channel adds them in order
    extern __shared__ float sums[];  // [warps * per_warp][d]
    const int nw = blockDim.x >> 5, warp = threadIdx.x >> 5;
    for (int o = 0; o < 2; ++o) {
      __syncthreads();
#pragma unroll
      for (int s = 0; s < SL; ++s) {
        if (!valid[s]) continue;
        float* const to = sums + static_cast<size_t>(warp * per_warp + seg) * P.d;
#pragma unroll
        for (int i = 0; i < 2 * V; ++i) to[(i < V ? lo[s] : hi[s] - V) + i] = o == 0 ? acc[0][s][i] : acc[1][s][i];
      }
      __syncthreads();
      for (int c = threadIdx.x; c < P.d; c += blockDim.x) {
        float t = 0.f;
        for (int k = 0; k < nw * per_warp; ++k) t += sums[static_cast<size_t>(k) * P.d + c];
        P.partial[(static_cast<size_t>(blockIdx.x) * 2 + o) * P.d + c] = t;
      }
    }
  }
}

// dg[o][c] = sum over blocks of partial[block][o][c]: 32 columns a block, 32 threads a column, joined in order
__global__ void __launch_bounds__(1024) weight_grad_kernel(const float* __restrict__ partial, int blocks, int d,
                                                           void* dq_weight, void* dk_weight, int bf16) {
  __shared__ float part[32][33];
  const int c = blockIdx.x * 32 + (threadIdx.x & 31), k0 = threadIdx.x >> 5;
  float t = 0.f;
  if (c < 2 * d)
    for (int b = k0; b < blocks; b += 32) t += partial[static_cast<size_t>(b) * 2 * d + c];
  part[k0][threadIdx.x & 31] = t;
  __syncthreads();
  if (k0 == 0 && c < 2 * d) {
    t = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += part[k][threadIdx.x];
    void* const out = c < d ? dq_weight : dk_weight;
    const int i = c < d ? c : c - d;
    if (out) {
      if (bf16) static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(t);
      else static_cast<float*>(out)[i] = t;
    }
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
// follows from it: V = 8 and 4 need at most 32 lanes for 256 channels, V = 2 two slots, V = 1 four.
int choose_v(const Params& P, bool inter, int dtype, bool bwd, int nops) {
  const int es = dtype == MSL_DTYPE_BF16 ? 2 : 4;
  for (int v = 8; v > 1; v /= 2) {
    // 8 pairs a lane only where it makes 16-byte loads out of 8-byte ones (split pairs of bf16)
    if (v == 8 && (inter || es == 4)) continue;
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

template <typename T, int V, int SL, bool INTER, bool NORM, bool BWD>
cudaError_t launch(Params P, cudaStream_t s, int blocks_fixed) {
  P.lanes = (P.d / (2 * V) + SL - 1) / SL;
  const int per_warp = 32 / P.lanes;
  const int units = (P.heads[0] + per_warp - 1) / per_warp + (P.heads[1] + per_warp - 1) / per_warp;
  // few tokens: several warps share a token's heads, until every SM has some
  const long long want = static_cast<long long>(sm_count()) * kWarps;
  long long splits = P.rows >= want ? 1 : (want + P.rows - 1) / P.rows;
  if (splits > units) splits = units;
  P.splits = static_cast<int>(splits);
  long long blocks = (P.rows * splits + kWarps - 1) / kWarps;
  if (blocks_fixed) blocks = blocks_fixed;
  if (blocks > 0x7fffffffLL) blocks = 0x7fffffffLL;  // the kernel strides over the rest
  const size_t smem = BWD && P.partial ? sizeof(float) * kWarps * per_warp * P.d : 0;
  rotary_kernel<T, V, SL, INTER, NORM, BWD><<<static_cast<unsigned>(blocks), kWarps * 32, smem, s>>>(P);
  return cudaGetLastError();
}

template <typename T, bool INTER, bool NORM, bool BWD>
cudaError_t by_v(const Params& P, int v, cudaStream_t s, int blocks) {
  switch (v) {
    case 8:
      if constexpr (!INTER && sizeof(T) == 2) return launch<T, 8, 1, INTER, NORM, BWD>(P, s, blocks);
      return cudaErrorInvalidValue;
    case 4: return launch<T, 4, 1, INTER, NORM, BWD>(P, s, blocks);
    case 2: return launch<T, 2, 2, INTER, NORM, BWD>(P, s, blocks);
    default: return launch<T, 1, 4, INTER, NORM, BWD>(P, s, blocks);
  }
}

template <bool NORM, bool BWD>
cudaError_t dispatch(const Params& P, bool inter, int dtype, cudaStream_t s, int blocks) {
  const int v = choose_v(P, inter, dtype, BWD, 2);
  if (dtype == MSL_DTYPE_BF16)
    return inter ? by_v<__nv_bfloat16, true, NORM, BWD>(P, v, s, blocks) : by_v<__nv_bfloat16, false, NORM, BWD>(P, v, s, blocks);
  return inter ? by_v<float, true, NORM, BWD>(P, v, s, blocks) : by_v<float, false, NORM, BWD>(P, v, s, blocks);
}

// Blocks of a backward whose weights' gradients are wanted: resident ones only, each keeps its sums.
int bwd_blocks(const msl_rotary_geometry* g, const msl_qk_norm_io* io) {
  const long long most = static_cast<long long>(sm_count()) * kBwdBlocksPerSm;
  const long long units = g->rows * (static_cast<long long>(io->heads) + io->kv_heads);  // at least as many as items
  const long long need = (units + kWarps - 1) / kWarps;
  return static_cast<int>(need < most ? (need > 0 ? need : 1) : most);
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
  const cudaError_t e = rot::dispatch<false, false>(P, geom->interleaved != 0, geom->dtype, static_cast<cudaStream_t>(stream), 0);
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
  const cudaError_t e = rot::dispatch<true, false>(P, geom->interleaved != 0, geom->dtype, static_cast<cudaStream_t>(stream), 0);
  if (e != cudaSuccess) return cuda_failf(e, "rotary_kernel launch");
  count_launches(1);
  return MSL_OK;
}

size_t msl_qk_norm_rope_bwd_workspace_bytes(const msl_rotary_geometry* geom, const msl_qk_norm_io* io) {
  rot::Params P;
  if (rot::fill_norm(geom, io, P)) return 0;
  if (!io->dq_weight && !io->dk_weight) return 0;
  return sizeof(float) * 2 * P.d * rot::bwd_blocks(geom, io);
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
  const int blocks = rot::bwd_blocks(geom, io);
  if (dw) {
    const size_t need = sizeof(float) * 2 * P.d * blocks;
    if (!workspace || workspace_bytes < need)
      return failf(MSL_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : 0);
    if (!multiple_of(workspace, 4)) return failf(MSL_ERR_INVALID, "workspace must be 4-byte aligned");
    P.partial = static_cast<float*>(workspace);
  }
  cudaError_t e = rot::dispatch<true, true>(P, geom->interleaved != 0, geom->dtype, s, dw ? blocks : 0);
  if (e != cudaSuccess) return cuda_failf(e, "rotary_kernel launch");
  if (dw) {
    rot::weight_grad_kernel<<<(2 * P.d + 31) / 32, 1024, 0, s>>>(P.partial, blocks, P.d, io->dq_weight, io->dk_weight,
                                                                io->weight_dtype == MSL_DTYPE_BF16);
    e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_failf(e, "weight_grad_kernel launch");
  }
  count_launches(dw ? 2 : 1);
  return MSL_OK;
}

}  // extern "C"
