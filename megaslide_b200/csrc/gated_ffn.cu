// Gated feed-forward block, forward and backward: which kernel takes a product, the bias gradients, and the entry points.
//
//   [g u] = x w_in^T + b_in;  h = act(g) u;  y = h w_out^T + b_out
//   dh = dy w_out;  dg = dh (u act'(g));  du = dh act(g), of which the forward keeps the two factors;
//   dx = [dg du] w_in;  dw_in = [dg du]^T x;  dw_out = dy^T h;  db_in, db_out = column sums of [dg du], dy

#include <initializer_list>

#include "gated_ffn.cuh"

namespace msl {
namespace ffn {

// ------------------------------------------------------------------------------------------ column sums

// The sums of up to two matrices' columns in one launch.  Bound by bytes (604 MB for the 32768 x 9216 gradients of
// the projections in bf16): every element is read once, V adjacent columns a thread (16 bytes), 8 warps a block on
// alternate rows, four rows' loads in flight.  partial[slice][c] = sum of the slice's rows, or out[c] where there
// is one slice.
struct Columns {
  const void* x;
  void* out;
  float* partial;
  long long ld;
  int cols, blocks;
};
struct ColumnArgs {
  Columns of[2];
  long long rows, per;
};

template <typename T, int V>
__global__ void __launch_bounds__(256) column_sum_kernel(const __grid_constant__ ColumnArgs A) {
  __shared__ float part[8][32 * V + 1];
  const int second = static_cast<int>(blockIdx.x) >= A.of[0].blocks;
  const Columns& C = A.of[second];
  const int block = static_cast<int>(blockIdx.x) - (second ? A.of[0].blocks : 0);
  const int lane = threadIdx.x & 31, y = threadIdx.x >> 5;
  const int c = (block * 32 + lane) * V;
  const long long r1 = min(A.rows, (blockIdx.y + 1LL) * A.per);
  float t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = 0.f;
  if (c < C.cols) {
    const T* p = static_cast<const T*>(C.x) + (blockIdx.y * A.per + y) * C.ld + c;
    long long r = blockIdx.y * A.per + y;
    if constexpr (V == 1) {
      for (; r < r1; r += 8, p += 8 * C.ld) t[0] += to_f32<T>(p[0]);
    } else {
      for (; r + 24 < r1; r += 32, p += 32 * C.ld) {
        uint4 w[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) w[u] = __ldg(reinterpret_cast<const uint4*>(p + u * 8 * C.ld));
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int i = 0; i < V; ++i) t[i] += to_f32<T>(reinterpret_cast<const T*>(&w[u])[i]);
      }
      for (; r < r1; r += 8, p += 8 * C.ld) {
        const uint4 w = __ldg(reinterpret_cast<const uint4*>(p));
#pragma unroll
        for (int i = 0; i < V; ++i) t[i] += to_f32<T>(reinterpret_cast<const T*>(&w)[i]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < V; ++i) part[y][lane * V + i] = t[i];
  __syncthreads();
  for (int k = threadIdx.x; k < 32 * V; k += 256) {
    const int col = block * 32 * V + k;
    if (col >= C.cols) break;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += part[i][k];
    if (gridDim.y == 1) static_cast<T*>(C.out)[col] = from_f32<T>(sum);
    else C.partial[static_cast<size_t>(blockIdx.y) * C.cols + col] = sum;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) column_join_kernel(const __grid_constant__ ColumnArgs A, int slices) {
  const Columns& C = A.of[blockIdx.y];
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= C.cols) return;
  float t = 0.f;
#pragma unroll 8
  for (int s = 0; s < slices; ++s) t += C.partial[static_cast<size_t>(s) * C.cols + c];
  static_cast<T*>(C.out)[c] = from_f32<T>(t);
}

constexpr int kSlices = 64;

template <typename T>
static cudaError_t column_sums_t(ColumnArgs a, cudaStream_t s) {
  constexpr int kVec = 16 / static_cast<int>(sizeof(T));
  const int count = a.of[1].out ? 2 : 1;
  a.per = a.rows > 128 * kSlices ? (a.rows + kSlices - 1) / kSlices : 128;
  const int slices = static_cast<int>((a.rows + a.per - 1) / a.per);
  bool vec = true;
  for (int i = 0; i < count; ++i) vec = vec && multiple_of(a.of[i].x, 16) && a.of[i].ld % kVec == 0 && a.of[i].cols % kVec == 0;
  const int v = vec ? kVec : 1;
  int blocks = 0, widest = 0;
  for (int i = 0; i < count; ++i) {
    a.of[i].blocks = (a.of[i].cols + 32 * v - 1) / (32 * v);
    blocks += a.of[i].blocks;
    widest = a.of[i].cols > widest ? a.of[i].cols : widest;
  }
  const dim3 grid(blocks, slices);
  if (vec) column_sum_kernel<T, kVec><<<grid, 256, 0, s>>>(a);
  else column_sum_kernel<T, 1><<<grid, 256, 0, s>>>(a);
  if (slices > 1) column_join_kernel<T><<<dim3((widest + 255) / 256, count), 256, 0, s>>>(a, slices);
  count_launches(slices > 1 ? 2 : 1);
  return cudaGetLastError();
}

// The workspace's slots for planes, and the matrix whose planes each holds in this call.  Two operands may begin at one
// address (w_out or x as the first rows of w_in, say), so a matrix is its shape and row stride as well.
struct Held {
  const void* src;
  long long rows, cols, ld;
};
struct Slots {
  char* at[3];
  size_t bytes[3];
  Held of[3];
};

static const char* const kOff16 = "an address or a row stride is no multiple of 16 bytes and the geometry's unaligned is 0";

static int run(const Product& p, Slots& slots, int slot_a, int slot_b, cudaStream_t s, bool rows = false) {
  cudaError_t e;
  if (rows) {
    e = launch_product_rows(p, s);
    if (e != cudaSuccess) return cuda_failf(e, "rows_kernel launch");
  } else if (tc_applies(p)) {
    e = launch_product_tc(p, s);
    if (e != cudaSuccess) return cuda_failf(e, "product_kernel launch");
  } else if (few_apply(p)) {
    e = launch_product_few(p, s);
    if (e != cudaSuccess) return cuda_failf(e, "few_kernel launch");
  } else if (slots.at[0] && planes_apply(p)) {
    const long long rows[2] = {p.a_major ? p.K : p.M, p.b_major ? p.K : (p.epilogue == kGate ? 2 * p.N : p.N)};
    const long long cols[2] = {p.a_major ? p.M : p.K, p.b_major ? p.N : p.K};
    const void* const src[2] = {p.a, p.b};
    const long long ld[2] = {p.lda, p.ldb};
    const int slot[2] = {slot_a, slot_b};
    PlaneJob jobs[2];
    int count = 0;
    for (int i = 0; i < 2; ++i) {
      Held& held = slots.of[slot[i]];
      if (held.src == src[i] && held.rows == rows[i] && held.cols == cols[i] && held.ld == ld[i]) continue;
      if (planes_bytes(p.dtype, rows[i], cols[i]) > slots.bytes[slot[i]]) return failf(MSL_ERR_WORKSPACE, "planes beyond their slot");
      jobs[count++] = {src[i], ld[i], rows[i], cols[i], slots.at[slot[i]]};
      held = {src[i], rows[i], cols[i], ld[i]};
    }
    if (count) {
      e = launch_planes(p.dtype, jobs, count, s);
      if (e != cudaSuccess) return cuda_failf(e, "split_kernel launch");
    }
    // the gradient of h passes through slot 1, as wide and not yet used: the gradients of g and u come after it
    if (p.epilogue == kDgate && p.dtype == MSL_DTYPE_BF16 && sizeof(float) * p.M * p.N > slots.bytes[1])
      return failf(MSL_ERR_WORKSPACE, "the gradient of h beyond its slot");
    e = launch_product_planes(p, slots.at[slot_a], slots.at[slot_b], reinterpret_cast<float*>(slots.at[1]), s);
    if (e != cudaSuccess) return cuda_failf(e, "planes_kernel launch");
  } else if (p.dtype == MSL_DTYPE_F32) {
    e = launch_product_skinny(p, s);
    if (e != cudaSuccess) return cuda_failf(e, "skinny_kernel launch");
  } else if (!slots.at[0]) {
    return failf(MSL_ERR_INVALID, kOff16);
  } else {
    return failf(MSL_ERR_UNSUPPORTED, "the driver encodes no tensor maps, or the product has over 2^30 tiles");
  }
  count_launches(1);
  return MSL_OK;
}

static int check(const msl_ffn_geometry* g, const msl_ffn_io* io) {
  if (!g) return failf(MSL_ERR_INVALID, "geometry is NULL");
  if (g->rows < 0 || g->dim < 1 || g->hidden < 1) return failf(MSL_ERR_INVALID, "rows must be >= 0, dim and hidden >= 1");
  if (g->dtype != MSL_DTYPE_F32 && g->dtype != MSL_DTYPE_BF16) return failf(MSL_ERR_INVALID, "unknown dtype %d", g->dtype);
  if (g->activation != MSL_ACT_SILU && g->activation != MSL_ACT_GELU) return failf(MSL_ERR_INVALID, "unknown activation %d", g->activation);
  if (g->dim > (1 << 21)) return failf(MSL_ERR_UNSUPPORTED, "dim is over 2^21");
  if (g->hidden > (1 << 20)) return failf(MSL_ERR_UNSUPPORTED, "hidden is over 2^20");
  if (g->rows > (1LL << 31) - 256) return failf(MSL_ERR_UNSUPPORTED, "rows is over 2^31 - 256");
  if (!io) return failf(MSL_ERR_INVALID, "io is NULL");
  return MSL_OK;
}

// Workspace: the sums of parts of tiles of one product at a time, the column sums' slices, and planes of
// operands: forward, x or h and one weight; backward, dy, the gradients of g and u, and the product's other operand.
struct Workspace {
  size_t partial, columns, planes[3], total;
};
// A bf16 forward that the kernels for few rows do whole, if the operands lie on 16 bytes as the geometry says.
static bool few_rows(const msl_ffn_geometry* g, bool backward) {
  return !backward && g->dtype == MSL_DTYPE_BF16 && g->rows <= rows_most(g->dtype, 2LL * g->hidden * g->dim) && g->dim % 8 == 0 &&
         g->hidden % 8 == 0 && !g->unaligned;
}
static Workspace workspace_of(const msl_ffn_geometry* g, bool backward) {
  Workspace w{};
  const long long M = g->rows, C = g->dim, F = g->hidden;
  const bool f32 = g->dtype == MSL_DTYPE_F32, copies = !f32 && (C % 8 || F % 8 || g->unaligned);
  if (few_rows(g, backward)) return w;
  bool planes = false;  // some product takes planes
  auto need = [&](long long m, long long n, long long k, int epilogue, bool b_major, bool a_major = false) {
    if (M == 0) return;
    Product p{};
    p.dtype = g->dtype;
    p.epilogue = epilogue;
    p.M = m;
    p.N = n;
    p.K = k;
    size_t b = 0;
    if ((f32 || copies) && planes_apply(p)) {
      planes = true;
      b = planes_partial_bytes(g->dtype, m, n, k, epilogue);
    } else if (f32) {
      b = skinny_bytes(m, n, k, epilogue, a_major);
    }
    if (f32 && few_shape(m, epilogue == kGate ? 2 * n : n, k, a_major, b_major)) {
      const size_t few = few_bytes(m, n, k, epilogue);
      b = few > b ? few : b;
    }
    // some products of a bf16 block may be addressable though others are not
    const size_t t = f32 ? 0 : tc_partial_bytes(m, n, k, epilogue, b_major);
    if (b > w.partial) w.partial = b;
    if (t > w.partial) w.partial = t;
  };
  auto most = [](std::initializer_list<size_t> v) {
    size_t m = 0;
    for (size_t x : v) m = x > m ? x : m;
    return m;
  };
  auto size = [&](long long rows, long long cols) { return planes_bytes(g->dtype, rows, cols); };
  if (backward) {
    need(M, F, C, kDgate, true);
    need(M, C, 2 * F, kPlain, true);
    need(2 * F, C, M, kPlain, true, true);
    need(C, F, M, kPlain, true, true);
    w.columns = sizeof(float) * kSlices * static_cast<size_t>(2 * F + C);
    w.columns = (w.columns + 255) / 256 * 256;
    if (planes && M > 0) {
      w.planes[0] = size(M, C);
      w.planes[1] = size(M, 2 * F);
      w.planes[2] = most({size(C, F), size(2 * F, C), size(M, C), size(M, F)});
    }
  } else {
    need(M, F, C, kGate, false);
    need(M, C, F, kPlain, false);
    if (planes && M > 0) {
      w.planes[0] = most({size(M, C), size(M, F)});
      w.planes[1] = most({size(2 * F, C), size(C, F)});
    }
  }
  w.partial = (w.partial + 255) / 256 * 256;
  w.total = w.partial + w.columns + w.planes[0] + w.planes[1] + w.planes[2];
  return w;
}
static Slots slots_of(const Workspace& w, void* workspace) {
  Slots s{};
  char* at = static_cast<char*>(workspace) + w.partial + w.columns;
  for (int i = 0; i < 3; ++i) {
    s.at[i] = w.planes[0] ? at : nullptr;
    s.bytes[i] = w.planes[i];
    at += w.planes[i];
  }
  return s;
}
static int check_workspace(const Workspace& w, const void* p, size_t bytes) {
  if (w.total == 0) return MSL_OK;
  if (!p || bytes < w.total) return failf(MSL_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", w.total, p ? bytes : 0);
  if (!multiple_of(p, 16)) return failf(MSL_ERR_INVALID, "workspace must be 16-byte aligned");
  return MSL_OK;
}

static Product product(const msl_ffn_geometry* g, const msl_ffn_io* io, const Workspace& w, void* workspace) {
  Product p{};
  p.dtype = g->dtype;
  p.act = g->activation;
  p.status = io->status;
  p.partial = static_cast<float*>(workspace);
  p.partial_bytes = w.partial;
  return p;
}

}  // namespace ffn
}  // namespace msl

using namespace msl;

extern "C" {

size_t msl_gated_ffn_workspace_bytes(const msl_ffn_geometry* geom, int32_t backward) {
  msl_ffn_io none{};
  return ffn::check(geom, &none) ? 0 : ffn::workspace_of(geom, backward != 0).total;
}

int msl_gated_ffn_fwd(const msl_ffn_geometry* geom, const msl_ffn_io* io, void* workspace, size_t workspace_bytes,
                      void* stream) {
  int rc = ffn::check(geom, io);
  if (rc) return rc;
  const long long M = geom->rows, C = geom->dim, F = geom->hidden;
  if (!io->w_in || !io->w_out) return failf(MSL_ERR_INVALID, "w_in and w_out are required");
  if (M == 0) return MSL_OK;
  if (!io->x || !io->h || !io->y) return failf(MSL_ERR_INVALID, "x, h and y are required");
  if (io->x_ld < C || io->y_ld < C) return failf(MSL_ERR_INVALID, "row strides must be >= dim = %lld", C);
  if (io->kept && geom->dtype == MSL_DTYPE_BF16 && !io->kept_low) return failf(MSL_ERR_INVALID, "kept_low is required beside kept in bf16");
  const ffn::Workspace W = ffn::workspace_of(geom, false);
  rc = ffn::check_workspace(W, workspace, workspace_bytes);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  ffn::Slots slots = ffn::slots_of(W, workspace);
  ffn::Product p = ffn::product(geom, io, W, workspace);
  p.epilogue = ffn::kGate;
  p.a = io->x; p.lda = io->x_ld;
  p.b = io->w_in; p.ldb = C;
  p.out = io->h; p.ldo = F;
  p.bias = io->b_in;
  p.kept_out = io->kept;
  p.low = static_cast<uint8_t*>(io->kept_low);
  p.M = M; p.N = F; p.K = C;
  ffn::Product q = ffn::product(geom, io, W, workspace);
  q.epilogue = ffn::kPlain;
  q.a = io->h; q.lda = F;
  q.b = io->w_out; q.ldb = F;
  q.out = io->y; q.ldo = io->y_ld;
  q.bias = io->b_out;
  q.M = M; q.N = C; q.K = F;
  // by rows, where each one's operands allow it (the second is launched into what comes before it)
  const bool few = M <= ffn::rows_most(geom->dtype, 2 * F * C), first = few && ffn::rows_apply(p), second = few && ffn::rows_apply(q);
  if (!(first && second) && ffn::few_rows(geom, false)) return failf(MSL_ERR_INVALID, ffn::kOff16);
  rc = ffn::run(p, slots, 0, 1, s, first);
  return rc ? rc : ffn::run(q, slots, 0, 1, s, second);
}

int msl_gated_ffn_bwd(const msl_ffn_geometry* geom, const msl_ffn_io* io, void* workspace, size_t workspace_bytes,
                      void* stream) {
  int rc = ffn::check(geom, io);
  if (rc) return rc;
  const long long M = geom->rows, C = geom->dim, F = geom->hidden;
  const size_t es = geom->dtype == MSL_DTYPE_BF16 ? 2 : 4;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (M == 0) {
    struct { void* p; size_t n; } zero[] = {{io->dw_in, 2 * F * C * es}, {io->dw_out, C * F * es}, {io->db_in, 2 * F * es}, {io->db_out, C * es}};
    for (const auto& z : zero) {
      const cudaError_t e = z.p ? cudaMemsetAsync(z.p, 0, z.n, s) : cudaSuccess;
      if (e != cudaSuccess) return cuda_failf(e, "clearing the weights' gradients");
    }
    return MSL_OK;
  }
  const bool inner = io->dx || io->dw_in || io->db_in;  // wants the gradients of g and u
  if (!io->dy || io->dy_ld < C) return failf(MSL_ERR_INVALID, "dy (row stride >= dim) is required");
  if (inner && (!io->w_out || !io->kept || !io->dgu)) return failf(MSL_ERR_INVALID, "w_out, kept and dgu are required");
  if (inner && geom->dtype == MSL_DTYPE_BF16 && !io->kept_low) return failf(MSL_ERR_INVALID, "kept_low is required beside kept in bf16");
  if (io->dx && (!io->w_in || io->dx_ld < C)) return failf(MSL_ERR_INVALID, "dx needs w_in and a row stride >= dim");
  if (io->dw_in && (!io->x || io->x_ld < C)) return failf(MSL_ERR_INVALID, "dw_in needs x");
  if (io->dw_out && !io->h) return failf(MSL_ERR_INVALID, "dw_out needs h");
  const ffn::Workspace W = ffn::workspace_of(geom, true);
  rc = ffn::check_workspace(W, workspace, workspace_bytes);
  if (rc) return rc;
  ffn::Slots slots = ffn::slots_of(W, workspace);
  ffn::Product p;
  if (inner) {
    p = ffn::product(geom, io, W, workspace);
    p.epilogue = ffn::kDgate;
    p.a = io->dy; p.lda = io->dy_ld;
    p.b = io->w_out; p.ldb = F; p.b_major = true;  // [K = dim, N = hidden]
    p.out = io->dgu; p.ldo = 2 * F;
    p.kept = io->kept;
    p.low = static_cast<uint8_t*>(io->kept_low);
    p.M = M; p.N = F; p.K = C;
    rc = ffn::run(p, slots, 0, 2, s);
    if (rc) return rc;
  }
  if (io->dx) {
    p = ffn::product(geom, io, W, workspace);
    p.a = io->dgu; p.lda = 2 * F;
    p.b = io->w_in; p.ldb = C; p.b_major = true;  // [K = 2 hidden, N = dim]
    p.out = io->dx; p.ldo = io->dx_ld;
    p.M = M; p.N = C; p.K = 2 * F;
    rc = ffn::run(p, slots, 1, 2, s);
    if (rc) return rc;
  }
  if (io->dw_in) {
    p = ffn::product(geom, io, W, workspace);
    p.a = io->dgu; p.lda = 2 * F; p.a_major = true;  // [K = rows, M = 2 hidden]
    p.b = io->x; p.ldb = io->x_ld; p.b_major = true;  // [K = rows, N = dim]
    p.out = io->dw_in; p.ldo = C;
    p.M = 2 * F; p.N = C; p.K = M;
    rc = ffn::run(p, slots, 1, 2, s);
    if (rc) return rc;
  }
  if (io->dw_out) {
    p = ffn::product(geom, io, W, workspace);
    p.a = io->dy; p.lda = io->dy_ld; p.a_major = true;  // [K = rows, M = dim]
    p.b = io->h; p.ldb = F; p.b_major = true;           // [K = rows, N = hidden]
    p.out = io->dw_out; p.ldo = F;
    p.M = C; p.N = F; p.K = M;
    rc = ffn::run(p, slots, 0, 2, s);
    if (rc) return rc;
  }
  if (io->db_in || io->db_out) {
    float* const partial = reinterpret_cast<float*>(static_cast<char*>(workspace) + W.partial);
    ffn::ColumnArgs a{};
    a.rows = M;
    int i = 0;
    if (io->db_in) a.of[i++] = {io->dgu, io->db_in, partial, 2 * F, static_cast<int>(2 * F), 0};
    if (io->db_out) a.of[i] = {io->dy, io->db_out, partial + 2 * F * ffn::kSlices, io->dy_ld, static_cast<int>(C), 0};
    const cudaError_t e = geom->dtype == MSL_DTYPE_BF16 ? ffn::column_sums_t<__nv_bfloat16>(a, s) : ffn::column_sums_t<float>(a, s);
    if (e != cudaSuccess) return cuda_failf(e, "column_sum_kernel launch");
  }
  return MSL_OK;
}

}  // extern "C"
