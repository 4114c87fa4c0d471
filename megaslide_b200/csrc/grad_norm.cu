// Global gradient norm over many tensors, and clipping.
//
//   norm = sqrt(extra + sum over tensors of sum_i g_i^2),   out = g * min(1, max_norm / (norm + 1e-6))
//
// Bound by bytes: the norm reads everything once, the scaling reads it again (the factor is known only
// when the last element has been read; backwards, so that it begins with what the caches still hold) and writes
// it.  The tensors are cut into chunks, which the blocks take in turn, whatever the tensors' sizes, so two
// launches serve any number of tensors up to kMaxTensors (more take further launches).  Chunks grow with the
// total from 2048 elements (a few megabytes still reach every SM) to 32768.  Measured with 504 bf16 tensors of
// 1.63 GB, results not aligned with their sources: norm 260 us, 6.3 TB/s, scaling 588 us, 5.5 TB/s (a
// contiguous share of the chunks for every block: 650 us; chunks of 8192: 284 and 641; 4 blocks a SM instead
// of 8: 880 us).
// The table of tensors travels in the kernel's parameters: no copy to the device, nothing to keep alive.
// Sums: float32 in a thread's part of a chunk, double from there on, joined in a fixed order (the same result on
// every run on the same kind of GPU).

#include <math.h>

#include <algorithm>
#include <new>

#include "msl_abi.cuh"
#include "msl_common.cuh"

namespace msl {
namespace clip {

constexpr int kThreads = 256;
constexpr int kLeastChunk = 2048, kMostChunk = 32768;  // elements
constexpr int kMaxTensors = 896;   // of a launch
constexpr int kBlocksPerSm = 8;

struct Table {
  const void* src[kMaxTensors];
  void* dst[kMaxTensors];
  long long numel[kMaxTensors];
  unsigned first[kMaxTensors + 1];  // chunks before the tensor; [count] = all
  unsigned char bf16[kMaxTensors];
  int count, chunk;
};
static_assert(sizeof(Table) + 64 <= 32764, "a kernel's parameters may take 32764 bytes, other ones than the table 40 of them");

// last tensor whose first chunk is <= c (tensors without elements have no chunk and are never it)
__device__ __forceinline__ int tensor_of(const Table& t, unsigned c) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= c) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ void sum_span(const T* p, int n, float& acc) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T)));
  for (int i = threadIdx.x; i < head; i += kThreads) { const float v = to_f32<T>(p[i]); acc = fmaf(v, v, acc); }
  const uint4* const q = reinterpret_cast<const uint4*>(p + head);
  const int nv = (n - head) / kPer;
#pragma unroll 4
  for (int i = threadIdx.x; i < nv; i += kThreads) {
    const uint4 w = __ldg(q + i);
    const T* e = reinterpret_cast<const T*>(&w);
#pragma unroll
    for (int j = 0; j < kPer; ++j) { const float v = to_f32<T>(e[j]); acc = fmaf(v, v, acc); }
  }
  for (int i = head + nv * kPer + threadIdx.x; i < n; i += kThreads) { const float v = to_f32<T>(p[i]); acc = fmaf(v, v, acc); }
}

template <typename T>
__device__ __forceinline__ uint4 scaled(uint4 w, float c) {
  T* const e = reinterpret_cast<T*>(&w);
#pragma unroll
  for (int j = 0; j < 16 / static_cast<int>(sizeof(T)); ++j) e[j] = from_f32<T>(to_f32<T>(e[j]) * c);
  return w;
}

// 16 bytes from `shift` bytes into two adjacent aligned 16-byte words (shift a multiple of 2, 0 < shift < 16)
__device__ __forceinline__ uint4 window(uint4 a, uint4 b, int shift) {
  const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
  uint32_t t[5], o[4];
  const int words = shift >> 2, bits = (shift & 3) * 8;
#pragma unroll
  for (int i = 0; i < 5; ++i) t[i] = words == 0 ? w[i] : words == 1 ? w[i + 1] : words == 2 ? w[i + 2] : w[i + 3 < 8 ? i + 3 : 7];
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = __funnelshift_r(t[i], t[i + 1], bits);
  return make_uint4(o[0], o[1], o[2], o[3]);
}

// Stores are whole aligned 16-byte words.  Where the source is not aligned alike, each word comes out of two
// aligned loads of the source (the second is the neighbour's first: it hits L1).
template <typename T>
__device__ __forceinline__ void scale_span(const T* p, T* o, int n, float c) {
  constexpr int kPer = 16 / static_cast<int>(sizeof(T));
  const int head = min(n, static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(o) & 15)) & 15) / sizeof(T)));
  const int shift = static_cast<int>(reinterpret_cast<uintptr_t>(p + head) & 15);
  // the two loads of a word stay inside the span: one word less where the last would reach past it, and the
  // first is done apart where its loads would begin before it
  const int before = shift != 0 && head * static_cast<int>(sizeof(T)) < shift ? 1 : 0;
  int nv = (n - head) / kPer;
  if (shift != 0 && nv > 0 && (n - head - nv * kPer) * static_cast<int>(sizeof(T)) < 16 - shift) --nv;
  const int start = min(head + before * kPer, n);  // elements before the words
  nv = max(nv - before, 0);
  for (int i = threadIdx.x; i < start; i += kThreads) o[i] = from_f32<T>(to_f32<T>(p[i]) * c);
  uint4* const r = reinterpret_cast<uint4*>(o + start);
  const uint4* const q = reinterpret_cast<const uint4*>(reinterpret_cast<uintptr_t>(p + start) - shift);
  if (shift == 0) {
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += kThreads) r[i] = scaled<T>(q[i], c);
  } else {
#pragma unroll 4
    for (int i = threadIdx.x; i < nv; i += kThreads) r[i] = scaled<T>(window(q[i], q[i + 1], shift), c);
  }
  for (int i = start + nv * kPer + threadIdx.x; i < n; i += kThreads) o[i] = from_f32<T>(to_f32<T>(p[i]) * c);
}

__device__ __forceinline__ double block_sum(double v) {
  __shared__ double part[kThreads / 32];
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0;
#pragma unroll
  for (int i = 0; i < kThreads / 32; ++i) v += part[i];
  __syncthreads();
  return v;
}

__global__ void __launch_bounds__(kThreads, kBlocksPerSm) sumsq_kernel(const __grid_constant__ Table t, double* __restrict__ partial) {
  // a chunk's squares of a thread (128 at most) add up in float32, the chunks in double: thousands of squares of
  // bf16 numbers, whose few bits leave many ties, drift by 5e-6 in one float32 sum
  double sum = 0.0;
  const unsigned all = t.first[t.count];
  for (unsigned c = blockIdx.x; c < all; c += gridDim.x) {
    const int k = tensor_of(t, c);
    const long long at = static_cast<long long>(c - t.first[k]) * t.chunk;
    const int n = static_cast<int>(min(static_cast<long long>(t.chunk), t.numel[k] - at));
    float acc = 0.f;
    if (t.bf16[k]) sum_span(static_cast<const __nv_bfloat16*>(t.src[k]) + at, n, acc);
    else sum_span(static_cast<const float*>(t.src[k]) + at, n, acc);
    sum += static_cast<double>(acc);
  }
  const double s = block_sum(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

// every block joins the same sums in the same order
__device__ __forceinline__ float join(const double* __restrict__ partial, int n, double extra) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v += partial[i];
  return static_cast<float>(sqrt(block_sum(v) + extra));
}

__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_kernel(const double* __restrict__ partial, int n, double extra, float* norm) {
  const float v = join(partial, n, extra);
  if (threadIdx.x == 0) *norm = v;
}

__global__ void __launch_bounds__(kThreads, kBlocksPerSm)
    scale_kernel(const __grid_constant__ Table t, const double* __restrict__ partial, int n, double extra, float max_norm, float* norm) {
  const float v = join(partial, n, extra);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  float f = max_norm / (v + 1e-6f);
  f = f > 1.f ? 1.f : f;  // a NaN stays a NaN
  const unsigned all = t.first[t.count];
  for (unsigned i = blockIdx.x; i < all; i += gridDim.x) {
    const unsigned c = all - 1 - i;
    const int k = tensor_of(t, c);
    const long long at = static_cast<long long>(c - t.first[k]) * t.chunk;
    const int m = static_cast<int>(min(static_cast<long long>(t.chunk), t.numel[k] - at));
    if (t.bf16[k]) scale_span(static_cast<const __nv_bfloat16*>(t.src[k]) + at, static_cast<__nv_bfloat16*>(t.dst[k]) + at, m, f);
    else scale_span(static_cast<const float*>(t.src[k]) + at, static_cast<float*>(t.dst[k]) + at, m, f);
  }
}

// ------------------------------------------------------------------------------------------ host

long long chunks_of(int64_t n, int chunk) { return (n + chunk - 1) / chunk; }

int grid_of(long long chunks) {
  const long long most = static_cast<long long>(sm_count()) * kBlocksPerSm;
  return static_cast<int>(chunks < most ? (chunks > 0 ? chunks : 1) : most);
}

// The chunk that gives every resident block one, within the limits; the same for all launches of a call.
int chunk_of(const int64_t* numel, int count) {
  long long total = 0;
  for (int i = 0; i < count; ++i) total += numel[i];
  const long long each = total / (static_cast<long long>(sm_count()) * kBlocksPerSm);
  int chunk = kLeastChunk;
  while (chunk < kMostChunk && chunk < each) chunk *= 2;
  return chunk;
}

// The tensors of a launch, up to kMaxTensors from `at` on: visit(tensor, chunks before it); returns the next tensor.
template <typename F>
int each_of(const int64_t* numel, int count, int at, int chunk, long long* all, F visit) {
  long long chunks = 0;
  int k = 0;
  for (; at < count && k < kMaxTensors; ++at) {
    const long long c = chunks_of(numel[at], chunk);
    if (c <= 0) continue;
    if (chunks + c > 0x7fffffffLL && k > 0) break;
    visit(at, k++, chunks);
    chunks += c;
  }
  *all = chunks;
  return at;
}

int fill(Table& t, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int count, int at, int chunk) {
  long long all = 0;
  t.count = 0;
  t.chunk = chunk;
  at = each_of(numel, count, at, chunk, &all, [&](int i, int k, long long before) {
    t.src[k] = src[i];
    t.dst[k] = dst ? dst[i] : nullptr;
    t.numel[k] = numel[i];
    t.bf16[k] = dtype[i] == MSL_DTYPE_BF16;
    t.first[k] = static_cast<unsigned>(before);
    t.count = k + 1;
  });
  t.first[t.count] = static_cast<unsigned>(all);
  return at;
}

// Blocks of every launch over these tensors together (the sums of a launch follow those before it).
long long all_blocks(const int64_t* numel, int count) {
  const int chunk = chunk_of(numel, count);
  long long n = 0, all = 0;
  int at = 0;
  do {
    at = each_of(numel, count, at, chunk, &all, [](int, int, long long) {});
    n += grid_of(all);
  } while (at < count);
  return n;
}

// Results must not share memory with one another, nor with a source other than their own in place: blocks read and write
// them in no order, so an element would be scaled once or twice, by chance.  504 tensors: 11 us of the host's time.
int check_overlap(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int32_t count) {
  struct Range {
    uintptr_t begin, end;
    int tensor;
  };
  Range* const r = new (std::nothrow) Range[count > 0 ? count : 1];
  if (!r) return failf(MSL_ERR_UNSUPPORTED, "no host memory for %d tensors", count);
  auto bytes = [&](int i) { return static_cast<uintptr_t>(numel[i]) * (dtype[i] == MSL_DTYPE_BF16 ? 2 : 4); };
  int n = 0;
  bool in_place = true;
  for (int i = 0; i < count; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t at = reinterpret_cast<uintptr_t>(dst[i]);
    r[n++] = {at, at + bytes(i), i};
    in_place = in_place && dst[i] == src[i];
  }
  std::sort(r, r + n, [](const Range& a, const Range& b) { return a.begin < b.begin; });
  int one = -1, other = -1;
  const char* what = "result";
  for (int k = 1; k < n && one < 0; ++k)
    if (r[k].begin < r[k - 1].end) { one = r[k].tensor; other = r[k - 1].tensor; }
  for (int i = 0; i < count && one < 0 && !in_place; ++i) {
    if (numel[i] == 0) continue;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(src[i]), end = begin + bytes(i);
    for (const Range* q = std::upper_bound(r, r + n, begin, [](uintptr_t b, const Range& a) { return b < a.end; }); q < r + n && q->begin < end; ++q) {
      if (q->tensor == i && q->begin == begin) continue;
      one = q->tensor;
      other = i;
      what = "source";
      break;
    }
  }
  delete[] r;
  return one < 0 ? MSL_OK : failf(MSL_ERR_INVALID, "tensor %d: its result overlaps the %s of tensor %d", one, what, other);
}

int check(const void* const* src, void* const* dst, bool scale, const int64_t* numel, const int32_t* dtype, int32_t count,
          double extra, const float* norm, void* workspace, size_t bytes) {
  if (count < 0) return failf(MSL_ERR_INVALID, "count must be >= 0");
  if (count > 0 && (!src || !numel || !dtype || (scale && !dst))) return failf(MSL_ERR_INVALID, "src, dst, numel and dtype are required");
  if (!norm) return failf(MSL_ERR_INVALID, "norm is required");
  if (!(extra >= 0.0)) return failf(MSL_ERR_INVALID, "extra_sumsq must be >= 0");
  for (int i = 0; i < count; ++i) {
    if (numel[i] < 0) return failf(MSL_ERR_INVALID, "tensor %d: numel must be >= 0", i);
    if (dtype[i] != MSL_DTYPE_F32 && dtype[i] != MSL_DTYPE_BF16) return failf(MSL_ERR_INVALID, "tensor %d: unknown dtype %d", i, dtype[i]);
    if (numel[i] == 0) continue;
    if (!src[i] || (scale && !dst[i])) return failf(MSL_ERR_INVALID, "tensor %d: NULL", i);
    const unsigned es = dtype[i] == MSL_DTYPE_BF16 ? 2 : 4;
    if (!multiple_of(src[i], es) || (scale && !multiple_of(dst[i], es)))
      return failf(MSL_ERR_INVALID, "tensor %d: not aligned to its elements", i);
    if (chunks_of(numel[i], kLeastChunk) > 0x7fffffffLL) return failf(MSL_ERR_UNSUPPORTED, "tensor %d: too many elements", i);
  }
  const int rc = scale ? check_overlap(src, dst, numel, dtype, count) : MSL_OK;
  if (rc) return rc;
  const size_t need = sizeof(double) * static_cast<size_t>(all_blocks(numel, count));
  if (!workspace || bytes < need) return failf(MSL_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? bytes : 0);
  if (!multiple_of(workspace, 8)) return failf(MSL_ERR_INVALID, "workspace must be 8-byte aligned");
  return MSL_OK;
}

}  // namespace clip
}  // namespace msl

using namespace msl;

static int sum_squares(clip::Table& t, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype,
                       int32_t count, double* partial, cudaStream_t s, int* blocks) {
  const int chunk = clip::chunk_of(numel, count);
  int at = 0, n = 0;
  do {
    at = clip::fill(t, src, dst, numel, dtype, count, at, chunk);
    const int g = clip::grid_of(t.first[t.count]);
    clip::sumsq_kernel<<<g, clip::kThreads, 0, s>>>(t, partial + n);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_failf(e, "sumsq_kernel launch");
    count_launches(1);
    n += g;
  } while (at < count);
  *blocks = n;
  return MSL_OK;
}

extern "C" {

size_t msl_grad_norm_workspace_bytes(const int64_t* numel, int32_t count) {
  if (count < 0 || (count > 0 && !numel)) return 0;
  return sizeof(double) * static_cast<size_t>(clip::all_blocks(numel, count));
}

int msl_grad_norm(const void* const* src, const int64_t* numel, const int32_t* dtype, int32_t count,
                  double extra_sumsq, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = clip::check(src, nullptr, false, numel, dtype, count, extra_sumsq, norm, workspace, workspace_bytes);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  double* const partial = static_cast<double*>(workspace);
  static thread_local clip::Table t;
  int n = 0;
  rc = sum_squares(t, src, nullptr, numel, dtype, count, partial, s, &n);
  if (rc) return rc;
  clip::norm_kernel<<<1, clip::kThreads, 0, s>>>(partial, n, extra_sumsq, norm);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return cuda_failf(e, "norm_kernel launch");
  count_launches(1);
  return MSL_OK;
}

int msl_grad_clip(const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype, int32_t count,
                  double extra_sumsq, float max_norm, float* norm, void* workspace, size_t workspace_bytes,
                  void* stream) {
  if (!(max_norm >= 0.f)) return failf(MSL_ERR_INVALID, "max_norm must be >= 0");
  int rc = clip::check(src, dst, true, numel, dtype, count, extra_sumsq, norm, workspace, workspace_bytes);
  if (rc) return rc;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  double* const partial = static_cast<double*>(workspace);
  static thread_local clip::Table t;
  int n = 0;
  rc = sum_squares(t, src, dst, numel, dtype, count, partial, s, &n);
  if (rc) return rc;
  const int chunk = t.chunk;
  int at = 0;
  do {
    at = clip::fill(t, src, dst, numel, dtype, count, at, chunk);
    clip::scale_kernel<<<clip::grid_of(t.first[t.count]), clip::kThreads, 0, s>>>(t, partial, n, extra_sumsq, max_norm, norm);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return cuda_failf(e, "scale_kernel launch");
    count_launches(1);
  } while (at < count);
  return MSL_OK;
}

}  // extern "C"
