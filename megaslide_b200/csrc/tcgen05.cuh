// tcgen05 and TMA building blocks for products on pairs of CTAs (cta_group::2), and the host's tensor-map encoder.
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>
#include <stdint.h>

#include "megaslide_b200.h"

namespace msl {
namespace t5 {

constexpr long long kWaitClocks = 4000000000ll;  // two seconds, at most four

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
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
// Waits for phase `parity` of a barrier, at most kWaitClocks (counted on the SM's own clock: reading
// the global timer takes longer than most waits): then the CTA is marked dead and every role leaves.
__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* dead, uint32_t* status) {
  if (mbar_try(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (*dead) return false;
    if (clock64() - t0 > kWaitClocks) {
      *dead = 1;
      if (status) atomicOr(status, MSL_STATUS_TIMEOUT);
      return false;
    }
  }
  return true;
}
// The same for a whole warp: its lanes may see the end of a wait and the mark in any order, and must leave or go on together
// (what follows is executed by all of them or none).
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* dead, uint32_t* status) {
  return __all_sync(0xffffffffu, wait(bar, parity, dead, status));
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
template <int LEFT>
__device__ __forceinline__ void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(LEFT) : "memory"); }
__device__ __forceinline__ void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int x, int y, int z) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// arrives on the first CTA's barrier at the same place as `bar`.  Nothing that the thread itself wrote goes with
// it (the operands are the TMA's, the sums were read), so the plain form will do: .release.cluster took a
// microsecond, four times a block of 64 k.
__device__ __forceinline__ void arrive_first(uint32_t bar) {
  asm volatile("{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, 0;\n mbarrier.arrive.shared::cluster.b64 _, [a];\n}" ::"r"(bar)
               : "memory");
}

__device__ __forceinline__ void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile("{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
               "l"(b), "r"(idesc), "r"(accumulate ? 1 : 0) : "memory");
}
// arrives on the barrier at this place in both CTAs when the multiplications issued so far are done
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"(static_cast<uint16_t>(3)) : "memory");
}
// A CTA that gives up: the multiplications issued so far end (within the limit) before their operands' CTAs leave and their
// tensor memory is freed.
__device__ __forceinline__ void mma_drain(uint32_t bar) {
  mma_commit(bar);
  const long long since = clock64();
  while (!mbar_try(bar, 0) && clock64() - since < kWaitClocks) {
  }
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

// Driver entry that makes tensor maps; NULL where there is none.
using Encode = PFN_cuTensorMapEncodeTiled_v12000;

inline Encode encoder() {
  static const Encode encode = []() -> Encode {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<Encode>(fn);
  }();
  return encode;
}

// The encoder is a driver call and works only with the device's context current on the calling thread.  A thread that has
// made no runtime call of its own has none yet: autograd's, say, where its memory came out of torch's cache.
inline cudaError_t bind_context() {
  int device = 0;
  const cudaError_t e = cudaGetDevice(&device);
  return e != cudaSuccess ? e : cudaSetDevice(device);
}

}  // namespace t5
}  // namespace msl
