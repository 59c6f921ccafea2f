// PTX wrappers and operand descriptors of the dense product kernels (dense_*.cu).
// Shared-memory operands are 32-bit addresses in the shared window.
#pragma once
#include <cuda.h>

#include "common.cuh"

// Status word of the dense kernels on the current device: bit 0 = a bounded wait ran out.
int dmoq_dense_status(int* out);
int dmoq_dense_pair_status(int* out);
int dmoq_dense_mid_status(int* out);

namespace dense {

constexpr uint32_t kSpinLimit = 1u << 26;
constexpr long long kWaitCycles = 2000000000LL;   // about one second

// The kernels of the dense operators are launched so that one may be set up while its predecessor in the stream still runs
// (launch_overlapped).  overlap_point stands behind a kernel's set-up, which touches no global memory but for L2 prefetches:
// every block waits there until all that comes before the kernel in the stream has completed, and only then lets the next
// kernel's blocks in, so that at most two kernels overlap.  TMEM is allocated in front of it: the blocks that come in early
// never take columns that this kernel has yet to get.  What is read behind it is read with ordinary loads, not as constant.
__device__ __forceinline__ void overlap_point() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <class Kernel, class... Params>
int launch_overlapped(Kernel* kernel, unsigned grid, unsigned block, size_t smem, unsigned cluster, cudaStream_t s, const Params&... params) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(block);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = cluster;
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;   // 0: as the kernel was compiled
  if (cudaLaunchKernelEx(&cfg, kernel, params...) == cudaSuccess) return DMOQ_OK;
  (void)cudaGetLastError();   // reported by the return value; the next call on this thread starts clean
  return DMOQ_ELAUNCH;
}

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// One look at a barrier phase, without waiting: its result is used only after other instructions have been issued.
__device__ __forceinline__ uint32_t mbar_peek(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(100000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ int flag_get(uint32_t flag) {
  int v;
  asm volatile("ld.volatile.shared.u32 %0, [%1];" : "=r"(v) : "r"(flag) : "memory");
  return v;
}
__device__ __forceinline__ void flag_set(uint32_t flag) {
  asm volatile("st.volatile.shared.u32 [%0], %1;" ::"r"(flag), "r"(1) : "memory");
}
// Bounded wait for a barrier phase.  Returns false and raises the block's abort flag and the device status word when the
// phase does not complete in about a second; once the flag is up every later wait returns at once.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, uint32_t abort_flag, int* status) {
  if (mbar_try(bar, parity)) return true;
  if (flag_get(abort_flag)) return false;
  const long long t0 = clock64();
  for (uint32_t spin = 0; spin < kSpinLimit; ++spin) {
    if (mbar_try(bar, parity)) return true;
    if ((spin & 31u) == 31u) {
      if (flag_get(abort_flag)) return false;
      if (clock64() - t0 > kWaitCycles) break;
    }
  }
  flag_set(abort_flag);
  atomicOr(status, 1);
  return false;
}
// The same without the flag: only bounded in time, for the teardown after an abort.
__device__ __forceinline__ void mbar_wait_quiet(uint32_t bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try(bar, parity)) {
    if (clock64() - t0 > kWaitCycles) break;
  }
}

// 2-D box of a tensor map -> this block's shared memory (128-byte swizzle); completion counted in bytes on the barrier.
// The inner coordinate x is a multiple of 16 bytes; boxes that start past an edge read as zero.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
               "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar)
               : "memory");
}

__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

// 32 lanes x 32 columns: thread t receives columns 0..31 of lane base + t
__device__ __forceinline__ void tc_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}

// Operand tiles are 128-byte rows in the 128-byte swizzle (16-byte chunk c of row r at slot c ^ (r & 7)), as the TMA copy
// writes them.  K-major operand: a tile row is a row of the operand with 128 bytes of K; eight rows are 1024 bytes apart.
// MN-major operand: a tile row is one k with 64 consecutive 16-bit elements of the other axis; eight k are 1024 bytes
// apart (stride offset), the next 64 elements `lead` bytes away (leading offset).
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem_addr, uint32_t lead) {
  return (uint64_t)((smem_addr >> 4) & 0x3FFF) | ((uint64_t)((lead >> 4) & 0x3FFF) << 16) | ((uint64_t)(1024 >> 4) << 32) |
         ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t smem_addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr), "r"(rank));
  return r;
}
__device__ __forceinline__ uint4 ld_cluster_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared::cluster.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
// The sum over the cluster's blocks of four values at this offset of their shared memory, in rank order.  All loads are issued
// before the first is used: one round trip, not one a block.
template <bool INTEGER>
__device__ __forceinline__ void sum_over_cluster(uint32_t addr, uint32_t blocks, uint32_t (&v)[4]) {
  uint4 p[8];
#pragma unroll
  for (uint32_t q = 0; q < 8; ++q)
    if (q < blocks) p[q] = ld_cluster_v4(map_to_rank(addr, q));
  v[0] = p[0].x, v[1] = p[0].y, v[2] = p[0].z, v[3] = p[0].w;
#pragma unroll
  for (uint32_t q = 1; q < 8; ++q) {
    if (q >= blocks) break;
    const uint32_t e[4] = {p[q].x, p[q].y, p[q].z, p[q].w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = INTEGER ? v[j] + e[j] : __float_as_uint(__uint_as_float(v[j]) + __uint_as_float(e[j]));
  }
}
__device__ __forceinline__ uint4 ld_global_v4(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p) : "memory");
  return v;
}
__device__ __forceinline__ uint4 ld_shared_v4(uint32_t addr) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Two fp32 values -> two 16-bit values of the tensor's type, low half first.
__device__ __forceinline__ uint32_t pack16(float lo, float hi, bool bf16) {
  uint32_t r;
  if (bf16) {
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  } else {
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  }
  return r;
}
__device__ __forceinline__ float unpack16(uint32_t bits16, bool bf16) {
  return bf16 ? __uint_as_float(bits16 << 16) : __half2float(__ushort_as_half((unsigned short)bits16));
}
// sigmoid in fp32, of the exponential of -|x|, which does not overflow: far below zero the result is that exponential (as
// 1 / (1 + e^-x) the fast division returns 0 once 1 + e^-x passes 2^126, at -87).  The exponential is off by at most
// 2 + 1.173 |x| units of 2^-23: for x < 0 so is the result (2^-19 of it at -12, 2^-16 at -90), below the 16-bit rounding of what
// is made of it; for x > 0 that is divided by e^x.
__device__ __forceinline__ float sigmoid(float x) {
  const float e = __expf(-fabsf(x));
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(__fadd_rn(1.f, e)));   // of 1 to 2: nothing to flush
  return __fmul_rn(x < 0.f ? e : 1.f, r);
}

}  // namespace dense
