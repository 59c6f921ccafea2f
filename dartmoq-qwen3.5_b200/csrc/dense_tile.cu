// Dense products on the tensor cores, one 128-row output tile a cluster: the K axis is split over the cluster's blocks and
// their partial sums are joined through distributed shared memory, in rank order, so that a result does not depend on
// timing.
//
// A block multiplies its share of K steps (128 bytes of K each) into one TMEM accumulator: warp 0 brings the operand boxes in
// by TMA, warp 1 issues tcgen05.mma, warps 4-7 take the accumulator to shared memory (over the operand stages, which are
// idle by then); after a cluster barrier every block finishes 128 / splits rows of the tile.
// For products with too few tiles for pairs of SMs, which one long K would bind to a few of them: 257 x 1032 by K = 5456 13.0 us in 4
// parts, 32 unsplit, 31 in pairs; 1024 x 2048 by K = 16384 64 us in 2 parts at two blocks an SM (1.07 PFLOP/s), 77 in pairs.
#include "dense.cuh"

__device__ int g_dmoq_dense_status = 0;

namespace dense {
namespace {

constexpr int BN = 128;                                   // columns of a tile
constexpr int kStageBytes = 128 * 128 + BN * 128;
// Six operand stages where the blocks have an SM each, three where two share one: what is on its way into an SM is the same, and
// one block's products cover the other's start and end.
constexpr int kMostStages = 6;
constexpr int kPitch = BN * 4 + 16;                       // accumulator rows in shared memory: 16 bytes of padding against bank conflicts
constexpr int smem_bytes(int stages) { return 1024 + 256 + stages * kStageBytes; }
static_assert(128 * kPitch <= 3 * kStageBytes, "the accumulator rows lie over the operand stages");
static_assert(2 * (smem_bytes(3) + 1024) <= 228 * 1024, "two blocks an SM");

template <int KIND, bool AMN, bool BMN, int EPI>
__global__ void __launch_bounds__(256, 2) dense_tile_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a, int stages) {
  constexpr bool kDual = is_dual(EPI);
  constexpr int kCols = kDual ? BN / 2 : BN;              // output columns of the tile
  constexpr int kBK = KIND == KIND_I8 ? 128 : 64;         // elements of K in a step
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t bars = sb + stages * kStageBytes;
  auto stage_a = [&](uint32_t s) { return sb + s * kStageBytes; };
  auto stage_b = [&](uint32_t s) { return sb + s * kStageBytes + 128 * 128; };
  auto bar_full = [&](uint32_t s) { return bars + 8 * s; };
  auto bar_empty = [&](uint32_t s) { return bars + 64 + 8 * s; };
  const uint32_t bar_acc = bars + 128, tmem_slot = bars + 136, abort_flag = bars + 140;
  struct Ring {                                            // a position in the ring of stages and the parity of its use
    uint32_t s = 0, parity = 0;
    __device__ __forceinline__ void next(int stages) {
      if (++s == (uint32_t)stages) s = 0, parity ^= 1;
    }
  };

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t rank = cluster_rank(), splits = cluster_size();
  const int tiles_n = (a.N + kCols - 1) / kCols;
  const int tile = blockIdx.x / splits;
  const int m0 = tile / tiles_n * 128, n0 = tile % tiles_n * kCols;
  const int seg_steps = (a.K + kBK - 1) / kBK;
  const int steps = seg_steps * a.segs;
  const int it0 = (int)((long long)steps * rank / splits), it1 = (int)((long long)steps * (rank + 1) / splits);

  if (tid == 0) {
    for (int s = 0; s < stages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    mbar_init(bar_acc, 1);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(abort_flag), "r"(0) : "memory");
    mbar_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(BN));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  overlap_point();

  bool mine_plain = true;
  if (warp == 0) {
    if (lane == 0) {
      int done = 0;
      Ring at;
      for (int it = it0; it < it1; ++it, ++done, at.next(stages)) {
        const uint32_t s = at.s;
        if (done >= stages && !mbar_wait(bar_empty(s), at.parity ^ 1, abort_flag, &g_dmoq_dense_status)) break;
        const int seg = it >= seg_steps ? 1 : 0, k = (it - seg * seg_steps) * kBK;
        mbar_arrive_expect_tx(bar_full(s), kStageBytes);
        if (AMN) {
          tma_load(stage_a(s), &maps.a[seg], m0, k, bar_full(s));
          tma_load(stage_a(s) + 8192, &maps.a[seg], m0 + 64, k, bar_full(s));
        } else {
          tma_load(stage_a(s), &maps.a[seg], k, m0, bar_full(s));
        }
        if (BMN) {
#pragma unroll
          for (int j = 0; j < BN / 64; ++j) tma_load(stage_b(s) + 8192 * j, &maps.b[seg], n0 + 64 * j, k, bar_full(s));
        } else if (kDual) {
          tma_load(stage_b(s), &maps.b[0], k, n0, bar_full(s));
          tma_load(stage_b(s) + BN * 64, &maps.b[1], k, n0, bar_full(s));
        } else {
          tma_load(stage_b(s), &maps.b[seg], k, n0, bar_full(s));
        }
      }
      // nothing may still be on its way into this block's shared memory when it is reused or the block ends (matters after an abort)
      for (int j = done > stages ? done - stages : 0; j < done; ++j) mbar_wait_quiet(bar_full(j % stages), (j / stages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t shape = ((uint32_t)(BN >> 3) << 17) | (8u << 24);
      const uint32_t type = a.bf16 ? 1u : 0u;
      const uint32_t idesc = KIND == KIND_I8 ? (2u << 4) | (1u << 7) | (1u << 10) | shape
                                             : (1u << 4) | (type << 7) | (type << 10) | (AMN ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u) | shape;
      // 32 bytes of K an instruction: 32 bytes along a K-major row, sixteen 128-byte rows of an MN-major tile
      constexpr uint32_t step_a = AMN ? 128 : 2, step_b = BMN ? 128 : 2;
      uint32_t ready = 0;
      Ring at;
      for (int done = 0; done < it1 - it0; ++done) {
        const uint32_t s = at.s;
        if (!ready && !mbar_wait(bar_full(s), at.parity, abort_flag, &g_dmoq_dense_status)) break;
        tc_fence_after();
        at.next(stages);
        ready = mbar_peek(bar_full(at.s), at.parity);      // used after this step's products
        const uint64_t da = operand_desc(stage_a(s), AMN ? 8192 : 16), db = operand_desc(stage_b(s), BMN ? 8192 : 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t acc = (done > 0 || k > 0) ? 1u : 0u;
          if (KIND == KIND_I8) {
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                         "l"(da + step_a * k), "l"(db + step_b * k), "r"(idesc), "r"(acc)
                         : "memory");
          } else {
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                         "l"(da + step_a * k), "l"(db + step_b * k), "r"(idesc), "r"(acc)
                         : "memory");
          }
        }
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_empty(s)) : "memory");
      }
      asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_acc) : "memory");
    }
  } else if (warp < 4) {
    if (KIND == KIND_I8) mine_plain = plain_tile(a, m0, 128, n0, kCols, kDual, tid - 64, 64);
  } else {
    mbar_wait(bar_acc, 0, abort_flag, &g_dmoq_dense_status);
    if (flag_get(abort_flag)) mbar_wait_quiet(bar_acc, 0);
    tc_fence_after();
    const int w = warp - 4;
    const uint32_t row = sb + (uint32_t)(w * 32 + lane) * kPitch;
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
      uint32_t v[32];
      tc_ld32(tmem + ((uint32_t)(w * 32) << 16) + c, v);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; i += 4) st_shared_v4(row + (c + i) * 4, v[i], v[i + 1], v[i + 2], v[i + 3]);
    }
    tc_fence_before();
  }
  __syncwarp();
  const bool plain = __syncthreads_and(mine_plain);
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(BN));
  }
  if (splits > 1) cluster_sync();

  // join and finish: this block's rows of the tile
  finish_rows<KIND, EPI, kCols>(a, sb, kPitch, 128 * rank / splits, 128 * (rank + 1) / splits, m0, n0, splits, tid, plain);
  if (splits > 1) cluster_sync();   // a block's shared memory lives until the others have read it
}

}  // namespace

// Blocks of this kernel that run at once in clusters of `splits` (a power of two up to 8), an SM each: clusters do not fill
// every processing cluster of the device, so this is less than there are SMs.  With three stages twice as many fit.
int tile_blocks_at_once(int splits) {
  static std::atomic<int> known[64][4] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return dmoq_sm_count();
  int log = 0;
  while ((1 << log) < splits) ++log;
  int n = known[dev][log];
  if (n == 0) {
    auto* kernel = dense_tile_kernel<KIND_16, false, false, EPI_OUT>;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(splits);
    cfg.blockDim = dim3(256);
    cfg.dynamicSmemBytes = smem_bytes(kMostStages);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = splits;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    int clusters = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kMostStages)) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&clusters, kernel, &cfg) != cudaSuccess || clusters < 1) {
      (void)cudaGetLastError();
      clusters = dmoq_sm_count() / splits;
    }
    known[dev][log] = n = clusters * splits;
  }
  return n;
}

namespace {

template <int KIND, bool AMN, bool BMN, int EPI>
int launch(const Maps& maps, const Args& a, int splits, cudaStream_t s) {
  static DmoqOncePerDevice once;
  std::atomic<bool>* configured = once.slot();
  if (configured == nullptr) return DMOQ_EDEVICE;
  auto* kernel = dense_tile_kernel<KIND, AMN, BMN, EPI>;
  if (!*configured) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes(kMostStages)) != cudaSuccess) return DMOQ_ELAUNCH;
    *configured = true;
  }
  constexpr int kCols = is_dual(EPI) ? BN / 2 : BN;
  const long long blocks = (long long)dmoq_ceil_div(a.M, 128) * dmoq_ceil_div(a.N, kCols) * splits;
  if (blocks > 0x7fffffffLL) return DMOQ_ESIZE;
  const int stages = blocks <= tile_blocks_at_once(splits) ? kMostStages : 3;
  return launch_overlapped(kernel, (unsigned)blocks, 256, smem_bytes(stages), splits, s, maps, a, stages);
}

}  // namespace

int tile_product(int kind, bool a_mn, bool b_mn, int epi, const Maps& maps, const Args& a, int splits, cudaStream_t s) {
  const int key = kind * 1000 + a_mn * 200 + b_mn * 100 + epi;
  switch (key) {
    case EPI_OUT: return launch<KIND_16, false, false, EPI_OUT>(maps, a, splits, s);
    case EPI_SILU: return launch<KIND_16, false, false, EPI_SILU>(maps, a, splits, s);
    case EPI_SILU_SAVE: return launch<KIND_16, false, false, EPI_SILU_SAVE>(maps, a, splits, s);
    case 100 + EPI_OUT: return launch<KIND_16, false, true, EPI_OUT>(maps, a, splits, s);
    case 100 + EPI_GRAD: return launch<KIND_16, false, true, EPI_GRAD>(maps, a, splits, s);
    case 300 + EPI_OUT: return launch<KIND_16, true, true, EPI_OUT>(maps, a, splits, s);
    case 1000 + EPI_SCALE: return launch<KIND_I8, false, false, EPI_SCALE>(maps, a, splits, s);
    case 1000 + EPI_SILU: return launch<KIND_I8, false, false, EPI_SILU>(maps, a, splits, s);
    default: return DMOQ_EINVAL;
  }
}

}  // namespace dense

int dmoq_dense_status(int* out) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_dmoq_dense_status, sizeof(int)) != cudaSuccess) return DMOQ_EDEVICE;
  int w = 0, m = 0;
  int rc = dmoq_dense_pair_status(&w);
  if (rc == DMOQ_OK) rc = dmoq_dense_mid_status(&m);
  if (rc != DMOQ_OK) return rc;
  *out = v | w | m;
  return DMOQ_OK;
}
