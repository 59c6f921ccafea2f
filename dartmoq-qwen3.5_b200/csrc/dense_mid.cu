// Dense products of 9 to 256 tokens: bound by reading the weights once.
//
// The weights are the M operand of tcgen05.mma (128 rows a block; when dual 64 rows of either weight) and the tokens its N
// operand, padded to 32, 64, 128 or 256, so that most of what a block brings in is weights.  Up to 128 tokens its ring of
// operand stages takes less than half of the shared memory: two blocks share an SM, and one streams while the other starts or
// finishes.  Where
// there are few tiles the K axis is split over a cluster's blocks, whose sums are joined through distributed shared memory
// in rank order.  The accumulator (a lane an output, a column a token) passes through shared memory, a row a token.
// 64 tokens, 16 bits: 13824 x 5120 twice 51 us = 5.6 TB/s of weights (86 % of the measured bandwidth), and with 5120 x 13824 in 4
// parts behind it 78 us (40 tiles of that: their start, join and end show).  8 bits: 13824 x 5120 13 us.
#include "dense.cuh"

__device__ int g_dmoq_dense_mid_status = 0;

namespace dense {
namespace {

template <int BN>
struct MidCfg {
  static constexpr int kStageBytes = 128 * 128 + BN * 128;
  static constexpr int kStages = BN == 32 ? 5 : BN == 128 ? 3 : 4;
  static constexpr int kPitch = 128 * 4;                  // sums of a token
  static constexpr int kBar = kStages * kStageBytes;
  static constexpr int kSmem = kBar + 256 + 1024;
  static_assert(BN * kPitch <= kBar, "the sums lie over the operand stages");
  static constexpr int kBlocks = BN == 256 ? 1 : 2;        // of an SM
  static_assert(kBlocks * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

template <int KIND, int EPI, int BN>
__global__ void __launch_bounds__(256, MidCfg<BN>::kBlocks) dense_mid_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Args a) {
  using C = MidCfg<BN>;
  constexpr bool kDual = is_dual(EPI);
  constexpr int kRows = kDual ? 64 : 128;                  // outputs of a tile
  constexpr int kBK = KIND == KIND_I8 ? 128 : 64;
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
  auto stage_w = [&](uint32_t s) { return sb + s * C::kStageBytes; };
  auto stage_x = [&](uint32_t s) { return sb + s * C::kStageBytes + 128 * 128; };
  auto bar_full = [&](uint32_t s) { return sb + C::kBar + 8 * s; };
  auto bar_empty = [&](uint32_t s) { return sb + C::kBar + 64 + 8 * s; };
  const uint32_t bar_acc = sb + C::kBar + 128, tmem_slot = sb + C::kBar + 136, abort_flag = sb + C::kBar + 140;
  int* status = &g_dmoq_dense_mid_status;

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t rank = cluster_rank(), splits = cluster_size();
  const int n0 = (int)(blockIdx.x / splits) * kRows;
  const int steps = (a.K + kBK - 1) / kBK;
  const int it0 = (int)((long long)steps * rank / splits), it1 = (int)((long long)steps * (rank + 1) / splits);

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
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
      for (int it = it0; it < it1; ++it, ++done) {
        const uint32_t s = done % kStages;
        if (done >= kStages && !mbar_wait(bar_empty(s), (done / kStages - 1) & 1, abort_flag, status)) break;
        mbar_arrive_expect_tx(bar_full(s), C::kStageBytes);
        const int k = it * kBK;
        tma_load(stage_w(s), &maps.a[0], k, n0, bar_full(s));
        if (kDual) tma_load(stage_w(s) + 64 * 128, &maps.a[1], k, n0, bar_full(s));
        tma_load(stage_x(s), &maps.b[0], k, 0, bar_full(s));
      }
      // nothing may still be on its way into this block's shared memory when it is reused or the block ends (matters after an abort)
      for (int j = done > kStages ? done - kStages : 0; j < done; ++j) mbar_wait_quiet(bar_full(j % kStages), (j / kStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t shape = ((uint32_t)(BN >> 3) << 17) | (8u << 24);
      const uint32_t type = a.bf16 ? 1u : 0u;
      const uint32_t idesc = KIND == KIND_I8 ? (2u << 4) | (1u << 7) | (1u << 10) | shape : (1u << 4) | (type << 7) | (type << 10) | shape;
      uint32_t ready = 0;
      for (int done = 0; done < it1 - it0; ++done) {
        const uint32_t s = done % kStages;
        if (!ready && !mbar_wait(bar_full(s), (done / kStages) & 1, abort_flag, status)) break;
        tc_fence_after();
        ready = mbar_peek(bar_full((done + 1) % kStages), ((done + 1) / kStages) & 1);   // used after this step's products
        const uint64_t da = operand_desc(stage_w(s), 16), db = operand_desc(stage_x(s), 16);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t acc = (done > 0 || k > 0) ? 1u : 0u;
          if (KIND == KIND_I8) {
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                         "l"(da + 2 * k), "l"(db + 2 * k), "r"(idesc), "r"(acc)
                         : "memory");
          } else {
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem),
                         "l"(da + 2 * k), "l"(db + 2 * k), "r"(idesc), "r"(acc)
                         : "memory");
          }
        }
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_empty(s)) : "memory");
      }
      asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_acc) : "memory");
    }
  } else if (warp < 4) {
    if (KIND == KIND_I8) mine_plain = plain_tile(a, 0, a.M, n0, kRows, kDual, tid - 64, 64);
  } else {
    mbar_wait(bar_acc, 0, abort_flag, status);
    if (flag_get(abort_flag)) mbar_wait_quiet(bar_acc, 0);
    tc_fence_after();
    const int w = warp - 4;
    const uint32_t out = sb + (uint32_t)(w * 32 + lane) * 4;
#pragma unroll 1
    for (int c = 0; c < BN; c += 32) {
      uint32_t v[32];
      tc_ld32(tmem + ((uint32_t)(w * 32) << 16) + c, v);
      tc_wait_ld();
#pragma unroll
      for (int i = 0; i < 32; ++i) asm volatile("st.shared.u32 [%0], %1;" ::"r"(out + (c + i) * C::kPitch), "r"(v[i]) : "memory");
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

  // join and finish: this block's share of the tokens
  finish_rows<KIND, EPI, kRows>(a, sb, C::kPitch, (int)((long long)a.M * rank / splits), (int)((long long)a.M * (rank + 1) / splits), 0, n0,
                                splits, tid, plain);
  if (splits > 1) cluster_sync();   // a block's shared memory lives until the others have read it
}

template <int KIND, int EPI, int BN>
int launch(const Maps& maps, const Args& a, int splits, cudaStream_t s) {
  using C = MidCfg<BN>;
  static DmoqOncePerDevice once;
  std::atomic<bool>* configured = once.slot();
  if (configured == nullptr) return DMOQ_EDEVICE;
  auto* kernel = dense_mid_kernel<KIND, EPI, BN>;
  if (!*configured) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) return DMOQ_ELAUNCH;
    *configured = true;
  }
  const long long blocks = (long long)dmoq_ceil_div(a.N, is_dual(EPI) ? 64 : 128) * splits;
  if (blocks > 0x7fffffffLL) return DMOQ_ESIZE;
  return launch_overlapped(kernel, (unsigned)blocks, 256, C::kSmem, splits, s, maps, a);
}

template <int KIND, int EPI>
int launch_tokens(const Maps& maps, const Args& a, int splits, cudaStream_t s) {
  if (a.M <= 32) return launch<KIND, EPI, 32>(maps, a, splits, s);
  if (a.M <= 64) return launch<KIND, EPI, 64>(maps, a, splits, s);
  if (a.M <= 128) return launch<KIND, EPI, 128>(maps, a, splits, s);
  return launch<KIND, EPI, 256>(maps, a, splits, s);
}

}  // namespace

int mid_token_box(int tokens) { return tokens <= 32 ? 32 : tokens <= 64 ? 64 : tokens <= 128 ? 128 : 256; }

// maps.a: the weights in boxes of 128 rows (dual: both, of 64), maps.b[0]: the tokens in one box of mid_token_box rows.
int mid_product(int kind, int epi, const Maps& maps, const Args& a, int splits, cudaStream_t s) {
  switch (kind * 1000 + epi) {
    case EPI_OUT: return launch_tokens<KIND_16, EPI_OUT>(maps, a, splits, s);
    case EPI_SILU: return launch_tokens<KIND_16, EPI_SILU>(maps, a, splits, s);
    case EPI_SILU_SAVE: return launch_tokens<KIND_16, EPI_SILU_SAVE>(maps, a, splits, s);
    case 1000 + EPI_SCALE: return launch_tokens<KIND_I8, EPI_SCALE>(maps, a, splits, s);
    case 1000 + EPI_SILU: return launch_tokens<KIND_I8, EPI_SILU>(maps, a, splits, s);
    default: return DMOQ_EINVAL;
  }
}

}  // namespace dense

int dmoq_dense_mid_status(int* out) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_dmoq_dense_mid_status, sizeof(int)) != cudaSuccess) return DMOQ_EDEVICE;
  *out = v;
  return DMOQ_OK;
}
