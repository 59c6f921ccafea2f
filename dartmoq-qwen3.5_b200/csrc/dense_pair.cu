// Dense products on the tensor cores, large outputs: a persistent pair of blocks (two SMs, tcgen05 cta_group::2) walks 256 x 256
// output tiles.
//
// Each block of a pair holds 128 of the tile's rows: it loads its own 128 rows of A and one half of the tile's 256 columns of B
// (when dual: the first block the gate's 128 columns, the second the up projection's), the leader's MMA thread multiplies both
// halves, and each block finds its 128 rows x 256 columns of sums in its own TMEM.  Two such accumulators fill TMEM, so the
// epilogue of a tile runs beside the products of the next one.  One launch may hold several products: the gradients of a
// block, whose tiles differ in length, share the SMs.
//   warp 0      loads the operands by TMA (six steps of 128 bytes of K ahead)
//   warp 1      issues tcgen05.mma (leader only)
//   warps 4-11  take the sums out of TMEM, finish them, and write 32 x 32 blocks out through shared memory (plain
//               stores of 64-byte rows: a TMA store costs each warp a proxy fence of about 500 cycles a block, which made the
//               epilogue the longer half of tiles with a short K)
// Bound by the tensor cores at the clock that the power limit leaves: 16384 x 4096 by K = 4096 in 8 bits 170 us = 3.2 Pop/s in a
// burst and 195 us = 2.8 Pop/s held for seconds (tensor pipe 89 % active), 8192 x 14336 twice by K = 4096 in bf16 with the saved
// planes 1.34 ms = 1.44 PFLOP/s in a burst.  A product of one round of tiles shows its epilogue: 8192 x 512 twice by K = 2048 with
// the saved planes takes 33 us, 10 of them for 34 MB of outputs.
// Pairs rather than single blocks: each SM reads half as much of B from shared memory and L2.
#include "dense.cuh"

#include <algorithm>

__device__ int g_dmoq_dense_pair_status = 0;

namespace dense {
namespace {

constexpr int kStages = 6;
constexpr int kStageBytes = 2 * 128 * 128;
constexpr int kEpiWarps = 8;
constexpr int kUnitBytes = 32 * 64;                       // 32 rows of 32 16-bit outputs on their way out
constexpr int kUnits = 2;                                 // per epilogue warp
constexpr int kUnitBase = kStages * kStageBytes;
constexpr int kBarBase = kUnitBase + kEpiWarps * kUnits * kUnitBytes;
constexpr int kSmem = kBarBase + 256 + 1024;
constexpr int kThreads = 32 * (4 + kEpiWarps);
constexpr int kGroupM = 8;                                // tile rows that are walked together, so that both operands are shared in L2

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t leader_bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3}], [%4];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(leader_bar)
      : "memory");
}
// completes on the barrier at this address in both blocks of the pair
__device__ __forceinline__ void commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar),
               "h"((uint16_t)3)
               : "memory");
}

// NP products of one launch.  Their tiles come in two lengths (steps of K): first the long ones go round the pairs, then the
// pairs that got one fewer take `fill` short tiles each, which is about as long, and the rest of the short ones goes round.
template <int NP>
struct Work {
  Maps maps[NP];
  Args p[NP];
  int a_mn[NP];
  int tiles[NP];             // 256-row tiles of each product
  int n_long;                // products 0 .. n_long - 1 have the long tiles
  int long_tiles, fill;
};

// AMN is that of a single product; a group's products say it themselves.
template <int KIND, bool AMN, bool BMN, int EPI, int NP>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1) dense_pair_kernel(const __grid_constant__ Work<NP> work) {
  constexpr bool kDual = is_dual(EPI);
  constexpr int kCols = kDual ? 128 : 256;                 // output columns of a tile
  constexpr int kBK = KIND == KIND_I8 ? 128 : 64;
  extern __shared__ uint8_t smem_raw[];
  uint32_t sb = (smem_u32(smem_raw) + 1023u) & ~1023u;
  asm volatile("" : "+r"(sb));
  auto stage_a = [&](uint32_t s) { return sb + s * kStageBytes; };
  auto stage_b = [&](uint32_t s) { return sb + s * kStageBytes + 128 * 128; };
  auto bar_full = [&](uint32_t s) { return sb + kBarBase + 8 * s; };
  auto bar_empty = [&](uint32_t s) { return sb + kBarBase + 64 + 8 * s; };
  auto bar_acc_full = [&](uint32_t b) { return sb + kBarBase + 128 + 8 * b; };
  auto bar_acc_empty = [&](uint32_t b) { return sb + kBarBase + 144 + 8 * b; };
  const uint32_t bar_drain = sb + kBarBase + 160, tmem_slot = sb + kBarBase + 168, abort_flag = sb + kBarBase + 172;
  int* status = &g_dmoq_dense_pair_status;

  const int tid = threadIdx.x, lane = tid & 31, warp = __shfl_sync(0xffffffffu, tid >> 5, 0);
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  struct Tile {
    int q, m0, n0, seg_steps, steps;                       // product, first row of this block, first column, steps of K
  };
  auto next_tile = [&](int i, Tile& o) {                   // the pair's i-th tile; false after the last one
    int t = pair + i * pairs, q = 0;
    if (NP > 1) {
      const int ahead = work.long_tiles % pairs;           // pairs that have one long tile more than the others
      const int mine = work.long_tiles / pairs + (pair < ahead ? 1 : 0);
      int last = work.n_long;
      if (i >= mine) {
        const int j = i - mine, fill = pair < ahead ? 0 : work.fill, others = pairs - ahead;
        t = j < fill ? j * others + pair - ahead : work.fill * others + (j - fill) * pairs + pair;
        q = work.n_long;
        last = NP;
      }
      while (q < last && t >= work.tiles[q]) t -= work.tiles[q++];
      if (q >= last) return false;
    } else if (t >= work.tiles[0]) {
      return false;
    }
    const Args& a = work.p[q];
    const int tiles_n = (a.N + kCols - 1) / kCols, tiles_m = (a.M + 255) / 256;
    // columns of up to kGroupM tile rows, one tile column after the other
    const int group = t / (kGroupM * tiles_n), first = group * kGroupM;
    const int height = min(kGroupM, tiles_m - first), local = t - group * kGroupM * tiles_n;
    o.q = q;
    o.m0 = (first + local % height) * 256 + (int)rank * 128;
    o.n0 = local / height * kCols;
    o.seg_steps = (a.K + kBK - 1) / kBK;
    o.steps = o.seg_steps * a.segs;
    return true;
  };

  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_full(s), 1);
      mbar_init(bar_empty(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(bar_acc_full(b), 1);
      mbar_init(bar_acc_empty(b), 2 * kEpiWarps);
    }
    mbar_init(bar_drain, 1);
    asm volatile("st.shared.u32 [%0], %1;" ::"r"(abort_flag), "r"(0) : "memory");
    mbar_init_fence();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(tmem_slot), "r"(512));
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::);
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  tc_fence_after();
  uint32_t tmem;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
  overlap_point();

  if (warp == 0) {
    if (lane == 0) {
      uint32_t done = 0;
      bool ok = true;
      Tile w;
      for (int i = 0; ok && next_tile(i, w); ++i) {
        const Maps& maps = work.maps[w.q];
        const bool a_mn = NP > 1 ? work.a_mn[w.q] != 0 : AMN;
        const int m0 = w.m0, n0 = w.n0, seg_steps = w.seg_steps;
        for (int it = 0; it < w.steps; ++it, ++done) {
          const uint32_t s = done % kStages;
          if (done >= kStages && !mbar_wait(bar_empty(s), (done / kStages - 1) & 1, abort_flag, status)) {
            ok = false;
            break;
          }
          const uint32_t full = map_to_rank(bar_full(s), 0);
          if (rank == 0) mbar_arrive_expect_tx(bar_full(s), 2 * kStageBytes);
          const int seg = it >= seg_steps ? 1 : 0, k = (it - seg * seg_steps) * kBK;
          if (a_mn) {
            tma_load_pair(stage_a(s), &maps.a[seg], m0, k, full);
            tma_load_pair(stage_a(s) + 8192, &maps.a[seg], m0 + 64, k, full);
          } else {
            tma_load_pair(stage_a(s), &maps.a[seg], k, m0, full);
          }
          const int nb = kDual ? n0 : n0 + (int)rank * 128;
          const CUtensorMap* mb = &maps.b[kDual ? (int)rank : seg];
          if (BMN) {
            tma_load_pair(stage_b(s), mb, nb, k, full);
            tma_load_pair(stage_b(s) + 8192, mb, nb + 64, k, full);
          } else {
            tma_load_pair(stage_b(s), mb, k, nb, full);
          }
        }
      }
      // after an abort copies may still be on their way into either block; the leader's barriers count both blocks' bytes
      if (!ok && rank == 0)
        for (uint32_t j = done > kStages ? done - kStages : 0u; j < done; ++j) mbar_wait_quiet(bar_full(j % kStages), (j / kStages) & 1);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr uint32_t shape = (32u << 17) | (16u << 24);
      const uint32_t type = work.p[0].bf16 ? 1u : 0u;
      constexpr uint32_t step_b = BMN ? 128 : 2;
      uint32_t done = 0, ready = 0;
      bool ok = true;
      Tile w;
      for (int i = 0; ok && next_tile(i, w); ++i) {
        const bool a_mn = NP > 1 ? work.a_mn[w.q] != 0 : AMN;
        const uint32_t step_a = a_mn ? 128 : 2, lead_a = a_mn ? 8192 : 16;
        const uint32_t idesc = KIND == KIND_I8 ? (2u << 4) | (1u << 7) | (1u << 10) | shape
                                               : (1u << 4) | (type << 7) | (type << 10) | (a_mn ? 1u << 15 : 0u) | (BMN ? 1u << 16 : 0u) | shape;
        const uint32_t b = i & 1, d = tmem + b * 256;
        if (i >= 2 && !mbar_wait(bar_acc_empty(b), (i / 2 - 1) & 1, abort_flag, status)) {
          ok = false;
          break;
        }
        tc_fence_after();
        for (int it = 0; it < w.steps; ++it, ++done) {
          const uint32_t s = done % kStages;
          if (!ready && !mbar_wait(bar_full(s), (done / kStages) & 1, abort_flag, status)) {
            ok = false;
            break;
          }
          tc_fence_after();
          // look at the next step now and use the answer after this one's products: the barrier's latency (about 110 cycles of
          // the 512 that a step takes) would otherwise stand between them
          ready = mbar_peek(bar_full((done + 1) % kStages), ((done + 1) / kStages) & 1);
          const uint64_t da = operand_desc(stage_a(s), lead_a), db = operand_desc(stage_b(s), BMN ? 8192 : 16);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t acc = (it > 0 || k > 0) ? 1u : 0u;
            if (KIND == KIND_I8) {
              asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                           "l"(da + step_a * k), "l"(db + step_b * k), "r"(idesc), "r"(acc)
                           : "memory");
            } else {
              asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                           "l"(da + step_a * k), "l"(db + step_b * k), "r"(idesc), "r"(acc)
                           : "memory");
            }
          }
          commit_pair(bar_empty(s));
        }
        if (ok) commit_pair(bar_acc_full(b));
      }
      if (!ok) {   // no product may still read shared memory when the blocks end
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar_drain) : "memory");
        mbar_wait_quiet(bar_drain, 0);
      }
    }
  } else if (warp >= 4) {
    const int e = warp - 4, quarter = e & 3, side = e >> 2;
    const uint32_t units = sb + kUnitBase + e * (kUnits * kUnitBytes);
    uint32_t n_out = 0;
    Tile at_tile;
    for (int i = 0; next_tile(i, at_tile); ++i) {
      const Args& a = work.p[at_tile.q];
      const int m0 = at_tile.m0, n0 = at_tile.n0;
      const uint32_t b = i & 1;
      const int row0 = m0 + quarter * 32;
      const long long row = row0 + lane;
      const float sa = KIND == KIND_I8 && row < a.M ? a.a_scale[row] : 0.f;
      // The gradient's planes are loaded a block ahead in whole 64-byte row pieces (four lanes a row; a row a lane would touch 32
      // lines an instruction) and turned into a row a lane through shared memory, like the outputs on their way out.
      uint4 in[3][4];
      auto load_planes = [&](int col0) {
#pragma unroll
        for (int p = 0; p < 3; ++p)
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = row0 + 8 * r + (lane >> 2), col = col0 + 8 * (lane & 3);   // rows are whole groups of eight elements
            in[p][r] = at < a.M && col < a.N ? ld_global_v4(a.in[p] + at * a.ld_in + col) : make_uint4(0u, 0u, 0u, 0u);
          }
      };
      if (EPI == EPI_GRAD) load_planes(n0 + side * 128);
      if (!mbar_wait(bar_acc_full(b), (i / 2) & 1, abort_flag, status)) break;
      tc_fence_after();
      const uint32_t acc = tmem + ((uint32_t)(quarter * 32) << 16) + b * 256;
      constexpr int kBlocks = kDual ? 2 : 4;               // 32-column blocks of this warp
#pragma unroll 1
      for (int u = 0; u < kBlocks; ++u) {
        const int c = side * (kBlocks * 32) + u * 32, col0 = n0 + c;
        uint32_t v[32], w[32];
        tc_ld32(acc + c, v);
        if (kDual) tc_ld32(acc + 128 + c, w);
        uint4 plane[3][4];                                 // of this lane's row
        if (EPI == EPI_GRAD) {
#pragma unroll
          for (int p = 0; p < 3; ++p, ++n_out) {
            const uint32_t unit = units + (n_out % kUnits) * kUnitBytes;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = 8 * r + (lane >> 2);
              st_shared_v4(unit + at * 64 + (((lane & 3) ^ ((at >> 1) & 3)) << 4), in[p][r].x, in[p][r].y, in[p][r].z, in[p][r].w);
            }
            __syncwarp();
#pragma unroll
            for (int j = 0; j < 4; ++j) plane[p][j] = ld_shared_v4(unit + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4));
          }
          if (u + 1 < kBlocks) load_planes(col0 + 32);
        }
        float sc0 = 1.f, sc1 = 1.f, bias = 0.f;            // of column col0 + lane
        if (KIND == KIND_I8 && col0 + lane < a.N) {
          sc0 = a.b_scale[0][col0 + lane];
          if (kDual) sc1 = a.b_scale[1][col0 + lane];
          if (EPI == EPI_SCALE && a.bias) bias = unpack16(a.bias[col0 + lane], a.bf16);
        }
        tc_wait_ld();
        if (u == kBlocks - 1) {                            // the sums are in registers: the accumulator goes back to the leader
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            const uint32_t remote = map_to_rank(bar_acc_empty(b), 0);
            // block scope: what is handed over are TMEM columns whose loads have completed; at cluster scope the release would
            // wait for this warp's outstanding global stores
            asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(remote) : "memory");
          }
        }
        if (KIND == KIND_I8) {                             // sums -> values; one look at all of the block's scales (see scaled)
          auto values = [&](auto&& scale) {
#pragma unroll
            for (int q = 0; q < 32; ++q) {
              v[q] = __float_as_uint(scale(v[q], sa, __shfl_sync(0xffffffffu, sc0, q)));
              if (kDual) w[q] = __float_as_uint(scale(w[q], sa, __shfl_sync(0xffffffffu, sc1, q)));
            }
          };
          if (__all_sync(0xffffffffu, plain_scale(sa) && plain_scale(sc0) && plain_scale(sc1)))
            values([](uint32_t sum, float s, float r) { return scaled_plain(sum, s, r); });
          else
            values([](uint32_t sum, float s, float r) { return scaled(sum, s, r); });
        }
        uint32_t o[outputs_of(EPI)][16];
#pragma unroll
        for (int j = 0; j < 16; ++j) {
          float x[2], y[2];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const int q = 2 * j + h;
            x[h] = __uint_as_float(v[q]);
            if (kDual) y[h] = __uint_as_float(w[q]);
            if (EPI == EPI_SCALE && a.bias) x[h] = __fadd_rn(x[h], __shfl_sync(0xffffffffu, bias, q));
          }
          if (EPI == EPI_OUT || EPI == EPI_SCALE) {
            o[0][j] = pack16(x[0], x[1], a.bf16);
          } else if (EPI == EPI_SILU) {
            o[0][j] = pack16(gated(x[0], y[0]), gated(x[1], y[1]), a.bf16);
          } else if (EPI == EPI_SILU_SAVE) {
            float si[2], sl[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const float s = sigmoid(x[h]);
              si[h] = __fmul_rn(x[h], s);
              sl[h] = slope_of(s, si[h], y[h]);
            }
            o[0][j] = pack16(si[0] * y[0], si[1] * y[1], a.bf16);
            o[1 % outputs_of(EPI)][j] = (__float_as_uint(si[0]) >> 16) | (__float_as_uint(si[1]) & 0xffff0000u);
            o[2 % outputs_of(EPI)][j] = (__float_as_uint(sl[0]) >> 16) | (__float_as_uint(sl[1]) & 0xffff0000u);
            o[3 % outputs_of(EPI)][j] = saved_low(si[0], sl[0]) | (saved_low(si[1], sl[1]) << 16);
          } else {
            auto word = [&](int p) {
              const uint4 q = plane[p][j / 4];
              return (j & 3) == 0 ? q.x : (j & 3) == 1 ? q.y : (j & 3) == 2 ? q.z : q.w;
            };
            const uint32_t s2 = word(0), p2 = word(1), l2 = word(2);
            o[0][j] = pack16(x[0] * saved_slope(p2 & 0xffffu, l2 & 0xffffu), x[1] * saved_slope(p2 >> 16, l2 >> 16), a.bf16);
            o[1 % outputs_of(EPI)][j] = pack16(x[0] * saved_silu(s2 & 0xffffu, l2 & 0xffffu), x[1] * saved_silu(s2 >> 16, l2 >> 16), a.bf16);
          }
        }
        if (row0 >= a.M || col0 >= a.N) continue;
#pragma unroll
        for (int p = 0; p < outputs_of(EPI); ++p, ++n_out) {
          const uint32_t unit = units + (n_out % kUnits) * kUnitBytes;
          const uint32_t line = unit + lane * 64, swz = (lane >> 1) & 3;
#pragma unroll
          for (int j = 0; j < 4; ++j) st_shared_v4(line + ((j ^ swz) << 4), o[p][4 * j], o[p][4 * j + 1], o[p][4 * j + 2], o[p][4 * j + 3]);
          __syncwarp();                                    // also: what this unit held two outputs ago has been read
          if (a.vec) {
            const long long ld = EPI == EPI_SILU_SAVE && p > 0 ? a.ld_saved : a.ld_out;
            const int q = lane & 3, col = col0 + 8 * q;    // 16 bytes a thread: eight rows of 64 bytes an instruction
            uint16_t* dst = a.out[p] + (row0 + (lane >> 2)) * ld + col;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = 8 * r + (lane >> 2);
              const uint4 val = ld_shared_v4(unit + at * 64 + ((q ^ ((at >> 1) & 3)) << 4));
              if (row0 + at < a.M && col < a.N) *reinterpret_cast<uint4*>(dst + 8 * r * ld) = val;
            }
          } else {                                         // rows that are not 16-byte aligned: 64-byte runs of a row at a time
            for (int r = 0; r < 32 && row0 + r < a.M; ++r) {
              const uint32_t at = unit + r * 64 + ((((uint32_t)lane >> 3) ^ ((r >> 1) & 3)) << 4) + (lane & 7) * 2;
              uint16_t val;
              asm volatile("ld.shared.u16 %0, [%1];" : "=h"(val) : "r"(at) : "memory");
              if (col0 + lane < a.N) a.out[p][(row0 + r) * a.ld_out + col0 + lane] = val;
            }
          }
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync();
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
  }
}

template <int KIND, bool AMN, bool BMN, int EPI, int NP>
int launch(Work<NP>& work, cudaStream_t s) {
  static DmoqOncePerDevice once;
  std::atomic<bool>* configured = once.slot();
  if (configured == nullptr) return DMOQ_EDEVICE;
  auto* kernel = dense_pair_kernel<KIND, AMN, BMN, EPI, NP>;
  if (!*configured) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return DMOQ_ELAUNCH;
    *configured = true;
  }
  constexpr int kCols = is_dual(EPI) ? 128 : 256;
  long long tiles = 0;
  for (int q = 0; q < NP; ++q) {
    const long long t = (long long)dmoq_ceil_div(work.p[q].M, 256) * dmoq_ceil_div(work.p[q].N, kCols);
    tiles += t;
    if (tiles > 0x3fffffffLL) return DMOQ_ESIZE;
    work.tiles[q] = (int)t;
  }
  const int pairs = (int)std::min<long long>(tiles, dmoq_sm_count() / 2);
  if (NP > 1) {
    auto steps = [&](int q) { return (long long)dmoq_ceil_div(work.p[q].K, 64) * work.p[q].segs; };
    work.long_tiles = 0;
    for (int q = 0; q < work.n_long; ++q) work.long_tiles += work.tiles[q];
    const long long shorts = tiles - work.long_tiles;
    const int ahead = work.long_tiles % pairs;
    work.fill = ahead == 0 || shorts == 0 ? 0 : (int)std::min<long long>(steps(0) / steps(work.n_long), shorts / (pairs - ahead));
  }
  return launch_overlapped(kernel, 2 * pairs, kThreads, kSmem, 0, s, work);
}

template <int KIND, bool AMN, bool BMN, int EPI>
int launch1(const Maps& maps, const Args& a, cudaStream_t s) {
  Work<1> w{};
  w.maps[0] = maps;
  w.p[0] = a;
  return launch<KIND, AMN, BMN, EPI, 1>(w, s);
}

}  // namespace

int pair_product(int kind, bool a_mn, bool b_mn, int epi, const Maps& maps, const Args& a, cudaStream_t s) {
  const int key = kind * 1000 + a_mn * 200 + b_mn * 100 + epi;
  switch (key) {
    case EPI_OUT: return launch1<KIND_16, false, false, EPI_OUT>(maps, a, s);
    case EPI_SILU: return launch1<KIND_16, false, false, EPI_SILU>(maps, a, s);
    case EPI_SILU_SAVE: return launch1<KIND_16, false, false, EPI_SILU_SAVE>(maps, a, s);
    case 100 + EPI_OUT: return launch1<KIND_16, false, true, EPI_OUT>(maps, a, s);
    case 100 + EPI_GRAD: return launch1<KIND_16, false, true, EPI_GRAD>(maps, a, s);
    case 300 + EPI_OUT: return launch1<KIND_16, true, true, EPI_OUT>(maps, a, s);
    case 1000 + EPI_SCALE: return launch1<KIND_I8, false, false, EPI_SCALE>(maps, a, s);
    case 1000 + EPI_SILU: return launch1<KIND_I8, false, false, EPI_SILU>(maps, a, s);
    default: return DMOQ_EINVAL;
  }
}

// Two or three 16-bit products with MN-major B in one launch, ordered so that the first n_long have the longer tiles.
int pair_group(const Maps* maps, const Args* p, const bool* a_mn, int n, int n_long, cudaStream_t s) {
  Work<3> w{};
  for (int q = 0; q < n; ++q) {
    w.maps[q] = maps[q];
    w.p[q] = p[q];
    w.a_mn[q] = a_mn[q];
  }
  w.n_long = n_long;
  return launch<KIND_16, false, true, EPI_OUT, 3>(w, s);
}

}  // namespace dense

int dmoq_dense_pair_status(int* out) {
  int v = 0;
  if (cudaMemcpyFromSymbol(&v, g_dmoq_dense_pair_status, sizeof(int)) != cudaSuccess) return DMOQ_EDEVICE;
  *out = v;
  return DMOQ_OK;
}
