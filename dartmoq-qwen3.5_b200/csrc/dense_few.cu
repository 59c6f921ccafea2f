// Dense products of a few tokens (T <= 16): bound by reading the weights once, and below a few megabytes by latency.
//
// The weights are the M operand of warp-level MMAs, 16 rows a block (when dual: eight rows of either weight, so that a thread
// ends with the gate and the up value of the same output), and go from global memory straight to registers.  A thread's 16
// bytes of a row hold consecutive k and feed two MMA steps: the order of k inside a step is permuted the same way for both
// operands, which leaves the sums as they are.  The eight warps split K in steps of 128 bytes; their partial sums are joined
// in a fixed order.  8-bit: with FUSE the block makes the codes of up to 8 tokens itself, in shared memory, while its first
// weights are on their way (few_can_fuse), which saves a launch.
// One token through 14336 x 4096 twice and back, 16 bits: 68 us for both launches = 5.2 TB/s (80 % of the measured bandwidth: each
// launch pays for its start and its join); 512 x 2048 twice and back: 5.0 us, of which the weights account for 1.0.
#include "token_codes.cuh"

namespace dense {
namespace {

constexpr int kWarps = 8;
constexpr int kFuseBytes = 17408;

// Rows of codes in shared memory start 64 bytes off a multiple of 128, so that the rows of two tokens that are read at once lie
// in different banks.
__host__ __device__ inline int code_pitch(int K) { return (K + 127) / 128 * 128 + 64; }

struct FewArgs {
  Args p;
  const uint8_t* w[2];
  const uint8_t* x;          // 16-bit rows, or codes
  long long x_pitch, w_pitch[2];   // bytes
  int first_blocks;          // that run at once
};

enum Type { BF16 = 0, FP16 = 1, INT8 = 2 };

__device__ __forceinline__ void prefetch_l2(const uint8_t* p) { asm volatile("prefetch.global.L2 [%0];" ::"l"(p)); }

template <int TYPE>
__device__ __forceinline__ void mma(uint32_t (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if (TYPE == INT8) {
    asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else if (TYPE == BF16) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  } else {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  }
}

template <int TYPE, int EPI, bool FUSE, int NT>
__global__ void __launch_bounds__(32 * kWarps) dense_few_kernel(const __grid_constant__ FewArgs f) {
  constexpr int kKind = TYPE == INT8 ? KIND_I8 : KIND_16;
  constexpr bool kDual = is_dual(EPI);
  constexpr int kRows = kDual ? 8 : 16;                    // outputs of a block
  constexpr int kAhead = NT == 1 ? 4 : 2;                  // 128-byte steps of K in flight per warp
  const Args& a = f.p;
  __shared__ uint32_t part[kWarps][16][NT * 8 + 1];
  __shared__ __align__(16) uint8_t codes[FUSE ? kFuseBytes : 16];
  __shared__ uint32_t top[8];
  __shared__ float token_scale[8];
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
  const int n0 = blockIdx.x * kRows;
  const int kb = kKind == KIND_I8 ? a.K : 2 * a.K;         // bytes of a row
  // rows past the end repeat the last one; their outputs are not written
  const uint8_t* row_a = f.w[0] + min(n0 + g, a.N - 1) * f.w_pitch[0] + 16 * t;
  const uint8_t* row_b = kDual ? f.w[1] + min(n0 + g, a.N - 1) * f.w_pitch[1] + 16 * t
                               : f.w[0] + min(n0 + g + 8, a.N - 1) * f.w_pitch[0] + 16 * t;
  uint4 wa[kAhead][2], wb[kAhead][2];
  auto load_weights = [&](int base) {                      // base: byte of K of the warp's next step
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int b = base + i * (kWarps * 128) + 64 * h;
        const bool in = b + 16 * t < kb;
        wa[i][h] = in ? ld_global_v4(row_a + b) : make_uint4(0u, 0u, 0u, 0u);
        wb[i][h] = in ? ld_global_v4(row_b + b) : make_uint4(0u, 0u, 0u, 0u);
      }
  };
  // The first blocks bring their weights into L2 while the kernel before this one ends (2048 / 4096, one token: 14.4 us a block
  // for 15.0); later ones would only load everything twice (8192 / 8192: 66 us became 78).
  for (int b = warp * 128; b < kb && (int)blockIdx.x < f.first_blocks; b += kWarps * 128) {
    if (t == 0) prefetch_l2(row_a + b), prefetch_l2(row_b + b);   // 128 bytes of either row
  }
  overlap_point();
  load_weights(warp * 128);
  // the scales of this thread's output, long before they are needed
  const int r = tid % kRows, token = tid / kRows, col = n0 + r;
  float sa = 1.f, weight_scale[2] = {1.f, 1.f};
  if (kKind == KIND_I8 && token < a.M && col < a.N) {
    if (!FUSE) sa = a.a_scale[token];
    weight_scale[0] = a.b_scale[0][col];
    if (kDual) weight_scale[1] = a.b_scale[1][col];
  }

  if (FUSE) {
    if (tid < 8) top[tid] = 0u;
    __syncthreads();
    const int per = 32 * kWarps / (a.M <= 1 ? 1 : a.M <= 2 ? 2 : a.M <= 4 ? 4 : 8);   // threads of a token
    const int of = tid / per, j0 = tid % per, n8 = a.K / 8;
    const uint4* src = reinterpret_cast<const uint4*>(f.x + of * f.x_pitch);
    if (of < a.M) {
      uint32_t top2 = 0u;
      for (int i = j0; i < n8; i += per) top2 = magnitude_max(top2, src[i]);
      atomicMax(&top[of], magnitude_join(top2));           // a maximum: the order does not matter
    }
    __syncthreads();
    if (of < a.M) {
      const RowScale s = row_scale(top[of], a.bf16);
      if (j0 == 0) token_scale[of] = s.scale;
      for (int i = j0; i < n8; i += per) *reinterpret_cast<uint2*>(codes + of * code_pitch(a.K) + 8 * i) = codes8(src[i], s, a.bf16);
    }
    __syncthreads();
  }

  uint32_t acc[NT][4];
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[n][e] = 0u;
  for (int base = warp * 128; base < kb; base += kAhead * kWarps * 128) {
    uint4 xb[NT][kAhead][2];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < kAhead; ++i)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int b = base + i * (kWarps * 128) + 64 * h + 16 * t, token = 8 * n + g;
          uint4 v = make_uint4(0u, 0u, 0u, 0u);
          if (token < a.M && b < kb)
            v = FUSE ? *reinterpret_cast<const uint4*>(codes + token * code_pitch(a.K) + b)
                     : *reinterpret_cast<const uint4*>(f.x + token * f.x_pitch + b);
          xb[n][i][h] = v;
        }
#pragma unroll
    for (int i = 0; i < kAhead; ++i)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int n = 0; n < NT; ++n) {
          mma<TYPE>(acc[n], wa[i][h].x, wb[i][h].x, wa[i][h].y, wb[i][h].y, xb[n][i][h].x, xb[n][i][h].y);
          mma<TYPE>(acc[n], wa[i][h].z, wb[i][h].z, wa[i][h].w, wb[i][h].w, xb[n][i][h].z, xb[n][i][h].w);
        }
    if (base + kAhead * kWarps * 128 < kb) load_weights(base + kAhead * kWarps * 128);
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) part[warp][g + 8 * (e >> 1)][8 * n + 2 * t + (e & 1)] = acc[n][e];
  __syncthreads();

  if (tid >= kRows * a.M || col >= a.N) return;            // an output a thread: at most 16 rows by 16 tokens
  uint32_t v[2] = {0u, 0u};
#pragma unroll
  for (int d = 0; d < (kDual ? 2 : 1); ++d)
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const uint32_t p = part[w][r + 8 * d][token];
      v[d] = kKind == KIND_I8 ? v[d] + p : __float_as_uint(__uint_as_float(v[d]) + __uint_as_float(p));
    }
  if (kKind == KIND_I8) {
    if (FUSE) sa = token_scale[token];
#pragma unroll
    for (int d = 0; d < (kDual ? 2 : 1); ++d) v[d] = __float_as_uint(scaled(v[d], sa, weight_scale[d]));
  }
  float o[3];
  finish<EPI>(a, col, __uint_as_float(v[0]), __uint_as_float(v[1]), o);
  a.out[0][token * a.ld_out + col] = (uint16_t)(pack16(o[0], 0.f, a.bf16) & 0xffffu);
}

template <int TYPE, int EPI, bool FUSE>
int launch(const FewArgs& f, cudaStream_t s) {
  const int blocks = dmoq_ceil_div(f.p.N, is_dual(EPI) ? 8 : 16);
  if (FUSE || f.p.M <= 8) return launch_overlapped(dense_few_kernel<TYPE, EPI, FUSE, 1>, blocks, 32 * kWarps, 0, 0, s, f);
  return launch_overlapped(dense_few_kernel<TYPE, EPI, false, 2>, blocks, 32 * kWarps, 0, 0, s, f);
}

}  // namespace

// Every block makes all codes again.  In a graph the quantiser's own launch costs 0.2 us more than that saves at the least (2048
// x 512, one token: 3.5 us fused, 3.3 not; 2048 x 4096 twice: 8.1 and 6.8), but a call by itself has 5 us less to do on the
// host; so only as long as the blocks' codes are few in all.
bool few_can_fuse(int T, int K, int N, bool dual) {
  return T <= 8 && (long long)T * code_pitch(K) <= kFuseBytes && (long long)T * K * dmoq_ceil_div(N, dual ? 8 : 16) <= 1 << 20;
}

// x: 16-bit rows, or codes where a.a_scale is given; w1 only when dual; pitches in bytes.
int few_product(int kind, int epi, const void* x, long long x_pitch, const void* w0, long long w0_pitch, const void* w1, long long w1_pitch,
                const Args& a, cudaStream_t s) {
  const FewArgs f = {a, {static_cast<const uint8_t*>(w0), static_cast<const uint8_t*>(w1)}, static_cast<const uint8_t*>(x),
                     x_pitch, {w0_pitch, w1_pitch}, 2 * dmoq_sm_count()};
  if (kind == KIND_I8) {
    const bool fuse = a.a_scale == nullptr;
    if (epi == EPI_SCALE) return fuse ? launch<INT8, EPI_SCALE, true>(f, s) : launch<INT8, EPI_SCALE, false>(f, s);
    if (epi == EPI_SILU) return fuse ? launch<INT8, EPI_SILU, true>(f, s) : launch<INT8, EPI_SILU, false>(f, s);
    return DMOQ_EINVAL;
  }
  if (epi == EPI_OUT) return a.bf16 ? launch<BF16, EPI_OUT, false>(f, s) : launch<FP16, EPI_OUT, false>(f, s);
  if (epi == EPI_SILU) return a.bf16 ? launch<BF16, EPI_SILU, false>(f, s) : launch<FP16, EPI_SILU, false>(f, s);
  return DMOQ_EINVAL;
}

}  // namespace dense
