// Per-token symmetric 8-bit codes: scale = max|x| / 127 over a row, code = rint(127 x / max|x|), ties to even (token_codes.cuh has
// the arithmetic).  Bound by memory: 2 bytes read and 1 written a value; a row stays in registers between its maximum and
// its codes, so it is read once.  16384 x 4096: 36 us = 5.6 TB/s (87 % of the measured bandwidth); a division a value took 64 us.
#include "token_codes.cuh"

namespace dense {
namespace {

// A row belongs to WARPS warps, NV vectors of eight values a thread: K <= 8 * 32 * WARPS * NV.
template <int NV, int WARPS>
__global__ void __launch_bounds__(256) token_quant_kernel(const uint16_t* x, int bf16, int rows, int K, long long pitch, int8_t* codes, long long code_pitch,
                                                          float* scales) {
  constexpr int kThreads = 32 * WARPS;                     // threads of a row
  const int tid = threadIdx.x % kThreads, n8 = K / 8;
  overlap_point();
  const long long row = (long long)blockIdx.x * (256 / kThreads) + threadIdx.x / kThreads;
  if (WARPS == 1 && row >= rows) return;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * pitch);
  uint4 v[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = tid + j * kThreads;
    v[j] = i < n8 ? src[i] : make_uint4(0u, 0u, 0u, 0u);
  }
  uint32_t top2 = 0u;
#pragma unroll
  for (int j = 0; j < NV; ++j) top2 = magnitude_max(top2, v[j]);
  uint32_t top = __reduce_max_sync(0xffffffffu, magnitude_join(top2));
  if (WARPS > 1) {
    __shared__ uint32_t part[WARPS];
    if ((tid & 31) == 0) part[tid >> 5] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) top = max(top, part[w]);
  }
  const RowScale s = row_scale(top, bf16);
  if (tid == 0) scales[row] = s.scale;
  uint2* dst = reinterpret_cast<uint2*>(codes + row * code_pitch);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int i = tid + j * kThreads;
    if (i < n8) dst[i] = codes8(v[j], s, bf16);
  }
}

// Rows too long for registers: a block a row, the second pass reads the row again from L2.
__global__ void __launch_bounds__(256) token_quant_long_kernel(const uint16_t* x, int bf16, int K, long long pitch, int8_t* codes, long long code_pitch,
                                                               float* scales) {
  __shared__ uint32_t part[8];
  overlap_point();
  const long long row = blockIdx.x;
  const int tid = threadIdx.x, n8 = K / 8;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * pitch);
  uint32_t top2 = 0u;
  for (int i = tid; i < n8; i += 256) top2 = magnitude_max(top2, src[i]);
  uint32_t top = __reduce_max_sync(0xffffffffu, magnitude_join(top2));
  if ((tid & 31) == 0) part[tid >> 5] = top;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < 8; ++w) top = max(top, part[w]);
  const RowScale s = row_scale(top, bf16);
  if (tid == 0) scales[row] = s.scale;
  uint2* dst = reinterpret_cast<uint2*>(codes + row * code_pitch);
  for (int i = tid; i < n8; i += 256) dst[i] = codes8(src[i], s, bf16);
}

template <int NV, int WARPS>
int launch(const uint16_t* x, int bf16, int T, int K, long long pitch, int8_t* codes, long long code_pitch, float* scales, cudaStream_t s) {
  return launch_overlapped(token_quant_kernel<NV, WARPS>, dmoq_ceil_div(T, 8 / WARPS), 256, 0, 0, s, x, bf16, T, K, pitch, codes, code_pitch, scales);
}

}  // namespace
}  // namespace dense

// code_pitch: between the codes' rows, a multiple of 16
int dmoq_token_quant_launch(const void* xv, int bf16, int T, int K, long long pitch, int8_t* codes, long long code_pitch, float* scales, cudaStream_t s) {
  using namespace dense;
  const uint16_t* x = static_cast<const uint16_t*>(xv);
  // A warp a row streams best; few rows, or rows beyond a warp's registers, get a block each.
  if (T >= 4 * dmoq_sm_count() && K <= 4096) {
    if (K <= 1024) return launch<4, 1>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
    if (K <= 2048) return launch<8, 1>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
    return launch<16, 1>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
  }
  if (K <= 2048) return launch<1, 8>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
  if (K <= 4096) return launch<2, 8>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
  if (K <= 8192) return launch<4, 8>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
  if (K <= 16384) return launch<8, 8>(x, bf16, T, K, pitch, codes, code_pitch, scales, s);
  return launch_overlapped(token_quant_long_kernel, T, 256, 0, 0, s, x, bf16, K, pitch, codes, code_pitch, scales);
}
