// Per-token symmetric 8-bit codes: scale = max|x| / 127 over a row, code = rint(127 x / max|x|), ties to even.
//
// 127 x has at most 18 significant bits and the maximum at most 11, so a quotient that is not a tie differs from one by at
// least 2^-19 of its size: the correctly rounded 32-bit quotient rounds to the same code as the exact one.
#include "dense.cuh"

namespace {

constexpr int kThreads = 256;

// One block a row; the second pass reads the row again from L1 / L2.
__global__ void __launch_bounds__(kThreads) token_quant_kernel(const uint16_t* x, int bf16, int K, long long pitch, int8_t* codes,
                                                               float* scales) {
  __shared__ float part[kThreads / 32];
  __shared__ int bad;
  const long long row = blockIdx.x;
  const uint4* src = reinterpret_cast<const uint4*>(x + row * pitch);
  const int tid = threadIdx.x, n8 = K / 8;
  if (tid == 0) bad = 0;
  __syncthreads();
  float top = 0.f;
  bool odd = false;                      // infinities and NaN
  for (int i = tid; i < n8; i += kThreads) {
    const uint4 v = src[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float f = fabsf(dense::unpack16((w[j / 2] >> (16 * (j & 1))) & 0xffffu, bf16));
      odd |= !(f <= 3.4028235e38f);
      top = fmaxf(top, f);
    }
  }
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  if ((tid & 31) == 0) part[tid >> 5] = top;
  if (odd) bad = 1;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kThreads / 32; ++w) top = fmaxf(top, part[w]);
  const bool void_row = bad != 0;
  if (tid == 0) scales[row] = void_row ? __int_as_float(0x7fc00000) : __fdiv_rn(top, 127.f);
  // 127 x must not overflow: rows of huge bf16 values are brought down by a power of two first
  const float down = top > 1e30f ? 0x1p-8f : 1.f;
  const float den = top * down;
  uint2* dst = reinterpret_cast<uint2*>(codes + row * (long long)K);
  for (int i = tid; i < n8; i += kThreads) {
    const uint4 v = src[i];
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t o[2] = {0u, 0u};
    if (!void_row && top > 0.f) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float f = dense::unpack16((w[j / 2] >> (16 * (j & 1))) & 0xffffu, bf16) * down;
        const int q = __float2int_rn(__fdiv_rn(127.f * f, den));
        o[j / 4] |= (uint32_t)(q & 0xff) << (8 * (j & 3));
      }
    }
    dst[i] = make_uint2(o[0], o[1]);
  }
}

}  // namespace

int dmoq_token_quant_launch(const void* x, int bf16, int T, int K, long long pitch, int8_t* codes, float* scales, cudaStream_t s) {
  token_quant_kernel<<<T, kThreads, 0, s>>>(static_cast<const uint16_t*>(x), bf16, K, pitch, codes, scales);
  return dmoq_launch_status();
}
