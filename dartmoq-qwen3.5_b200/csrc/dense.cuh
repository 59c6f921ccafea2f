// Dense products y = A B^T of the operators beside the packed experts: what a launch is given, and its epilogues.
//
//   kind 16-bit (bf16 or fp16, fp32 sums) or 8-bit integers (int32 sums); an operand is K-major (its rows run along K) or
//   MN-major (its rows run along the output axis), as the caller's tensors lie in memory: nothing is transposed or copied.
#pragma once
#include "dense_ptx.cuh"

namespace dense {

enum Kind { KIND_16 = 0, KIND_I8 = 1 };
enum Epi {
  EPI_OUT = 0,        // out[0] = v                                       (16-bit products)
  EPI_SCALE = 1,      // out[0] = v * a_scale[row] * b_scale[col] + bias  (8-bit products)
  EPI_SILU = 2,       // g, u from two weights: out[0] = silu(g) u
  EPI_SILU_SAVE = 3,  // the same, and silu(g), u silu'(g) for the gradients in three planes (see Saved)
  EPI_GRAD = 4        // v = dh: out[0] = dg = dh * u silu'(g), out[1] = du = dh * silu(g), from those planes
};
constexpr __host__ __device__ bool is_dual(int epi) { return epi == EPI_SILU || epi == EPI_SILU_SAVE; }

constexpr __host__ __device__ int outputs_of(int epi) { return epi == EPI_SILU_SAVE ? 4 : epi == EPI_GRAD ? 2 : 1; }

struct Maps {
  CUtensorMap a[2], b[2];
};

// silu(g) and u silu'(g) are kept to the upper 24 bits of their 32-bit floats, whatever the tensors' 16-bit type: planes 1 and 2
// hold the upper 16 bits of either, plane 3 the next eight of both.  Rounded to 16 bits they would add a third rounding of the
// type to dg and du, which are themselves rounded as operands of the next products; this costs half as much traffic
// again and leaves less than 2^-15, always toward zero (2^-16 on average; a rounding of the types is up to 2^-9 or 2^-12).
// The lower bits are cut off, not rounded, so that a NaN stays one.
__device__ __forceinline__ uint32_t saved_low(float silu, float slope) {
  return ((__float_as_uint(silu) >> 8) & 0xffu) | (__float_as_uint(slope) & 0xff00u);
}
__device__ __forceinline__ float saved_silu(uint32_t hi, uint32_t low) { return __uint_as_float((hi << 16) | ((low & 0xffu) << 8)); }
__device__ __forceinline__ float saved_slope(uint32_t hi, uint32_t low) { return __uint_as_float((hi << 16) | (low & 0xff00u)); }

struct Args {
  int M, N, K;              // output rows, output columns (of one of the two products when dual), length of a K segment
  int segs;                 // K segments: segment s multiplies a[s] by b[s], all into one sum
  int bf16;                 // 16-bit type of inputs and outputs: bf16, else fp16
  int vec;                  // output rows may be written four elements at a time
  const float* a_scale;     // 8-bit: one per row
  const float* b_scale[2];  // 8-bit: one per column (of each product when dual)
  const uint16_t* bias;     // 8-bit, optional, type of the output
  const uint16_t* in[3];    // the saved planes
  uint16_t* out[4];
  long long ld_in, ld_out;  // row pitches in elements (ld_in: of the planes that are read)
  long long ld_saved;       // of the planes that are written, out[1] to out[3]
};

// The arithmetic of the epilogues, with its roundings spelled out (no contraction left to the compiler), so that an 8-bit result
// does not depend on the kernel that a batch's size selects.
//
// sum * token_scale * row_scale: the scales are multiplied first.  With either outside 2^-60 .. 2^48 their product may leave the
// normal 32-bit numbers although the result does not (a subnormal factor of 1e-45 times a sum of 1e8, infinity times a sum of
// zero), and neither other order of two products holds everywhere; there the three are multiplied in 64 bits, whose range holds
// any of them.  The rule looks at the element's own scales alone: its result is the same in every batch and every kernel.
__device__ __forceinline__ bool plain_scale(float s) {
  const uint32_t magnitude = __float_as_uint(s) & 0x7fffffffu;
  return magnitude - (67u << 23) < (108u << 23) || magnitude == 0u;
}
__device__ __forceinline__ float scaled_plain(uint32_t sum, float token_scale, float row_scale) {
  return __fmul_rn((float)(int)sum, __fmul_rn(token_scale, row_scale));
}
__device__ __forceinline__ float scaled(uint32_t sum, float token_scale, float row_scale) {
  if (plain_scale(token_scale) && plain_scale(row_scale)) return scaled_plain(sum, token_scale, row_scale);
  return __double2float_rn(__dmul_rn(__dmul_rn((double)(int)sum, (double)token_scale), (double)row_scale));
}
__device__ __forceinline__ float gated(float g, float u) { return __fmul_rn(__fmul_rn(g, sigmoid(g)), u); }
// silu'(g) = s (1 + g (1 - s)) = s + silu(g) (1 - s), s = sigmoid(g)
__device__ __forceinline__ float slope_of(float s, float silu, float u) { return __fmul_rn(u, __fmaf_rn(silu, __fsub_rn(1.f, s), s)); }

// One output element's value: x (and y of the second product) are the products.
template <int EPI>
__device__ __forceinline__ void finish(const Args& a, int col, float x, float y, float (&o)[3]) {
  if (EPI == EPI_OUT) {
    o[0] = x;
  } else if (EPI == EPI_SCALE) {
    o[0] = a.bias ? __fadd_rn(x, unpack16(a.bias[col], a.bf16)) : x;
  } else if (EPI == EPI_SILU) {
    o[0] = gated(x, y);
  } else if (EPI == EPI_SILU_SAVE) {
    const float s = sigmoid(x), si = __fmul_rn(x, s);
    o[0] = __fmul_rn(si, y);
    o[1] = si;
    o[2] = slope_of(s, si, y);
  }
}

// Rows row_lo .. row_hi - 1 of a tile whose sums lie in shared memory (rows `pitch` bytes apart, kCols 32-bit columns and, when
// dual, kCols more of the second product), split over the cluster's blocks: joined, finished and written, four columns a
// thread.  Neighbouring threads read neighbouring columns: a warp's read of another block's memory is whole lines (a row a
// lane made joining eight blocks slower than leaving the product unsplit).
template <int KIND, int EPI, int kCols, bool PLAIN>
__device__ __forceinline__ void finish_rows_of(const Args& a, uint32_t sums, uint32_t pitch, int row_lo, int row_hi, int m0, int n0,
                                            uint32_t blocks, int tid) {
  constexpr int kQuads = kCols / 4;
  constexpr bool kDual = is_dual(EPI);
#pragma unroll 2
  for (int i = row_lo * kQuads + tid; i < row_hi * kQuads; i += 256) {
    const int r = i / kQuads, c = i % kQuads * 4;
    const long long row = m0 + r;
    const int col = n0 + c;
    if (row >= a.M || col >= a.N) continue;
    uint32_t v[4], u[4] = {0u, 0u, 0u, 0u};
    const uint32_t at = sums + r * pitch + c * 4;
    sum_over_cluster<KIND == KIND_I8>(at, blocks, v);
    if (kDual) sum_over_cluster<KIND == KIND_I8>(at + kCols * 4, blocks, u);
    const int n = min(4, a.N - col);
    const float sa = KIND == KIND_I8 ? a.a_scale[row] : 1.f;
    auto product = [&](uint32_t sum, int d, int j) {
      if (KIND == KIND_16) return __uint_as_float(sum);
      const float s = a.b_scale[d][col + j];
      return PLAIN ? scaled_plain(sum, sa, s) : scaled(sum, sa, s);
    };
    const long long at_out = row * a.ld_out + col;
    float o[3][4];
    if (EPI == EPI_GRAD) {
      const long long at_in = row * a.ld_in + col;   // the planes' rows are whole groups of four (sizes are multiples of 8)
      uint2 pl[3];
#pragma unroll
      for (int e = 0; e < 3; ++e) pl[e] = *reinterpret_cast<const uint2*>(a.in[e] + at_in);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        auto half = [&](const uint2 w) { return ((j < 2 ? w.x : w.y) >> (16 * (j & 1))) & 0xffffu; };
        const float dh = __uint_as_float(v[j]);
        o[0][j] = dh * saved_slope(half(pl[1]), half(pl[2]));
        o[1][j] = dh * saved_silu(half(pl[0]), half(pl[2]));
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float e[3] = {0.f, 0.f, 0.f};
        if (j < n) finish<EPI>(a, col + j, product(v[j], 0, j), kDual ? product(u[j], 1, j) : 0.f, e);
        o[0][j] = e[0], o[1][j] = e[1], o[2][j] = e[2];
      }
    }
#pragma unroll
    for (int e = 0; e < outputs_of(EPI); ++e) {
      uint32_t lo, hi;
      if (EPI == EPI_SILU_SAVE && e > 0) {
        auto word = [&](int j) {
          return e == 3 ? saved_low(o[1][j], o[2][j]) : __float_as_uint(o[e < 3 ? e : 0][j]) >> 16;
        };
        lo = word(0) | (word(1) << 16), hi = word(2) | (word(3) << 16);
      } else {
        lo = pack16(o[e < 3 ? e : 0][0], o[e < 3 ? e : 0][1], a.bf16), hi = pack16(o[e < 3 ? e : 0][2], o[e < 3 ? e : 0][3], a.bf16);
      }
      uint16_t* dst = a.out[e] + (EPI == EPI_SILU_SAVE && e > 0 ? row * a.ld_saved + col : at_out);
      if (a.vec) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(lo, hi);
      } else {
        const uint32_t h[4] = {lo & 0xffffu, lo >> 16, hi & 0xffffu, hi >> 16};
        for (int j = 0; j < n; ++j) dst[j] = (uint16_t)h[j];
      }
    }
  }
}

// Whether all scales of a tile are plain, by `threads` threads of which this is the t-th: their part of the answer.  Looked at
// once, beside the products: a look at every element kept the epilogue's loads apart (200 x 2048 by K = 4096 9.4 us for 8.5).
__device__ __forceinline__ bool plain_tile(const Args& a, int m0, int rows, int n0, int cols, bool dual, int t, int threads) {
  bool plain = true;
  for (int i = t; i < rows && m0 + i < a.M; i += threads) plain = plain && plain_scale(a.a_scale[m0 + i]);
  for (int i = t; i < cols && n0 + i < a.N; i += threads)
    plain = plain && plain_scale(a.b_scale[0][n0 + i]) && (!dual || plain_scale(a.b_scale[1][n0 + i]));
  return plain;
}
template <int KIND, int EPI, int kCols>
__device__ __forceinline__ void finish_rows(const Args& a, uint32_t sums, uint32_t pitch, int row_lo, int row_hi, int m0, int n0,
                                            uint32_t blocks, int tid, bool plain) {
  if (KIND == KIND_16 || plain)
    finish_rows_of<KIND, EPI, kCols, true>(a, sums, pitch, row_lo, row_hi, m0, n0, blocks, tid);
  else
    finish_rows_of<KIND, EPI, kCols, false>(a, sums, pitch, row_lo, row_hi, m0, n0, blocks, tid);
}

}  // namespace dense
