// C entry points of the dense operators: argument checks, tensor maps, choice of the kernel.
#include <algorithm>
#include <cmath>

#include "dense.cuh"

int dmoq_token_quant_launch(const void* x, int bf16, int T, int K, long long pitch, int8_t* codes, long long code_pitch, float* scales,
                            cudaStream_t s);

namespace dense {

int tile_product(int kind, bool a_mn, bool b_mn, int epi, const Maps& maps, const Args& a, int splits, cudaStream_t s);
int tile_blocks_at_once(int splits);
int pair_product(int kind, bool a_mn, bool b_mn, int epi, const Maps& maps, const Args& a, cudaStream_t s);
int pair_group(const Maps* maps, const Args* p, const bool* a_mn, int n, int n_long, cudaStream_t s);

int mid_product(int kind, int epi, const Maps& maps, const Args& a, int splits, cudaStream_t s);
int mid_token_box(int tokens);
int few_product(int kind, int epi, const void* x, long long x_pitch, const void* w0, long long w0_pitch, const void* w1, long long w1_pitch,
                const Args& a, cudaStream_t s);
bool few_can_fuse(int T, int K, int N, bool dual);

namespace {

constexpr int kMidTokens = 256;  // up to here the kernel whose M operand is the weights

// The kernel that streams the weights through registers: always up to 8 tokens, and up to 16 (its second token tile halves the
// loads it keeps in flight) where there are so few weights that latency counts.  16 tokens, gate and up: 4 MB 4.8 us against
// 6.4, 67 MB 24.9 us against 16.7.
bool few_tokens(int T, long long weight_bytes) { return T <= 8 || (T <= 16 && weight_bytes <= (16LL << 20)); }

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn() {
  static std::atomic<EncodeTiledFn> known{nullptr};
  EncodeTiledFn fn = known;
  if (fn == nullptr) {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess || q != cudaDriverEntryPointSuccess)
      return nullptr;
    known = fn = reinterpret_cast<EncodeTiledFn>(p);
  }
  return fn;
}

// A matrix of `rows` rows of `cols` elements (1 or 2 bytes), `pitch` elements apart.
struct Matrix {
  const void* p;
  long long rows, cols, pitch;
};

// Every check comes before the first launch of a call.
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
bool tma_ok(const Matrix& m, int es) { return aligned16(m.p) && (m.pitch * es) % 16 == 0 && m.pitch >= m.cols; }

// Copied in boxes of 128 bytes x box_rows rows with the 128-byte swizzle; what lies past the matrix reads as zero.
int make_map(CUtensorMap* map, const Matrix& m, int es, int box_rows) {
  EncodeTiledFn fn = encode_tiled_fn();
  if (fn == nullptr) return DMOQ_EDEVICE;
  const cuuint64_t dims[2] = {(cuuint64_t)m.cols, (cuuint64_t)m.rows};
  const cuuint64_t strides[1] = {(cuuint64_t)m.pitch * es};
  const cuuint32_t box[2] = {(cuuint32_t)(128 / es), (cuuint32_t)box_rows};
  const cuuint32_t estr[2] = {1, 1};
  auto encode = [&] {
    return fn(map, es == 1 ? CU_TENSOR_MAP_DATA_TYPE_UINT8 : CU_TENSOR_MAP_DATA_TYPE_UINT16, 2, const_cast<void*>(m.p), dims,
              strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
              CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = encode();
  if (rc == CUDA_ERROR_INVALID_CONTEXT || rc == CUDA_ERROR_NOT_INITIALIZED) {
    // a thread that has made no runtime call yet (autograd runs backward passes on threads of its own) has no context bound
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaSetDevice(dev) != cudaSuccess) return DMOQ_EDEVICE;
    rc = encode();
  }
  return rc == CUDA_SUCCESS ? DMOQ_OK : DMOQ_EINVAL;
}

// A product of operands as they lie in memory: a_mn / b_mn say that a matrix runs along the output axis (its rows are K).
struct Product {
  int kind = KIND_16, epi = EPI_OUT;
  bool a_mn = false, b_mn = false;
  Matrix a[2] = {}, b[2] = {};
  Args args = {};
};

// The tensor maps of a product: boxes of 128 rows of A and `b_box` rows of B (K-major), or of a step of K (MN-major).
int make_maps(Maps& maps, const Product& p, int b_box) {
  const int es = p.kind == KIND_I8 ? 1 : 2, bk = 128 / es;
  const int n_a = p.args.segs, n_b = is_dual(p.epi) ? 2 : p.args.segs;
  for (int i = 0; i < n_a + n_b; ++i) {
    const bool is_a = i < n_a;
    const Matrix& m = is_a ? p.a[i] : p.b[i - n_a];
    if (!tma_ok(m, es)) return DMOQ_EINVAL;
    const int rc = make_map(is_a ? &maps.a[i] : &maps.b[i - n_a], m, es, is_a ? (p.a_mn ? bk : 128) : (p.b_mn ? bk : b_box));
    if (rc != DMOQ_OK) return rc;
  }
  return DMOQ_OK;
}
// The pair kernel's arguments: outputs leave as 16-byte stores of eight columns where their memory allows.
Args pair_args(const Product& p) {
  Args args = p.args;
  args.vec = args.N % 8 == 0;
  for (int e = 0; e < outputs_of(p.epi); ++e) args.vec = args.vec && aligned16(args.out[e]) && args.ld_out % 8 == 0;
  return args;
}
long long pair_tiles(const Product& p) {
  return (long long)dmoq_ceil_div(p.args.M, 256) * dmoq_ceil_div(p.args.N, is_dual(p.epi) ? 128 : 256);
}
long long steps_of(const Product& p) { return (long long)dmoq_ceil_div(p.args.K, p.kind == KIND_I8 ? 128 : 64) * p.args.segs; }

// What a product costs in each kernel, in microseconds, to choose among them: fits to measurements on a B200 of products
// of 64 to 16384 rows by 512 to 5456 columns and 1 to 256 steps of K (a step is 128 bytes), about 15 % off at worst.  Whole
// tiles go round the SMs, so a product that fills them badly in wide tiles may be better off in narrow ones or with K split:
//                                            pairs    tiles (K in parts)
//   300 x 4096 by K = 4096 (64 steps)        23.7     21.5 (2)     1000 x 4096, K = 4096    26.2     34.1 (1)
//   1024 x 2048 by K = 16384 (256)           77.0     64.1 (2)     2048 x 2048, K = 16384   94.6    119.8 (1)
//   257 x 1032 by K = 5456 (86)              31.1     13.0 (4)     1000 x 2728, K = 1032    12.1     20.3 (1)
double pair_cost(const Product& p) {
  const double rounds = std::ceil((double)pair_tiles(p) / (dmoq_sm_count() / 2));
  return 4.6 + rounds * 0.30 * steps_of(p) + (rounds - 1) * 2.0;
}
double join_cost(int splits) { return splits == 1 ? 0.0 : splits == 2 ? 0.7 : splits == 4 ? 1.0 : 1.8; }
double tile_cost(const Product& p, int splits) {
  const double blocks = (double)dmoq_ceil_div(p.args.M, 128) * dmoq_ceil_div(p.args.N, is_dual(p.epi) ? 64 : 128) * splits;
  const double steps = std::ceil((double)steps_of(p) / splits);
  if (blocks <= tile_blocks_at_once(splits)) return 5.0 + 0.29 * steps + join_cost(splits);
  const double rounds = std::ceil(blocks / (2 * tile_blocks_at_once(splits)));                             // two blocks an SM
  return 2.0 + rounds * (5.0 + 0.45 * steps) + join_cost(splits);   // a round's start and end are not covered by the next
}
double mid_cost(const Product& p, int splits) {   // 129 to 256 tokens
  const double blocks = (double)dmoq_ceil_div(p.args.N, is_dual(p.epi) ? 64 : 128) * splits;
  return std::ceil(blocks / dmoq_sm_count()) * (5.0 + 0.38 * std::ceil((double)steps_of(p) / splits)) + join_cost(splits);
}

struct Choice {
  enum Kernel { PAIR, TILE, MID } kernel;
  int splits;
  double cost;
};
Choice choose(const Product& p) {
  const long long steps = steps_of(p);
  Choice best = {Choice::PAIR, 1, pair_cost(p)};
  for (int splits = 1; splits <= 8 && splits <= steps; splits *= 2) {
    const double c = tile_cost(p, splits);
    if (c < best.cost) best = {Choice::TILE, splits, c};
  }
  if (p.args.M <= kMidTokens && !p.a_mn && !p.b_mn && p.args.segs == 1) {
    if (p.args.M <= 128) {
      // Reading the weights is all that counts.  Up to two blocks an SM stream at once.  Below half the SMs a split pays from
      // 2 steps a block on, above from 8: 32 tiles of 32 steps take 10.4 us in 4 parts and 11.6 in 8; 64 tiles of 64 steps
      // 22.4 us in 2 and 19.3 in 4; 216 tiles of 80 steps 50 us whole and 56 in 2.
      const long long tiles = dmoq_ceil_div(p.args.N, is_dual(p.epi) ? 64 : 128);
      int splits = 1;
      while (splits < 8 && tiles * splits <= dmoq_sm_count() && steps >= splits * (tiles * splits * 2 < dmoq_sm_count() ? 4 : 16)) splits *= 2;
      return {Choice::MID, splits, 0.0};
    }
    for (int splits = 1; splits <= 8 && splits <= steps; splits *= 2) {
      const double c = mid_cost(p, splits);
      if (c < best.cost) best = {Choice::MID, splits, c};
    }
  }
  return best;
}

int run(const Product& p, const Choice& choice, cudaStream_t s) {
  Maps maps;
  int rc;
  switch (choice.kernel) {
    case Choice::PAIR:
      rc = make_maps(maps, p, 128);
      return rc != DMOQ_OK ? rc : pair_product(p.kind, p.a_mn, p.b_mn, p.epi, maps, pair_args(p), s);
    case Choice::TILE:
      rc = make_maps(maps, p, is_dual(p.epi) ? 64 : 128);
      return rc != DMOQ_OK ? rc : tile_product(p.kind, p.a_mn, p.b_mn, p.epi, maps, p.args, choice.splits, s);
    default: {
      const int es = p.kind == KIND_I8 ? 1 : 2, rows = is_dual(p.epi) ? 64 : 128;
      rc = tma_ok(p.a[0], es) && tma_ok(p.b[0], es) ? make_map(&maps.b[0], p.a[0], es, mid_token_box(p.args.M)) : DMOQ_EINVAL;
      if (rc == DMOQ_OK) rc = make_map(&maps.a[0], p.b[0], es, rows);
      if (rc == DMOQ_OK && is_dual(p.epi)) rc = tma_ok(p.b[1], es) ? make_map(&maps.a[1], p.b[1], es, rows) : DMOQ_EINVAL;
      return rc != DMOQ_OK ? rc : mid_product(p.kind, p.epi, maps, p.args, choice.splits, s);
    }
  }
}
int run(const Product& p, cudaStream_t s) { return run(p, choose(p), s); }

// Independent products (MN-major B, plain outputs) in one launch: their tiles fill the SMs together.  That takes as long as a
// pair's share of all tiles, each with about 2 us that the next one's products do not cover, or the longest tile.
double group_cost(const Product* const* p, int n) {
  double all = 0.0, longest = 0.0;
  for (int i = 0; i < n; ++i) {
    const double tile = 2.0 + 0.30 * steps_of(*p[i]);
    all += pair_tiles(*p[i]) * tile;
    longest = std::max(longest, tile);
  }
  return 4.6 + std::max(all / (dmoq_sm_count() / 2), longest);
}
int run_group(const Product* const* p, int n, cudaStream_t s) {
  long long longest = 0, shortest = 1LL << 60;
  for (int i = 0; i < n; ++i) {
    longest = std::max(longest, steps_of(*p[i]));
    shortest = std::min(shortest, steps_of(*p[i]));
  }
  Maps maps[3];
  Args args[3];
  bool a_mn[3];
  int m = 0, n_long = 0;
  for (int side = 0; side < 2; ++side) {      // the products with the longer tiles first
    for (int i = 0; i < n; ++i) {
      const Product& q = *p[i];
      if ((2 * steps_of(q) >= longest + shortest) != (side == 0)) continue;
      const int rc = make_maps(maps[m], q, 128);
      if (rc != DMOQ_OK) return rc;
      args[m] = pair_args(q);
      a_mn[m++] = q.a_mn;
    }
    if (side == 0) n_long = m;
  }
  return pair_group(maps, args, a_mn, n, n_long, s);
}
// The three products behind dg and du: each by itself, all in one launch, or the two weight gradients in one (8192 tokens of 2048 /
// 512: 56 us in one launch, 107 in three; 257 tokens of 1032 / 2728: dx is better off with its long K split).
int run_gradients(const Product& dx, const Product& dw_in, const Product& dw_out, cudaStream_t s) {
  const Product* all[3] = {&dx, &dw_in, &dw_out};
  const Choice x = choose(dx), in = choose(dw_in), out = choose(dw_out);
  const double weights = group_cost(all + 1, 2), apart = in.cost + out.cost;
  if (group_cost(all, 3) <= x.cost + std::min(weights, apart)) return run_group(all, 3, s);
  int rc = run(dx, x, s);
  if (rc != DMOQ_OK) return rc;
  if (weights <= apart) return run_group(all + 1, 2, s);
  rc = run(dw_in, in, s);
  return rc != DMOQ_OK ? rc : run(dw_out, out, s);
}

// four-element accesses to a 16-bit matrix
bool vec4(const void* p, long long n, long long pitch) { return reinterpret_cast<uintptr_t>(p) % 8 == 0 && n % 4 == 0 && pitch % 4 == 0; }

constexpr int kMaxK8 = 131056;   // |sum of K products of codes| <= 128 * 128 K stays inside 32 bits

bool usable(const void* p) { return p != nullptr && aligned16(p); }
bool rows_usable(const void* p, long long pitch, int cols) { return usable(p) && pitch >= cols && pitch % 8 == 0; }   // 16-bit rows

constexpr int kMaxDim = 1 << 30;   // rows and columns: tile coordinates stay inside 32 bits
// The weights' gradients sum over the tokens in one pass: at this many a tile takes a third of the second after which a wait
// inside a kernel gives up.
constexpr int kMaxGradTokens = 1 << 26;

int check_sizes8(int T, int N, int K) {
  if (T < 0 || N < 1 || K < 16 || K % 16 != 0) return DMOQ_EINVAL;
  return K > kMaxK8 || T > kMaxDim || N > kMaxDim ? DMOQ_ESIZE : DMOQ_OK;
}
bool quant_ok(const void* x, long long pitch, int K, const void* codes, const void* scales) {
  return rows_usable(x, pitch, K) && usable(codes) && scales;
}
struct Weight8 {   // rows of K codes, `pitch` apart, one scale each
  const int8_t* w;
  long long pitch;
  const float* scale;
};
bool weight8_ok(const Weight8& w, int K) { return usable(w.w) && w.scale && w.pitch >= K && w.pitch % 16 == 0; }
int check_ffn(int T, int H, int I) {
  if (T < 0 || H < 8 || I < 8 || H % 8 != 0 || I % 8 != 0) return DMOQ_EINVAL;
  // the gradients of both projections are one product of 2 I rows, and the bytes of a row are counted in 32 bits
  return T > kMaxDim || H > kMaxDim / 2 || I > kMaxDim / 2 ? DMOQ_ESIZE : DMOQ_OK;
}

// The products of `codes`, or of the 16-bit rows x (pitch in elements), whose codes then go into `codes` / `scales` first unless
// the kernel makes them itself.
int int8_product(const void* x, long long x_pitch, int8_t* codes, long long code_pitch, float* scales, const Weight8& w, const Weight8* up,
                 const void* bias, int bf16, int T, int N, int K, void* out, cudaStream_t s) {
  const bool few = few_tokens(T, (long long)N * K * (up ? 2 : 1));
  const bool fuse = x != nullptr && few_can_fuse(T, K, N, up != nullptr);   // implies few
  if (x != nullptr && !fuse) {
    const int rc = dmoq_token_quant_launch(x, bf16, T, K, x_pitch, codes, code_pitch, scales, s);
    if (rc != DMOQ_OK) return rc;
  }
  Product p;
  p.kind = KIND_I8;
  p.epi = up ? EPI_SILU : EPI_SCALE;
  Args& a = p.args;
  a.M = T, a.N = N, a.K = K, a.segs = 1, a.bf16 = bf16;
  a.a_scale = fuse ? nullptr : scales, a.b_scale[0] = w.scale, a.b_scale[1] = up ? up->scale : nullptr;
  a.bias = static_cast<const uint16_t*>(bias);
  a.out[0] = static_cast<uint16_t*>(out);
  a.ld_out = N;
  a.vec = vec4(out, N, N);
  if (few)
    return few_product(KIND_I8, p.epi, fuse ? x : codes, fuse ? 2 * x_pitch : code_pitch, w.w, w.pitch, up ? up->w : nullptr,
                       up ? up->pitch : 0, a, s);
  p.a[0] = {codes, T, K, code_pitch};
  p.b[0] = {w.w, N, K, w.pitch};
  if (up) p.b[1] = {up->w, N, K, up->pitch};
  return run(p, s);
}

}  // namespace
}  // namespace dense

using namespace dense;

extern "C" int dmoq_token_quant(const void* x, int32_t is_bf16, int32_t T, int32_t K, int64_t x_pitch, int8_t* codes, float* scales,
                                void* stream) {
  DMOQ_CHECK_ARG(T >= 0 && K >= 16 && K % 16 == 0);
  if (T > kMaxDim) return DMOQ_ESIZE;
  if (T == 0) return DMOQ_OK;
  DMOQ_CHECK_ARG(quant_ok(x, x_pitch, K, codes, scales));
  return dmoq_token_quant_launch(x, is_bf16, T, K, x_pitch, codes, K, scales, static_cast<cudaStream_t>(stream));
}

extern "C" int dmoq_int8_gemm(const int8_t* codes, const float* scales, const int8_t* w, int64_t w_pitch, const float* w_scale, const void* bias,
                              int32_t is_bf16, int32_t T, int32_t N, int32_t K, void* out, void* stream) {
  const int rc = check_sizes8(T, N, K);
  if (rc != DMOQ_OK || T == 0) return rc;
  const Weight8 weight = {w, w_pitch, w_scale};
  DMOQ_CHECK_ARG(usable(codes) && scales && weight8_ok(weight, K) && out);
  return int8_product(nullptr, 0, const_cast<int8_t*>(codes), K, const_cast<float*>(scales), weight, nullptr, bias, is_bf16, T, N, K, out,
                      static_cast<cudaStream_t>(stream));
}

extern "C" int dmoq_int8_gated_gemm(const int8_t* codes, const float* scales, const int8_t* w_gate, int64_t gate_pitch, const float* gate_scale,
                                    const int8_t* w_up, int64_t up_pitch, const float* up_scale, int32_t is_bf16, int32_t T, int32_t I,
                                    int32_t K, void* out, void* stream) {
  const int rc = check_sizes8(T, I, K);
  if (rc != DMOQ_OK || T == 0) return rc;
  const Weight8 gate = {w_gate, gate_pitch, gate_scale}, up = {w_up, up_pitch, up_scale};
  DMOQ_CHECK_ARG(usable(codes) && scales && weight8_ok(gate, K) && weight8_ok(up, K) && out);
  return int8_product(nullptr, 0, const_cast<int8_t*>(codes), K, const_cast<float*>(scales), gate, &up, nullptr, is_bf16, T, I, K, out,
                      static_cast<cudaStream_t>(stream));
}

namespace {
// Scratch of the two calls below: the codes, then the scales.  A row of codes starts on a 128-byte line whatever K is: a box row
// that straddles two lines costs the L2 a quarter more sectors (1111 tokens, 10936 x 4112 twice: 98 us became 83).
long long scratch_pitch(int K) { return (K + 127) / 128 * 128; }
float* scratch_scales(void* scratch, int T, int K) {
  return reinterpret_cast<float*>(static_cast<char*>(scratch) + (size_t)T * scratch_pitch(K));
}
}  // namespace

extern "C" size_t dmoq_int8_scratch_bytes(int32_t T, int32_t N, int32_t K, int32_t gated) {
  if (check_sizes8(T, N, K) != DMOQ_OK || few_can_fuse(T, K, N, gated != 0)) return 0;
  return (size_t)T * scratch_pitch(K) + (size_t)T * sizeof(float);
}

extern "C" int dmoq_int8_linear(const void* x, int32_t is_bf16, int64_t x_pitch, const int8_t* w, int64_t w_pitch, const float* w_scale,
                                const void* bias, int32_t T, int32_t N, int32_t K, void* scratch, void* out, void* stream) {
  const int rc = check_sizes8(T, N, K);
  if (rc != DMOQ_OK || T == 0) return rc;
  const Weight8 weight = {w, w_pitch, w_scale};
  DMOQ_CHECK_ARG(rows_usable(x, x_pitch, K) && weight8_ok(weight, K) && out && (few_can_fuse(T, K, N, false) || usable(scratch)));
  return int8_product(x, x_pitch, static_cast<int8_t*>(scratch), scratch_pitch(K), scratch_scales(scratch, T, K), weight, nullptr, bias, is_bf16,
                      T, N, K, out, static_cast<cudaStream_t>(stream));
}

extern "C" int dmoq_int8_gated_linear(const void* x, int32_t is_bf16, int64_t x_pitch, const int8_t* w_gate, int64_t gate_pitch,
                                      const float* gate_scale, const int8_t* w_up, int64_t up_pitch, const float* up_scale, int32_t T,
                                      int32_t I, int32_t K, void* scratch, void* out, void* stream) {
  const int rc = check_sizes8(T, I, K);
  if (rc != DMOQ_OK || T == 0) return rc;
  const Weight8 gate = {w_gate, gate_pitch, gate_scale}, up = {w_up, up_pitch, up_scale};
  DMOQ_CHECK_ARG(rows_usable(x, x_pitch, K) && weight8_ok(gate, K) && weight8_ok(up, K) && out &&
                 (few_can_fuse(T, K, I, true) || usable(scratch)));
  return int8_product(x, x_pitch, static_cast<int8_t*>(scratch), scratch_pitch(K), scratch_scales(scratch, T, K), gate, &up, nullptr, is_bf16, T,
                      I, K, out, static_cast<cudaStream_t>(stream));
}

extern "C" int dmoq_gated_ffn(const void* x, int32_t is_bf16, int64_t x_pitch, const void* w_gate, int64_t gate_pitch, const void* w_up,
                              int64_t up_pitch, const void* w_down, int64_t down_pitch, int32_t T, int32_t H, int32_t I,
                              void* h, int64_t h_pitch, void* saved, void* y, void* stream) {
  const int size = check_ffn(T, H, I);
  if (size != DMOQ_OK || T == 0) return size;
  DMOQ_CHECK_ARG(rows_usable(x, x_pitch, H) && rows_usable(w_gate, gate_pitch, H) && rows_usable(w_up, up_pitch, H) &&
                 rows_usable(w_down, down_pitch, I) && rows_usable(h, h_pitch, I) && usable(y));
  DMOQ_CHECK_ARG(aligned16(saved));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  Product up;
  up.epi = saved ? EPI_SILU_SAVE : EPI_SILU;
  up.a[0] = {x, T, H, x_pitch};
  up.b[0] = {w_gate, I, H, gate_pitch};
  up.b[1] = {w_up, I, H, up_pitch};
  up.args.M = T, up.args.N = I, up.args.K = H, up.args.segs = 1, up.args.bf16 = is_bf16, up.args.vec = 1;
  up.args.out[0] = static_cast<uint16_t*>(h);
  for (int e = 0; saved && e < 3; ++e) up.args.out[1 + e] = static_cast<uint16_t*>(saved) + e * (size_t)T * I;
  up.args.ld_out = h_pitch;
  up.args.ld_saved = I;
  const long long w_bytes = 2LL * H * I;
  int rc = few_tokens(T, 2 * w_bytes) && !saved
               ? few_product(KIND_16, EPI_SILU, x, 2 * x_pitch, w_gate, 2 * gate_pitch, w_up, 2 * up_pitch, up.args, s)
               : run(up, s);
  if (rc != DMOQ_OK) return rc;
  Product down;
  down.a[0] = {h, T, I, h_pitch};
  down.b[0] = {w_down, H, I, down_pitch};
  down.args.M = T, down.args.N = H, down.args.K = I, down.args.segs = 1, down.args.bf16 = is_bf16, down.args.vec = 1;
  down.args.out[0] = static_cast<uint16_t*>(y);
  down.args.ld_out = H;
  return few_tokens(T, w_bytes) ? few_product(KIND_16, EPI_OUT, h, 2 * h_pitch, w_down, 2 * down_pitch, nullptr, 0, down.args, s) : run(down, s);
}

extern "C" int dmoq_gated_ffn_backward(const void* dy, int64_t dy_pitch, const void* x, int32_t is_bf16, int64_t x_pitch, const void* w_gate,
                                       int64_t gate_pitch, const void* w_up, int64_t up_pitch, const void* w_down, int64_t down_pitch, int32_t T,
                                       int32_t H, int32_t I, const void* h,
                                       int64_t h_pitch, const void* saved, void* d_gate_up, int64_t d_pitch, void* dx, void* dw_gate, void* dw_up,
                                       void* dw_down, void* stream) {
  const int size = check_ffn(T, H, I);
  if (size != DMOQ_OK) return size;
  if (T > kMaxGradTokens) return DMOQ_ESIZE;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const size_t w_bytes = (size_t)H * I * 2;
  if (T == 0) {   // no tokens: the weights' gradients are zero
    void* dw[3] = {dw_gate, dw_up, dw_down};
    for (void* p : dw)
      if (p && cudaMemsetAsync(p, 0, w_bytes, s) != cudaSuccess) return DMOQ_ELAUNCH;
    return DMOQ_OK;
  }
  const bool inner = dx || dw_gate || dw_up;    // anything behind the hidden values
  DMOQ_CHECK_ARG(aligned16(dx) && aligned16(dw_gate) && aligned16(dw_up) && aligned16(dw_down));
  DMOQ_CHECK_ARG(!(inner || dw_down) || rows_usable(dy, dy_pitch, H));
  DMOQ_CHECK_ARG(!dw_down || rows_usable(h, h_pitch, I));
  DMOQ_CHECK_ARG(!inner || (rows_usable(w_down, down_pitch, I) && usable(saved) && rows_usable(d_gate_up, d_pitch, 2 * I)));
  DMOQ_CHECK_ARG(!dx || (rows_usable(w_gate, gate_pitch, H) && rows_usable(w_up, up_pitch, H)));
  DMOQ_CHECK_ARG(!(dw_gate || dw_up) || rows_usable(x, x_pitch, H));
  uint16_t* dg = static_cast<uint16_t*>(d_gate_up);
  int rc = DMOQ_OK;
  if (inner) {   // dh = dy Wd; dg = dh u silu'(g), du = dh silu(g), side by side in rows of 2 I
    Product p;
    p.epi = EPI_GRAD;
    p.b_mn = true;
    p.a[0] = {dy, T, H, dy_pitch};
    p.b[0] = {w_down, H, I, down_pitch};
    p.args.M = T, p.args.N = I, p.args.K = H, p.args.segs = 1, p.args.bf16 = is_bf16, p.args.vec = 1;
    for (int e = 0; e < 3; ++e) p.args.in[e] = static_cast<const uint16_t*>(saved) + e * (size_t)T * I;
    p.args.ld_in = I;
    p.args.out[0] = dg;
    p.args.out[1] = dg + I;
    p.args.ld_out = d_pitch;
    if ((rc = run(p, s)) != DMOQ_OK) return rc;
  }
  Product px, pg, pd;   // dx, dw_gate and dw_up, dw_down
  auto output = [&](Product& p, int M, int N, int K, int segs, void* out) {
    p.args.M = M, p.args.N = N, p.args.K = K, p.args.segs = segs, p.args.bf16 = is_bf16, p.args.vec = 1;
    p.args.out[0] = static_cast<uint16_t*>(out);
    p.args.ld_out = N;
  };
  if (dx) {             // dg Wg + du Wu: one sum over two K segments
    px.b_mn = true;
    px.a[0] = {dg, T, I, d_pitch};
    px.a[1] = {dg + I, T, I, d_pitch};
    px.b[0] = {w_gate, I, H, gate_pitch};
    px.b[1] = {w_up, I, H, up_pitch};
    output(px, T, H, I, 2, dx);
  }
  auto weight_grad = [&](Product& p, const Matrix& a, const Matrix& b, void* out) {   // a^T b, both along the tokens
    p.a_mn = p.b_mn = true;
    p.a[0] = a;
    p.b[0] = b;
    output(p, (int)a.cols, (int)b.cols, T, 1, out);
  };
  const Matrix xm = {x, T, H, x_pitch};
  const bool joined = dw_gate && dw_up && static_cast<char*>(dw_up) == static_cast<char*>(dw_gate) + w_bytes;
  if (joined) weight_grad(pg, {dg, T, 2 * (long long)I, d_pitch}, xm, dw_gate);   // one product for both halves
  if (dw_down) weight_grad(pd, {dy, T, H, dy_pitch}, {h, T, I, h_pitch}, dw_down);
  if (dx && joined && dw_down) return run_gradients(px, pg, pd, s);
  if (dx && (rc = run(px, s)) != DMOQ_OK) return rc;
  if (joined) {
    if ((rc = run(pg, s)) != DMOQ_OK) return rc;
  } else {
    Product p;
    if (dw_gate) {
      weight_grad(p, {dg, T, I, d_pitch}, xm, dw_gate);
      if ((rc = run(p, s)) != DMOQ_OK) return rc;
    }
    if (dw_up) {
      weight_grad(p, {dg + I, T, I, d_pitch}, xm, dw_up);
      if ((rc = run(p, s)) != DMOQ_OK) return rc;
    }
  }
  return dw_down ? run(pd, s) : DMOQ_OK;
}
