// linear_int8: out = act(xs ws (x W^T) + bias) + residual for int8 codes x and
// W with a scale for each row (of tokens, and of channels).
//
// The products' sums are whole numbers in 32 bits, exact: a term is at most
// 2^14, and there are fewer than 2^17 of them.  They are scaled in registers
// on their way to the epilogue, each of the two scales and the sum's way to
// fp32 one rounding.  (Where few outputs leave CUs idle, the reduction is cut
// into up to 16 parts, which are scaled each and added in fp32.)
#include "mhc_operand.hpp"

namespace mhc {
namespace {

using gemm::Cut;
using gemm::Epilogue;
using gemm::Operand;
using gemm::Product;

constexpr int64_t kMaxK = 1 << 17;

struct Scales {
  const float* x;     // [M]
  const float* w;     // [N]
  const float* bias;  // [N], or NULL
};

// int32 sums to fp32 values, with the bias (in the first of a reduction's
// parts).  The tile's scales are loaded before its sums are formed, one or two
// numbers a thread, and shared through LDS after them.  So that the residuals
// are in L2 by then, one of each of their lines is loaded too, and dropped
// (1001 x 2050 x 1100, operands from memory: 15.4 to 14.3 us).
template <typename O>
struct Scaled {
  Scales s;

  static constexpr int kMost = 4;
  struct Own {
    float scale, bias;
    uint32_t touched[kMost];
  };

  template <int BM, int BN, int WM, int WN>
  MHC_DEV Own ahead(const Product& p, const gemm::Place<BM, BN, WM, WN>& at) const {
    constexpr int kThreads = 64 * WM * WN, kLine = 128, kLines = BN * (int)sizeof(O) / kLine;  // of a row of the tile
    constexpr int kTouch = (BM * kLines + kThreads - 1) / kThreads;
    static_assert(BM + BN <= kThreads, "a scale for each thread");
    static_assert(kTouch <= kMost, "lines of a tile's residuals");
    const int t = threadIdx.x;
    const int64_t n = min(at.n0 + (t < BM ? 0 : t - BM), p.N - 1);
    const float* const scale = t < BM ? s.x + min(at.m0 + t, p.M - 1) : s.w + n;
    Own own = {*scale, s.bias != nullptr && t >= BM ? s.bias[n] : 0.f, {}};
#pragma unroll
    for (int i = 0; i < kTouch; ++i) {
      const int line = i * kThreads + t;
      const int64_t m = min(at.m0 + line / kLines, p.M - 1), c = min(at.n0 + line % kLines * (kLine / (int)sizeof(O)), p.N - 1);
      // (without residuals a scale: a load under a condition would wait for itself)
      const void* const from = p.e.residual != nullptr ? static_cast<const void*>(static_cast<const O*>(p.e.residual) + m * p.N + c) : s.x;
      if constexpr (sizeof(O) == 4) own.touched[i] = *static_cast<const uint32_t*>(from);
      else own.touched[i] = *static_cast<const uint16_t*>(from);
    }
    return own;
  }

  template <int BM, int BN, int WM, int WN, int JM, int JN>
  MHC_DEV void operator()(const Product&, const gemm::Place<BM, BN, WM, WN>& at, int split, char* smem, const Own& own,
                          f32x4 (&acc)[JN][JM]) const {
    float* const lds = reinterpret_cast<float*>(smem);  // of rows, of columns, biases
    const int t = threadIdx.x;
#pragma unroll
    for (int i = 0; i < kMost; ++i) asm volatile("" ::"v"(own.touched[i]));
    lds_barrier();  // nobody reads the stages any more
    if (t < BM + BN) lds[t] = own.scale;
    if (t >= BM && t < BM + BN) lds[BN + t] = own.bias;
    lds_barrier();
    float x[JM];
#pragma unroll
    for (int j = 0; j < JM; ++j) x[j] = lds[at.wm + j * 16 + at.lane % 16];
#pragma unroll
    for (int i = 0; i < JN; ++i) {
      const float* const of_columns = lds + BM + at.wn + i * 16 + at.lane / 16 * 4;
      const f32x4 w = *reinterpret_cast<const f32x4*>(of_columns);
      f32x4 b = {0.f, 0.f, 0.f, 0.f};
      if (split == 0) b = *reinterpret_cast<const f32x4*>(of_columns + BN);
#pragma unroll
      for (int j = 0; j < JM; ++j) {
        const gemm::i32x4 sum = __builtin_bit_cast(gemm::i32x4, acc[i][j]);
        f32x4 v;
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = fmaf((float)sum[k] * x[j], w[k], b[k]);
        acc[i][j] = v;
      }
    }
  }
};

template <typename O, int BM, int BN, int WM, int WN, int NS>
__global__ __launch_bounds__(64 * WM * WN) void int8_tile_kernel(const Product p, const Scaled<O> then) {
  __shared__ __attribute__((aligned(1024))) char smem[gemm::TileBytes<int8_t, BM, BN, WM, WN, NS>::kAll];
  Product q = p;
  q.e.dact = nullptr;  // (known here, so that no derivative is formed)
  // (without a derivative, large tiles have the registers for four rows at a time: with a residual and gelu_tanh 2048 x 8192 x
  // 4096 79 to 72 us)
  gemm::run_tile<int8_t, true, true, BM, BN, WM, WN, NS, O, BM * BN == 65536 ? 4 : 2>(q, smem, blockIdx.x, (int)blockIdx.y, p.M * p.N, p.N, then);
}

// Up to 64 rows: as few_rows_kernel, with the waves' sums joined as whole numbers.
template <typename O, int MT, int NT, int NS>
__global__ __launch_bounds__(64 * gemm::kFewWaves) void int8_few_rows_kernel(const Operand x, const Operand w, int M, int64_t N, int K,
                                                                            const Scales s, const Epilogue e) {
  constexpr int kN = 16 * NT, kSums = MT * 16 * kN;
  __shared__ __attribute__((aligned(1024))) char smem[std::max(gemm::kFewBytes<MT, NT, NS>, gemm::kFewWaves * kSums * 4)];
  const int64_t n0 = (int64_t)blockIdx.x * kN;
  f32x4 acc[NT][MT] = {};
  gemm::sum_few_rows<int8_t, MT, NT, NS>(x, w, M, n0, N, K, smem, acc);
  int* const sums = reinterpret_cast<int*>(smem);
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) *reinterpret_cast<f32x4*>(sums + ((wave * MT + j) * 16 + lane % 16) * kN + i * 16 + lane / 16 * 4) = acc[i][j];
  __syncthreads();
  for (int at = threadIdx.x; at < kSums; at += 64 * gemm::kFewWaves) {
    const int m = at / kN;
    const int64_t n = n0 + at % kN;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < gemm::kFewWaves; ++v) sum += sums[v * kSums + at];
    if (m < M && n < N) {
      const float none[1] = {};
      float z[1][1] = {{fmaf((float)sum * s.x[m], s.w[n], s.bias != nullptr ? s.bias[n] : 0.f)}}, residual[1][1];
      Epilogue f = e;
      f.dact = nullptr;  // (known here, so that no derivative is formed)
      gemm::residual_of<O, true>(f, m, 0, M, n, N, 1, residual);
      gemm::finish<O, true>(f, m, 0, M, n, N, 1, z, none, residual);
    }
  }
}

template <typename O, int BM, int BN, int WM, int WN, int NS>
int launch_tile(const Product& p, const Scaled<O>& then, hipStream_t s) {
  const dim3 grid((unsigned)(ceil_div(p.M, BM) * ceil_div(p.N, BN)), (unsigned)p.splits), block(64 * WM * WN);
  hipLaunchKernelGGL((int8_tile_kernel<O, BM, BN, WM, WN, NS>), grid, block, 0, s, p, then);
  MHC_CHECK_LAUNCH("int8_tile_kernel");
  return MHC_OK;
}

template <typename O>
int run_tiles(Product p, const Cut& c, const Scaled<O>& then, float* part, hipStream_t s) {
  const Epilogue e = p.e;
  p.splits = c.splits;
  p.kper = c.kper;
  if (c.splits > 1) p.e = Epilogue{nullptr, nullptr, part, nullptr, MHC_ACT_NONE, 1};
  int rc;
  switch (c.tile) {
    case 0: rc = launch_tile<O, 256, 256, 2, 4, 2>(p, then, s); break;
    case 1: rc = launch_tile<O, 128, 256, 2, 4, 2>(p, then, s); break;
    case 2: rc = launch_tile<O, 128, 128, 4, 2, 2>(p, then, s); break;
    case 3: rc = launch_tile<O, 64, 128, 4, 2, 3>(p, then, s); break;
    default: rc = launch_tile<O, 64, 64, 4, 1, 3>(p, then, s); break;
  }
  if (rc != MHC_OK || c.splits == 1) return rc;
  return gemm::launch_join<O>(e, part, c.splits, p.M, p.N, s);
}

template <typename O, int MT>
int run_few(const Operand& x, const Operand& w, int64_t M, int64_t N, int64_t K, const Scales& scales, const Epilogue& e, hipStream_t s) {
  hipLaunchKernelGGL((int8_few_rows_kernel<O, MT, 1, MT == 1 ? 2 : 1>), dim3((unsigned)ceil_div(N, 16)), dim3(64 * gemm::kFewWaves), 0, s, x, w,
                     (int)M, N, (int)K, scales, e);
  MHC_CHECK_LAUNCH("int8_few_rows_kernel");
  return MHC_OK;
}

// Whether the product goes to the kernel for few rows: up to 64 of them, unless
// tiles are estimated faster.  A workgroup of it has 16 columns and reads all of
// x, and takes 0.35, 0.65 or 1.05 us for 1024 k of 16, 32 or 64 rows (64 x 4096 x
// 4096 8.1 us, tiles 11.7; 64 x 16384 x 1024 10.0 and 6.3); W's bytes go by at 5
// TB/s there, in tiles at 6 (16 x 32000 x 4096 25.5 and 21.9, 48 rows 37.6 and 22.5).
bool few_rows(int64_t M, int64_t N, int64_t K) {
  if (M > 64) return false;
  const float of_cu = std::max(1.f, (float)N / 16.f / (float)device_cu_count()), bytes = (float)(N * K) * 1e-6f;
  const float few = 2.5f + of_cu * (float)ceil_div(K, 1024) * (M <= 16 ? 0.35f : M <= 32 ? 0.65f : 1.05f);
  return std::max(few, bytes / 5.f) <= std::max(gemm::cut_of(M, N, K, kI8, true, true).us, bytes / 6.f);
}

template <typename O>
int run(const Product& p, const Scales& scales, float* part, hipStream_t s) {
  if (few_rows(p.M, p.N, p.K)) {
    if (p.M <= 16) return run_few<O, 1>(p.a, p.b, p.M, p.N, p.K, scales, p.e, s);
    if (p.M <= 32) return run_few<O, 2>(p.a, p.b, p.M, p.N, p.K, scales, p.e, s);
    return run_few<O, 4>(p.a, p.b, p.M, p.N, p.K, scales, p.e, s);
  }
  return run_tiles<O>(p, gemm::cut_of(p.M, p.N, p.K, kI8, true, true), Scaled<O>{scales}, part, s);
}

}  // namespace
}  // namespace mhc

extern "C" size_t mhc_linear_int8_workspace_bytes(const int8_t* x, int64_t ldx, const int8_t* w, int64_t ldw, int64_t M, int64_t N, int64_t K) {
  using namespace mhc;
  if (M <= 0 || N <= 0 || K <= 0 || K >= kMaxK) return 0;
  return gemm::pack_bytes(x, M, ldx, K, kI8) + gemm::pack_bytes(w, N, ldw, K, kI8) +
         (few_rows(M, N, K) ? 0 : gemm::part_bytes(gemm::cut_of(M, N, K, kI8, true, true), M, N));
}

extern "C" int mhc_linear_int8(const int8_t* x, int64_t ldx, const float* x_scales, const int8_t* w, int64_t ldw, const float* w_scales,
                               const float* bias, const void* residual, void* out, int out_dtype, int act, int64_t M, int64_t N, int64_t K,
                               void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  MHC_CHECK_ARG(M >= 0 && N >= 1 && K >= 1, "M must be >= 0, N and K >= 1 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
  MHC_CHECK_ARG(M < ((int64_t)1 << 28) && N < ((int64_t)1 << 22), "M must be below 2^28, N below 2^22 (got %lld, %lld)", (long long)M, (long long)N);
  // (a launch has fewer than 2^32 threads: tiles of 256 x 256 with 512 each, or of 64 x 64 with 256 for small M or N)
  MHC_CHECK_ARG((M / 256 + 1) * (N / 256 + 1) < ((int64_t)1 << 22), "M times N is too large (got %lld, %lld)", (long long)M, (long long)N);
  MHC_CHECK_ARG(K < kMaxK, "K must be below 2^17, so that sums stay in 32 bits (got %lld)", (long long)K);
  MHC_CHECK_ARG(out_dtype == kF32 || out_dtype == kBF16 || out_dtype == kF16, "unsupported out_dtype %d", out_dtype);
  MHC_CHECK_ARG(act >= MHC_ACT_NONE && act <= MHC_ACT_SILU, "unknown activation %d", act);
  if (M == 0) return MHC_OK;
  MHC_CHECK_ARG(x && x_scales && w && w_scales && out, "null pointer");
  MHC_CHECK_ARG((ldx >= K || M == 1) && (ldw >= K || N == 1), "ldx and ldw must be at least K");
  MHC_CHECK_ARG(workspace_bytes >= mhc_linear_int8_workspace_bytes(x, ldx, w, ldw, M, N, K), "workspace too small");
  MHC_CHECK_ARG(workspace_bytes == 0 || workspace != nullptr, "null workspace");
  MHC_CHECK_ARG(aligned(workspace, 16), "workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  Product p = {{}, {}, M, N, K, Epilogue{nullptr, residual, out, nullptr, act, out_dtype == kF32}, 1, 0};
  if (const int rc = gemm::operand(p.a, x, M, ldx, K, kI8, ws, s)) return rc;
  if (const int rc = gemm::operand(p.b, w, N, ldw, K, kI8, ws, s)) return rc;
  const Scales scales = {x_scales, w_scales, bias};
  float* const part = reinterpret_cast<float*>(ws);
  if (out_dtype == kF32) return run<float>(p, scales, part, s);
  if (out_dtype == kBF16) return run<__bf16>(p, scales, part, s);
  return run<_Float16>(p, scales, part, s);
}
