// RMS norm with the residual's addition, its int8 form, and its gradients.
//
//   h = x + r, rounded to their type: what the next block adds to is what is normed
//   s = 1 / sqrt(mean h^2 + eps);  y = h s w
//   int8: a = max |h w|;  code = rint(127 h w / a);  scale = a s / 127
//   g = dy w;  n = h s;  dx = dr = s (g - n mean(g n)) + dh;  dw = sum_t dy n
//
// s cancels in the codes, so that they need only a row's largest product: of
// 16-bit values and weights the products and 127 times them are exact in fp32,
// and so is the code, ties included.
//
// Bound by memory: a row is read once and written once.
#include "mhc_gemm.hpp"
#include "mhc_plan.hpp"

namespace mhc {
namespace {

constexpr int kLongThreads = 1024;  // of the kernels for rows of any length
constexpr int kMaxRows = 1 << 20;   // workgroups of a launch; further rows go round again

struct NormArgs {
  const void* x;
  const void* r;   // or NULL
  const void* w;   // or NULL: ones
  int64_t ldx, ldr;
  void* h;         // [T, C], written if there is an r
  void* y;         // [T, C], or int8 codes
  float* scales;   // [T] of the codes
  float* rstd;     // [T], or NULL
  int64_t T;
  int C;
  float eps;
};

enum Mode { kPlain, kCodes, kCodesOnly };  // kCodesOnly: of x itself, without a norm

template <typename T> constexpr int kV = 16 / (int)sizeof(T);  // elements of a vector

// a value over all of a workgroup's threads, in every thread, in a fixed order
template <int THREADS, typename Op>
MHC_DEV float join_threads(float v, Op op, float* lds) {
  v = group_reduce<kWave>(v, op);
  if constexpr (THREADS == kWave) return v;
  const int wave = threadIdx.x / kWave;
  __syncthreads();
  if (threadIdx.x % kWave == 0) lds[wave] = v;
  __syncthreads();
  v = lds[0];
#pragma unroll
  for (int k = 1; k < THREADS / kWave; ++k) v = op(v, lds[k]);
  return v;
}

// The larger of two magnitudes, as bit patterns: NaN is larger than infinity, and that than any number.
struct LargerOp {
  MHC_DEV float operator()(float a, float b) const {
    return __builtin_bit_cast(float, max(__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)));
  }
};

// Codes of values p from the largest magnitude of their row.  Both are scaled
// by a power of two first, so that 127 p and the quotient stay in range; the
// quotient is corrected by its remainder, which makes it the nearest number to
// 127 p / top.  A row of zeros has codes of 0 and the scale 0, one with an
// infinity or NaN codes of 0 and the scale NaN.
struct Coder {
  float up, top, inv;
  bool some;

  MHC_DEV explicit Coder(float t) {
    const uint32_t e = min(max(__builtin_bit_cast(uint32_t, t) >> 23, 1u), 253u);
    up = __builtin_bit_cast(float, (254u - e) << 23);
    some = t > 0.f && t < __builtin_inff();
    top = some ? t * up : 1.f;
    inv = 1.f / top;
  }
  MHC_DEV int code(float p) const {
    const float a = 127.f * (p * up), q = a * inv;
    return some ? (int)rintf(fmaf(fmaf(-q, top, a), inv, q)) : 0;
  }
  static MHC_DEV float scale(float t, float s) { return t < __builtin_inff() ? t * s / 127.f : __builtin_nanf(""); }
};

template <bool WHOLE, int V>
MHC_DEV void put_codes(int8_t* p, const Coder& c, const float (&v)[V], int left) {
  uint32_t w[V / 4];
#pragma unroll
  for (int k = 0; k < V / 4; ++k)
    w[k] = (uint32_t)(c.code(v[4 * k]) & 255) | (uint32_t)(c.code(v[4 * k + 1]) & 255) << 8 | (uint32_t)(c.code(v[4 * k + 2]) & 255) << 16 |
           (uint32_t)c.code(v[4 * k + 3]) << 24;
  if constexpr (WHOLE) {
    __builtin_memcpy(p, w, V);
  } else {
#pragma unroll
    for (int k = 0; k < V; ++k)
      if (k < left) p[k] = (int8_t)(w[k / 4] >> (8 * (k % 4)));
  }
}

// the weights of a vector's elements
template <bool WHOLE, typename T, int V>
MHC_DEV void weights_of(const void* w, bool f32, int64_t n, int left, float (&v)[V]) {
  if (w == nullptr) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = 1.f;
  } else if (f32) {
    gemm::take<WHOLE>(static_cast<const float*>(w) + n, v, left);
  } else if constexpr (sizeof(T) == 2) {
    gemm::take<WHOLE>(static_cast<const T*>(w) + n, v, left);
  }
}

// s of a row from its sum of squares.  Squares past fp32's range are summed
// once more, of values scaled by the row's largest (sum(k) gives that of the
// values times k, largest() their largest magnitude).
template <typename Sum, typename Largest>
MHC_DEV float factor_of(float squares, int C, float eps, Sum sum, Largest largest) {
  if (squares < __builtin_inff()) return 1.f / sqrtf(squares / (float)C + eps);
  const float top = largest();
  if (!(top < __builtin_inff())) return top == __builtin_inff() ? 0.f : top;
  const float k = __builtin_bit_cast(float, (254u - min(__builtin_bit_cast(uint32_t, top) >> 23, 253u)) << 23);
  return k / sqrtf(sum(k) / (float)C + eps * k * k);
}

// --------------------------------------------------------------------------
// Rows of any length: a workgroup goes over a row twice
// --------------------------------------------------------------------------

template <typename T, int MODE>
__global__ __launch_bounds__(kLongThreads) void norm_long_kernel(const NormArgs a, int w_f32) {
  constexpr int V = kV<T>;
  __shared__ float lds[kLongThreads / kWave];
  const int C = a.C, vecs = (C + V - 1) / V;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const T* row = static_cast<const T*>(a.x) + t * a.ldx;
    const auto each = [&](const T* from, auto&& use) {
      for (int v = threadIdx.x; v < vecs; v += kLongThreads) {
        const int left = min(V, C - v * V);
        float z[V];
        if (left == V) {
          gemm::take<true>(from + v * V, z, V);
          use(v * V, left, z, std::true_type{});
        } else {
          gemm::take<false>(from + v * V, z, left);
          use(v * V, left, z, std::false_type{});
        }
      }
    };
    float squares = 0.f, top = 0.f;
    T* const h = static_cast<T*>(a.h) + t * C;
    each(row, [&](int n, int left, float(&z)[V], auto whole) {
      constexpr bool W = decltype(whole)::value;
      if (a.r != nullptr) {
        float r[V];
        gemm::take<W>(static_cast<const T*>(a.r) + t * a.ldr + n, r, left);
#pragma unroll
        for (int k = 0; k < V; ++k) {
          z[k] += r[k];
          if constexpr (sizeof(T) == 2) z[k] = from16<T>(bits16<T>(z[k]));
        }
        gemm::put<W>(h + n, z, left);
      }
      float w[V];
      if (MODE != kPlain) weights_of<W, T>(a.w, w_f32, n, left, w);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        squares = fmaf(z[k], z[k], squares);
        if (MODE != kPlain) top = LargerOp{}(top, fabsf(z[k] * w[k]));
      }
    });
    if (a.r != nullptr) row = h;  // (each thread reads what it wrote)
    float s = 1.f;
    if constexpr (MODE != kCodesOnly) {
      squares = join_threads<kLongThreads>(squares, SumOp{}, lds);
      s = factor_of(
          squares, C, a.eps,
          [&](float by) {
            float q = 0.f;
            each(row, [&](int, int, float(&z)[V], auto) {
#pragma unroll
              for (int k = 0; k < V; ++k) q = fmaf(z[k] * by, z[k] * by, q);
            });
            return join_threads<kLongThreads>(q, SumOp{}, lds);
          },
          [&] {
            float m = 0.f;
            each(row, [&](int, int, float(&z)[V], auto) {
#pragma unroll
              for (int k = 0; k < V; ++k) m = LargerOp{}(m, fabsf(z[k]));
            });
            return join_threads<kLongThreads>(m, LargerOp{}, lds);
          });
    }
    if constexpr (MODE != kPlain) top = join_threads<kLongThreads>(top, LargerOp{}, lds);
    if (threadIdx.x == 0) {
      if (MODE == kPlain && a.rstd != nullptr) a.rstd[t] = s;
      if (MODE != kPlain) a.scales[t] = Coder::scale(top, s);
    }
    const Coder coder(top);
    each(row, [&](int n, int left, float(&z)[V], auto whole) {
      constexpr bool W = decltype(whole)::value;
      float w[V];
      weights_of<W, T>(a.w, w_f32, n, left, w);
      if constexpr (MODE == kPlain) {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] = z[k] * s * w[k];
        gemm::put<W>(static_cast<T*>(a.y) + t * C + n, z, left);
      } else {
#pragma unroll
        for (int k = 0; k < V; ++k) z[k] *= w[k];
        put_codes<W>(static_cast<int8_t*>(a.y) + t * C + n, coder, z, left);
      }
    });
  }
}

// --------------------------------------------------------------------------
// Gradients
// --------------------------------------------------------------------------

struct NormBwdArgs {
  const void* dy;
  const void* dh;  // or NULL
  const void* h;
  const float* rstd;
  const void* w;   // or NULL
  int64_t lddy, lddh, ldh;
  void* dx;        // [T, C], or NULL
  float* part;     // sums of dw, [workgroups, C], or NULL
  int64_t T;
  int C;
};

template <typename T>
__global__ __launch_bounds__(kLongThreads) void norm_bwd_long_kernel(const NormBwdArgs a, int w_f32) {
  constexpr int V = kV<T>;
  __shared__ float lds[kLongThreads / kWave];
  const int C = a.C, vecs = (C + V - 1) / V;
  for (int64_t t = blockIdx.x; t < a.T; t += gridDim.x) {
    const float s = a.rstd[t];
    // g and n of a vector
    const auto each = [&](auto&& use) {
      for (int v = threadIdx.x; v < vecs; v += kLongThreads) {
        const int n = v * V, left = min(V, C - n);
        const auto one = [&](auto whole) {
          constexpr bool W = decltype(whole)::value;
          float g[V], h[V], w[V];
          gemm::take<W>(static_cast<const T*>(a.dy) + t * a.lddy + n, g, left);
          gemm::take<W>(static_cast<const T*>(a.h) + t * a.ldh + n, h, left);
          weights_of<W, T>(a.w, w_f32, n, left, w);
#pragma unroll
          for (int k = 0; k < V; ++k) {
            g[k] *= w[k];
            h[k] *= s;
          }
          use(n, left, g, h, whole);
        };
        if (left == V) one(std::true_type{});
        else one(std::false_type{});
      }
    };
    float along = 0.f;
    each([&](int, int, float(&g)[V], float(&h)[V], auto) {
#pragma unroll
      for (int k = 0; k < V; ++k) along = fmaf(g[k], h[k], along);
    });
    along = join_threads<kLongThreads>(along, SumOp{}, lds) / (float)C;
    each([&](int n, int left, float(&g)[V], float(&h)[V], auto whole) {
      constexpr bool W = decltype(whole)::value;
      float d[V] = {};
      if (a.dh != nullptr) gemm::take<W>(static_cast<const T*>(a.dh) + t * a.lddh + n, d, left);
#pragma unroll
      for (int k = 0; k < V; ++k) d[k] = fmaf(s, g[k] - h[k] * along, d[k]);
      gemm::put<W>(static_cast<T*>(a.dx) + t * C + n, d, left);
    });
  }
}

constexpr int kDwCols = 64 * 8;  // columns of a workgroup of norm_dw_kernel

int dw_rows(int64_t T, int C) { return (int)std::max<int64_t>(16, ceil_div(T * ceil_div(C, kDwCols), 4 * device_cu_count())); }

// sums of dy n over a workgroup's rows, to part[block of rows][C]: for rows too long to be held by norm_bwd_kernel
template <typename T>
__global__ __launch_bounds__(256) void norm_dw_kernel(const NormBwdArgs a, int rows, uint32_t wide) {
  __shared__ float lds[4][kDwCols];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t block = blockIdx.x / wide;
  const int n0 = (int)(blockIdx.x % wide) * kDwCols, n = n0 + lane * 8, left = min(8, a.C - n);
  const int64_t t0 = (int64_t)block * rows, t1 = min(t0 + rows, a.T);
  float sum[8] = {};
  if (left > 0) {
    for (int64_t t = t0 + wave; t < t1; t += 4) {
      float g[8], h[8];
      if (left == 8) {
        gemm::take<true>(static_cast<const T*>(a.dy) + t * a.lddy + n, g, 8);
        gemm::take<true>(static_cast<const T*>(a.h) + t * a.ldh + n, h, 8);
      } else {
        gemm::take<false>(static_cast<const T*>(a.dy) + t * a.lddy + n, g, left);
        gemm::take<false>(static_cast<const T*>(a.h) + t * a.ldh + n, h, left);
      }
      const float s = a.rstd[t];
#pragma unroll
      for (int k = 0; k < 8; ++k) sum[k] = fmaf(g[k], h[k] * s, sum[k]);
    }
  }
#pragma unroll
  for (int k = 0; k < 8; ++k) lds[wave][lane * 8 + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < kDwCols; c += 256)
    if (n0 + c < a.C) a.part[(int64_t)block * a.C + n0 + c] = (lds[0][c] + lds[1][c]) + (lds[2][c] + lds[3][c]);
}

template <typename W>
__global__ __launch_bounds__(256) void norm_dw_join_kernel(const float* part, W* dw, int64_t rows, int64_t C) {
  __shared__ float lds[8][gemm::kSumCols];
  gemm::sum_columns<256>(lds, part, dw, rows, C, blockIdx.x);
}

unsigned grid_of(int64_t T) { return (unsigned)std::min<int64_t>(T, kMaxRows); }

template <typename T, int MODE>
int run_norm(const NormArgs& a, int w_f32, hipStream_t s) {
  hipLaunchKernelGGL((norm_long_kernel<T, MODE>), dim3(grid_of(a.T)), dim3(kLongThreads), 0, s, a, w_f32);
  MHC_CHECK_LAUNCH("norm_long_kernel");
  return MHC_OK;
}

template <int MODE>
int run_norm(const NormArgs& a, int dtype, int w_f32, hipStream_t s) {
  if (dtype == kF32) return run_norm<float, MODE>(a, w_f32, s);
  if (dtype == kBF16) return run_norm<__bf16, MODE>(a, w_f32, s);
  return run_norm<_Float16, MODE>(a, w_f32, s);
}

// rows of the sums of dw
int64_t part_rows(int64_t T, int C) { return ceil_div(T, dw_rows(T, C)); }

template <typename T>
int run_bwd(const NormBwdArgs& a, int w_f32, void* dw, hipStream_t s) {
  if (a.dx != nullptr) {
    hipLaunchKernelGGL((norm_bwd_long_kernel<T>), dim3(grid_of(a.T)), dim3(kLongThreads), 0, s, a, w_f32);
    MHC_CHECK_LAUNCH("norm_bwd_long_kernel");
  }
  if (dw == nullptr) return MHC_OK;
  const int64_t blocks = part_rows(a.T, a.C);
  const uint32_t wide = (uint32_t)ceil_div(a.C, kDwCols);
  hipLaunchKernelGGL((norm_dw_kernel<T>), dim3(wide * (uint32_t)blocks), dim3(256), 0, s, a, dw_rows(a.T, a.C), wide);
  MHC_CHECK_LAUNCH("norm_dw_kernel");
  const dim3 grid((unsigned)ceil_div(a.C, gemm::kSumCols));
  if (w_f32) hipLaunchKernelGGL((norm_dw_join_kernel<float>), grid, dim3(256), 0, s, (const float*)a.part, static_cast<float*>(dw), blocks, a.C);
  else hipLaunchKernelGGL((norm_dw_join_kernel<T>), grid, dim3(256), 0, s, (const float*)a.part, static_cast<T*>(dw), blocks, a.C);
  MHC_CHECK_LAUNCH("norm_dw_join_kernel");
  return MHC_OK;
}

int check_shape(int64_t T, int64_t C, int dtype) {
  MHC_CHECK_ARG(T >= 0 && C >= 1, "T must be >= 0 and C >= 1 (got %lld, %lld)", (long long)T, (long long)C);
  MHC_CHECK_ARG(C < ((int64_t)1 << 24), "C must be below 2^24 (got %lld)", (long long)C);  // (vectors of a row are counted in 32 bits)
  MHC_CHECK_ARG(dtype == kF32 || dtype == kBF16 || dtype == kF16, "unsupported dtype %d", dtype);
  return MHC_OK;
}

int check_norm(const void* x, int64_t ldx, const void* r, int64_t ldr, const void* w, int w_dtype, const void* h, int64_t T, int64_t C,
               int dtype, float eps) {
  if (const int rc = check_shape(T, C, dtype)) return rc;
  MHC_CHECK_ARG(w == nullptr || w_dtype == dtype || w_dtype == kF32, "w_dtype must be the rows' or fp32 (got %d)", w_dtype);
  MHC_CHECK_ARG(eps > 0.f && eps < __builtin_inff(), "eps must be positive (got %g)", (double)eps);
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(x != nullptr && (r == nullptr || h != nullptr), "null pointer");
  MHC_CHECK_ARG((ldx >= C || T == 1) && (r == nullptr || ldr >= C || T == 1), "ldx and ldr must be at least C");
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

extern "C" int mhc_add_rms_norm_fwd(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, void* h,
                                    void* y, float* rstd, int64_t T, int64_t C, int dtype, float eps, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_norm(x, ldx, residual, ldr, w, w_dtype, h, T, C, dtype, eps)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(y != nullptr, "null pointer");
  const NormArgs a = {x, residual, w, ldx, ldr, h, y, nullptr, rstd, T, (int)C, eps};
  return run_norm<kPlain>(a, dtype, w_dtype == kF32, static_cast<hipStream_t>(stream));
}

extern "C" int mhc_add_rms_norm_int8(const void* x, int64_t ldx, const void* residual, int64_t ldr, const void* w, int w_dtype, void* h,
                                     int8_t* codes, float* scales, int64_t T, int64_t C, int dtype, float eps, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_norm(x, ldx, residual, ldr, w, w_dtype, h, T, C, dtype, eps)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(codes != nullptr && scales != nullptr, "null pointer");
  const NormArgs a = {x, residual, w, ldx, ldr, h, codes, scales, nullptr, T, (int)C, eps};
  return run_norm<kCodes>(a, dtype, w_dtype == kF32, static_cast<hipStream_t>(stream));
}

extern "C" int mhc_quantize_int8(const void* x, int64_t ldx, int8_t* codes, float* scales, int64_t T, int64_t C, int dtype, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(T, C, dtype)) return rc;
  if (T == 0) return MHC_OK;
  MHC_CHECK_ARG(x != nullptr && codes != nullptr && scales != nullptr, "null pointer");
  MHC_CHECK_ARG(ldx >= C || T == 1, "ldx must be at least C");
  const NormArgs a = {x, nullptr, nullptr, ldx, 0, nullptr, codes, scales, nullptr, T, (int)C, 1.f};
  return run_norm<kCodesOnly>(a, dtype, 0, static_cast<hipStream_t>(stream));
}

extern "C" size_t mhc_add_rms_norm_bwd_workspace_bytes(int64_t T, int64_t C, int dtype) {
  (void)dtype;
  if (T <= 0 || C <= 0 || C >= ((int64_t)1 << 24)) return 0;
  return (size_t)(mhc::part_rows(T, (int)C) * C) * sizeof(float);
}

extern "C" int mhc_add_rms_norm_bwd(const void* dy, int64_t lddy, const void* dh, int64_t lddh, const void* h, int64_t ldh, const float* rstd,
                                    const void* w, int w_dtype, void* dx, void* dw, int64_t T, int64_t C, int dtype, void* workspace,
                                    size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(T, C, dtype)) return rc;
  MHC_CHECK_ARG(T > 0, "T must be > 0");
  MHC_CHECK_ARG((w == nullptr && dw == nullptr) || w_dtype == dtype || w_dtype == kF32, "w_dtype must be the rows' or fp32 (got %d)", w_dtype);
  MHC_CHECK_ARG(dy != nullptr && h != nullptr && rstd != nullptr, "null pointer");
  MHC_CHECK_ARG((lddy >= C && ldh >= C && (dh == nullptr || lddh >= C)) || T == 1, "rows must be at least C apart");
  MHC_CHECK_ARG(dw == nullptr || (workspace != nullptr && workspace_bytes >= mhc_add_rms_norm_bwd_workspace_bytes(T, C, dtype)),
                "workspace too small");
  MHC_CHECK_ARG(aligned(workspace, 16), "workspace must be 16-byte aligned");
  if (dx == nullptr && dw == nullptr) return MHC_OK;
  const NormBwdArgs a = {dy, dh, h, rstd, w, lddy, lddh, ldh, dx, static_cast<float*>(workspace), T, (int)C};
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == kF32) return run_bwd<float>(a, 1, dw, s);
  if (dtype == kBF16) return run_bwd<__bf16>(a, w_dtype == kF32, dw, s);
  return run_bwd<_Float16>(a, w_dtype == kF32, dw, s);
}
