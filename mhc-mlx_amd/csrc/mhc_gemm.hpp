// Matrix products out[m, n] = sum_k A(m, k) B(n, k) on MFMA with a fused
// epilogue (gfx950), for fp32, bf16 and fp16 operands.
//
// Each operand is either "k-major" (its k are contiguous: x and W of x W^T)
// or not (its rows are k: W of dz W, and both operands of dz^T x).
#pragma once

#include "mhc_device.hpp"
#include "mhc_host.hpp"

namespace mhc {
namespace gemm {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// --------------------------------------------------------------------------
// Epilogue: out = act(sum + bias) + residual, and act' for a backward
// --------------------------------------------------------------------------

struct Epilogue {
  const void* bias;      // [N] of the operands' type, or NULL
  const void* residual;  // [M, N] of the output's type, or NULL
  void* out;             // [M, N]
  void* dact;            // [M, N] fp32 (fp32 operands) or fp16, or NULL
  int act;               // MHC_ACT_*
  int out_f32;           // out and residual are fp32, else of the operands' type
  int vec;               // four outputs from a column that is a multiple of four are one vector of each array
};

// an epilogue whose `vec` goes by the row length and the addresses (residuals start anywhere)
inline Epilogue epilogue(const void* bias, const void* residual, void* out, void* dact, int act, int out_dtype, int dtype,
                         int64_t N) {
  const int eo = out_dtype == kF32 ? 16 : 8, ed = dtype == kF32 ? 16 : 8;
  const bool vec = N % 4 == 0 && aligned(out, eo) && aligned(residual, eo) && aligned(dact, ed);
  return Epilogue{bias, residual, out, dact, act, out_dtype == kF32, vec};
}

struct Act {
  float y, d;
};

MHC_DEV float sigmoid(float x) { return 1.f / (1.f + expf(-x)); }

// act(z) and act'(z).  NaN goes through each of them.
MHC_DEV Act activate(float z, int act) {
  switch (act) {
    case MHC_ACT_RELU: return {z < 0.f ? 0.f : z, z > 0.f ? 1.f : 0.f};
    case MHC_ACT_GELU: {
      const float p = 0.5f * (1.f + erff(z * 0.70710678f));
      return {z * p, p + z * expf(-0.5f * z * z) * 0.39894228f};
    }
    case MHC_ACT_GELU_TANH: {  // (1 + tanh u) / 2 is sigmoid(2 u)
      const float p = sigmoid(1.59576912f * (z + 0.044715f * z * z * z));
      return {z * p, p + z * p * (1.f - p) * 1.59576912f * (1.f + 0.134145f * z * z)};
    }
    case MHC_ACT_SILU: {
      const float p = sigmoid(z);
      return {z * p, p * (1.f + z * (1.f - p))};
    }
    default: return {z, 1.f};
  }
}

template <typename T> struct DactOf { using Type = _Float16; };
template <> struct DactOf<float> { using Type = float; };

// `C` consecutive outputs of one row, from column n; vec: all C are stored as one vector
template <typename T, int C>
MHC_DEV void finish(const Epilogue& e, int64_t m, int64_t n, int64_t N, float (&z)[C], bool vec) {
  using D = typename DactOf<T>::Type;
  const int64_t at = m * N + n;
  const int left = vec ? C : (int)min((int64_t)C, N - n);
  float d[C];
#pragma unroll
  for (int k = 0; k < C; ++k) {
    if (e.bias != nullptr && k < left) z[k] += load1(static_cast<const T*>(e.bias) + n + k);
    const Act a = activate(z[k], e.act);
    z[k] = a.y;
    d[k] = a.d;
  }
  if (vec) {
    if (e.out_f32) {
      if (e.residual != nullptr) {
        Vec<float, C> r;
        r.load(static_cast<const float*>(e.residual) + at);
#pragma unroll
        for (int k = 0; k < C; ++k) z[k] += r.get(k);
      }
      float* const o = static_cast<float*>(e.out) + at;
#pragma unroll
      for (int k = 0; k < C; k += 4) *reinterpret_cast<f32x4*>(o + k) = f32x4{z[k], z[k + 1], z[k + 2], z[k + 3]};
    } else if constexpr (sizeof(T) == 2) {
      if (e.residual != nullptr) {
        Vec<T, C> r;
        r.load(static_cast<const T*>(e.residual) + at);
#pragma unroll
        for (int k = 0; k < C; ++k) z[k] += r.get(k);
      }
      T* const o = static_cast<T*>(e.out) + at;
#pragma unroll
      for (int k = 0; k < C; k += 4)
        *reinterpret_cast<u32x2*>(o + k) = u32x2{pack2<T>(z[k], z[k + 1]), pack2<T>(z[k + 2], z[k + 3])};
    }
    if (e.dact != nullptr) {
      D* const o = static_cast<D*>(e.dact) + at;
#pragma unroll
      for (int k = 0; k < C; k += 4) {
        if constexpr (sizeof(D) == 4) *reinterpret_cast<f32x4*>(o + k) = f32x4{d[k], d[k + 1], d[k + 2], d[k + 3]};
        else *reinterpret_cast<u32x2*>(o + k) = u32x2{pack2<D>(d[k], d[k + 1]), pack2<D>(d[k + 2], d[k + 3])};
      }
    }
  } else {
#pragma unroll
    for (int k = 0; k < C; ++k) {
      if (k >= left) break;
      if (e.out_f32) {
        if (e.residual != nullptr) z[k] += static_cast<const float*>(e.residual)[at + k];
        static_cast<float*>(e.out)[at + k] = z[k];
      } else {
        if (e.residual != nullptr) z[k] += load1(static_cast<const T*>(e.residual) + at + k);
        store1(static_cast<T*>(e.out) + at + k, z[k]);
      }
      if (e.dact != nullptr) store1(static_cast<D*>(e.dact) + at + k, d[k]);
    }
  }
}

// --------------------------------------------------------------------------
// MFMA
// --------------------------------------------------------------------------

// Sixteen bytes of one row's k a lane: lane l has row l % 16 and the group
// l / 16 of the step's k.  Which k a place holds does not matter as long as
// both operands agree.
template <typename T>
MHC_DEV f32x4 mfma16(const u32x4& a, const u32x4& b, f32x4 c) {
  if constexpr (sizeof(T) == 4) {
    // (the vectors are cast whole: a bit cast of one element of a vector takes its first)
    const f32x4 af = __builtin_bit_cast(f32x4, a), bf = __builtin_bit_cast(f32x4, b);
#pragma unroll
    for (int k = 0; k < 4; ++k) c = __builtin_amdgcn_mfma_f32_16x16x4f32(af[k], bf[k], c, 0, 0, 0);
    return c;
  } else if constexpr (__is_same(T, __bf16)) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  } else {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
}

// --------------------------------------------------------------------------
// The tile kernel: 128 x 128 outputs a workgroup, four waves of 64 x 64
// --------------------------------------------------------------------------

struct Product {
  const void* a;
  const void* b;
  int64_t lda, ldb;  // elements between rows as they are stored
  int64_t M, N, K;
  Epilogue e;
};

constexpr int kTile = 128;
constexpr int kTileThreads = 256;

// LDS holds an operand's tile as rows of its index with eight 16-byte chunks
// of k each; chunk c of row r is at c ^ (r % 8), so that 16 lanes that read
// the same chunk of 16 rows meet different banks.
template <typename T>
struct Stage {
  static constexpr int kE = 16 / (int)sizeof(T);  // elements of a chunk
  static constexpr int kK = 8 * kE;               // k of a stage
  static constexpr int kElems = kTile * kK;
};

template <typename T>
MHC_DEV int lds_at(int row, int chunk) { return (row * 8 + (chunk ^ (row & 7))) * Stage<T>::kE; }

// a chunk of kE elements along k of row i (zeros past the ends)
template <typename T, bool KMAJOR>
MHC_DEV u32x4 fetch(const T* p, int64_t ld, int64_t i, int64_t rows, int64_t k, int64_t K) {
  constexpr int kE = Stage<T>::kE;
  u32x4 r = {0, 0, 0, 0};
  if (i >= rows) return r;
  if (KMAJOR && k + kE <= K) {
    __builtin_memcpy(&r, p + i * ld + k, 16);
    return r;
  }
  T v[kE];
#pragma unroll
  for (int j = 0; j < kE; ++j) v[j] = k + j < K ? (KMAJOR ? p[i * ld + k + j] : p[(k + j) * ld + i]) : (T)0;
  __builtin_memcpy(&r, v, 16);
  return r;
}

template <typename T, bool AK, bool BK>
__global__ __launch_bounds__(kTileThreads) void tile_kernel(const Product p) {
  using S = Stage<T>;
  __shared__ T sa[S::kElems];
  __shared__ T sb[S::kElems];
  const int tid = threadIdx.x, lane = tid % kWave, wave = tid / kWave;
  const int64_t m0 = (int64_t)blockIdx.y * kTile, n0 = (int64_t)blockIdx.x * kTile;
  const int wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  f32x4 acc[4][4] = {};  // [n][m]: the first operand's index runs over a lane's four values
  for (int64_t k0 = 0; k0 < p.K; k0 += S::kK) {
    u32x4 ra[4], rb[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = j * 32 + tid / 8, chunk = tid % 8;
      ra[j] = fetch<T, AK>(static_cast<const T*>(p.a), p.lda, m0 + row, p.M, k0 + chunk * S::kE, p.K);
      rb[j] = fetch<T, BK>(static_cast<const T*>(p.b), p.ldb, n0 + row, p.N, k0 + chunk * S::kE, p.K);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int row = j * 32 + tid / 8, chunk = tid % 8;
      *reinterpret_cast<u32x4*>(sa + lds_at<T>(row, chunk)) = ra[j];
      *reinterpret_cast<u32x4*>(sb + lds_at<T>(row, chunk)) = rb[j];
    }
    __syncthreads();
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 fa[4], fb[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        fa[j] = *reinterpret_cast<const u32x4*>(sa + lds_at<T>(wm + j * 16 + lane % 16, s * 4 + lane / 16));
        fb[j] = *reinterpret_cast<const u32x4*>(sb + lds_at<T>(wn + j * 16 + lane % 16, s * 4 + lane / 16));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = mfma16<T>(fb[i], fa[j], acc[i][j]);
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int64_t m = m0 + wm + j * 16 + lane % 16;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t n = n0 + wn + i * 16 + lane / 16 * 4;
      if (m < p.M && n < p.N) {
        float z[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        finish<T, 4>(p.e, m, n, p.N, z, p.e.vec != 0);
      }
    }
  }
}

// The product of one type; a_k / b_k: the operand's k are contiguous.
template <typename T>
int run_product(const Product& p, bool a_k, bool b_k, hipStream_t s) {
  const dim3 grid((unsigned)ceil_div(p.N, kTile), (unsigned)ceil_div(p.M, kTile));
  if (a_k && b_k) hipLaunchKernelGGL((tile_kernel<T, true, true>), grid, dim3(kTileThreads), 0, s, p);
  else if (a_k) hipLaunchKernelGGL((tile_kernel<T, true, false>), grid, dim3(kTileThreads), 0, s, p);
  else hipLaunchKernelGGL((tile_kernel<T, false, false>), grid, dim3(kTileThreads), 0, s, p);
  MHC_CHECK_LAUNCH("tile_kernel");
  return MHC_OK;
}

int run_product_f32(const Product& p, bool a_k, bool b_k, hipStream_t s);
int run_product_bf16(const Product& p, bool a_k, bool b_k, hipStream_t s);
int run_product_f16(const Product& p, bool a_k, bool b_k, hipStream_t s);

}  // namespace gemm
}  // namespace mhc
