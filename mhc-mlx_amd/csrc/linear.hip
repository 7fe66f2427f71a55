// linear_act: out = act(x W^T + bias) + residual and its gradients.
//
// The forward is one product with the epilogue in its kernel; for a training
// step it also stores d = act'(z), so that the backward needs neither z nor
// an exponential: dz = dout d is one streaming pass, which also forms db from
// the unrounded dz, and dx = dz W and dW = dz^T x are two more products.
#include "mhc_operand.hpp"

namespace mhc {
namespace {

using gemm::operand;
using gemm::Operand;
using gemm::pack_bytes;
using gemm::padded;
using gemm::part_bytes;
using gemm::Product;
using gemm::up256;

constexpr int kDzCols = 64 * 8;   // columns of a workgroup of dz_kernel: eight for each lane of a wave

// rows of a workgroup: sixteen for each wave, four where those would be too few to fill the card
int dz_rows(int64_t M, int64_t N) { return ceil_div(M, 64) * ceil_div(N, kDzCols) < 2 * device_cu_count() ? 16 : 64; }

// dz = dout dact (dact NULL: dout), rounded to T, in rows of N elements `ld`
// (a multiple of eight) apart with zeros between (not stored if dz is NULL),
// and sums of dz over this workgroup's rows, before rounding, to
// part[block of rows][N] (if not NULL).  One pass at the card's streaming
// rate (8192 x 4096 bf16: 41 us, 4.9 TB/s): a lane has eight columns of every
// fourth row, and loads four rows at a time.
template <typename T, typename G, bool WHOLE>
MHC_DEV void dz_columns(const G* dout, const typename gemm::DactOf<T>::Type* d, T* dz, int64_t ld, int64_t m0, int64_t m1, int64_t n,
                        int64_t N, int left, float (&sum)[8]) {
  for (int64_t m = m0; m < m1; m += 16) {
    float v[4][8], f[4][8];
#pragma unroll
    for (int q = 0; q < 4; ++q) gemm::take<WHOLE>(dout + min(m + 4 * q, m1 - 1) * N + n, v[q], left);
    if (d != nullptr) {
#pragma unroll
      for (int q = 0; q < 4; ++q) gemm::take_dact<WHOLE>(d + min(m + 4 * q, m1 - 1) * N + n, f[q], left);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (m + 4 * q >= m1) break;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (d != nullptr) v[q][k] *= f[q][k];  // (not WHOLE: zeros from `left` on)
        sum[k] += v[q][k];
      }
      if (dz != nullptr) gemm::put<true>(dz + (m + 4 * q) * ld + n, v[q], 8);
    }
  }
}

template <typename T, typename G>
__global__ __launch_bounds__(256) void dz_kernel(const G* dout, const void* dact, T* dz, int64_t ld, float* part, int64_t M,
                                                 int64_t N, int rows, uint32_t wide) {
  __shared__ float lds[4][kDzCols];
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t block = blockIdx.x / wide;  // of rows; `wide` workgroups have its columns
  const int64_t n0 = (int64_t)(blockIdx.x % wide) * kDzCols, n = n0 + lane * 8, m0 = (int64_t)block * rows, m1 = min(m0 + rows, M);
  const auto* const d = static_cast<const typename gemm::DactOf<T>::Type*>(dact);
  float sum[8] = {};
  if (n + 8 <= N) dz_columns<T, G, true>(dout, d, dz, ld, m0 + wave, m1, n, N, 8, sum);
  else if (n < N) dz_columns<T, G, false>(dout, d, dz, ld, m0 + wave, m1, n, N, (int)(N - n), sum);
  if (part == nullptr) return;
#pragma unroll
  for (int k = 0; k < 8; ++k) lds[wave][lane * 8 + k] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < kDzCols; c += 256)
    if (n0 + c < N) part[(int64_t)block * N + n0 + c] = (lds[0][c] + lds[1][c]) + (lds[2][c] + lds[3][c]);
}

// db[n] = sum over the blocks of rows
template <typename T>
__global__ __launch_bounds__(256) void db_kernel(const float* part, T* db, int64_t rows, int64_t N) {
  __shared__ float lds[8][gemm::kSumCols];
  gemm::sum_columns<256>(lds, part, db, rows, N, blockIdx.x);
}

// ws: part_bytes of the product
int run_product(const Product& p, bool a_k, bool b_k, const gemm::Cut& c, int dtype, char* ws, hipStream_t s) {
  float* const part = reinterpret_cast<float*>(ws);
  if (dtype == kF32) return gemm::run_product_f32(p, a_k, b_k, c, part, s);
  if (dtype == kBF16) return gemm::run_product_bf16(p, a_k, b_k, c, part, s);
  return gemm::run_product_f16(p, a_k, b_k, c, part, s);
}

struct BwdPlan {
  size_t dz, part, x, w, total;  // bytes; the products' sums (of one after the other, unless they go together) come last
  gemm::PairCut cut;
};

BwdPlan plan_bwd(const void* dout, int dout_dtype, bool dact, const void* x, int64_t ldx, const void* w, int64_t ldw, bool dx, bool dw,
                 bool db, int64_t M, int64_t N, int64_t K, int dtype) {
  BwdPlan b = {};
  if ((dx || dw) && (dact || dout_dtype != dtype || !gemm::in_words(dout, N, N, gemm::elem_bytes(dtype))))
    b.dz = up256((size_t)(M * padded(N, dtype)) * gemm::elem_bytes(dtype));
  if (db) b.part = up256((size_t)(ceil_div(M, dz_rows(M, N)) * N) * sizeof(float));
  if (dx) b.w = pack_bytes(w, N, ldw, K, dtype);
  if (dw) b.x = pack_bytes(x, M, ldx, K, dtype);
  if (dx && dw) b.cut = gemm::pair_of(M, N, K, dtype);
  else if (dx) b.cut.dx = gemm::cut_of(M, K, N, dtype, true, false);
  else if (dw) b.cut.dw = gemm::cut_of(N, K, M, dtype, false, false);
  const size_t of_dx = dx ? part_bytes(b.cut.dx, M, K) : 0, of_dw = dw ? part_bytes(b.cut.dw, N, K) : 0;
  b.total = b.dz + b.part + b.x + b.w + (b.cut.together ? of_dx + of_dw : std::max(of_dx, of_dw));
  return b;
}

template <typename T, typename G>
int run_dz(const void* dout, const void* dact, void* dz, int64_t ld, float* part, void* db, int64_t M, int64_t N, hipStream_t s) {
  const int rows = dz_rows(M, N);
  const int64_t blocks = ceil_div(M, rows);
  const uint32_t wide = (uint32_t)ceil_div(N, kDzCols);
  hipLaunchKernelGGL((dz_kernel<T, G>), dim3(wide * (uint32_t)blocks), dim3(256), 0, s, static_cast<const G*>(dout), dact,
                     static_cast<T*>(dz), ld, part, M, N, rows, wide);
  MHC_CHECK_LAUNCH("dz_kernel");
  if (db != nullptr) {
    hipLaunchKernelGGL((db_kernel<T>), dim3((unsigned)ceil_div(N, gemm::kSumCols)), dim3(256), 0, s, (const float*)part,
                       static_cast<T*>(db), blocks, N);
    MHC_CHECK_LAUNCH("db_kernel");
  }
  return MHC_OK;
}

int check_shape(int64_t M, int64_t N, int64_t K, int dtype) {
  MHC_CHECK_ARG(M >= 0 && N >= 1 && K >= 1, "M must be >= 0, N and K >= 1 (got %lld, %lld, %lld)", (long long)M,
                (long long)N, (long long)K);
  // (M: the reduction of dW is counted in 32 bits, and a launch has fewer than 2^32 threads; N and K: see gemm::most_rows)
  MHC_CHECK_ARG(M < ((int64_t)1 << 28) && N < ((int64_t)1 << 22) && K < ((int64_t)1 << 22),
                "M must be below 2^28, N and K below 2^22 (got %lld, %lld, %lld)", (long long)M, (long long)N, (long long)K);
  MHC_CHECK_ARG(dtype == kF32 || dtype == kBF16 || dtype == kF16, "unsupported dtype %d", dtype);
  return MHC_OK;
}

}  // namespace
}  // namespace mhc

extern "C" size_t mhc_linear_act_fwd_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M,
                                                     int64_t N, int64_t K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0 || mhc::gemm::few_rows(x, ldx, w, ldw, M, N, K, dtype)) return 0;
  return mhc::gemm::pack_bytes(x, M, ldx, K, dtype) + mhc::gemm::pack_bytes(w, N, ldw, K, dtype) +
         mhc::gemm::part_bytes(mhc::gemm::cut_of(M, N, K, dtype, true, true), M, N);
}

extern "C" int mhc_linear_act_fwd(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                  const void* residual, void* out, int out_dtype, void* dact, int act, int64_t M,
                                  int64_t N, int64_t K, int dtype, void* workspace, size_t workspace_bytes,
                                  void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(M, N, K, dtype)) return rc;
  MHC_CHECK_ARG(out_dtype == dtype || out_dtype == kF32, "out_dtype must be the operands' or fp32 (got %d)", out_dtype);
  MHC_CHECK_ARG(act >= MHC_ACT_NONE && act <= MHC_ACT_SILU, "unknown activation %d", act);
  MHC_CHECK_ARG(act != MHC_ACT_NONE || dact == nullptr, "dact is for an activation");
  if (M == 0) return MHC_OK;
  MHC_CHECK_ARG(x && w && out, "null pointer");
  MHC_CHECK_ARG((ldx >= K || M == 1) && (ldw >= K || N == 1), "ldx and ldw must be at least K");
  MHC_CHECK_ARG(workspace_bytes >= mhc_linear_act_fwd_workspace_bytes(x, ldx, w, ldw, M, N, K, dtype), "workspace too small");
  MHC_CHECK_ARG(aligned(workspace, 16), "workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  if (gemm::few_rows(x, ldx, w, ldw, M, N, K, dtype)) {
    const gemm::Epilogue e = gemm::Epilogue{bias, residual, out, dact, act, out_dtype == kF32};
    if (dtype == kF32) return gemm::run_few_rows_f32(x, ldx, w, ldw, M, N, K, e, s);
    if (dtype == kBF16) return gemm::run_few_rows_bf16(x, ldx, w, ldw, M, N, K, e, s);
    return gemm::run_few_rows_f16(x, ldx, w, ldw, M, N, K, e, s);
  }
  Product p = {{}, {}, M, N, K, gemm::Epilogue{bias, residual, out, dact, act, out_dtype == kF32}, 1, 0};
  if (const int rc = operand(p.a, x, M, ldx, K, dtype, ws, s)) return rc;
  if (const int rc = operand(p.b, w, N, ldw, K, dtype, ws, s)) return rc;
  return run_product(p, true, true, gemm::cut_of(M, N, K, dtype, true, true), dtype, ws, s);
}

extern "C" size_t mhc_linear_act_bwd_workspace_bytes(const void* dout, int dout_dtype, const void* dact, const void* x,
                                                     int64_t ldx, const void* w, int64_t ldw, int want_dx, int want_dw,
                                                     int want_db, int64_t M, int64_t N, int64_t K, int dtype) {
  if (M <= 0 || N <= 0 || K <= 0) return 0;
  return mhc::plan_bwd(dout, dout_dtype, dact != nullptr, x, ldx, w, ldw, want_dx != 0, want_dw != 0, want_db != 0, M, N, K, dtype)
      .total;
}

extern "C" int mhc_linear_act_bwd(const void* dout, int dout_dtype, const void* dact, const void* x, int64_t ldx,
                                  const void* w, int64_t ldw, void* dx, void* dw, void* db, int64_t M, int64_t N,
                                  int64_t K, int dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace mhc;
  clear_error();
  if (const int rc = check_shape(M, N, K, dtype)) return rc;
  MHC_CHECK_ARG(dout_dtype == dtype || dout_dtype == kF32, "dout_dtype must be the operands' or fp32 (got %d)", dout_dtype);
  MHC_CHECK_ARG(M > 0, "M must be > 0");
  MHC_CHECK_ARG(dout && (dw == nullptr || x) && (dx == nullptr || w), "null pointer");
  MHC_CHECK_ARG((dw == nullptr || ldx >= K || M == 1) && (dx == nullptr || ldw >= K || N == 1), "ldx and ldw must be at least K");
  const BwdPlan b = plan_bwd(dout, dout_dtype, dact != nullptr, x, ldx, w, ldw, dx != nullptr, dw != nullptr, db != nullptr, M, N, K,
                             dtype);
  MHC_CHECK_ARG(workspace_bytes >= b.total && (b.total == 0 || workspace != nullptr), "workspace too small");
  MHC_CHECK_ARG(aligned(workspace, 16), "workspace must be 16-byte aligned");
  hipStream_t s = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  void* const dz = b.dz > 0 ? ws : nullptr;
  float* const part = b.part > 0 ? reinterpret_cast<float*>(ws + b.dz) : nullptr;
  if (dz != nullptr || db != nullptr) {
    void* const sum = b.cut.together ? nullptr : db;  // (else by the products' launch)
    int rc;
    if (dtype == kF32) rc = run_dz<float, float>(dout, dact, dz, padded(N, dtype), part, sum, M, N, s);
    else if (dtype == kBF16)
      rc = dout_dtype == kF32 ? run_dz<__bf16, float>(dout, dact, dz, padded(N, dtype), part, sum, M, N, s)
                              : run_dz<__bf16, __bf16>(dout, dact, dz, padded(N, dtype), part, sum, M, N, s);
    else
      rc = dout_dtype == kF32 ? run_dz<_Float16, float>(dout, dact, dz, padded(N, dtype), part, sum, M, N, s)
                              : run_dz<_Float16, _Float16>(dout, dact, dz, padded(N, dtype), part, sum, M, N, s);
    if (rc != MHC_OK) return rc;
  }
  ws += b.dz + b.part;
  const Operand g = dz != nullptr ? Operand{dz, padded(N, dtype), padded(N, dtype)} : Operand{dout, N, N};
  // dx[m, k] = sum_n dz[m, n] W[n, k],  dw[n, k] = sum_m dz[m, n] x[m, k]
  Product px = {g, {}, M, K, N, gemm::Epilogue{nullptr, nullptr, dx, nullptr, MHC_ACT_NONE, dtype == kF32}, 1, 0};
  Product pw = {g, {}, N, K, M, gemm::Epilogue{nullptr, nullptr, dw, nullptr, MHC_ACT_NONE, dtype == kF32}, 1, 0};
  if (dx != nullptr) {
    if (const int rc = operand(px.b, w, N, ldw, K, dtype, ws, s)) return rc;
  }
  if (dw != nullptr) {
    if (const int rc = operand(pw.b, x, M, ldx, K, dtype, ws, s)) return rc;
  }
  if (b.cut.together) {
    const gemm::Pair p = {px, pw, 0, 0, 0, 0, part, db, ceil_div(M, dz_rows(M, N)), N};
    float* const sums = reinterpret_cast<float*>(ws);
    if (dtype == kF32) return gemm::run_pair_f32(p, b.cut, sums, s);
    if (dtype == kBF16) return gemm::run_pair_bf16(p, b.cut, sums, s);
    return gemm::run_pair_f16(p, b.cut, sums, s);
  }
  if (dx != nullptr) {
    if (const int rc = run_product(px, true, false, b.cut.dx, dtype, ws, s)) return rc;
  }
  if (dw != nullptr) {
    if (const int rc = run_product(pw, false, false, b.cut.dw, dtype, ws, s)) return rc;
  }
  return MHC_OK;
}
