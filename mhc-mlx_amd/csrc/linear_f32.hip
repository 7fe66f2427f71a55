// The matrix products' kernels for fp32 operands.
#include "mhc_gemm.hpp"

namespace mhc {
namespace gemm {

int run_product_f32(const Product& p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s) {
  return run_product<float>(p, a_k, b_k, c, part, s);
}

int run_pair_f32(const Pair& p, const PairCut& c, float* part, hipStream_t s) { return run_pair<float>(p, c, part, s); }

int run_few_rows_f32(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e,
                 hipStream_t s) {
  return run_few_rows<float>(x, ldx, w, ldw, M, N, K, e, s);
}

}  // namespace gemm
}  // namespace mhc
