// The matrix products' kernels for fp16 operands.
#include "mhc_gemm.hpp"

namespace mhc {
namespace gemm {

int run_product_f16(const Product& p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s) {
  return run_product<_Float16>(p, a_k, b_k, c, part, s);
}

int run_pair_f16(const Pair& p, const PairCut& c, float* part, hipStream_t s) { return run_pair<_Float16>(p, c, part, s); }

int run_few_rows_f16(const void* x, int64_t ldx, const void* w, int64_t ldw, int64_t M, int64_t N, int64_t K, const Epilogue& e,
                 hipStream_t s) {
  return run_few_rows<_Float16>(x, ldx, w, ldw, M, N, K, e, s);
}

}  // namespace gemm
}  // namespace mhc
