// The matrix products' kernels for fp16 operands.
#include "mhc_gemm.hpp"

namespace mhc {
namespace gemm {

int run_product_f16(const Product& p, bool a_k, bool b_k, const Cut& c, float* part, hipStream_t s) {
  return run_product<_Float16>(p, a_k, b_k, c, part, s);
}

}  // namespace gemm
}  // namespace mhc
