// linear_cross_entropy's logits of fp32 operands as products of fp16 parts.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

int run_sums_halves(const Product& p, const Cut& c, const int* live, const SumsOf& of, const Halves& halves, hipStream_t s) {
  return run_sums<_Float16, true>(p, RowsOf{nullptr, p.M}, c, live, of, halves, s);
}

int run_dz_halves(const Product& p, const Cut& c, const int* live, int64_t width, const Gradient& g, const Halves& halves, hipStream_t s) {
  return run_live<_Float16, true, true, false, float>(p, c, live, width, GradientOfHalves{g, halves}, nullptr, s);
}

}  // namespace ce
}  // namespace mhc
