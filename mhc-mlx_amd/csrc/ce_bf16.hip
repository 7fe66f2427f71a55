// linear_cross_entropy's products for bf16 operands.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

const Runs& runs_bf16() { return runs_of<__bf16>(); }

}  // namespace ce
}  // namespace mhc
