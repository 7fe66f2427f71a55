// linear_cross_entropy's products for fp16 operands.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

const Runs& runs_f16() { return runs_of<_Float16>(); }

}  // namespace ce
}  // namespace mhc
