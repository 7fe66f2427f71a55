// linear_cross_entropy's products for fp32 operands.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

const Runs& runs_f32() { return runs_of<float>(); }

}  // namespace ce
}  // namespace mhc
