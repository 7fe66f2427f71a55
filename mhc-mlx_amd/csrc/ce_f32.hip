// linear_cross_entropy's products for fp32 operands.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

MHC_CE_DEFINE(f32, float)

}  // namespace ce
}  // namespace mhc
