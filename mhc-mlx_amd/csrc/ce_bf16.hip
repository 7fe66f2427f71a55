// linear_cross_entropy's products for bf16 operands.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

MHC_CE_DEFINE(bf16, __bf16)

}  // namespace ce
}  // namespace mhc
