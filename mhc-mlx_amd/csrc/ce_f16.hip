// linear_cross_entropy's products for fp16 operands.
#include "mhc_ce.hpp"

namespace mhc {
namespace ce {

MHC_CE_DEFINE(f16, _Float16)

}  // namespace ce
}  // namespace mhc
