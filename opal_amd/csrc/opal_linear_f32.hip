// The matrix products of the score head for elements of type float (opal_linear.h).
#include "opal_linear.h"

namespace opal_head {
template <> hipError_t launch_linear<float>(const Linear &g, int product, int tile, bool dma, hipStream_t stream)
{
    OPAL_LINEAR_FEW_WEIGHT(float)
    OPAL_LINEAR_SMALL(float, FWD)
    OPAL_LINEAR_SMALL(float, GIN)
    OPAL_LINEAR_CASES(float, GWT)
    OPAL_LINEAR_FEW(float, FWD, 1)
    OPAL_LINEAR_FEW(float, FWD, 2)
    OPAL_LINEAR_FEW(float, FWD, 4)
    OPAL_LINEAR_FEW(float, GIN, 1)
    OPAL_LINEAR_FEW(float, GIN, 2)
    OPAL_LINEAR_FEW(float, GIN, 4)
    return hipErrorInvalidValue;
}
}  // namespace opal_head
