// The matrix products of the score head for elements of type bf16_t (opal_linear.h).
#include "opal_linear_pair.h"

namespace opal_head {
template <> hipError_t launch_linear<bf16_t>(const Linear &g, int product, int tile, bool dma, hipStream_t stream)
{
    if (tile == 4 && dma && product == FWD) return launch_pair<bf16_t>(g, stream);
    if (tile == 2 && dma) return launch_big<bf16_t>(g, product, stream);
    OPAL_LINEAR_FEW_WEIGHT(bf16_t)
    OPAL_LINEAR_CASES(bf16_t, FWD)
    OPAL_LINEAR_CASES(bf16_t, GIN)
    OPAL_LINEAR_CASES(bf16_t, GWT)
    OPAL_LINEAR_FEW(bf16_t, FWD, 1)
    OPAL_LINEAR_FEW(bf16_t, FWD, 2)
    OPAL_LINEAR_FEW(bf16_t, FWD, 4)
    OPAL_LINEAR_FEW(bf16_t, GIN, 1)
    OPAL_LINEAR_FEW(bf16_t, GIN, 2)
    OPAL_LINEAR_FEW(bf16_t, GIN, 4)
    return hipErrorInvalidValue;
}
}  // namespace opal_head
