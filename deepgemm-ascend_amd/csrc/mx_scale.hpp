// The scale of a microscaled block (mx_quant.hip, mx_product.hip).
#pragma once

#include "dg_common.hpp"

namespace dg {

// Exponent byte of a block whose largest magnitude has the fp32 bits `a`.
template <bool FP4>
__device__ __forceinline__ uint32_t scale_byte(uint32_t a) {
    if (a >= 0x7f800000u) return 255u;
    // (adding what lies between l and 2 carries into the exponent where the mantissa passes l)
    const uint32_t e = (a + (FP4 ? 0x3fffffu : 0x1fffffu)) >> 23;
    return max(e, FP4 ? 3u : 9u) - (FP4 ? 2u : 8u);
}

}  // namespace dg
