// Dense product over 4-bit floating-point blocks: the tiles on the bf16 matrix cores (f4_wide.h has the kernel).
#include "f4_wide.h"

namespace mx {
namespace f4 {
namespace {

template <int P, bool OI>
int run_tile(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int tile, int slices) {
  if constexpr (P == 1) {
    switch (tile) {
      case 0: return run_f4_wide<WideTile<4, 4, OI ? 3 : 2, 1, OI>>(b, name, d, x, slices);
      case 1: return run_f4_wide<WideTile<4, 2, OI ? 4 : 3, 1, OI>>(b, name, d, x, slices);
      case 2: return run_f4_wide<WideTile<2, 2, OI ? 3 : 2, 1, OI>>(b, name, d, x, slices);
      case 3: return run_f4_wide<WideTile<2, 1, 3, 1, OI>>(b, name, d, x, slices);
      default: return run_f4_wide<WideTile<1, 1, 4, 1, OI>>(b, name, d, x, slices);
    }
  } else {
    if constexpr (OI)  // (no LDS for the other layout's)
      if (tile == 0) return run_f4_wide<WideTile<4, 2, 2, P, OI>>(b, name, d, x, slices);
    switch (tile) {
      case 1: return run_f4_wide<WideTile<4, 1, 2, P, OI>>(b, name, d, x, slices);
      case 3: return run_f4_wide<WideTile<2, 1, 2, P, OI>>(b, name, d, x, slices);
      default: return run_f4_wide<WideTile<1, 1, 3, P, OI>>(b, name, d, x, slices);
    }
  }
}

}  // namespace

int wide_run(mx_backend* b, const char* name, const F4DenseDesc& d, const WideX& x, int tile, int slices) {
  if (x.parts == 3)
    return d.oi ? run_tile<3, true>(b, name, d, x, tile, slices) : run_tile<3, false>(b, name, d, x, tile, slices);
  return d.oi ? run_tile<1, true>(b, name, d, x, tile, slices) : run_tile<1, false>(b, name, d, x, tile, slices);
}

}  // namespace f4
}  // namespace mx
