// The tiles of the dense product over 8-bit blocks whose operands do not lie in whole aligned 16-byte chunks (odd K, odd N
// of [K, N] weights, arrays from any byte, sizes past 32-bit offsets).  A translation unit of its own, so that the two
// forms compile side by side.
#include "f8_dense_tiles.h"

namespace mx {
namespace f8 {

int staged_run(mx_backend* b, const char* name, const DenseArgs& a, bool wide, int tile, int slices) {
  using Tile128x128 = DenseTile<2, 4, 2, 2>;
  using Tile128x64 = DenseTile<2, 2, 2, 2>;
  using Tile64x64 = DenseTile<1, 2, 2, 2>;
  switch (tile) {
    case 2: return run_dense_tiles<Tile128x128, false, false>(b, name, a, slices);  // (of bfloat16 results alone)
    case 3: return wide ? run_dense_tiles<Tile128x64, true, false>(b, name, a, slices) : run_dense_tiles<Tile128x64, false, false>(b, name, a, slices);
    default: return wide ? run_dense_tiles<Tile64x64, true, false>(b, name, a, slices) : run_dense_tiles<Tile64x64, false, false>(b, name, a, slices);
  }
}

}  // namespace f8
}  // namespace mx
