// Dense product over 4-bit floating-point blocks: the tiles on the 4-bit matrix cores (f4_tiles.h has the kernel).
#include "f4_tiles.h"

namespace mx {
namespace f4 {

int tiles_run(mx_backend* b, const char* name, const F4DenseDesc& d, int tile, int slices) {
  switch (tile) {
    case 0: return run_f4_tiles<Tile4<4, 2, 4, 2, 4>>(b, name, d, slices);
    case 1: return run_f4_tiles<Tile4<4, 2, 2, 3, 2>>(b, name, d, slices);
    case 2: return run_f4_tiles<Tile4<2, 4, 1, 3, 4>>(b, name, d, slices);
    case 3: return run_f4_tiles<Tile4<2, 2, 1, 3, 4>>(b, name, d, slices);
    default: return run_f4_tiles<Tile4<1, 2, 1, 4, 4>>(b, name, d, slices);
  }
}

}  // namespace f4
}  // namespace mx
