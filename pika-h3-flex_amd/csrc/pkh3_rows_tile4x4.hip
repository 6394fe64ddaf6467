// The products of pkh3_rows_tile.h with tiles of 128 rows of A and 128 of B.
#include "pkh3_rows_tile.h"

namespace pkh3 {

hipError_t launch_tiles_4x4(const ProductParams& p, const ProductPlan& plan, bool a_across, bool b_across, int mode, hipStream_t s) {
  return launch_tiles_of<4, 4>(p, plan, a_across, b_across, mode, s);
}

}  // namespace pkh3
