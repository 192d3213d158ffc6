// Attention of drafted tokens over Q8_0 caches: the matrix-instruction kernels.
#include "tree_mma.cuh"

namespace mlb {

bool LaunchTreeQ80(DeviceContext& ctx, const TreeArgs& a) { return LaunchBlocks<MLB_Q8_0>(ctx, a); }

}  // namespace mlb
