// Attention of drafted tokens over Q4_0 caches: the matrix-instruction kernels.
#include "tree_mma.cuh"

namespace mlb {

bool LaunchTreeQ40(DeviceContext& ctx, const TreeArgs& a) { return LaunchBlocks<MLB_Q4_0>(ctx, a); }

}  // namespace mlb
