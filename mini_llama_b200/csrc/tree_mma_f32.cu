// Attention of drafted tokens over fp32 caches: the matrix-instruction kernels.
#include "tree_mma.cuh"

namespace mlb {

bool LaunchTreeF32(DeviceContext& ctx, const TreeArgs& a) { return LaunchBlocks<MLB_F32>(ctx, a); }

}  // namespace mlb
