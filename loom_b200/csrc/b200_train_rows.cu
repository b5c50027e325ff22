// The norms around a block for one pair of element types (LOOM_ROWS_X of the
// residual stream, LOOM_ROWS_B of the branch) and one direction
// (LOOM_ROWS_BACKWARD), compiled once for each: the kernels are many, and this
// way they compile side by side.
#include "loom_b200_block_norm.cuh"

namespace loomb {
#if LOOM_ROWS_BACKWARD
template int launch_block_norm_grad<LOOM_ROWS_X, LOOM_ROWS_B>(const BlockNorm&, BlockNormGrad,
                                                              int64_t, void*, void*, void*,
                                                              cudaStream_t);
#else
template int launch_block_norm<LOOM_ROWS_X, LOOM_ROWS_B>(const BlockNorm&, const BlockNormOut&,
                                                         cudaStream_t);
#endif
}  // namespace loomb
