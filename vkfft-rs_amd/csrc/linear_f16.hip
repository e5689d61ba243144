// linear_f16.hip -- chunk kernels of linear attention for f16 elements.
#include "linear_chunk.hpp"

namespace vkfx {

const ChunkKernel* chunk_kernel_f16(int dk, int dv, bool gradient) { return pick_chunk_kernel<_Float16>(dk, dv, gradient); }

}  // namespace vkfx
