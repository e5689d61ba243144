// linear_f32.hip -- chunk kernels of linear attention for f32 elements.
#include "linear_chunk.hpp"

namespace vkfx {

const ChunkKernel* chunk_kernel_f32(int dk, int dv, bool gradient) { return pick_chunk_kernel<float>(dk, dv, gradient); }

}  // namespace vkfx
