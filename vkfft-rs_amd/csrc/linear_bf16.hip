// linear_bf16.hip -- chunk kernels of linear attention for bf16 elements.
#include "linear_chunk.hpp"

namespace vkfx {

const ChunkKernel* chunk_kernel_bf16(int dk, int dv, bool gradient) { return pick_chunk_kernel<__bf16>(dk, dv, gradient); }

}  // namespace vkfx
