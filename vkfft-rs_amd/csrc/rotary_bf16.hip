// rotary_bf16.hip -- rotary positions and head norms of bf16 elements.
#include "rotary_kernels.hpp"

namespace vkfx {

int launch_rotary_bf16(const RotaryArgs& a, hipStream_t s, bool back) { return launch_layout<__bf16>(a, s, back); }

}  // namespace vkfx
