// rotary_f32.hip -- rotary positions and head norms of f32 elements.
#include "rotary_kernels.hpp"

namespace vkfx {

int launch_rotary_f32(const RotaryArgs& a, hipStream_t s, bool back) { return launch_layout<float>(a, s, back); }

}  // namespace vkfx
