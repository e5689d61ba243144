// rotary_f16.hip -- rotary positions and head norms of f16 elements.
#include "rotary_kernels.hpp"

namespace vkfx {

int launch_rotary_f16(const RotaryArgs& a, hipStream_t s, bool back) { return launch_layout<_Float16>(a, s, back); }

}  // namespace vkfx
