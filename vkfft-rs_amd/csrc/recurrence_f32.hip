// recurrence_f32.hip -- the gated recurrence of f32 elements.
#include "recurrence_kernels.hpp"

namespace vkfx {

int launch_recurrence_f32(const RecurrenceArgs& a, hipStream_t s, bool back) { return launch_channels<float>(a, s, back); }

}  // namespace vkfx
