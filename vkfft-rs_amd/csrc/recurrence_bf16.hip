// recurrence_bf16.hip -- the gated recurrence of bf16 elements.
#include "recurrence_kernels.hpp"

namespace vkfx {

int launch_recurrence_bf16(const RecurrenceArgs& a, hipStream_t s, bool back) { return launch_channels<__bf16>(a, s, back); }

}  // namespace vkfx
