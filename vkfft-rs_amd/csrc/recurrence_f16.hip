// recurrence_f16.hip -- the gated recurrence of f16 elements.
#include "recurrence_kernels.hpp"

namespace vkfx {

int launch_recurrence_f16(const RecurrenceArgs& a, hipStream_t s, bool back) { return launch_channels<_Float16>(a, s, back); }

}  // namespace vkfx
