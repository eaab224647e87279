// The backward kernels of the linear recurrence, in a unit of their own (recurrence.hip has the formulas).
#include "igx_recurrence.hpp"

namespace igx {

template void launch_recurrence<true>(int dtype, const Plan &p, hipStream_t s);

}  // namespace igx
