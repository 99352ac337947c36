// The 128 x 128 tiles of the dense products, in a file of their own for the time they take to compile.
#include "linear_ring.h"

namespace moe {
template void run_dense<128, 128, 160 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
template void run_dense<128, 128, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
}  // namespace moe
