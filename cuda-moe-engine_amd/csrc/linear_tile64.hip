// The 64 x 64 tiles of the dense products, in a file of their own for the time they take to compile.
#include "linear_ring.h"

namespace moe {
template void run_dense<64, 64, 53 * 1024, 2>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
}  // namespace moe
