// The 256 x 256 tiles of the dense products, in a file of their own for the time they take to compile.
#include "linear_ring.h"

namespace moe {
template void run_dense<256, 256, 160 * 1024, true>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
}  // namespace moe
