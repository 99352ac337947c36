// The tiles of 64 and 96 rows of the dense products, in a file of their own for the time they take to compile.
#include "linear_ring.h"

namespace moe {
template void run_dense<96, 128, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
template void run_dense<64, 128, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
template void run_dense<64, 64, 80 * 1024, false>(const LinearArgs&, const LinearPlan&, int, hipStream_t);
}  // namespace moe
