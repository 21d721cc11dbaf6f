// The forward walk of the gated recurrence for one storage type.
#include "recurrence.cuh"

namespace dsb {

template <>
int run_recurrence_forward<__half>(const RecurrenceLaunch& c, cudaStream_t s) { return run_walk<__half, true>(c, s); }

}  // namespace dsb
