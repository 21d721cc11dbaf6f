// The backward walk of the gated recurrence for one storage type.
#include "recurrence.cuh"

namespace dsb {

template <>
int run_recurrence_backward<__half>(const RecurrenceLaunch& c, cudaStream_t s) { return run_walk<__half, false>(c, s); }

}  // namespace dsb
