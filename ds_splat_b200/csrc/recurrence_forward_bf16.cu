// The forward walk of the gated recurrence for one storage type.
#include "recurrence.cuh"

namespace dsb {

template <>
int run_recurrence_forward<__nv_bfloat16>(const RecurrenceLaunch& c, cudaStream_t s) { return run_walk<__nv_bfloat16, true>(c, s); }

}  // namespace dsb
