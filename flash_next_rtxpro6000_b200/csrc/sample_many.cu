// Sampling (sample.cuh) for many rows.
#include "sample.cuh"

namespace fnx {

const void* sample_fn_many(int type) { return sample_fn<true, false>(type); }

}  // namespace fnx
