// Sampling (sample.cuh): a token of each row.
#include "sample.cuh"

namespace fnx {

const void* sample_fn_one(int type) { return sample_fn<false, false>(type); }

int launch_sample(SampleArgs a, cudaStream_t stream) { return launch_rows<false>(a, stream); }

}  // namespace fnx
