// Sampling (sample.cuh): a token of each row.
#include "sample.cuh"

namespace fnx {

int launch_sample(SampleArgs a, cudaStream_t stream) { return launch_rows<false>(a, stream); }

}  // namespace fnx
