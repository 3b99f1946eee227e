// Sampling (sample.cuh): a token of each row.
//
// Here the compiler inlines the steps' lambdas by itself, and in another order than when it is made to: fp32 rows keep
// their registers (20 bytes of spills otherwise), and a row of 151,936 with a top-k of 50 takes 10.6 us against 11.0, 16 rows
// without top-k 40.7 against 41.8.  In the units of the other forms some are left out then.
#define FNX_INLINE_STEP
#include "sample.cuh"

namespace fnx {

const void* sample_fn_one(int type) { return sample_fn<false, false>(type); }

int launch_sample(SampleArgs a, cudaStream_t stream) { return launch_rows<false>(a, stream); }

}  // namespace fnx
