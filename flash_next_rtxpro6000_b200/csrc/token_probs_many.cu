// The kept tokens of many rows (sample.cuh), for their probabilities.
#include "sample.cuh"

namespace fnx {

const void* probs_fn_many(int type) { return sample_fn<true, true>(type); }

}  // namespace fnx
