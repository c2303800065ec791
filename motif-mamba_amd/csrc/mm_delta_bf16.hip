// mm_delta_bf16.hip -- the bfloat16 instances of the gated delta rule's kernels of mm_delta.hip
// (compiled once per input type, so that the three sets build in parallel).
#define MM_DELTA_TYPE bf16_t
#include "mm_delta.hip"
