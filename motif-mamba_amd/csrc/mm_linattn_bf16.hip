// mm_linattn_bf16.hip -- the bfloat16 instances of the linear-attention kernels of mm_linattn.hip
// (compiled once per input type, so that the three sets build in parallel).
#define MM_LINATTN_TYPE bf16_t
#include "mm_linattn.hip"
