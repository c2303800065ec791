// mm_linattn_f16.hip -- the float16 instances of the linear-attention kernels of mm_linattn.hip
// (compiled once per input type, so that the three sets build in parallel).
#define MM_LINATTN_TYPE f16_t
#include "mm_linattn.hip"
