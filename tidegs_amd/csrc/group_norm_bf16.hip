// The group norm's kernels for bfloat16 tensors.
#define GN_TYPE bf16_t
#include "group_norm.cuh"
