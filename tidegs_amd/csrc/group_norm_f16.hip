// The group norm's kernels for half tensors.
#define GN_TYPE f16_t
#include "group_norm.cuh"
