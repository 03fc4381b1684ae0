// The group norm's kernels for float32 tensors.
#define GN_TYPE float
#include "group_norm.cuh"
