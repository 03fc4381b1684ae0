// The gated feed-forward block over narrow rows of f32 values.
#include "gated_ffn_rows.cuh"

template struct RowKernels<float>;
