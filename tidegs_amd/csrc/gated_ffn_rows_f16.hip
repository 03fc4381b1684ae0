// The gated feed-forward block over narrow rows of f16 values.
#include "gated_ffn_rows.cuh"

template struct RowKernels<f16_t>;
