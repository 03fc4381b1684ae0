// The gated feed-forward block over narrow rows of bf16 values.
#include "gated_ffn_rows.cuh"

template struct RowKernels<bf16_t>;
