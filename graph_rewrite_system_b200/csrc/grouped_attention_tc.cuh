// The tensor-core launcher of the grouped attention (bf16).
#pragma once

#include "grouped_attention.cuh"

namespace grs {

// whether both slots of a CTA take the same rows and halves of a slice's keys
// (the batch fits one tile of 128 rows); slices then come in pairs
inline bool grouped_tc_split(int positions, int group) { return positions <= 128 / group; }

// Widths that are multiples of 8 up to 128, groups up to 128, 16-byte aligned
// rows with positive strides.
bool grouped_tc_takes(const GroupedArgs<__nv_bfloat16>& a);
int grouped_tc_launch(const GroupedArgs<__nv_bfloat16>& a, cudaStream_t stream);

}  // namespace grs
