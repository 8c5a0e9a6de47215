// Entry to the kernel for requests with few rows (chunk_attn_few.cu).
#pragma once

#include "chunk_attn.cuh"

namespace subspec {

// Tensor map of a layer's rows for tiles (of a CTA or a warp) of `rows` cache rows; sets ka.box_rows.
void chunk_tensor_map(ChunkArgs& ka, int rows, CUtensorMap* map);
// Scratch for ka.few_rows (16 or 32).
size_t chunk_few_scratch_bytes(const ChunkArgs& ka);
// Every request of ka.few_rows rows (token, head of the group) or less.  `scratch` 16-byte aligned.
int launch_chunk_few(ChunkArgs& ka, float* scratch, cudaStream_t stream);

}  // namespace subspec
