// The 128-row tile form of corm_llm_paged_attn (paged_tile.cu).
#pragma once

#include <cuda_runtime.h>

#include "cormorant_b200.h"

namespace paged {

// whether the form takes the job: 64 or 128 dimensions, row coordinates in 31 bits
bool tile_takes(const corm_llm_paged_attn_desc& d);
// d checked, max_q within the rows; tab: the softmax unit's table, err: the status word
int launch_tiles(const corm_llm_paged_attn_desc& d, const int32_t* tab, int* err, cudaStream_t st);

}  // namespace paged
