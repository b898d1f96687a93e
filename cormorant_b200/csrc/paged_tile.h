// The 128-row tile form of corm_llm_paged_attn (paged_tile.cu).
#pragma once

#include <cuda_runtime.h>

#include "cormorant_b200.h"

namespace paged {

// the most (tile, sequence, KV head) with rows, of `tiles` a sequence: the packed rows hold
// no more tiles of n rows (a row being a token and a head of the group) and a part of one a
// sequence
inline uint64_t live_tiles(const corm_llm_paged_attn_desc& d, uint32_t n, uint64_t tiles) {
  const uint64_t packed = ((uint64_t)d.c.rows * (d.H / d.c.KV) + (uint64_t)(n - 1u) * d.c.B) / n, all = tiles * d.c.B;
  return (packed < all ? packed : all) * d.c.KV;
}

// whether the form takes the job: 64 or 128 dimensions, row coordinates in 31 bits
bool tile_takes(const corm_llm_paged_attn_desc& d);
// d checked, max_q within the rows; tab: the softmax unit's table, err: the status word
int launch_tiles(const corm_llm_paged_attn_desc& d, const int32_t* tab, int* err, cudaStream_t st);

}  // namespace paged
