// The chunk form of the attention (attention_chunk.cu) as attention.cu calls it.
#pragma once
#include "attention.cuh"

namespace mpt {

struct ChunkPlan {
    int tiles_per_seq, runs;
    size_t tile_bytes, partial_floats, stats_floats;      // expanded K and V; shares of row tiles that are cut
};

bool chunk_kernel_exists(int dim, int dtype);
ChunkPlan chunk_plan(const CacheView& c, int q_heads);
int launch_chunk(AttentionParams p, const ChunkPlan& pl, uint8_t* tiles, bool fp4, cudaStream_t st);

}  // namespace mpt
