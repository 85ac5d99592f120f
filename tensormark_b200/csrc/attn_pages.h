// attn_pages.h — the kernels behind tm_cuda_attn_paged_dev and tm_cuda_attn_window_dev, and which of them serves what.
#pragma once

#include "kv_pages.cuh"

namespace tmc {

struct AttnCall {
    KvBatch c;
    KvMask mask;
    const float* q;
    float* out;
    uint32_t H, rep;            // query heads; of them to a K/V head
    uint32_t max_q;             // a sequence with more new tokens is out of range
    uint32_t few;               // rows (new tokens x rep) of a sequence up to which attn_few.cu serves it; 0: none
    bool others;                // sequences with more rows are served by another launch of the same call
    float scale;
    int* status;
    bool tiled;                 // attn_few.cu: rows in tiles (launch_attn_tiled sets it)
};

// attn_few.cu: sequences with at most 8 or 16 query rows per K/V head (attn_pages.cu, split)
constexpr uint32_t kChunkRows = 256, kFewRows = 16, kFewCtas = 296;       // two CTAs on each of 148 SMs
size_t attn_few_scratch(uint32_t rows, uint32_t dh);
bool launch_attn_few(const AttnCall& a, bool half, float* scratch, cudaStream_t st);

// Sequences with more rows, in tiles of row_tile: 256 over fp16 caches (attn_chunk.cu), 16 over fp32 ones (attn_few.cu).
// The keys of a tile of rows are split over the CTAs of a cluster, which merge: as many as keep the SMs busy, a power of two up to 8.
struct ChunkPlan { uint32_t slots, splits; };           // (sequence, tile of rows) at most; parts
ChunkPlan plan_attn_chunk(uint32_t T, uint32_t B, uint32_t KVH, uint32_t rep, uint32_t few, uint32_t row_tile);
bool launch_attn_chunk(const AttnCall& a, const ChunkPlan& pl, cudaStream_t st);
bool launch_attn_tiled(AttnCall a, const ChunkPlan& pl, cudaStream_t st);

}  // namespace tmc
