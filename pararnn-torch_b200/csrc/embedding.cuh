// Embedding lookup and its gradient: arguments shared by the kernels (embedding.cu) and the C ABI.
#pragma once
#include "kernels.h"

namespace prb {

struct EmbedArgs {
    const void* ids;    // (tokens,) int32 or int64
    const void* table;  // (vocab, channels)
    const void* dy;     // (tokens, channels)
    void* out;          // (tokens, channels), or (vocab, channels) gradient
    long long tokens;
    int vocab, channels, ids64;
    float scale;
};

// workspace of the gradient, offsets in bytes
struct EmbedPlan {
    size_t counters, counts, offsets, rank, pos, sorted, segs, piece_seg, partial, total;
    long long max_segs, max_pieces;
};

EmbedPlan embedding_plan(long long tokens, int vocab, int channels);
cudaError_t launch_embedding(const EmbedArgs& a, int dtype, cudaStream_t s);
cudaError_t launch_embedding_grad(const EmbedArgs& a, int dtype, void* ws, cudaStream_t s);

}  // namespace prb
