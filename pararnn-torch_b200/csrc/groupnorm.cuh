// Group norm with an activation: arguments shared by the kernels (groupnorm.cu) and the C ABI.
#pragma once
#include "kernels.h"

namespace prb {

enum Activation : int { kActNone = 0, kActSilu = 1, kActGelu = 2 };

struct GroupNormArgs {
    const void *x, *dy, *w, *b;  // w, b (channels,) or null
    void *y, *dx, *dw, *db;
    float2* stats;      // (samples, groups): mean, rstd
    float* partial;     // rows of [2][channels]: sum du xhat, sum du
    float* group_part;  // float4 per (sample of the piece, slab, group, channel block of the group)
    long long samples, sample0, sample1;  // all samples; first and end of the piece
    int positions, channels, groups, act, w_f32, slabs, span;
    float eps;
};

struct GroupNormPlan {
    int rows, vec, nv, lanes, blocks, slabs;
    int span;           // channel blocks that a group can touch
    int walkers;        // CTAs per slab that share the samples of a piece (backward sums)
    long long piece;    // samples per pair of launches
    long long part_rows;
    size_t group_floats;
};

GroupNormPlan groupnorm_plan(int dtype, long long samples, int positions, int channels, int groups, bool backward);
cudaError_t launch_groupnorm(const GroupNormArgs& a, int dtype, bool backward, cudaStream_t s);

}  // namespace prb
