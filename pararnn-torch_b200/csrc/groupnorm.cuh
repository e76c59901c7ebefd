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
    float* group_part;  // per (sample, slab, channel block, group) float4
    long long samples, sample0;
    int positions, channels, groups, act, w_f32, slabs;
    float eps;
};

struct GroupNormPlan {
    int rows, vec, nv, lanes, blocks, slabs;
    long long part_rows;
    size_t group_floats;
};

GroupNormPlan groupnorm_plan(int dtype, long long samples, int positions, int channels, int groups, bool backward);
cudaError_t launch_groupnorm(const GroupNormArgs& a, int dtype, bool backward, cudaStream_t s);

}  // namespace prb
