// Arguments of the channels-last group norm's kernels and its launchers.
#pragma once

#include "exb_seq_common.cuh"

namespace exb {

constexpr int NORM_MAX_GROUP = 16384;      // channels of a group

struct NormArgs {
    View x;                              // (sample, position, channel)
    const void *weight, *bias;           // [C] or null; float when params_f32, else the type of x
    void *y;                             // contiguous
    float *mean, *rstd;                  // [R][G]
    int64_t R, S;
    int C, G, act, params_f32;
    float eps;
    // backward
    View dy;
    void *dx;                            // contiguous
    float *part;                         // partial sums: statistics [R][chunks][G][2] or gradients [rows][2][C]
    int64_t chunk;                       // positions of a block
    int chunks, slab, slabs;             // blocks of a sample; groups of a block; blocks of a row
    int per;                             // channels of a group
    int smem;                            // pairs of shared memory that the map kernels work in
};

int64_t norm_workspace_bytes(int64_t R, int64_t S, int C, int G, int dtype, bool backward);
cudaError_t launch_norm_forward(NormArgs a, int dtype, void *ws, cudaStream_t stream);
cudaError_t launch_norm_backward(NormArgs a, int dtype, void *dweight, void *dbias, void *ws, cudaStream_t stream);

}  // namespace exb
