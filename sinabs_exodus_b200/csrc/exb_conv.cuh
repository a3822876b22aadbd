// Arguments of the short causal convolution's kernels and its launchers.
#pragma once

#include "exb_seq_common.cuh"

namespace exb {

constexpr int CONV_MAX_WIDTH = 8;

struct ConvArgs {
    View x;
    const void *weight, *bias;           // [M][W], [M] or null; float when params_f32, else the type of x
    const void *state;                   // [B][W-1][M] or null (zeros): the rows in front of x
    const int32_t *lengths;              // [B] or null
    void *y, *last;                      // [B][T][M]; [B][W-1][M] or null
    int64_t B, T;
    int M, W, silu, params_f32;
    // backward
    View dy;
    const void *dlast;                   // [B][W-1][M] or null
    void *dx, *dstate;                   // [B][T][M]; [B][W-1][M] or null
    float *part;                         // [blocks of a channel tile][W + 1][M]
    int64_t run;                         // steps of a thread
};

int64_t conv_backward_workspace_bytes(int64_t B, int64_t T, int M, int W);
cudaError_t launch_conv_forward(ConvArgs a, int dtype, cudaStream_t stream);
cudaError_t launch_conv_backward(ConvArgs a, int dtype, void *dweight, void *dbias, void *ws, cudaStream_t stream);

struct ConvStepArgs {
    View x;                              // st unused
    const void *weight, *bias;
    void *state;                         // [B][W-1][M], shifted by one row
    int64_t ss;                          // elements between two batch items of state
    void *y;                             // [B][M]
    int64_t B;
    int M, W, silu, params_f32;
};
cudaError_t launch_conv_step(const ConvStepArgs &a, int dtype, cudaStream_t stream);

}  // namespace exb
