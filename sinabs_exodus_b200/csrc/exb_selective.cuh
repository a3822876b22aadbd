// Arguments of the selective scan's kernels and its launchers.
#pragma once

#include "exb_seq_common.cuh"

namespace exb {

constexpr int SEL_CHUNK = EXB_SELECTIVE_CHECKPOINT;      // steps between two checkpoints of the state

struct SelArgs {
    View x, dt, z, Bm, Cm;               // z.p may be null
    const float *A, *D, *dt_bias, *h0;   // [M][N], [M], [M], [B][M][N]; all but A may be null
    const int32_t *lengths;              // [B] or null
    int64_t B, T;
    int M, N, G;
    int softplus;
    // forward
    void *y;                             // contiguous
    float *h_last;                       // [B][M][N]
    float *ckpt;                         // [B][ceil(T / SEL_CHUNK)][M][NP], or null
    // backward
    View dy;
    const float *dh_last;                // [B][M][N] or null
    void *dx, *ddt, *dz;                 // contiguous
    float *dh0;                          // [B][M][N] or null
    float *part_bc;                      // [tiles][B][T][G][2][NP]
    float *part_a;                       // [B * segments][M][NP]
    float *part_d;                       // [B * segments][2][M]   (D, dt_bias)
    // time split: `segments` pieces of `seg` steps; what each hands on (state or gradient), and its sum of step sizes
    int segments;
    int64_t seg;
    float *seg_h;                        // [B][segments][M][NP]
    float *seg_dt;                       // [B][segments][M]
};

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether rows can be read four elements at a time.
template <typename T>
bool pack_aligned(const View &v)
{
    return !v.p || (reinterpret_cast<uintptr_t>(v.p) % (4 * sizeof(T)) == 0 && v.sb % 4 == 0 && v.st % 4 == 0);
}

// Rates are kept finite: an infinite one times the step size 0 (of a row behind the sequence, or the input's own) would not be
// the 0 it stands for.
__device__ __forceinline__ float finite_rate(float v) { return min_nan(max_nan(v, -2.0e38f), 2.0e38f); }

// What to add to the exponent e of a decay 2^e, before it is rounded, so that ex2.approx is right on average.  A decay is
// applied over and over: what its errors have in common adds up over a state's memory of 1 / (dt |A|) steps, what is random
// about them does not.  By itself it is low by 1.6e-8 to 2.7e-8 of the value for e from -1 to -2^-8 and by 5e-9 to 9e-9 for
// those nearer to 0, the states with the longest memory (means of a million exponents in each octave).  With this it is right
// to 6.5e-9, and to 2e-9 from -2^-8 to -2^-17; small positive exponents are high by 1.3e-8 to 2e-8 instead of 1e-8.  The
// exponent 0 still gives 1.
__device__ __forceinline__ float decay_lift(float e) { return e < -0x1p-8f ? 2.9e-8f : 8.7e-9f; }

// Lanes per channel: four states in each.
inline int sel_lanes(int N)
{
    int l = 1;
    while (4 * l < N) l *= 2;
    return l;
}

// States of a channel as the scan's kernels keep them (the single step has no use for a second lane of padding).
inline int sel_padded(int N) { const int l = sel_lanes(N); return 4 * (l < 2 ? 2 : l); }

struct SelPlan {
    int L, S, NP, CC, tiles, segments;      // lanes of a channel, states of a lane, their product; channels of a block
    int64_t seg;
    int64_t off_h, off_dt, off_bc, off_a, off_d, bytes;      // offsets into the workspace
};
SelPlan sel_plan(int64_t B, int64_t T, int M, int N, int G, bool backward);

// One translation unit per element type (exb_selective_f32.cu and so on): the kernels come in many shapes.
template <typename T> cudaError_t selective_forward_typed(const SelArgs &a, const SelPlan &p, cudaStream_t s);
template <typename T> cudaError_t selective_backward_typed(const SelArgs &a, const SelPlan &p, void *dB, void *dC, cudaStream_t s);

cudaError_t launch_selective_forward(SelArgs a, int dtype, void *ws, cudaStream_t stream);
cudaError_t launch_selective_backward(SelArgs a, int dtype, void *dB, void *dC, float *dA, float *dD, float *dbias, void *ws,
                                      cudaStream_t stream);

struct SelStepArgs {
    View x, dt, z, Bm, Cm;               // st unused
    const float *A, *D, *dt_bias;
    float *h;                            // [B][M][N], updated
    int64_t sh;                          // elements between two batch items of h
    void *y;                             // [B][M]
    int64_t B;
    int M, N, G;
    int softplus;
};
cudaError_t launch_selective_step(const SelStepArgs &a, int dtype, cudaStream_t stream);

}  // namespace exb
