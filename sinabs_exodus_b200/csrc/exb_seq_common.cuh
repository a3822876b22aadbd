// Pieces shared by the sequence operators (selective scan, causal convolution, group norm): element types, strided
// (batch, time, channel) views, four-element accesses, lane reductions.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/exodus_b200.h"

namespace exb {

// Element (b, t, c) of a tensor at p + b*sb + t*st + c (strides in elements).
struct View {
    void *p = nullptr;
    int64_t sb = 0, st = 0;
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }

template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// V neighbouring elements as they lie in memory; VEC: the address is a multiple of the pack's size, else element by element.
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack {
    T v[V];
};

// `n` elements of the pack exist (n <= 0: none); missing ones read as zero.  VEC implies that n is 0 or at least V.
template <bool VEC, typename T, int V>
__device__ __forceinline__ void load_pack(Pack<T, V> &r, const T *p, int n)
{
    if (VEC) {
        if (n > 0) {
            r = *reinterpret_cast<const Pack<T, V> *>(p);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) r.v[i] = from_f32<T>(0.0f);
        }
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) r.v[i] = i < n ? p[i] : from_f32<T>(0.0f);
    }
}

template <bool VEC, typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &r, int n)
{
    if (VEC) {
        if (n > 0) *reinterpret_cast<Pack<T, V> *>(p) = r;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) p[i] = r.v[i];
    }
}

__device__ __forceinline__ float sigmoid_f(float v) { return 1.0f / (1.0f + expf(-v)); }
__device__ __forceinline__ float silu_f(float v) { return v / (1.0f + expf(-v)); }

// 2^v, two units in the last place at worst over the range that matters; results below 2^-126 become 0.
__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}

constexpr float LOG2E = 1.4426950408889634f;

// Sums v[0..V) over the W lanes that differ in the lane bits W/2*UNIT ... UNIT, by halving: in each exchange a lane
// passes on the half that it will not end up with, so that V values cost about V exchanges instead of V*log2(W).
// Afterwards v[0..max(1, V/W)) holds the totals number first_of<V, W>(rank) + 0, 1, ..., rank being the lane's position
// among the W.
template <int V, int W, int UNIT>
__device__ __forceinline__ void reduce_scatter(float (&v)[V], int lane)
{
    int n = V;
#pragma unroll
    for (int m = W / 2; m >= 1; m >>= 1) {
        if (n > 1) {
            n >>= 1;
            const bool upper = lane & (m * UNIT);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                if (i < n) {
                    const float send = upper ? v[i] : v[i + n];
                    const float keep = upper ? v[i + n] : v[i];
                    v[i] = keep + __shfl_xor_sync(0xffffffffu, send, m * UNIT);
                }
            }
        } else {
            v[0] += __shfl_xor_sync(0xffffffffu, v[0], m * UNIT);
        }
    }
}

// Position of the first total that the lane of rank `rank` holds after reduce_scatter.
template <int V, int W>
__device__ __forceinline__ int first_of(int rank)
{
    return V >= W ? rank * (V / W) : rank / (W / V);
}

// Whether the lane of rank `rank` is the one of those holding a total that writes it.
template <int V, int W>
__device__ __forceinline__ bool writes_total(int rank)
{
    return V >= W || rank % (W / V) == 0;
}

// Sums the rows of part[rows][cols], in double and in an order that depends on `rows` alone, and hands the total of
// each column to out(column, total).  A block takes 32 columns; its 32 rows of threads take every 32nd row each.
template <typename Out>
__global__ void __launch_bounds__(1024) column_sum_kernel(Out out, const float *part, int64_t rows, int64_t cols)
{
    __shared__ double s[32][33];
    const int64_t c = blockIdx.x * 32ll + threadIdx.x;
    double sum = 0.0;
    if (c < cols)
#pragma unroll 4
        for (int64_t r = threadIdx.y; r < rows; r += 32) sum += part[r * cols + c];
    s[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
    if (threadIdx.y != 0 || c >= cols) return;
    sum = 0.0;
#pragma unroll
    for (int k = 0; k < 32; ++k) sum += s[k][threadIdx.x];
    out(c, (float)sum);
}

template <typename Out>
void launch_column_sum(const Out &out, const float *part, int64_t rows, int64_t cols, cudaStream_t stream)
{
    column_sum_kernel<Out><<<(unsigned)((cols + 31) / 32), dim3(32, 32), 0, stream>>>(out, part, rows, cols);
}

}  // namespace exb
