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

// The value whose bits stand in the low end of a word.
__device__ __forceinline__ float word_to_f32(const float *, uint32_t w) { return __uint_as_float(w); }
__device__ __forceinline__ float word_to_f32(const __nv_bfloat16 *, uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float word_to_f32(const __half *, uint32_t w) { return __half2float(__ushort_as_half((unsigned short)w)); }

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

// The same kept as the words that were loaded, for loads that stay in flight over much other work: the elements of a
// Pack would be taken apart, and waited for, where the load stands.
template <typename T, int V, bool VEC>
struct RawPack {
    static constexpr int PER = VEC ? 4 / (int)sizeof(T) : 1;      // elements of a word
    static constexpr int WORDS = V / PER;
    uint32_t w[WORDS];

    __device__ __forceinline__ void load(const T *p, int n)
    {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < WORDS; ++i) w[i] = 0u;
            if (n > 0) {
                if constexpr (WORDS == 4) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(p);
                    w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
                } else if constexpr (WORDS == 2) {
                    const uint2 v = *reinterpret_cast<const uint2 *>(p);
                    w[0] = v.x; w[1] = v.y;
                } else {
                    w[0] = *reinterpret_cast<const uint32_t *>(p);
                }
            }
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = i < n ? *reinterpret_cast<const unsigned short *>(p + i) : 0u;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) w[i] = i < n ? *reinterpret_cast<const uint32_t *>(p + i) : 0u;
        }
    }
    __device__ __forceinline__ void store(T *p, int n) const
    {
        if constexpr (VEC) {
            if (n > 0) {
                if constexpr (WORDS == 4) *reinterpret_cast<uint4 *>(p) = make_uint4(w[0], w[1], w[2], w[3]);
                else if constexpr (WORDS == 2) *reinterpret_cast<uint2 *>(p) = make_uint2(w[0], w[1]);
                else *reinterpret_cast<uint32_t *>(p) = w[0];
            }
        } else if constexpr (sizeof(T) == 2) {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) *reinterpret_cast<unsigned short *>(p + i) = (unsigned short)w[i];
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < n) *reinterpret_cast<uint32_t *>(p + i) = w[i];
        }
    }
    __device__ __forceinline__ float get(int j) const
    {
        const uint32_t v = PER == 2 && (j & 1) ? w[j / PER] >> 16 : w[j / PER];
        return word_to_f32((const T *)nullptr, v);
    }
    __device__ __forceinline__ float2 pair(int i) const { return make_float2(get(2 * i), get(2 * i + 1)); }
};

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

constexpr float LOG2E = 1.4426950408889634f, LN2 = 0.6931471805599453f;

// 2^v, two units in the last place at worst over the range that matters; results below 2^-126 become 0.
__device__ __forceinline__ float exp2_fast(float v)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// 1 / v to one unit in the last place.
__device__ __forceinline__ float rcp_fast(float v)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
    return r;
}
// The larger of two values, NaN if either is.
__device__ __forceinline__ float max_nan(float a, float b)
{
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ float min_nan(float a, float b)
{
    float r;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// The exponent's rounding makes these good to (2 + |v|) * 2^-23: at most a few units where the result matters.
__device__ __forceinline__ float sigmoid_f(float v) { return rcp_fast(1.0f + exp2_fast(-LOG2E * v)); }
__device__ __forceinline__ float silu_f(float v) { return v * sigmoid_f(v); }

// Two float32 operations in one instruction.
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) { return __ffma2_rn(a, b, c); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

__device__ __forceinline__ float2 sigmoid2(float2 v)
{
    const float2 e = mul2(v, both(-LOG2E));
    const float2 n = add2(make_float2(exp2_fast(e.x), exp2_fast(e.y)), both(1.0f));
    return make_float2(rcp_fast(n.x), rcp_fast(n.y));
}
__device__ __forceinline__ float2 silu2(float2 v) { return mul2(v, sigmoid2(v)); }
// d (v sigmoid(v)) / dv = s + v s (1 - s)
__device__ __forceinline__ float2 silu_slope2(float2 v)
{
    const float2 s = sigmoid2(v), f = mul2(v, s);
    return fma2(f, fma2(s, both(-1.0f), both(1.0f)), s);
}

// log(1 + e^v) = max(v, 0) + log(1 + u), u = e^-|v|, and log(1 + u) = 2 artanh(u / (2 + u)) by its series, whose argument is
// at most 1/3: seven terms leave 1.4e-8.  u keeps the digits that rounding |v| log2(e) would cost (step sizes are the
// small end of softplus: v = -7 gives 0.001, and they are multiplied over many steps).
__device__ __forceinline__ float2 softplus2(float2 v)
{
    const float2 w = make_float2(min_nan(fabsf(v.x), 87.0f), min_nan(fabsf(v.y), 87.0f));
    const float2 t = mul2(w, both(-LOG2E));
    // what the rounding of t lost, with the second word of log2(e)
    const float2 lost = fma2(w, both(-1.92596299e-8f), fma2(w, both(-LOG2E), make_float2(-t.x, -t.y)));
    float2 u = make_float2(exp2_fast(t.x), exp2_fast(t.y));
    u = fma2(u, mul2(lost, both(LN2)), u);
    const float2 n = add2(u, both(2.0f));
    const float2 s = mul2(u, make_float2(rcp_fast(n.x), rcp_fast(n.y))), q = mul2(s, s);
    float2 p = both(2.0f / 13.0f);
    p = fma2(p, q, both(2.0f / 11.0f));
    p = fma2(p, q, both(2.0f / 9.0f));
    p = fma2(p, q, both(2.0f / 7.0f));
    p = fma2(p, q, both(2.0f / 5.0f));
    p = fma2(p, q, both(2.0f / 3.0f));
    p = fma2(p, q, both(2.0f));
    return fma2(s, p, make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f)));
}
__device__ __forceinline__ float softplus_f(float v) { return softplus2(both(v)).x; }

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
// each column to out(column, total).  A block takes TX columns; its TY rows of threads take every TY-th row each.
template <typename Out, int TX, int TY>
__global__ void __launch_bounds__(TX * TY) column_sum_kernel(Out out, const float *part, int64_t rows, int64_t cols)
{
    __shared__ double s[TY][TX + 1];
    const int64_t c = blockIdx.x * (int64_t)TX + threadIdx.x;
    double sum = 0.0;
    if (c < cols)
#pragma unroll 8
        for (int64_t r = threadIdx.y; r < rows; r += TY) sum += part[r * cols + c];
    s[threadIdx.y][threadIdx.x] = sum;
    __syncthreads();
#pragma unroll
    for (int half = TY / 2; half >= 1; half /= 2) {
        if (threadIdx.y < half) s[threadIdx.y][threadIdx.x] += s[threadIdx.y + half][threadIdx.x];
        __syncthreads();
    }
    if (threadIdx.y == 0 && c < cols) out(c, (float)s[0][threadIdx.x]);
}

// Many rows (of few columns, as they come): narrow blocks, so that each column has many loads on their way.
// 2048 x 128: 3.9 us with blocks of 8 x 128 threads, 11.5 with 32 x 32; 128 x 20480: 16 and 8; 4 x 32768: 19.6 and 6.
template <typename Out>
void launch_column_sum(const Out &out, const float *part, int64_t rows, int64_t cols, cudaStream_t stream)
{
    if (rows > 512) column_sum_kernel<Out, 8, 64><<<(unsigned)((cols + 7) / 8), dim3(8, 64), 0, stream>>>(out, part, rows, cols);
    else if (rows > 8) column_sum_kernel<Out, 32, 16><<<(unsigned)((cols + 31) / 32), dim3(32, 16), 0, stream>>>(out, part, rows, cols);
    else column_sum_kernel<Out, 128, 2><<<(unsigned)((cols + 127) / 128), dim3(128, 2), 0, stream>>>(out, part, rows, cols);
}

}  // namespace exb
