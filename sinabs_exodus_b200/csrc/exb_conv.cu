// Short causal convolution along time, one filter per channel:
//
//   y_t[m] = act(bias[m] + sum_k w[m,k] x_{t-W+1+k}[m]),   x_{-1}, x_{-2}, ... from the state of the call before.
//
// Bound by memory: a thread owns a pack of neighbouring channels and a run of time steps, keeps the last W - 1 rows in
// registers and so reads every row once, W - 1 rows per run twice.
#include "exb_conv.cuh"

namespace exb {

namespace {

constexpr int TX = 32, TY = 4;      // packs and runs of a block
constexpr int STEP = 4;             // rows in flight per thread

__device__ __forceinline__ float param(const void *p, int64_t i, int f32, const float *) { (void)f32; return static_cast<const float *>(p)[i]; }
template <typename T>
__device__ __forceinline__ float param(const void *p, int64_t i, int f32, const T *)
{
    return f32 ? static_cast<const float *>(p)[i] : to_f32(static_cast<const T *>(p)[i]);
}

struct Spot {
    int64_t b, t0, t1, len, row;      // batch item, run, valid steps, index of the block among those of its channels
    int m;
};
template <int V>
__device__ __forceinline__ Spot place(const ConvArgs &a)
{
    const int tiles = (a.M + TX * V - 1) / (TX * V);
    const int64_t runs = (a.T + a.run * TY - 1) / (a.run * TY);
    int64_t i = blockIdx.x;
    Spot s;
    s.m = ((int)(i % tiles) * TX + threadIdx.x) * V;
    i /= tiles;
    s.row = i;
    s.b = i / runs;
    s.t0 = ((i % runs) * TY + threadIdx.y) * a.run;
    s.t1 = s.t0 + a.run < a.T ? s.t0 + a.run : a.T;
    int64_t n = a.lengths ? (int64_t)a.lengths[s.b] : a.T;
    s.len = n < 0 ? 0 : (n > a.T ? a.T : n);
    return s;
}

// Row t of the sequence with the state in front of it (t >= -(W - 1)).
template <typename T, int V, int W, bool VEC>
__device__ __forceinline__ void load_row(Pack<T, V> &r, const ConvArgs &a, const Spot &s, int64_t t, int left)
{
    if (t >= 0)
        load_pack<VEC>(r, static_cast<const T *>(a.x.p) + s.b * a.x.sb + t * a.x.st + s.m, t < s.len ? left : 0);
    else
        load_pack<VEC>(r, static_cast<const T *>(a.state) + (s.b * (W - 1) + (t + W - 1)) * a.M + s.m, (a.state && t >= 1 - W) ? left : 0);
}

template <typename T, int V, int W, bool VEC>
__global__ void __launch_bounds__(TX * TY) conv_forward_kernel(const ConvArgs a)
{
    const Spot s = place<V>(a);
    const int left = a.M - s.m;
    if (left <= 0) return;
    if (s.t0 == 0 && a.last) {      // the rows that the next call starts from
        for (int j = 0; j < W - 1; ++j) {
            Pack<T, V> r;
            load_row<T, V, W, VEC>(r, a, s, s.len + j - (W - 1), left);
            store_pack<VEC>(static_cast<T *>(a.last) + (s.b * (W - 1) + j) * a.M + s.m, r, left);
        }
    }
    if (s.t0 >= a.T) return;
    float w[W][V], bias[V], win[W][V];      // win[k]: row t - W + 1 + k
#pragma unroll
    for (int v = 0; v < V; ++v) {
        const bool there = v < left;
        bias[v] = (there && a.bias) ? param(a.bias, s.m + v, a.params_f32, (const T *)nullptr) : 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) w[k][v] = there ? param(a.weight, (int64_t)(s.m + v) * W + k, a.params_f32, (const T *)nullptr) : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        Pack<T, V> r;
        load_row<T, V, W, VEC>(r, a, s, s.t0 - (W - 1) + k, left);
#pragma unroll
        for (int v = 0; v < V; ++v) win[k + 1][v] = to_f32(r.v[v]);
    }
    for (int64_t t = s.t0; t < s.t1; t += STEP) {
        Pack<T, V> in[STEP];
#pragma unroll
        for (int i = 0; i < STEP; ++i) load_row<T, V, W, VEC>(in[i], a, s, t + i, t + i < s.t1 ? left : 0);
#pragma unroll
        for (int i = 0; i < STEP; ++i) {
            if (t + i >= s.t1) break;
            Pack<T, V> out;
#pragma unroll
            for (int v = 0; v < V; ++v) {
#pragma unroll
                for (int k = 0; k < W - 1; ++k) win[k][v] = win[k + 1][v];
                win[W - 1][v] = to_f32(in[i].v[v]);
                float y = bias[v];
#pragma unroll
                for (int k = 0; k < W; ++k) y = fmaf(w[k][v], win[k][v], y);
                if (a.silu) y = silu_f(y);
                out.v[v] = from_f32<T>(t + i < s.len ? y : 0.0f);
            }
            store_pack<VEC>(static_cast<T *>(a.y) + (s.b * a.T + t + i) * a.M + s.m, out, left);
        }
    }
}

// A thread forms d pre_t for its run and for the W - 1 steps behind it (which the rows of its run feed), and from
// those dx; filter and bias gradients only take the run's own steps.
template <typename T, int V, int W, bool VEC>
__global__ void __launch_bounds__(TX * TY) conv_backward_kernel(const ConvArgs a)
{
    extern __shared__ float s_part[];      // [TY][W + 1][TX * V]
    const Spot s = place<V>(a);
    const int left = a.M - s.m;
    float dw[W + 1][V];
#pragma unroll
    for (int v = 0; v < V; ++v)
#pragma unroll
        for (int k = 0; k <= W; ++k) dw[k][v] = 0.0f;
    if (left > 0 && s.t0 < a.T) {
        float w[W][V], bias[V], win[W][V], dp[W][V];      // dp[k]: d pre of step t - W + 1 + k
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const bool there = v < left;
            bias[v] = (there && a.bias) ? param(a.bias, s.m + v, a.params_f32, (const T *)nullptr) : 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) {
                w[k][v] = there ? param(a.weight, (int64_t)(s.m + v) * W + k, a.params_f32, (const T *)nullptr) : 0.0f;
                dp[k][v] = 0.0f;
            }
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            Pack<T, V> r;
            load_row<T, V, W, VEC>(r, a, s, s.t0 - (W - 1) + k, left);
#pragma unroll
            for (int v = 0; v < V; ++v) win[k + 1][v] = to_f32(r.v[v]);
        }
        const int64_t end = s.t1 + W - 1;      // rows t - W + 1 in [t0 (or the state's), t1) come out
        for (int64_t t = s.t0; t < end; t += STEP) {
            Pack<T, V> in[STEP], up[STEP];
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                const bool valid = t + i < end && t + i < s.len;
                load_row<T, V, W, VEC>(in[i], a, s, t + i, valid ? left : 0);
                load_pack<VEC>(up[i], static_cast<const T *>(a.dy.p) + s.b * a.dy.sb + (t + i) * a.dy.st + s.m, valid ? left : 0);
            }
#pragma unroll
            for (int i = 0; i < STEP; ++i) {
                const int64_t now = t + i, row = now - (W - 1);
                if (now >= end) break;
                Pack<T, V> out;
#pragma unroll
                for (int v = 0; v < V; ++v) {
#pragma unroll
                    for (int k = 0; k < W - 1; ++k) {
                        win[k][v] = win[k + 1][v];
                        dp[k][v] = dp[k + 1][v];
                    }
                    win[W - 1][v] = to_f32(in[i].v[v]);
                    float d = to_f32(up[i].v[v]);
                    if (a.silu) {
                        float pre = bias[v];
#pragma unroll
                        for (int k = 0; k < W; ++k) pre = fmaf(w[k][v], win[k][v], pre);
                        const float sg = sigmoid_f(pre);
                        d *= sg * (1.0f + pre * (1.0f - sg));
                    }
                    if (now >= s.len) d = 0.0f;
                    dp[W - 1][v] = d;
                    if (now < s.t1 && now < s.len) {
#pragma unroll
                        for (int k = 0; k < W; ++k) dw[k][v] = fmaf(d, win[k][v], dw[k][v]);
                        dw[W][v] += d;
                    }
                    float g = 0.0f;
#pragma unroll
                    for (int k = 0; k < W; ++k) g = fmaf(w[W - 1 - k][v], dp[k][v], g);
                    const int64_t f = row + (W - 1) - s.len;      // row of `last` that this row became
                    if (a.dlast && f >= 0 && f < W - 1 && v < left)
                        g += to_f32(static_cast<const T *>(a.dlast)[(s.b * (W - 1) + f) * a.M + s.m + v]);
                    out.v[v] = from_f32<T>(g);
                }
                if (row >= s.t0)
                    store_pack<VEC>(static_cast<T *>(a.dx) + (s.b * a.T + row) * a.M + s.m, out, left);
                else if (s.t0 == 0 && a.dstate)
                    store_pack<VEC>(static_cast<T *>(a.dstate) + (s.b * (W - 1) + now) * a.M + s.m, out, left);
            }
        }
    }
#pragma unroll
    for (int k = 0; k <= W; ++k)
#pragma unroll
        for (int v = 0; v < V; ++v) s_part[(threadIdx.y * (W + 1) + k) * (TX * V) + threadIdx.x * V + v] = dw[k][v];
    __syncthreads();
    const int m0 = s.m - threadIdx.x * V;
    for (int i = threadIdx.y * TX + threadIdx.x; i < (W + 1) * TX * V; i += TX * TY) {
        const int k = i / (TX * V), m = m0 + i % (TX * V);
        if (m >= a.M) continue;
        float sum = 0.0f;
#pragma unroll
        for (int q = 0; q < TY; ++q) sum += s_part[q * (W + 1) * (TX * V) + i];
        a.part[(s.row * (W + 1) + k) * a.M + m] = sum;
    }
}

// Columns [W + 1][M] of the blocks' partial sums become dweight[m][k] and dbias[m].
template <typename O>
struct PutParams {
    O *dweight, *dbias;
    int M, W;
    __device__ void operator()(int64_t col, float v) const
    {
        const int k = (int)(col / M), m = (int)(col % M);
        if (k < W) dweight[(int64_t)m * W + k] = from_f32<O>(v);
        else if (dbias) dbias[m] = from_f32<O>(v);
    }
};

template <typename T, int V, int W, bool VEC>
__global__ void conv_step_kernel(const ConvStepArgs a)
{
    const int packs = (a.M + V - 1) / V;
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= a.B * packs) return;
    const int64_t b = i / packs;
    const int m = (int)(i % packs) * V, left = a.M - m;
    Pack<T, V> row[W];
    T *st = static_cast<T *>(a.state) + b * a.ss + m;
#pragma unroll
    for (int k = 0; k < W - 1; ++k) load_pack<VEC>(row[k], st + (int64_t)k * a.M, left);
    load_pack<VEC>(row[W - 1], static_cast<const T *>(a.x.p) + b * a.x.sb + m, left);
#pragma unroll
    for (int k = 0; k < W - 1; ++k) store_pack<VEC>(st + (int64_t)k * a.M, row[k + 1], left);
    Pack<T, V> out;
#pragma unroll
    for (int v = 0; v < V; ++v) {
        float y = 0.0f;
        if (v < left) {
            y = a.bias ? param(a.bias, m + v, a.params_f32, (const T *)nullptr) : 0.0f;
#pragma unroll
            for (int k = 0; k < W; ++k) y = fmaf(param(a.weight, (int64_t)(m + v) * W + k, a.params_f32, (const T *)nullptr), to_f32(row[k].v[v]), y);
            if (a.silu) y = silu_f(y);
        }
        out.v[v] = from_f32<T>(y);
    }
    store_pack<VEC>(static_cast<T *>(a.y) + b * a.M + m, out, left);
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Steps of a thread: long runs re-read less (W - 1 rows each), short ones give every SM work on small problems.
int64_t run_of(int64_t B, int64_t T, int M, int V, int64_t longest)
{
    int64_t run = longest;
    while (run > 4 && B * ceil_div(M, TX * V) * ceil_div(T, run * TY) < 2 * 148) run /= 2;
    return run;
}

template <typename T>
bool rows_aligned(const View &v, int V)
{
    return reinterpret_cast<uintptr_t>(v.p) % (V * sizeof(T)) == 0 && v.sb % V == 0 && v.st % V == 0;
}
template <typename T>
bool ptr_aligned(const void *p, int V)
{
    return reinterpret_cast<uintptr_t>(p) % (V * sizeof(T)) == 0;
}

template <typename T, int V, int W, bool VEC>
cudaError_t forward_typed(ConvArgs a, cudaStream_t s)
{
    a.run = run_of(a.B, a.T, a.M, V, 32);
    const int64_t runs = a.T > 0 ? ceil_div(a.T, a.run * TY) : 1;
    conv_forward_kernel<T, V, W, VEC><<<(unsigned)(ceil_div(a.M, TX * V) * runs * a.B), dim3(TX, TY), 0, s>>>(a);
    return cudaGetLastError();
}

constexpr int BV = 4;      // channels of a thread in the backward pass: 16-byte packs of 16-bit types would need 200 registers

template <typename T, int V, int W, bool VEC>
cudaError_t backward_typed(ConvArgs a, void *dweight, void *dbias, cudaStream_t s)
{
    a.run = run_of(a.B, a.T, a.M, BV, 64);
    const int64_t rows = a.B * ceil_div(a.T, a.run * TY);
    constexpr int smem = TY * (W + 1) * TX * V * (int)sizeof(float);
    static_assert(smem <= 48 * 1024, "");
    conv_backward_kernel<T, V, W, VEC><<<(unsigned)(ceil_div(a.M, TX * V) * rows), dim3(TX, TY), smem, s>>>(a);
    const int64_t cols = (int64_t)(W + 1) * a.M;
    if (a.params_f32) launch_column_sum(PutParams<float>{(float *)dweight, (float *)dbias, a.M, W}, a.part, rows, cols, s);
    else launch_column_sum(PutParams<T>{(T *)dweight, (T *)dbias, a.M, W}, a.part, rows, cols, s);
    return cudaGetLastError();
}

template <typename T, int V, int W, bool VEC>
cudaError_t step_typed(const ConvStepArgs &a, cudaStream_t s)
{
    conv_step_kernel<T, V, W, VEC><<<(unsigned)ceil_div(a.B * ceil_div(a.M, V), 128), 128, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t forward_width(const ConvArgs &a, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool vec = a.M % V == 0 && rows_aligned<T>(a.x, V) && ptr_aligned<T>(a.y, V) && ptr_aligned<T>(a.state, V) && ptr_aligned<T>(a.last, V);
    return vec ? forward_typed<T, V, W, true>(a, s) : forward_typed<T, 1, W, false>(a, s);
}
template <typename T, int W>
cudaError_t backward_width(const ConvArgs &a, void *dweight, void *dbias, cudaStream_t s)
{
    const bool vec = a.M % BV == 0 && rows_aligned<T>(a.x, BV) && rows_aligned<T>(a.dy, BV) && ptr_aligned<T>(a.dx, BV) &&
                     ptr_aligned<T>(a.state, BV) && ptr_aligned<T>(a.dstate, BV);
    return vec ? backward_typed<T, BV, W, true>(a, dweight, dbias, s) : backward_typed<T, 1, W, false>(a, dweight, dbias, s);
}
template <typename T, int W>
cudaError_t step_width(const ConvStepArgs &a, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const bool vec = a.M % V == 0 && a.x.sb % V == 0 && a.ss % V == 0 && ptr_aligned<T>(a.x.p, V) && ptr_aligned<T>(a.y, V) && ptr_aligned<T>(a.state, V);
    return vec ? step_typed<T, V, W, true>(a, s) : step_typed<T, 1, W, false>(a, s);
}

#define EXB_CONV_WIDTHS(CALL)                                                                                                  \
    switch (a.W) {                                                                                                             \
    case 1: return CALL(1);                                                                                                    \
    case 2: return CALL(2);                                                                                                    \
    case 3: return CALL(3);                                                                                                    \
    case 4: return CALL(4);                                                                                                    \
    case 5: return CALL(5);                                                                                                    \
    case 6: return CALL(6);                                                                                                    \
    case 7: return CALL(7);                                                                                                    \
    default: return CALL(8);                                                                                                   \
    }

template <typename T>
cudaError_t forward_dispatch(const ConvArgs &a, cudaStream_t s)
{
#define EXB_CALL(W) forward_width<T, W>(a, s)
    EXB_CONV_WIDTHS(EXB_CALL)
#undef EXB_CALL
}
template <typename T>
cudaError_t backward_dispatch(const ConvArgs &a, void *dweight, void *dbias, cudaStream_t s)
{
#define EXB_CALL(W) backward_width<T, W>(a, dweight, dbias, s)
    EXB_CONV_WIDTHS(EXB_CALL)
#undef EXB_CALL
}
template <typename T>
cudaError_t step_dispatch(const ConvStepArgs &a, cudaStream_t s)
{
#define EXB_CALL(W) step_width<T, W>(a, s)
    EXB_CONV_WIDTHS(EXB_CALL)
#undef EXB_CALL
}

}  // namespace

int64_t conv_backward_workspace_bytes(int64_t B, int64_t T, int M, int W)
{
    // the run does not depend on how many channels a thread takes, so that both kernels fill the same partial sums
    const int64_t run = run_of(B, T, M, BV, 64);
    return B * ceil_div(T, run * TY) * (W + 1) * M * (int64_t)sizeof(float);
}

cudaError_t launch_conv_forward(ConvArgs a, int dtype, cudaStream_t stream)
{
    if (dtype == EXB_F32) return forward_dispatch<float>(a, stream);
    if (dtype == EXB_BF16) return forward_dispatch<__nv_bfloat16>(a, stream);
    return forward_dispatch<__half>(a, stream);
}

cudaError_t launch_conv_backward(ConvArgs a, int dtype, void *dweight, void *dbias, void *ws, cudaStream_t stream)
{
    a.part = static_cast<float *>(ws);
    if (dtype == EXB_F32) return backward_dispatch<float>(a, dweight, dbias, stream);
    if (dtype == EXB_BF16) return backward_dispatch<__nv_bfloat16>(a, dweight, dbias, stream);
    return backward_dispatch<__half>(a, dweight, dbias, stream);
}

cudaError_t launch_conv_step(const ConvStepArgs &a, int dtype, cudaStream_t stream)
{
    if (dtype == EXB_F32) return step_dispatch<float>(a, stream);
    if (dtype == EXB_BF16) return step_dispatch<__nv_bfloat16>(a, stream);
    return step_dispatch<__half>(a, stream);
}

}  // namespace exb
