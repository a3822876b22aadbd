// Short causal convolution along time, one filter per channel:
//
//   y_t[m] = act(bias[m] + sum_k w[m,k] x_{t-W+1+k}[m]),   x_{-1}, x_{-2}, ... from the state of the call before.
//
// Bound by memory: a thread owns V neighbouring channels and a run of time steps.  It takes STEP rows at a time, with the
// next STEP already on their way, and keeps the W - 1 rows in front of them in registers, so that every row is read once,
// W - 1 rows per run twice.  Rows that do not exist are predicated loads and stores: a branch would keep the rows apart.
#include "exb_conv.cuh"

namespace exb {

namespace {

constexpr int TX = 32, TY = 4;      // packs and runs of a block
constexpr int STEP = 4;

__device__ __forceinline__ float param(const void *p, int64_t i, int f32, const float *) { (void)f32; return static_cast<const float *>(p)[i]; }
template <typename T>
__device__ __forceinline__ float param(const void *p, int64_t i, int f32, const T *)
{
    return f32 ? static_cast<const float *>(p)[i] : to_f32(static_cast<const T *>(p)[i]);
}

struct Spot {
    int64_t b, t0, t1, len, row;      // batch item, run, valid steps, index of the block among those of its channels
    int m, left;                      // first channel, channels from there on
};
template <int V>
__device__ __forceinline__ Spot place(const ConvArgs &a)
{
    const int tiles = (a.M + TX * V - 1) / (TX * V);
    const int64_t runs = (a.T + a.run * TY - 1) / (a.run * TY);
    int64_t i = blockIdx.x;
    Spot s;
    s.m = ((int)(i % tiles) * TX + threadIdx.x) * V;
    s.left = a.M - s.m;
    i /= tiles;
    s.row = i;
    s.b = runs > 0 ? i / runs : i;
    s.t0 = (runs > 0 ? (i % runs) * TY + threadIdx.y : threadIdx.y) * a.run;
    s.t1 = s.t0 + a.run < a.T ? s.t0 + a.run : a.T;
    int64_t n = a.lengths ? (int64_t)a.lengths[s.b] : a.T;
    s.len = n < 0 ? 0 : (n > a.T ? a.T : n);
    return s;
}

// Row t of the sequence with the state in front of it; 0 in front of that and behind the sequence.
template <typename T, int V, int W, bool VEC>
__device__ __forceinline__ void load_row(RawPack<T, V, VEC> &r, const ConvArgs &a, const Spot &s, int64_t t)
{
    const bool from_x = t >= 0;
    const T *p = from_x ? static_cast<const T *>(a.x.p) + s.b * a.x.sb + t * a.x.st + s.m
                        : static_cast<const T *>(a.state) + (s.b * (W - 1) + (t + W - 1)) * a.M + s.m;
    r.load(p, (from_x ? t < s.len : (a.state && t >= 1 - W)) ? s.left : 0);
}

// Filter of V channels as pairs.
template <typename T, int V, int W>
struct Filter {
    float2 w[W][V / 2], bias[V / 2];
    __device__ __forceinline__ Filter(const ConvArgs &a, const Spot &s)
    {
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const int m = s.m + 2 * i;
            const bool one = 2 * i < s.left, two = 2 * i + 1 < s.left;
            const T *tag = nullptr;
            bias[i] = make_float2(one && a.bias ? param(a.bias, m, a.params_f32, tag) : 0.0f, two && a.bias ? param(a.bias, m + 1, a.params_f32, tag) : 0.0f);
#pragma unroll
            for (int k = 0; k < W; ++k)
                w[k][i] = make_float2(one ? param(a.weight, (int64_t)m * W + k, a.params_f32, tag) : 0.0f,
                                      two ? param(a.weight, (int64_t)(m + 1) * W + k, a.params_f32, tag) : 0.0f);
        }
    }
};

// 8 x 2048 x 4096, W = 4, silu, bfloat16 (268 MB read and written): 63 us, 4.3 TB/s; 5 x 1999 x 1023, W = 3, float16, rows that
// start at odd addresses: 17.8 us, 2.3 TB/s, bound by the single-element accesses.
template <typename T, int V, int W, bool VEC>
__global__ void __launch_bounds__(TX * TY) conv_forward_kernel(const ConvArgs a)
{
    const Spot s = place<V>(a);
    if (s.left <= 0) return;
    if (s.t0 == 0 && a.last) {      // the rows that the next call starts from
        for (int j = 0; j < W - 1; ++j) {
            RawPack<T, V, VEC> r;
            load_row<T, V, W, VEC>(r, a, s, s.len + j - (W - 1));
            r.store(static_cast<T *>(a.last) + (s.b * (W - 1) + j) * a.M + s.m, s.left);
        }
    }
    if (s.t0 >= a.T) return;
    const Filter<T, V, W> f(a, s);
    RawPack<T, V, VEC> next[STEP];
    float2 row[STEP + W - 1][V / 2];      // row j: step t - (W - 1) + j
#pragma unroll
    for (int k = 0; k < W - 1; ++k) {
        RawPack<T, V, VEC> r;
        load_row<T, V, W, VEC>(r, a, s, s.t0 - (W - 1) + k);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) row[k][i] = r.pair(i);
    }
#pragma unroll
    for (int j = 0; j < STEP; ++j) load_row<T, V, W, VEC>(next[j], a, s, s.t0 + j);
    T *out = static_cast<T *>(a.y) + (s.b * a.T + s.t0) * a.M + s.m;
    for (int64_t t = s.t0; t < s.t1; t += STEP) {
#pragma unroll
        for (int j = 0; j < STEP; ++j)
#pragma unroll
            for (int i = 0; i < V / 2; ++i) row[W - 1 + j][i] = next[j].pair(i);
        if (t + STEP < s.t1) {
#pragma unroll
            for (int j = 0; j < STEP; ++j) load_row<T, V, W, VEC>(next[j], a, s, t + STEP + j);
        }
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
            Pack<T, V> y;
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                float2 v = f.bias[i];
#pragma unroll
                for (int k = 0; k < W; ++k) v = fma2(f.w[k][i], row[j + k][i], v);
                if (a.silu) v = silu2(v);
                y.v[2 * i] = from_f32<T>(t + j < s.len ? v.x : 0.0f);
                y.v[2 * i + 1] = from_f32<T>(t + j < s.len ? v.y : 0.0f);
            }
            store_pack<VEC>(out, y, t + j < s.t1 ? s.left : 0);
            out += a.M;
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k)
#pragma unroll
            for (int i = 0; i < V / 2; ++i) row[k][i] = row[k + STEP][i];
    }
}

// Rows of x and dy on their way to one thread: STEP rows at a time, DEPTH times ahead, through a ring in shared memory that
// only this thread writes (asynchronous copies, which fill in zeros for rows that do not exist) and reads.  In registers they
// would cost the occupancy that the backward pass needs.  Rows that are not aligned are loaded when they are needed.
template <typename T, int V, bool VEC>
struct Rows {
    static constexpr int DEPTH = 3, BYTES = V * (int)sizeof(T);
    static constexpr int RING = VEC ? DEPTH * STEP * 2 * TX * TY * BYTES : 0;
    char *ring;
    int slot = 0;      // group that is taken next

    __device__ __forceinline__ explicit Rows(char *base) : ring(base + (threadIdx.y * TX + threadIdx.x) * BYTES) {}
    __device__ __forceinline__ char *at(int group, int j, int which) const { return ring + ((group * STEP + j) * 2 + which) * (TX * TY * BYTES); }
    __device__ __forceinline__ static void copy(char *to, const T *from, bool there)
    {
        const unsigned dst = (unsigned)__cvta_generic_to_shared(to), bytes = there ? BYTES : 0;
        if constexpr (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
        else asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(dst), "l"(from), "r"(bytes) : "memory");
    }
    // Rows t .. t + STEP of both tensors on their way into group `group` (rows that do not exist: any valid address).
    template <typename There>
    __device__ __forceinline__ void issue(int group, const T *x, int64_t step_x, const T *g, int64_t step_g, int64_t t, const There &there) const
    {
#pragma unroll
        for (int j = 0; j < STEP; ++j) {
            const bool h = there(t + j);
            copy(at(group, j, 0), h ? x + (t + j) * step_x : x, h);
            copy(at(group, j, 1), h ? g + (t + j) * step_g : g, h);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    __device__ __forceinline__ static void take(RawPack<T, V, VEC> &r, const char *from)
    {
        if constexpr (BYTES == 16) {
            const uint4 v = *reinterpret_cast<const uint4 *>(from);
            r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
        } else {
            const uint2 v = *reinterpret_cast<const uint2 *>(from);
            r.w[0] = v.x; r.w[1] = v.y;
        }
    }
};

// A thread forms the gradient in front of the activation, d, for its run and for the W - 1 steps behind it (which the rows
// of its run feed), and from those dx; filter and bias gradients only take the run's own steps.
// 8 x 2048 x 4096, W = 4, silu, bfloat16 (403 MB): 144 us, 2.8 TB/s; half of the issue slots are busy with 12 warps on an SM
// (168 registers: filter, its gradient, and the windows of x and d).  With the rows ahead in registers: 184 us.
template <typename T, int V, int W, bool VEC>
__global__ void __launch_bounds__(TX * TY, W <= 4 ? 3 : 1) conv_backward_kernel(const ConvArgs a)
{
    extern __shared__ uint4 s_raw[];      // the rings, and at the end the sums [TY][W + 1][TX * V]
    float *s_part = reinterpret_cast<float *>(s_raw);
    const Spot s = place<V>(a);
    float2 dw[W + 1][V / 2];
#pragma unroll
    for (int i = 0; i < V / 2; ++i)
#pragma unroll
        for (int k = 0; k <= W; ++k) dw[k][i] = both(0.0f);
    if (s.left > 0 && s.t0 < a.T) {
        const Filter<T, V, W> f(a, s);
        using Ring = Rows<T, V, VEC>;
        Ring ring(reinterpret_cast<char *>(s_raw));
        float2 row[STEP + W - 1][V / 2], d[STEP + W - 1][V / 2];      // entry j: step t - (W - 1) + j
        const int64_t own_end = s.t1 < s.len ? s.t1 : s.len;
        const int64_t end = s.t1 + W - 1;      // rows t - (W - 1) in [t0 (or the state's), t1) come out
        const T *x = static_cast<const T *>(a.x.p) + s.b * a.x.sb + s.m, *dy = static_cast<const T *>(a.dy.p) + s.b * a.dy.sb + s.m;
        auto there = [&](int64_t t) { return t < s.len && t < end; };
        if constexpr (VEC) {
#pragma unroll
            for (int q = 0; q < Ring::DEPTH; ++q) ring.issue(q, x, a.x.st, dy, a.dy.st, s.t0 + q * STEP, there);
        }
#pragma unroll
        for (int k = 0; k < W - 1; ++k) {
            RawPack<T, V, VEC> r;
            load_row<T, V, W, VEC>(r, a, s, s.t0 - (W - 1) + k);
#pragma unroll
            for (int i = 0; i < V / 2; ++i) {
                row[k][i] = r.pair(i);
                d[k][i] = both(0.0f);
            }
        }
        T *out = static_cast<T *>(a.dx) + (s.b * a.T + s.t0 - (W - 1)) * a.M + s.m;
        T *out_state = (s.t0 == 0 && a.dstate) ? static_cast<T *>(a.dstate) + s.b * (W - 1) * a.M + s.m : nullptr;
        for (int64_t t = s.t0; t < end; t += STEP) {
            float2 up[STEP][V / 2];
            if constexpr (VEC) asm volatile("cp.async.wait_group %0;" ::"n"(Ring::DEPTH - 1) : "memory");
#pragma unroll
            for (int j = 0; j < STEP; ++j) {
                RawPack<T, V, VEC> rx, rg;
                if constexpr (VEC) {
                    Ring::take(rx, ring.at(ring.slot, j, 0));
                    Ring::take(rg, ring.at(ring.slot, j, 1));
                } else {
                    rx.load(x + (t + j) * a.x.st, there(t + j) ? s.left : 0);
                    rg.load(dy + (t + j) * a.dy.st, there(t + j) ? s.left : 0);
                }
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    row[W - 1 + j][i] = rx.pair(i);
                    up[j][i] = rg.pair(i);
                }
            }
            if constexpr (VEC) {
                ring.issue(ring.slot, x, a.x.st, dy, a.dy.st, t + Ring::DEPTH * STEP, there);
                ring.slot = ring.slot == Ring::DEPTH - 1 ? 0 : ring.slot + 1;
            }
#pragma unroll
            for (int j = 0; j < STEP; ++j) {
                const int64_t now = t + j, r = now - (W - 1);
                const bool counts = now < own_end;
                Pack<T, V> g;
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    // rows without an output have up = 0; their pre is finite, because rows behind the sequence read as 0
                    float2 e = up[j][i];
                    if (a.silu) {
                        float2 pre = f.bias[i];
#pragma unroll
                        for (int k = 0; k < W; ++k) pre = fma2(f.w[k][i], row[j + k][i], pre);
                        const float2 slope = silu_slope2(pre);
                        e = now < s.len ? mul2(e, slope) : both(0.0f);
                    }
                    d[W - 1 + j][i] = e;
                    if (counts) {      // not e = 0: the rows may hold infinities, which belong to others' sums or to none
#pragma unroll
                        for (int k = 0; k < W; ++k) dw[k][i] = fma2(e, row[j + k][i], dw[k][i]);
                        dw[W][i] = add2(dw[W][i], e);
                    }
                    float2 v = mul2(f.w[0][i], d[W - 1 + j][i]);
#pragma unroll
                    for (int k = 1; k < W; ++k) v = fma2(f.w[k][i], d[W - 1 + j - k][i], v);
                    const int64_t q = now - s.len;      // row of `last` that row r became
                    if (a.dlast && q >= 0 && q < W - 1) {
                        const T *at = static_cast<const T *>(a.dlast) + (s.b * (W - 1) + q) * a.M + s.m + 2 * i;
                        if (2 * i < s.left) v.x += to_f32(at[0]);
                        if (2 * i + 1 < s.left) v.y += to_f32(at[1]);
                    }
                    g.v[2 * i] = from_f32<T>(v.x);
                    g.v[2 * i + 1] = from_f32<T>(v.y);
                }
                store_pack<VEC>(out, g, (r >= s.t0 && r < s.t1) ? s.left : 0);
                if (out_state && now < W - 1) store_pack<VEC>(out_state + now * a.M, g, s.left);
                out += a.M;
            }
#pragma unroll
            for (int k = 0; k < W - 1; ++k)
#pragma unroll
                for (int i = 0; i < V / 2; ++i) {
                    row[k][i] = row[k + STEP][i];
                    d[k][i] = d[k + STEP][i];
                }
        }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    __syncthreads();      // nobody's rows are on their way any more
#pragma unroll
    for (int k = 0; k <= W; ++k)
#pragma unroll
        for (int i = 0; i < V / 2; ++i) *reinterpret_cast<float2 *>(s_part + (threadIdx.y * (W + 1) + k) * (TX * V) + threadIdx.x * V + 2 * i) = dw[k][i];
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

// One step: a thread takes V channels of `items` batch items, with their filters in registers.  512 x 4096, W = 4, bfloat16
// (34 MB): 6.6 us, 5.1 TB/s.
template <typename T, int V, int W, bool VEC>
__global__ void __launch_bounds__(128) conv_step_kernel(const ConvStepArgs a, int items)
{
    const int packs = (a.M + V - 1) / V;
    const int64_t i = blockIdx.x * 128ll + threadIdx.x;
    const int64_t b0 = i / packs * items;
    if (b0 >= a.B) return;
    ConvArgs c{};
    c.M = a.M; c.weight = a.weight; c.bias = a.bias; c.params_f32 = a.params_f32;
    Spot s{};
    s.m = (int)(i % packs) * V;
    s.left = a.M - s.m;
    const Filter<T, V, W> f(c, s);
    const int64_t b1 = b0 + items < a.B ? b0 + items : a.B;
#pragma unroll 2
    for (int64_t b = b0; b < b1; ++b) {
        RawPack<T, V, VEC> row[W];
        T *st = static_cast<T *>(a.state) + b * a.ss + s.m;
#pragma unroll
        for (int k = 0; k < W - 1; ++k) row[k].load(st + (int64_t)k * a.M, s.left);
        row[W - 1].load(static_cast<const T *>(a.x.p) + b * a.x.sb + s.m, s.left);
#pragma unroll
        for (int k = 0; k < W - 1; ++k) row[k + 1].store(st + (int64_t)k * a.M, s.left);
        Pack<T, V> y;
#pragma unroll
        for (int q = 0; q < V / 2; ++q) {
            float2 v = f.bias[q];
#pragma unroll
            for (int k = 0; k < W; ++k) v = fma2(f.w[k][q], row[k].pair(q), v);
            if (a.silu) v = silu2(v);
            y.v[2 * q] = from_f32<T>(v.x);
            y.v[2 * q + 1] = from_f32<T>(v.y);
        }
        store_pack<VEC>(static_cast<T *>(a.y) + b * a.M + s.m, y, s.left);
    }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

constexpr int V = 4;      // channels of a thread where rows are aligned, two where they are not

// Steps of a thread: long runs re-read less (W - 1 rows each), short ones give every SM work on small problems.
int64_t run_of(int64_t B, int64_t T, int M, int64_t longest)
{
    int64_t run = longest;
    while (run > 4 && B * ceil_div(M, TX * V) * ceil_div(T, run * TY) < 4 * 148) run /= 2;
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

template <typename T, int N, int W, bool VEC>
cudaError_t forward_typed(ConvArgs a, cudaStream_t s)
{
    a.run = run_of(a.B, a.T, a.M, 64);
    const int64_t runs = a.T > 0 ? ceil_div(a.T, a.run * TY) : 1;
    conv_forward_kernel<T, N, W, VEC><<<(unsigned)(ceil_div(a.M, TX * N) * runs * a.B), dim3(TX, TY), 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int N, int W, bool VEC>
cudaError_t backward_typed(ConvArgs a, void *dweight, void *dbias, cudaStream_t s)
{
    a.run = run_of(a.B, a.T, a.M, 64);
    const int64_t rows = a.B * ceil_div(a.T, a.run * TY);
    constexpr int sums = TY * (W + 1) * TX * N * (int)sizeof(float), ring = Rows<T, N, VEC>::RING, smem = sums > ring ? sums : ring;
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(conv_backward_kernel<T, N, W, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    conv_backward_kernel<T, N, W, VEC><<<(unsigned)(ceil_div(a.M, TX * N) * rows), dim3(TX, TY), smem, s>>>(a);
    const int64_t cols = (int64_t)(W + 1) * a.M;
    if (a.params_f32) launch_column_sum(PutParams<float>{(float *)dweight, (float *)dbias, a.M, W}, a.part, rows, cols, s);
    else launch_column_sum(PutParams<T>{(T *)dweight, (T *)dbias, a.M, W}, a.part, rows, cols, s);
    return cudaGetLastError();
}

template <typename T, int N, int W, bool VEC>
cudaError_t step_typed(const ConvStepArgs &a, cudaStream_t s)
{
    const int64_t packs = ceil_div(a.M, N);
    // several batch items per thread once there are two blocks of threads for every SM
    int64_t items = a.B * packs / (2 * 148 * 128);
    items = items < 1 ? 1 : (items > 8 ? 8 : items);
    conv_step_kernel<T, N, W, VEC><<<(unsigned)ceil_div(ceil_div(a.B, items) * packs, 128), 128, 0, s>>>(a, (int)items);
    return cudaGetLastError();
}

template <typename T, int W>
cudaError_t forward_width(const ConvArgs &a, cudaStream_t s)
{
    const bool vec = a.M % V == 0 && rows_aligned<T>(a.x, V) && ptr_aligned<T>(a.y, V) && ptr_aligned<T>(a.state, V) && ptr_aligned<T>(a.last, V);
    return vec ? forward_typed<T, V, W, true>(a, s) : forward_typed<T, 2, W, false>(a, s);
}
template <typename T, int W>
cudaError_t backward_width(const ConvArgs &a, void *dweight, void *dbias, cudaStream_t s)
{
    const bool vec = a.M % V == 0 && rows_aligned<T>(a.x, V) && rows_aligned<T>(a.dy, V) && ptr_aligned<T>(a.dx, V) &&
                     ptr_aligned<T>(a.state, V) && ptr_aligned<T>(a.dstate, V);
    return vec ? backward_typed<T, V, W, true>(a, dweight, dbias, s) : backward_typed<T, 2, W, false>(a, dweight, dbias, s);
}
template <typename T, int W>
cudaError_t step_width(const ConvStepArgs &a, cudaStream_t s)
{
    const bool vec = a.M % V == 0 && a.x.sb % V == 0 && a.ss % V == 0 && ptr_aligned<T>(a.x.p, V) && ptr_aligned<T>(a.y, V) && ptr_aligned<T>(a.state, V);
    return vec ? step_typed<T, V, W, true>(a, s) : step_typed<T, 2, W, false>(a, s);
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
    const int64_t run = run_of(B, T, M, 64);
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
