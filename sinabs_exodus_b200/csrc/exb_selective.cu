// Selective scan: a leaky integrator whose decay, input weight and readout depend on the input.
//
//   h_t[d,n] = exp(dt_t[d] A[d,n]) h_{t-1}[d,n] + dt_t[d] x_t[d] B_t[g,n]        g = d / (M / G)
//   y_t[d]   = (sum_n C_t[g,n] h_t[d,n] + D[d] x_t[d]) * silu(z_t[d])
//
// Mapping: L neighbouring lanes hold the N <= 4L states of a channel, four each; a block owns CC channels of one group
// and one batch item and walks a piece of the time axis.  The block first turns the chunk's x, dt (and z, dy) into
// what the recurrence needs, one thread per element and not per state, and leaves it in shared memory.
#include "exb_selective.cuh"

namespace exb {

namespace {

template <int L> struct Geo {
    static constexpr int CC = L == 1 ? 128 : 256 / L;
    static constexpr int NT = CC * L;
    static constexpr int NP = 4 * L;
    static constexpr int COLS = CC / 4;      // four-channel packs of a row
};

__device__ __forceinline__ float step_size(float dt, float bias, int softplus)
{
    const float v = dt + bias;
    return (softplus && v <= 20.0f) ? log1pf(expf(v)) : v;      // beyond 20 the difference is below 2^-31 of the value
}

// Which tile, piece of time and batch item a block works on.
struct Where {
    int tile, seg, g, ch0;
    int64_t b;
};
template <int CC>
__device__ __forceinline__ Where locate(const SelArgs &a)
{
    Where w;
    const int per = a.M / a.G;
    const int tiles = (per + CC - 1) / CC;
    int64_t i = blockIdx.x;
    const int gt = (int)(i % ((int64_t)a.G * tiles));
    i /= (int64_t)a.G * tiles;
    w.seg = (int)(i % a.segments);
    w.b = i / a.segments;
    w.g = gt / tiles;
    w.tile = gt % tiles;
    w.ch0 = w.tile * CC;
    return w;
}

__device__ __forceinline__ int64_t sequence_length(const SelArgs &a, int64_t b)
{
    if (!a.lengths) return a.T;
    const int64_t n = a.lengths[b];
    return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// Four states of a channel from a [.., N] array (columns n0 ...; missing ones are 0).
__device__ __forceinline__ void load_states(float (&v)[4], const float *p, int n0, int N)
{
    if ((N & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        if (n0 < N) f = *reinterpret_cast<const float4 *>(p + n0);
        v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = n0 + j < N ? p[n0 + j] : 0.0f;
    }
}
__device__ __forceinline__ void store_states(float *p, const float (&v)[4], int n0, int N)
{
    if ((N & 3) == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        if (n0 < N) *reinterpret_cast<float4 *>(p + n0) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (n0 + j < N) p[n0 + j] = v[j];
    }
}

// Stages rows t0 .. t0 + K of B (and C) of one group as float, zero beyond `steps` rows and N columns.
template <typename T, int NT, int NP, int K>
__device__ __forceinline__ void stage_group(float *dst, const View &v, int64_t b, int64_t t0, int steps, int g, int N)
{
    const T *base = static_cast<const T *>(v.p) + b * v.sb + (int64_t)g * N;
    for (int i = threadIdx.x; i < K * NP; i += NT) {
        const int t = i / NP, n = i % NP;
        dst[i] = (t < steps && n < N) ? to_f32(base[(t0 + t) * v.st + n]) : 0.0f;
    }
}

// ---------------------------------------------------------------------------------------------- forward

constexpr int KF = 16;      // steps staged at a time

// STATE_ONLY: the state a piece of time ends with when it starts from zero, and its sum of step sizes.
template <typename T, int L, bool VEC, bool STATE_ONLY>
__global__ void __launch_bounds__(Geo<L>::NT) sel_forward_kernel(const SelArgs a)
{
    using Q = Geo<L>;
    constexpr int CC = Q::CC, NT = Q::NT, NP = Q::NP, COLS = Q::COLS;
    constexpr int GS = L < SEL_CHUNK ? L : SEL_CHUNK;      // steps whose readouts are summed over the lanes together
    __shared__ float2 s_in[KF * CC];         // dt, dt * x
    __shared__ float s_b[KF * NP], s_c[STATE_ONLY ? 4 : KF * NP];
    __shared__ float s_y[STATE_ONLY ? 4 : KF * CC];
    const Where w = locate<CC>(a);
    const int per = a.M / a.G;
    const int tid = threadIdx.x, c = tid / L, l = tid % L, n0 = 4 * l;
    const bool alive = w.ch0 + c < per;
    const int m = w.g * per + w.ch0 + c;
    const int64_t len = sequence_length(a, w.b);
    const int64_t t_lo = w.seg * a.seg, t_hi = t_lo + a.seg < a.T ? t_lo + a.seg : a.T;
    const int64_t t_end = t_hi < len ? t_hi : len;
    const int64_t nchunks = (a.T + SEL_CHUNK - 1) / SEL_CHUNK;

    float A2[4] = {0.f, 0.f, 0.f, 0.f}, h[4] = {0.f, 0.f, 0.f, 0.f};
    if (alive) {
        load_states(A2, a.A + (int64_t)m * a.N, n0, a.N);
#pragma unroll
        for (int j = 0; j < 4; ++j) A2[j] *= LOG2E;
        if (!STATE_ONLY) {
            if (a.segments > 1) load_states(h, a.seg_h + ((w.b * a.segments + w.seg) * a.M + m) * NP, n0, NP);
            else if (a.h0) load_states(h, a.h0 + (w.b * a.M + m) * a.N, n0, a.N);
        }
    }
    float dt_sum = 0.0f;

    for (int64_t tc = t_lo; tc < t_end; tc += KF) {
        const int steps = t_end - tc < KF ? (int)(t_end - tc) : KF;
        __syncthreads();      // the previous chunk's readouts have been taken
        for (int i = tid; i < KF * COLS; i += NT) {
            const int row = i / COLS, col = (i % COLS) * 4;
            const int left = row < steps ? per - (w.ch0 + col) : 0;
            const int ch = w.g * per + w.ch0 + col;
            Pack<T, 4> px, pd;
            load_pack<VEC>(px, static_cast<const T *>(a.x.p) + w.b * a.x.sb + (tc + row) * a.x.st + ch, left);
            load_pack<VEC>(pd, static_cast<const T *>(a.dt.p) + w.b * a.dt.sb + (tc + row) * a.dt.st + ch, left);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float d = 0.0f, u = 0.0f;
                if (j < left) {
                    d = step_size(to_f32(pd.v[j]), a.dt_bias ? a.dt_bias[ch + j] : 0.0f, a.softplus);
                    u = d * to_f32(px.v[j]);
                }
                s_in[row * CC + col + j] = make_float2(d, u);
            }
        }
        stage_group<T, NT, NP, KF>(s_b, a.Bm, w.b, tc, steps, w.g, a.N);
        if (!STATE_ONLY) stage_group<T, NT, NP, KF>(s_c, a.Cm, w.b, tc, steps, w.g, a.N);
        __syncthreads();
#pragma unroll
        for (int t0 = 0; t0 < KF; t0 += GS) {
            if (!STATE_ONLY && a.ckpt && t0 % SEL_CHUNK == 0 && t0 < steps && alive)
                store_states(a.ckpt + ((w.b * nchunks + (tc + t0) / SEL_CHUNK) * a.M + m) * NP, h, n0, NP);
            float v[GS];
#pragma unroll
            for (int i = 0; i < GS; ++i) {
                const int t = t0 + i;
                v[i] = 0.0f;
                if (t < steps) {
                    const float2 in = s_in[t * CC + c];
                    const float4 b4 = *reinterpret_cast<const float4 *>(s_b + t * NP + n0);
                    const float bb[4] = {b4.x, b4.y, b4.z, b4.w};
                    float cc[4] = {0.f, 0.f, 0.f, 0.f};
                    if (!STATE_ONLY) {
                        const float4 c4 = *reinterpret_cast<const float4 *>(s_c + t * NP + n0);
                        cc[0] = c4.x; cc[1] = c4.y; cc[2] = c4.z; cc[3] = c4.w;
                    } else {
                        dt_sum += in.x;
                    }
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        h[j] = fmaf(exp2_fast(in.x * A2[j]), h[j], in.y * bb[j]);
                        if (!STATE_ONLY) v[i] = fmaf(cc[j], h[j], v[i]);
                    }
                }
            }
            if (!STATE_ONLY) {
                reduce_scatter<GS, L, 1>(v, tid);
                if (writes_total<GS, L>(l)) s_y[(t0 + first_of<GS, L>(l)) * CC + c] = v[0];
            }
        }
        if (STATE_ONLY) continue;
        __syncthreads();
        for (int i = tid; i < KF * COLS; i += NT) {
            const int row = i / COLS, col = (i % COLS) * 4;
            const int left = row < steps ? per - (w.ch0 + col) : 0;
            const int ch = w.g * per + w.ch0 + col;
            if (left <= 0) continue;
            Pack<T, 4> px, pz, out;
            load_pack<VEC>(px, static_cast<const T *>(a.x.p) + w.b * a.x.sb + (tc + row) * a.x.st + ch, left);
            if (a.z.p) load_pack<VEC>(pz, static_cast<const T *>(a.z.p) + w.b * a.z.sb + (tc + row) * a.z.st + ch, left);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float y = s_y[row * CC + col + j];
                if (j < left && a.D) y = fmaf(a.D[ch + j], to_f32(px.v[j]), y);
                if (a.z.p) y *= silu_f(to_f32(pz.v[j]));
                out.v[j] = from_f32<T>(y);
            }
            store_pack<VEC>(static_cast<T *>(a.y) + (w.b * a.T + tc + row) * a.M + ch, out, left);
        }
    }
    if (STATE_ONLY) {
        if (alive) {
            store_states(a.seg_h + ((w.b * a.segments + w.seg) * a.M + m) * NP, h, n0, NP);
            if (l == 0) a.seg_dt[(w.b * a.segments + w.seg) * a.M + m] = dt_sum;
        }
        return;
    }
    if (alive && w.seg == a.segments - 1) store_states(a.h_last + (w.b * a.M + m) * a.N, h, n0, a.N);
    // rows behind the sequence
    const int64_t z_lo = t_end > t_lo ? t_end : t_lo;
    for (int64_t i = tid; i < (t_hi - z_lo) * CC; i += NT) {
        const int ch = w.ch0 + (int)(i % CC);
        if (ch < per) static_cast<T *>(a.y)[(w.b * a.T + z_lo + i / CC) * a.M + w.g * per + ch] = from_f32<T>(0.0f);
    }
}

// Turns every piece's own end state (started from zero) into the state that enters it, in place.  REVERSE: the same for
// the gradient, from the last piece to the first.  One thread per state.
template <bool REVERSE>
__global__ void sel_carry_kernel(const SelArgs a, int NP)
{
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= a.B * a.M * NP) return;
    const int n = (int)(i % NP);
    const int64_t bm = i / NP, b = bm / a.M, m = bm % a.M;
    const float *start = REVERSE ? a.dh_last : a.h0;
    float carry = (start && n < a.N) ? start[bm * a.N + n] : 0.0f;
    const float A2 = n < a.N ? a.A[m * a.N + n] * LOG2E : 0.0f;
    for (int k = 0; k < a.segments; ++k) {
        const int s = REVERSE ? a.segments - 1 - k : k;
        const int64_t at = (b * a.segments + s) * a.M + m;
        const float own = a.seg_h[at * NP + n], sum = a.seg_dt[at];
        a.seg_h[at * NP + n] = carry;
        carry = fmaf(sum == 0.0f ? 1.0f : exp2_fast(sum * A2), carry, own);
    }
}

// ---------------------------------------------------------------------------------------------- backward

constexpr int KB = SEL_CHUNK;

// What the elementwise part of the backward derives from one element of dt, x, z and dy.
struct Elem {
    float dt, x, p;
};

// Gradient that a piece of time sends to the step in front of it when nothing enters from behind, and its sum of step sizes.
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(Geo<L>::NT) sel_backward_state_kernel(const SelArgs a)
{
    using Q = Geo<L>;
    constexpr int CC = Q::CC, NT = Q::NT, NP = Q::NP, COLS = Q::COLS;
    __shared__ float2 s_in[KB * CC];         // dt, p
    __shared__ float s_c[KB * NP];
    const Where w = locate<CC>(a);
    const int per = a.M / a.G;
    const int tid = threadIdx.x, c = tid / L, l = tid % L, n0 = 4 * l;
    const bool alive = w.ch0 + c < per;
    const int m = w.g * per + w.ch0 + c;
    const int64_t len = sequence_length(a, w.b);
    const int64_t t_lo = w.seg * a.seg, t_hi = t_lo + a.seg < a.T ? t_lo + a.seg : a.T;
    const int64_t t_end = t_hi < len ? t_hi : len;
    float A2[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
    if (alive) {
        load_states(A2, a.A + (int64_t)m * a.N, n0, a.N);
#pragma unroll
        for (int j = 0; j < 4; ++j) A2[j] *= LOG2E;
    }
    float dt_sum = 0.0f;
    const int64_t count = t_end > t_lo ? (t_end - t_lo + KB - 1) / KB : 0;
    for (int64_t k = count - 1; k >= 0; --k) {
        const int64_t tc = t_lo + k * KB;
        const int steps = t_end - tc < KB ? (int)(t_end - tc) : KB;
        __syncthreads();
        for (int i = tid; i < KB * COLS; i += NT) {
            const int row = i / COLS, col = (i % COLS) * 4;
            const int left = row < steps ? per - (w.ch0 + col) : 0;
            const int ch = w.g * per + w.ch0 + col;
            Pack<T, 4> pd, pz, pg;
            load_pack<VEC>(pd, static_cast<const T *>(a.dt.p) + w.b * a.dt.sb + (tc + row) * a.dt.st + ch, left);
            load_pack<VEC>(pg, static_cast<const T *>(a.dy.p) + w.b * a.dy.sb + (tc + row) * a.dy.st + ch, left);
            if (a.z.p) load_pack<VEC>(pz, static_cast<const T *>(a.z.p) + w.b * a.z.sb + (tc + row) * a.z.st + ch, left);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float d = 0.0f, p = 0.0f;
                if (j < left) {
                    d = step_size(to_f32(pd.v[j]), a.dt_bias ? a.dt_bias[ch + j] : 0.0f, a.softplus);
                    p = to_f32(pg.v[j]);
                    if (a.z.p) p *= silu_f(to_f32(pz.v[j]));
                }
                s_in[row * CC + col + j] = make_float2(d, p);
            }
        }
        stage_group<T, NT, NP, KB>(s_c, a.Cm, w.b, tc, steps, w.g, a.N);
        __syncthreads();
#pragma unroll
        for (int t = KB - 1; t >= 0; --t) {
            if (t < steps) {
                const float2 in = s_in[t * CC + c];
                const float4 c4 = *reinterpret_cast<const float4 *>(s_c + t * NP + n0);
                const float cc[4] = {c4.x, c4.y, c4.z, c4.w};
                dt_sum += in.x;
#pragma unroll
                for (int j = 0; j < 4; ++j) r[j] = exp2_fast(in.x * A2[j]) * fmaf(cc[j], in.y, r[j]);
            }
        }
    }
    if (alive) {
        store_states(a.seg_h + ((w.b * a.segments + w.seg) * a.M + m) * NP, r, n0, NP);
        if (l == 0) a.seg_dt[(w.b * a.segments + w.seg) * a.M + m] = dt_sum;
    }
}

template <int L>
constexpr int backward_smem_bytes()
{
    using Q = Geo<L>;
    const int warps = Q::NT / 32;
    return (int)sizeof(float) * (KB * Q::CC * 6 + KB * Q::NP * 2 + warps * KB * 2 * Q::NP + 8 * Q::NT);
}

// Walks its piece of time backwards, one chunk of KB steps after the other.  In each it rebuilds the states from the
// chunk's checkpoint, keeping the decays a_t and the decayed states a_t h_{t-1} in registers, and then runs the reverse
// recurrence  g_t = C_t p_t + a_{t+1} g_{t+1}  (p = dy silu(z)) on them.
template <typename T, int L, bool VEC>
__global__ void __launch_bounds__(Geo<L>::NT) sel_backward_kernel(const SelArgs a)
{
    using Q = Geo<L>;
    constexpr int CC = Q::CC, NT = Q::NT, NP = Q::NP, COLS = Q::COLS, WARPS = NT / 32;
    constexpr int GS = L < KB ? L : KB;             // steps whose sums over the lanes of a channel are formed together
    constexpr int CW = 32 / L;                      // channels of a warp
    constexpr int SC = CW <= 4 ? 1 : (CW / 4 < KB ? CW / 4 : KB);      // steps whose sums over the channels are formed together
    constexpr int VC = 4 * SC, RC = VC >= CW ? VC / CW : 1;
    static_assert(KB % GS == 0 && KB % SC == 0, "");
    extern __shared__ float smem[];
    float2 *s_in = reinterpret_cast<float2 *>(smem);      // dt, dt * x
    float *s_p = smem + 2 * KB * CC;
    float *s_y = s_p + KB * CC, *s_gb = s_y + KB * CC, *s_ga = s_gb + KB * CC;
    float *s_b = s_ga + KB * CC, *s_c = s_b + KB * NP;
    float *s_bc = s_c + KB * NP;                          // [warp][step][B, C][NP]
    float *s_d = s_bc + WARPS * KB * 2 * NP;              // [thread][8]
    const Where w = locate<CC>(a);
    const int per = a.M / a.G;
    const int tid = threadIdx.x, c = tid / L, l = tid % L, n0 = 4 * l, warp = tid / 32, cw = (tid % 32) / L;
    const bool alive = w.ch0 + c < per;
    const int m = w.g * per + w.ch0 + c;
    const int64_t len = sequence_length(a, w.b);
    const int64_t t_lo = w.seg * a.seg, t_hi = t_lo + a.seg < a.T ? t_lo + a.seg : a.T;
    const int64_t t_end = t_hi < len ? t_hi : len;
    const int64_t nchunks = (a.T + SEL_CHUNK - 1) / SEL_CHUNK;
    const int tiles = (per + CC - 1) / CC;

    float A2[4] = {0.f, 0.f, 0.f, 0.f}, A1[4] = {0.f, 0.f, 0.f, 0.f}, g[4] = {0.f, 0.f, 0.f, 0.f}, dA[4] = {0.f, 0.f, 0.f, 0.f};
    if (alive) {
        load_states(A1, a.A + (int64_t)m * a.N, n0, a.N);
#pragma unroll
        for (int j = 0; j < 4; ++j) A2[j] = A1[j] * LOG2E;
        if (a.segments > 1) load_states(g, a.seg_h + ((w.b * a.segments + w.seg) * a.M + m) * NP, n0, NP);
        else if (a.dh_last) load_states(g, a.dh_last + (w.b * a.M + m) * a.N, n0, a.N);
    }
    float dD[4] = {0.f, 0.f, 0.f, 0.f}, dbias[4] = {0.f, 0.f, 0.f, 0.f};      // of the elementwise part's channels

    const int64_t count = t_end > t_lo ? (t_end - t_lo + KB - 1) / KB : 0;
    for (int64_t k = count - 1; k >= 0; --k) {
        const int64_t tc = t_lo + k * KB;
        const int steps = t_end - tc < KB ? (int)(t_end - tc) : KB;
        float h[4] = {0.f, 0.f, 0.f, 0.f};
        if (alive) load_states(h, a.ckpt + ((w.b * nchunks + tc / SEL_CHUNK) * a.M + m) * NP, n0, NP);
        __syncthreads();
        for (int i = tid; i < KB * COLS; i += NT) {
            const int row = i / COLS, col = (i % COLS) * 4;
            const int left = row < steps ? per - (w.ch0 + col) : 0;
            const int ch = w.g * per + w.ch0 + col;
            Pack<T, 4> px, pd, pz, pg;
            load_pack<VEC>(px, static_cast<const T *>(a.x.p) + w.b * a.x.sb + (tc + row) * a.x.st + ch, left);
            load_pack<VEC>(pd, static_cast<const T *>(a.dt.p) + w.b * a.dt.sb + (tc + row) * a.dt.st + ch, left);
            load_pack<VEC>(pg, static_cast<const T *>(a.dy.p) + w.b * a.dy.sb + (tc + row) * a.dy.st + ch, left);
            if (a.z.p) load_pack<VEC>(pz, static_cast<const T *>(a.z.p) + w.b * a.z.sb + (tc + row) * a.z.st + ch, left);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float d = 0.0f, u = 0.0f, p = 0.0f;
                if (j < left) {
                    d = step_size(to_f32(pd.v[j]), a.dt_bias ? a.dt_bias[ch + j] : 0.0f, a.softplus);
                    u = d * to_f32(px.v[j]);
                    p = to_f32(pg.v[j]);
                    if (a.z.p) p *= silu_f(to_f32(pz.v[j]));
                }
                s_in[row * CC + col + j] = make_float2(d, u);
                s_p[row * CC + col + j] = p;
            }
        }
        stage_group<T, NT, NP, KB>(s_b, a.Bm, w.b, tc, steps, w.g, a.N);
        stage_group<T, NT, NP, KB>(s_c, a.Cm, w.b, tc, steps, w.g, a.N);
        __syncthreads();

        // forward through the chunk: decays, decayed states, readout, gradient of C
        float av[KB][4], ah[KB][4];
        {
            float y[GS], vc[VC];
#pragma unroll
            for (int t = 0; t < KB; ++t) {
                const float2 in = s_in[t * CC + c];
                const float p = s_p[t * CC + c];
                const float4 b4 = *reinterpret_cast<const float4 *>(s_b + t * NP + n0);
                const float4 c4 = *reinterpret_cast<const float4 *>(s_c + t * NP + n0);
                const float bb[4] = {b4.x, b4.y, b4.z, b4.w}, cc[4] = {c4.x, c4.y, c4.z, c4.w};
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    av[t][j] = t < steps ? exp2_fast(in.x * A2[j]) : 1.0f;
                    ah[t][j] = av[t][j] * h[j];
                    h[j] = fmaf(in.y, bb[j], ah[t][j]);
                    sum = fmaf(cc[j], h[j], sum);
                    vc[(t % SC) * 4 + j] = p * h[j];
                }
                y[t % GS] = sum;
                if (t % GS == GS - 1 && a.z.p) {
                    reduce_scatter<GS, L, 1>(y, tid);
                    if (writes_total<GS, L>(l)) s_y[(t - (GS - 1) + first_of<GS, L>(l)) * CC + c] = y[0];
                }
                if (t % SC == SC - 1) {
                    reduce_scatter<VC, CW, L>(vc, tid);
                    if (writes_total<VC, CW>(cw)) {
#pragma unroll
                        for (int r = 0; r < RC; ++r) {
                            const int e = first_of<VC, CW>(cw) + r;
                            s_bc[((warp * KB + t - (SC - 1) + e / 4) * 2 + 1) * NP + n0 + e % 4] = vc[r];
                        }
                    }
                }
            }
        }
        // backward through it
        {
            float gb[GS], ga[GS], vb[VC], dA_c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int t = KB - 1; t >= 0; --t) {
                const float2 in = s_in[t * CC + c];
                const float p = s_p[t * CC + c];
                const float4 b4 = *reinterpret_cast<const float4 *>(s_b + t * NP + n0);
                const float4 c4 = *reinterpret_cast<const float4 *>(s_c + t * NP + n0);
                const float bb[4] = {b4.x, b4.y, b4.z, b4.w}, cc[4] = {c4.x, c4.y, c4.z, c4.w};
                float sb = 0.0f, sa = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    g[j] = fmaf(cc[j], p, g[j]);
                    vb[(t % SC) * 4 + j] = g[j] * in.y;
                    sb = fmaf(g[j], bb[j], sb);
                    const float u = g[j] * ah[t][j];
                    sa = fmaf(u, A1[j], sa);
                    dA_c[j] = fmaf(u, in.x, dA_c[j]);
                    g[j] *= av[t][j];
                }
                gb[t % GS] = sb;
                ga[t % GS] = sa;
                if (t % GS == 0) {
                    reduce_scatter<GS, L, 1>(gb, tid);
                    reduce_scatter<GS, L, 1>(ga, tid);
                    if (writes_total<GS, L>(l)) {
                        s_gb[(t + first_of<GS, L>(l)) * CC + c] = gb[0];
                        s_ga[(t + first_of<GS, L>(l)) * CC + c] = ga[0];
                    }
                }
                if (t % SC == 0) {
                    reduce_scatter<VC, CW, L>(vb, tid);
                    if (writes_total<VC, CW>(cw)) {
#pragma unroll
                        for (int r = 0; r < RC; ++r) {
                            const int e = first_of<VC, CW>(cw) + r;
                            s_bc[((warp * KB + t + e / 4) * 2) * NP + n0 + e % 4] = vb[r];
                        }
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) dA[j] += dA_c[j];
        }
        __syncthreads();
        for (int i = tid; i < steps * 2 * NP; i += NT) {
            float s = 0.0f;
#pragma unroll
            for (int q = 0; q < WARPS; ++q) s += s_bc[q * KB * 2 * NP + i];
            const int64_t row = ((w.tile * a.B + w.b) * a.T + tc + i / (2 * NP)) * a.G + w.g;
            a.part_bc[row * 2 * NP + i % (2 * NP)] = s;
        }
        for (int i = tid; i < KB * COLS; i += NT) {
            const int row = i / COLS, col = (i % COLS) * 4;
            const int left = row < steps ? per - (w.ch0 + col) : 0;
            const int ch = w.g * per + w.ch0 + col;
            if (left <= 0) continue;
            Pack<T, 4> px, pd, pz, pg, ox, od, oz;
            load_pack<VEC>(px, static_cast<const T *>(a.x.p) + w.b * a.x.sb + (tc + row) * a.x.st + ch, left);
            load_pack<VEC>(pd, static_cast<const T *>(a.dt.p) + w.b * a.dt.sb + (tc + row) * a.dt.st + ch, left);
            if (a.z.p) {
                load_pack<VEC>(pg, static_cast<const T *>(a.dy.p) + w.b * a.dy.sb + (tc + row) * a.dy.st + ch, left);
                load_pack<VEC>(pz, static_cast<const T *>(a.z.p) + w.b * a.z.sb + (tc + row) * a.z.st + ch, left);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int at = row * CC + col + j;
                const float x = to_f32(px.v[j]), p = s_p[at];
                const float skip = (j < left && a.D) ? a.D[ch + j] : 0.0f;
                const float pre = to_f32(pd.v[j]) + ((j < left && a.dt_bias) ? a.dt_bias[ch + j] : 0.0f);
                float d = fmaf(s_gb[at], x, s_ga[at]);
                if (a.softplus) d *= sigmoid_f(pre);
                ox.v[j] = from_f32<T>(fmaf(s_in[at].x, s_gb[at], skip * p));
                od.v[j] = from_f32<T>(d);
                if (a.z.p) {
                    const float z = to_f32(pz.v[j]), sg = sigmoid_f(z);
                    const float raw = fmaf(skip, x, s_y[at]);
                    oz.v[j] = from_f32<T>(to_f32(pg.v[j]) * raw * (sg * (1.0f + z * (1.0f - sg))));
                }
                if (j < left) {
                    dD[j] = fmaf(p, x, dD[j]);
                    dbias[j] += d;
                }
            }
            const int64_t at = (w.b * a.T + tc + row) * a.M + ch;
            store_pack<VEC>(static_cast<T *>(a.dx) + at, ox, left);
            store_pack<VEC>(static_cast<T *>(a.ddt) + at, od, left);
            if (a.z.p) store_pack<VEC>(static_cast<T *>(a.dz) + at, oz, left);
        }
    }
    if (alive) {
        store_states(a.part_a + ((w.b * a.segments + w.seg) * a.M + m) * NP, dA, n0, NP);
        if (a.dh0 && w.seg == 0) store_states(a.dh0 + (w.b * a.M + m) * a.N, g, n0, a.N);
    }
    // a thread's elementwise part always has the same four columns (NT is a multiple of COLS): sum over the threads
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        s_d[tid * 8 + j] = dD[j];
        s_d[tid * 8 + 4 + j] = dbias[j];
    }
    __syncthreads();
    for (int i = tid; i < 2 * CC; i += NT) {
        const int ch = i % CC, which = i / CC;
        float s = 0.0f;
        for (int q = ch / 4; q < NT; q += COLS) s += s_d[q * 8 + which * 4 + ch % 4];
        if (w.ch0 + ch < per) a.part_d[((w.b * a.segments + w.seg) * 2 + which) * a.M + w.g * per + w.ch0 + ch] = s;
    }
    // rows behind the sequence have no gradient
    const int64_t z_lo = t_end > t_lo ? t_end : t_lo;
    for (int64_t i = tid; i < (t_hi - z_lo) * CC; i += NT) {
        const int ch = w.ch0 + (int)(i % CC);
        if (ch >= per) continue;
        const int64_t at = (w.b * a.T + z_lo + i / CC) * a.M + w.g * per + ch;
        static_cast<T *>(a.dx)[at] = from_f32<T>(0.0f);
        static_cast<T *>(a.ddt)[at] = from_f32<T>(0.0f);
        if (a.z.p) static_cast<T *>(a.dz)[at] = from_f32<T>(0.0f);
    }
    for (int64_t i = tid; i < (t_hi - z_lo) * 2 * NP; i += NT) {
        const int64_t row = ((w.tile * a.B + w.b) * a.T + z_lo + i / (2 * NP)) * a.G + w.g;
        a.part_bc[row * 2 * NP + i % (2 * NP)] = 0.0f;
    }
    (void)tiles;
}

// Gradients of B and C: sum over the channel tiles.  One thread per (b, t, g, B or C, n).
template <typename T>
__global__ void sel_sum_bc_kernel(T *dB, T *dC, const float *part, int tiles, int64_t rows, int N, int NP)
{
    const int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x;
    if (i >= rows * 2 * N) return;
    const int64_t row = i / (2 * N);
    const int k = (int)(i % (2 * N)), which = k / N, n = k % N;
    float s = 0.0f;
    for (int q = 0; q < tiles; ++q) s += part[((q * rows + row) * 2 + which) * NP + n];
    (which ? dC : dB)[row * N + n] = from_f32<T>(s);
}

// Where the sums over batch items and pieces of time go: d A from columns [M][NP], d D and d dt_bias from columns [2][M].
struct PutA {
    float *dA;
    int N, NP;
    __device__ void operator()(int64_t col, float v) const
    {
        const int n = (int)(col % NP);
        if (n < N) dA[col / NP * N + n] = v;
    }
};
struct PutD {
    float *dD, *dbias;
    int M;
    __device__ void operator()(int64_t col, float v) const
    {
        float *out = col < M ? dD : dbias;
        if (out) out[col % M] = v;
    }
};

// ---------------------------------------------------------------------------------------------- one token

template <typename T, int L>
__global__ void __launch_bounds__(256) sel_step_kernel(const SelStepArgs a)
{
    const int64_t i = (blockIdx.x * (int64_t)256 + threadIdx.x) / L;
    const int l = threadIdx.x % L, n0 = 4 * l;
    const bool alive = i < a.B * a.M;
    const int64_t b = alive ? i / a.M : 0;
    const int m = alive ? (int)(i % a.M) : 0, g = m / (a.M / a.G);
    float y = 0.0f, x = 0.0f;
    if (alive) {
        float h[4], A[4], bb[4], cc[4];
        float *hp = a.h + b * a.sh + (int64_t)m * a.N;
        load_states(h, hp, n0, a.N);
        load_states(A, a.A + (int64_t)m * a.N, n0, a.N);
        x = to_f32(static_cast<const T *>(a.x.p)[b * a.x.sb + m]);
        const float d = step_size(to_f32(static_cast<const T *>(a.dt.p)[b * a.dt.sb + m]), a.dt_bias ? a.dt_bias[m] : 0.0f, a.softplus);
        const T *bp = static_cast<const T *>(a.Bm.p) + b * a.Bm.sb + (int64_t)g * a.N;
        const T *cp = static_cast<const T *>(a.Cm.p) + b * a.Cm.sb + (int64_t)g * a.N;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            bb[j] = n0 + j < a.N ? to_f32(bp[n0 + j]) : 0.0f;
            cc[j] = n0 + j < a.N ? to_f32(cp[n0 + j]) : 0.0f;
        }
        const float u = d * x;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h[j] = fmaf(exp2_fast(d * A[j] * LOG2E), h[j], u * bb[j]);
            y = fmaf(cc[j], h[j], y);
        }
        store_states(hp, h, n0, a.N);
    }
#pragma unroll
    for (int s = 1; s < L; s <<= 1) y += __shfl_xor_sync(0xffffffffu, y, s);
    if (alive && l == 0) {
        if (a.D) y = fmaf(a.D[m], x, y);
        if (a.z.p) y *= silu_f(to_f32(static_cast<const T *>(a.z.p)[b * a.z.sb + m]));
        static_cast<T *>(a.y)[b * a.M + m] = from_f32<T>(y);
    }
}

// ---------------------------------------------------------------------------------------------- launchers

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

template <typename T>
bool pack_aligned(const View &v)
{
    return !v.p || (reinterpret_cast<uintptr_t>(v.p) % (4 * sizeof(T)) == 0 && v.sb % 4 == 0 && v.st % 4 == 0);
}

template <typename T, int L, bool VEC>
cudaError_t forward_typed(const SelArgs &a, const SelPlan &p, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.B * a.G * p.tiles * p.segments);
    if (p.segments > 1) {
        sel_forward_kernel<T, L, VEC, true><<<grid, Geo<L>::NT, 0, s>>>(a);
        sel_carry_kernel<false><<<(unsigned)ceil_div(a.B * a.M * p.NP, 128), 128, 0, s>>>(a, p.NP);
    }
    sel_forward_kernel<T, L, VEC, false><<<grid, Geo<L>::NT, 0, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int L, bool VEC>
cudaError_t backward_typed(const SelArgs &a, const SelPlan &p, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.B * a.G * p.tiles * p.segments);
    if (p.segments > 1) {
        sel_backward_state_kernel<T, L, VEC><<<grid, Geo<L>::NT, 0, s>>>(a);
        sel_carry_kernel<true><<<(unsigned)ceil_div(a.B * a.M * p.NP, 128), 128, 0, s>>>(a, p.NP);
    }
    constexpr int smem = backward_smem_bytes<L>();
    if (smem > 48 * 1024) {
        cudaError_t e = cudaFuncSetAttribute(sel_backward_kernel<T, L, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e != cudaSuccess) return e;
    }
    sel_backward_kernel<T, L, VEC><<<grid, Geo<L>::NT, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t forward_dispatch(const SelArgs &a, const SelPlan &p, cudaStream_t s)
{
    const bool vec = (a.M / a.G) % 4 == 0 && pack_aligned<T>(a.x) && pack_aligned<T>(a.dt) && pack_aligned<T>(a.z) &&
                     reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0;
    switch (p.L) {
    case 1: return vec ? forward_typed<T, 1, true>(a, p, s) : forward_typed<T, 1, false>(a, p, s);
    case 2: return vec ? forward_typed<T, 2, true>(a, p, s) : forward_typed<T, 2, false>(a, p, s);
    case 4: return vec ? forward_typed<T, 4, true>(a, p, s) : forward_typed<T, 4, false>(a, p, s);
    case 8: return vec ? forward_typed<T, 8, true>(a, p, s) : forward_typed<T, 8, false>(a, p, s);
    case 16: return vec ? forward_typed<T, 16, true>(a, p, s) : forward_typed<T, 16, false>(a, p, s);
    default: return vec ? forward_typed<T, 32, true>(a, p, s) : forward_typed<T, 32, false>(a, p, s);
    }
}

template <typename T>
cudaError_t backward_dispatch(const SelArgs &a, const SelPlan &p, void *dB, void *dC, cudaStream_t s)
{
    const bool vec = (a.M / a.G) % 4 == 0 && pack_aligned<T>(a.x) && pack_aligned<T>(a.dt) && pack_aligned<T>(a.z) && pack_aligned<T>(a.dy) &&
                     ((reinterpret_cast<uintptr_t>(a.dx) | reinterpret_cast<uintptr_t>(a.ddt) | reinterpret_cast<uintptr_t>(a.dz)) %
                      (4 * sizeof(T))) == 0;
    cudaError_t e;
    switch (p.L) {
    case 1: e = vec ? backward_typed<T, 1, true>(a, p, s) : backward_typed<T, 1, false>(a, p, s); break;
    case 2: e = vec ? backward_typed<T, 2, true>(a, p, s) : backward_typed<T, 2, false>(a, p, s); break;
    case 4: e = vec ? backward_typed<T, 4, true>(a, p, s) : backward_typed<T, 4, false>(a, p, s); break;
    case 8: e = vec ? backward_typed<T, 8, true>(a, p, s) : backward_typed<T, 8, false>(a, p, s); break;
    case 16: e = vec ? backward_typed<T, 16, true>(a, p, s) : backward_typed<T, 16, false>(a, p, s); break;
    default: e = vec ? backward_typed<T, 32, true>(a, p, s) : backward_typed<T, 32, false>(a, p, s); break;
    }
    if (e != cudaSuccess) return e;
    const int64_t rows = a.B * a.T * a.G;
    sel_sum_bc_kernel<T><<<(unsigned)ceil_div(rows * 2 * a.N, 256), 256, 0, s>>>(static_cast<T *>(dB), static_cast<T *>(dC), a.part_bc,
                                                                                p.tiles, rows, a.N, p.NP);
    return cudaGetLastError();
}

template <typename T>
cudaError_t step_dispatch(const SelStepArgs &a, cudaStream_t s)
{
    const int L = sel_lanes(a.N);
    const unsigned grid = (unsigned)ceil_div(a.B * a.M * L, 256);
    switch (L) {
    case 1: sel_step_kernel<T, 1><<<grid, 256, 0, s>>>(a); break;
    case 2: sel_step_kernel<T, 2><<<grid, 256, 0, s>>>(a); break;
    case 4: sel_step_kernel<T, 4><<<grid, 256, 0, s>>>(a); break;
    case 8: sel_step_kernel<T, 8><<<grid, 256, 0, s>>>(a); break;
    case 16: sel_step_kernel<T, 16><<<grid, 256, 0, s>>>(a); break;
    default: sel_step_kernel<T, 32><<<grid, 256, 0, s>>>(a); break;
    }
    return cudaGetLastError();
}

void place(SelArgs &a, const SelPlan &p, void *ws)
{
    char *base = static_cast<char *>(ws);
    a.segments = p.segments;
    a.seg = p.seg;
    a.seg_h = reinterpret_cast<float *>(base + p.off_h);
    a.seg_dt = reinterpret_cast<float *>(base + p.off_dt);
    a.part_bc = reinterpret_cast<float *>(base + p.off_bc);
    a.part_a = reinterpret_cast<float *>(base + p.off_a);
    a.part_d = reinterpret_cast<float *>(base + p.off_d);
}

}  // namespace

SelPlan sel_plan(int64_t B, int64_t T, int M, int N, int G, bool backward)
{
    SelPlan p{};
    p.L = sel_lanes(N);
    p.NP = 4 * p.L;
    p.CC = sel_channels(p.L);
    p.tiles = (int)ceil_div(M / G, p.CC);
    const int64_t blocks = B * G * p.tiles, unit = KF;
    // A block per SM at least: split the time axis when there are fewer, down to pieces of 64 steps.
    int64_t want = blocks >= 148 ? 1 : ceil_div(296, blocks);
    const int64_t most = T / 64 > 1 ? T / 64 : 1;
    if (want > most) want = most;
    p.seg = ceil_div(ceil_div(T, want), unit) * unit;
    p.segments = (int)ceil_div(T, p.seg);
    p.chunks = ceil_div(T, SEL_CHUNK);
    int64_t at = 0;
    auto take = [&at](int64_t floats) { const int64_t o = at; at += (floats * 4 + 255) / 256 * 256; return o; };
    if (p.segments > 1) {
        p.off_h = take(B * p.segments * M * p.NP);
        p.off_dt = take(B * p.segments * M);
    }
    if (backward) {
        p.off_bc = take((int64_t)p.tiles * B * T * G * 2 * p.NP);
        p.off_a = take(B * p.segments * M * p.NP);
        p.off_d = take(B * p.segments * 2 * M);
    }
    p.bytes = at;
    return p;
}

cudaError_t launch_selective_forward(SelArgs a, int dtype, void *ws, cudaStream_t stream)
{
    const SelPlan p = sel_plan(a.B, a.T, a.M, a.N, a.G, false);
    place(a, p, ws);
    if (dtype == EXB_F32) return forward_dispatch<float>(a, p, stream);
    if (dtype == EXB_BF16) return forward_dispatch<__nv_bfloat16>(a, p, stream);
    return forward_dispatch<__half>(a, p, stream);
}

cudaError_t launch_selective_backward(SelArgs a, int dtype, void *dB, void *dC, float *dA, float *dD, float *dbias, void *ws,
                                      cudaStream_t stream)
{
    const SelPlan p = sel_plan(a.B, a.T, a.M, a.N, a.G, true);
    place(a, p, ws);
    cudaError_t e;
    if (dtype == EXB_F32) e = backward_dispatch<float>(a, p, dB, dC, stream);
    else if (dtype == EXB_BF16) e = backward_dispatch<__nv_bfloat16>(a, p, dB, dC, stream);
    else e = backward_dispatch<__half>(a, p, dB, dC, stream);
    if (e != cudaSuccess) return e;
    launch_column_sum(PutA{dA, a.N, p.NP}, a.part_a, a.B * a.segments, (int64_t)a.M * p.NP, stream);
    if (dD || dbias) launch_column_sum(PutD{dD, dbias, a.M}, a.part_d, a.B * a.segments, 2 * (int64_t)a.M, stream);
    return cudaGetLastError();
}

cudaError_t launch_selective_step(const SelStepArgs &a, int dtype, cudaStream_t stream)
{
    if (dtype == EXB_F32) return step_dispatch<float>(a, stream);
    if (dtype == EXB_BF16) return step_dispatch<__nv_bfloat16>(a, stream);
    return step_dispatch<__half>(a, stream);
}

}  // namespace exb
