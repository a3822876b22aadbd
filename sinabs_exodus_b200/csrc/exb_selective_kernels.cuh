// Selective scan: kernels of the forward pass, of its time split and of the backward pass.  A leaky integrator whose decay,
// input weight and readout depend on the input:
//
//   h_t[d,n] = exp(dt_t[d] A[d,n]) h_{t-1}[d,n] + dt_t[d] x_t[d] B_t[g,n]        g = d / (M / G)
//   y_t[d]   = (sum_n C_t[g,n] h_t[d,n] + D[d] x_t[d]) * silu(z_t[d])
//
// What bounds it.  Per step, channel and state an exponential and some seven other operations, for two or three bytes: the
// exponentials alone (16 per SM and clock, 4.6e12 / s) take three times as long as the bytes at N = 16 in 16 bits, and
// issuing the rest takes longer still.  So: states in registers, pairs of float32 per instruction, everything that is not
// per state done once per (step, channel) by warps of their own, sums over lanes without selections.
#pragma once

#include "exb_selective.cuh"

namespace exb {

namespace {

// L lanes of S states each hold a channel, a thread has two channels: with two, the values that all channels share (B, C)
// are read from shared memory half as often, which is what bounds these kernels next to the exponentials.  S is 4 where
// there are blocks enough for two on every SM, and 2, with twice the warps for the same channels, where there are not.
template <int L, int S> struct Geo {
    static constexpr int NT = S == 4 ? 128 : 256;   // threads of the recurrence
    static constexpr int NH = NT;                   // threads that prepare its inputs and take its results away
    static constexpr int CC = 2 * NT / L;           // channels of a block
    static constexpr int NP = S * L;
    static constexpr int WARPS = NT / 32;
    static constexpr int KF = CC > 64 ? 8 : 16;     // steps of a chunk in the forward direction
    static constexpr int BLOCKS = S == 4 ? 2 : 1;   // blocks on an SM that registers are kept for
};

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

// S states of a channel from a [.., N] array (columns n0 ...; missing ones are 0).
template <int S>
__device__ __forceinline__ void load_states(float (&v)[S], const float *p, int n0, int N)
{
    if (N % S == 0 && reinterpret_cast<uintptr_t>(p) % (4 * S) == 0) {
        Pack<float, S> f;
        load_pack<true>(f, p + n0, N - n0);
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = f.v[j];
    } else {
#pragma unroll
        for (int j = 0; j < S; ++j) v[j] = n0 + j < N ? p[n0 + j] : 0.0f;
    }
}
template <int S>
__device__ __forceinline__ void store_states(float *p, const float (&v)[S], int n0, int N)
{
    Pack<float, S> f;
#pragma unroll
    for (int j = 0; j < S; ++j) f.v[j] = v[j];
    if (N % S == 0 && reinterpret_cast<uintptr_t>(p) % (4 * S) == 0) store_pack<true>(p + n0, f, N - n0);
    else store_pack<false>(p + n0, f, N - n0);
}

template <int S>
__device__ __forceinline__ void load_rates(float (&v)[S], const float *p, int n0, int N)
{
    load_states(v, p, n0, N);
#pragma unroll
    for (int j = 0; j < S; ++j) v[j] = finite_rate(v[j]);
}

// Two kinds of warps.  The first NT threads of a block run the recurrence; NH more prepare its inputs and take its
// results away.  They meet at one barrier per chunk of K steps: while the recurrence runs through chunk k, the others
// store chunk k - 1's results, prepare chunk k + 1 and have chunk k + 2 on its way from memory.  A training problem has
// few channels for the size of the GPU (8192 channels are two recurrence warps on each scheduler), so the elementwise
// work, which has long chains of dependent instructions, must not stand between two of their steps.
template <int THREADS>
__device__ __forceinline__ void meet()
{
    asm volatile("bar.sync 0, %0;" ::"n"(THREADS) : "memory");
}

// The elementwise work of a chunk of K steps on CC channels by NH threads: packs of V channels, ITEMS per thread, all of
// a thread in the same columns (its channels' D and dt_bias stay in registers).
template <int K, int CC, int NH> struct Items {
    static constexpr int V = K * CC / NH >= 4 ? 4 : 2;
    static constexpr int COLS = CC / V;
    static constexpr int ROWS = NH / COLS;      // rows between two items of a thread
    static constexpr int ITEMS = (K + ROWS - 1) / ROWS;
    static_assert(NH % COLS == 0, "");
};

// A block's piece of the problem.
template <int K, int CC>
struct Block {
    Where w;
    int per;                        // channels of a group
    int64_t t_lo, t_hi, t_end;      // its steps; those that belong to the sequence end at t_end
    int64_t count;                  // chunks

    __device__ __forceinline__ explicit Block(const SelArgs &a)
    {
        w = locate<CC>(a);
        per = a.M / a.G;
        const int64_t len = sequence_length(a, w.b);
        t_lo = w.seg * a.seg;
        t_hi = t_lo + a.seg < a.T ? t_lo + a.seg : a.T;
        t_end = t_hi < len ? t_hi : len;
        count = t_end > t_lo ? (t_end - t_lo + K - 1) / K : 0;
    }
    __device__ __forceinline__ int64_t time(int64_t k) const { return t_lo + k * K; }
    __device__ __forceinline__ int steps(int64_t k) const { return t_end - time(k) < K ? (int)(t_end - time(k)) : K; }
};

// A preparing thread's part of a chunk.
template <int K, int CC, int NH>
struct Part {
    using I = Items<K, CC, NH>;
    static constexpr int V = I::V;
    int row, col, ch, left;      // first row, column, channel and number of channels of its packs

    __device__ __forceinline__ Part(const Block<K, CC> &b, int thread)
    {
        row = thread / I::COLS;
        col = thread % I::COLS * V;
        ch = b.w.g * b.per + b.w.ch0 + col;
        left = b.per - (b.w.ch0 + col);
    }
    // Number of the pack's channels that exist in row `r` of a chunk of `steps` rows (0 or less: none).
    __device__ __forceinline__ int there(int steps, int r) const { return r < steps ? left : 0; }

    template <typename T, bool VEC>
    __device__ __forceinline__ void fetch(RawPack<T, V, VEC> (&p)[I::ITEMS], const View &v, const Block<K, CC> &b, int64_t k) const
    {
        const T *at = static_cast<const T *>(v.p) + b.w.b * v.sb + (b.time(k) + row) * v.st + ch;
        const int steps = b.steps(k);
#pragma unroll
        for (int i = 0; i < I::ITEMS; ++i, at += I::ROWS * v.st) p[i].load(at, there(steps, row + i * I::ROWS));
    }
    __device__ __forceinline__ void channel_values(float (&v)[V], const float *p) const
    {
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = (p && j < left) ? p[ch + j] : 0.0f;
    }
};

// Step sizes of a pack; channels and rows that do not exist get 0, which changes no state.
template <typename R, int V>
__device__ __forceinline__ void step_sizes(float (&d)[V], float (&pre)[V], const R &raw, const float (&bias)[V], int softplus, int have)
{
#pragma unroll
    for (int j = 0; j < V; j += 2) {
        pre[j] = raw.get(j) + bias[j];
        pre[j + 1] = raw.get(j + 1) + bias[j + 1];
        float2 s = make_float2(pre[j], pre[j + 1]);
        if (softplus) s = softplus2(s);
        d[j] = j < have ? s.x : 0.0f;
        d[j + 1] = j + 1 < have ? s.y : 0.0f;
    }
}

// Rows of B or C of one group: fetched as they are, and left in shared memory as float, 0 beyond the sequence and N.
// COPIES of each row, the i-th with column n at n ^ i (see the backward kernel).
template <typename T, int K, int CC, int NP, int NH, int COPIES = 1>
struct GroupRows {
    static constexpr int ITEMS = (K * NP + NH - 1) / NH;
    RawPack<T, 1, false> r[ITEMS];

    __device__ __forceinline__ void fetch(const Block<K, CC> &b, const View &v, int N, int64_t k, int thread)
    {
        const T *base = static_cast<const T *>(v.p) + b.w.b * v.sb + b.time(k) * v.st + (int64_t)b.w.g * N;
        const int steps = b.steps(k);
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int e = thread + i * NH, t = e / NP, n = e % NP;
            r[i].load(base + t * v.st + n, (t < steps && n < N) ? 1 : 0);
        }
    }
    __device__ __forceinline__ void stage(float *dst, int thread) const
    {
#pragma unroll
        for (int i = 0; i < ITEMS; ++i) {
            const int e = thread + i * NH, t = e / NP, n = e % NP;
            if (t < K) {
#pragma unroll
                for (int q = 0; q < COPIES; ++q) dst[(t * COPIES + q) * NP + (n ^ q)] = r[i].get(0);
            }
        }
    }
};

// A thread's two channels, and how sums over their states are formed.  Lanes with odd l have them in the other order
// (channel k ^ 1 at place k): what a lane keeps in the first exchange and what it sends then always lie at the same
// places, and no selection is needed.
template <int L, int STEPS>
struct Pair {
    static constexpr int REST = L / 2;                                 // lanes left after the first exchange
    static constexpr int GS = REST < STEPS ? REST : STEPS;             // steps that share the other exchanges
    int l, first;      // state lane; first of the two channels (in the block)
    __device__ __forceinline__ explicit Pair(int tid) : l(tid % L), first(tid / L * 2) {}
    __device__ __forceinline__ int channel(int k) const { return first + (k ^ (l & 1)); }
    // Leaves the totals of GS steps from t on in out[step][CC].
    __device__ __forceinline__ void total(float (&v)[GS], float *out, int CC, int t) const
    {
        reduce_scatter<GS, REST, 2>(v, l);
        if (writes_total<GS, REST>(l >> 1)) out[(t + first_of<GS, REST>(l >> 1)) * CC + first + (l & 1)] = v[0];
    }
    __device__ __forceinline__ static float exchange(float keep, float send) { return keep + __shfl_xor_sync(0xffffffffu, send, 1); }
};

// S states of a lane as pairs.
template <int S>
struct States {
    static constexpr int Q = S / 2;
    float2 q[Q];
    __device__ __forceinline__ void set(const float (&v)[S])
    {
#pragma unroll
        for (int i = 0; i < Q; ++i) q[i] = make_float2(v[2 * i], v[2 * i + 1]);
    }
    __device__ __forceinline__ void get(float (&v)[S]) const
    {
#pragma unroll
        for (int i = 0; i < Q; ++i) { v[2 * i] = q[i].x; v[2 * i + 1] = q[i].y; }
    }
    __device__ __forceinline__ void fill(float v)
    {
#pragma unroll
        for (int i = 0; i < Q; ++i) q[i] = both(v);
    }
    __device__ __forceinline__ void load(const float *p)      // aligned
    {
        const Pack<float, S> f = *reinterpret_cast<const Pack<float, S> *>(p);
        set(f.v);
    }
};

// What to add to the exponents of a chunk's decays (see decay_lift), by those of its first step: one choice for all steps of a
// chunk costs nothing per step, and a choice that does not fit one of them is off by 2e-8 there.
template <int S>
__device__ __forceinline__ void set_lift(States<S> &lift, float dt, const States<S> &A2)
{
#pragma unroll
    for (int q = 0; q < S / 2; ++q) lift.q[q] = make_float2(decay_lift(dt * A2.q[q].x), decay_lift(dt * A2.q[q].y));
}
__device__ __forceinline__ float2 exponent(float dt, float2 A2, float2 lift) { return fma2(both(dt), A2, lift); }

// State that enters piece `seg` of channel m (S states from n0 on): what the pieces in front of it hand on by
// themselves, each decayed through those behind it; or (REVERSE) the gradient that enters from behind.  Every block folds
// that for itself: a launch less, and the loads of several pieces are in flight together.
// Where states grow (positive rates or negative step sizes), the factor of a whole piece may be beyond float32 although
// what it applies to is 0, or so small that the product is not: so 0 stays 0, and the factor is applied in two parts (the
// second is 1 for all others).
constexpr float ENTER_PART = 120.0f;
template <bool REVERSE, int NP, int S>
__device__ __forceinline__ void enter(float (&v)[S], const SelArgs &a, const Where &w, int m, int n0, const States<S> &A2)
{
    const float *start = REVERSE ? a.dh_last : a.h0;
    if (start) load_states(v, start + (w.b * a.M + m) * a.N, n0, a.N);
    const int count = REVERSE ? a.segments - 1 - w.seg : w.seg;
    float rate[S];
    A2.get(rate);
#pragma unroll 8
    for (int k = 0; k < count; ++k) {
        const int64_t at = (w.b * a.segments + (REVERSE ? a.segments - 1 - k : k)) * a.M + m;
        const Pack<float, S> own = *reinterpret_cast<const Pack<float, S> *>(a.seg_h + at * NP + n0);
        const float sum = a.seg_dt[at];
#pragma unroll
        for (int j = 0; j < S; ++j) {
            const float t = sum * rate[j], e = t + decay_lift(t), part = exp2_fast(min_nan(e, ENTER_PART)) * v[j];
            v[j] = v[j] == 0.0f ? own.v[j] : fmaf(exp2_fast(fmaxf(e - ENTER_PART, 0.0f)), part, own.v[j]);
        }
    }
}

// ---------------------------------------------------------------------------------------------- forward


// Stores a checkpoint without a branch, which would keep the steps on its two sides apart.
template <int S>
__device__ __forceinline__ void keep_states(float *p, const States<S> &h, bool there)
{
    if constexpr (S == 4)
        asm volatile("{ .reg .pred p; setp.ne.u32 p, %0, 0; @p st.global.v4.f32 [%1], {%2, %3, %4, %5}; }"
                     :: "r"((unsigned)there), "l"(p), "f"(h.q[0].x), "f"(h.q[0].y), "f"(h.q[S / 4].x), "f"(h.q[S / 4].y) : "memory");
    else
        asm volatile("{ .reg .pred p; setp.ne.u32 p, %0, 0; @p st.global.v2.f32 [%1], {%2, %3}; }"
                     :: "r"((unsigned)there), "l"(p), "f"(h.q[0].x), "f"(h.q[0].y) : "memory");
}

template <int L, int S>
constexpr int forward_smem_bytes()
{
    using Q = Geo<L, S>;
    return (int)sizeof(float) * 2 * (Q::KF * Q::CC * 5 + 2 * Q::KF * Q::NP);
}

// Measured (N = 16, bfloat16, gated): 1 x 16384 x 1024 in 18 pieces 128 us, half of the issue slots busy, the rest barrier
// and fixed latencies; 4 x 2048 x 2048 whole, with checkpoints, 160 us on 128 of the 148 SMs (S = 2; with S = 4 one
// recurrence warp per scheduler, 182 us).  Exponentials: 58 us of either.
template <typename T, int L, int S, bool VEC>
__global__ void __launch_bounds__(Geo<L, S>::NT + Geo<L, S>::NH, Geo<L, S>::BLOCKS) sel_forward_kernel(const SelArgs a)
{
    using Q = Geo<L, S>;
    constexpr int K = Q::KF, CC = Q::CC, NT = Q::NT, NP = Q::NP, NH = Q::NH;
    extern __shared__ float smem[];
    float2 *s_in = reinterpret_cast<float2 *>(smem);       // [2][K][CC]: dt, dt x
    float *s_skip = smem + 4 * K * CC, *s_gate = s_skip + 2 * K * CC;      // [2][K][CC]: D x, silu(z)
    float *s_y = s_gate + 2 * K * CC;                      // [2][K][CC]
    float *s_b = s_y + 2 * K * CC, *s_c = s_b + 2 * K * NP;      // [2][K][NP]
    const Block<K, CC> blk(a);

    if (threadIdx.x >= NT) {
        using P = Part<K, CC, NH>;
        constexpr int V = P::V, ITEMS = P::I::ITEMS, ROWS = P::I::ROWS;
        const int tid = threadIdx.x - NT;
        const P part(blk, tid);
        float skip[V], bias[V];
        part.channel_values(skip, a.D);
        part.channel_values(bias, a.dt_bias);
        struct Raw {
            RawPack<T, V, VEC> x[ITEMS], dt[ITEMS], z[ITEMS];
            GroupRows<T, K, CC, NP, NH> b, c;
        } raw[2];
        auto fetch = [&](Raw &f, int64_t k) {
            if (k >= blk.count) return;
            part.fetch(f.x, a.x, blk, k);
            part.fetch(f.dt, a.dt, blk, k);
            if (a.z.p) part.fetch(f.z, a.z, blk, k);
            f.b.fetch(blk, a.Bm, a.N, k, tid);
            f.c.fetch(blk, a.Cm, a.N, k, tid);
        };
        auto stage = [&](const Raw &f, int64_t k) {
            if (k >= blk.count) return;
            const int buf = (int)(k & 1) * K * CC, steps = blk.steps(k);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int r = part.row + i * ROWS, at = buf + r * CC + part.col;
                if (r >= K) continue;
                float d[V], pre[V];
                step_sizes(d, pre, f.dt[i], bias, a.softplus, part.there(steps, r));
                Pack<float, V> sk, ga;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float x = f.x[i].get(j), u = d[j] * x;
                    s_in[at + j] = make_float2(d[j], u);
                    sk.v[j] = skip[j] * x;
                    ga.v[j] = a.z.p ? silu_f(f.z[i].get(j)) : 1.0f;
                }
                *reinterpret_cast<Pack<float, V> *>(s_skip + at) = sk;
                *reinterpret_cast<Pack<float, V> *>(s_gate + at) = ga;
            }
            f.b.stage(s_b + (k & 1) * K * NP, tid);
            f.c.stage(s_c + (k & 1) * K * NP, tid);
        };
        auto emit = [&](int64_t k) {
            if (k < 0) return;
            const int buf = (int)(k & 1) * K * CC, steps = blk.steps(k);
            T *to = static_cast<T *>(a.y) + (blk.w.b * a.T + blk.time(k) + part.row) * a.M + part.ch;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i, to += ROWS * (int64_t)a.M) {
                const int r = part.row + i * ROWS, have = part.there(steps, r), at = buf + r * CC + part.col;
                if (have <= 0) continue;
                const Pack<float, V> y = *reinterpret_cast<const Pack<float, V> *>(s_y + at), sk = *reinterpret_cast<const Pack<float, V> *>(s_skip + at),
                                     ga = *reinterpret_cast<const Pack<float, V> *>(s_gate + at);
                Pack<T, V> out;
#pragma unroll
                for (int j = 0; j < V; ++j) out.v[j] = from_f32<T>((y.v[j] + sk.v[j]) * ga.v[j]);
                store_pack<VEC>(to, out, have);
            }
        };
        fetch(raw[0], 0);
        fetch(raw[1], 1);
        stage(raw[0], 0);
        fetch(raw[0], 2);
        for (int64_t k = 0; k < blk.count; k += 2) {
            meet<NT + NH>();
            emit(k - 1);
            stage(raw[1], k + 1);
            fetch(raw[1], k + 3);
            if (k + 1 >= blk.count) break;
            meet<NT + NH>();
            emit(k);
            stage(raw[0], k + 2);
            fetch(raw[0], k + 4);
        }
        meet<NT + NH>();
        emit(blk.count - 1);
        // rows behind the sequence
        const int64_t z_lo = blk.t_end > blk.t_lo ? blk.t_end : blk.t_lo;
        for (int64_t i = tid; i < (blk.t_hi - z_lo) * CC; i += NH) {
            const int ch = blk.w.ch0 + (int)(i % CC);
            if (ch < blk.per) static_cast<T *>(a.y)[(blk.w.b * a.T + z_lo + i / CC) * a.M + blk.w.g * blk.per + ch] = from_f32<T>(0.0f);
        }
        return;
    }

    using R = Pair<L, SEL_CHUNK>;
    constexpr int GS = R::GS;
    const R pair(threadIdx.x);
    const int n0 = S * pair.l;
    const int64_t nchunks = (a.T + SEL_CHUNK - 1) / SEL_CHUNK;
    States<S> A2[2], h[2];
    float *ckpt[2];
    bool keeps[2];      // not told from the pointer, which moves on
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = pair.channel(k), m = blk.w.g * blk.per + blk.w.ch0 + c;
        const bool alive = blk.w.ch0 + c < blk.per;
        float r[S] = {}, v[S] = {};
        if (alive) load_rates(r, a.A + (int64_t)m * a.N, n0, a.N);
        A2[k].set(r);
#pragma unroll
        for (int q = 0; q < S / 2; ++q) A2[k].q[q] = mul2(A2[k].q[q], both(LOG2E));
        if (alive) enter<false, NP, S>(v, a, blk.w, m, n0, A2[k]);
        h[k].set(v);
        keeps[k] = a.ckpt && alive;
        ckpt[k] = keeps[k] ? a.ckpt + ((blk.w.b * nchunks + blk.t_lo / SEL_CHUNK) * a.M + m) * NP + n0 : nullptr;
    }
    const int64_t ckpt_step = a.ckpt ? (int64_t)a.M * NP : 0;
    for (int64_t j = 0; j < blk.count; ++j) {
        meet<NT + NH>();
        const float2 *in = s_in + (j & 1) * K * CC;
        const float *b = s_b + (j & 1) * K * NP + n0, *cc = s_c + (j & 1) * K * NP + n0;
        float *y = s_y + (j & 1) * K * CC;
        const int steps = blk.steps(j);
        States<S> lift[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) set_lift(lift[k], in[pair.channel(k)].x, A2[k]);
#pragma unroll
        for (int t0 = 0; t0 < K; t0 += GS) {
            if (t0 % SEL_CHUNK == 0) {
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    keep_states(ckpt[k], h[k], keeps[k] && t0 < steps);
                    ckpt[k] += ckpt_step;
                }
            }
            float v[GS];
#pragma unroll
            for (int i = 0; i < GS; ++i) {
                const int t = t0 + i;
                States<S> bb, ccv;
                bb.load(b + t * NP);
                ccv.load(cc + t * NP);
                float sum[2];
#pragma unroll
                for (int k = 0; k < 2; ++k) {
                    const float2 d = in[t * CC + pair.channel(k)];
                    float2 s;
#pragma unroll
                    for (int q = 0; q < S / 2; ++q) {
                        const float2 e = exponent(d.x, A2[k].q[q], lift[k].q[q]);
                        h[k].q[q] = fma2(make_float2(exp2_fast(e.x), exp2_fast(e.y)), h[k].q[q], mul2(both(d.y), bb.q[q]));
                        s = q ? fma2(ccv.q[q], h[k].q[q], s) : mul2(ccv.q[q], h[k].q[q]);
                    }
                    sum[k] = s.x + s.y;
                }
                v[i] = R::exchange(sum[0], sum[1]);
            }
            pair.total(v, y, CC, t0);
        }
    }
    meet<NT + NH>();
    if (blk.w.seg == a.segments - 1) {
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int c = blk.w.ch0 + pair.channel(k);
            float v[S];
            h[k].get(v);
            if (c < blk.per) store_states(a.h_last + (blk.w.b * a.M + blk.w.g * blk.per + c) * a.N, v, n0, a.N);
        }
    }
}

// ---------------------------------------------------------------------------------------------- time split

template <int L, int S>
constexpr int state_smem_bytes()
{
    using Q = Geo<L, S>;
    return (int)sizeof(float) * 2 * (Q::KF * Q::CC * 2 + Q::KF * Q::NP);
}

// What a piece of time hands on when nothing enters it, and its sum of step sizes: the state behind its last step, or
// (REVERSE) the gradient that goes to the step in front of its first one.  1 x 16384 x 1024 x 16 in 18 pieces: 92 us.
template <typename T, int L, int S, bool VEC, bool REVERSE>
__global__ void __launch_bounds__(Geo<L, S>::NT + Geo<L, S>::NH, Geo<L, S>::BLOCKS) sel_state_kernel(const SelArgs a)
{
    using Q = Geo<L, S>;
    constexpr int K = Q::KF, CC = Q::CC, NT = Q::NT, NP = Q::NP, NH = Q::NH;
    extern __shared__ float smem[];
    float2 *s_in = reinterpret_cast<float2 *>(smem);      // [2][K][CC]: dt, and dt x or p
    float *s_w = smem + 4 * K * CC;                       // [2][K][NP]: B or C
    const Block<K, CC> blk(a);
    if (blk.w.seg == (REVERSE ? 0 : a.segments - 1)) return;      // nobody comes after it

    if (threadIdx.x >= NT) {
        using P = Part<K, CC, NH>;
        constexpr int V = P::V, ITEMS = P::I::ITEMS, ROWS = P::I::ROWS;
        const int tid = threadIdx.x - NT;
        const P part(blk, tid);
        float bias[V];
        part.channel_values(bias, a.dt_bias);
        struct Raw {
            RawPack<T, V, VEC> dt[ITEMS], w[ITEMS], z[ITEMS];
            GroupRows<T, K, CC, NP, NH> g;
        } raw[2];
        const bool gated = REVERSE && a.z.p;
        // k counts in the order of the walk
        auto chunk = [&](int64_t k) { return REVERSE ? blk.count - 1 - k : k; };
        auto fetch = [&](Raw &f, int64_t k) {
            if (k >= blk.count) return;
            part.fetch(f.dt, a.dt, blk, chunk(k));
            part.fetch(f.w, REVERSE ? a.dy : a.x, blk, chunk(k));
            if (gated) part.fetch(f.z, a.z, blk, chunk(k));
            f.g.fetch(blk, REVERSE ? a.Cm : a.Bm, a.N, chunk(k), tid);
        };
        auto stage = [&](const Raw &f, int64_t k) {
            if (k >= blk.count) return;
            const int buf = (int)(k & 1) * K * CC, steps = blk.steps(chunk(k));
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int r = part.row + i * ROWS;
                if (r >= K) continue;
                float d[V], pre[V];
                step_sizes(d, pre, f.dt[i], bias, a.softplus, part.there(steps, r));
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    float v = f.w[i].get(j);
                    if (!REVERSE) v *= d[j];
                    else if (gated) v *= silu_f(f.z[i].get(j));
                    s_in[buf + r * CC + part.col + j] = make_float2(d[j], v);
                }
            }
            f.g.stage(s_w + (k & 1) * K * NP, tid);
        };
        fetch(raw[0], 0);
        fetch(raw[1], 1);
        stage(raw[0], 0);
        fetch(raw[0], 2);
        for (int64_t k = 0; k < blk.count; k += 2) {
            meet<NT + NH>();
            stage(raw[1], k + 1);
            fetch(raw[1], k + 3);
            if (k + 1 >= blk.count) break;
            meet<NT + NH>();
            stage(raw[0], k + 2);
            fetch(raw[0], k + 4);
        }
        return;
    }

    const Pair<L, K> pair(threadIdx.x);
    const int n0 = S * pair.l;
    States<S> A2[2], h[2];
    float dt_sum[2] = {0.0f, 0.0f};
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = blk.w.ch0 + pair.channel(k);
        float r[S] = {};
        if (c < blk.per) load_rates(r, a.A + (int64_t)(blk.w.g * blk.per + c) * a.N, n0, a.N);
        A2[k].set(r);
#pragma unroll
        for (int q = 0; q < S / 2; ++q) {
            A2[k].q[q] = mul2(A2[k].q[q], both(LOG2E));
            h[k].q[q] = both(0.0f);
        }
    }
    for (int64_t j = 0; j < blk.count; ++j) {
        meet<NT + NH>();
        const float2 *in = s_in + (j & 1) * K * CC;
        const float *w = s_w + (j & 1) * K * NP + n0;
        States<S> lift[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) set_lift(lift[k], in[pair.channel(k)].x, A2[k]);
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int t = REVERSE ? K - 1 - i : i;
            States<S> ww;
            ww.load(w + t * NP);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const float2 d = in[t * CC + pair.channel(k)];
                dt_sum[k] += d.x;
#pragma unroll
                for (int q = 0; q < S / 2; ++q) {
                    const float2 e = exponent(d.x, A2[k].q[q], lift[k].q[q]), f = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                    h[k].q[q] = REVERSE ? mul2(f, fma2(ww.q[q], both(d.y), h[k].q[q])) : fma2(f, h[k].q[q], mul2(both(d.y), ww.q[q]));
                }
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = blk.w.ch0 + pair.channel(k);
        if (c >= blk.per) continue;
        const int64_t at = (blk.w.b * a.segments + blk.w.seg) * a.M + blk.w.g * blk.per + c;
        float v[S];
        h[k].get(v);
        store_states(a.seg_h + at * NP, v, n0, NP);
        if (pair.l == 0) a.seg_dt[at] = dt_sum[k];
    }
}

// ---------------------------------------------------------------------------------------------- backward

// How the sums over the channels of a warp (gradients of B and C) are formed.  The CW channels of a warp lie in the
// lane bits above the state lanes.  The first exchanges halve the S states of a lane: lanes of different channels keep
// their states in different orders (state j at place j ^ order), so that what a lane keeps and what it sends always lie
// at the same places and no selection is needed.  The other exchanges halve SC consecutive steps.
template <int L, int S> struct Across {
    static constexpr int CW = 32 / L;
    static constexpr int PERM = CW >= S ? S : CW;               // orders (powers of two; 1: none)
    static constexpr int REST = CW / PERM;                      // lanes left to sum over after the states
    static constexpr int SC = REST;                             // consecutive steps whose sums share the other exchanges
    static constexpr int KEPT = S / PERM;                       // states that a lane is left with
    static constexpr int COPIES = PERM > 1 ? S : 1;             // of a staged row; with S = 4, orders 0 and 2 leave two unused
    // order of a lane's states: its highest channel bits, the highest exchanges the halves
    __device__ static __forceinline__ int order(int cw) { return PERM > 1 ? cw / REST * (S / PERM) : 0; }
    // sums v over the lanes that the states are halved over; the first KEPT of them are left
    __device__ static __forceinline__ void halve_states(States<S> &v)
    {
        if constexpr (S == 4) {
            if (PERM >= 2) v.q[0] = add2(v.q[0], make_float2(__shfl_xor_sync(0xffffffffu, v.q[S / 4].x, 16), __shfl_xor_sync(0xffffffffu, v.q[S / 4].y, 16)));
            if (PERM == 4) v.q[0].x += __shfl_xor_sync(0xffffffffu, v.q[0].y, 8);
        } else {
            if (PERM == 2) v.q[0].x += __shfl_xor_sync(0xffffffffu, v.q[0].y, 16);
        }
    }
};

// v[j] = u[j ^ order]
template <int S>
__device__ __forceinline__ void reorder(float (&v)[S], int order)
{
    if (order & 1) {
#pragma unroll
        for (int j = 0; j < S; j += 2) { const float t = v[j]; v[j] = v[j + 1]; v[j + 1] = t; }
    }
    if constexpr (S == 4) {
        if (order & 2) {
#pragma unroll
            for (int j = 0; j < 2; ++j) { const float t = v[j]; v[j] = v[j + 2]; v[j + 2] = t; }
        }
    }
}

constexpr int KB = SEL_CHUNK;
// Sums over time (gradients of A, D and dt_bias) are kept in registers for so many chunks and then added to their totals in
// shared memory: one by one, the 2048 terms of a thread that walks 16384 steps alone would drift by some 1e-5 of their sum (equal
// terms, whose roundings all go the same way), in blocks by less than 1e-6.
constexpr int SUM_CHUNKS = 32;
template <int S> constexpr int in_registers = S == 4 ? KB / 2 : KB;      // steps whose decays and states are

template <int L, int S>
constexpr int backward_smem_bytes()
{
    using Q = Geo<L, S>;
    return (int)sizeof(float) * 2 * (KB * Q::CC * 9 + 2 * KB * Across<L, S>::COPIES * Q::NP + Q::WARPS * KB * 2 * Q::NP +
                                     Items<KB, Q::CC, Q::NH>::V * Q::NH + S * Q::NT);
}

// Walks its piece of time backwards.  It rebuilds the states of a chunk from the chunk's checkpoint, keeping them and the
// decays a_t in registers, and runs the reverse recurrence  g_t = C_t p_t + a_{t+1} g_{t+1}  (p = dy silu(z)) on them.
// With four states to a lane it does so by halves of a chunk, the later one first, for which the earlier one is run through
// once more: a quarter more exponentials, and registers for two blocks on an SM, whose barriers then do not stop all of it.
// The launch gives every thread 128 registers, of which the preparing warps hand 40 to those of the recurrence.
// Measured (N = 16, bfloat16, gated): 4 x 2048 x 2048 whole 445 us, issue slots 61 % busy, a third of the
// recurrence's instructions for the sums over lanes.  Before the decays' correction, whole 424 us, S = 4 in this place 495, and
// split into nine pieces 338 us and 80 more for what enters them.  Sums over channels through shared memory instead would cost 1 KB per warp and step.
template <typename T, int L, int S, bool VEC>
__global__ void __launch_bounds__(Geo<L, S>::NT + Geo<L, S>::NH, Geo<L, S>::BLOCKS) sel_backward_kernel(const SelArgs a)
{
    using Q = Geo<L, S>;
    using X = Across<L, S>;
    constexpr int CC = Q::CC, NT = Q::NT, NP = Q::NP, NH = Q::NH, COPIES = X::COPIES;
    extern __shared__ float smem[];
    float2 *s_in = reinterpret_cast<float2 *>(smem);      // [2][KB][CC]: dt, dt x
    float *s_p = smem + 4 * KB * CC;                      // [2][KB][CC]: p
    float *s_x = s_p + 2 * KB * CC;                       // x
    float *s_s = s_x + 2 * KB * CC;                       // slope of the step size
    float *s_q = s_s + 2 * KB * CC;                       // dy times the slope of silu(z)
    float *s_y = s_q + 2 * KB * CC, *s_gb = s_y + 2 * KB * CC, *s_ga = s_gb + 2 * KB * CC;      // sums over the states: C h, g B, g a h A log2(e)
    float *s_b = s_ga + 2 * KB * CC, *s_c = s_b + 2 * KB * COPIES * NP;              // [2][KB][COPIES][NP]
    float *s_bc = s_c + 2 * KB * COPIES * NP;             // [2][warp][KB][B, C][NP]
    float *s_sum = s_bc + 2 * Q::WARPS * KB * 2 * NP;     // totals over time: [2 V][preparing thread], [2 S][recurrence thread]
    const Block<KB, CC> blk(a);
    const bool gated = a.z.p != nullptr;
    const int64_t nchunks = (a.T + SEL_CHUNK - 1) / SEL_CHUNK;

    if (threadIdx.x >= NT) {
        using P = Part<KB, CC, NH>;
        constexpr int V = P::V, ITEMS = P::I::ITEMS, ROWS = P::I::ROWS, COLS = P::I::COLS;
        using F = Pack<float, V>;
        asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
        const int tid = threadIdx.x - NT;
        const P part(blk, tid);
        float skip[V], bias[V], dD[V], dbias[V];
        part.channel_values(skip, a.D);
        part.channel_values(bias, a.dt_bias);
#pragma unroll
        for (int j = 0; j < V; ++j) dD[j] = dbias[j] = s_sum[j * NH + tid] = s_sum[(V + j) * NH + tid] = 0.0f;
        struct Raw {
            RawPack<T, V, VEC> x[ITEMS], dt[ITEMS], z[ITEMS], dy[ITEMS];
            GroupRows<T, KB, CC, NP, NH, COPIES> b, c;
        } raw[2];
        // chunks are numbered in time and walked backwards
        auto fetch = [&](Raw &f, int64_t k) {
            if (k < 0) return;
            part.fetch(f.x, a.x, blk, k);
            part.fetch(f.dt, a.dt, blk, k);
            part.fetch(f.dy, a.dy, blk, k);
            if (gated) part.fetch(f.z, a.z, blk, k);
            f.b.fetch(blk, a.Bm, a.N, k, tid);
            f.c.fetch(blk, a.Cm, a.N, k, tid);
        };
        auto stage = [&](const Raw &f, int64_t k) {
            if (k < 0) return;
            const int buf = (int)(k & 1) * KB * CC, steps = blk.steps(k);
#pragma unroll
            for (int i = 0; i < ITEMS; ++i) {
                const int r = part.row + i * ROWS, at = buf + r * CC + part.col;
                if (r >= KB) continue;
                float d[V], pre[V];
                step_sizes(d, pre, f.dt[i], bias, a.softplus, part.there(steps, r));
                F fx, fs, fq, fp;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float x = f.x[i].get(j), up = f.dy[i].get(j), u = d[j] * x;
                    s_in[at + j] = make_float2(d[j], u);
                    fx.v[j] = x;
                    fs.v[j] = a.softplus ? sigmoid_f(pre[j]) : 1.0f;
                    float p = up;
                    if (gated) {
                        const float z = f.z[i].get(j), sg = sigmoid_f(z), gate = z * sg;
                        p = up * gate;
                        fq.v[j] = up * fmaf(gate, 1.0f - sg, sg);
                    }
                    fp.v[j] = p;
                }
                *reinterpret_cast<F *>(s_p + at) = fp;
                *reinterpret_cast<F *>(s_x + at) = fx;
                *reinterpret_cast<F *>(s_s + at) = fs;
                if (gated) *reinterpret_cast<F *>(s_q + at) = fq;
            }
            f.b.stage(s_b + (k & 1) * KB * COPIES * NP, tid);
            f.c.stage(s_c + (k & 1) * KB * COPIES * NP, tid);
        };
        auto emit = [&](int64_t k) {
            if (k >= blk.count) return;
            const int buf = (int)(k & 1) * KB * CC, steps = blk.steps(k);
            const float *sums = s_bc + (k & 1) * Q::WARPS * KB * 2 * NP;
            float *to = a.part_bc + (((blk.w.tile * a.B + blk.w.b) * a.T + blk.time(k)) * a.G + blk.w.g) * 2 * NP;
            for (int i = tid; i < steps * 2 * NP; i += NH) {
                float s = 0.0f;
#pragma unroll
                for (int q = 0; q < Q::WARPS; ++q) s += sums[q * KB * 2 * NP + i];
                to[(int64_t)(i / (2 * NP)) * a.G * 2 * NP + i % (2 * NP)] = s;
            }
            int64_t out = (blk.w.b * a.T + blk.time(k) + part.row) * a.M + part.ch;
#pragma unroll
            for (int i = 0; i < ITEMS; ++i, out += ROWS * (int64_t)a.M) {
                const int r = part.row + i * ROWS, have = part.there(steps, r), at = buf + r * CC + part.col;
                if (have <= 0) continue;
                const F fx = *reinterpret_cast<const F *>(s_x + at), fs = *reinterpret_cast<const F *>(s_s + at),
                        fb = *reinterpret_cast<const F *>(s_gb + at), fa = *reinterpret_cast<const F *>(s_ga + at),
                        fp = *reinterpret_cast<const F *>(s_p + at);
                F fq, fy;
                if (gated) {
                    fq = *reinterpret_cast<const F *>(s_q + at);
                    fy = *reinterpret_cast<const F *>(s_y + at);
                }
                Pack<T, V> ox, od, oz;
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float p = fp.v[j], x = fx.v[j];
                    const float d = fmaf(fb.v[j], x, fa.v[j] * LN2) * fs.v[j];
                    ox.v[j] = from_f32<T>(fmaf(s_in[at + j].x, fb.v[j], skip[j] * p));
                    od.v[j] = from_f32<T>(d);
                    if (gated) oz.v[j] = from_f32<T>(fq.v[j] * fmaf(skip[j], x, fy.v[j]));
                    dD[j] = fmaf(p, x, dD[j]);
                    dbias[j] += d;
                }
                store_pack<VEC>(static_cast<T *>(a.dx) + out, ox, have);
                store_pack<VEC>(static_cast<T *>(a.ddt) + out, od, have);
                if (gated) store_pack<VEC>(static_cast<T *>(a.dz) + out, oz, have);
            }
            if (k % SUM_CHUNKS == 0) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    s_sum[j * NH + tid] += dD[j];
                    s_sum[(V + j) * NH + tid] += dbias[j];
                    dD[j] = dbias[j] = 0.0f;
                }
            }
        };
        fetch(raw[0], blk.count - 1);
        fetch(raw[1], blk.count - 2);
        stage(raw[0], blk.count - 1);
        fetch(raw[0], blk.count - 3);
        for (int64_t k = blk.count - 1; k >= 0; k -= 2) {
            meet<NT + NH>();
            emit(k + 1);
            stage(raw[1], k - 1);
            fetch(raw[1], k - 3);
            if (k < 1) break;
            meet<NT + NH>();
            emit(k);
            stage(raw[0], k - 2);
            fetch(raw[0], k - 4);
        }
        meet<NT + NH>();
        emit(0);
        // sums of the threads that had the same columns (chunk 0, the last one, has left them all in the totals)
        asm volatile("bar.sync 1, %0;" ::"n"(NH) : "memory");
        for (int i = tid; i < 2 * CC; i += NH) {
            const int ch = i % CC, which = i / CC;
            double s = 0.0;
            for (int q = ch / V; q < NH; q += COLS) s += s_sum[(which * V + ch % V) * NH + q];
            if (blk.w.ch0 + ch < blk.per) a.part_d[((blk.w.b * a.segments + blk.w.seg) * 2 + which) * a.M + blk.w.g * blk.per + blk.w.ch0 + ch] = (float)s;
        }
        // rows behind the sequence have no gradient
        const int64_t z_lo = blk.t_end > blk.t_lo ? blk.t_end : blk.t_lo;
        for (int64_t i = tid; i < (blk.t_hi - z_lo) * CC; i += NH) {
            const int ch = blk.w.ch0 + (int)(i % CC);
            if (ch >= blk.per) continue;
            const int64_t at = (blk.w.b * a.T + z_lo + i / CC) * a.M + blk.w.g * blk.per + ch;
            static_cast<T *>(a.dx)[at] = from_f32<T>(0.0f);
            static_cast<T *>(a.ddt)[at] = from_f32<T>(0.0f);
            if (gated) static_cast<T *>(a.dz)[at] = from_f32<T>(0.0f);
        }
        for (int64_t i = tid; i < (blk.t_hi - z_lo) * 2 * NP; i += NH) {
            const int64_t row = ((blk.w.tile * a.B + blk.w.b) * a.T + z_lo + i / (2 * NP)) * a.G + blk.w.g;
            a.part_bc[row * 2 * NP + i % (2 * NP)] = 0.0f;
        }
        return;
    }

    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    constexpr int KH = in_registers<S>;
    using R = Pair<L, KH>;
    constexpr int GS = R::GS, SC = X::SC;
    static_assert(KH % GS == 0 && KH % SC == 0 && X::REST <= SC, "");
    const R pair(threadIdx.x);
    const int n0 = S * pair.l, warp = threadIdx.x / 32, cw = threadIdx.x % 32 / L;
    const int order = X::order(cw);
    States<S> A2[2], g[2], dA[2];
    States<S> state[2];      // the chunk's checkpoint
    float *sum_A = s_sum + 2 * Items<KB, CC, NH>::V * NH + threadIdx.x;
#pragma unroll
    for (int i = 0; i < 2 * S; ++i) sum_A[i * NT] = 0.0f;
    const float *ckpt[2];
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = blk.w.ch0 + pair.channel(k), m = blk.w.g * blk.per + c;
        float r[S] = {}, v[S] = {};
        if (c < blk.per) load_rates(r, a.A + (int64_t)m * a.N, n0, a.N);
        States<S> A2_here;
        A2_here.set(r);
        reorder(r, order);
        A2[k].set(r);
#pragma unroll
        for (int q = 0; q < S / 2; ++q) {
            A2_here.q[q] = mul2(A2_here.q[q], both(LOG2E));
            A2[k].q[q] = mul2(A2[k].q[q], both(LOG2E));
            dA[k].q[q] = both(0.0f);
        }
        if (c < blk.per) enter<true, NP, S>(v, a, blk.w, m, n0, A2_here);
        reorder(v, order);
        g[k].set(v);
        state[k].fill(0.0f);
        ckpt[k] = c < blk.per ? a.ckpt + ((blk.w.b * nchunks + blk.t_lo / SEL_CHUNK + blk.count - 1) * a.M + m) * NP + n0 : nullptr;
    }
    auto fetch_state = [&](bool there) {
#pragma unroll
        for (int k = 0; k < 2; ++k)
            if (there && ckpt[k]) {
                state[k].load(ckpt[k]);
                ckpt[k] -= (int64_t)a.M * NP;
            }
    };
    fetch_state(blk.count > 0);
    for (int64_t j = blk.count - 1; j >= 0; --j) {
        meet<NT + NH>();
        const float2 *in = s_in + (j & 1) * KB * CC;
        const float *p = s_p + (j & 1) * KB * CC;
        const float *b = s_b + ((j & 1) * KB * COPIES + order) * NP + n0, *cc = s_c + ((j & 1) * KB * COPIES + order) * NP + n0;
        float *y_out = s_y + (j & 1) * KB * CC, *gb_out = s_gb + (j & 1) * KB * CC, *ga_out = s_ga + (j & 1) * KB * CC;
        float *bc_out = s_bc + ((j & 1) * Q::WARPS + warp) * KB * 2 * NP + n0;
        // Leaves the warp's totals of `v`, gathered over SC steps from t on, in row `which` (B, C) of the steps.
        auto across = [&](States<S> (&v)[SC], int t, int which) {
#pragma unroll
            for (int i = 0; i < SC; ++i) X::halve_states(v[i]);
            if (X::REST > 1) {
                float s[SC];
#pragma unroll
                for (int i = 0; i < SC; ++i) s[i] = v[i].q[0].x;
                reduce_scatter<SC, X::REST, L>(s, threadIdx.x);
                bc_out[((t + cw % X::REST) * 2 + which) * NP + order] = s[0];
            } else {
                float s[S];
                v[0].get(s);
#pragma unroll
                for (int i = 0; i < X::KEPT; ++i) bc_out[(t * 2 + which) * NP + (i ^ order)] = s[i];
            }
        };
        States<S> lift[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) set_lift(lift[k], in[pair.channel(k)].x, A2[k]);
#pragma unroll 1      // unrolled, the halves are interleaved beyond what the registers hold
        for (int half = KB / KH - 1; half >= 0; --half) {
            States<S> h[2], av[KH][2], before[KH][2];      // decays, and the states in front of the steps
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float v[S];
                state[k].get(v);
                reorder(v, order);
                h[k].set(v);
            }
            if (KH < KB && half == 1) {
#pragma unroll
                for (int t = 0; t < KH; ++t) {
                    States<S> bb;
                    bb.load(b + t * COPIES * NP);
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float2 d = in[t * CC + pair.channel(k)];
#pragma unroll
                        for (int q = 0; q < S / 2; ++q) {
                            const float2 e = exponent(d.x, A2[k].q[q], lift[k].q[q]);
                            h[k].q[q] = fma2(make_float2(exp2_fast(e.x), exp2_fast(e.y)), h[k].q[q], mul2(both(d.y), bb.q[q]));
                        }
                    }
                }
            } else {
                fetch_state(j > 0);
            }
            {      // forward: decays, states, readout (also without a gate, a branch would keep the steps apart), gradient of C
                float y[GS];
                States<S> vc[SC];
#pragma unroll
                for (int i = 0; i < KH; ++i) {
                    const int t = half * KH + i;
                    States<S> bb, ccv;
                    bb.load(b + t * COPIES * NP);
                    ccv.load(cc + t * COPIES * NP);
                    float sum[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float2 d = in[t * CC + pair.channel(k)];
                        const float pt = p[t * CC + pair.channel(k)];
                        before[i][k] = h[k];
#pragma unroll
                        for (int q = 0; q < S / 2; ++q) {
                            const float2 e = exponent(d.x, A2[k].q[q], lift[k].q[q]);
                            av[i][k].q[q] = make_float2(exp2_fast(e.x), exp2_fast(e.y));
                            h[k].q[q] = fma2(av[i][k].q[q], h[k].q[q], mul2(both(d.y), bb.q[q]));
                            vc[i % SC].q[q] = k ? fma2(both(pt), h[k].q[q], vc[i % SC].q[q]) : mul2(both(pt), h[k].q[q]);
                        }
                        float2 s = mul2(ccv.q[0], h[k].q[0]);
                        if constexpr (S == 4) s = fma2(ccv.q[S / 4], h[k].q[S / 4], s);
                        sum[k] = s.x + s.y;
                    }
                    y[i % GS] = R::exchange(sum[0], sum[1]);
                    if (i % GS == GS - 1) pair.total(y, y_out, CC, t - (GS - 1));
                    if (i % SC == SC - 1) across(vc, t - (SC - 1), 1);
                }
            }
            {      // backward
                float sb[GS], sa[GS];
                States<S> vb[SC], dA_c[2];      // of these steps
                dA_c[0].fill(0.0f);
                dA_c[1].fill(0.0f);
#pragma unroll
                for (int i = KH - 1; i >= 0; --i) {
                    const int t = half * KH + i;
                    States<S> bb, ccv;
                    bb.load(b + t * COPIES * NP);
                    ccv.load(cc + t * COPIES * NP);
                    float tb[2], ta[2];
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        const float2 d = in[t * CC + pair.channel(k)];
                        const float pt = p[t * CC + pair.channel(k)];
                        float2 rb, ra;
#pragma unroll
                        for (int q = 0; q < S / 2; ++q) {
                            g[k].q[q] = fma2(ccv.q[q], both(pt), g[k].q[q]);
                            vb[i % SC].q[q] = k ? fma2(g[k].q[q], both(d.y), vb[i % SC].q[q]) : mul2(g[k].q[q], both(d.y));
                            rb = q ? fma2(g[k].q[q], bb.q[q], rb) : mul2(g[k].q[q], bb.q[q]);
                            g[k].q[q] = mul2(g[k].q[q], av[i][k].q[q]);
                            const float2 u = mul2(g[k].q[q], before[i][k].q[q]);
                            ra = q ? fma2(u, A2[k].q[q], ra) : mul2(u, A2[k].q[q]);
                            dA_c[k].q[q] = fma2(u, both(d.x), dA_c[k].q[q]);
                        }
                        tb[k] = rb.x + rb.y;
                        ta[k] = ra.x + ra.y;
                    }
                    sb[i % GS] = R::exchange(tb[0], tb[1]);
                    sa[i % GS] = R::exchange(ta[0], ta[1]);
                    if (i % GS == 0) {
                        pair.total(sb, gb_out, CC, t);
                        pair.total(sa, ga_out, CC, t);
                    }
                    if (i % SC == 0) across(vb, t, 0);
                }
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int q = 0; q < S / 2; ++q) dA[k].q[q] = add2(dA[k].q[q], dA_c[k].q[q]);
            }
        }
        if (j % SUM_CHUNKS == 0) {
#pragma unroll
            for (int i = 0; i < S; ++i) {
                float2 *d = &dA[i / (S / 2)].q[i % (S / 2)];
                sum_A[2 * i * NT] += d->x;
                sum_A[(2 * i + 1) * NT] += d->y;
                *d = both(0.0f);
            }
        }
    }
    meet<NT + NH>();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int c = blk.w.ch0 + pair.channel(k), m = blk.w.g * blk.per + c;
        if (c >= blk.per) continue;
        float v[S], r[S];
#pragma unroll
        for (int i = 0; i < S; ++i) v[i] = sum_A[(k * S + i) * NT];
        g[k].get(r);
        reorder(v, order);
        reorder(r, order);
        store_states(a.part_a + ((blk.w.b * a.segments + blk.w.seg) * a.M + m) * NP, v, n0, NP);
        if (a.dh0 && blk.w.seg == 0) store_states(a.dh0 + (blk.w.b * a.M + m) * a.N, r, n0, a.N);
    }
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
    for (int q0 = 0; q0 < tiles; q0 += 32) {      // in blocks, as above
        float block = 0.0f;
        for (int q = q0; q < min(q0 + 32, tiles); ++q) block += part[((q * rows + row) * 2 + which) * NP + n];
        s += block;
    }
    (which ? dC : dB)[row * N + n] = from_f32<T>(s);
}

// ---------------------------------------------------------------------------------------------- launchers

template <typename K>
cudaError_t allow_smem(K kernel, int bytes)
{
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : cudaSuccess;
}

// What every piece of time hands on.
template <typename T, int L, int S, bool VEC, bool REVERSE>
cudaError_t piece_states(const SelArgs &a, unsigned grid, cudaStream_t s)
{
    constexpr int smem = state_smem_bytes<L, S>();
    cudaError_t e = allow_smem(sel_state_kernel<T, L, S, VEC, REVERSE>, smem);
    if (e != cudaSuccess) return e;
    sel_state_kernel<T, L, S, VEC, REVERSE><<<grid, Geo<L, S>::NT + Geo<L, S>::NH, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int L, int S, bool VEC>
cudaError_t forward_typed(const SelArgs &a, const SelPlan &p, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.B * a.G * p.tiles * p.segments);
    constexpr int smem = forward_smem_bytes<L, S>();
    cudaError_t e = allow_smem(sel_forward_kernel<T, L, S, VEC>, smem);
    if (e == cudaSuccess && p.segments > 1) e = piece_states<T, L, S, VEC, false>(a, grid, s);
    if (e != cudaSuccess) return e;
    sel_forward_kernel<T, L, S, VEC><<<grid, Geo<L, S>::NT + Geo<L, S>::NH, smem, s>>>(a);
    return cudaGetLastError();
}

template <typename T, int L, int S, bool VEC>
cudaError_t backward_typed(const SelArgs &a, const SelPlan &p, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.B * a.G * p.tiles * p.segments);
    constexpr int smem = backward_smem_bytes<L, S>();
    // The kernel moves registers between its warps, out of the 128 that a thread is launched with; with fewer its warps
    // would wait for registers that nobody has.
    static const int registers = [] {
        cudaFuncAttributes f{};
        return cudaFuncGetAttributes(&f, sel_backward_kernel<T, L, S, VEC>) == cudaSuccess ? f.numRegs : 0;
    }();
    if (registers != 128) return cudaErrorInvalidKernelImage;
    cudaError_t e = allow_smem(sel_backward_kernel<T, L, S, VEC>, smem);
    if (e == cudaSuccess && p.segments > 1) e = piece_states<T, L, S, VEC, true>(a, grid, s);
    if (e != cudaSuccess) return e;
    sel_backward_kernel<T, L, S, VEC><<<grid, Geo<L, S>::NT + Geo<L, S>::NH, smem, s>>>(a);
    return cudaGetLastError();
}

// f.run<L, S>() for the lanes and states per lane of a plan.
template <typename F>
cudaError_t with_lanes(const SelPlan &p, const F &f)
{
    if (p.S == 2) {
        switch (p.L) {
        case 4: return f.template run<4, 2>();
        case 8: return f.template run<8, 2>();
        case 16: return f.template run<16, 2>();
        default: return f.template run<32, 2>();
        }
    }
    switch (p.L) {
    case 2: return f.template run<2, 4>();
    case 4: return f.template run<4, 4>();
    case 8: return f.template run<8, 4>();
    case 16: return f.template run<16, 4>();
    default: return f.template run<32, 4>();
    }
}
template <typename T, bool VEC>
struct Forward {
    const SelArgs &a;
    const SelPlan &p;
    cudaStream_t s;
    template <int L, int S> cudaError_t run() const { return forward_typed<T, L, S, VEC>(a, p, s); }
};
template <typename T, bool VEC>
struct Backward {
    const SelArgs &a;
    const SelPlan &p;
    cudaStream_t s;
    template <int L, int S> cudaError_t run() const { return backward_typed<T, L, S, VEC>(a, p, s); }
};

}  // namespace

// The scan on tensors of type T.
template <typename T>
cudaError_t selective_forward_typed(const SelArgs &a, const SelPlan &p, cudaStream_t s)
{
    const bool vec = (a.M / a.G) % 4 == 0 && pack_aligned<T>(a.x) && pack_aligned<T>(a.dt) && pack_aligned<T>(a.z) &&
                     reinterpret_cast<uintptr_t>(a.y) % (4 * sizeof(T)) == 0;
    return vec ? with_lanes(p, Forward<T, true>{a, p, s}) : with_lanes(p, Forward<T, false>{a, p, s});
}

template <typename T>
cudaError_t selective_backward_typed(const SelArgs &a, const SelPlan &p, void *dB, void *dC, cudaStream_t s)
{
    const bool vec = (a.M / a.G) % 4 == 0 && pack_aligned<T>(a.x) && pack_aligned<T>(a.dt) && pack_aligned<T>(a.z) && pack_aligned<T>(a.dy) &&
                     ((reinterpret_cast<uintptr_t>(a.dx) | reinterpret_cast<uintptr_t>(a.ddt) | reinterpret_cast<uintptr_t>(a.dz)) %
                      (4 * sizeof(T))) == 0;
    const cudaError_t e = vec ? with_lanes(p, Backward<T, true>{a, p, s}) : with_lanes(p, Backward<T, false>{a, p, s});
    if (e != cudaSuccess) return e;
    const int64_t rows = a.B * a.T * a.G;
    sel_sum_bc_kernel<T><<<(unsigned)ceil_div(rows * 2 * a.N, 256), 256, 0, s>>>(static_cast<T *>(dB), static_cast<T *>(dC), a.part_bc,
                                                                                p.tiles, rows, a.N, p.NP);
    return cudaGetLastError();
}

}  // namespace exb
