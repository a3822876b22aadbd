// Group norm with an activation on channels-last tensors (sample, position, channel):
//
//   y = act((x - mean) rstd w + b),  mean and variance over the positions and the channels of a group of one sample.
//
// Three mappings.  One position per sample (tokens): a few lanes hold a group in registers.  Maps: a cluster of blocks takes
// a sample, each block a run of positions and all channels of some groups; the blocks exchange their sums over distributed
// shared memory and read their run again, from the L2 cache, to apply them.  Few large maps: the same as two kernels, with
// as many blocks as the GPU takes.
#include "exb_norm.cuh"

#include <cooperative_groups.h>

namespace exb {

namespace {

constexpr int NT = 256;

template <typename T>
__device__ __forceinline__ float param(const void *p, int64_t i, int f32)
{
    return f32 ? static_cast<const float *>(p)[i] : to_f32(static_cast<const T *>(p)[i]);
}

// The activation of all pairs, and d times its slope; one branch for all of them.
template <int P>
__device__ __forceinline__ void activate(float2 (&v)[P], int act)
{
    if (act == EXB_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = silu2(v[i]);
    } else if (act == EXB_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < P; ++i) v[i] = make_float2(max_nan(v[i].x, 0.0f), max_nan(v[i].y, 0.0f));
    }
}
template <int P>
__device__ __forceinline__ void activate_backward(float2 (&d)[P], const float2 (&pre)[P], int act)
{
    if (act == EXB_ACT_SILU) {
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = mul2(d[i], silu_slope2(pre[i]));
    } else if (act == EXB_ACT_RELU) {
#pragma unroll
        for (int i = 0; i < P; ++i) d[i] = make_float2(pre[i].x > 0.0f ? d[i].x : 0.0f, pre[i].y > 0.0f ? d[i].y : 0.0f);
    }
}

// Weight or bias of V channels from c on (the first `left` of them exist), `absent` where there is none.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void load_params(float (&v)[V], const void *p, int64_t c, int left, int f32, float absent)
{
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = absent;
    if (!p) return;
    if (VEC && f32 && V % 4 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {
#pragma unroll
        for (int i = 0; i + 3 < V; i += 4) {
            const float4 q = left > 0 ? *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + c + i) : make_float4(absent, absent, absent, absent);
            v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < V; ++i)
        if (i < left) v[i] = param<T>(p, c + i, f32);
}

// 1 / sqrt(v), the approximation refined once.
__device__ __forceinline__ float inverse_sqrt(float v)
{
    const float r = rsqrtf(v);
    return v > 0.0f && r < 1e18f ? r * fmaf(-0.5f * v * r, r, 1.5f) : r;
}

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Number of values, their mean and the sum of their squared distances from it.
struct Moments {
    float n, mean, m2;
};

// Moments of `count` sets of values together, by one warp: the mean about the first set's, then every set's distances with
// n (mean - total mean)^2, so that a large common offset costs no digits.  get(i): the i-th set; the same in all lanes.
template <typename Get>
__device__ __forceinline__ Moments join(int count, const Get &get)
{
    const int lane = threadIdx.x % 32;
    const float base = get(0).mean;
    float n = 0.0f, sum = 0.0f;
    for (int i = lane; i < count; i += 32) {
        const Moments m = get(i);
        n += m.n;
        sum = fmaf(m.n, m.mean - base, sum);
    }
    n = warp_sum(n);
    const float off = warp_sum(sum) / n, mean = base + off;
    float m2 = 0.0f;
    for (int i = lane; i < count; i += 32) {
        const Moments m = get(i);
        const float d = (m.mean - base) - off;
        m2 += fmaf(m.n * d, d, m.m2);
    }
    return Moments{n, mean, warp_sum(m2)};
}

// ---------------------------------------------------------------------------------------------- tokens

// L lanes hold the channels of a group, K packs of V each; lane l has packs l, l + L, ...  A lane group keeps to its group
// and takes every `strides`-th sample, the next one on its way: weight and bias stay in registers, and so do the sums of
// their gradients.  V is 1 where rows are not aligned (a pair then is a channel and nothing).
// Several samples at a time, as many as the registers of four blocks on an SM hold: 8191 x 1536 in 24 groups takes 15.7 us in
// float32 (101 MB, 6.4 TB/s) with three at a time, 22 with four, which spill, and 29 with one; in bfloat16 (50 MB) 12.7 us
// with two and 20 with four.
template <typename T, int V, int L, int K, bool VEC>
struct Token {
    static constexpr int P = V > 1 ? V / 2 : 1;      // pairs of a pack
    static constexpr int ROWS = K * V <= 4 ? 3 : (K * V <= 16 ? 2 : 1);      // samples at a time
    int64_t first;
    int l, per, g;
    bool alive;

    __device__ __forceinline__ Token(const NormArgs &a, int64_t strides)
    {
        const int64_t q = (blockIdx.x * (int64_t)NT + threadIdx.x) / L;
        l = threadIdx.x % L;
        per = a.C / a.G;
        g = (int)(q % a.G);
        first = q / a.G;
        alive = first < strides;
    }
    __device__ __forceinline__ int channel(int k) const { return (k * L + l) * V; }
    // x points to the group's first channel of a sample
    __device__ __forceinline__ void fetch(RawPack<T, V, VEC> (&r)[K], const T *x, bool here) const
    {
#pragma unroll
        for (int k = 0; k < K; ++k) r[k].load(x + channel(k), here ? per - channel(k) : 0);
    }
    __device__ __forceinline__ static float2 pair(const RawPack<T, V, VEC> &r, int i)
    {
        if constexpr (V > 1) return r.pair(i);
        else return make_float2(r.get(0), 0.0f);
    }
    __device__ __forceinline__ void values(float2 (&v)[K][P], const void *p, int f32, float absent) const
    {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = channel(k) + 2 * i;
                v[k][i].x = (p && c < per) ? param<T>(p, g * per + c, f32) : absent;
                v[k][i].y = (p && V > 1 && c + 1 < per) ? param<T>(p, g * per + c + 1, f32) : absent;
            }
    }
    // 0 for channels that do not exist
    __device__ __forceinline__ void mask(float2 (&v)[K][P]) const
    {
        if (per == L * K * V && V > 1) return;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const int c = channel(k) + 2 * i;
                if (c >= per) v[k][i].x = 0.0f;
                if (V == 1 || c + 1 >= per) v[k][i].y = 0.0f;
            }
    }
    __device__ __forceinline__ void store(T *y, const float2 (&v)[K][P]) const
    {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Pack<T, V> out;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                out.v[2 * i] = from_f32<T>(v[k][i].x);
                if constexpr (V > 1) out.v[2 * i + 1] = from_f32<T>(v[k][i].y);
            }
            store_pack<VEC>(y + channel(k), out, per - channel(k));
        }
    }
};
template <int L>
__device__ __forceinline__ float lane_sum(float v)
{
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

template <typename T, int V, int L, int K, bool VEC>
__global__ void __launch_bounds__(NT, K * V <= 8 ? 4 : 1) norm_token_forward_kernel(const NormArgs a, int64_t strides)
{
    using U = Token<T, V, L, K, VEC>;
    constexpr int P = U::P, ROWS = U::ROWS;
    const U u(a, strides);
    float2 w[K][P], b[K][P];
    u.values(w, a.weight, a.params_f32, 1.0f);
    u.values(b, a.bias, a.params_f32, 0.0f);
    RawPack<T, V, VEC> next[ROWS][K];
    // samples of this lane group; rounds of ROWS samples, as many for every lane of the warp
    const int mine = u.alive && u.first < a.R ? (int)((a.R - u.first + strides - 1) / strides) : 0;
    const int rounds = (int)((a.R + ROWS * strides - 1) / (ROWS * strides));
    const int64_t first = u.alive ? u.first : 0;
    const T *x = static_cast<const T *>(a.x.p) + first * a.x.sb + u.g * u.per;
    T *y = static_cast<T *>(a.y) + first * a.C + u.g * u.per;
    float *stat = (u.l == 0 ? a.mean : a.rstd) + first * a.G + u.g;      // lane 0 keeps the mean, lane 1 (or 0 too) the rest
    const int64_t dx = strides * a.x.sb, dy = strides * a.C, ds = strides * a.G;
#pragma unroll
    for (int q = 0; q < ROWS; ++q, x += dx) u.fetch(next[q], x, q < mine);
    const float inv = 1.0f / u.per;
    for (int j = 0; j < rounds; ++j) {
        float2 v[ROWS][K][P];
        float base[ROWS], mean[ROWS], rstd[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {      // about the group's first value: a large common offset costs no digits
            base[q] = U::pair(next[q][0], 0).x;
            if (L > 1) base[q] = __shfl_sync(0xffffffffu, base[q], threadIdx.x % 32 - u.l);
            float2 sum = both(0.0f);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) v[q][k][i] = add2(U::pair(next[q][k], i), both(-base[q]));
            u.mask(v[q]);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) sum = add2(sum, v[q][k][i]);
            mean[q] = sum.x + sum.y;
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q, x += dx) u.fetch(next[q], x, (j + 1) * ROWS + q < mine);
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            mean[q] = lane_sum<L>(mean[q]) * inv;
            if (u.l == 0 && j * ROWS + q < mine) stat[q * ds] = base[q] + mean[q];
            float2 sq = both(0.0f);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) v[q][k][i] = add2(v[q][k][i], both(-mean[q]));
            u.mask(v[q]);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) sq = fma2(v[q][k][i], v[q][k][i], sq);
            rstd[q] = sq.x + sq.y;
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q) rstd[q] = inverse_sqrt(lane_sum<L>(rstd[q]) * inv + a.eps);
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
#pragma unroll
            for (int k = 0; k < K; ++k) {
#pragma unroll
                for (int i = 0; i < P; ++i) v[q][k][i] = fma2(mul2(v[q][k][i], both(rstd[q])), w[k][i], b[k][i]);
                activate(v[q][k], a.act);
            }
            if (j * ROWS + q < mine) {
                u.store(y, v[q]);
                if (u.l == 1) *stat = rstd[q];
                if (L == 1) a.rstd[stat - a.mean] = rstd[q];
            }
            y += dy;
            stat += ds;
        }
    }
}

// Sums over samples and positions are kept in registers for so many of them (rounds: one or two samples each) and then added to
// their totals in memory: thousands of equal terms (as the gradient of a mean has) one by one would drift by 1e-5 of their
// sum, because each addition rounds the same way.
constexpr int SUM_ROUNDS = 64, SUM_POSITIONS = 64;

template <typename T, int V, int L, int K, bool VEC>
__global__ void __launch_bounds__(NT, K * V <= 8 ? 2 : 1) norm_token_backward_kernel(const NormArgs a, int64_t strides)
{
    using U = Token<T, V, L, K, VEC>;
    constexpr int P = U::P;
    const U u(a, strides);
    float2 w[K][P], b[K][P], dw[K][P], db[K][P];
    u.values(w, a.weight, a.params_f32, 1.0f);
    u.values(b, a.bias, a.params_f32, 0.0f);
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i) dw[k][i] = db[k][i] = both(0.0f);
    constexpr int ROWS = U::ROWS > 2 ? 2 : U::ROWS;
    const int mine = u.alive && u.first < a.R ? (int)((a.R - u.first + strides - 1) / strides) : 0;
    const int rounds = (int)((a.R + ROWS * strides - 1) / (ROWS * strides));      // the same for every lane of the warp
    const int64_t first = u.alive ? u.first : 0;
    const T *x = static_cast<const T *>(a.x.p) + first * a.x.sb + u.g * u.per, *dy = static_cast<const T *>(a.dy.p) + first * a.dy.sb + u.g * u.per;
    T *out = static_cast<T *>(a.dx) + first * a.C + u.g * u.per;
    int64_t stat = first * a.G + u.g;
    const int64_t step_x = strides * a.x.sb, step_dy = strides * a.dy.sb, step_out = strides * a.C, step_stat = strides * a.G;
    const float inv = 1.0f / u.per;
    RawPack<T, V, VEC> px[ROWS][K], pg[ROWS][K];
    float next_mean[ROWS], next_rstd[ROWS];
    auto fetch = [&](int q, bool here) {
        u.fetch(px[q], x, here);
        u.fetch(pg[q], dy, here);
        next_mean[q] = here ? a.mean[stat] : 0.0f;
        next_rstd[q] = here ? a.rstd[stat] : 0.0f;
        x += step_x;
        dy += step_dy;
        stat += step_stat;
    };
#pragma unroll
    for (int q = 0; q < ROWS; ++q) fetch(q, q < mine);
    // adds the sums to the lane group's row of a.part, which only it touches, or starts the row with them
    auto settle = [&](bool add) {
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
#pragma unroll
                for (int h = 0; h < (V > 1 ? 2 : 1); ++h) {
                    const int c = u.channel(k) + 2 * i + h;
                    if (!u.alive || c >= u.per) continue;
                    float *to = a.part + u.first * 2 * a.C + u.g * u.per + c;
                    const float w_sum = h ? dw[k][i].y : dw[k][i].x, b_sum = h ? db[k][i].y : db[k][i].x;
                    to[0] = add ? to[0] + w_sum : w_sum;
                    to[a.C] = add ? to[a.C] + b_sum : b_sum;
                }
                dw[k][i] = db[k][i] = both(0.0f);
            }
    };
    for (int j = 0; j < rounds; ++j) {
        if (j > 0 && j % SUM_ROUNDS == 0) settle(j > SUM_ROUNDS);
        float2 n[ROWS][K][P], e[ROWS][K][P];
        float u1[ROWS], u2[ROWS], rstd[ROWS];
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            const float mean = next_mean[q];
            rstd[q] = next_rstd[q];
            float2 s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    n[q][k][i] = mul2(add2(U::pair(px[q][k], i), both(-mean)), both(rstd[q]));
                    e[q][k][i] = U::pair(pg[q][k], i);      // 0 where there is no channel
                }
            fetch(q, (j + 1) * ROWS + q < mine);
            u.mask(n[q]);
#pragma unroll
            for (int k = 0; k < K; ++k) {
                float2 pre[P];
#pragma unroll
                for (int i = 0; i < P; ++i) pre[i] = fma2(n[q][k][i], w[k][i], b[k][i]);
                activate_backward(e[q][k], pre, a.act);
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 d = e[q][k][i];
                    dw[k][i] = fma2(d, n[q][k][i], dw[k][i]);
                    db[k][i] = add2(db[k][i], d);
                    e[q][k][i] = mul2(d, w[k][i]);
                    s1 = add2(s1, e[q][k][i]);
                    s2 = fma2(e[q][k][i], n[q][k][i], s2);
                }
            }
            u1[q] = s1.x + s1.y;
            u2[q] = s2.x + s2.y;
        }
#pragma unroll
        for (int q = 0; q < ROWS; ++q) {
            u1[q] = lane_sum<L>(u1[q]) * inv;
            u2[q] = lane_sum<L>(u2[q]) * inv;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
                for (int i = 0; i < P; ++i) e[q][k][i] = mul2(both(rstd[q]), fma2(n[q][k][i], both(-u2[q]), add2(e[q][k][i], both(-u1[q]))));
            if (j * ROWS + q < mine) u.store(out, e[q]);
            out += step_out;
        }
    }
    settle(rounds > SUM_ROUNDS);
}

// ---------------------------------------------------------------------------------------------- maps

// A block's sample, positions and channels; its threads as columns of packs times rows of positions.
struct Spot {
    int64_t r, p0, p1;
    int g0, groups, c0, chans, chunk, packs, wide, px, ty, rows, count;
};
template <int V>
__device__ __forceinline__ Spot place(const NormArgs &a)
{
    Spot s;
    unsigned i = blockIdx.x;
    s.chunk = (int)(i % (unsigned)a.chunks);      // neighbours: the blocks of a cluster
    i /= (unsigned)a.chunks;
    const int sl = (int)(i % (unsigned)a.slabs);
    s.r = i / (unsigned)a.slabs;
    s.g0 = sl * a.slab;
    s.groups = s.g0 + a.slab < a.G ? a.slab : a.G - s.g0;
    s.c0 = s.g0 * a.per;
    s.chans = s.groups * a.per;
    s.packs = (s.chans + V - 1) / V;
    s.wide = s.packs < NT ? s.packs : NT;
    s.rows = NT / s.wide;
    s.ty = threadIdx.x / s.wide;
    s.px = threadIdx.x - s.ty * s.wide;
    s.p0 = s.chunk * a.chunk;
    s.p1 = s.p0 + a.chunk < a.S ? s.p0 + a.chunk : a.S;
    s.count = s.ty < s.rows ? ((int)(s.p1 - s.p0) - s.ty + s.rows - 1) / s.rows : 0;      // positions of the thread
    if (s.ty >= s.rows) s.packs = 0;      // threads left over
    return s;
}
// Number of positions that the threads of row `ty` have.
__device__ __forceinline__ float positions(const Spot &s, int ty)
{
    const int n = (int)(s.p1 - s.p0), each = n / s.rows;
    return (float)(each + (ty < n - each * s.rows ? 1 : 0));
}

// The positions of a thread, walked with AHEAD of them on their way.  Aligned rows come through a ring in shared memory that
// only this thread writes (asynchronous copies) and reads, so that nothing but the copies themselves is waited for and no
// registers are held; others are loaded into registers.
constexpr int AHEAD = 8;
template <typename T, int V, bool VEC, bool TWO>
struct Walk {
    using R = RawPack<T, V, VEC>;
    static constexpr int RING = VEC ? NT * AHEAD * 16 * (TWO ? 2 : 1) : 0;      // bytes
    const T *x, *g;
    int64_t step_x, step_g;
    int left, count, issued = 0;
    uint4 *ring;

    __device__ __forceinline__ Walk(const NormArgs &a, const Spot &s, int p, uint4 *ring_) : ring(ring_ + threadIdx.x)
    {
        left = s.chans - p * V;
        count = s.count;
        x = static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V + (s.p0 + s.ty) * a.x.st;
        g = TWO ? static_cast<const T *>(a.dy.p) + s.r * a.dy.sb + s.c0 + p * V + (s.p0 + s.ty) * a.dy.st : nullptr;
        step_x = s.rows * a.x.st;
        step_g = TWO ? s.rows * a.dy.st : 0;
        if (VEC) {
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) issue();
        }
    }
    __device__ __forceinline__ void issue()
    {
        if (issued < count) {
            uint4 *to = ring + (issued % AHEAD) * NT;
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to)), "l"(x) : "memory");
            if (TWO) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((unsigned)__cvta_generic_to_shared(to + AHEAD * NT)), "l"(g) : "memory");
            x += step_x;
            g += step_g;
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
        ++issued;
    }
    __device__ __forceinline__ static void take(R &r, const uint4 *from)
    {
        if constexpr (VEC) {
            const uint4 v = *from;
            r.w[0] = v.x; r.w[1] = v.y; r.w[2] = v.z; r.w[3] = v.w;
        }
    }
    // f(pack of x, pack of dy) for the positions q ... end; peek(pack of x) sees the first of all before.
    template <typename F, typename Peek>
    __device__ __forceinline__ void some(int q, int end, const F &f, const Peek &peek)
    {
        R cx, cg;
        if constexpr (VEC) {
#pragma unroll 4
            for (; q < end; ++q) {
                asm volatile("cp.async.wait_group %0;" ::"n"(AHEAD - 1) : "memory");
                const uint4 *from = ring + (q % AHEAD) * NT;
                take(cx, from);
                if (TWO) take(cg, from + AHEAD * NT);
                if (q == 0) peek(cx);
                issue();
                f(cx, cg);
            }
        } else {
            for (; q < end; ++q) {
                cx.load(x, left);
                if (TWO) cg.load(g, left);
                if (q == 0) peek(cx);
                f(cx, cg);
                x += step_x;
                g += step_g;
            }
        }
    }
    // All positions.
    template <typename F>
    __device__ __forceinline__ void run(const F &f)
    {
        some(0, count, f, [](const R &) {});
        if (VEC) asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // All positions; after the first `stop` of them settle(stop) is called, which returns the number to stop at next.
    template <typename F, typename Peek, typename Settle>
    __device__ __forceinline__ void run(const F &f, const Peek &peek, int stop, const Settle &settle)
    {
        int q = 0;
        while (stop < count) {
            some(q, stop, f, peek);
            q = stop;
            stop = settle(q);
        }
        some(q, count, f, peek);
        if (VEC) asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
};
template <typename T, int V, bool VEC>
__device__ __forceinline__ float2 pair_of(const RawPack<T, V, VEC> &r, int i)
{
    if constexpr (V > 1) return r.pair(i);
    else return make_float2(r.get(0), 0.0f);
}

// Moments of every group over the block's positions, in s_m (see map_smem), passed to out(group of the block, moments).
// A thread takes the moments of its channels about their first value, so that a large common offset costs no digits, and moves
// them to their mean after 8, 64, 512, ... positions: where the first value lies far off, it would cost the digits of all that
// follow (a first value of 1e4 among 2048 of deviation 1: 1e-3 of the variance).  Where whole packs belong to one group, it
// joins those of a pack.
template <typename T, int V, bool VEC, typename Out>
__device__ __forceinline__ void block_moments(const NormArgs &a, const Spot &s, float2 *s_m, uint4 *ring, const Out &out)
{
    using W = Walk<T, V, VEC, false>;
    constexpr int P = V > 1 ? V / 2 : 1;
    const bool whole = V > 1 && a.per % V == 0;
    const int entries = whole ? s.chans / V : s.chans;      // of a row in s_m
    for (int p = s.px; p < s.packs; p += s.wide) {
        float2 k[P], sum[P], sq[P];
        const int left = s.chans - p * V;
#pragma unroll
        for (int i = 0; i < P; ++i) k[i] = sum[i] = sq[i] = both(0.0f);
        W(a, s, p, ring).run([&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 d = add2(pair_of(x, i), k[i]);
                sum[i] = add2(sum[i], d);
                sq[i] = fma2(d, d, sq[i]);
            }
        }, [&](const RawPack<T, V, VEC> &x) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 f = pair_of(x, i);
                k[i] = make_float2(-f.x, -f.y);
            }
        }, 8, [&](int n) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 mean = mul2(sum[i], both(1.0f / n)), from = k[i];
                k[i] = add2(from, make_float2(-mean.x, -mean.y));
                const float2 moved = add2(from, make_float2(-k[i].x, -k[i].y));      // the mean but for the rounding of k
                sq[i] = fma2(make_float2(-mean.x, -mean.y), sum[i], sq[i]);
                sq[i] = make_float2(max_nan(sq[i].x, 0.0f), max_nan(sq[i].y, 0.0f));
                sum[i] = fma2(both(-(float)n), moved, sum[i]);
            }
            return n < 1 << 27 ? 8 * n : 0x7fffffff;
        });
        const float n = (float)s.count, inv = s.count > 0 ? 1.0f / n : 0.0f;
        float mean[V], m2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float t = (i & 1) ? sum[i / 2].y : sum[i / 2].x, u = (i & 1) ? sq[i / 2].y : sq[i / 2].x, b = (i & 1) ? k[i / 2].y : k[i / 2].x;
            mean[i] = fmaf(t, inv, -b);
            m2[i] = max_nan(fmaf(-t * inv, t, u), 0.0f);
        }
        if (whole) {
            float off = 0.0f, total = 0.0f;
#pragma unroll
            for (int i = 1; i < V; ++i) off += mean[i] - mean[0];
            off *= 1.0f / V;
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = (mean[i] - mean[0]) - off;
                total += fmaf(n * d, d, m2[i]);
            }
            s_m[s.ty * entries + p] = make_float2(mean[0] + off, total);
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (i < left) s_m[s.ty * entries + p * V + i] = make_float2(mean[i], m2[i]);
        }
    }
    __syncthreads();
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int each = whole ? a.per / V : a.per;             // entries of a group in a row
    const int rows = s.p1 - s.p0 < s.rows ? (int)(s.p1 - s.p0) : s.rows;
    const float weight = whole ? (float)V : 1.0f;
    for (int g = warp; g < s.groups; g += NT / 32) {
        const Moments m = join(rows * each, [&](int i) {
            const int row = i / each;
            const float2 f = s_m[row * entries + g * each + i - row * each];
            return Moments{positions(s, row) * weight, f.x, f.y};
        });
        if (lane == 0) out(g, m);
    }
}

// Group of a channel, for channels one after the other.
struct GroupOf {
    int g, rest;      // group, channels of it that are left
    __device__ __forceinline__ GroupOf(int c, int per) : g(c / per) { rest = per - (c - g * per); }
    __device__ __forceinline__ void step(int per)
    {
        if (--rest == 0) {
            rest = per;
            ++g;
        }
    }
};

// y from x with the groups' mean and rstd in s_m.  ready() is called when the first positions are on their way: it waits
// for what s_m holds.
template <typename T, int V, bool VEC, typename Ready>
__device__ __forceinline__ void block_apply(const NormArgs &a, const Spot &s, const float2 *s_m, uint4 *ring, const Ready &ready)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    const int passes = (s.chans + V * s.wide - 1) / (V * s.wide);      // the same for all threads: ready() may be a barrier
    for (int k = 0; k < passes; ++k) {
        const int p = s.px + k * s.wide;
        const bool there = p < s.packs;
        const int left = there ? s.chans - p * V : 0;
        Spot mine = s;
        if (!there) mine.count = 0;
        Walk<T, V, VEC, false> walk(a, mine, there ? p : 0, ring);
        if (k == 0) ready();
        if (!there) continue;
        float2 mean[P], scale[P], shift[P];
        float wv[V], bv[V];
        load_params<T, V, VEC>(wv, a.weight, s.c0 + p * V, left, a.params_f32, 1.0f);
        load_params<T, V, VEC>(bv, a.bias, s.c0 + p * V, left, a.params_f32, 0.0f);
        GroupOf group(p * V, a.per);
#pragma unroll
        for (int i = 0; i < V; ++i, group.step(a.per)) {
            const float2 f = p * V + i < s.chans ? s_m[group.g] : both(0.0f);
            const float m = -f.x, sc = f.y * wv[i], sh = bv[i];
            if (i % 2 == 0) { mean[i / 2] = both(m); scale[i / 2] = both(sc); shift[i / 2] = both(sh); }
            else { mean[i / 2].y = m; scale[i / 2].y = sc; shift[i / 2].y = sh; }
        }
        T *out = static_cast<T *>(a.y) + (s.r * a.S + s.p0 + s.ty) * a.C + s.c0 + p * V;
        const int64_t step = (int64_t)s.rows * a.C;
        walk.run([&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &) {
            Pack<T, V> y;
            float2 v[P];
#pragma unroll
            for (int i = 0; i < P; ++i) v[i] = fma2(add2(pair_of(x, i), mean[i]), scale[i], shift[i]);
            activate(v, a.act);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                y.v[2 * i] = from_f32<T>(v[i].x);
                if constexpr (V > 1) y.v[2 * i + 1] = from_f32<T>(v[i].y);
            }
            store_pack<VEC>(out, y, left);
            out += step;
        });
    }
}

// What the backward needs of a pack's channels: (x - mean) rstd = x rstd + centre would lose digits, so both are kept.
template <typename T, int V, bool VEC>
struct Channels {
    static constexpr int P = V > 1 ? V / 2 : 1;
    float2 mean[P], rstd[P], w[P], b[P];
    __device__ __forceinline__ Channels(const NormArgs &a, const Spot &s, int p)
    {
        float wv[V], bv[V];
        load_params<T, V, VEC>(wv, a.weight, s.c0 + p * V, s.chans - p * V, a.params_f32, 1.0f);
        load_params<T, V, VEC>(bv, a.bias, s.c0 + p * V, s.chans - p * V, a.params_f32, 0.0f);
        GroupOf group(p * V, a.per);
        const int64_t at = s.r * a.G + s.g0;
        float m = -a.mean[at + group.g], r = a.rstd[at + group.g];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            if (i % 2 == 0) { mean[i / 2] = both(m); rstd[i / 2] = both(r); w[i / 2] = both(wv[i]); b[i / 2] = both(bv[i]); }
            else { mean[i / 2].y = m; rstd[i / 2].y = r; w[i / 2].y = wv[i]; b[i / 2].y = bv[i]; }
            const int before = group.g;
            group.step(a.per);
            if (i + 1 < V && group.g != before && p * V + i + 1 < s.chans) {
                m = -a.mean[at + group.g];
                r = a.rstd[at + group.g];
            }
        }
    }
    // normed x, and the gradient in front of the activation
    template <typename R>
    __device__ __forceinline__ void get(float2 (&n)[P], float2 (&d)[P], const R &x, const R &up, int act) const
    {
        float2 pre[P];
#pragma unroll
        for (int i = 0; i < P; ++i) {
            n[i] = mul2(add2(pair_of(x, i), mean[i]), rstd[i]);
            d[i] = pair_of(up, i);
            pre[i] = fma2(n[i], w[i], b[i]);
        }
        activate_backward(d, pre, act);
    }
};

// Per channel, over the block's positions: the sums of d n and of d (d: gradient in front of the activation, n: normed x),
// left in s_m[channel] and in the block's row of a.part.  s_m: see map_smem.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void block_gradient_sums(const NormArgs &a, const Spot &s, float2 *s_m, uint4 *ring)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    for (int p = s.px; p < s.packs; p += s.wide) {
        const int left = s.chans - p * V;
        Walk<T, V, VEC, true> walk(a, s, p, ring);
        const Channels<T, V, VEC> h(a, s, p);
        float2 s1[P], s2[P];
#pragma unroll
        for (int i = 0; i < P; ++i) s1[i] = s2[i] = both(0.0f);
        float2 *own = s_m + s.ty * s.chans + p * V;
        auto put = [&]() {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                if (2 * i < left) own[2 * i] = make_float2(s1[i].x, s2[i].x);
                if (V > 1 && 2 * i + 1 < left) own[2 * i + 1] = make_float2(s1[i].y, s2[i].y);
            }
        };
        auto settle = [&](int q) {
            if (q > SUM_POSITIONS) {
#pragma unroll
                for (int i = 0; i < P; ++i) {
                    const float2 x = 2 * i < left ? own[2 * i] : both(0.0f), y = V > 1 && 2 * i + 1 < left ? own[2 * i + 1] : both(0.0f);
                    s1[i] = add2(s1[i], make_float2(x.x, y.x));
                    s2[i] = add2(s2[i], make_float2(x.y, y.y));
                }
            }
            put();
#pragma unroll
            for (int i = 0; i < P; ++i) s1[i] = s2[i] = both(0.0f);
            return q + SUM_POSITIONS;
        };
        walk.run([&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &g) {
            float2 n[P], d[P];
            h.get(n, d, x, g, a.act);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                s1[i] = add2(s1[i], d[i]);
                s2[i] = fma2(d[i], n[i], s2[i]);
            }
        }, [](const RawPack<T, V, VEC> &) {}, SUM_POSITIONS, settle);
        if (s.count > SUM_POSITIONS) settle(s.count);
        else put();
    }
    __syncthreads();
    float *out = a.part + (s.r * a.chunks + s.chunk) * 2 * a.C + s.c0;
    for (int c = threadIdx.x; c < s.chans; c += NT) {
        float2 t = both(0.0f);
        for (int k = 0; k < s.rows; ++k) t = add2(t, s_m[k * s.chans + c]);
        out[c] = t.y;
        out[a.C + c] = t.x;
        s_m[c] = t;      // of this column only this thread has read
    }
    __syncthreads();
}

// Sums of a group from sums per channel: weighted, one warp per group.
template <typename T, typename Get, typename Out>
__device__ __forceinline__ void group_sums(const NormArgs &a, const Spot &s, const Get &get, const Out &out)
{
    const int per = a.per, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int g = warp; g < s.groups; g += NT / 32) {
        float2 t = both(0.0f);
        for (int i = lane; i < per; i += 32) {
            const int c = g * per + i;
            t = fma2(both(a.weight ? param<T>(a.weight, s.c0 + c, a.params_f32) : 1.0f), get(c), t);
        }
        t = make_float2(warp_sum(t.x), warp_sum(t.y));
        if (lane == 0) out(g, t);
    }
}

// dx with the groups' two sums over their number of values in s_g; ready() as above.
template <typename T, int V, bool VEC, typename Ready>
__device__ __forceinline__ void block_gradient(const NormArgs &a, const Spot &s, const float2 *s_g, uint4 *ring, const Ready &ready)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    const int passes = (s.chans + V * s.wide - 1) / (V * s.wide);
    for (int k = 0; k < passes; ++k) {
        const int p = s.px + k * s.wide;
        const bool there = p < s.packs;
        const int left = there ? s.chans - p * V : 0;
        Spot mine = s;
        if (!there) mine.count = 0;
        Walk<T, V, VEC, true> walk(a, mine, there ? p : 0, ring);
        if (k == 0) ready();
        if (!there) continue;
        const Channels<T, V, VEC> h(a, s, p);
        float2 u[P], v[P];
        GroupOf group(p * V, a.per);
#pragma unroll
        for (int i = 0; i < V; ++i, group.step(a.per)) {
            const float2 f = s_g[p * V + i < s.chans ? group.g : 0];
            if (i % 2 == 0) { u[i / 2] = both(-f.x); v[i / 2] = both(-f.y); }
            else { u[i / 2].y = -f.x; v[i / 2].y = -f.y; }
        }
        T *out = static_cast<T *>(a.dx) + (s.r * a.S + s.p0 + s.ty) * a.C + s.c0 + p * V;
        const int64_t step = (int64_t)s.rows * a.C;
        walk.run([&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &g) {
            Pack<T, V> o;
            float2 n[P], d[P];
            h.get(n, d, x, g, a.act);
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 e = mul2(h.rstd[i], fma2(n[i], v[i], fma2(d[i], h.w[i], u[i])));
                o.v[2 * i] = from_f32<T>(e.x);
                if constexpr (V > 1) o.v[2 * i + 1] = from_f32<T>(e.y);
            }
            store_pack<VEC>(out, o, left);
            out += step;
        });
    }
}

// Final mean and rstd of a group.
__device__ __forceinline__ void finish_group(const NormArgs &a, const Spot &s, float2 *s_m, int g, const Moments &m, bool write)
{
    const float rstd = inverse_sqrt(m.m2 / m.n + a.eps);
    s_m[g] = make_float2(m.mean, rstd);
    if (write) {
        a.mean[s.r * a.G + s.g0 + g] = m.mean;
        a.rstd[s.r * a.G + s.g0 + g] = rstd;
    }
}

// ---- one cluster per sample (and slab of groups): a.chunks blocks, which is the cluster's size
//
// 256 x 4096 x 64 in 8 groups, silu, bfloat16: forward 93 us (268 MB past the second reading, which the L2 cache serves),
// backward 155 us (403 MB); about half of the issue slots busy, the rest the cluster's barriers and the memory latency at
// both ends of a block's run.  Two kernels: 155 and 279 us.

// Dynamic shared memory of the map kernels: the rings, then a.smem pairs (see map_smem), then what each says.
template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_cluster_forward_kernel(const NormArgs a)
{
    extern __shared__ uint4 ring[];
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const Spot s = place<V>(a);
    float2 *s_m = reinterpret_cast<float2 *>(reinterpret_cast<char *>(ring) + Walk<T, V, VEC, false>::RING);
    Moments *own = reinterpret_cast<Moments *>(s_m + a.smem);      // [groups]
    block_moments<T, V, VEC>(a, s, s_m, ring, [&](int g, const Moments &m) { own[g] = m; });
    block_apply<T, V, VEC>(a, s, s_m, ring, [&]() {
        cluster.sync();
        for (int g = threadIdx.x / 32; g < s.groups; g += NT / 32) {
            const Moments m = join(a.chunks, [&](int r) { return cluster.map_shared_rank(own, r)[g]; });
            if (threadIdx.x % 32 == 0) finish_group(a, s, s_m, g, m, s.chunk == 0);
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");      // done with the other blocks' moments (not .aligned: lanes may be apart here)
        __syncthreads();
    });
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");      // nobody reads this block's any more
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 2) norm_cluster_backward_kernel(const NormArgs a)
{
    extern __shared__ uint4 ring[];
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const Spot s = place<V>(a);
    float2 *s_m = reinterpret_cast<float2 *>(reinterpret_cast<char *>(ring) + Walk<T, V, VEC, true>::RING);
    float2 *own = s_m + a.smem;      // [groups] sums of the block
    block_gradient_sums<T, V, VEC>(a, s, s_m, ring);
    block_gradient<T, V, VEC>(a, s, s_m, ring, [&]() {
        group_sums<T>(a, s, [&](int c) { return s_m[c]; }, [&](int g, float2 t) { own[g] = t; });
        cluster.sync();
        const float inv = 1.0f / ((float)a.S * (float)a.per);
        for (int g = threadIdx.x; g < s.groups; g += NT) {
            float2 t = both(0.0f);
            for (int r = 0; r < a.chunks; ++r) t = add2(t, cluster.map_shared_rank(own, r)[g]);
            s_m[g] = mul2(t, both(inv));
        }
        asm volatile("barrier.cluster.arrive.release;" ::: "memory");      // as above
        __syncthreads();
    });
    asm volatile("barrier.cluster.wait.acquire;" ::: "memory");
}

// ---- two kernels

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_stats_kernel(const NormArgs a)
{
    extern __shared__ uint4 ring[];
    float2 *s_m = reinterpret_cast<float2 *>(reinterpret_cast<char *>(ring) + Walk<T, V, VEC, false>::RING);
    const Spot s = place<V>(a);
    block_moments<T, V, VEC>(a, s, s_m, ring, [&](int g, const Moments &m) {
        float *out = a.part + ((s.r * a.chunks + s.chunk) * a.G + s.g0 + g) * 2;
        out[0] = m.mean;
        out[1] = m.m2;
    });
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_apply_kernel(const NormArgs a)
{
    extern __shared__ uint4 ring[];
    float2 *s_m = reinterpret_cast<float2 *>(reinterpret_cast<char *>(ring) + Walk<T, V, VEC, false>::RING);      // [groups]
    const Spot s = place<V>(a);
    block_apply<T, V, VEC>(a, s, s_m, ring, [&]() {
        for (int g = threadIdx.x / 32; g < s.groups; g += NT / 32) {
            const Moments m = join(a.chunks, [&](int i) {
                const int64_t lo = i * a.chunk, hi = lo + a.chunk < a.S ? lo + a.chunk : a.S;
                const float *in = a.part + ((s.r * a.chunks + i) * a.G + s.g0 + g) * 2;
                return Moments{(float)((hi - lo) * a.per), in[0], in[1]};
            });
            if (threadIdx.x % 32 == 0) finish_group(a, s, s_m, g, m, s.chunk == 0);
        }
        __syncthreads();
    });
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 2) norm_backward_sums_kernel(const NormArgs a)
{
    extern __shared__ uint4 ring[];
    float2 *s_m = reinterpret_cast<float2 *>(reinterpret_cast<char *>(ring) + Walk<T, V, VEC, true>::RING);
    const Spot s = place<V>(a);
    block_gradient_sums<T, V, VEC>(a, s, s_m, ring);
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 2) norm_backward_apply_kernel(const NormArgs a)
{
    extern __shared__ uint4 ring[];
    float2 *s_m = reinterpret_cast<float2 *>(reinterpret_cast<char *>(ring) + Walk<T, V, VEC, true>::RING);      // [groups]
    const Spot s = place<V>(a);
    block_gradient<T, V, VEC>(a, s, s_m, ring, [&]() {
        const float inv = 1.0f / ((float)a.S * (float)a.per);
        group_sums<T>(a, s, [&](int c) {
            float2 t = both(0.0f);
#pragma unroll 4
            for (int k = 0; k < a.chunks; ++k) {
                const float *in = a.part + (s.r * a.chunks + k) * 2 * a.C + s.c0 + c;
                t = add2(t, make_float2(in[a.C], in[0]));
            }
            return t;
        }, [&](int g, float2 t) { s_m[g] = mul2(t, both(inv)); });
        __syncthreads();
    });
}

// ---------------------------------------------------------------------------------------------- launchers

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

struct Plan {
    bool tokens, packs, cluster;     // packs: whole packs fit a block's shared memory
    int64_t strides;                 // tokens: samples that are walked side by side
    int64_t chunk;
    int chunks, slab, slabs;
    int64_t forward_bytes, backward_bytes;
};

constexpr int TOKEN_MAX_GROUP = 1024;      // channels that a warp holds, 32 in a lane

// Lanes and packs that hold a group of `per` channels in packs of V.
void token_shape(int per, int V, int *L, int *K)
{
    const int packs = (per + V - 1) / V;
    *L = 1;
    while (*L < packs && *L < 32) *L *= 2;
    *K = 1;
    while (*L * *K < packs) *K *= 2;
}

Plan plan_of(int64_t R, int64_t S, int C, int G, int dtype, bool backward)
{
    Plan p{};
    const int per = C / G, V = dtype == EXB_F32 ? 4 : 8;
    p.tokens = S == 1 && per <= TOKEN_MAX_GROUP;
    // groups of a block: whole packs, up to 1024 channels.  Where whole packs would take more channels than a block's
    // shared memory has room for, one group and single channels.
    int unit = V / gcd(per, V);
    p.packs = per * unit <= NORM_MAX_GROUP;
    if (!p.packs) unit = 1;
    p.slab = (1024 / per) / unit * unit;
    if (p.slab < unit) p.slab = unit;
    if (p.slab > G) p.slab = G;
    p.slabs = (int)ceil_div(G, p.slab);
    // A cluster of 1, 2, 4 or 8 blocks per sample when that gives every SM two blocks, as large as leaves each thread
    // eight positions; otherwise two kernels, whose blocks need not run together: eight for every SM.
    const int packs = p.slab * per / V > 1 ? p.slab * per / V : 1, rows = packs < NT ? NT / packs : 1;
    int cluster = 1;
    while (cluster < 8 && S / (2 * cluster) >= 8 * rows) cluster *= 2;
    p.cluster = R * p.slabs * cluster >= 2 * 148;
    int64_t chunks = cluster;
    if (!p.cluster) {
        chunks = ceil_div(8 * 148, R * p.slabs);
        const int64_t most = ceil_div(S, 2 * rows);
        if (chunks > most) chunks = most;
        if (chunks > 256) chunks = 256;
    }
    p.chunk = ceil_div(S, chunks);
    p.chunks = p.cluster ? cluster : (int)ceil_div(S, p.chunk);
    // tokens: as many threads as are resident at once, so that no block waits for another's end; backward at least four
    // samples each, which leave one partial sum
    int L, K;
    token_shape(per, V, &L, &K);
    int64_t strides = (148ll * NT * (K * V > 8 ? 1 : (backward ? 2 : 4))) / ((int64_t)G * L);
    if (strides < 1) strides = 1;
    if (backward && strides > R / 4) strides = R / 4 > 64 ? R / 4 : 64;
    p.strides = strides < R ? strides : R;
    p.forward_bytes = p.tokens || p.cluster ? 0 : R * p.chunks * G * 2 * 4;
    p.backward_bytes = (p.tokens ? p.strides : R * p.chunks) * 2 * C * 4;
    return p;
}

template <typename T>
bool aligned(const View &x, const View &dy, const void *out, int C, int V)
{
    const int64_t bytes = V * sizeof(T);
    return C % V == 0 && reinterpret_cast<uintptr_t>(x.p) % bytes == 0 && x.sb % V == 0 && x.st % V == 0 &&
           reinterpret_cast<uintptr_t>(dy.p) % bytes == 0 && dy.sb % V == 0 && dy.st % V == 0 && reinterpret_cast<uintptr_t>(out) % bytes == 0;
}

// Columns [2][C] of the partial sums become dweight and dbias.
template <typename O>
struct PutParams {
    O *dweight, *dbias;
    int C;
    __device__ void operator()(int64_t col, float v) const
    {
        O *out = col < C ? dweight : dbias;
        if (out) out[col % C] = from_f32<O>(v);
    }
};

// Calls f.template run<V, L, K, VEC>() for the shape of a group.
template <typename T, int V, bool VEC, typename F>
cudaError_t with_token_shape(int per, const F &f)
{
    int L, K;
    token_shape(per, V, &L, &K);
    if (K == 1) {
        switch (L) {
        case 1: return f.template run<V, 1, 1, VEC>();
        case 2: return f.template run<V, 2, 1, VEC>();
        case 4: return f.template run<V, 4, 1, VEC>();
        case 8: return f.template run<V, 8, 1, VEC>();
        case 16: return f.template run<V, 16, 1, VEC>();
        default: return f.template run<V, 32, 1, VEC>();
        }
    }
    if (K == 2) return f.template run<V, 32, 2, VEC>();
    if (K == 4) return f.template run<V, 32, 4, VEC>();
    if constexpr (V <= 4) {
        if (K == 8) return f.template run<V, 32, 8, VEC>();
    }
    if constexpr (V == 1) {
        return K == 16 ? f.template run<V, 32, 16, VEC>() : f.template run<V, 32, 32, VEC>();
    }
    return cudaErrorInvalidValue;
}

template <typename T>
struct TokenForward {
    const NormArgs &a;
    int64_t strides;
    cudaStream_t s;
    template <int V, int L, int K, bool VEC>
    cudaError_t run() const
    {
        norm_token_forward_kernel<T, V, L, K, VEC><<<(unsigned)ceil_div(strides * a.G * L, NT), NT, 0, s>>>(a, strides);
        return cudaGetLastError();
    }
};
template <typename T>
struct TokenBackward {
    const NormArgs &a;
    int64_t strides;
    cudaStream_t s;
    template <int V, int L, int K, bool VEC>
    cudaError_t run() const
    {
        norm_token_backward_kernel<T, V, L, K, VEC><<<(unsigned)ceil_div(strides * a.G * L, NT), NT, 0, s>>>(a, strides);
        return cudaGetLastError();
    }
};

// Pairs of shared memory that a map kernel works in: one per thread row and channel (one per group at least).
template <int V>
int map_smem(const NormArgs &a)
{
    const int per = a.C / a.G, chans = a.slab * per, packs = (chans + V - 1) / V, wide = packs < NT ? packs : NT;
    return (NT / wide) * chans;
}

template <typename K>
cudaError_t allow_smem(K kernel, int bytes)
{
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : cudaSuccess;
}

// Launches `kernel` with clusters of a.chunks blocks.
template <typename K>
cudaError_t launch_clusters(K kernel, const NormArgs &a, unsigned grid, int smem, cudaStream_t s)
{
    cudaError_t e = allow_smem(kernel, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(NT);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = a.chunks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, a);
}

template <typename T, int V, bool VEC>
cudaError_t maps_forward(NormArgs a, bool cluster, cudaStream_t s)
{
    constexpr int RING = Walk<T, V, VEC, false>::RING;
    const int64_t blocks = a.R * a.chunks * a.slabs;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    const unsigned grid = (unsigned)blocks;
    a.smem = map_smem<V>(a);
    const int smem = RING + a.smem * (int)sizeof(float2), apply = RING + a.slab * (int)sizeof(float2);
    if (cluster) return launch_clusters(norm_cluster_forward_kernel<T, V, VEC>, a, grid, smem + a.slab * (int)sizeof(Moments), s);
    cudaError_t e = allow_smem(norm_stats_kernel<T, V, VEC>, smem);
    if (e == cudaSuccess) e = allow_smem(norm_apply_kernel<T, V, VEC>, apply);
    if (e != cudaSuccess) return e;
    norm_stats_kernel<T, V, VEC><<<grid, NT, smem, s>>>(a);
    norm_apply_kernel<T, V, VEC><<<grid, NT, apply, s>>>(a);
    return cudaGetLastError();
}
template <typename T, int V, bool VEC>
cudaError_t maps_backward(NormArgs a, bool cluster, cudaStream_t s)
{
    constexpr int RING = Walk<T, V, VEC, true>::RING;
    const int64_t blocks = a.R * a.chunks * a.slabs;
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    const unsigned grid = (unsigned)blocks;
    a.smem = map_smem<V>(a);
    const int smem = RING + a.smem * (int)sizeof(float2), apply = RING + a.slab * (int)sizeof(float2);
    if (cluster) return launch_clusters(norm_cluster_backward_kernel<T, V, VEC>, a, grid, smem + a.slab * (int)sizeof(float2), s);
    cudaError_t e = allow_smem(norm_backward_sums_kernel<T, V, VEC>, smem);
    if (e == cudaSuccess) e = allow_smem(norm_backward_apply_kernel<T, V, VEC>, apply);
    if (e != cudaSuccess) return e;
    norm_backward_sums_kernel<T, V, VEC><<<grid, NT, smem, s>>>(a);
    norm_backward_apply_kernel<T, V, VEC><<<grid, NT, apply, s>>>(a);
    return cudaGetLastError();
}

template <typename T>
cudaError_t forward_typed(const NormArgs &a, const Plan &p, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const int per = a.C / a.G;
    const bool vec = aligned<T>(a.x, View{}, a.y, a.C, V);
    if (p.tokens) {
        const TokenForward<T> f{a, p.strides, s};
        return vec && per % V == 0 ? with_token_shape<T, V, true>(per, f) : with_token_shape<T, 1, false>(per, f);
    }
    return vec && p.packs ? maps_forward<T, V, true>(a, p.cluster, s) : maps_forward<T, 1, false>(a, p.cluster, s);
}

template <typename T>
cudaError_t backward_typed(const NormArgs &a, const Plan &p, void *dweight, void *dbias, cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    const int per = a.C / a.G;
    const bool vec = aligned<T>(a.x, a.dy, a.dx, a.C, V);
    cudaError_t e;
    if (p.tokens) {
        const TokenBackward<T> f{a, p.strides, s};
        e = vec && per % V == 0 ? with_token_shape<T, V, true>(per, f) : with_token_shape<T, 1, false>(per, f);
    } else {
        e = vec && p.packs ? maps_backward<T, V, true>(a, p.cluster, s) : maps_backward<T, 1, false>(a, p.cluster, s);
    }
    if (e != cudaSuccess || (!dweight && !dbias)) return e;
    const int64_t rows = p.tokens ? p.strides : a.R * a.chunks;
    if (a.params_f32) launch_column_sum(PutParams<float>{(float *)dweight, (float *)dbias, a.C}, a.part, rows, 2 * (int64_t)a.C, s);
    else launch_column_sum(PutParams<T>{(T *)dweight, (T *)dbias, a.C}, a.part, rows, 2 * (int64_t)a.C, s);
    return cudaGetLastError();
}

Plan apply_plan(NormArgs &a, int dtype, void *ws, bool backward)
{
    const Plan p = plan_of(a.R, a.S, a.C, a.G, dtype, backward);
    a.chunk = p.chunk;
    a.chunks = p.chunks;
    a.slab = p.slab;
    a.slabs = p.slabs;
    a.per = a.C / a.G;
    a.part = static_cast<float *>(ws);
    return p;
}

}  // namespace

int64_t norm_workspace_bytes(int64_t R, int64_t S, int C, int G, int dtype, bool backward)
{
    const Plan p = plan_of(R, S, C, G, dtype, backward);
    return backward ? p.backward_bytes : p.forward_bytes;
}

cudaError_t launch_norm_forward(NormArgs a, int dtype, void *ws, cudaStream_t stream)
{
    const Plan p = apply_plan(a, dtype, ws, false);
    if (dtype == EXB_F32) return forward_typed<float>(a, p, stream);
    if (dtype == EXB_BF16) return forward_typed<__nv_bfloat16>(a, p, stream);
    return forward_typed<__half>(a, p, stream);
}

cudaError_t launch_norm_backward(NormArgs a, int dtype, void *dweight, void *dbias, void *ws, cudaStream_t stream)
{
    const Plan p = apply_plan(a, dtype, ws, true);
    if (dtype == EXB_F32) return backward_typed<float>(a, p, dweight, dbias, stream);
    if (dtype == EXB_BF16) return backward_typed<__nv_bfloat16>(a, p, dweight, dbias, stream);
    return backward_typed<__half>(a, p, dweight, dbias, stream);
}

}  // namespace exb
