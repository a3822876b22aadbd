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

__device__ __forceinline__ float2 activate2(float2 v, int act)
{
    if (act == EXB_ACT_SILU) return silu2(v);
    if (act == EXB_ACT_RELU) return make_float2(max_nan(v.x, 0.0f), max_nan(v.y, 0.0f));
    return v;
}
__device__ __forceinline__ float2 activate_slope2(float2 v, int act)
{
    if (act == EXB_ACT_SILU) return silu_slope2(v);
    if (act == EXB_ACT_RELU) return make_float2(v.x > 0.0f ? 1.0f : 0.0f, v.y > 0.0f ? 1.0f : 0.0f);
    return both(1.0f);
}

// Number of values, their mean and the sum of their squared distances from it.
struct Moments {
    float n, mean, m2;
};
__device__ __forceinline__ Moments merge(const Moments &a, const Moments &b)
{
    Moments r;
    r.n = a.n + b.n;
    if (b.n == 0.0f) return a;
    if (a.n == 0.0f) return b;
    const float d = b.mean - a.mean, f = b.n / r.n;
    r.mean = fmaf(d, f, a.mean);
    r.m2 = a.m2 + b.m2 + d * d * (a.n * f);
    return r;
}
__device__ __forceinline__ Moments merge_lanes(Moments v)
{
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) {
        Moments o;
        o.n = __shfl_xor_sync(0xffffffffu, v.n, m);
        o.mean = __shfl_xor_sync(0xffffffffu, v.mean, m);
        o.m2 = __shfl_xor_sync(0xffffffffu, v.m2, m);
        // the same order in both lanes, so that they agree to the last bit
        v = (threadIdx.x & m) ? merge(o, v) : merge(v, o);
    }
    return v;
}

// ---------------------------------------------------------------------------------------------- tokens

// L lanes hold the channels of a group, K packs of V each; lane l has packs l, l + L, ...  A lane group keeps to its group
// and takes every `strides`-th sample, the next one on its way: weight and bias stay in registers, and so do the sums of
// their gradients.  V is 1 where rows are not aligned (a pair then is a channel and nothing).
template <typename T, int V, int L, int K, bool VEC>
struct Token {
    static constexpr int P = V > 1 ? V / 2 : 1;      // pairs of a pack
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
    __device__ __forceinline__ void fetch(RawPack<T, V, VEC> (&r)[K], const View &v, int64_t row, bool here) const
    {
#pragma unroll
        for (int k = 0; k < K; ++k) r[k].load(static_cast<const T *>(v.p) + row * v.sb + g * per + channel(k), here ? per - channel(k) : 0);
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
    // 1 where the pair's channels exist
    __device__ __forceinline__ float2 there(int k, int i) const
    {
        const int c = channel(k) + 2 * i;
        return make_float2(c < per ? 1.0f : 0.0f, V > 1 && c + 1 < per ? 1.0f : 0.0f);
    }
    __device__ __forceinline__ void store(T *p, int64_t row, int C, const float2 (&v)[K][P]) const
    {
#pragma unroll
        for (int k = 0; k < K; ++k) {
            Pack<T, V> out;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                out.v[2 * i] = from_f32<T>(v[k][i].x);
                if constexpr (V > 1) out.v[2 * i + 1] = from_f32<T>(v[k][i].y);
            }
            store_pack<VEC>(p + row * C + g * per + channel(k), out, per - channel(k));
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
__global__ void __launch_bounds__(NT) norm_token_forward_kernel(const NormArgs a, int64_t strides)
{
    using U = Token<T, V, L, K, VEC>;
    constexpr int P = U::P;
    const U u(a, strides);
    float2 w[K][P], b[K][P];
    u.values(w, a.weight, a.params_f32, 1.0f);
    u.values(b, a.bias, a.params_f32, 0.0f);
    RawPack<T, V, VEC> next[K];
    u.fetch(next, a.x, u.first, u.alive && u.first < a.R);
    const int64_t rounds = (a.R + strides - 1) / strides;      // the same for every lane of the warp
    const float inv = 1.0f / u.per;
    for (int64_t j = 0; j < rounds; ++j) {
        const int64_t r = u.first + j * strides;
        const bool here = u.alive && r < a.R;
        float2 v[K][P], sum = both(0.0f), sq = both(0.0f);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                v[k][i] = U::pair(next[k], i);
                sum = add2(sum, v[k][i]);
            }
        u.fetch(next, a.x, r + strides, u.alive && r + strides < a.R);
        const float mean = lane_sum<L>(sum.x + sum.y) * inv;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                v[k][i] = add2(v[k][i], both(-mean));
                const float2 d = mul2(v[k][i], u.there(k, i));
                sq = fma2(d, d, sq);
            }
        const float rstd = 1.0f / sqrtf(lane_sum<L>(sq.x + sq.y) * inv + a.eps);
        if (!here) continue;
        if (u.l == 0) {
            a.mean[r * a.G + u.g] = mean;
            a.rstd[r * a.G + u.g] = rstd;
        }
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) v[k][i] = activate2(fma2(mul2(v[k][i], both(rstd)), w[k][i], b[k][i]), a.act);
        u.store(static_cast<T *>(a.y), r, a.C, v);
    }
}

template <typename T, int V, int L, int K, bool VEC>
__global__ void __launch_bounds__(NT) norm_token_backward_kernel(const NormArgs a, int64_t strides)
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
    const int64_t rounds = (a.R + strides - 1) / strides;      // the same for every lane of the warp
    const float inv = 1.0f / u.per;
    for (int64_t j = 0; j < rounds; ++j) {
        const int64_t r = u.first + j * strides;
        const bool here = u.alive && r < a.R;
        RawPack<T, V, VEC> px[K], pg[K];
        u.fetch(px, a.x, r, here);
        u.fetch(pg, a.dy, r, here);
        const float mean = here ? a.mean[r * a.G + u.g] : 0.0f, rstd = here ? a.rstd[r * a.G + u.g] : 0.0f;
        float2 n[K][P], e[K][P], s1 = both(0.0f), s2 = both(0.0f);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) {
                n[k][i] = mul2(mul2(add2(U::pair(px[k], i), both(-mean)), both(rstd)), u.there(k, i));
                float2 d = U::pair(pg[k], i);      // 0 where there is no channel
                if (a.act) d = mul2(d, activate_slope2(fma2(n[k][i], w[k][i], b[k][i]), a.act));
                dw[k][i] = fma2(d, n[k][i], dw[k][i]);
                db[k][i] = add2(db[k][i], d);
                e[k][i] = mul2(d, w[k][i]);
                s1 = add2(s1, e[k][i]);
                s2 = fma2(e[k][i], n[k][i], s2);
            }
        const float u1 = lane_sum<L>(s1.x + s1.y) * inv, u2 = lane_sum<L>(s2.x + s2.y) * inv;
        if (!here) continue;
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int i = 0; i < P; ++i) e[k][i] = mul2(both(rstd), fma2(n[k][i], both(-u2), add2(e[k][i], both(-u1))));
        u.store(static_cast<T *>(a.dx), r, a.C, e);
    }
    if (!u.alive) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < P; ++i)
#pragma unroll
            for (int h = 0; h < (V > 1 ? 2 : 1); ++h) {
                const int c = u.channel(k) + 2 * i + h;
                if (c >= u.per) continue;
                a.part[(u.first * 2 + 0) * a.C + u.g * u.per + c] = h ? dw[k][i].y : dw[k][i].x;
                a.part[(u.first * 2 + 1) * a.C + u.g * u.per + c] = h ? db[k][i].y : db[k][i].x;
            }
}

// ---------------------------------------------------------------------------------------------- maps

// A block's sample, positions and channels; its threads as columns of packs times rows of positions.
struct Spot {
    int64_t r, p0, p1;
    int g0, groups, c0, chans, chunk, packs, px, ty, rows;
};
template <int V>
__device__ __forceinline__ Spot place(const NormArgs &a)
{
    Spot s;
    int64_t i = blockIdx.x;
    s.chunk = (int)(i % a.chunks);      // neighbours: the blocks of a cluster
    i /= a.chunks;
    const int sl = (int)(i % a.slabs);
    s.r = i / a.slabs;
    s.g0 = sl * a.slab;
    s.groups = s.g0 + a.slab < a.G ? a.slab : a.G - s.g0;
    const int per = a.C / a.G;
    s.c0 = s.g0 * per;
    s.chans = s.groups * per;
    s.packs = (s.chans + V - 1) / V;
    const int wide = s.packs < NT ? s.packs : NT;
    s.px = threadIdx.x % wide;
    s.ty = threadIdx.x / wide;
    s.rows = NT / wide;
    if (s.ty >= s.rows) s.packs = 0;      // threads left over
    s.p0 = s.chunk * a.chunk;
    s.p1 = s.p0 + a.chunk < a.S ? s.p0 + a.chunk : a.S;
    return s;
}
__device__ __forceinline__ int columns(const Spot &s, int V) { const int p = (s.chans + V - 1) / V; return p < NT ? p : NT; }

__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Calls f(pack of x, pack of dy, position) for the positions of a thread, AHEAD of them on their way.
template <typename T, int V, bool VEC, bool TWO, typename F>
__device__ __forceinline__ void walk(const NormArgs &a, const Spot &s, int p, const F &f)
{
    using R = RawPack<T, V, VEC>;
    constexpr int AHEAD = TWO ? 2 : 4;
    const int left = s.chans - p * V;
    const T *x = static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V;
    const T *g = TWO ? static_cast<const T *>(a.dy.p) + s.r * a.dy.sb + s.c0 + p * V : nullptr;
    R px[AHEAD], pg[AHEAD];
    auto fetch = [&](int i, int64_t q) {
        px[i].load(x + q * a.x.st, q < s.p1 ? left : 0);
        if (TWO) pg[i].load(g + q * a.dy.st, q < s.p1 ? left : 0);
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) fetch(i, s.p0 + s.ty + (int64_t)i * s.rows);
    for (int64_t q = s.p0 + s.ty; q < s.p1; q += (int64_t)AHEAD * s.rows) {
#pragma unroll
        for (int i = 0; i < AHEAD; ++i) {
            const int64_t at = q + (int64_t)i * s.rows;
            const R cx = px[i], cg = pg[i];
            fetch(i, at + (int64_t)AHEAD * s.rows);
            if (at < s.p1) f(cx, cg, at);
        }
    }
}
template <typename T, int V, bool VEC>
__device__ __forceinline__ float2 pair_of(const RawPack<T, V, VEC> &r, int i)
{
    if constexpr (V > 1) return r.pair(i);
    else return make_float2(r.get(0), 0.0f);
}

// Moments of every group over the block's positions, in s_m (see map_smem), passed to out(group of the block, moments).
// A thread takes the moments of its channels about their first value, so that a large common offset costs no digits.
template <typename T, int V, bool VEC, typename Out>
__device__ __forceinline__ void block_moments(const NormArgs &a, const Spot &s, float2 *s_m, const Out &out)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        float2 k[P], sum[P], sq[P];
        int count = 0;
        const int left = s.chans - p * V;
#pragma unroll
        for (int i = 0; i < P; ++i) k[i] = sum[i] = sq[i] = both(0.0f);
        if (s.p0 + s.ty < s.p1) {
            RawPack<T, V, VEC> head;
            head.load(static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V + (s.p0 + s.ty) * a.x.st, left);
#pragma unroll
            for (int i = 0; i < P; ++i) k[i] = pair_of(head, i);
        }
        walk<T, V, VEC, false>(a, s, p, [&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &, int64_t) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 f = pair_of(x, i), d = make_float2(f.x - k[i].x, f.y - k[i].y);
                sum[i] = add2(sum[i], d);
                sq[i] = fma2(d, d, sq[i]);
            }
            ++count;
        });
        const float inv = count ? 1.0f / count : 0.0f;
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float2 *to = s_m + s.ty * s.chans + p * V + 2 * i;
            if (2 * i < left) to[0] = make_float2(fmaf(sum[i].x, inv, k[i].x), max_nan(sq[i].x - sum[i].x * sum[i].x * inv, 0.0f));
            if (V > 1 && 2 * i + 1 < left) to[1] = make_float2(fmaf(sum[i].y, inv, k[i].y), max_nan(sq[i].y - sum[i].y * sum[i].y * inv, 0.0f));
        }
    }
    __syncthreads();
    const int per = a.C / a.G, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t n = s.p1 - s.p0;
    for (int g = warp; g < s.groups; g += NT / 32) {
        Moments m = {0.f, 0.f, 0.f};
        int row = lane / per, c = lane % per;
        const int step_row = 32 / per, step_c = 32 % per;
        while (row < s.rows && row < n) {
            const float2 f = s_m[row * s.chans + g * per + c];
            m = merge(m, Moments{(float)((n - row + s.rows - 1) / s.rows), f.x, f.y});
            row += step_row;
            c += step_c;
            if (c >= per) {
                c -= per;
                ++row;
            }
        }
        m = merge_lanes(m);
        if (lane == 0) out(g, m);
    }
}

// y from x with the groups' mean and rstd in s_m.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void block_apply(const NormArgs &a, const Spot &s, const float2 *s_m)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    const int per = a.C / a.G;
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        const int left = s.chans - p * V;
        float2 mean[P], scale[P], shift[P];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = p * V + i;
            float m = 0.0f, sc = 0.0f, sh = 0.0f;
            if (c < s.chans) {
                const float2 f = s_m[c / per];
                m = f.x;
                sc = a.weight ? f.y * param<T>(a.weight, s.c0 + c, a.params_f32) : f.y;
                sh = a.bias ? param<T>(a.bias, s.c0 + c, a.params_f32) : 0.0f;
            }
            if (i % 2 == 0) { mean[i / 2] = both(-m); scale[i / 2] = both(sc); shift[i / 2] = both(sh); }
            else { mean[i / 2].y = -m; scale[i / 2].y = sc; shift[i / 2].y = sh; }
        }
        T *out = static_cast<T *>(a.y) + s.r * a.S * a.C + s.c0 + p * V;
        walk<T, V, VEC, false>(a, s, p, [&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &, int64_t q) {
            Pack<T, V> y;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 v = activate2(fma2(add2(pair_of(x, i), mean[i]), scale[i], shift[i]), a.act);
                y.v[2 * i] = from_f32<T>(v.x);
                if constexpr (V > 1) y.v[2 * i + 1] = from_f32<T>(v.y);
            }
            store_pack<VEC>(out + q * a.C, y, left);
        });
    }
}

// What the backward needs of a pack's channels: (x - mean) rstd = x rstd + centre would lose digits, so both are kept.
template <typename T, int V>
struct Channels {
    static constexpr int P = V > 1 ? V / 2 : 1;
    float2 mean[P], rstd[P], w[P], b[P];
    __device__ __forceinline__ Channels(const NormArgs &a, const Spot &s, int p)
    {
        const int per = a.C / a.G;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = p * V + i;
            const bool there = c < s.chans;
            const int64_t g = s.r * a.G + (there ? (s.c0 + c) / per : s.g0);
            const float m = -a.mean[g], r = a.rstd[g];
            const float wv = (there && a.weight) ? param<T>(a.weight, s.c0 + c, a.params_f32) : 1.0f;
            const float bv = (there && a.bias) ? param<T>(a.bias, s.c0 + c, a.params_f32) : 0.0f;
            if (i % 2 == 0) { mean[i / 2] = both(m); rstd[i / 2] = both(r); w[i / 2] = both(wv); b[i / 2] = both(bv); }
            else { mean[i / 2].y = m; rstd[i / 2].y = r; w[i / 2].y = wv; b[i / 2].y = bv; }
        }
    }
    __device__ __forceinline__ float2 normed(float2 x, int i) const { return mul2(add2(x, mean[i]), rstd[i]); }
    // gradient in front of the activation
    __device__ __forceinline__ float2 inner(float2 n, float2 up, int act, int i) const { return act ? mul2(up, activate_slope2(fma2(n, w[i], b[i]), act)) : up; }
};

// Per channel, over the block's positions: the sums of d n and of d (d: gradient in front of the activation, n: normed x),
// in s_c [2][channels] and in the block's row of a.part.  s_m: see map_smem.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void block_gradient_sums(const NormArgs &a, const Spot &s, float2 *s_m, float2 *s_c)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        const int left = s.chans - p * V;
        const Channels<T, V> h(a, s, p);
        float2 s1[P], s2[P];
#pragma unroll
        for (int i = 0; i < P; ++i) s1[i] = s2[i] = both(0.0f);
        walk<T, V, VEC, true>(a, s, p, [&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &g, int64_t) {
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 n = h.normed(pair_of(x, i), i), d = h.inner(n, pair_of(g, i), a.act, i);
                s1[i] = add2(s1[i], d);
                s2[i] = fma2(d, n, s2[i]);
            }
        });
#pragma unroll
        for (int i = 0; i < P; ++i) {
            float2 *to = s_m + s.ty * s.chans + p * V + 2 * i;
            if (2 * i < left) to[0] = make_float2(s1[i].x, s2[i].x);
            if (V > 1 && 2 * i + 1 < left) to[1] = make_float2(s1[i].y, s2[i].y);
        }
    }
    __syncthreads();
    float *out = a.part + (s.r * a.chunks + s.chunk) * 2 * a.C + s.c0;
    for (int c = threadIdx.x; c < s.chans; c += NT) {
        float2 t = both(0.0f);
        for (int k = 0; k < s.rows; ++k) t = add2(t, s_m[k * s.chans + c]);
        out[c] = t.y;
        out[a.C + c] = t.x;
        s_c[c] = t;
    }
    __syncthreads();
}

// Sums of a group from sums per channel: weighted, one warp per group.
template <typename T, typename Get, typename Out>
__device__ __forceinline__ void group_sums(const NormArgs &a, const Spot &s, const Get &get, const Out &out)
{
    const int per = a.C / a.G, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
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

// dx with the groups' two sums over their number of values in s_g.
template <typename T, int V, bool VEC>
__device__ __forceinline__ void block_gradient(const NormArgs &a, const Spot &s, const float2 *s_g)
{
    constexpr int P = V > 1 ? V / 2 : 1;
    const int per = a.C / a.G;
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        const int left = s.chans - p * V;
        const Channels<T, V> h(a, s, p);
        float2 u[P], v[P];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 f = s_g[p * V + i < s.chans ? (p * V + i) / per : 0];
            if (i % 2 == 0) { u[i / 2] = both(-f.x); v[i / 2] = both(-f.y); }
            else { u[i / 2].y = -f.x; v[i / 2].y = -f.y; }
        }
        T *out = static_cast<T *>(a.dx) + s.r * a.S * a.C + s.c0 + p * V;
        walk<T, V, VEC, true>(a, s, p, [&](const RawPack<T, V, VEC> &x, const RawPack<T, V, VEC> &g, int64_t q) {
            Pack<T, V> o;
#pragma unroll
            for (int i = 0; i < P; ++i) {
                const float2 n = h.normed(pair_of(x, i), i), d = h.inner(n, pair_of(g, i), a.act, i);
                const float2 e = mul2(h.rstd[i], fma2(n, v[i], fma2(d, h.w[i], u[i])));
                o.v[2 * i] = from_f32<T>(e.x);
                if constexpr (V > 1) o.v[2 * i + 1] = from_f32<T>(e.y);
            }
            store_pack<VEC>(out + q * a.C, o, left);
        });
    }
}

// Final mean and rstd of a group.
__device__ __forceinline__ void finish_group(const NormArgs &a, const Spot &s, float2 *s_m, int g, const Moments &m, bool write)
{
    const float rstd = 1.0f / sqrtf(m.m2 / m.n + a.eps);
    s_m[g] = make_float2(m.mean, rstd);
    if (write) {
        a.mean[s.r * a.G + s.g0 + g] = m.mean;
        a.rstd[s.r * a.G + s.g0 + g] = rstd;
    }
}

// ---- one cluster per sample (and slab of groups): a.chunks blocks, which is the cluster's size

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_cluster_forward_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // map_smem; behind it [groups] moments of the block
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const Spot s = place<V>(a);
    Moments *own = reinterpret_cast<Moments *>(s_m + a.smem);
    block_moments<T, V, VEC>(a, s, s_m, [&](int g, const Moments &m) { own[g] = m; });
    cluster.sync();
    for (int g = threadIdx.x; g < s.groups; g += NT) {
        Moments m = {0.f, 0.f, 0.f};
        for (int r = 0; r < a.chunks; ++r) m = merge(m, cluster.map_shared_rank(own, r)[g]);
        finish_group(a, s, s_m, g, m, s.chunk == 0);
    }
    cluster.sync();      // nobody reads another block's moments any more; s_m is written
    block_apply<T, V, VEC>(a, s, s_m);
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_cluster_backward_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // map_smem; [channels] sums; [groups] sums of the block
    namespace cg = cooperative_groups;
    const cg::cluster_group cluster = cg::this_cluster();
    const Spot s = place<V>(a);
    float2 *s_c = s_m + a.smem, *own = s_c + a.slab * (a.C / a.G);
    block_gradient_sums<T, V, VEC>(a, s, s_m, s_c);
    group_sums<T>(a, s, [&](int c) { return s_c[c]; }, [&](int g, float2 t) { own[g] = t; });
    cluster.sync();
    const float inv = 1.0f / ((float)a.S * (float)(a.C / a.G));
    for (int g = threadIdx.x; g < s.groups; g += NT) {
        float2 t = both(0.0f);
        for (int r = 0; r < a.chunks; ++r) t = add2(t, cluster.map_shared_rank(own, r)[g]);
        s_m[g] = mul2(t, both(inv));
    }
    cluster.sync();
    block_gradient<T, V, VEC>(a, s, s_m);
}

// ---- two kernels

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_stats_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];
    const Spot s = place<V>(a);
    block_moments<T, V, VEC>(a, s, s_m, [&](int g, const Moments &m) {
        float *out = a.part + ((s.r * a.chunks + s.chunk) * a.G + s.g0 + g) * 2;
        out[0] = m.mean;
        out[1] = m.m2;
    });
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_apply_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // [groups]
    const Spot s = place<V>(a);
    const int per = a.C / a.G, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int g = warp; g < s.groups; g += NT / 32) {
        Moments m = {0.f, 0.f, 0.f};
        for (int i = lane; i < a.chunks; i += 32) {
            const int64_t lo = i * a.chunk, hi = lo + a.chunk < a.S ? lo + a.chunk : a.S;
            const float *in = a.part + ((s.r * a.chunks + i) * a.G + s.g0 + g) * 2;
            m = merge(m, Moments{(float)((hi - lo) * per), in[0], in[1]});
        }
        m = merge_lanes(m);
        if (lane == 0) finish_group(a, s, s_m, g, m, s.chunk == 0);
    }
    __syncthreads();
    block_apply<T, V, VEC>(a, s, s_m);
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_backward_sums_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];
    const Spot s = place<V>(a);
    block_gradient_sums<T, V, VEC>(a, s, s_m, s_m + a.smem);
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT, 3) norm_backward_apply_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // [groups]
    const Spot s = place<V>(a);
    const float inv = 1.0f / ((float)a.S * (float)(a.C / a.G));
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
    block_gradient<T, V, VEC>(a, s, s_m);
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
    // tokens: half of the threads that the GPU holds; backward at least four samples each, which leave one partial sum
    int L, K;
    token_shape(per, V, &L, &K);
    int64_t strides = ceil_div(148 * 1024, (int64_t)G * L);
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

// Pairs of shared memory in front of what a map kernel keeps besides: one per thread row and channel (one per group at least).
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
    const unsigned grid = (unsigned)(a.R * a.chunks * a.slabs);
    a.smem = map_smem<V>(a);
    int smem = a.smem * (int)sizeof(float2);
    if (cluster) return launch_clusters(norm_cluster_forward_kernel<T, V, VEC>, a, grid, smem + a.slab * (int)sizeof(Moments), s);
    cudaError_t e = allow_smem(norm_stats_kernel<T, V, VEC>, smem);
    if (e != cudaSuccess) return e;
    norm_stats_kernel<T, V, VEC><<<grid, NT, smem, s>>>(a);
    norm_apply_kernel<T, V, VEC><<<grid, NT, a.slab * sizeof(float2), s>>>(a);
    return cudaGetLastError();
}
template <typename T, int V, bool VEC>
cudaError_t maps_backward(NormArgs a, bool cluster, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.R * a.chunks * a.slabs);
    a.smem = map_smem<V>(a);
    const int chans = a.slab * (a.C / a.G);
    const int smem = (a.smem + chans) * (int)sizeof(float2);
    if (cluster) return launch_clusters(norm_cluster_backward_kernel<T, V, VEC>, a, grid, smem + a.slab * (int)sizeof(float2), s);
    cudaError_t e = allow_smem(norm_backward_sums_kernel<T, V, VEC>, smem);
    if (e != cudaSuccess) return e;
    norm_backward_sums_kernel<T, V, VEC><<<grid, NT, smem, s>>>(a);
    norm_backward_apply_kernel<T, V, VEC><<<grid, NT, a.slab * sizeof(float2), s>>>(a);
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
