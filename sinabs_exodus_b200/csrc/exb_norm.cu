// Group norm with an activation on channels-last tensors (sample, position, channel):
//
//   y = act((x - mean) rstd w + b),  mean and variance over the positions and the channels of a group of one sample.
//
// Two mappings.  One position per sample (tokens): a few lanes hold a group in registers.  Maps: a block takes a run of
// positions of a sample and all channels of some groups; statistics first, then the map is read again.
#include "exb_norm.cuh"

namespace exb {

namespace {

constexpr int NT = 256;

template <typename T>
__device__ __forceinline__ float param(const void *p, int64_t i, int f32)
{
    return f32 ? static_cast<const float *>(p)[i] : to_f32(static_cast<const T *>(p)[i]);
}

__device__ __forceinline__ float activate(float v, int act)
{
    if (act == EXB_ACT_SILU) return silu_f(v);
    if (act == EXB_ACT_RELU) return v > 0.0f ? v : (v != v ? v : 0.0f);
    return v;
}
__device__ __forceinline__ float activate_slope(float v, int act)
{
    if (act == EXB_ACT_SILU) {
        const float s = sigmoid_f(v);
        return s * (1.0f + v * (1.0f - s));
    }
    if (act == EXB_ACT_RELU) return v > 0.0f ? 1.0f : 0.0f;
    return 1.0f;
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

// L lanes hold the channels of a group, K packs of V each; lane l has packs l, l + L, ...
template <typename T, int V, int L, int K, bool VEC>
__global__ void __launch_bounds__(NT) norm_token_forward_kernel(const NormArgs a)
{
    const int64_t u = (blockIdx.x * (int64_t)NT + threadIdx.x) / L;
    const int l = threadIdx.x % L, per = a.C / a.G;
    const bool alive = u < a.R * a.G;
    const int64_t r = alive ? u / a.G : 0;
    const int g = alive ? (int)(u % a.G) : 0;
    float v[K][V], sum = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * L + l) * V;
        Pack<T, V> p;
        load_pack<VEC>(p, static_cast<const T *>(a.x.p) + r * a.x.sb + g * per + c, alive ? per - c : 0);
#pragma unroll
        for (int i = 0; i < V; ++i) {
            v[k][i] = to_f32(p.v[i]);
            sum += v[k][i];
        }
    }
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, m);
    const float mean = sum / per;
    float sq = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float d = v[k][i] - mean;
            if ((k * L + l) * V + i < per) sq = fmaf(d, d, sq);
        }
#pragma unroll
    for (int m = L / 2; m >= 1; m >>= 1) sq += __shfl_xor_sync(0xffffffffu, sq, m);
    if (!alive) return;
    const float rstd = 1.0f / sqrtf(sq / per + a.eps);
    if (l == 0) {
        a.mean[r * a.G + g] = mean;
        a.rstd[r * a.G + g] = rstd;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int c = (k * L + l) * V, ch = g * per + c;
        if (c >= per) continue;
        Pack<T, V> p;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float y = (v[k][i] - mean) * rstd;
            if (c + i < per) {
                if (a.weight) y *= param<T>(a.weight, ch + i, a.params_f32);
                if (a.bias) y += param<T>(a.bias, ch + i, a.params_f32);
            }
            p.v[i] = from_f32<T>(activate(y, a.act));
        }
        store_pack<VEC>(static_cast<T *>(a.y) + r * a.C + ch, p, per - c);
    }
}

// A lane group keeps to its group and takes every `strides`-th sample, so that the gradients of weight and bias add up
// in registers.
template <typename T, int V, int L, int K, bool VEC>
__global__ void __launch_bounds__(NT) norm_token_backward_kernel(const NormArgs a, int64_t strides)
{
    const int64_t q = (blockIdx.x * (int64_t)NT + threadIdx.x) / L;
    const int l = threadIdx.x % L, per = a.C / a.G, g = (int)(q % a.G);
    const int64_t first = q / a.G;
    const bool alive = first < strides;
    float w[K][V], b[K][V], dw[K][V], db[K][V];
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (k * L + l) * V + i;
            w[k][i] = (c < per && a.weight) ? param<T>(a.weight, g * per + c, a.params_f32) : 1.0f;
            b[k][i] = (c < per && a.bias) ? param<T>(a.bias, g * per + c, a.params_f32) : 0.0f;
            dw[k][i] = db[k][i] = 0.0f;
        }
    const int64_t rounds = (a.R + strides - 1) / strides;      // the same for every lane of the warp
    for (int64_t j = 0; j < rounds; ++j) {
        const int64_t r = first + j * strides;
        const bool here = alive && r < a.R;
        const float mean = here ? a.mean[r * a.G + g] : 0.0f, rstd = here ? a.rstd[r * a.G + g] : 0.0f;
        float n[K][V], e[K][V], s1 = 0.0f, s2 = 0.0f;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * L + l) * V;
            Pack<T, V> px, pg;
            load_pack<VEC>(px, static_cast<const T *>(a.x.p) + r * a.x.sb + g * per + c, here ? per - c : 0);
            load_pack<VEC>(pg, static_cast<const T *>(a.dy.p) + r * a.dy.sb + g * per + c, here ? per - c : 0);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                n[k][i] = (to_f32(px.v[i]) - mean) * rstd;
                float d = to_f32(pg.v[i]);
                if (a.act) d *= activate_slope(fmaf(n[k][i], w[k][i], b[k][i]), a.act);
                if (!here || c + i >= per) d = n[k][i] = 0.0f;
                dw[k][i] = fmaf(d, n[k][i], dw[k][i]);
                db[k][i] += d;
                e[k][i] = d * w[k][i];
                s1 += e[k][i];
                s2 = fmaf(e[k][i], n[k][i], s2);
            }
        }
#pragma unroll
        for (int m = L / 2; m >= 1; m >>= 1) {
            s1 += __shfl_xor_sync(0xffffffffu, s1, m);
            s2 += __shfl_xor_sync(0xffffffffu, s2, m);
        }
        if (!here) continue;
        s1 /= per;
        s2 /= per;
#pragma unroll
        for (int k = 0; k < K; ++k) {
            const int c = (k * L + l) * V;
            if (c >= per) continue;
            Pack<T, V> p;
#pragma unroll
            for (int i = 0; i < V; ++i) p.v[i] = from_f32<T>(rstd * (e[k][i] - s1 - n[k][i] * s2));
            store_pack<VEC>(static_cast<T *>(a.dx) + r * a.C + g * per + c, p, per - c);
        }
    }
    if (!alive) return;
#pragma unroll
    for (int k = 0; k < K; ++k)
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = (k * L + l) * V + i;
            if (c >= per) continue;
            a.part[(first * 2 + 0) * a.C + g * per + c] = dw[k][i];
            a.part[(first * 2 + 1) * a.C + g * per + c] = db[k][i];
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
    const int sl = (int)(i % a.slabs);
    i /= a.slabs;
    s.chunk = (int)(i % a.chunks);
    s.r = i / a.chunks;
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

// Sums over a group of values that lie one per channel in shared memory; a warp per group.
__device__ __forceinline__ float warp_sum(float v)
{
#pragma unroll
    for (int m = 16; m >= 1; m >>= 1) v += __shfl_xor_sync(0xffffffffu, v, m);
    return v;
}

// Mean and squared distances of every group over the block's positions.  A thread takes the moments of its channels
// about their first value, so that a large common offset costs no digits.
template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT) norm_stats_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // [rows][channels]: mean, squared distances
    const Spot s = place<V>(a);
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        float k[V], sum[V], sq[V];
        int count = 0;
        const int left = s.chans - p * V;
        const T *base = static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V;
#pragma unroll
        for (int i = 0; i < V; ++i) k[i] = sum[i] = sq[i] = 0.0f;
#pragma unroll 4
        for (int64_t q = s.p0 + s.ty; q < s.p1; q += s.rows) {
            Pack<T, V> v;
            load_pack<VEC>(v, base + q * a.x.st, left);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float f = to_f32(v.v[i]);
                if (count == 0) k[i] = f;
                const float d = f - k[i];
                sum[i] += d;
                sq[i] = fmaf(d, d, sq[i]);
            }
            ++count;
        }
        const float inv = count ? 1.0f / count : 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) s_m[s.ty * s.chans + p * V + i] = make_float2(fmaf(sum[i], inv, k[i]), fmaxf(sq[i] - sum[i] * sum[i] * inv, 0.0f));
    }
    __syncthreads();
    const int per = a.C / a.G, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int64_t n = s.p1 - s.p0;
    for (int g = warp; g < s.groups; g += NT / 32) {
        Moments m = {0.f, 0.f, 0.f};
        for (int i = lane; i < s.rows * per; i += 32) {
            const int row = i / per;
            if (row >= n) break;
            const float2 f = s_m[row * s.chans + g * per + i % per];
            m = merge(m, Moments{(float)((n - row + s.rows - 1) / s.rows), f.x, f.y});
        }
        m = merge_lanes(m);
        if (lane == 0) {
            float *out = a.part + ((s.r * a.chunks + s.chunk) * a.G + s.g0 + g) * 2;
            out[0] = m.mean;
            out[1] = m.m2;
        }
    }
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT) norm_apply_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // [groups]: mean, rstd
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
        if (lane == 0) {
            const float rstd = 1.0f / sqrtf(m.m2 / m.n + a.eps);
            s_m[g] = make_float2(m.mean, rstd);
            if (s.chunk == 0) {
                a.mean[s.r * a.G + s.g0 + g] = m.mean;
                a.rstd[s.r * a.G + s.g0 + g] = rstd;
            }
        }
    }
    __syncthreads();
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        const int left = s.chans - p * V;
        float mean[V], scale[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const int c = p * V + i;
            mean[i] = scale[i] = shift[i] = 0.0f;
            if (c < s.chans) {
                const float2 m = s_m[c / per];
                mean[i] = m.x;
                scale[i] = a.weight ? m.y * param<T>(a.weight, s.c0 + c, a.params_f32) : m.y;
                shift[i] = a.bias ? param<T>(a.bias, s.c0 + c, a.params_f32) : 0.0f;
            }
        }
        const T *base = static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V;
        T *out = static_cast<T *>(a.y) + s.r * a.S * a.C + s.c0 + p * V;
#pragma unroll 4
        for (int64_t q = s.p0 + s.ty; q < s.p1; q += s.rows) {
            Pack<T, V> v;
            load_pack<VEC>(v, base + q * a.x.st, left);
#pragma unroll
            for (int i = 0; i < V; ++i) v.v[i] = from_f32<T>(activate(fmaf(to_f32(v.v[i]) - mean[i], scale[i], shift[i]), a.act));
            store_pack<VEC>(out + q * a.C, v, left);
        }
    }
}

// What the backward needs of a channel.
template <int V>
struct Channel {
    float mean[V], rstd[V], w[V], b[V];
};
template <typename T, int V>
__device__ __forceinline__ void load_channels(Channel<V> &h, const NormArgs &a, const Spot &s, int p)
{
    const int per = a.C / a.G;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const int c = p * V + i;
        const bool there = c < s.chans;
        const int g = there ? (s.c0 + c) / per : s.g0;
        h.mean[i] = a.mean[s.r * a.G + g];
        h.rstd[i] = a.rstd[s.r * a.G + g];
        h.w[i] = (there && a.weight) ? param<T>(a.weight, s.c0 + c, a.params_f32) : 1.0f;
        h.b[i] = (there && a.bias) ? param<T>(a.bias, s.c0 + c, a.params_f32) : 0.0f;
    }
}

// Per channel, over the block's positions: the sums of d and of d * (x - mean) rstd, d being the gradient in front of
// the activation.
template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT) norm_backward_sums_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // [rows][channels]
    const Spot s = place<V>(a);
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        const int left = s.chans - p * V;
        Channel<V> h;
        load_channels<T, V>(h, a, s, p);
        float s1[V], s2[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.0f;
        const T *xb = static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V;
        const T *gb = static_cast<const T *>(a.dy.p) + s.r * a.dy.sb + s.c0 + p * V;
#pragma unroll 2
        for (int64_t q = s.p0 + s.ty; q < s.p1; q += s.rows) {
            Pack<T, V> vx, vg;
            load_pack<VEC>(vx, xb + q * a.x.st, left);
            load_pack<VEC>(vg, gb + q * a.dy.st, left);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float n = (to_f32(vx.v[i]) - h.mean[i]) * h.rstd[i];
                float d = to_f32(vg.v[i]);
                if (a.act) d *= activate_slope(fmaf(n, h.w[i], h.b[i]), a.act);
                s1[i] += d;
                s2[i] = fmaf(d, n, s2[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < left) s_m[s.ty * s.chans + p * V + i] = make_float2(s1[i], s2[i]);
    }
    __syncthreads();
    float *out = a.part + (s.r * a.chunks + s.chunk) * 2 * a.C + s.c0;
    for (int c = threadIdx.x; c < s.chans; c += NT) {
        float u = 0.0f, v = 0.0f;
        for (int k = 0; k < s.rows; ++k) {
            const float2 f = s_m[k * s.chans + c];
            u += f.x;
            v += f.y;
        }
        out[c] = v;
        out[a.C + c] = u;
    }
}

template <typename T, int V, bool VEC>
__global__ void __launch_bounds__(NT) norm_backward_apply_kernel(const NormArgs a)
{
    extern __shared__ float2 s_m[];      // [groups]: the two sums of the group over its number of values
    const Spot s = place<V>(a);
    const int per = a.C / a.G, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    for (int g = warp; g < s.groups; g += NT / 32) {
        float u = 0.0f, v = 0.0f;
        for (int i = lane; i < per; i += 32) {
            const int c = s.c0 + g * per + i;
            float cu = 0.0f, cv = 0.0f;
            for (int k = 0; k < a.chunks; ++k) {
                const float *in = a.part + (s.r * a.chunks + k) * 2 * a.C + c;
                cv += in[0];
                cu += in[a.C];
            }
            const float w = a.weight ? param<T>(a.weight, c, a.params_f32) : 1.0f;
            u = fmaf(w, cu, u);
            v = fmaf(w, cv, v);
        }
        u = warp_sum(u);
        v = warp_sum(v);
        const float n = (float)(a.S * per);
        if (lane == 0) s_m[g] = make_float2(u / n, v / n);
    }
    __syncthreads();
    for (int p = s.px; p < s.packs; p += columns(s, V)) {
        const int left = s.chans - p * V;
        Channel<V> h;
        load_channels<T, V>(h, a, s, p);
        float u[V], v[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 f = s_m[p * V + i < s.chans ? (p * V + i) / per : 0];
            u[i] = f.x;
            v[i] = f.y;
        }
        const T *xb = static_cast<const T *>(a.x.p) + s.r * a.x.sb + s.c0 + p * V;
        const T *gb = static_cast<const T *>(a.dy.p) + s.r * a.dy.sb + s.c0 + p * V;
        T *out = static_cast<T *>(a.dx) + s.r * a.S * a.C + s.c0 + p * V;
#pragma unroll 2
        for (int64_t q = s.p0 + s.ty; q < s.p1; q += s.rows) {
            Pack<T, V> vx, vg;
            load_pack<VEC>(vx, xb + q * a.x.st, left);
            load_pack<VEC>(vg, gb + q * a.dy.st, left);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float n = (to_f32(vx.v[i]) - h.mean[i]) * h.rstd[i];
                float d = to_f32(vg.v[i]);
                if (a.act) d *= activate_slope(fmaf(n, h.w[i], h.b[i]), a.act);
                vx.v[i] = from_f32<T>(h.rstd[i] * (fmaf(d, h.w[i], -u[i]) - n * v[i]));
            }
            store_pack<VEC>(out + q * a.C, vx, left);
        }
    }
}

// ---------------------------------------------------------------------------------------------- launchers

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

struct Plan {
    bool tokens, packs;
    int64_t strides;                 // tokens, backward: samples that are walked side by side
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

Plan plan_of(int64_t R, int64_t S, int C, int G, int dtype)
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
    // positions of a block: eight blocks per SM if the samples do not give them
    int64_t chunks = ceil_div(8 * 148, R * p.slabs);
    const int64_t most = ceil_div(S, 32);
    if (chunks > most) chunks = most;
    if (chunks > 256) chunks = 256;
    p.chunk = ceil_div(S, chunks);
    p.chunks = (int)ceil_div(S, p.chunk);
    p.strides = ceil_div(8 * 148 * (NT / 32), G) < R ? ceil_div(8 * 148 * (NT / 32), G) : R;
    p.forward_bytes = p.tokens ? 0 : R * p.chunks * G * 2 * 4;
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
    cudaStream_t s;
    template <int V, int L, int K, bool VEC>
    cudaError_t run() const
    {
        norm_token_forward_kernel<T, V, L, K, VEC><<<(unsigned)ceil_div(a.R * a.G * L, NT), NT, 0, s>>>(a);
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

// Shared memory of the map kernels: one pair per thread row and channel, at least one per group.
template <int V>
int map_smem(const NormArgs &a)
{
    const int per = a.C / a.G, chans = a.slab * per, packs = (chans + V - 1) / V, wide = packs < NT ? packs : NT;
    return (NT / wide) * chans * (int)sizeof(float2);
}

template <typename K>
cudaError_t allow_smem(K kernel, int bytes)
{
    return bytes > 48 * 1024 ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) : cudaSuccess;
}

template <typename T, int V, bool VEC>
cudaError_t maps_forward(const NormArgs &a, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.R * a.chunks * a.slabs);
    const int smem = map_smem<V>(a);
    cudaError_t e = allow_smem(norm_stats_kernel<T, V, VEC>, smem);
    if (e != cudaSuccess) return e;
    norm_stats_kernel<T, V, VEC><<<grid, NT, smem, s>>>(a);
    norm_apply_kernel<T, V, VEC><<<grid, NT, a.slab * sizeof(float2), s>>>(a);
    return cudaGetLastError();
}
template <typename T, int V, bool VEC>
cudaError_t maps_backward(const NormArgs &a, cudaStream_t s)
{
    const unsigned grid = (unsigned)(a.R * a.chunks * a.slabs);
    const int smem = map_smem<V>(a);
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
        const TokenForward<T> f{a, s};
        return vec && per % V == 0 ? with_token_shape<T, V, true>(per, f) : with_token_shape<T, 1, false>(per, f);
    }
    return vec && p.packs ? maps_forward<T, V, true>(a, s) : maps_forward<T, 1, false>(a, s);
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
        e = vec && p.packs ? maps_backward<T, V, true>(a, s) : maps_backward<T, 1, false>(a, s);
    }
    if (e != cudaSuccess || (!dweight && !dbias)) return e;
    const int64_t rows = p.tokens ? p.strides : a.R * a.chunks;
    if (a.params_f32) launch_column_sum(PutParams<float>{(float *)dweight, (float *)dbias, a.C}, a.part, rows, 2 * (int64_t)a.C, s);
    else launch_column_sum(PutParams<T>{(T *)dweight, (T *)dbias, a.C}, a.part, rows, 2 * (int64_t)a.C, s);
    return cudaGetLastError();
}

Plan apply_plan(NormArgs &a, int dtype, void *ws)
{
    const Plan p = plan_of(a.R, a.S, a.C, a.G, dtype);
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
    const Plan p = plan_of(R, S, C, G, dtype);
    return backward ? p.backward_bytes : p.forward_bytes;
}

cudaError_t launch_norm_forward(NormArgs a, int dtype, void *ws, cudaStream_t stream)
{
    const Plan p = apply_plan(a, dtype, ws);
    if (dtype == EXB_F32) return forward_typed<float>(a, p, stream);
    if (dtype == EXB_BF16) return forward_typed<__nv_bfloat16>(a, p, stream);
    return forward_typed<__half>(a, p, stream);
}

cudaError_t launch_norm_backward(NormArgs a, int dtype, void *dweight, void *dbias, void *ws, cudaStream_t stream)
{
    const Plan p = apply_plan(a, dtype, ws);
    if (dtype == EXB_F32) return backward_typed<float>(a, p, dweight, dbias, stream);
    if (dtype == EXB_BF16) return backward_typed<__nv_bfloat16>(a, p, dweight, dbias, stream);
    return backward_typed<__half>(a, p, dweight, dbias, stream);
}

}  // namespace exb
