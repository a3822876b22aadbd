// Selective scan: the single step, the plan of the scan and its launchers (kernels: exb_selective_kernels.cuh).
#include "exb_selective.cuh"

namespace exb {

namespace {

// ---------------------------------------------------------------------------------------------- one token

// A thread takes four states of a channel in ITEMS batch items, `apart` of them between two: the rates are loaded once, and
// all states are on their way together (the state is what has to move).  The channel's first ITEMS lanes do the work that is
// not per state for one batch item each.  256 x 4096 x 16, bfloat16: 32.7 us, 4.4 TB/s of states and inputs (with one batch
// item per thread, and all lanes doing that work, 55 us); 1 x 1024 x 16: 2 us, the launch.
template <typename T, int L, int ITEMS, bool VEC>
__global__ void __launch_bounds__(256) sel_step_kernel(const SelStepArgs a, unsigned apart)
{
    const unsigned i = (blockIdx.x * 256u + threadIdx.x) / L;
    const int l = threadIdx.x % L, n0 = 4 * l, lane = threadIdx.x % 32;
    const unsigned b0 = i / (unsigned)a.M;
    const bool alive = b0 < apart;
    const int m = (int)(i - b0 * (unsigned)a.M), g = m / (a.M / a.G);
    RawPack<float, 4, VEC> vh[ITEMS], va;
    RawPack<T, 4, VEC> vb[ITEMS], vc[ITEMS];
    va.load(a.A + (int64_t)m * a.N + n0, alive ? a.N - n0 : 0);
    float *h0 = a.h + b0 * a.sh + (int64_t)m * a.N + n0;
    const int64_t hs = apart * a.sh, bs = apart * a.Bm.sb, cs = apart * a.Cm.sb;
    const T *bp = static_cast<const T *>(a.Bm.p) + b0 * a.Bm.sb + g * a.N + n0, *cp = static_cast<const T *>(a.Cm.p) + b0 * a.Cm.sb + g * a.N + n0;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int have = alive && b0 + k * apart < a.B ? a.N - n0 : 0;
        vh[k].load(h0 + k * hs, have);
        vb[k].load(bp + k * bs, have);
        vc[k].load(cp + k * cs, have);
    }
    const int64_t own = b0 + (int64_t)(l < ITEMS ? l : 0) * apart;      // batch item that this lane prepares
    const int mine = alive && own < a.B;
    RawPack<T, 1, false> vx, vd, vz;
    vx.load(static_cast<const T *>(a.x.p) + own * a.x.sb + m, mine);
    vd.load(static_cast<const T *>(a.dt.p) + own * a.dt.sb + m, mine);
    vz.load(static_cast<const T *>(a.z.p) + own * a.z.sb + m, mine && a.z.p);
    const float bias = alive && a.dt_bias ? a.dt_bias[m] : 0.0f, skip = alive && a.D ? a.D[m] : 0.0f;
    const float x = vx.get(0);
    float dt = vd.get(0) + bias;
    if (a.softplus) dt = softplus_f(dt);
    const float u = dt * x;
    float y[ITEMS], A2[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) A2[j] = finite_rate(va.get(j)) * LOG2E;
#pragma unroll
    for (int k = 0; k < ITEMS; ++k) {
        const int from = (lane & ~(L - 1)) + (ITEMS > 1 ? k : 0);
        const float d = ITEMS > 1 ? __shfl_sync(0xffffffffu, dt, from) : dt, w = ITEMS > 1 ? __shfl_sync(0xffffffffu, u, from) : u;
        y[k] = 0.0f;
        Pack<float, 4> h;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            h.v[j] = fmaf(exp2_fast(fmaf(d, A2[j], decay_lift(d * A2[j]))), vh[k].get(j), w * vb[k].get(j));
            y[k] = fmaf(vc[k].get(j), h.v[j], y[k]);
        }
        store_pack<VEC>(h0 + k * hs, h, alive && b0 + k * apart < a.B ? a.N - n0 : 0);
    }
    // the lanes of rank k L/ITEMS end up with batch item k, which the lane l = k holds the inputs of
    reduce_scatter<ITEMS, L, 1>(y, lane);
    float sum = y[0];
    if (ITEMS > 1 && L > ITEMS) sum = __shfl_sync(0xffffffffu, sum, (lane & ~(L - 1)) + (l < ITEMS ? l : 0) * (L / ITEMS));
    if (mine && l < ITEMS) {
        float out = fmaf(skip, x, sum);
        if (a.z.p) out *= silu_f(vz.get(0));
        static_cast<T *>(a.y)[own * a.M + m] = from_f32<T>(out);
    }
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

template <typename T, int L, bool VEC>
cudaError_t step_typed(const SelStepArgs &a, cudaStream_t s)
{
    // Several batch items per thread once that leaves two blocks for every SM.
    constexpr int ITEMS = L < 4 ? L : 4;
    const bool many = ceil_div(a.B, ITEMS) * a.M * L >= 2 * 148 * 256;
    const int64_t apart = many ? ceil_div(a.B, ITEMS) : a.B;
    const unsigned grid = (unsigned)ceil_div(apart * a.M * L, 256);
    if (many) sel_step_kernel<T, L, ITEMS, VEC><<<grid, 256, 0, s>>>(a, (unsigned)apart);
    else sel_step_kernel<T, L, 1, VEC><<<grid, 256, 0, s>>>(a, (unsigned)apart);
    return cudaGetLastError();
}

template <typename T, bool VEC>
cudaError_t step_lanes(const SelStepArgs &a, cudaStream_t s)
{
    switch (sel_lanes(a.N)) {
    case 1: return step_typed<T, 1, VEC>(a, s);
    case 2: return step_typed<T, 2, VEC>(a, s);
    case 4: return step_typed<T, 4, VEC>(a, s);
    case 8: return step_typed<T, 8, VEC>(a, s);
    case 16: return step_typed<T, 16, VEC>(a, s);
    default: return step_typed<T, 32, VEC>(a, s);
    }
}

template <typename T>
cudaError_t step_dispatch(const SelStepArgs &a, cudaStream_t s)
{
    const bool vec = a.N % 4 == 0 && pack_aligned<T>(a.Bm) && pack_aligned<T>(a.Cm) && a.sh % 4 == 0 &&
                     ((reinterpret_cast<uintptr_t>(a.h) | reinterpret_cast<uintptr_t>(a.A)) & 15) == 0;
    return vec ? step_lanes<T, true>(a, s) : step_lanes<T, false>(a, s);
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
    p.NP = sel_padded(N);
    p.CC = 1024 / p.NP;
    p.tiles = (int)ceil_div(M / G, p.CC);
    const int64_t blocks = B * G * p.tiles, unit = 16;
    // Splitting the time axis costs a pass over the states of all pieces (half of the forward pass, a quarter of the
    // backward one), so it has to bring more than 1.5 times the blocks, for two on each of 148 SMs.  1 x 4096 steps of 64
    // channels x 16 states per block, prompt and training, whole against split: 64 blocks 311 and 1206 us against 231 and
    // 755; 96 blocks 311 and 1209 against 311 and 1005; 112 blocks 310 and 1211 against 392 and 1409.  At 16 blocks
    // (1 x 16384 x 1024 x 16, prompt) 9, 18, 27 and 37 pieces take 282, 221, 236 and 226 us.  A piece is no shorter than 32
    // steps and than the number of pieces that its block has to fold.
    int64_t want = blocks >= 96 ? 1 : 296 / blocks;
    while (want > 1 && (T / want < 32 || T / want < want)) --want;
    p.seg = ceil_div(ceil_div(T, want), unit) * unit;
    p.segments = (int)ceil_div(T, p.seg);
    // One block per SM: two states per lane and twice the warps (4 x 2048 x 2048 x 16, training: 622 us against 699).  More blocks than
    // SMs: four, and two blocks on an SM (288 blocks: 212 us against 277).
    p.S = (blocks * p.segments > 148 || p.NP > 64) ? 4 : 2;
    p.L = p.NP / p.S;
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
    if (dtype == EXB_F32) return selective_forward_typed<float>(a, p, stream);
    if (dtype == EXB_BF16) return selective_forward_typed<__nv_bfloat16>(a, p, stream);
    return selective_forward_typed<__half>(a, p, stream);
}

cudaError_t launch_selective_backward(SelArgs a, int dtype, void *dB, void *dC, float *dA, float *dD, float *dbias, void *ws,
                                      cudaStream_t stream)
{
    const SelPlan p = sel_plan(a.B, a.T, a.M, a.N, a.G, true);
    place(a, p, ws);
    cudaError_t e;
    if (dtype == EXB_F32) e = selective_backward_typed<float>(a, p, dB, dC, stream);
    else if (dtype == EXB_BF16) e = selective_backward_typed<__nv_bfloat16>(a, p, dB, dC, stream);
    else e = selective_backward_typed<__half>(a, p, dB, dC, stream);
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
