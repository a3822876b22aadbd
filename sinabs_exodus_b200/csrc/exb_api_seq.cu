// C-ABI front end of the sequence operators: selective scan, causal convolution, group norm.
// Argument validation, device selection, dispatch; nothing here allocates device memory or keeps state.
#include "exb_conv.cuh"
#include "exb_host.cuh"
#include "exb_norm.cuh"
#include "exb_selective.cuh"

namespace {

using exb::DeviceGuard;
using exb::fail;

int64_t element_size(int dtype) { return dtype == EXB_F32 ? 4 : 2; }

bool dtype_ok(int dtype) { return dtype == EXB_F32 || dtype == EXB_BF16 || dtype == EXB_F16; }

// A tensor is there, aligned to its element and walked forwards.
int check_rows(const char *who, const char *name, const exb_rows *r, int64_t es, bool required)
{
    if (!r || !r->data) return required ? fail(EXB_ERR_ARG, "%s: %s is required", who, name) : EXB_OK;
    if (reinterpret_cast<uintptr_t>(r->data) % es) return fail(EXB_ERR_ALIGN, "%s: %s is not aligned to its element size", who, name);
    if (r->stride_b < 0 || r->stride_t < 0) return fail(EXB_ERR_ARG, "%s: negative stride of %s", who, name);
    return EXB_OK;
}
int check_ptr(const char *who, const char *name, const void *p, int64_t es, bool required)
{
    if (!p) return required ? fail(EXB_ERR_ARG, "%s: %s is required", who, name) : EXB_OK;
    if (reinterpret_cast<uintptr_t>(p) % es) return fail(EXB_ERR_ALIGN, "%s: %s is not aligned to its element size", who, name);
    return EXB_OK;
}

// A dimension of size one has no stride (whatever the caller's says, it must not keep aligned rows from being seen as such).
exb::View view(const exb_rows *r, int64_t B, int64_t T)
{
    exb::View v;
    if (r) { v.p = r->data; v.sb = B > 1 ? r->stride_b : 0; v.st = T > 1 ? r->stride_t : 0; }
    return v;
}

constexpr int64_t GRID_MAX = 0x7fffffffll;

int check_scan_sizes(const char *who, int64_t B, int64_t T, int64_t M, int64_t N, int64_t G)
{
    if (B < 0 || T < 0 || M < 0) return fail(EXB_ERR_ARG, "%s: negative size (B=%lld T=%lld M=%lld)", who, (long long)B, (long long)T, (long long)M);
    if (N < 1 || N > EXB_SELECTIVE_MAX_STATES) return fail(EXB_ERR_ARG, "%s: 1 to %d states per channel, got %lld", who, EXB_SELECTIVE_MAX_STATES, (long long)N);
    if (G < 1 || M % G) return fail(EXB_ERR_ARG, "%s: the %lld groups must divide the %lld channels", who, (long long)G, (long long)M);
    if (M > 0x7fffffffll / 512 || (double)B * (double)T > 1.0e15) return fail(EXB_ERR_ARG, "%s: sizes too large", who);
    return EXB_OK;
}

// Blocks of the scan's kernels (every block has at least 8 channels, every piece of time at least 16 steps).
int check_scan_grid(const char *who, const exb::SelPlan &p, int64_t B, int64_t T, int64_t M, int64_t N, int64_t G)
{
    const double blocks = (double)B * G * p.tiles * p.segments, sums = (double)B * T * G * 2 * N / 256;
    if (blocks > GRID_MAX || sums > GRID_MAX) return fail(EXB_ERR_ARG, "%s: sizes too large for one launch", who);
    return EXB_OK;
}

#define EXB_TRY(x)                 \
    do {                           \
        const int st_ = (x);       \
        if (st_ != EXB_OK) return st_; \
    } while (0)

int launched(const char *who, cudaError_t e)
{
    return e == cudaSuccess ? EXB_OK : fail(EXB_ERR_LAUNCH, "%s: %s", who, cudaGetErrorString(e));
}

}  // namespace

extern "C" {

int64_t exb_selective_checkpoint_floats(int64_t B, int64_t T, int64_t M, int64_t N)
{
    if (B <= 0 || T <= 0 || M <= 0 || N < 1 || N > EXB_SELECTIVE_MAX_STATES) return 0;
    return B * ((T + EXB_SELECTIVE_CHECKPOINT - 1) / EXB_SELECTIVE_CHECKPOINT) * M * exb::sel_padded((int)N);
}

int64_t exb_selective_workspace_bytes(int64_t B, int64_t T, int64_t M, int64_t N, int64_t G, int backward)
{
    if (check_scan_sizes("exb_selective_workspace_bytes", B, T, M, N, G) != EXB_OK || B == 0 || T == 0 || M == 0) return 0;
    return exb::sel_plan(B, T, (int)M, (int)N, (int)G, backward != 0).bytes;
}

int exb_selective_forward(void *y, float *h_last, float *ckpt, const exb_rows *x, const exb_rows *dt, const float *A, const exb_rows *Bm,
                          const exb_rows *Cm, const float *D, const exb_rows *z, const float *dt_bias, const float *h0,
                          const int32_t *lengths, int softplus, void *workspace, int64_t workspace_bytes, int dtype, int64_t B, int64_t T,
                          int64_t M, int64_t N, int64_t G, int device, void *stream)
{
    const char *who = "exb_selective_forward";
    EXB_TRY(check_scan_sizes(who, B, T, M, N, G));
    if (!dtype_ok(dtype)) return fail(EXB_ERR_ARG, "%s: unknown element type %d", who, dtype);
    if (B == 0 || T == 0 || M == 0) return EXB_OK;
    const int64_t es = element_size(dtype);
    EXB_TRY(check_ptr(who, "y", y, es, true));
    EXB_TRY(check_ptr(who, "h_last", h_last, 4, true));
    EXB_TRY(check_ptr(who, "ckpt", ckpt, 16, false));
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_rows(who, "dt", dt, es, true));
    EXB_TRY(check_ptr(who, "A", A, 4, true));
    EXB_TRY(check_rows(who, "B", Bm, es, true));
    EXB_TRY(check_rows(who, "C", Cm, es, true));
    EXB_TRY(check_ptr(who, "D", D, 4, false));
    EXB_TRY(check_rows(who, "z", z, es, false));
    EXB_TRY(check_ptr(who, "dt_bias", dt_bias, 4, false));
    EXB_TRY(check_ptr(who, "h0", h0, 4, false));
    EXB_TRY(check_ptr(who, "lengths", lengths, 4, false));
    const exb::SelPlan p = exb::sel_plan(B, T, (int)M, (int)N, (int)G, false);
    EXB_TRY(check_scan_grid(who, p, B, T, M, N, G));
    if (p.bytes > 0 && (!workspace || workspace_bytes < p.bytes))
        return fail(EXB_ERR_ARG, "%s: needs %lld bytes of workspace, got %lld", who, (long long)p.bytes, (long long)(workspace ? workspace_bytes : 0));
    EXB_TRY(check_ptr(who, "workspace", workspace, 16, false));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::SelArgs a{};
    a.x = view(x, B, T); a.dt = view(dt, B, T); a.z = view(z, B, T); a.Bm = view(Bm, B, T); a.Cm = view(Cm, B, T);
    a.A = A; a.D = D; a.dt_bias = dt_bias; a.h0 = h0; a.lengths = lengths;
    a.B = B; a.T = T; a.M = (int)M; a.N = (int)N; a.G = (int)G; a.softplus = softplus;
    a.y = y; a.h_last = h_last; a.ckpt = ckpt;
    return launched(who, exb::launch_selective_forward(a, dtype, workspace, (cudaStream_t)stream));
}

int exb_selective_backward(void *dx, void *ddt, float *dA, void *dB, void *dC, float *dD, void *dz, float *ddt_bias, float *dh0,
                           const exb_rows *dy, const float *dh_last, const float *ckpt, const exb_rows *x, const exb_rows *dt,
                           const float *A, const exb_rows *Bm, const exb_rows *Cm, const float *D, const exb_rows *z,
                           const float *dt_bias, const int32_t *lengths, int softplus, void *workspace, int64_t workspace_bytes,
                           int dtype, int64_t B, int64_t T, int64_t M, int64_t N, int64_t G, int device, void *stream)
{
    const char *who = "exb_selective_backward";
    EXB_TRY(check_scan_sizes(who, B, T, M, N, G));
    if (!dtype_ok(dtype)) return fail(EXB_ERR_ARG, "%s: unknown element type %d", who, dtype);
    if (B == 0 || T == 0 || M == 0) return EXB_OK;
    const int64_t es = element_size(dtype);
    const bool gated = z && z->data;
    EXB_TRY(check_ptr(who, "dx", dx, es, true));
    EXB_TRY(check_ptr(who, "ddt", ddt, es, true));
    EXB_TRY(check_ptr(who, "dA", dA, 4, true));
    EXB_TRY(check_ptr(who, "dB", dB, es, true));
    EXB_TRY(check_ptr(who, "dC", dC, es, true));
    EXB_TRY(check_ptr(who, "dD", dD, 4, false));
    EXB_TRY(check_ptr(who, "dz", dz, es, gated));
    EXB_TRY(check_ptr(who, "ddt_bias", ddt_bias, 4, false));
    EXB_TRY(check_ptr(who, "dh0", dh0, 4, false));
    EXB_TRY(check_rows(who, "dy", dy, es, true));
    EXB_TRY(check_ptr(who, "dh_last", dh_last, 4, false));
    EXB_TRY(check_ptr(who, "ckpt", ckpt, 16, true));
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_rows(who, "dt", dt, es, true));
    EXB_TRY(check_ptr(who, "A", A, 4, true));
    EXB_TRY(check_rows(who, "B", Bm, es, true));
    EXB_TRY(check_rows(who, "C", Cm, es, true));
    EXB_TRY(check_ptr(who, "D", D, 4, false));
    EXB_TRY(check_rows(who, "z", z, es, false));
    EXB_TRY(check_ptr(who, "dt_bias", dt_bias, 4, false));
    EXB_TRY(check_ptr(who, "lengths", lengths, 4, false));
    const exb::SelPlan p = exb::sel_plan(B, T, (int)M, (int)N, (int)G, true);
    EXB_TRY(check_scan_grid(who, p, B, T, M, N, G));
    if (!workspace || workspace_bytes < p.bytes)
        return fail(EXB_ERR_ARG, "%s: needs %lld bytes of workspace, got %lld", who, (long long)p.bytes, (long long)(workspace ? workspace_bytes : 0));
    EXB_TRY(check_ptr(who, "workspace", workspace, 16, true));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::SelArgs a{};
    a.x = view(x, B, T); a.dt = view(dt, B, T); a.z = view(z, B, T); a.Bm = view(Bm, B, T); a.Cm = view(Cm, B, T); a.dy = view(dy, B, T);
    a.A = A; a.D = D; a.dt_bias = dt_bias; a.lengths = lengths; a.dh_last = dh_last;
    a.B = B; a.T = T; a.M = (int)M; a.N = (int)N; a.G = (int)G; a.softplus = softplus;
    a.ckpt = const_cast<float *>(ckpt);
    a.dx = dx; a.ddt = ddt; a.dz = dz; a.dh0 = dh0;
    return launched(who, exb::launch_selective_backward(a, dtype, dB, dC, dA, dD, ddt_bias, workspace, (cudaStream_t)stream));
}

int exb_selective_step(void *y, float *h, int64_t h_stride, const exb_rows *x, const exb_rows *dt, const float *A, const exb_rows *Bm,
                       const exb_rows *Cm, const float *D, const exb_rows *z, const float *dt_bias, int softplus, int dtype, int64_t B,
                       int64_t M, int64_t N, int64_t G, int device, void *stream)
{
    const char *who = "exb_selective_step";
    EXB_TRY(check_scan_sizes(who, B, 1, M, N, G));
    if (!dtype_ok(dtype)) return fail(EXB_ERR_ARG, "%s: unknown element type %d", who, dtype);
    if (B == 0 || M == 0) return EXB_OK;
    const int64_t es = element_size(dtype);
    EXB_TRY(check_ptr(who, "y", y, es, true));
    EXB_TRY(check_ptr(who, "h", h, 4, true));
    if (h_stride < M * N && B > 1) return fail(EXB_ERR_ARG, "%s: the batch items of h overlap", who);
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_rows(who, "dt", dt, es, true));
    EXB_TRY(check_ptr(who, "A", A, 4, true));
    EXB_TRY(check_rows(who, "B", Bm, es, true));
    EXB_TRY(check_rows(who, "C", Cm, es, true));
    EXB_TRY(check_ptr(who, "D", D, 4, false));
    EXB_TRY(check_rows(who, "z", z, es, false));
    EXB_TRY(check_ptr(who, "dt_bias", dt_bias, 4, false));
    if ((double)B * M * exb::sel_lanes((int)N) > 4.0e9)      // threads are counted in 32 bits
        return fail(EXB_ERR_ARG, "%s: sizes too large for one launch", who);
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::SelStepArgs a{};
    a.x = view(x, B, 1); a.dt = view(dt, B, 1); a.z = view(z, B, 1); a.Bm = view(Bm, B, 1); a.Cm = view(Cm, B, 1);
    a.A = A; a.D = D; a.dt_bias = dt_bias; a.h = h; a.sh = h_stride; a.y = y;
    a.B = B; a.M = (int)M; a.N = (int)N; a.G = (int)G; a.softplus = softplus;
    return launched(who, exb::launch_selective_step(a, dtype, (cudaStream_t)stream));
}

namespace {

int check_conv_sizes(const char *who, int64_t B, int64_t T, int64_t M, int64_t W, int dtype)
{
    if (B < 0 || T < 0 || M < 0) return fail(EXB_ERR_ARG, "%s: negative size (B=%lld T=%lld M=%lld)", who, (long long)B, (long long)T, (long long)M);
    if (W < 1 || W > exb::CONV_MAX_WIDTH) return fail(EXB_ERR_ARG, "%s: filters of 1 to %d steps, got %lld", who, exb::CONV_MAX_WIDTH, (long long)W);
    if (!dtype_ok(dtype)) return fail(EXB_ERR_ARG, "%s: unknown element type %d", who, dtype);
    // blocks of 32 or more channels and 16 or more steps
    if (M > 0x7fffffffll / 16 || (double)B * (double)(T / 16 + 1) * (double)(M / 32 + 1) > GRID_MAX)
        return fail(EXB_ERR_ARG, "%s: sizes too large for one launch", who);
    return EXB_OK;
}

}  // namespace

int64_t exb_causal_conv_workspace_bytes(int64_t B, int64_t T, int64_t M, int64_t W)
{
    if (check_conv_sizes("exb_causal_conv_workspace_bytes", B, T, M, W, EXB_F32) != EXB_OK || B == 0 || T == 0 || M == 0) return 0;
    return exb::conv_backward_workspace_bytes(B, T, (int)M, (int)W);
}

int exb_causal_conv_forward(void *y, void *last, const exb_rows *x, const void *weight, const void *bias, const void *state,
                            const int32_t *lengths, int activation, int params_f32, int dtype, int64_t B, int64_t T, int64_t M, int64_t W,
                            int device, void *stream)
{
    const char *who = "exb_causal_conv_forward";
    EXB_TRY(check_conv_sizes(who, B, T, M, W, dtype));
    if (activation != EXB_ACT_NONE && activation != EXB_ACT_SILU) return fail(EXB_ERR_ARG, "%s: unknown activation %d", who, activation);
    if (B == 0 || T == 0 || M == 0) return EXB_OK;
    const int64_t es = element_size(dtype), ps = params_f32 ? 4 : es;
    EXB_TRY(check_ptr(who, "y", y, es, true));
    EXB_TRY(check_ptr(who, "last", last, es, false));
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_ptr(who, "weight", weight, ps, true));
    EXB_TRY(check_ptr(who, "bias", bias, ps, false));
    EXB_TRY(check_ptr(who, "state", state, es, false));
    EXB_TRY(check_ptr(who, "lengths", lengths, 4, false));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::ConvArgs a{};
    a.x = view(x, B, T); a.weight = weight; a.bias = bias; a.state = state; a.lengths = lengths; a.y = y; a.last = last;
    a.B = B; a.T = T; a.M = (int)M; a.W = (int)W; a.silu = activation == EXB_ACT_SILU; a.params_f32 = params_f32 || dtype == EXB_F32;
    return launched(who, exb::launch_conv_forward(a, dtype, (cudaStream_t)stream));
}

int exb_causal_conv_backward(void *dx, void *dweight, void *dbias, void *dstate, const exb_rows *dy, const void *dlast, const exb_rows *x,
                             const void *weight, const void *bias, const void *state, const int32_t *lengths, int activation,
                             int params_f32, void *workspace, int64_t workspace_bytes, int dtype, int64_t B, int64_t T, int64_t M,
                             int64_t W, int device, void *stream)
{
    const char *who = "exb_causal_conv_backward";
    EXB_TRY(check_conv_sizes(who, B, T, M, W, dtype));
    if (activation != EXB_ACT_NONE && activation != EXB_ACT_SILU) return fail(EXB_ERR_ARG, "%s: unknown activation %d", who, activation);
    if (B == 0 || T == 0 || M == 0) return EXB_OK;
    const int64_t es = element_size(dtype), ps = params_f32 ? 4 : es;
    EXB_TRY(check_ptr(who, "dx", dx, es, true));
    EXB_TRY(check_ptr(who, "dweight", dweight, ps, true));
    EXB_TRY(check_ptr(who, "dbias", dbias, ps, false));
    EXB_TRY(check_ptr(who, "dstate", dstate, es, false));
    EXB_TRY(check_rows(who, "dy", dy, es, true));
    EXB_TRY(check_ptr(who, "dlast", dlast, es, false));
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_ptr(who, "weight", weight, ps, true));
    EXB_TRY(check_ptr(who, "bias", bias, ps, false));
    EXB_TRY(check_ptr(who, "state", state, es, false));
    EXB_TRY(check_ptr(who, "lengths", lengths, 4, false));
    const int64_t need = exb::conv_backward_workspace_bytes(B, T, (int)M, (int)W);
    if (!workspace || workspace_bytes < need)
        return fail(EXB_ERR_ARG, "%s: needs %lld bytes of workspace, got %lld", who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
    EXB_TRY(check_ptr(who, "workspace", workspace, 16, true));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::ConvArgs a{};
    a.x = view(x, B, T); a.dy = view(dy, B, T); a.weight = weight; a.bias = bias; a.state = state; a.lengths = lengths; a.dlast = dlast;
    a.dx = dx; a.dstate = dstate;
    a.B = B; a.T = T; a.M = (int)M; a.W = (int)W; a.silu = activation == EXB_ACT_SILU; a.params_f32 = params_f32 || dtype == EXB_F32;
    return launched(who, exb::launch_conv_backward(a, dtype, dweight, dbias, workspace, (cudaStream_t)stream));
}

int exb_causal_conv_step(void *y, void *state, int64_t state_stride, const exb_rows *x, const void *weight, const void *bias,
                         int activation, int params_f32, int dtype, int64_t B, int64_t M, int64_t W, int device, void *stream)
{
    const char *who = "exb_causal_conv_step";
    EXB_TRY(check_conv_sizes(who, B, 1, M, W, dtype));
    if (activation != EXB_ACT_NONE && activation != EXB_ACT_SILU) return fail(EXB_ERR_ARG, "%s: unknown activation %d", who, activation);
    if (B == 0 || M == 0) return EXB_OK;
    const int64_t es = element_size(dtype), ps = params_f32 ? 4 : es;
    EXB_TRY(check_ptr(who, "y", y, es, true));
    EXB_TRY(check_ptr(who, "state", state, es, W > 1));
    if (state_stride < (W - 1) * M && B > 1) return fail(EXB_ERR_ARG, "%s: the batch items of state overlap", who);
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_ptr(who, "weight", weight, ps, true));
    EXB_TRY(check_ptr(who, "bias", bias, ps, false));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::ConvStepArgs a{};
    a.x = view(x, B, 1); a.weight = weight; a.bias = bias; a.state = state; a.ss = state_stride; a.y = y;
    a.B = B; a.M = (int)M; a.W = (int)W; a.silu = activation == EXB_ACT_SILU; a.params_f32 = params_f32 || dtype == EXB_F32;
    return launched(who, exb::launch_conv_step(a, dtype, (cudaStream_t)stream));
}

namespace {

int check_norm_sizes(const char *who, int64_t R, int64_t S, int64_t C, int64_t G, int dtype)
{
    if (R < 0 || S < 0 || C < 0) return fail(EXB_ERR_ARG, "%s: negative size (R=%lld S=%lld C=%lld)", who, (long long)R, (long long)S, (long long)C);
    if (G < 1 || C % G) return fail(EXB_ERR_ARG, "%s: the %lld groups must divide the %lld channels", who, (long long)G, (long long)C);
    if (C / G > exb::NORM_MAX_GROUP) return fail(EXB_ERR_ARG, "%s: at most %d channels in a group, got %lld", who, exb::NORM_MAX_GROUP, (long long)(C / G));
    if (!dtype_ok(dtype)) return fail(EXB_ERR_ARG, "%s: unknown element type %d", who, dtype);
    // 32 lanes per sample and group at most, blocks of 256; a sample's positions are counted in int
    if (C > 0x7fffffffll / 4 || S > 0x7fffffffll - 1024 || (double)R * (double)G > GRID_MAX) return fail(EXB_ERR_ARG, "%s: sizes too large for one launch", who);
    return EXB_OK;
}

}  // namespace

int64_t exb_group_norm_workspace_bytes(int64_t R, int64_t S, int64_t C, int64_t G, int dtype, int backward)
{
    if (check_norm_sizes("exb_group_norm_workspace_bytes", R, S, C, G, dtype) != EXB_OK || R == 0 || S == 0 || C == 0) return 0;
    return exb::norm_workspace_bytes(R, S, (int)C, (int)G, dtype, backward != 0);
}

int exb_group_norm_forward(void *y, float *mean, float *rstd, const exb_rows *x, const void *weight, const void *bias, float eps,
                           int activation, int params_f32, void *workspace, int64_t workspace_bytes, int dtype, int64_t R, int64_t S,
                           int64_t C, int64_t G, int device, void *stream)
{
    const char *who = "exb_group_norm_forward";
    EXB_TRY(check_norm_sizes(who, R, S, C, G, dtype));
    if (activation < EXB_ACT_NONE || activation > EXB_ACT_RELU) return fail(EXB_ERR_ARG, "%s: unknown activation %d", who, activation);
    if (!(eps >= 0.0f)) return fail(EXB_ERR_ARG, "%s: eps must not be negative", who);
    if (R == 0 || S == 0 || C == 0) return EXB_OK;
    const int64_t es = element_size(dtype), ps = params_f32 ? 4 : es;
    EXB_TRY(check_ptr(who, "y", y, es, true));
    EXB_TRY(check_ptr(who, "mean", mean, 4, true));
    EXB_TRY(check_ptr(who, "rstd", rstd, 4, true));
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_ptr(who, "weight", weight, ps, false));
    EXB_TRY(check_ptr(who, "bias", bias, ps, false));
    const int64_t need = exb::norm_workspace_bytes(R, S, (int)C, (int)G, dtype, false);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(EXB_ERR_ARG, "%s: needs %lld bytes of workspace, got %lld", who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
    EXB_TRY(check_ptr(who, "workspace", workspace, 16, false));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::NormArgs a{};
    a.x = view(x, R, S); a.weight = weight; a.bias = bias; a.y = y; a.mean = mean; a.rstd = rstd;
    a.R = R; a.S = S; a.C = (int)C; a.G = (int)G; a.act = activation; a.params_f32 = params_f32 || dtype == EXB_F32; a.eps = eps;
    return launched(who, exb::launch_norm_forward(a, dtype, workspace, (cudaStream_t)stream));
}

int exb_group_norm_backward(void *dx, void *dweight, void *dbias, const exb_rows *dy, const exb_rows *x, const float *mean,
                            const float *rstd, const void *weight, const void *bias, int activation, int params_f32, void *workspace,
                            int64_t workspace_bytes, int dtype, int64_t R, int64_t S, int64_t C, int64_t G, int device, void *stream)
{
    const char *who = "exb_group_norm_backward";
    EXB_TRY(check_norm_sizes(who, R, S, C, G, dtype));
    if (activation < EXB_ACT_NONE || activation > EXB_ACT_RELU) return fail(EXB_ERR_ARG, "%s: unknown activation %d", who, activation);
    if (R == 0 || S == 0 || C == 0) return EXB_OK;
    const int64_t es = element_size(dtype), ps = params_f32 ? 4 : es;
    EXB_TRY(check_ptr(who, "dx", dx, es, true));
    EXB_TRY(check_ptr(who, "dweight", dweight, ps, false));
    EXB_TRY(check_ptr(who, "dbias", dbias, ps, false));
    EXB_TRY(check_rows(who, "dy", dy, es, true));
    EXB_TRY(check_rows(who, "x", x, es, true));
    EXB_TRY(check_ptr(who, "mean", mean, 4, true));
    EXB_TRY(check_ptr(who, "rstd", rstd, 4, true));
    EXB_TRY(check_ptr(who, "weight", weight, ps, false));
    EXB_TRY(check_ptr(who, "bias", bias, ps, false));
    const int64_t need = exb::norm_workspace_bytes(R, S, (int)C, (int)G, dtype, true);
    if (!workspace || workspace_bytes < need)
        return fail(EXB_ERR_ARG, "%s: needs %lld bytes of workspace, got %lld", who, (long long)need, (long long)(workspace ? workspace_bytes : 0));
    EXB_TRY(check_ptr(who, "workspace", workspace, 16, true));
    DeviceGuard guard(device);
    if (!guard.ok) return fail(EXB_ERR_DEVICE, "%s: cannot select device %d", who, device);
    exb::NormArgs a{};
    a.x = view(x, R, S); a.dy = view(dy, R, S); a.weight = weight; a.bias = bias; a.dx = dx; a.mean = const_cast<float *>(mean); a.rstd = const_cast<float *>(rstd);
    a.R = R; a.S = S; a.C = (int)C; a.G = (int)G; a.act = activation; a.params_f32 = params_f32 || dtype == EXB_F32;
    return launched(who, exb::launch_norm_backward(a, dtype, dweight, dbias, workspace, (cudaStream_t)stream));
}

}  // extern "C"
