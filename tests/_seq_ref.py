"""Plain float64 forms of the sequence operators, with their gradients, and bounds on what float32 may lose.

Every function returns the value of each output and a majorant: the same sums with every term's absolute value.  A
float32 evaluation whose factors are each off by a relative ``d`` is off by at most ``terms * d * majorant``, which is what
the tolerances of the tests count.
"""
from __future__ import annotations

import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def silu(v):
    return v * torch.sigmoid(v)


def silu_slope(v):
    s = torch.sigmoid(v)
    return s * (1 + v * (1 - s))


def f64(*ts):
    return [None if t is None else t.detach().double() for t in ts]


def scan(x, dt, A, B, C, D=None, z=None, dt_bias=None, h0=None, lengths=None, dt_softplus=True, dy=None, dh=None):
    """(values, majorants) of ``selective_scan``, one step of time after the other; with ``dy`` the gradients too."""
    kinds = {"y": x.dtype, "dx": x.dtype, "ddt": x.dtype, "dB": x.dtype, "dC": x.dtype, "dz": x.dtype}
    x, dt, A, B, C, D, z, dt_bias, h0, dy, dh = f64(x, dt, A, B, C, D, z, dt_bias, h0, dy, dh)
    nb, T, M = x.shape
    if B.ndim == 3:
        B, C = B.unsqueeze(2), C.unsqueeze(2)
    G, N = B.shape[2:]
    own_group = torch.arange(M, device=x.device) // (M // G)
    pre = dt + (dt_bias if dt_bias is not None else 0)
    s = torch.nn.functional.softplus(pre, threshold=200.0) if dt_softplus else pre
    slope = torch.sigmoid(pre) if dt_softplus else torch.ones_like(pre)
    n_valid = torch.full((nb,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    skip = D if D is not None else torch.zeros(M, device=x.device, dtype=torch.float64)

    def sweep(x, s, A_in, B, C, h0, skip, dy, dh, z, absolute):
        decay_A = A                                              # the decays are those of the operator in both sweeps
        h = torch.zeros(nb, M, N, device=x.device, dtype=torch.float64) if h0 is None else h0
        hs, raws = [h], []
        for t in range(T):
            live = (t < n_valid)[:, None, None]
            a = torch.exp(s_true[:, t, :, None] * decay_A)
            new = a * h + (s[:, t] * x[:, t])[..., None] * B[:, t][:, own_group]
            h = torch.where(live, new, h)
            hs.append(h)
            raw = (h * C[:, t][:, own_group]).sum(-1) + skip * x[:, t]
            raws.append(torch.where(live[..., 0], raw, torch.zeros_like(raw)))
        raw = torch.stack(raws, 1)
        gate = None if z is None else (silu(z).abs() if absolute else silu(z))
        keep = (torch.arange(T, device=x.device)[None] < n_valid[:, None])[..., None]
        y = raw if gate is None else raw * torch.where(keep, gate, torch.zeros_like(gate))
        r = {"y": y, "h": h}
        if dy is None:
            return r
        p = dy if gate is None else dy * gate
        p = torch.where(keep, p, torch.zeros_like(p))
        g = torch.zeros_like(h) if dh is None else dh
        dx, ddt = torch.zeros_like(x), torch.zeros_like(x)
        dB, dC = torch.zeros_like(B), torch.zeros_like(C)
        dA, dD, dbias = torch.zeros_like(A), torch.zeros_like(skip), torch.zeros_like(skip)
        for t in range(T - 1, -1, -1):
            live = (t < n_valid)[:, None, None]
            Bt, Ct = B[:, t][:, own_group], C[:, t][:, own_group]
            a = torch.exp(s_true[:, t, :, None] * decay_A)
            gt = g + p[:, t, :, None] * Ct
            through = gt * a * hs[t]
            gb = (gt * Bt).sum(-1)
            ds = (through * A_in).sum(-1) + gb * x[:, t]
            dpre = torch.where(live[..., 0], ds * slope[:, t], torch.zeros_like(ds))
            dx[:, t] = torch.where(live[..., 0], p[:, t] * skip + s[:, t] * gb, torch.zeros_like(gb))
            ddt[:, t] = dpre
            per = M // G
            db = gt * (s[:, t] * x[:, t])[..., None]
            dc = p[:, t, :, None] * hs[t + 1]
            dB[:, t] = torch.where(live, db, torch.zeros_like(db)).view(nb, G, per, N).sum(2)
            dC[:, t] = torch.where(live, dc, torch.zeros_like(dc)).view(nb, G, per, N).sum(2)
            da = through * s[:, t, :, None]
            dA += torch.where(live, da, torch.zeros_like(da)).sum(0)
            dD += torch.where(live[..., 0], p[:, t] * x[:, t], torch.zeros_like(dpre)).sum(0)
            dbias += dpre.sum(0)
            g = torch.where(live, gt * a, g)
        r.update(dx=dx, ddt=ddt, dA=dA, dB=dB, dC=dC, dD=dD, ddt_bias=dbias, dh0=g)
        if z is not None:
            k = silu_slope(z)
            r["dz"] = dy * raw * (k.abs() + 1e-2 if absolute else k)
            r["dz"] = torch.where(keep, r["dz"], torch.zeros_like(r["dz"]))
        return r

    def clean(t):      # rows behind the sequence may hold anything
        if t is None:
            return None
        keep = (torch.arange(T, device=t.device)[None] < n_valid[:, None]).view(nb, T, *[1] * (t.ndim - 2))
        return torch.where(keep, t, torch.zeros_like(t))

    x, B, C, z, dy, s, slope = (clean(t) for t in (x, B, C, z, dy, s, slope))
    s_true = s
    value = sweep(x, s, A, B, C, h0, skip, dy, dh, z, False)
    ab = [None if t is None else t.abs() for t in (x, s, A, B, C, h0, skip, dy, dh)]
    bound = sweep(*ab, z, True)
    emax = float((s.unsqueeze(-1) * A).abs().max()) if s.numel() else 0.0
    return value, bound, emax, kinds


def scan_tolerance(bound, emax, T, kind):
    """Relative error of one step's factors in float32: the step size (softplus: 6 roundings, amplified by at most the
    exponent), the exponent (two roundings), 2^v (2 ulp), the products: (12 + 8 emax) * 2^-24 with some room to 2^-20;
    at most T of them lie between a term and a sum; each sum over states or channels of a shape used here adds fewer
    than 16 roundings in its tree."""
    step = (12 + 8 * emax) * 2.0 ** -24
    return (step * (T + 1) + 32 * 2.0 ** -24) * bound


def assert_close(got, want, slack, kind, name):
    """|got - want| <= half a step of ``kind`` at the value + ``slack`` (elementwise), and nothing subnormal is asked of
    float16."""
    got64 = got.detach().double()
    assert got.dtype == kind, (name, got.dtype)
    assert got64.shape == want.shape, (name, got64.shape, want.shape)
    tiny = 2.0 ** -25 if kind == torch.float16 else 1e-36
    tol = HALF_STEP[kind] * (want.abs() + slack) + slack + tiny
    worst = (got64 - want).abs() - tol
    bad = ~((got64 - want).abs() <= tol)
    assert not bad.any(), f"{name}: {int(bad.sum())} of {bad.numel()} off, worst by {float(worst.max()):.3e} " \
        f"(largest value {float(want.abs().max()):.3e}, largest slack {float(torch.as_tensor(slack).max()):.3e})"


def conv(x, weight, bias=None, state=None, lengths=None, activation=None):
    """``causal_conv`` in float64, differentiable by autograd (arguments are float64 already)."""
    nb, T, M = x.shape
    W = weight.shape[1]
    n_valid = torch.full((nb,), T, device=x.device) if lengths is None else lengths.long().clamp(0, T)
    keep = (torch.arange(T, device=x.device)[None] < n_valid[:, None])[..., None]
    x = torch.where(keep, x, torch.zeros_like(x))
    head = torch.zeros(nb, W - 1, M, device=x.device, dtype=x.dtype) if state is None else state
    full = torch.cat([head, x], 1)
    pre = torch.zeros_like(x) + (bias if bias is not None else 0)
    for k in range(W):
        pre = pre + full[:, k:k + T] * weight[:, k]
    y = silu(pre) if activation == "silu" else pre
    y = torch.where(keep, y, torch.zeros_like(y))
    last = torch.stack([full[b, int(n_valid[b]):int(n_valid[b]) + W - 1] for b in range(nb)]) if nb else head
    return y, last


def norm(x, groups, weight=None, bias=None, eps=1e-5, activation=None):
    """``group_norm`` of (samples, positions, channels) in float64, differentiable by autograd."""
    R, S, C = x.shape
    v = x.view(R, S, groups, C // groups)
    mean = v.mean((1, 3), keepdim=True)
    var = ((v - mean) ** 2).mean((1, 3), keepdim=True)
    n = ((v - mean) / torch.sqrt(var + eps)).reshape(R, S, C)
    pre = n * (weight if weight is not None else 1) + (bias if bias is not None else 0)
    return silu(pre) if activation == "silu" else torch.relu(pre) if activation == "relu" else pre
