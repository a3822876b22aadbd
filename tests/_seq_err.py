"""Bounds on what ``selective_scan`` may lose in float32, carried through the recurrence: an error of one step decays with the
state that it is in, so that the bounds do not grow with the length of the sequence."""
from __future__ import annotations

import torch

from tests import _seq_ref as ref

U = 2.0 ** -24


def scan_bounds(x, dt, A, B, C, D=None, z=None, dt_bias=None, h0=None, dt_softplus=True, dy=None, dh=None):
    """Error bounds by output, in units that the caller scales: every rounding counts fully.

    One step: the step size (softplus: 8 roundings; the sums of step sizes over a piece of time: a random walk over some 100
    terms, 16), the exponent (2 roundings and those of the step size, each as large as the exponent), 2^v (4), the input
    (2 and the step size's), the update (1).  Sums over N states or M channels round N + 4 or M + 4 times, silu 12 times.
    """
    x, dt, A, B, C, D, z, dt_bias, h0, dy, dh = ref.f64(x, dt, A, B, C, D, z, dt_bias, h0, dy, dh)
    nb, T, M = x.shape
    G, N = B.shape[2:]
    per, f64 = M // G, dict(device=x.device, dtype=torch.float64)
    group = torch.arange(M, device=x.device) // per
    pre = dt + (dt_bias if dt_bias is not None else 0)
    s = torch.nn.functional.softplus(pre, threshold=200.0) if dt_softplus else pre
    slope = torch.sigmoid(pre) if dt_softplus else torch.ones_like(pre)
    rs = (8 if dt_softplus else 1) + 16
    skip = D if D is not None else torch.zeros(M, **f64)
    gate = ref.silu(z) if z is not None else torch.ones_like(x)
    egate = 12 * U * (gate.abs() + 0.1) if z is not None else torch.zeros_like(x)

    def factors(t):
        sA = s[:, t, :, None] * A
        return torch.exp(sA), (4 + (2 + rs) * sA.abs()) * U

    h = torch.zeros(nb, M, N, **f64) if h0 is None else h0
    e = torch.zeros_like(h)
    hs, es, raw, eraw = [h], [e], [], []
    for t in range(T):
        a, ra = factors(t)
        u = (s[:, t] * x[:, t])[..., None] * B[:, t][:, group]
        new = a * h + u
        e = a * e + (a * h).abs() * ra + u.abs() * (rs + 2) * U + new.abs() * U
        h = new
        hs.append(h)
        es.append(e)
        Ct = C[:, t][:, group]
        raw.append((h * Ct).sum(-1) + skip * x[:, t])
        eraw.append((e * Ct.abs()).sum(-1) + (N + 4) * U * ((h * Ct).abs().sum(-1) + (skip * x[:, t]).abs()))
    raw, eraw = torch.stack(raw, 1), torch.stack(eraw, 1)
    out = {"y": eraw * gate.abs() + raw.abs() * egate + 2 * U * (raw * gate).abs(), "h": e}
    if dy is None:
        return out
    p, ep = dy * gate, dy.abs() * egate + U * (dy * gate).abs()
    g = torch.zeros_like(h) if dh is None else dh
    eg = torch.zeros_like(g)
    ex, edt, eB, eC = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(B), torch.zeros_like(C)
    eA, eD, ebias = torch.zeros_like(A), torch.zeros(M, **f64), torch.zeros(M, **f64)
    for t in range(T - 1, -1, -1):
        a, ra = factors(t)
        Bt, Ct = B[:, t][:, group], C[:, t][:, group]
        cp = p[:, t, :, None] * Ct
        gt = g + cp
        egt = eg + ep[:, t, :, None] * Ct.abs() + 2 * U * cp.abs() + U * gt.abs()
        through = gt * a * hs[t]
        eth = a * (egt * hs[t].abs() + gt.abs() * es[t]) + through.abs() * (ra + 2 * U)
        gb, egb = (gt * Bt).sum(-1), (egt * Bt.abs()).sum(-1) + (N + 4) * U * (gt * Bt).abs().sum(-1)
        ds = (through * A).sum(-1) + gb * x[:, t]
        eds = (eth * A.abs()).sum(-1) + (N + 8) * U * (through * A).abs().sum(-1) + egb * x[:, t].abs() + 2 * U * (gb * x[:, t]).abs()
        dpre, edpre = ds * slope[:, t], eds * slope[:, t] + 12 * U * ds.abs()
        sx = (s[:, t] * x[:, t])[..., None]
        ex[:, t] = s[:, t].abs() * (egb + (rs + 2) * U * gb.abs()) + skip.abs() * ep[:, t] + 3 * U * (p[:, t] * skip).abs()
        edt[:, t] = edpre
        db, dc = gt * sx, p[:, t, :, None] * hs[t + 1]
        edb = egt * sx.abs() + (rs + 2) * U * db.abs()
        edc = ep[:, t, :, None] * hs[t + 1].abs() + p[:, t, :, None].abs() * es[t + 1] + U * dc.abs()
        eB[:, t] = (edb + (per + 4) * U * db.abs()).view(nb, G, per, N).sum(2)
        eC[:, t] = (edc + (per + 4) * U * dc.abs()).view(nb, G, per, N).sum(2)
        # sums over time: blocks of 8 and 32 steps and of those
        da = through * s[:, t, :, None]
        eA += (eth * s[:, t, :, None].abs() + (rs + 2 + 104) * U * da.abs()).sum(0)
        eD += (ep[:, t] * x[:, t].abs() + 104 * U * (p[:, t] * x[:, t]).abs()).sum(0)
        ebias += (edpre + 104 * U * dpre.abs()).sum(0)
        g = gt * a
        eg = a * egt + g.abs() * (ra + U)
    out.update(dx=ex, ddt=edt, dA=eA, dB=eB, dC=eC, dD=eD, ddt_bias=ebias, dh0=eg)
    if z is not None:
        k = ref.silu_slope(z)
        out["dz"] = dy.abs() * (eraw * k.abs() + raw.abs() * 16 * U * (k.abs() + 0.1))
    return out
