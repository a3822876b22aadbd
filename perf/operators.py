"""The workloads on which the selective scan, its short convolution, their single-token forms and the group norm are
measured: inputs, one pass of each operator in plain torch operations or through the package, and the work of a pass.

Every tensor is time-major / channels last, as the package's layers use it: ``(batch, time, channels)``.
"""
import math

import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


# ------------------------------------------------------------------------------------------------ cases

def listed():
    return [
        # the first tokens of a short request: a call of a few microseconds
        dict(name="scan_prompt_short", op="scan", train=False, B=1, T=128, D=512, N=16, G=1, type="bf16", gate=True, carry=False, ragged=False),
        # one long document: few rows, so the time axis has to be split; the state carries on from an earlier chunk
        dict(name="scan_prompt_long", op="scan", train=False, B=1, T=16384, D=1024, N=16, G=1, type="bf16", gate=True, carry=True, ragged=False),
        # a training step of a wide layer: the largest case
        dict(name="scan_train_wide", op="scan", train=True, B=4, T=2048, D=2048, N=16, G=1, type="bf16", gate=True, carry=False, ragged=False),
        # odd sizes in full precision: a padded batch with several groups and a carried state
        dict(name="scan_train_odd", op="scan", train=True, B=3, T=777, D=510, N=10, G=3, type="f32", gate=False, carry=True, ragged=True),
        # decoding one token for one request, and for many requests at once
        dict(name="step_single", op="scan_step", B=1, D=1024, N=16, G=1, type="bf16", gate=True),
        dict(name="step_batch", op="scan_step", B=256, D=4096, N=16, G=1, type="bf16", gate=True),
        # the short convolution in front of the scan: training, and a padded batch of prompts with odd sizes
        dict(name="conv_train", op="conv", train=True, B=8, T=2048, D=4096, W=4, type="bf16", act="silu", carry=False, ragged=False),
        dict(name="conv_prompt_odd", op="conv", train=False, B=5, T=1999, D=1023, W=3, type="f16", act="silu", carry=True, ragged=True),
        # the convolution of one token
        dict(name="conv_step_single", op="conv_step", B=1, D=1024, W=4, type="bf16", act="silu"),
        dict(name="conv_step_batch", op="conv_step", B=512, D=4096, W=4, type="bf16", act="silu"),
        # feature maps between a convolution and a spiking layer, trained (256 frames of 64 x 64, 64 channels)
        dict(name="norm_maps_train", op="norm", train=True, R=256, S=4096, C=64, G=8, type="bf16", act="silu"),
        # one token per row behind the scan, full precision
        dict(name="norm_tokens", op="norm", train=False, R=8191, S=1, C=1536, G=24, type="f32", act=None),
    ]


def _log(rng, low, high):
    return max(low, min(high, int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))))


def draw(rng):
    """A case of the ranges above: sizes spread over their logarithm, odd ones among them."""
    kind = rng.choice(["scan", "scan", "scan_step", "conv", "conv_step", "norm"])
    c = dict(op=kind, type=rng.choice(["bf16", "bf16", "f16", "f32"]))
    if kind in ("scan", "scan_step"):
        c["N"] = rng.choice([4, 8, 10, 16, 16, 16, 32, 64])
        c["G"] = rng.choice([1, 1, 2, 4])
        c["gate"] = rng.random() < 0.6
    if kind == "scan":
        c["B"] = _log(rng, 1, 16)
        c["D"] = c["G"] * _log(rng, 64 // c["G"], 2048 // c["G"])
        c["T"] = max(1, min(_log(rng, 16, 16384), (1 << 27) // (c["B"] * c["D"] * c["N"])))
        c.update(train=rng.random() < 0.5, carry=rng.random() < 0.5, ragged=rng.random() < 0.3)
    elif kind == "scan_step":
        c["B"] = _log(rng, 1, 256)
        c["D"] = c["G"] * _log(rng, 64 // c["G"], 4096 // c["G"])
        c["N"] = min(c["N"], 32)
    elif kind == "conv":
        c.update(B=_log(rng, 1, 16), D=_log(rng, 64, 4096), W=rng.choice([2, 3, 4, 4, 5]), act=rng.choice(["silu", None]))
        c["T"] = max(1, min(_log(rng, 16, 8192), (1 << 25) // (c["B"] * c["D"])))
        c.update(train=rng.random() < 0.5, carry=rng.random() < 0.5, ragged=rng.random() < 0.3)
    elif kind == "conv_step":
        c.update(B=_log(rng, 1, 512), D=_log(rng, 64, 4096), W=rng.choice([2, 3, 4, 4, 5]), act=rng.choice(["silu", None]))
    else:
        c["G"] = rng.choice([1, 2, 4, 8, 16, 32])
        c["C"] = c["G"] * _log(rng, 2, 64)
        if rng.random() < 0.6:
            side = _log(rng, 4, 96)
            c["S"] = side * side
        else:
            c["S"] = 1
        c["R"] = max(1, min(_log(rng, 1, 16384), (1 << 25) // (c["S"] * c["C"])))
        c.update(train=rng.random() < 0.5, act=rng.choice(["silu", "relu", None]))
    return c


# ------------------------------------------------------------------------------------------------ inputs

def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind = _TYPES[case["type"]]

    def normal(*shape, std=1.0, mean=0.0, dtype=kind):
        return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)

    def uniform(*shape, low=0.0, high=1.0):
        return torch.rand(*shape, generator=gen, device="cuda") * (high - low) + low

    s = {"case": case}
    op = case["op"]
    if op in ("scan", "scan_step"):
        B, D, N, G = case["B"], case["D"], case["N"], case["G"]
        rows = (B, case["T"]) if op == "scan" else (B,)
        x = normal(*rows, D)
        s["x"] = (x * torch.sigmoid(x.float())).to(kind)
        s["dt"] = normal(*rows, D, std=0.5)
        s["B"] = normal(*rows, G, N)
        s["C"] = normal(*rows, G, N)
        # step sizes between 0.001 and 0.1 before the input moves them; rates around 1 ... N
        first = torch.exp(uniform(D, low=math.log(0.001), high=math.log(0.1)))
        s["dt_bias"] = first + torch.log(-torch.expm1(-first))
        s["A"] = -(torch.arange(1, N + 1, device="cuda", dtype=torch.float32) * uniform(D, N, low=0.8, high=1.2))
        s["skip"] = normal(D, std=0.2, mean=1.0, dtype=torch.float32)
        s["z"] = normal(*rows, D) if case["gate"] else None
        if op == "scan_step":
            s["h"] = normal(B, D, N, std=0.3, dtype=torch.float32)
            return s
        s["h0"] = normal(B, D, N, std=0.3, dtype=torch.float32) if case["carry"] else None
        leaves = ("x", "dt", "A", "B", "C", "skip", "z", "dt_bias", "h0")
    elif op in ("conv", "conv_step"):
        B, D, W = case["B"], case["D"], case["W"]
        s["weight"] = normal(D, W, std=W ** -0.5)
        s["bias"] = normal(D, std=0.1)
        if op == "conv_step":
            s["x"] = normal(B, D)
            s["state"] = normal(B, W - 1, D)
            return s
        s["x"] = normal(B, case["T"], D)
        s["state"] = normal(B, W - 1, D) if case["carry"] else None
        leaves = ("x", "weight", "bias", "state")
    else:
        shape = (case["R"], case["S"], case["C"])
        s["x"] = normal(*shape, std=1.5, mean=0.5)
        s["weight"] = normal(case["C"], std=0.2, mean=1.0, dtype=torch.float32)
        s["bias"] = normal(case["C"], std=0.2, dtype=torch.float32)
        if case["train"]:
            s["dy"] = normal(*shape)
        leaves = ("x", "weight", "bias")
    if op != "norm":
        B, T = case["B"], case["T"]
        s["lengths"] = None
        if case["ragged"]:
            s["lengths"] = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        if case["train"]:
            s["dy"] = normal(B, T, case["D"])
            if op == "scan":
                s["dh"] = normal(B, case["D"], case["N"], dtype=torch.float32) if case["carry"] else None
    s["leaves"] = [k for k in leaves if s[k] is not None]
    if case["train"]:
        for k in s["leaves"]:
            s[k].requires_grad_(True)
    return s


# ------------------------------------------------------------------------------------------------ one pass

def run(state):
    op = state["case"]["op"]
    if own:
        return _OWN[op](state)
    with torch.no_grad():
        return _PLAIN[op](state)


def _gradients(state, outputs, upstream):
    grads = torch.autograd.grad(outputs, [state[k] for k in state["leaves"]], upstream)
    return {"d_" + k: g for k, g in zip(state["leaves"], grads)}


def _own_scan(s):
    import sinabs_exodus_b200 as ex

    y, h = ex.selective_scan(s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], dt_bias=s["dt_bias"],
                             h0=s["h0"], lengths=s["lengths"], dt_softplus=True)
    out = {"y": y, "h": h}
    if s["case"]["train"]:
        if s["dh"] is None:
            out.update(_gradients(s, [y], [s["dy"]]))
        else:
            out.update(_gradients(s, [y, h], [s["dy"], s["dh"]]))
    return {k: v.detach() for k, v in out.items()}


def _own_scan_step(s):
    import sinabs_exodus_b200 as ex

    y = ex.selective_step(s["h"], s["x"], s["dt"], s["A"], s["B"], s["C"], D=s["skip"], z=s["z"], dt_bias=s["dt_bias"],
                          dt_softplus=True)
    return {"y": y, "h": s["h"]}


def _own_conv(s):
    import sinabs_exodus_b200 as ex

    y, last = ex.causal_conv(s["x"], s["weight"], s["bias"], state=s["state"], lengths=s["lengths"],
                             activation=s["case"]["act"])
    out = {"y": y, "last": last}
    if s["case"]["train"]:
        out.update(_gradients(s, [y], [s["dy"]]))
    return {k: v.detach() for k, v in out.items()}


def _own_conv_step(s):
    import sinabs_exodus_b200 as ex

    y = ex.causal_conv_step(s["state"], s["x"], s["weight"], s["bias"], activation=s["case"]["act"])
    return {"y": y, "state": s["state"]}


def _own_norm(s):
    import sinabs_exodus_b200 as ex

    y = ex.group_norm(s["x"], s["case"]["G"], s["weight"], s["bias"], eps=1e-5, activation=s["case"]["act"])
    out = {"y": y}
    if s["case"]["train"]:
        out.update(_gradients(s, [y], [s["dy"]]))
    return {k: v.detach() for k, v in out.items()}


_OWN = {"scan": _own_scan, "scan_step": _own_scan_step, "conv": _own_conv, "conv_step": _own_conv_step, "norm": _own_norm}


# ------------------------------------------------------------------------------------------------ plain form

def _softplus(v):
    return torch.clamp(v, min=0) + torch.log1p(torch.exp(-v.abs()))


def _linear_scan(a, b):
    """``h_t = a_t h_{t-1} + b_t`` along dimension 1 by doubling the reach log2(T) times; overwrites its arguments."""
    reach = 1
    while reach < b.shape[1]:
        b[:, reach:] = torch.addcmul(b[:, reach:], a[:, reach:], b[:, :-reach])
        a[:, reach:] = a[:, reach:] * a[:, :-reach]
        reach *= 2
    return b


def _valid(s, T):
    """(B, T, 1) mask of the rows that belong to a sequence, or None."""
    if s["lengths"] is None:
        return None
    return (torch.arange(T, device="cuda")[None, :] < s["lengths"][:, None])[..., None]


def _plain_scan(s):
    case, kind = s["case"], s["x"].dtype
    B, T, D, N, G = case["B"], case["T"], case["D"], case["N"], case["G"]
    per_group = (B, T, G, D // G)
    x, Bt, Ct = s["x"].float(), s["B"].float(), s["C"].float()
    pre = s["dt"].float() + s["dt_bias"]
    dt = _softplus(pre)
    valid = _valid(s, T)
    if valid is not None:
        dt = torch.where(valid, dt, 0.0)
    h0 = s["h0"] if s["h0"] is not None else torch.zeros(B, D, N, device="cuda")
    a = torch.exp(dt[..., None] * s["A"])
    b = ((dt * x).view(*per_group, 1) * Bt[:, :, :, None]).view(B, T, D, N)
    b[:, 0] += a[:, 0] * h0
    keep = a.clone() if case["train"] else None
    h = _linear_scan(a, b)
    del a
    raw = (h.view(*per_group, N) * Ct[:, :, :, None]).sum(-1).view(B, T, D) + s["skip"] * x
    z = s["z"].float() if s["z"] is not None else None
    gate = z * torch.sigmoid(z) if z is not None else None
    y = raw * gate if gate is not None else raw
    if valid is not None:
        y = torch.where(valid, y, 0.0)
    out = {"y": y.to(kind), "h": h[:, -1].clone()}
    if not case["train"]:
        return out
    dy = s["dy"].float()
    if valid is not None:
        dy = torch.where(valid, dy, 0.0)
    p = dy * gate if gate is not None else dy
    out["d_x"] = out["d_dt"] = None          # the order of the leaves
    # reverse recurrence of the gradient of h
    later = torch.zeros_like(keep)
    later[:, :-1] = keep[:, 1:]
    g = (p.view(*per_group, 1) * Ct[:, :, :, None]).view(B, T, D, N)
    if s["dh"] is not None:
        g[:, -1] += s["dh"]
    g = _linear_scan(later.flip(1), g.flip(1)).flip(1)
    del later
    d_c = (p.view(*per_group, 1) * h.view(*per_group, N)).sum(3)
    d_b = (g.view(*per_group, N) * (dt * x).view(*per_group, 1)).sum(3)
    from_b = (g.view(*per_group, N) * Bt[:, :, :, None]).sum(-1).view(B, T, D)
    before = torch.cat([h0[:, None], h[:, :-1]], 1)
    del h
    through = g * keep * before
    d_dt = (through * s["A"]).sum(-1) + from_b * x
    d_pre = d_dt * torch.sigmoid(pre)
    d_x = s["skip"] * p + dt * from_b
    if valid is not None:
        d_pre = torch.where(valid, d_pre, 0.0)
    out["d_x"], out["d_dt"] = d_x.to(kind), d_pre.to(kind)
    out["d_A"] = (through * dt[..., None]).sum((0, 1))
    out["d_B"], out["d_C"] = d_b.to(kind), d_c.to(kind)
    out["d_skip"] = (p * x).sum((0, 1))
    if z is not None:
        sig = torch.sigmoid(z)
        out["d_z"] = (dy * raw * sig * (1 + z * (1 - sig))).to(kind)
    out["d_dt_bias"] = d_pre.sum((0, 1))
    if s["h0"] is not None:
        out["d_h0"] = g[:, 0] * keep[:, 0]
    return out


def _plain_scan_step(s):
    case, kind = s["case"], s["x"].dtype
    B, D, N, G = case["B"], case["D"], case["N"], case["G"]
    x = s["x"].float()
    dt = _softplus(s["dt"].float() + s["dt_bias"])
    h = torch.exp(dt[..., None] * s["A"]) * s["h"]
    h += ((dt * x).view(B, G, D // G, 1) * s["B"].float()[:, :, None]).view(B, D, N)
    y = (h.view(B, G, D // G, N) * s["C"].float()[:, :, None]).sum(-1).view(B, D) + s["skip"] * x
    if s["z"] is not None:
        z = s["z"].float()
        y = y * z * torch.sigmoid(z)
    s["h"].copy_(h)
    return {"y": y.to(kind), "h": s["h"]}


def _plain_conv(s):
    case, kind = s["case"], s["x"].dtype
    B, T, D, W = case["B"], case["T"], case["D"], case["W"]
    x, w = s["x"].float(), s["weight"].float()
    head = s["state"].float() if s["state"] is not None else torch.zeros(B, W - 1, D, device="cuda")
    full = torch.cat([head, x], 1)
    pre = s["bias"].float().expand(B, T, D)
    for k in range(W):
        pre = torch.addcmul(pre, full[:, k:k + T], w[:, k])
    sig = torch.sigmoid(pre) if case["act"] == "silu" else None
    y = pre * sig if sig is not None else pre
    valid = _valid(s, T)
    if valid is not None:
        y = torch.where(valid, y, 0.0)
    end = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    rows = end[:, None] + torch.arange(W - 1, device="cuda")
    last = torch.gather(full, 1, rows[..., None].expand(B, W - 1, D).long())
    out = {"y": y.to(kind), "last": last.to(kind)}
    if not case["train"]:
        return out
    d = s["dy"].float()
    if sig is not None:
        d = d * sig * (1 + pre * (1 - sig))
    if valid is not None:
        d = torch.where(valid, d, 0.0)
    d_full = torch.zeros_like(full)
    d_w = torch.empty_like(w)
    for k in range(W):
        d_full[:, k:k + T] += d * w[:, k]
        d_w[:, k] = (d * full[:, k:k + T]).sum((0, 1))
    out["d_x"] = d_full[:, W - 1:].to(kind)
    out["d_weight"], out["d_bias"] = d_w.to(kind), d.sum((0, 1)).to(kind)
    if s["state"] is not None:
        out["d_state"] = d_full[:, :W - 1].to(kind)
    return out


def _plain_conv_step(s):
    kind = s["x"].dtype
    window = torch.cat([s["state"], s["x"][:, None]], 1)
    y = (window.float() * s["weight"].float().t()).sum(1) + s["bias"].float()
    if s["case"]["act"] == "silu":
        y = y * torch.sigmoid(y)
    s["state"].copy_(window[:, 1:])
    return {"y": y.to(kind), "state": s["state"]}


def _plain_norm(s):
    case, kind = s["case"], s["x"].dtype
    R, S, C, G = case["R"], case["S"], case["C"], case["G"]
    shape = (R, S, G, C // G)
    x = s["x"].float().view(shape)
    mean = x.mean((1, 3), keepdim=True)
    centred = x - mean
    rstd = torch.rsqrt((centred * centred).mean((1, 3), keepdim=True) + 1e-5)
    norm = (centred * rstd).view(R, S, C)
    pre = norm * s["weight"] + s["bias"]
    if case["act"] == "silu":
        sig = torch.sigmoid(pre)
        y, slope = pre * sig, sig * (1 + pre * (1 - sig))
    elif case["act"] == "relu":
        y, slope = torch.clamp(pre, min=0), (pre > 0).float()
    else:
        y, slope = pre, None
    out = {"y": y.to(kind)}
    if not case["train"]:
        return out
    d = s["dy"].float()
    if slope is not None:
        d = d * slope
    d_norm = (d * s["weight"]).view(shape)
    n = norm.view(shape)
    d_x = rstd * (d_norm - d_norm.mean((1, 3), keepdim=True) - n * (d_norm * n).mean((1, 3), keepdim=True))
    out["d_x"] = d_x.view(R, S, C).to(kind)
    out["d_weight"], out["d_bias"] = (d * norm).sum((0, 1)), d.sum((0, 1))
    return out


_PLAIN = {"scan": _plain_scan, "scan_step": _plain_scan_step, "conv": _plain_conv, "conv_step": _plain_conv_step,
          "norm": _plain_norm}


# ------------------------------------------------------------------------------------------------ in 64 bits

def exact(case, seed):
    """What ``run`` returns, from the definitions in float64: one step of time after the other, gradients by autograd."""
    s = prepare(case, seed)
    train = case.get("train", False)
    e = {}
    for k, v in s.items():
        if torch.is_tensor(v) and v.is_floating_point():
            e[k] = v.detach().double().requires_grad_(train and k in s.get("leaves", ()))
        else:
            e[k] = v
    with torch.set_grad_enabled(train):
        out = _EXACT[case["op"]](case, e)
        if train:
            up = [(out["y"], e["dy"])]
            if e.get("dh") is not None:
                up.append((out["h"], e["dh"]))
            grads = torch.autograd.grad([u[0] for u in up], [e[k] for k in s["leaves"]], [u[1] for u in up])
            out.update({"d_" + k: g for k, g in zip(s["leaves"], grads)})
    return {k: v.detach() for k, v in out.items()}


def _exact_step(case, e, h, x, dt, Bt, Ct, z, alive=None):
    """One step of the recurrence on ``(batch, channels)`` rows: the new state and the output."""
    per = case["D"] // case["G"]
    dt = torch.nn.functional.softplus(dt + e["dt_bias"], threshold=100.0)
    Bd, Cd = Bt.repeat_interleave(per, 1), Ct.repeat_interleave(per, 1)
    new = torch.exp(dt.unsqueeze(-1) * e["A"]) * h + (dt * x).unsqueeze(-1) * Bd
    y = torch.matmul(new.unsqueeze(-2), Cd.unsqueeze(-1))[..., 0, 0] + e["skip"] * x
    if z is not None:
        y = y * torch.nn.functional.silu(z)
    if alive is not None:
        new = torch.where(alive[:, None, None], new, h)
        y = torch.where(alive[:, None], y, torch.zeros_like(y))
    return new, y


def _exact_scan(case, e):
    h = e["h0"] if e["h0"] is not None else torch.zeros(case["B"], case["D"], case["N"], device="cuda", dtype=torch.float64)
    rows = []
    parts = [v.unbind(1) if v is not None else None for v in (e["x"], e["dt"], e["B"], e["C"], e["z"])]
    for t in range(case["T"]):
        row = [p[t] if p is not None else None for p in parts]
        h, y = _exact_step(case, e, h, *row, alive=None if e["lengths"] is None else t < e["lengths"])
        rows.append(y)
    return {"y": torch.stack(rows, 1), "h": h}


def _exact_scan_step(case, e):
    h, y = _exact_step(case, e, e["h"], e["x"], e["dt"], e["B"], e["C"], e["z"])
    return {"y": y, "h": h}


def _exact_conv(case, e):
    B, T, D, W = case["B"], case["T"], case["D"], case["W"]
    head = e["state"] if e["state"] is not None else torch.zeros(B, W - 1, D, device="cuda", dtype=torch.float64)
    rows, ends = [], []
    for b in range(B):
        n = T if e["lengths"] is None else int(e["lengths"][b])
        window = torch.cat([head[b], e["x"][b, :n]]).t()
        ends.append(window.t()[n:])
        y = (window.unfold(1, W, 1) * e["weight"][:, None]).sum(-1) if n else window[:, :0]
        y = y + e["bias"][:, None]
        if case["act"] == "silu":
            y = torch.nn.functional.silu(y)
        rows.append(torch.nn.functional.pad(y, (0, T - n)).t())
    return {"y": torch.stack(rows), "last": torch.stack(ends)}


def _exact_conv_step(case, e):
    window = torch.cat([e["state"], e["x"].unsqueeze(1)], 1)
    y = torch.einsum("bwd,dw->bd", window, e["weight"]) + e["bias"]
    if case["act"] == "silu":
        y = torch.nn.functional.silu(y)
    return {"y": y, "state": window[:, 1:].clone()}


def _exact_norm(case, e):
    R, S, C, G = case["R"], case["S"], case["C"], case["G"]
    x = e["x"].transpose(1, 2).reshape(R, G, -1)
    var, mean = torch.var_mean(x, dim=-1, unbiased=False, keepdim=True)
    y = ((x - mean) / torch.sqrt(var + 1e-5)).reshape(R, C, S).transpose(1, 2) * e["weight"] + e["bias"]
    if case["act"] is not None:
        y = getattr(torch.nn.functional, case["act"])(y)
    return {"y": y}


_EXACT = {"scan": _exact_scan, "scan_step": _exact_scan_step, "conv": _exact_conv, "conv_step": _exact_conv_step,
          "norm": _exact_norm}


# ------------------------------------------------------------------------------------------------ work

def work(case):
    """Bytes and operations of one pass: each input read once, each output written once."""
    es, op, train = _SIZE[case["type"]], case["op"], case.get("train", False)
    if op in ("scan", "scan_step"):
        B, D, N, G = case["B"], case["D"], case["N"], case["G"]
        T = case.get("T", 1)
        rows = B * T * D
        ends = 4 * B * D * N
        # x, dt, y (and z); B and C; A, D and dt_bias; the states at both ends
        moved = rows * es * (4 if case["gate"] else 3) + 2 * B * T * G * N * es + 4 * D * (N + 2)
        moved += ends * (2 if op == "scan_step" or case["carry"] else 1)
        # decay (product, exp), input (product), update and readout (a multiply-add each)
        done = rows * (7 * N + 8)
        if train:
            # dy read; the gradients of x, dt, z, B, C, A, D, dt_bias and of both states
            moved += rows * es * (4 if case["gate"] else 3) + 2 * B * T * G * N * es + 4 * D * (N + 2)
            moved += 2 * ends if case["carry"] else 0
            # reverse update, and the products of it with B, x, h and A that the five gradients sum
            done += rows * (16 * N + 16)
        return {"bytes": moved, "flops": done}
    if op in ("conv", "conv_step"):
        B, D, W = case["B"], case["D"], case["W"]
        T = case.get("T", 1)
        rows, state = B * T * D, B * (W - 1) * D
        kept = 2 if op == "conv_step" or case["carry"] else 1
        moved = es * (2 * rows + kept * state + D * (W + 1))
        done = rows * (2 * W + (4 if case["act"] else 0))
        if train:
            moved += es * (2 * rows + (state if case["carry"] else 0) + D * (W + 1))
            done += rows * (4 * W + (6 if case["act"] else 0))
        return {"bytes": moved, "flops": done}
    rows = case["R"] * case["S"] * case["C"]
    moved = es * 2 * rows + 8 * case["C"]
    done = rows * (8 + (4 if case["act"] else 0))
    if train:
        moved += es * 2 * rows + 8 * case["C"]
        done += rows * (16 + (6 if case["act"] else 0))
    return {"bytes": moved, "flops": done}
