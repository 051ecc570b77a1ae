"""Linear attention and the norms of `pathsig_amd.sequence` in 64 bits, token by token and row by row, with their gradients by
formula.  Run on absolute values, the same formulas bound what roundings of their terms add up to."""
from __future__ import annotations

import torch


def attention(q, k, v, g, s0=None, lengths=None, scale=None, do=None, ds=None):
    """dict of out, last and, with `do`, the gradients dq, dk, dv, dg (per head), ds0.  All arguments double."""
    B, L, H, Dk = q.shape
    Hkv, Dv = v.shape[2:]
    group = H // Hkv
    scale = Dk ** -0.5 if scale is None else scale
    n = torch.full((B,), L) if lengths is None else lengths.cpu().clamp(0, L)
    live = (torch.arange(L)[None] < n[:, None]).to(q.device)          # (B, L)
    q, k, v = (torch.where(live[..., None, None], t, torch.zeros_like(t)) for t in (q, k, v))
    k, v = (t.repeat_interleave(group, dim=2) for t in (k, v))
    decay = torch.exp(g)[None, :, None, None]
    S = torch.zeros(B, H, Dk, Dv, dtype=q.dtype, device=q.device) if s0 is None else s0.clone()
    before, out = [], torch.zeros(B, L, H, Dv, dtype=q.dtype, device=q.device)
    for t in range(L):
        before.append(S)
        new = decay * S + k[:, t, :, :, None] * v[:, t, :, None, :]
        S = torch.where(live[:, t, None, None, None], new, S)
        out[:, t] = scale * (q[:, t, :, :, None] * S).sum(2) * live[:, t, None, None]
    result = {"out": out, "last": S}
    if do is None:
        return result
    do = torch.where(live[..., None, None], do, torch.zeros_like(do))
    R = torch.zeros_like(S) if ds is None else ds.clone()              # dL/dS after token t
    dq, dk, dv, dg = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v), torch.zeros_like(g)
    for t in reversed(range(L)):
        on = live[:, t, None, None, None]
        after = decay * before[t] + k[:, t, :, :, None] * v[:, t, :, None, :]
        dq[:, t] = scale * (after * do[:, t, :, None, :]).sum(3) * live[:, t, None, None]
        full = R + scale * q[:, t, :, :, None] * do[:, t, :, None, :]
        dk[:, t] = (full * v[:, t, :, None, :]).sum(3) * live[:, t, None, None]
        dv[:, t] = (full * k[:, t, :, :, None]).sum(2) * live[:, t, None, None]
        dg += torch.where(on, decay * before[t] * full, torch.zeros_like(full)).sum((0, 2, 3))
        R = torch.where(on, decay * full, R)
    dk, dv = (t.unflatten(2, (Hkv, group)).sum(3) for t in (dk, dv))
    result.update(dq=dq, dk=dk, dv=dv, dg=dg, ds0=R)
    return result


def attention_bound(q, k, v, g, s0=None, lengths=None, scale=None, do=None, ds=None):
    parts = [None if t is None else t.abs() for t in (q, k, v, s0, do, ds)]
    return attention(parts[0], parts[1], parts[2], g, parts[3], lengths, scale, parts[4], parts[5])


def gate_of(gate, activation):
    """act(g) and its derivative."""
    s = torch.sigmoid(gate)
    return {"silu": (gate * s, s + gate * s * (1 - s)), "sigmoid": (s, s * (1 - s)), "linear": (gate, torch.ones_like(gate))}[activation]


def norms(x, weight=None, gate=None, residual=None, scale=None, next_weight=None, eps=1e-6, activation="silu", do=None, dn=None):
    """dict of out, next and, with gradients from above, those of every argument; under "bound" what the terms of each add up to
    in absolute value."""
    one = torch.ones(x.shape[-1], dtype=x.dtype, device=x.device)
    w, s, nw = (one if t is None else t for t in (weight, scale, next_weight))
    u, du = (one, 0 * one) if gate is None else gate_of(gate, activation)
    res = torch.zeros_like(x) if residual is None else residual
    r = (x.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit = x * r
    joined = unit * w * u
    out = res + s * joined
    r2 = (out.square().mean(-1, keepdim=True) + eps).rsqrt()
    unit2 = out * r2
    size = res.abs() + (s * joined).abs()
    got = {"out": out, "next": unit2 * nw}
    bound = {"out": size, "next": (size * r2 + unit2.abs() * ((size * r2) * unit2.abs()).mean(-1, keepdim=True)) * nw.abs()}
    if do is None:
        return got, bound
    d, D = do, do.abs()
    if dn is not None:
        a = dn * nw
        d = d + r2 * (a - unit2 * (a * unit2).mean(-1, keepdim=True))
        # (out itself is a sum whose terms may cancel)
        size2 = size * r2
        D = D + r2 * (a.abs() + 2 * size2 * (a.abs() * size2).mean(-1, keepdim=True))
        got["next_weight"], bound["next_weight"] = (dn * unit2).sum(0), (dn.abs() * size2).sum(0)
    got["residual"], bound["residual"] = d, D
    got["scale"], bound["scale"] = (d * joined).sum(0), (D * joined.abs()).sum(0)
    got["gate"], bound["gate"] = d * s * unit * w * du, D * (s * unit * w).abs() * (du.abs() + u.abs())
    b, B = d * s * u * w, D * (s * u * w).abs()
    got["weight"], bound["weight"] = (d * s * u * unit).sum(0), (D * (s * u * unit).abs()).sum(0)
    got["x"] = r * (b - unit * (b * unit).mean(-1, keepdim=True))
    bound["x"] = r * (B + unit.abs() * (B * unit.abs()).mean(-1, keepdim=True))
    return got, bound
