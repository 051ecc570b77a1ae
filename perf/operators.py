"""Workloads of the sequence operators (`pathsig_amd.sequence`): linear attention with a decay for each head, for whole
sequences and for single tokens, and the norms before and after a block of a sequence model.

A case is a dict of plain values.  `kind`:

* "prompt": `linear_attention` without gradients, from a state to the state after the last token;
* "train":  `linear_attention` and the gradients of its inputs;
* "step":   `linear_attention_step`, one token of every sequence, the state updated in place;
* "before": `norm_before`; "after": `norm_after`; both with (`grad`) or without gradients.

Attention: `B`, `L`, `H`, `Hkv` (heads of keys and values, shared by H / Hkv heads of queries), `Dk`, `Dv`; `fused`: q, k
and v are views of one projection's output; `ragged`: sequences of unequal lengths, padded; `carry`: starts from a state
and hands one on; `learn`: the decays have a gradient.  Norms: `rows`, `C`, and for "after" `gate`, `residual` (with its
learned scale) and `next` (the norm before the next block).  `dtype`: "bf16" or "f32".
"""
import math

import torch

own = False

_DTYPE = {"f32": torch.float32, "bf16": torch.bfloat16}
_EPS = 1e-6
_CHUNK = 64


def _attention(name, kind, B, L, H, Hkv, Dk, Dv, dtype="bf16", fused=False, ragged=False, carry=False, learn=False):
    return dict(name=name, kind=kind, B=B, L=L, H=H, Hkv=Hkv, Dk=Dk, Dv=Dv, dtype=dtype, fused=fused, ragged=ragged,
                carry=carry, learn=learn)


def _norm(name, kind, rows, C, dtype="bf16", grad=True, gate=False, residual=False, next=False):
    return dict(name=name, kind=kind, rows=rows, C=C, dtype=dtype, grad=grad, gate=gate, residual=residual, next=next)


def listed():
    return [
        # one stream answered point by point while someone waits: nothing but latency
        _attention("step_one", "step", 1, 1, 4, 4, 64, 64),
        # a full serving batch: reads and writes the states of all streams
        _attention("step_batch", "step", 128, 1, 16, 16, 128, 128),
        # sizes that fit nothing, shared keys and values, single precision
        _attention("step_odd_f32", "step", 33, 1, 6, 2, 72, 40, dtype="f32"),
        # prompts of unequal length taken in before streaming starts, from one fused projection
        _attention("prompt_ragged", "prompt", 8, 2048, 16, 4, 128, 128, fused=True, ragged=True, carry=True),
        # one very long history
        _attention("prompt_long", "prompt", 1, 65536, 8, 8, 128, 128, carry=True),
        # the layer of a model in training, fixed decays: the largest
        _attention("train_base", "train", 16, 4096, 16, 16, 128, 128),
        # training with learned decays over pieces of longer sequences, the state and its gradient carried along
        _attention("train_learned", "train", 4, 8192, 8, 8, 64, 128, carry=True, learn=True),
        # odd lengths and head sizes in single precision (the batch of the odd workload of the signatures)
        _attention("train_odd_f32", "train", 50, 333, 6, 3, 40, 56, dtype="f32", ragged=True, carry=True, learn=True),
        # the norm in front of a block while streaming: latency
        _norm("before_step", "before", 128, 1024, grad=False),
        # the same in training
        _norm("before_train", "before", 32768, 2048),
        # the whole join of two blocks in training: norm, gate, residual scale, residual, next norm
        _norm("after_train", "after", 32768, 4096, gate=True, residual=True, next=True),
        # gated norm of every head's output, odd head size, single precision
        _norm("after_heads_f32", "after", 50 * 333 * 6, 56, dtype="f32", gate=True),
    ]


def _log_size(rng, lo, hi):
    return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))


def draw(rng):
    """One more case: 1 to 256 sequences of 1 to 65536 tokens, 1 to 32 heads of 8 to 256 channels, shared or not; norms of 1
    to 200 000 rows of 16 to 8192 channels; both types."""
    kind = rng.choice(("prompt", "prompt", "train", "train", "step", "before", "after"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    if kind in ("before", "after"):
        while True:
            rows, C = _log_size(rng, 1, 200000), _log_size(rng, 16, 8192)
            if rng.random() < 0.6:
                C = max(16, C // 64 * 64)
            if rows * C <= 32768 * 4096:
                break
        case = _norm("", kind, rows, C, dtype, grad=rng.random() < 0.7)
        if kind == "after":
            case.update(gate=rng.random() < 0.7, residual=rng.random() < 0.7, next=rng.random() < 0.5)
    else:
        while True:
            B, H = _log_size(rng, 1, 256), rng.randint(1, 32)
            L = 1 if kind == "step" else _log_size(rng, 1, 65536)
            Dk, Dv = _log_size(rng, 8, 256), _log_size(rng, 8, 256)
            if rng.random() < 0.6:
                Dk, Dv = (rng.choice((32, 64, 128, 256)) for _ in range(2))
            if B * H * Dk * Dv > 128 * 16 * 128 * 128:
                continue
            chunks = -(-L // _CHUNK)
            if B * H * L * max(Dk, Dv, 64) <= 16 * 4096 * 16 * 128 and B * H * chunks * Dk * Dv <= 16 * 64 * 16 * 128 * 128:
                break
        Hkv = rng.choice([n for n in range(1, H + 1) if H % n == 0])
        case = _attention("", kind, B, L, H, Hkv, Dk, Dv, dtype)
        if kind != "step":
            case.update(ragged=rng.random() < 0.4, carry=rng.random() < 0.5)
        if kind == "prompt":
            case.update(fused=rng.random() < 0.5)
        if kind == "train":
            case.update(learn=rng.random() < 0.5)
    del case["name"]
    return case


def prepare(case, seed):
    """Projections of normalised activations: unit variance; decays from fast to slow over the heads."""
    dtype = _DTYPE[case["dtype"]]
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=dtype, scale=1.0):
        return (torch.randn(*shape, device="cuda", generator=gen) * scale).to(dtype)

    if case["kind"] in ("before", "after"):
        rows, C = case["rows"], case["C"]

        def weight(mean=1.0):
            return (torch.randn(C, device="cuda", generator=gen) * 0.1 + mean).to(dtype)

        state = {"case": case, "x": randn(rows, C, scale=2.0), "weight": weight()}
        if case["kind"] == "after":
            state["gate"] = randn(rows, C) if case["gate"] else None
            state["residual"] = randn(rows, C, scale=3.0) if case["residual"] else None
            state["scale"] = weight(0.5) if case["residual"] else None
            state["next_weight"] = weight() if case["next"] else None
        if case["grad"]:
            state["upstream"] = [randn(rows, C) for _ in range(2 if case["next"] else 1)]
            for name in ("x", "weight", "gate", "residual", "scale", "next_weight"):
                if state.get(name) is not None:
                    state[name].requires_grad_(True)
        return state

    B, L, H, Hkv, Dk, Dv = (case[n] for n in ("B", "L", "H", "Hkv", "Dk", "Dv"))
    log_decay = torch.log1p(-torch.exp2(-torch.linspace(2, 9, H, dtype=torch.float64))).to("cuda", torch.float32)
    state = {"case": case, "log_decay": log_decay}
    if case["kind"] == "step":
        state.update(q=randn(B, H, Dk), k=randn(B, Hkv, Dk), v=randn(B, Hkv, Dv),
                     state=randn(B, H, Dk, Dv, dtype=torch.float32, scale=3.0))
        return state
    if case["fused"]:
        widths = (H * Dk, Hkv * Dk, Hkv * Dv)
        q, k, v = randn(B, L, sum(widths)).split(widths, dim=-1)
        state.update(q=q.unflatten(-1, (H, Dk)), k=k.unflatten(-1, (Hkv, Dk)), v=v.unflatten(-1, (Hkv, Dv)))
    else:
        state.update(q=randn(B, L, H, Dk), k=randn(B, L, Hkv, Dk), v=randn(B, L, Hkv, Dv))
    state["lengths"] = None
    if case["ragged"]:
        lengths = torch.randint(L // 8, L + 1, (B,), device="cuda", generator=gen, dtype=torch.int32)
        lengths[seed % B] = L
        state["lengths"] = lengths
    state["state"] = randn(B, H, Dk, Dv, dtype=torch.float32) if case["carry"] else None
    if case["kind"] == "train":
        state["upstream"] = [randn(B, L, H, Dv)]
        if case["carry"]:
            state["upstream"].append(randn(B, H, Dk, Dv, dtype=torch.float32, scale=0.1))
        for name in _leaves(case):
            state[name].requires_grad_(True)
    return state


def _leaves(case):
    if case["kind"] == "train":
        return ["q", "k", "v"] + (["log_decay"] if case["learn"] else []) + (["state"] if case["carry"] else [])
    names = ["x", "weight"]
    if case["kind"] == "after":
        names += (["gate"] if case["gate"] else []) + (["residual", "scale"] if case["residual"] else [])
        names += ["next_weight"] if case["next"] else []
    return names


def run(state):
    return (_run_own if own else _run_plain)(state)


# ---- the framework's operators ------------------------------------------------------------------------------------
def _run_own(state):
    from pathsig_amd import sequence

    case, kind = state["case"], state["case"]["kind"]
    if kind == "step":
        out = sequence.linear_attention_step(state["q"], state["k"], state["v"], state["log_decay"], state["state"])
        return out, state["state"]

    def forward():
        if kind in ("prompt", "train"):
            out = sequence.linear_attention(state["q"], state["k"], state["v"], state["log_decay"], state=state["state"],
                                            lengths=state["lengths"], return_state=case["carry"])
        elif kind == "before":
            out = sequence.norm_before(state["x"], state["weight"], eps=_EPS)
        else:
            out = sequence.norm_after(state["x"], state["weight"], gate=state["gate"], residual=state["residual"],
                                      scale=state["scale"], next_weight=state["next_weight"], eps=_EPS)
        return out if isinstance(out, tuple) else (out,)

    if "upstream" not in state:
        with torch.no_grad():
            return forward()
    outs = forward()
    return outs + torch.autograd.grad(outs, [state[n] for n in _leaves(case)], state["upstream"])


# ---- the same in elementary operations of 32 bits -----------------------------------------------------------------
def _run_plain(state):
    case, kind = state["case"], state["case"]["kind"]
    dtype = _DTYPE[case["dtype"]]
    if kind == "step":
        return _plain_step(state)
    args = {n: t.detach().float() if isinstance(t, torch.Tensor) and t.is_floating_point() else t for n, t in state.items()}
    grad = "upstream" in state
    if grad:
        for name in _leaves(case):
            args[name].requires_grad_(True)
    with torch.set_grad_enabled(grad):
        outs = {"before": _plain_before, "after": _plain_after}.get(kind, _plain_attention)(args)
    if not grad:
        return _rounded(outs, kind, dtype)
    leaves = _leaves(case)
    grads = torch.autograd.grad(outs, [args[n] for n in leaves], [u.float() for u in state["upstream"]])
    outs = [o.detach() for o in outs]
    return _rounded(outs, kind, dtype) + tuple(g.to(state[n].dtype) for g, n in zip(grads, leaves))


def _rounded(outs, kind, dtype):
    """The outputs in their types: a state stays in 32 bits."""
    return tuple(o if i == 1 and kind in ("prompt", "train") else o.to(dtype) for i, o in enumerate(outs))


def _plain_step(state):
    case = state["case"]
    group = case["H"] // case["Hkv"]
    q = state["q"].float() * case["Dk"] ** -0.5
    k, v = (state[n].float().repeat_interleave(group, dim=1) for n in ("k", "v"))
    new = state["state"] * state["log_decay"].exp()[:, None, None] + k[..., :, None] * v[..., None, :]
    state["state"].copy_(new)
    return (q[..., :, None] * new).sum(dim=2).to(state["q"].dtype), state["state"]


def _plain_attention(a):
    """Chunks of 64 tokens: products inside a chunk, and a state handed from chunk to chunk."""
    case = a["case"]
    B, L, H, Dk, Dv, C = (*(case[n] for n in ("B", "L", "H", "Dk", "Dv")), _CHUNK)
    group, n = H // case["Hkv"], -(-L // C)

    def chunks(t):  # (B, L, heads, D) -> (B, H, n, C, D)
        t = t.transpose(1, 2)
        if t.shape[1] != H:
            t = t.repeat_interleave(group, dim=1)
        return torch.nn.functional.pad(t, (0, 0, 0, n * C - L)).reshape(B, H, n, C, t.shape[-1])

    at = torch.arange(n * C, device="cuda")
    ends = at < L if a["lengths"] is None else at < a["lengths"][:, None]
    valid = ends.reshape(-1, 1, n, C, 1)
    q, k, v = (chunks(a[name]).where(valid, 0.0) for name in ("q", "k", "v"))
    q = q * Dk ** -0.5
    # tokens behind the end of a sequence neither decay nor add
    steps = valid[..., 0].cumsum(-1)                                       # (B or 1, 1, n, C)
    g = a["log_decay"][None, :, None, None]
    between = (steps[..., :, None] - steps[..., None, :]).tril()
    inside = (q @ k.transpose(-1, -2)) * (g[..., None] * between).exp().tril()
    out = inside @ v
    q = q * (g * steps).exp()[..., None]
    k = k * (g * (steps[..., -1:] - steps)).exp()[..., None]
    added = k.transpose(-1, -2) @ v                                        # (B, H, n, Dk, Dv)
    kept = (g[..., 0] * steps[..., -1]).exp()[..., None, None]
    held = a["state"] if a["state"] is not None else torch.zeros(B, H, Dk, Dv, device="cuda")
    starts = []
    for i in range(n):
        starts.append(held)
        held = held * kept[:, :, i] + added[:, :, i]
    out = out + q @ torch.stack(starts, dim=2)
    out = out.where(valid, 0.0).reshape(B, H, n * C, Dv)[:, :, :L].transpose(1, 2)
    return (out, held) if case["carry"] else (out,)


def _plain_norm(x, weight):
    return x / (x.square().mean(dim=-1, keepdim=True) + _EPS).sqrt() * weight


def _plain_before(a):
    return (_plain_norm(a["x"], a["weight"]),)


def _plain_after(a):
    out = _plain_norm(a["x"], a["weight"])
    if a["gate"] is not None:
        out = out * (a["gate"] / (1 + (-a["gate"]).exp()))
    if a["residual"] is not None:
        out = a["residual"] + out * a["scale"]
    return (out,) if a["next_weight"] is None else (out, _plain_norm(out, a["next_weight"]))


# ---- the definition in 64 bits ------------------------------------------------------------------------------------
def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        a = {n: t.detach().double() if isinstance(t, torch.Tensor) and t.is_floating_point() else t
             for n, t in state.items()}
        a["upstream"] = [u.double() for u in state["upstream"]] if "upstream" in state else None
        del state
        if case["kind"] == "step":
            return _exact_step(a)
        if case["kind"] in ("before", "after"):
            parts = [_exact_norms(a, slice(i, i + 4096)) for i in range(0, case["rows"], 4096)]
            names = ["y"] + (["n"] if case["next"] else []) + (_leaves(case) if case["grad"] else [])
            by_column = ("weight", "scale", "next_weight")
            return tuple(sum(p[n] for p in parts) if n in by_column else torch.cat([p[n] for p in parts]) for n in names)
        return _exact_attention(a)


def _exact_step(a):
    case = a["case"]
    B, H, group = case["B"], case["H"], case["H"] // case["Hkv"]
    out, new = torch.empty(B, H, case["Dv"], dtype=torch.float64, device="cuda"), torch.empty_like(a["state"])
    for h in range(H):
        k, v = a["k"][:, h // group], a["v"][:, h // group]
        new[:, h] = torch.exp(a["log_decay"][h]) * a["state"][:, h] + k.unsqueeze(2) * v.unsqueeze(1)
        out[:, h] = torch.bmm(a["q"][:, h].unsqueeze(1), new[:, h]).squeeze(1) / math.sqrt(case["Dk"])
    return out, new


def _exact_attention(a):
    """Every pair of tokens by itself: o_i = sum over j <= i of e^(g (i - j)) (q_i . k_j) v_j, in blocks of rows."""
    case, f64 = a["case"], torch.float64
    B, L, H, Hkv, Dk, Dv = (case[n] for n in ("B", "L", "H", "Hkv", "Dk", "Dv"))
    train = case["kind"] == "train"
    ends = [L] * B if a["lengths"] is None else a["lengths"].tolist()
    out = torch.zeros(B, L, H, Dv, dtype=f64, device="cuda")
    last = torch.zeros(B, H, Dk, Dv, dtype=f64, device="cuda")
    dq, dk, dv = (torch.zeros_like(a[n]) for n in ("q", "k", "v"))
    dg, d0 = torch.zeros(H, dtype=f64, device="cuda"), torch.zeros_like(last)
    for b in range(B):
        T = ends[b]
        for h in range(H):
            kv = h // (H // Hkv)
            q, k, v = a["q"][b, :T, h] / math.sqrt(Dk), a["k"][b, :T, kv], a["v"][b, :T, kv]
            g = a["log_decay"][h]
            at = torch.arange(T, device="cuda", dtype=f64)
            left = torch.exp(g * (T - 1 - at))[:, None]                    # decay from a token to the end
            last[b, h] = k.mT @ (left * v)
            first = None
            if a["state"] is not None:
                first = a["state"][b, h]
                since = torch.exp(g * (at + 1))[:, None]
                last[b, h] += torch.exp(g * T) * first
                out[b, :T, h] = since * (q @ first)
            if train:
                do = a["upstream"][0][b, :T, h]
                if first is not None:
                    end = a["upstream"][1][b, h]
                    pulled = since * (do @ first.mT)
                    dq[b, :T, h] += pulled
                    d0[b, h] = (since * q).mT @ do + torch.exp(g * T) * end
                    dk[b, :T, kv] += left * (v @ end.mT)
                    dv[b, :T, kv] += left * (k @ end)
                    dg[h] += ((at + 1)[:, None] * pulled * q).sum() + T * torch.exp(g * T) * (first * end).sum()
                    dg[h] += ((T - 1 - at)[:, None] * left * (k @ end) * v).sum()
            for i in range(0, T, 2048):
                rows = slice(i, min(T, i + 2048))
                cols = slice(0, rows.stop)
                gap = at[rows, None] - at[None, cols]
                decay = torch.exp(g * gap.clamp(min=0)).masked_fill_(gap < 0, 0.0)
                weights = (q[rows] @ k[cols].mT) * decay
                out[b, rows, h] += weights @ v[cols]
                if train:
                    dv[b, cols, kv] += weights.mT @ do[rows]
                    pulls = do[rows] @ v[cols].mT
                    if case["learn"]:
                        dg[h] += (gap * weights * pulls).sum()
                    pulls *= decay
                    dq[b, rows, h] += pulls @ k[cols]
                    dk[b, cols, kv] += pulls.mT @ q[rows]
    outs = (out, last) if case["carry"] else (out,)
    if not train:
        return outs
    outs += (dq / math.sqrt(Dk), dk, dv)
    return outs + ((dg,) if case["learn"] else ()) + ((d0,) if case["carry"] else ())


def _exact_norms(a, rows):
    case = a["case"]
    x, w, C = a["x"][rows], a["weight"], case["C"]
    inv = torch.rsqrt((x * x).sum(-1, keepdim=True) / C + _EPS)
    unit = x * inv
    u = s = None
    part = {"y": unit * w}
    if case["gate"]:
        gate = a["gate"][rows]
        sig = torch.sigmoid(gate)
        u = gate * sig
        part["y"] = part["y"] * u
    joined = part["y"]
    if case["residual"]:
        s = a["scale"]
        part["y"] = a["residual"][rows] + s * joined
    if case["next"]:
        inv2 = torch.rsqrt((part["y"] ** 2).sum(-1, keepdim=True) / C + _EPS)
        unit2 = part["y"] * inv2
        part["n"] = unit2 * a["next_weight"]
    if not case["grad"]:
        return part
    d = a["upstream"][0][rows]
    if case["next"]:
        dn = a["upstream"][1][rows]
        part["next_weight"] = (dn * unit2).sum(0)
        dn = dn * a["next_weight"]
        d = d + inv2 * (dn - unit2 * (dn * unit2).sum(-1, keepdim=True) / C)
    if case["residual"]:
        part["residual"] = d
        part["scale"] = (d * joined).sum(0)
        d = d * s
    if case["gate"]:
        part["gate"] = d * (unit * w) * (sig + gate * sig * (1 - sig))
        d = d * u
    part["weight"] = (d * unit).sum(0)
    d = d * w
    part["x"] = inv * (d - unit * (d * unit).sum(-1, keepdim=True) / C)
    return part


def work(case):
    """Bytes: inputs once, outputs once.  Flops of the attention: the recurrence, 4 Dk Dv a token and head, and in a step
    of training the same for the state once more and 8 Dk Dv for the gradients.  Norms: a handful for each element."""
    e = 2 if case["dtype"] == "bf16" else 4
    if case["kind"] in ("before", "after"):
        full = 2 + case["gate"] + case["residual"] + case["next"]
        if case["grad"]:  # the gradients from above and those of the inputs
            full += 1 + case["next"] + 1 + case["gate"] + case["residual"]
        columns = (1 + case["residual"] + case["next"]) * (1 + case["grad"])
        return {"bytes": e * (full * case["rows"] + columns) * case["C"],
                "flops": (30.0 if case["grad"] else 10.0) * case["rows"] * case["C"]}
    B, L, H, Hkv, Dk, Dv = (case[n] for n in ("B", "L", "H", "Hkv", "Dk", "Dv"))
    tokens = B * L * (1 - 7 / 16 * case["ragged"])
    read = tokens * (H * Dk + Hkv * (Dk + Dv))
    values = read + B * L * H * Dv
    states = 4.0 * B * H * Dk * Dv
    if case["kind"] == "step":
        return {"bytes": e * values + 2 * states, "flops": 5.0 * B * H * Dk * Dv}
    if case["kind"] == "prompt":
        return {"bytes": e * values + 2 * states * case["carry"], "flops": 4.0 * tokens * H * Dk * Dv}
    values += read + tokens * H * Dv + B * L * (H * Dk + Hkv * (Dk + Dv))
    return {"bytes": e * values + 4 * states * case["carry"], "flops": 14.0 * tokens * H * Dk * Dv}
