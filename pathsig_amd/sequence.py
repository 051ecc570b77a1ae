"""Layers of sequence models over (B, L, ...) features, e.g. the (log-)signatures of sliding windows of a path: linear
attention with a decay for each head, and the norms before and after a block with its gate and residual scale.

Linear attention carries S_t = exp(log_decay) S_(t-1) + k_t v_t^T along a sequence and answers scale * S_t^T q_t.  It is the
signatures' kind of operator: with no decay, k_t = x_(t-1) - x_0 + dx_t / 2 and v_t = dx_t, the last state is the second level
of the signature of x; a decay lets the far past fade.  The reference has no counterpart of this module.
"""
from __future__ import annotations

import torch
from torch import Tensor, nn

from . import _load

__all__ = ["linear_attention", "linear_attention_step", "norm_before", "norm_after", "LinearAttention", "NormBefore",
           "NormAfter"]

_ACTIVATIONS = {"silu": 0, "sigmoid": 1, "linear": 2}
_MAX_HEAD_DIM = 256
_MAX_CHANNELS = 8192
_direct = _load.direct
_ops = torch.ops.pathsig
_is_compiling = torch.compiler.is_compiling


# ------------------------------------------------------------------------------------------------
# functions
# ------------------------------------------------------------------------------------------------
def linear_attention(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, *, state: Tensor | None = None,
                     lengths: Tensor | None = None, scale: float | None = None, return_state: bool = False):
    """S_t = exp(log_decay) S_(t-1) + k_t v_t^T and out_t = scale * S_t^T q_t for whole sequences, differentiable in q, k, v,
    log_decay and state.

    q (B, L, H, Dk), k (B, L, Hkv, Dk), v (B, L, Hkv, Dv), float32 or bfloat16; H is a multiple of Hkv, and H / Hkv heads of
    queries share a head of keys and values.  log_decay (H,) float32.  state (B, H, Dk, Dv) float32: S before the first token
    (zero if not given).  lengths (B,) int32 or int64: tokens from there on are padding, which is neither read nor answered
    (zeros).  scale: 1 / sqrt(Dk) if not given.

    Returns out (B, L, H, Dv), with `return_state` also S after the last token of every sequence, (B, H, Dk, Dv) float32.
    """
    scale = max(q.shape[-1], 1) ** -0.5 if scale is None else float(scale)
    return_state = bool(return_state)
    if not _is_compiling():
        out = _direct.linear_attention(q, k, v, log_decay, state, lengths, scale, return_state)
        if out is not None:
            return out
    out, last = _ops.linear_attention.default(q, k, v, log_decay, state, lengths, scale, return_state)
    return (out, last) if return_state else out


def linear_attention_step(q: Tensor, k: Tensor, v: Tensor, log_decay: Tensor, state: Tensor, *,
                          scale: float | None = None) -> Tensor:
    """One token of every sequence: q (B, H, Dk), k (B, Hkv, Dk), v (B, Hkv, Dv); `state`, contiguous (B, H, Dk, Dv) float32,
    is updated in place.  Returns (B, H, Dv).  No gradient."""
    scale = max(q.shape[-1], 1) ** -0.5 if scale is None else float(scale)
    if not _is_compiling():
        out = _direct.linear_attention_step(q, k, v, log_decay, state, scale)
        if out is not None:
            return out
    return _ops.linear_attention_step.default(q, k, v, log_decay, state, scale)


def norm_before(x: Tensor, weight: Tensor | None = None, *, eps: float = 1e-6) -> Tensor:
    """x / sqrt(mean(x^2) + eps) * weight over the last axis: the norm in front of a block."""
    if not _is_compiling():
        out = _direct.norm_join(x, weight, None, None, None, None, float(eps), 0)
        if out is not None:
            return out
    return _ops.norm_join.default(x, weight, None, None, None, None, float(eps), 0, _wants_grad(x, weight))[0]


def norm_after(x: Tensor, weight: Tensor | None = None, *, gate: Tensor | None = None, residual: Tensor | None = None,
               scale: Tensor | None = None, next_weight: Tensor | None = None, eps: float = 1e-6,
               activation: str = "silu"):
    """What follows a block with output x, in one pass over it:

        out  = residual + scale * (x / sqrt(mean(x^2) + eps) * weight * act(gate))
        next = out / sqrt(mean(out^2) + eps) * next_weight         (the norm in front of the next block)

    x (..., C), float32 or bfloat16; gate and residual in its dtype, broadcast to its shape; weight, scale and next_weight (C,) in one
    dtype, float32 or that of x.  What is not given is left out.  activation: "silu", "sigmoid" or "linear".
    Returns out, with `next_weight` (out, next).
    """
    try:
        code = _ACTIVATIONS[activation]
    except KeyError:
        raise ValueError(f"activation must be one of {', '.join(map(repr, _ACTIVATIONS))}") from None
    if gate is not None and gate.shape != x.shape:
        gate = gate.expand(x.shape)
    if residual is not None and residual.shape != x.shape:
        residual = residual.expand(x.shape)
    if not _is_compiling():
        out = _direct.norm_join(x, weight, gate, residual, scale, next_weight, float(eps), code)
        if out is not None:
            return out
    out, normed, _ = _ops.norm_join.default(x, weight, gate, residual, scale, next_weight, float(eps), code,
                                            _wants_grad(x, weight, gate, residual, scale, next_weight))
    return out if next_weight is None else (out, normed)


def _wants_grad(*tensors) -> bool:
    return torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in tensors)


# ------------------------------------------------------------------------------------------------
# modules
# ------------------------------------------------------------------------------------------------
class LinearAttention(nn.Module):
    """`linear_attention` with the decays of its heads: exp(log_decay) = 1 - 2^-e with e spread evenly over [first, last] (the
    memory of a head is about 2^e tokens), or as given.  `learn_decay` makes them a parameter.  They stay float32 where the module
    is converted to another type."""

    def __init__(self, *, num_heads: int, log_decay=None, decay_exponents=(2.0, 9.0), learn_decay: bool = False, scale=None):
        super().__init__()
        if num_heads < 1:
            raise ValueError("num_heads must be at least 1.")
        if log_decay is None:
            first, last = decay_exponents
            if not (first > 0 and last > 0):
                raise ValueError("decay_exponents must be positive.")
            log_decay = torch.log1p(-torch.exp2(-torch.linspace(first, last, num_heads, dtype=torch.float64)))
        log_decay = torch.as_tensor(log_decay).detach().to(device="cuda", dtype=torch.float32).clone()
        if log_decay.shape != (num_heads,):
            raise ValueError("log_decay must hold one value for each head.")
        self.num_heads = num_heads
        self.scale = scale
        if learn_decay:
            self.log_decay = nn.Parameter(log_decay)
        else:
            self.register_buffer("log_decay", log_decay)

    def _apply(self, fn, recurse=True):
        # (a slow decay in bfloat16 would be none: 1 - 2^-9 rounds to 1)
        decays = self._parameters.get("log_decay", self._buffers.get("log_decay"))
        held = () if decays is None else (decays, decays.grad)

        def keep_float(t):
            new = fn(t)
            if new.dtype == t.dtype or not any(t is h for h in held):
                return new
            return t.to(new.device)
        return super()._apply(keep_float, recurse)

    def forward(self, q, k, v, *, state=None, lengths=None, return_state=False):
        return linear_attention(q, k, v, self.log_decay, state=state, lengths=lengths, scale=self.scale,
                                return_state=return_state)

    def step(self, q, k, v, state):
        return linear_attention_step(q, k, v, self.log_decay, state, scale=self.scale)

    def new_state(self, batch: int, key_dim: int, value_dim: int) -> Tensor:
        """A state before the first token."""
        return torch.zeros(batch, self.num_heads, key_dim, value_dim, dtype=torch.float32, device=self.log_decay.device)


class NormBefore(nn.Module):
    """`norm_before` with its weight."""

    def __init__(self, *, channels: int, eps: float = 1e-6, dtype=torch.float32):
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(channels, dtype=dtype, device="cuda"))

    def forward(self, x):
        return norm_before(x, self.weight, eps=self.eps)


class NormAfter(nn.Module):
    """`norm_after` with its weight, with `residual_scale` (a number: the scale of every channel at the start, learned) and
    with `next_norm` the weight of the norm in front of the next block."""

    def __init__(self, *, channels: int, residual_scale: float | None = None, next_norm: bool = False, activation: str = "silu",
                 eps: float = 1e-6, dtype=torch.float32):
        super().__init__()
        if activation not in _ACTIVATIONS:
            raise ValueError(f"activation must be one of {', '.join(map(repr, _ACTIVATIONS))}")
        self.eps = eps
        self.activation = activation
        self.weight = nn.Parameter(torch.ones(channels, dtype=dtype, device="cuda"))
        full = torch.full((channels,), 1.0 if residual_scale is None else float(residual_scale), dtype=dtype, device="cuda")
        self.scale = None if residual_scale is None else nn.Parameter(full)
        self.next_weight = nn.Parameter(torch.ones(channels, dtype=dtype, device="cuda")) if next_norm else None

    def forward(self, x, *, gate=None, residual=None):
        return norm_after(x, self.weight, gate=gate, residual=residual, scale=self.scale, next_weight=self.next_weight,
                          eps=self.eps, activation=self.activation)


# ------------------------------------------------------------------------------------------------
# shape inference for fake / meta tensors
# ------------------------------------------------------------------------------------------------
_library = torch.library.Library("pathsig", "FRAGMENT")


def _on_device(t: Tensor) -> bool:
    return t.device.type in ("cuda", "meta")


def _check_sequence(t: Tensor, what: str) -> None:
    torch._check(_on_device(t), lambda: f"{what} must be a CUDA tensor")
    torch._check(t.dtype in (torch.float32, torch.bfloat16), lambda: f"{what} must be float32 or bfloat16")


def _attention_dims(q, k, v, log_decay, state, lengths, dims):
    _check_sequence(q, "q")
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        torch._check(t.dim() == dims, lambda: f"{name} must have {dims} dimensions")
        torch._check(_on_device(t) and t.dtype == q.dtype, lambda: f"{name} must have same dtype and device as q")
        torch._check(tuple(t.shape[:dims - 2]) == tuple(q.shape[:dims - 2]),
                     lambda: f"{name} must have as many sequences and tokens as q")
    H, Hkv, Dk, Dv = q.shape[-2], k.shape[-2], q.shape[-1], v.shape[-1]
    torch._check(v.shape[-2] == Hkv, lambda: "k and v must have the same number of heads")
    torch._check(k.shape[-1] == Dk, lambda: "k must have as many channels as q")
    torch._check(H >= 1 and Hkv >= 1 and H % Hkv == 0, lambda: "the heads of q must be a multiple of those of k and v")
    torch._check(1 <= Dk <= _MAX_HEAD_DIM and 1 <= Dv <= _MAX_HEAD_DIM, lambda: f"heads have 1 to {_MAX_HEAD_DIM} channels")
    torch._check(log_decay.dtype == torch.float32 and tuple(log_decay.shape) == (H,), lambda: "log_decay must be (H,) float32")
    if state is not None:
        torch._check(state.dtype == torch.float32 and tuple(state.shape) == (q.shape[0], H, Dk, Dv),
                     lambda: "state must be (B, H, Dk, Dv) float32")
    if lengths is not None:
        torch._check(lengths.dtype in (torch.int32, torch.int64) and tuple(lengths.shape) == (q.shape[0],),
                     lambda: "lengths must be (B,) int32 or int64")
    return H, Hkv, Dk, Dv


@torch.library.register_fake("pathsig::linear_attention", lib=_library)
def _linear_attention_fake(q, k, v, log_decay, state, lengths, scale, return_state):
    H, _, Dk, Dv = _attention_dims(q, k, v, log_decay, state, lengths, 4)
    shape = (q.shape[0], H, Dk, Dv) if return_state else (0,)
    return q.new_empty((*q.shape[:2], H, Dv)), q.new_empty(shape, dtype=torch.float32)


@torch.library.register_fake("pathsig::linear_attention_backward", lib=_library)
def _linear_attention_backward_fake(grad_out, grad_state, q, k, v, log_decay, state, lengths, scale, want_log_decay,
                                    want_state):
    H, _, Dk, Dv = _attention_dims(q, k, v, log_decay, state, lengths, 4)
    torch._check(tuple(grad_out.shape) == (*q.shape[:2], H, Dv), lambda: "grad_out must be (B, L, H, Dv)")
    shape = (q.shape[0], H, Dk, Dv) if want_state else (0,)
    return (q.new_empty(q.shape), q.new_empty(k.shape), q.new_empty(v.shape),
            q.new_empty((H if want_log_decay else 0,), dtype=torch.float32), q.new_empty(shape, dtype=torch.float32))


@torch.library.register_fake("pathsig::linear_attention_step", lib=_library)
def _linear_attention_step_fake(q, k, v, log_decay, state, scale):
    H, _, _, Dv = _attention_dims(q, k, v, log_decay, state, None, 3)
    return q.new_empty((q.shape[0], H, Dv))


def _norm_dims(x, weight, gate, residual, scale, next_weight):
    _check_sequence(x, "x")
    torch._check(x.dim() >= 1 and 1 <= x.shape[-1] <= _MAX_CHANNELS, lambda: f"x must have 1 to {_MAX_CHANNELS} channels")
    for t, name in ((gate, "gate"), (residual, "residual")):
        if t is not None:
            torch._check(t.dtype == x.dtype and tuple(t.shape) == tuple(x.shape),
                         lambda: f"{name} must have the dtype and shape of x")
    params = [t for t in (weight, scale, next_weight) if t is not None]
    for t in params:
        torch._check(tuple(t.shape) == (x.shape[-1],), lambda: "weight, scale and next_weight must be (C,)")
        torch._check(t.dtype in (torch.float32, x.dtype), lambda: "parameters must be float32 or have the dtype of x")
        torch._check(t.dtype == params[0].dtype, lambda: "weight, scale and next_weight must have one dtype")
    return params[0].dtype if params else x.dtype


@torch.library.register_fake("pathsig::norm_join", lib=_library)
def _norm_join_fake(x, weight, gate, residual, scale, next_weight, eps, activation, keep):
    _norm_dims(x, weight, gate, residual, scale, next_weight)
    return (x.new_empty(x.shape), x.new_empty(x.shape if next_weight is not None else (0,)),
            x.new_empty((2 if keep else 0, x.numel() // x.shape[-1]), dtype=torch.float32))


@torch.library.register_fake("pathsig::norm_join_backward", lib=_library)
def _norm_join_backward_fake(grad_out, grad_next, x, weight, gate, residual, scale, next_weight, statistics, eps, activation):
    dtype = _norm_dims(x, weight, gate, residual, scale, next_weight)

    def like(t):
        return x.new_empty(x.shape if t is not None else (0,))

    def column(t):
        return x.new_empty((x.shape[-1] if t is not None else 0,), dtype=dtype)

    return x.new_empty(x.shape), column(weight), like(gate), like(residual), column(scale), column(next_weight)
