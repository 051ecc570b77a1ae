"""Sequence operators without a GPU: schemas, shapes of meta tensors, refusals of the wrappers, the modules' arguments, and the
argument checks of the C ABI, which come before anything is launched."""
from __future__ import annotations

import ctypes

import pytest
import torch

import pathsig_amd as ps
from pathsig_amd import _load, sequence

ERR_ARG, ERR_UNSUPPORTED, ERR_WORKSPACE = -1, -2, -3


@pytest.fixture(scope="module")
def lib():
    return _load.lib()


def _meta(*shape, dtype=torch.float32):
    return torch.empty(*shape, dtype=dtype, device="meta")


def test_submodule_is_reached_from_the_package():
    assert ps.sequence is sequence
    for name in sequence.__all__:
        assert hasattr(sequence, name)
    for op in ("linear_attention", "linear_attention_backward", "linear_attention_step", "norm_join", "norm_join_backward"):
        assert torch.Tag.pt2_compliant_tag in getattr(torch.ops.pathsig, op).default.tags


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_meta_shapes_of_attention(dtype):
    B, L, H, Hkv, Dk, Dv = 3, 17, 6, 2, 24, 40
    q, k, v = _meta(B, L, H, Dk, dtype=dtype), _meta(B, L, Hkv, Dk, dtype=dtype), _meta(B, L, Hkv, Dv, dtype=dtype)
    g, state, lengths = _meta(H), _meta(B, H, Dk, Dv), _meta(B, dtype=torch.int64)
    out, last = sequence.linear_attention(q, k, v, g, state=state, lengths=lengths, return_state=True)
    assert out.shape == (B, L, H, Dv) and out.dtype == dtype
    assert last.shape == (B, H, Dk, Dv) and last.dtype == torch.float32
    grads = torch.ops.pathsig.linear_attention_backward(out, last, q, k, v, g, state, lengths, 1.0, True, True)
    assert [tuple(t.shape) for t in grads] == [tuple(t.shape) for t in (q, k, v, g, state)]
    assert [t.dtype for t in grads] == [dtype] * 3 + [torch.float32] * 2
    grads = torch.ops.pathsig.linear_attention_backward(out, None, q, k, v, g, None, None, 1.0, False, False)
    assert grads[3].numel() == 0 and grads[4].numel() == 0
    step = sequence.linear_attention_step(q[:, 0], k[:, 0], v[:, 0], g, state)
    assert step.shape == (B, H, Dv) and step.dtype == dtype


def test_meta_gradients_reach_every_leaf():
    q, k, v, g, s = (t.requires_grad_(True) for t in (_meta(2, 5, 4, 8), _meta(2, 5, 2, 8), _meta(2, 5, 2, 12), _meta(4),
                                                       _meta(2, 4, 8, 12)))
    out, last = sequence.linear_attention(q, k, v, g, state=s, return_state=True)
    grads = torch.autograd.grad((out.sum() + last.sum(),), (q, k, v, g, s))
    assert [x.shape for x in grads] == [x.shape for x in (q, k, v, g, s)]
    x, w, gate, scale, nw = (t.requires_grad_(True) for t in (_meta(2, 5, 16), _meta(16), _meta(2, 1, 16), _meta(16), _meta(16)))
    r = _meta(5, 16).requires_grad_(True)
    out, nxt = sequence.norm_after(x, w, gate=gate, residual=r, scale=scale, next_weight=nw)
    leaves = (x, w, gate, r, scale, nw)
    grads = torch.autograd.grad((out.sum() + nxt.sum(),), leaves)
    assert [t.shape for t in grads] == [t.shape for t in leaves]
    (grad,) = torch.autograd.grad(sequence.norm_before(x).sum(), x)
    assert grad.shape == x.shape


@pytest.mark.parametrize("edit", [
    dict(k=(2, 5, 3, 8)), dict(k=(2, 5, 2, 9)), dict(v=(2, 5, 1, 12)), dict(v=(2, 6, 2, 12)), dict(g=(5,)), dict(state=(2, 4, 8, 11)),
    dict(lengths=(3,)), dict(q=(2, 5, 4, 257), k=(2, 5, 2, 257)), dict(q=(2, 5, 4))])
def test_meta_refuses_shapes_that_do_not_fit(edit):
    shapes = dict(q=(2, 5, 4, 8), k=(2, 5, 2, 8), v=(2, 5, 2, 12), g=(4,), state=(2, 4, 8, 12), lengths=(2,))
    shapes.update(edit)
    t = {n: _meta(*s, dtype=torch.int32 if n == "lengths" else torch.float32) for n, s in shapes.items()}
    with pytest.raises((RuntimeError, IndexError)):
        sequence.linear_attention(t["q"], t["k"], t["v"], t["g"], state=t["state"], lengths=t["lengths"])


def test_types_that_are_refused():
    q = _meta(2, 5, 4, 8)
    for bad in (torch.float16, torch.float64):
        with pytest.raises(RuntimeError, match="float32 or bfloat16"):
            sequence.linear_attention(q.to(bad), q.to(bad), q.to(bad), _meta(4))
        with pytest.raises(RuntimeError, match="float32 or bfloat16"):
            sequence.norm_before(q.to(bad))
    with pytest.raises(RuntimeError):
        sequence.linear_attention(q, q.to(torch.bfloat16), q, _meta(4))
    with pytest.raises(RuntimeError):
        sequence.linear_attention(q, q, q, _meta(4, dtype=torch.bfloat16))
    with pytest.raises(RuntimeError):
        sequence.norm_before(q, _meta(8, dtype=torch.bfloat16))  # parameters: float32 or the type of x
    with pytest.raises(RuntimeError, match="one dtype"):
        x = q.to(torch.bfloat16)
        sequence.norm_after(x, _meta(8), scale=_meta(8, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="activation"):
        sequence.norm_after(q, activation="tanh")
    with pytest.raises(RuntimeError):
        sequence.norm_before(_meta(3, 8193))


def test_tensors_on_the_cpu_are_refused():
    q = torch.zeros(2, 5, 4, 8)
    with pytest.raises((RuntimeError, NotImplementedError)):
        sequence.linear_attention(q, q, q, torch.zeros(4))
    with pytest.raises((RuntimeError, NotImplementedError)):
        sequence.norm_before(q)


def test_step_refuses_a_gradient():
    q = _meta(2, 4, 8).requires_grad_(True)
    with pytest.raises(RuntimeError, match="no gradient"):
        sequence.linear_attention_step(q, q.detach(), q.detach(), _meta(4), _meta(2, 4, 8, 8))
    with torch.no_grad():
        assert sequence.linear_attention_step(q, q, q, _meta(4), _meta(2, 4, 8, 8)).shape == (2, 4, 8)


# ---- C ABI ----------------------------------------------------------------------------------------------------------
def _attention(**edit):
    c = _load.LinearAttentionCall(dtype=2, B=2, L=300, H=4, Hkv=2, Dk=8, Dv=12, scale=1.0, learned_decay=0, log_decay=1, lengths=None)
    c.q_stride[:] = (300 * 32, 32, 8)
    c.k_stride[:] = (300 * 16, 16, 8)
    c.v_stride[:] = (300 * 24, 24, 12)
    for name, value in edit.items():
        if name.endswith("_stride"):
            getattr(c, name)[:] = value
        else:
            setattr(c, name, value)
    return c


def _forward(lib, call, q=1, out=1, ws=0, ws_bytes=0):
    ref = ctypes.byref(call) if call is not None else None
    return lib.pathsig_linattn_forward(ref, q, 1, 1, None, out, None, ws, ws_bytes, None)


@pytest.mark.parametrize("edit,code", [
    (dict(dtype=1), ERR_ARG), (dict(dtype=7), ERR_ARG), (dict(B=-1), ERR_ARG), (dict(L=-1), ERR_ARG), (dict(Hkv=3), ERR_ARG),
    (dict(Hkv=0), ERR_ARG), (dict(H=0), ERR_ARG), (dict(Dk=0), ERR_ARG), (dict(Dv=0), ERR_ARG), (dict(Dk=257), ERR_UNSUPPORTED),
    (dict(Dv=300), ERR_UNSUPPORTED), (dict(B=70000), ERR_UNSUPPORTED), (dict(H=70000, Hkv=70000), ERR_UNSUPPORTED),
    (dict(L=2 ** 31), ERR_UNSUPPORTED), (dict(log_decay=None), ERR_ARG), (dict(q_stride=(-1, 32, 8)), ERR_ARG),
    (dict(k_stride=(10 ** 10, 2 ** 25, 8)), ERR_UNSUPPORTED)])
def test_attention_refuses_bad_calls(lib, edit, code):
    assert _forward(lib, _attention(**edit)) == code
    assert lib.pathsig_last_error()
    assert lib.pathsig_linattn_forward_workspace(ctypes.byref(_attention(**edit))) == 0
    if edit.get("L") is None:
        assert lib.pathsig_linattn_step(ctypes.byref(_attention(L=1, **edit)), 1, 1, 1, 1, 1, None) == code


def test_attention_refuses_missing_buffers(lib):
    assert _forward(lib, None) == ERR_ARG
    assert _forward(lib, _attention(), q=None) == ERR_ARG and b"NULL" in lib.pathsig_last_error()
    assert _forward(lib, _attention(), out=None) == ERR_ARG
    long = _attention(L=65536)
    need = lib.pathsig_linattn_forward_workspace(ctypes.byref(long))
    assert need > 0
    assert _forward(lib, long) == ERR_WORKSPACE and b"workspace" in lib.pathsig_last_error()
    assert _forward(lib, long, ws=256, ws_bytes=need - 1) == ERR_WORKSPACE
    back = lib.pathsig_linattn_backward
    call = _attention(L=65536)
    ref = ctypes.byref(call)
    assert back(ref, 1, 1, 1, None, None, 0, 1, None, 1, 1, 1, None, None, None, 0, None) == ERR_WORKSPACE
    assert back(ref, 1, 1, 1, None, None, 0, None, None, 1, 1, 1, None, None, None, 0, None) == ERR_ARG
    assert back(ref, 1, 1, 1, None, 256, need - 1, 1, None, 1, 1, 1, None, None, None, 0, None) == ERR_ARG
    assert b"kept" in lib.pathsig_last_error()
    assert back(ref, 1, 1, 1, None, None, 0, 1, None, 1, 1, 1, 1, None, None, 0, None) == ERR_ARG
    assert b"learned_decay" in lib.pathsig_last_error()
    step = lib.pathsig_linattn_step
    assert step(ctypes.byref(_attention()), 1, 1, 1, 1, 1, None) == ERR_ARG and b"one token" in lib.pathsig_last_error()
    assert step(ctypes.byref(_attention(L=1, lengths=1)), 1, 1, 1, 1, 1, None) == ERR_ARG
    assert step(ctypes.byref(_attention(L=1)), 1, 1, 1, None, 1, None) == ERR_ARG
    # nothing to do
    assert _forward(lib, _attention(B=0), q=None, out=None) == 0
    assert step(ctypes.byref(_attention(L=1, B=0)), None, None, None, None, None, None) == 0


def _norm(**edit):
    fields = dict(dtype=2, param_dtype=0, activation=0, rows=5, C=16, x_stride=16, gate_stride=16, residual_stride=16, eps=1e-6, x=256,
                  gate=None, residual=None, weight=None, scale=None, next_weight=None)
    fields.update(edit)
    return _load.NormCall(**fields)


@pytest.mark.parametrize("edit,code", [
    (dict(dtype=1), ERR_ARG), (dict(param_dtype=1), ERR_ARG), (dict(dtype=0, param_dtype=2), ERR_ARG), (dict(activation=3), ERR_ARG),
    (dict(activation=-1), ERR_ARG), (dict(rows=-1), ERR_ARG), (dict(C=0), ERR_ARG), (dict(x_stride=-1), ERR_ARG),
    (dict(eps=-1.0), ERR_ARG), (dict(eps=float("nan")), ERR_ARG), (dict(C=8193), ERR_UNSUPPORTED), (dict(rows=2 ** 40, C=8192), ERR_UNSUPPORTED),
    (dict(x=None), ERR_ARG)])
def test_norms_refuse_bad_calls(lib, edit, code):
    assert lib.pathsig_norm_forward(ctypes.byref(_norm(**edit)), 256, None, None, None) == code
    assert lib.pathsig_last_error()
    assert lib.pathsig_norm_backward(ctypes.byref(_norm(**edit)), 256, 256, None, 256, None, None, None, None, None, None, 0,
                                     None) == code


def test_norms_refuse_missing_buffers(lib):
    call = _norm()
    ref = ctypes.byref(call)
    assert lib.pathsig_norm_forward(None, 256, None, None, None) == ERR_ARG
    assert lib.pathsig_norm_forward(ref, None, None, None, None) == ERR_ARG
    back = lib.pathsig_norm_backward
    need = lib.pathsig_norm_backward_workspace(ref)
    assert need > 0
    assert back(ref, None, 256, None, 256, None, None, None, None, None, None, 0, None) == ERR_ARG  # no statistics
    assert back(ref, 256, 256, None, 256, None, None, 256, None, None, None, 0, None) == ERR_WORKSPACE
    assert back(ref, 256, 256, None, 256, None, None, 256, None, None, 256, need - 1, None) == ERR_WORKSPACE
    assert back(ref, 256, 256, None, 256, 256, None, None, None, None, None, 0, None) == ERR_ARG  # a gradient of no gate
    assert b"gate" in lib.pathsig_last_error()
    assert lib.pathsig_norm_forward(ctypes.byref(_norm(rows=0, x=None)), None, None, None, None) == 0
