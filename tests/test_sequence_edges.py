"""Sequence operators at the edges of what their documents allow, without a GPU: buffers that a call of the C ABI must not share,
gradients of gradients, modules in other types."""
from __future__ import annotations

import ctypes

import pytest
import torch

from pathsig_amd import _load, sequence

ERR_ARG, ERR_WORKSPACE = -1, -3


@pytest.fixture(autouse=True)
def float32_by_default():
    """Tensors made here without a type are float32, whatever the tests before left as the default."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)


@pytest.fixture(scope="module")
def lib():
    return _load.lib()


def _attention(**edit):
    c = _load.LinearAttentionCall(dtype=2, B=2, L=300, H=4, Hkv=2, Dk=8, Dv=16, scale=1.0, learned_decay=0, log_decay=1, lengths=None)
    c.q_stride[:] = (300 * 32, 32, 8)
    c.k_stride[:] = (300 * 16, 16, 8)
    c.v_stride[:] = (300 * 32, 32, 16)
    for name, value in edit.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("state,above", [(None, 512), (512, None), (512, 512)])
def test_gradient_of_the_state_over_what_is_read(lib, state, above):
    """The gradient of the state in the place of the state or of the gradient from above: both are read after it is written."""
    rc = lib.pathsig_linattn_backward(ctypes.byref(_attention()), 256, 256, 256, state, None, 0, 256, above, 256, 256, 256, None, 512, None, 0,
                                      None)
    assert rc == ERR_ARG and b"grad_state" in lib.pathsig_last_error()


def test_gradients_that_are_not_wanted_may_be_missing(lib):
    """Their buffers are not asked for; the gradient of the state is worked out with that of the values."""
    call = _attention(L=65536)
    need = lib.pathsig_linattn_backward_workspace(ctypes.byref(call), 0)
    for grads in ((None, None, None), (256, None, None), (None, 256, None), (None, None, 256)):
        rc = lib.pathsig_linattn_backward(ctypes.byref(call), 256, 256, 256, None, None, 0, 256, None, *grads, None, None, 256, need - 1, None)
        assert rc == ERR_WORKSPACE  # (nothing is launched; missing buffers would be named before)
    rc = lib.pathsig_linattn_backward(ctypes.byref(call), 256, 256, 256, None, None, 0, 256, None, 256, 256, None, None, 512, 256, need, None)
    assert rc == ERR_ARG and b"grad_v" in lib.pathsig_last_error()


def _meta(*shape):
    return torch.empty(*shape, device="meta", requires_grad=True)


def _attention_out():
    q, k, v, g, s = _meta(2, 5, 4, 8), _meta(2, 5, 2, 8), _meta(2, 5, 2, 12), _meta(4), _meta(2, 4, 8, 12)
    return (q, k, v, g, s), sequence.linear_attention(q, k, v, g, state=s)


def _after_out():
    x, w, gate, r, s, nw = _meta(6, 16), _meta(16), _meta(6, 16), _meta(6, 16), _meta(16), _meta(16)
    return (x, w, gate, s, nw, r), sequence.norm_after(x, w, gate=gate, residual=r, scale=s, next_weight=nw)[1]


def _before_out():
    x, w = _meta(6, 16), _meta(16)
    return (x, w), sequence.norm_before(x, w)


@pytest.mark.parametrize("make", [_attention_out, _after_out, _before_out])
def test_gradients_of_gradients_are_refused(make):
    """A penalty on a gradient, which reaches the leaves through the output as well."""
    leaves, out = make()
    grads = torch.autograd.grad(out.sum(), leaves, create_graph=True)
    for grad in grads:
        penalty = out.sum() + grad.pow(2).sum()
        with pytest.raises(RuntimeError, match="not implemented"):
            penalty.backward(retain_graph=True)
    leaves, out = make()
    assert not any(grad.requires_grad for grad in torch.autograd.grad(out.sum(), leaves))


@pytest.mark.parametrize("learn", [False, True])
def test_decays_stay_float32_in_a_module_of_another_type(learn):
    """Conversions of a whole model leave the decays' values and type alone, alone or within another module, and their gradient."""
    class OnTheHost(sequence.LinearAttention):
        def __init__(self):
            torch.nn.Module.__init__(self)
            self.num_heads, self.scale = 3, None
            self.inner = torch.nn.Linear(4, 4)
            if learn:
                self.log_decay = torch.nn.Parameter(torch.tensor([-0.5, -2.0 ** -9, -1e-5]))
                self.log_decay.grad = torch.tensor([1.0, 1 + 2.0 ** -20, 3.0])
            else:
                self.register_buffer("log_decay", torch.tensor([-0.5, -2.0 ** -9, -1e-5]))

    for convert in (lambda m: m.bfloat16(), lambda m: m.half(), lambda m: m.to(torch.bfloat16), lambda m: m.to("cpu", torch.float64),
                    lambda m: m.type(torch.bfloat16), lambda m: m.float(), lambda m: m.bfloat16().float()):
        attend, other = OnTheHost(), torch.nn.Linear(4, 4)
        want, leaf = attend.log_decay.detach().clone(), attend.log_decay
        convert(torch.nn.Sequential(other, attend))
        assert attend.log_decay.dtype == torch.float32 and torch.equal(attend.log_decay, want)
        assert attend.inner.weight.dtype == other.weight.dtype
        assert ("log_decay" in dict(attend.named_parameters())) == learn and "log_decay" in attend.state_dict()
        if learn:
            assert attend.log_decay is leaf
            assert attend.log_decay.grad.dtype == torch.float32 and float(attend.log_decay.grad[1]) == 1 + 2.0 ** -20
    attend = OnTheHost().to("meta", torch.bfloat16)
    assert attend.log_decay.device.type == "meta" and attend.log_decay.dtype == torch.float32
