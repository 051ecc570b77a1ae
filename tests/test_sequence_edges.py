"""Sequence operators at the edges of what their documents allow, without a GPU: buffers that a call of the C ABI must not share."""
from __future__ import annotations

import ctypes

import pytest

from pathsig_amd import _load

ERR_ARG = -1


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
