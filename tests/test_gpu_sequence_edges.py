"""Sequence operators at the edges of what their documents allow: shared buffers, plans of pieces that few sizes reach, calls that
only part of the gradients is asked of, values that are no ordinary numbers."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests.test_gpu_sequence_attention import _inputs

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def float32_by_default():
    """Tensors made here without a type are float32, whatever the tests before left as the default."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)


# ---- the C ABI by itself ------------------------------------------------------------------------------------------
def _pointer(t):
    return None if t is None else t.data_ptr()


def _call(a, learned=0):
    """The call of `_inputs`, and the library."""
    from pathsig_amd import _load
    B, L, H, Dk = a["q"].shape
    c = _load.LinearAttentionCall(dtype=2 if a["q"].dtype == BF16 else 0, B=B, L=L, H=H, Hkv=a["k"].shape[2], Dk=Dk, Dv=a["v"].shape[3],
                                  scale=Dk ** -0.5, learned_decay=learned, log_decay=a["g"].data_ptr(), lengths=None)
    for n in ("q", "k", "v"):
        getattr(c, n + "_stride")[:] = a[n].stride()[:3]
    return _load.lib(), c


def _pieces(lib, c):
    """Pieces that sequences of whole units of 16 bytes are cut into: the workspace is a state for each."""
    return max(1, lib.pathsig_linattn_forward_workspace(ctypes.byref(c)) // (4 * c.B * c.H * c.Dk * c.Dv))


def _forward(a, state, last):
    lib, c = _call(a)
    size = lib.pathsig_linattn_forward_workspace(ctypes.byref(c))
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    out = torch.empty_like(a["do"])
    rc = lib.pathsig_linattn_forward(ctypes.byref(c), *(_pointer(a[n]) for n in ("q", "k", "v")), _pointer(state), _pointer(out), _pointer(last),
                                     _pointer(ws) if size else None, size, ctypes.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0, lib.pathsig_last_error()
    return out, ws


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,pieces", [
    # B, L, H, Hkv, Dk, Dv
    ((2, 60, 2, 1, 32, 48), {F32: 1, BF16: 1}), ((1, 192, 2, 1, 16, 16), {F32: 3, BF16: 3}), ((1, 256, 2, 2, 64, 64), {F32: 4, BF16: 2}),
    ((4, 2600, 2, 1, 16, 32), {F32: 21, BF16: 21})])
def test_last_state_over_the_first(shape, pieces, dtype):
    """The last state may be written over the first: one piece, up to four (whose blocks all read the first state) and more."""
    a = _inputs(*shape, dtype, seed=200)
    lib, c = _call(a)
    assert _pieces(lib, c) == pieces[dtype]
    last = torch.empty_like(a["s0"])
    out, ws = _forward(a, a["s0"], last)
    both = a["s0"].clone()
    out_both, ws_both = _forward(a, both, both)
    assert torch.equal(out_both, out) and torch.equal(both, last)
    # what a backward takes over is the same: the states in front of the second piece and all that follow
    state = 4 * both.numel()
    assert torch.equal(ws_both[state:_pieces(lib, c) * state], ws[state:_pieces(lib, c) * state])
