"""Sequence operators at the edges of what their documents allow: shared buffers, plans of pieces that few sizes reach, calls that
only part of the gradients is asked of, values that are no ordinary numbers."""
from __future__ import annotations

import ctypes

import pytest
import torch

from tests import sequence_reference as ref
from tests.test_gpu_sequence_attention import _compare, _double, _inputs, _run

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


# ---- precision ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("shape", [
    # B, L, H, Hkv, Dk, Dv
    (2, 33, 2, 1, 24, 40), (2, 64, 2, 2, 128, 128), (2, 65, 4, 2, 64, 128), (3, 100, 2, 2, 18, 10), (2, 130, 2, 2, 128, 20),
    (1, 700, 4, 2, 128, 128), (2, 200, 2, 1, 256, 24), (2, 90, 2, 2, 256, 200), (2, 40, 2, 1, 64, 16), (2, 300, 2, 1, 32, 32)])
def test_scores_and_states_in_bfloat16_keep_two_terms(shape):
    """bfloat16 answers and gradients are rounded once, at the end: half a step 2^-8 of the value.  With A the sum of the absolute values
    of the terms, before that: scores, the copy of the state and what is added to the state in two terms, 2^-16 A each, below
    2^-14 A together with what the last rounding makes of it; sums in 32 bits and powers of the decay as for float32,
    2^-24 (2 L + Dk + 64) A."""
    a = _inputs(*shape, BF16, seed=300)
    args = [_double(a[n]) for n in ("q", "k", "v", "g", "s0")] + [None, None, _double(a["do"]), _double(a["ds"])]
    want, bound = ref.attention(*args), ref.attention_bound(*args)
    got = _run(a)
    for n in ("out", "dq", "dk", "dv"):
        off = (got[n].double() - want[n]).abs()
        tol = 2 ** -8 * want[n].abs() + (2 ** -14 + 2 ** -24 * (2 * shape[1] + max(shape[4:]) + 64)) * bound[n]
        assert (off <= tol).all(), (n, float((off / tol).max()))
        if off.numel() > 2000:  # a rounding to the nearest alone: steps of 2^-7 at most, a third of whose half squared is the mean
            assert float(off.square().mean().sqrt()) <= 12 ** -0.5 * 2 ** -7 * float(want[n].square().mean().sqrt()), n


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_an_infinite_value_stays_infinite_in_the_state(dtype):
    from pathsig_amd import sequence
    a = _inputs(2, 150, 2, 1, 24, 40, dtype, seed=310)
    a["k"] = torch.where(a["k"] == 0, torch.ones_like(a["k"]), a["k"])
    a["v"][0, 20, 0, 3], a["v"][0, 149, 0, 5], a["v"][1, 70, 0, 0] = float("inf"), float("-inf"), float("inf")
    _, last = sequence.linear_attention(a["q"], a["k"], a["v"], torch.full((2,), -0.01, device=DEV), state=a["s0"], return_state=True)
    want = torch.isinf(torch.zeros_like(last))
    want[0, :, :, 3] = want[0, :, :, 5] = want[1, :, :, 0] = True
    assert torch.equal(torch.isinf(last), want) and not last.isnan().any()
    assert torch.equal(last[0, :, :, 5] > 0, (a["k"][0, 149] < 0).expand(2, 24))


# ---- gradients ----------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_gradients_of_gradients_are_refused(dtype):
    """A penalty on a gradient, which reaches the leaves through the output as well; a graph that nobody goes back through changes
    nothing."""
    from pathsig_amd import sequence
    a = _inputs(2, 40, 2, 1, 16, 24, dtype, seed=320)
    leaves = [a[n].requires_grad_(True) for n in ("q", "k", "v", "g", "s0")]
    x, w = a["q"].detach().requires_grad_(True), torch.ones(16, device=DEV, requires_grad=True)
    for out, of in ((sequence.linear_attention(*leaves[:4], state=leaves[4]), leaves), (sequence.norm_before(x, w), (x, w))):
        plain = torch.autograd.grad(out.float().sum(), of, retain_graph=True)
        grads = torch.autograd.grad(out.float().sum(), of, create_graph=True)
        for one, other in zip(plain, grads):
            assert torch.equal(one, other)
        for grad in grads:
            with pytest.raises(RuntimeError, match="not implemented"):
                (out.float().sum() + grad.float().pow(2).sum()).backward(retain_graph=True)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [40, 500])
def test_hooks_that_hand_saved_tensors_back_in_other_strides(L, dtype):
    """Views of a projection whose rows are no whole units of 16 bytes are copied by the forward; activations that were kept on the
    host come back contiguous, with rows of whole units, and need no copy."""
    from pathsig_amd import sequence
    B, H, Dk, Dv = 2, 2, 16, 24
    a = _inputs(B, L, H, H, Dk, Dv, dtype, seed=330)
    wide = torch.cat([a[n].flatten(2) for n in ("q", "k", "v")] + [torch.zeros(B, L, 3, dtype=dtype, device=DEV)], dim=-1)
    q, k, v, _ = wide.requires_grad_(True).split((H * Dk, H * Dk, H * Dv, 3), dim=-1)
    g, s0 = a["g"].requires_grad_(True), a["s0"].requires_grad_(True)

    def gradients():
        out, last = sequence.linear_attention(*(t.unflatten(-1, (H, -1)) for t in (q, k, v)), g, state=s0, return_state=True)
        return torch.autograd.grad((out, last), (wide, g, s0), (a["do"], a["ds"]), retain_graph=True)
    want = gradients()
    for hooks in (torch.autograd.graph.save_on_cpu(), torch.autograd.graph.save_on_cpu(pin_memory=True),
                  torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous(), lambda t: t),
                  # no unit of the workspace at its place
                  torch.autograd.graph.saved_tensors_hooks(
                      lambda t: torch.cat([t.flatten()[:1], t.flatten()])[1:].view(t.shape) if t.numel() else t, lambda t: t)):
        with hooks:
            got = gradients()
        for one, other in zip(got, want):
            assert torch.equal(one, other)


# ---- modules ------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("learn", [False, True])
def test_a_whole_block_converted_to_bfloat16(learn):
    """The block of test_gpu_sequence_block.py converted as models are, decays and all: what converting its other parts one by one
    gives, in training and token by token."""
    import copy
    from tests.test_gpu_sequence_block import Block
    torch.manual_seed(5)
    parts = Block(64, 4, 16, 16, learn)
    whole = copy.deepcopy(parts).to(BF16)
    for m in (parts.before, parts.project, parts.heads, parts.join, parts.after):
        m.to(BF16)
    x = torch.randn(2, 80, 64, device=DEV).to(BF16)
    results = []
    for block in (whole, parts):
        assert block.attend.log_decay.dtype == F32
        out, normed, last = block(x)
        grads = torch.autograd.grad(out.float().sum() + normed.float().square().sum() + last.sum(), list(block.parameters()))
        with torch.no_grad():
            results.append([out, normed, last, *grads, *block.step(x[:, 0], last.clone())])
    for one, other in zip(*results):
        assert one.dtype == other.dtype and torch.equal(one, other)


# ---- norms --------------------------------------------------------------------------------------------------------
def _norm_inputs(dtype, *shape):
    g = torch.Generator().manual_seed(400)
    make = lambda *s: torch.randn(*s, generator=g).to(DEV, dtype).requires_grad_(True)  # noqa: E731
    return {"x": make(*shape), "gate": make(*shape), "residual": make(*shape), "weight": make(shape[-1]), "scale": make(shape[-1])}


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_residual_that_changes_after_the_call(dtype):
    """Without a second norm the backward does not read the residual: a stream of features may be added to in place."""
    from pathsig_amd import sequence
    a = _norm_inputs(dtype, 5, 96)
    up = torch.randn(5, 96, device=DEV).to(dtype)
    x, rest = a["x"], {n: a[n] for n in ("gate", "residual", "scale")}
    want = torch.autograd.grad(sequence.norm_after(x, a["weight"], **rest), (x, *rest.values(), a["weight"]), up)
    assert torch.equal(want[2], up)
    stream = a["residual"] * 1
    out = sequence.norm_after(x, a["weight"], gate=a["gate"], residual=stream, scale=a["scale"])
    with torch.no_grad():
        stream.add_(1)
    got = torch.autograd.grad(out, (x, a["gate"], a["residual"], a["scale"], a["weight"]), up)
    for one, other in zip(got, want):
        assert torch.equal(one, other)
    # with a second norm it does, and autograd says so
    stream = a["residual"] * 1
    out, nxt = sequence.norm_after(x, a["weight"], residual=stream, next_weight=a["weight"])
    with torch.no_grad():
        stream.add_(1)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(nxt, x, up)
    # a residual of fewer axes: the sum over the rows
    one = a["residual"][0].detach().requires_grad_(True)
    (got,) = torch.autograd.grad(sequence.norm_after(x, residual=one), one, up)
    assert got.shape == one.shape and torch.equal(got, up.sum(0))


# ---- gradients that nobody asks for -------------------------------------------------------------------------------
def _subsets(names):
    return [[n for i, n in enumerate(names) if bits >> i & 1] for bits in range(1, 2 ** len(names))]


@pytest.mark.parametrize("dtype,shape", [(F32, (2, 300, 4, 2, 24, 32)), (BF16, (2, 300, 4, 2, 24, 32)), (BF16, (3, 45, 2, 2, 18, 10)), (F32, (2, 0, 2, 1, 8, 8))])
def test_each_gradient_of_attention_alone(shape, dtype):
    """Whatever part of the gradients is asked for, it is the same as in all of them."""
    from pathsig_amd import sequence
    a = _inputs(*shape, dtype, seed=340)
    lengths = torch.tensor([shape[1] - 7, 3, 0][:shape[0]], device=DEV)
    names = ("q", "k", "v", "g", "s0")
    bound = ref.attention_bound(*(_double(a[n]) for n in names), lengths, None, _double(a["do"]), _double(a["ds"]))
    want = None
    for some in [list(names)] + _subsets(names):
        leaves = {n: a[n].detach().requires_grad_(n in some) for n in names}
        outs = sequence.linear_attention(*(leaves[n] for n in names[:4]), state=leaves["s0"], lengths=lengths, return_state=True)
        got = dict(zip(some, torch.autograd.grad(outs, [leaves[n] for n in some], (a["do"], a["ds"]))))
        want = want or got
        for n in some:
            if dtype == F32 or ("g" in some and "s0" in some):
                assert torch.equal(got[n], want[n]), (some, n)
                continue
            # states that are not wanted in 32 bits carry a term of bfloat16 less: both sides are off by one rounding, 2^-8 of the value,
            # and 2^-14 A (test_scores_and_states_in_bfloat16_keep_two_terms); what is in 32 bits, by the states' terms, 2^-16 A, at most
            off, A = (got[n].double() - want[n].double()).abs(), bound["d" + n]
            u = 2 ** -8 if got[n].dtype == BF16 else 2 ** -23
            assert (off <= 2 * (u * want[n].double().abs() + 2 ** -14 * A)).all(), (some, n)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(40, 96), (5, 1030)])
def test_each_gradient_of_norms_alone(shape, dtype):
    from pathsig_amd import sequence
    a = _norm_inputs(dtype, *shape)
    a["next_weight"] = (a["weight"] * 0.5).detach()
    do, dn = (torch.randn(*shape, device=DEV).to(dtype) for _ in range(2))
    for last in (False, True):
        names = [n for n in a if last or n != "next_weight"]
        want = None
        for some in [names] + _subsets(names):
            leaves = {n: a[n].detach().requires_grad_(n in some) for n in names}
            outs = sequence.norm_after(leaves["x"], leaves["weight"], **{n: leaves[n] for n in names if n not in ("x", "weight")})
            got = dict(zip(some, torch.autograd.grad(outs, [leaves[n] for n in some], (do, dn) if last else do)))
            want = want or got
            for n in some:
                assert torch.equal(got[n], want[n]), (some, n)


def test_c_abi_without_some_of_the_gradients():
    a = _inputs(2, 700, 4, 2, 32, 48, BF16, seed=350)
    lib, c = _call(a)
    size = lib.pathsig_linattn_backward_workspace(ctypes.byref(c), 0)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)

    def backward(*which):
        got = [torch.full_like(a[n], float("nan")) if i in which else None for i, n in enumerate(("q", "k", "v"))]
        rc = lib.pathsig_linattn_backward(ctypes.byref(c), *(_pointer(a[n]) for n in ("q", "k", "v", "s0")), None, 0, _pointer(a["do"]),
                                          _pointer(a["ds"]), *map(_pointer, got), None, None, _pointer(ws), size, stream)
        assert rc == 0, lib.pathsig_last_error()
        return got
    want = backward(0, 1, 2)
    assert not any(t.isnan().any() for t in want)
    for which in ((0,), (1,), (2,), (0, 2), (1, 2), ()):
        for i, t in enumerate(backward(*which)):
            assert t is None or torch.equal(t, want[i])


# ---- decays above 1 -----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("state", [False, True])
@pytest.mark.parametrize("g,L", [(1.5, 42), (1.5, 33), (2.0, 32), (3.0, 20), (6.0, 9), (12.0, 5), (60.0, 1), (0.9, 70), (0.3, 200), (0.1, 640)])
def test_states_that_grow(g, L, state, dtype):
    """Positive log-decays are no memory that fades, but a learned one may become positive: as long as its powers over the tokens there
    are stay finite (here e^64), so do all results, whatever powers a whole chunk would have.  Tolerances as in
    test_gpu_sequence_attention.py."""
    for shape in ((2, L, 4, 2, 24, 40), (1, L, 4, 4, 130, 20)):
        a = _inputs(*shape, dtype, seed=360, state=state)
        a["g"] = torch.tensor([g, g / 2, 0.0, -g], device=DEV)
        got = _run(a)
        _compare(got, a, rms=False)
        a["g"] = torch.full((4,), g, device=DEV)
        lengths = torch.tensor([L, max(L - 3, 1)][:shape[0]], device=DEV)
        _compare(_run(a, lengths=lengths), a, lengths=lengths, rms=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("g,L", [(60.0, 2), (30.0, 3), (2.8, 32), (1.42, 63)])
def test_a_power_that_no_two_tokens_have(g, L, dtype):
    """From a state of zeros the largest power is that between the first token and the last: one more may overflow."""
    a = _inputs(2, L, 2, 1, 24, 40, dtype, seed=370, state=False)
    a["g"] = torch.full((2,), g, device=DEV)
    a["v"], a["ds"] = a["v"] * 2.0 ** -20, a["ds"] * 2.0 ** -20  # (the sums below stay finite too)
    a["do"] = a["do"] * 2.0 ** -20
    _compare(_run(a), a, rms=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("activation", ["silu", "sigmoid"])
def test_gates_to_the_last_places(activation, dtype):
    """On a row of ones without eps the norm is 1 and the answer the gate's: an exponential (two units of 2^-23), a sum, a reciprocal and
    two products, below 12 * 2^-24 of the value; of the derivative the same of the terms it adds up.  In bfloat16 the argument of
    the exponential, up to 85 / ln 2 in size, is rounded to half a step 2^-24: below 2^-16 together, and the answer is rounded, 2^-8."""
    from pathsig_amd import sequence
    gate = torch.cat([torch.linspace(-85, 85, 3401), torch.linspace(-2, 2, 695)]).view(-1, 64).to(DEV, dtype).requires_grad_(True)
    ones = torch.ones_like(gate)
    out = sequence.norm_after(ones, gate=gate, activation=activation, eps=0.0)
    (slope,) = torch.autograd.grad(out, gate, ones)
    g = gate.detach().double()
    up, down = 1 / (1 + (-g).exp()), 1 / (1 + g.exp())
    value, terms = (g * up, (up, g * up * down)) if activation == "silu" else (up, (up * down, 0 * up))
    u, last = (12 * 2 ** -24, 0.0) if dtype == F32 else (2 ** -16, (1 + 2 ** -16) * 2 ** -8)
    assert ((out.detach().double() - value).abs() <= (u + last) * value.abs()).all()
    off = (slope.double() - terms[0] - terms[1]).abs()
    assert (off <= u * (terms[0].abs() + terms[1].abs()) + last * (terms[0] + terms[1]).abs()).all()


def test_gates_at_their_ends():
    """Gates behind the range of the exponential, and what is no number."""
    from pathsig_amd import sequence
    inf = float("inf")
    for dtype in (F32, BF16):
        gate = torch.tensor([[-300.0, 300.0, -inf, inf, float("nan"), 0.0, -90.0, 90.0]], device=DEV, dtype=dtype, requires_grad=True)
        ones = torch.ones_like(gate)
        out = sequence.norm_after(ones, gate=gate, activation="sigmoid", eps=0.0)
        (slope,) = torch.autograd.grad(out, gate, ones)
        assert out[0, 4].isnan() and slope[0, 4].isnan()
        want = torch.tensor([0.0, 1.0, 0.0, 1.0, 0.5, 0.0, 1.0], device=DEV, dtype=dtype)
        some = [0, 1, 2, 3, 5, 6, 7]
        assert float((out.detach()[0, some] - want).abs().max()) <= 1e-38  # (e^-90 underflows)
        assert float((slope[0, some] - want * (1 - want)).abs().max()) <= 1e-38


# ---- every width of the state in chunks of each length ------------------------------------------------------------
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [19, 32, 33, 97])
@pytest.mark.parametrize("Dk", [24, 64, 128, 200])
@pytest.mark.parametrize("Dv", [32, 56, 128, 200])
def test_widths_and_lengths(L, Dk, Dv, dtype):
    """Up to 32 tokens, more, and more than a chunk, with sequences that end early and one without tokens; tolerances as in
    test_gpu_sequence_attention.py."""
    a = _inputs(4, L, 2, 1, Dk, Dv, dtype, seed=380)
    lengths = torch.tensor([L, L - 1, 0, L // 2], device=DEV)
    _compare(_run(a, lengths=lengths), a, lengths=lengths)


def test_rows_of_more_threads_than_a_launch_has():
    """2^29 rows of one channel, eight threads each: the last rows are answered like the same ones alone, and get their gradients."""
    from pathsig_amd import sequence
    rows = 2 ** 29 + 3001
    x = torch.full((rows, 1), 2.0, dtype=BF16, device=DEV)
    x[-5000:] = torch.randn(5000, 1, device=DEV).to(BF16)
    with torch.no_grad():
        out = sequence.norm_before(x, eps=0.25)
        assert torch.equal(out[-5000:], sequence.norm_before(x[-5000:], eps=0.25))
        assert bool((out[:-5000] == (2.0 / 4.25 ** 0.5 * torch.ones(1, device=DEV)).to(BF16)).all())
    x.requires_grad_(True)
    (grad,) = torch.autograd.grad(sequence.norm_before(x, eps=0.25), x, out)
    some = x.detach()[-5000:].requires_grad_(True)
    (want,) = torch.autograd.grad(sequence.norm_before(some, eps=0.25), some, out[-5000:])
    assert torch.equal(grad[-5000:], want)


def test_return_state_is_any_truth_value():
    import numpy as np
    from pathsig_amd import sequence
    a = _inputs(1, 5, 2, 1, 8, 8, F32, seed=390)
    args = [a[n] for n in ("q", "k", "v", "g")]
    want = sequence.linear_attention(*args, return_state=True)
    for yes in (1, np.True_, np.bool_(1)):
        got = sequence.linear_attention(*args, return_state=yes)
        assert isinstance(got, tuple) and all(torch.equal(x, y) for x, y in zip(got, want))
    for no in (0, np.False_, None):
        assert torch.equal(sequence.linear_attention(*args, return_state=no), want[0])


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L", [20, 700])
def test_what_a_sequence_without_tokens_holds_stays_there(L, dtype):
    """The state of a place in the batch that nothing uses, and the gradient from above for it, may be no numbers."""
    a = _inputs(3, L, 2, 1, 24, 40, dtype, seed=395)
    lengths = torch.tensor([L, 0, L // 2], device=DEV)
    want = _run(a, lengths=lengths)
    for n in ("s0", "ds"):
        a[n][1, :, :5], a[n][1, :, 5:] = float("nan"), float("inf")
    got = _run(a, lengths=lengths)
    assert torch.equal(got["dg"], want["dg"])
    for n in ("out", "last", "dq", "dk", "dv", "ds0"):
        assert torch.equal(got[n][::2], want[n][::2]), n
    assert (got["out"][1] == 0).all() and torch.equal(got["last"][1, :, 5:], a["s0"][1, :, 5:])


# ---- plans of pieces ----------------------------------------------------------------------------------------------
# Sequences are cut into pieces where there are few of them.  Up to four pieces are joined by the blocks that start from them, more by a
# launch of their own; 171 to 256 heads of more than 64 channels are folded in halves and swept two pieces to a block.
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape,pieces", [
    # B, L, H, Hkv, Dk, Dv: two pieces, three, four, more; rows times columns of the state no multiple of four; heads or rows that are no
    # whole units of 16 bytes and are copied first
    ((3, 250, 2, 1, 16, 128), 2), ((1, 192, 2, 1, 16, 16), 3), ((1, 500, 3, 3, 8, 8), 4), ((1, 2304, 1, 1, 16, 24), 36),
    ((1, 900, 3, 1, 5, 7), None), ((2, 700, 2, 1, 18, 10), None), ((1, 300, 2, 2, 33, 65), None), ((1, 1500, 2, 2, 129, 3), None)])
def test_pieces(shape, pieces, dtype):
    a = _inputs(*shape, dtype, seed=410)
    assert pieces is None or _pieces(*_call(a)) == pieces
    _compare(_run(a), a, rms=False)
    L = shape[1]
    lengths = torch.tensor([L - 70, 65, 1][:shape[0]], device=DEV)
    _compare(_run(a, lengths=lengths), a, lengths=lengths, rms=False)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("L,Dk,Dv,Hkv", [(616, 80, 72, 16), (617, 72, 80, 4), (640, 16, 96, 16), (1030, 128, 128, 16)])
def test_two_pieces_to_a_block(L, Dk, Dv, Hkv, dtype):
    """176 heads of sequences, folded in halves: all lengths alike, and sequences that end in each half, at its border and before it
    begins."""
    B, H = 11, 16
    a = _inputs(B, L, H, Hkv, Dk, Dv, dtype, seed=420)
    lib, c = _call(a)
    assert _pieces(lib, c) == 4
    _compare(_run(a), a)
    piece = -(-(-(-L // 4)) // 64) * 64
    lengths = torch.tensor([L, 0, 1, piece - 1, piece, piece + 1, 2 * piece - 3, 2 * piece, 2 * piece + 1, 3 * piece + 5, L - 1], device=DEV)
    got = _run(a, lengths=lengths)
    _compare(got, a, lengths=lengths)
    dead = torch.arange(L, device=DEV)[None] >= lengths[:, None]
    for n in ("out", "dq", "dk", "dv"):
        assert (got[n][dead] == 0).all(), n


@pytest.mark.parametrize("shape", [(2, 100, 4, 2, 24, 40), (1, 700, 4, 4, 64, 64), (2, 300, 2, 1, 130, 20), (2, 40, 3, 1, 18, 10), (1, 2304, 2, 2, 16, 24)])
def test_decays_gradient_in_bfloat16_is_summed_in_32_bits(shape):
    """Its terms enter in three parts of bfloat16, all their bits: the bound of float32."""
    a = _inputs(*shape, BF16, seed=430)
    args = [_double(a[n]) for n in ("q", "k", "v", "g", "s0")] + [None, None, _double(a["do"]), _double(a["ds"])]
    want, bound = ref.attention(*args)["dg"], ref.attention_bound(*args)["dg"]
    off = (_run(a)["dg"].double() - want).abs()
    assert (off <= 2 ** -24 * (2 * shape[1] + max(shape[4:]) + 64) * bound).all(), float((off / bound).max())
