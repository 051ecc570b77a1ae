"""The norms before and after a block on the GPU against their formulas in 64 bits (`sequence_reference.py`).

Tolerances: everything is worked out in 32 bits and rounded once.  Half a step of the type relative to the value (bfloat16 2^-8, float32
2^-24), and in 32 bits: sums over a row take eight terms a thread and at most ten steps of a tree, sums over rows
at most rows / 256 terms a block, 768 / 8 blocks and eight parts; about twenty products, exponentials and roots in a chain, each off by
one or two units: 2^-24 (64 + rows / 256 + 128 for sums over rows) of the sum of the absolute values of the terms."""
from __future__ import annotations

import ctypes
import itertools

import pytest
import torch

from tests import sequence_reference as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def float32_by_default():
    """Tensors made here without a type are float32, whatever the tests before left as the default."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)


BF16, F32 = torch.bfloat16, torch.float32
NAMES = ("x", "weight", "gate", "residual", "scale", "next_weight")
COLUMNS = ("weight", "scale", "next_weight")


def _randn(*shape, seed, dtype, scale=1.0, mean=0.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, dtype=torch.float64, generator=g) * scale + mean).to(dtype).to(DEV)


def _inputs(shape, dtype, param_dtype, have, seed=0):
    C = shape[-1]
    a = {"x": _randn(*shape, seed=seed + 1, dtype=dtype, scale=2.0)}
    for i, n in enumerate(("gate", "residual")):
        a[n] = _randn(*shape, seed=seed + 2 + i, dtype=dtype, scale=1.5) if n in have else None
    for i, n in enumerate(COLUMNS):
        a[n] = _randn(C, seed=seed + 5 + i, dtype=param_dtype, scale=0.3, mean=0.8) if n in have else None
    return a, _randn(*shape, seed=seed + 9, dtype=dtype), _randn(*shape, seed=seed + 10, dtype=dtype)


def _run(a, do, dn, **kw):
    from pathsig_amd import sequence
    leaves = {n: t.detach().requires_grad_(True) for n, t in a.items() if t is not None}
    out = sequence.norm_after(leaves["x"], leaves.get("weight"), **{n: leaves.get(n) for n in NAMES[2:]}, **kw)
    outs, ups = (out, (do, dn)) if isinstance(out, tuple) else ((out,), (do,))
    grads = torch.autograd.grad(outs, list(leaves.values()), ups)
    got = {"out": outs[0].detach(), **{n: g for n, g in zip(leaves, grads)}}
    if len(outs) == 2:
        got["next"] = outs[1].detach()
    return got


def _compare(got, a, do, dn, eps=1e-6, activation="silu"):
    C = a["x"].shape[-1]
    flat = {n: None if t is None else (t.double() if n in COLUMNS else t.double().reshape(-1, C)) for n, t in a.items()}
    rows = flat["x"].shape[0]
    want, bound = ref.norms(**flat, eps=eps, activation=activation, do=do.double().reshape(-1, C),
                            dn=dn.double().reshape(-1, C) if a["next_weight"] is not None else None)
    for n, x in got.items():
        assert torch.isfinite(x).all(), n
        w, A = want[n], bound[n]
        err = (x.double().reshape(w.shape) - w).abs()
        u = 2 ** -8 if x.dtype == BF16 else 2 ** -24
        tol = u * w.abs() + 2 ** -24 * (64 + (rows / 256 + 128 if n in COLUMNS else 0)) * A + 1e-37
        assert (err <= tol).all(), (n, float((err / tol).max()))


SHAPES = [(1, 1), (3, 5), (7, 64), (33, 63), (5, 65), (2, 3, 128), (9, 130), (2, 256), (3, 300), (5, 512), (2, 513), (2, 1000), (4, 1024),
          (2, 3, 1025), (2, 2048), (3, 2049), (2, 4096), (2, 4097), (1, 5000), (2, 8192), (3, 8191)]
EVERYTHING = ("weight", "gate", "residual", "scale", "next_weight")


@pytest.mark.parametrize("types", [(F32, F32), (BF16, BF16), (BF16, F32)])
@pytest.mark.parametrize("shape", SHAPES)
def test_everything_at_once(shape, types):
    a, do, dn = _inputs(shape, *types, EVERYTHING)
    _compare(_run(a, do, dn), a, do, dn)


@pytest.mark.parametrize("types", [(F32, F32), (BF16, F32)])
@pytest.mark.parametrize("have", [c for n in range(5) for c in itertools.combinations(EVERYTHING, n)])
def test_each_part_left_out(have, types):
    a, do, dn = _inputs((6, 192), *types, have, seed=20)
    _compare(_run(a, do, dn), a, do, dn)


@pytest.mark.parametrize("activation", ["silu", "sigmoid", "linear"])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_activations(activation, dtype):
    a, do, dn = _inputs((6, 200), dtype, dtype, EVERYTHING, seed=30)
    a["gate"][0, :4] = torch.tensor([0.0, 80.0, -80.0, 1e-3])
    _compare(_run(a, do, dn, activation=activation, eps=1e-3), a, do, dn, eps=1e-3, activation=activation)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(4, 6, 96), (1, 1), (5, 2050)])
def test_norm_before(shape, dtype):
    from pathsig_amd import sequence
    a, do, _ = _inputs(shape, dtype, dtype, ("weight",), seed=40)
    x, w = a["x"].clone().requires_grad_(True), a["weight"].clone().requires_grad_(True)
    y = sequence.norm_before(x, w, eps=1e-5)
    dx, dw = torch.autograd.grad(y, (x, w), do)
    _compare({"out": y.detach(), "x": dx, "weight": dw}, a, do, do, eps=1e-5)
    with torch.no_grad():
        assert torch.equal(sequence.norm_before(x, w, eps=1e-5), y)
    plain = sequence.norm_before(a["x"])
    _compare({"out": plain}, {**a, "weight": None}, do, do)


@pytest.mark.parametrize("rows,C", [(300001, 16), (70000, 64), (5000, 1024), (2000, 4096)])
def test_sums_over_many_rows(rows, C):
    a, do, dn = _inputs((rows, C), F32, F32, EVERYTHING, seed=50)
    _compare(_run(a, do, dn), a, do, dn)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_views_and_broadcasts(dtype):
    """Rows cut out of wider ones, other orders of the axes, an offset that leaves no address aligned, and gates and residuals
    broadcast over tokens, whose gradients are the sums."""
    from pathsig_amd import sequence
    B, L, C = 3, 5, 64
    a, do, dn = _inputs((B, L, C), dtype, dtype, EVERYTHING, seed=60)
    want = _run(a, do, dn)
    wide = torch.full((B, L, 3 * C + 1), float("nan"), dtype=dtype, device=DEV)
    views = {}
    for i, n in enumerate(("x", "gate", "residual")):
        views[n] = wide[..., i * C:(i + 1) * C]
        views[n].copy_(a[n])
    swapped = {n: a[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ("x", "gate", "residual")}
    apart = {n: a[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("x", "gate", "residual")}
    for view in (views, swapped, apart):
        got = _run({**a, **view}, do, dn)
        _compare(got, a, do, dn)
        # (rows that start anywhere are read element by element: thread t has columns t, t + T, ... instead of vectors of
        # neighbours, so a row's squares are added in another order and the last bit may differ)
        assert view is views or all(torch.equal(got[n], want[n]) for n in want)
    gate, residual = a["gate"][:, :1], a["residual"][0, 0]
    x = a["x"].clone().requires_grad_(True)
    g, r = gate.clone().requires_grad_(True), residual.clone().requires_grad_(True)
    out = sequence.norm_after(x, gate=g, residual=r)
    dx, dg, dr = torch.autograd.grad(out, (x, g, r), do)
    full = {"x": a["x"], "gate": gate.expand(B, L, C).contiguous(), "residual": residual.expand(B, L, C).contiguous(), "weight": None,
            "scale": None, "next_weight": None}
    whole = _run(full, do, dn)
    assert torch.equal(out, whole["out"]) and torch.equal(dx, whole["x"])
    u = 2 ** -8 if dtype == BF16 else 2 ** -22
    for got, rows in ((dg, whole["gate"].sum(1, keepdim=True)), (dr, whole["residual"].sum((0, 1)))):
        assert got.shape == rows.shape and float((got - rows).abs().max()) <= 2 * u * float(rows.abs().max())


def test_one_gradient_from_above():
    from pathsig_amd import sequence
    a, do, dn = _inputs((5, 100), F32, F32, EVERYTHING, seed=70)
    leaves = {n: t.clone().requires_grad_(True) for n, t in a.items()}
    zero = torch.zeros_like(do)
    for which in (0, 1):
        outs = sequence.norm_after(leaves["x"], leaves["weight"], **{n: leaves[n] for n in NAMES[2:]})
        grads = torch.autograd.grad(outs[which], list(leaves.values()), (do, dn)[which], allow_unused=True)
        got = {n: g for n, g in zip(leaves, grads) if g is not None}
        _compare(got, a, *((do, zero) if which == 0 else (zero, dn)))


def test_rows_do_not_touch_each_other():
    """Infinities and NaN stay in their row; a row of zeros is no division by zero."""
    from pathsig_amd import sequence
    for dtype, C in itertools.product((F32, BF16), (16, 100, 600)):
        x = _randn(40, C, seed=80, dtype=dtype)
        clean = sequence.norm_before(x)
        bad = x.clone()
        bad[3, 0], bad[7, 5], bad[9] = float("nan"), float("inf"), 0
        got = sequence.norm_before(bad)
        keep = [i for i in range(40) if i not in (3, 7, 9)]
        assert torch.equal(got[keep], clean[keep]) and (got[9] == 0).all() and got[3].isnan().any()


def test_refusals_on_the_device():
    from pathsig_amd import sequence
    x = torch.zeros(3, 16, device=DEV)
    for bad in (dict(weight=torch.ones(15, device=DEV)), dict(gate=torch.zeros(3, 16, device=DEV, dtype=BF16)),
                dict(gate=torch.zeros(4, 16, device=DEV)), dict(residual=torch.zeros(2, 16, device=DEV)), dict(scale=torch.ones(16)),
                dict(weight=torch.ones(16, device=DEV, dtype=BF16))):
        with pytest.raises(RuntimeError):
            sequence.norm_after(x, **bad)
    with pytest.raises(RuntimeError):
        sequence.norm_before(x.double())
    with pytest.raises(RuntimeError):
        sequence.norm_before(torch.zeros(2, 8193, device=DEV))
    with pytest.raises(RuntimeError):
        sequence.norm_before(x, eps=-1.0)


def test_nothing_to_do():
    from pathsig_amd import sequence
    x, w = torch.zeros(0, 7, 16, device=DEV, requires_grad=True), torch.ones(16, device=DEV, requires_grad=True)
    out, nxt = sequence.norm_after(x, w, next_weight=w)
    assert out.shape == nxt.shape == (0, 7, 16)
    dx, dw = torch.autograd.grad(out.sum() + nxt.sum(), (x, w))
    assert dx.shape == x.shape and (dw == 0).all()


def test_captured_and_replayed_and_on_two_streams():
    a, do, dn = _inputs((700, 96), BF16, F32, EVERYTHING, seed=90)
    want = _run(a, do, dn)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    results = []
    for s in streams:
        with torch.cuda.stream(s):
            results.append(_run(a, do, dn))
    torch.cuda.synchronize()
    for got in results:
        assert all(torch.equal(got[n], want[n]) for n in want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = _run(a, do, dn)
    for i in range(4):
        fresh, _, _ = _inputs((700, 96), BF16, F32, EVERYTHING, seed=100 + i)
        for n in a:
            a[n].copy_(fresh[n])
        graph.replay()
        eager = _run(a, do, dn)
        torch.cuda.synchronize()
        assert all(torch.equal(got[n], eager[n]) for n in eager)


def test_c_abi_by_itself():
    from pathsig_amd import _load
    lib = _load.lib()
    a, do, dn = _inputs((50, 96), BF16, BF16, EVERYTHING, seed=120)
    want = _run(a, do, dn)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    call = _load.NormCall(dtype=2, param_dtype=2, activation=0, rows=50, C=96, x_stride=96, gate_stride=96, residual_stride=96, eps=1e-6,
                          **{n: p(a[n]) for n in NAMES})
    c, stream = ctypes.byref(call), ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    out, nxt, stats = torch.empty_like(do), torch.empty_like(do), torch.empty(2, 50, device=DEV)
    assert lib.pathsig_norm_forward(c, p(out), p(nxt), p(stats), stream) == 0
    assert torch.equal(out, want["out"]) and torch.equal(nxt, want["next"])
    size = lib.pathsig_norm_backward_workspace(c)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    got = {n: torch.empty_like(a[n]) for n in NAMES}
    rc = lib.pathsig_norm_backward(c, p(stats), p(do), p(dn), p(got["x"]), p(got["gate"]), p(got["residual"]), p(got["weight"]),
                                   p(got["scale"]), p(got["next_weight"]), p(ws), size, stream)
    assert rc == 0, lib.pathsig_last_error()
    assert all(torch.equal(got[n], want[n]) for n in NAMES)
    # some gradients alone, without a workspace where no parameter's is among them
    dx = torch.empty_like(do)
    assert lib.pathsig_norm_backward(c, p(stats), p(do), p(dn), p(dx), None, None, None, None, None, None, 0, stream) == 0
    assert torch.equal(dx, want["x"])
    dw = torch.empty_like(a["weight"])
    assert lib.pathsig_norm_backward(c, p(stats), p(do), p(dn), None, None, None, p(dw), None, None, p(ws), size, stream) == 0
    assert torch.equal(dw, want["weight"])
