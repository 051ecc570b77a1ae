"""Linear attention with decays on the GPU against the token-by-token formulas in 64 bits (`sequence_reference.py`).

Tolerances, with u half a step of the type relative to the value (bfloat16 2^-8, float32 2^-24) and A the sum of the absolute values of the terms of
an answer (the same formulas on absolute values):
* bfloat16: an answer is rounded once (u |o|); its terms meet a rounded score (u) or a rounded copy of the state (u) whose terms
  were rounded (u): at most 2 u A.  Sums of up to L + Dk terms in 32 bits, powers of the decay: less than u A / 8.
* float32, and what is in 32 bits whatever the type (states, gradients of states and decays): sums of L + Dk terms, each sum in
  32 bits, 2^-24 (L + Dk) A, and decays that are powers of rounded exponentials, 3 * 2^-24 for each of the L / 32 chunks; together
  below 2^-24 (2 L + Dk + 64) A.  The gradient of the decays takes its terms in two parts of bfloat16: 2^-17 A more.
Roundings of independent terms also add up like independent numbers: the root mean square of the error of a bfloat16 answer stays below
sqrt(3) * (2^-8 / sqrt(3)) of that of the answers."""
from __future__ import annotations

import ctypes
import math

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


def _randn(*shape, seed, dtype=torch.float64, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(*shape, dtype=torch.float64, generator=g) * scale).to(dtype).to(DEV)


def _inputs(B, L, H, Hkv, Dk, Dv, dtype, seed=0, state=True):
    g = torch.log1p(-torch.exp2(-torch.linspace(1, 8, H, dtype=torch.float64))).to(F32).to(DEV)
    return dict(q=_randn(B, L, H, Dk, seed=seed + 1, dtype=dtype), k=_randn(B, L, Hkv, Dk, seed=seed + 2, dtype=dtype),
                v=_randn(B, L, Hkv, Dv, seed=seed + 3, dtype=dtype), g=g,
                s0=_randn(B, H, Dk, Dv, seed=seed + 4, dtype=F32) if state else None,
                do=_randn(B, L, H, Dv, seed=seed + 5, dtype=dtype), ds=_randn(B, H, Dk, Dv, seed=seed + 6, dtype=F32))


def _double(t):
    return None if t is None else t.detach().double()


def _run(a, lengths=None, scale=None, grads=True):
    """Results of the operators, by the names of the reference."""
    from pathsig_amd import sequence
    leaves = {n: a[n].detach().requires_grad_(True) for n in ("q", "k", "v", "g", "s0") if a[n] is not None}
    out, last = sequence.linear_attention(leaves["q"], leaves["k"], leaves["v"], leaves["g"], state=leaves.get("s0"),
                                          lengths=lengths, scale=scale, return_state=True)
    got = {"out": out.detach(), "last": last.detach()}
    if grads:
        g = torch.autograd.grad((out, last), list(leaves.values()), (a["do"], a["ds"]))
        got.update({"d" + n: x for n, x in zip(leaves, g)})
    return got


def _compare(got, a, lengths=None, scale=None, grads=True, rms=True):
    args = [_double(a[n]) for n in ("q", "k", "v", "g", "s0")] + [lengths, scale] + \
           ([_double(a["do"]), _double(a["ds"])] if grads else [])
    want, bound = ref.attention(*args), ref.attention_bound(*args)
    L, Dk = a["q"].shape[1], max(a["q"].shape[3], a["v"].shape[3])
    low = a["q"].dtype == BF16
    for name, x in got.items():
        assert torch.isfinite(x).all(), name
        err, w, A = (x.double() - want[name]).abs(), want[name], bound[name]
        if x.dtype == BF16:
            tol = 2 ** -8 * w.abs() + (2 + 1 / 8) * 2 ** -8 * A
        else:
            tol = 2 ** -24 * (2 * L + Dk + 64) * A
            if name == "dg" and low:
                tol = tol + 2 ** -17 * A
        # (an answer that only underflows: a few of the smallest float32)
        assert (err <= tol + 1e-37).all(), (name, float((err / (tol + 1e-37)).max()))
        if rms and x.dtype == BF16 and x.numel() > 2000:
            size = float(w.square().mean().sqrt())
            assert float(err.square().mean().sqrt()) <= 2 ** -8 * size, name


SHAPES = [
    # B, L, H, Hkv, Dk, Dv
    (2, 1, 1, 1, 1, 1), (1, 2, 3, 1, 5, 7), (3, 31, 2, 2, 16, 8), (2, 33, 2, 1, 32, 32), (2, 63, 4, 2, 24, 64), (1, 64, 2, 2, 64, 33),
    (2, 65, 2, 1, 40, 96), (1, 130, 2, 2, 128, 128), (2, 100, 3, 3, 100, 20), (1, 129, 2, 1, 256, 64), (2, 70, 2, 2, 20, 256),
    (1, 96, 1, 1, 255, 129),
    # in two, three and nine pieces
    (1, 512, 2, 1, 64, 64), (1, 900, 2, 2, 32, 128), (2, 2304, 1, 1, 16, 24),
]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", SHAPES)
def test_values_and_gradients(shape, dtype):
    a = _inputs(*shape, dtype)
    _compare(_run(a), a)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(5, 67, 2, 1, 24, 40), (6, 600, 2, 2, 64, 64), (5, 2500, 1, 1, 16, 16)])
def test_lengths_and_what_lies_behind_them(shape, dtype):
    """Padding is neither read nor answered: it holds NaN and infinities here, in gradients from above too."""
    B, L = shape[:2]
    a = _inputs(*shape, dtype, seed=10)
    lengths = torch.tensor([L, 0, 1, -3, L // 2 + 1, 2 * L][:B], device=DEV)
    dead = torch.arange(L, device=DEV)[None] >= lengths[:, None]
    clean = dict(a)
    for n, bad in (("q", math.nan), ("k", math.inf), ("v", -math.inf), ("do", math.nan)):
        a[n] = a[n].clone()
        a[n][dead] = bad
    for ln in (lengths, lengths.int()):
        got = _run(a, lengths=ln)
        _compare(got, clean, lengths=lengths)
        for n in ("out", "dq", "dk", "dv"):
            assert (got[n][dead] == 0).all(), n
    # no token at all: the state and its gradient pass through
    for b in (1, 3):
        assert torch.equal(got["last"][b], clean["s0"][b]) and torch.equal(got["ds0"][b], clean["ds"][b])


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_without_a_state_and_with_a_scale(dtype):
    from pathsig_amd import sequence
    a = _inputs(2, 150, 2, 1, 48, 80, dtype, seed=20, state=False)
    got = _run(a, scale=0.37)
    assert "ds0" not in got
    _compare(got, a, scale=0.37)
    with torch.no_grad():
        out = sequence.linear_attention(a["q"], a["k"], a["v"], a["g"], scale=0.37)
    want = ref.attention(*(_double(a[n]) for n in ("q", "k", "v", "g")), None, None, 0.37)["out"]
    A = ref.attention_bound(*(_double(a[n]) for n in ("q", "k", "v", "g")), None, None, 0.37)["out"]
    tol = 2 ** -8 * want.abs() + 2.125 * 2 ** -8 * A if dtype == BF16 else 2 ** -24 * (2 * 150 + 80 + 64) * A
    assert ((out.double() - want).abs() <= tol).all()


def test_gradients_of_one_output_alone():
    from pathsig_amd import sequence
    a = _inputs(2, 300, 2, 2, 32, 32, F32, seed=30)
    zero_o, zero_s = torch.zeros_like(a["do"]), torch.zeros_like(a["ds"])
    leaves = {n: a[n].detach().requires_grad_(True) for n in ("q", "k", "v", "g", "s0")}
    for which in (0, 1):
        outs = sequence.linear_attention(*(leaves[n] for n in ("q", "k", "v", "g")), state=leaves["s0"], return_state=True)
        grads = torch.autograd.grad(outs[which], list(leaves.values()), (a["do"], a["ds"])[which])
        got = {"d" + n: x for n, x in zip(leaves, grads)}
        _compare(got, {**a, **({"ds": zero_s} if which == 0 else {"do": zero_o})})


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_strides_and_views(dtype):
    """Views of a fused projection, heads before tokens, a head shared by stride zero, channels cut out of wider rows (whose
    other channels hold NaN), and an offset that leaves no address aligned."""
    from pathsig_amd import sequence
    B, L, H, Dk, Dv = 2, 75, 2, 24, 40
    a = _inputs(B, L, H, H, Dk, Dv, dtype, seed=40)
    want = _run(a)
    fused = torch.cat([a[n].flatten(2) for n in ("q", "k", "v")], dim=-1)
    q, k, v = fused.split((H * Dk, H * Dk, H * Dv), dim=-1)
    views = {"fused": {"q": q.unflatten(-1, (H, Dk)), "k": k.unflatten(-1, (H, Dk)), "v": v.unflatten(-1, (H, Dv))},
             "heads first": {n: a[n].transpose(1, 2).contiguous().transpose(1, 2) for n in ("q", "k", "v")},
             "tokens first": {n: a[n].transpose(0, 1).contiguous().transpose(0, 1) for n in ("q", "k", "v")},
             "channels apart": {n: a[n].transpose(2, 3).contiguous().transpose(2, 3) for n in ("q", "k", "v")}}
    odd = {}
    for n in ("q", "k", "v"):
        wide = torch.full((*a[n].shape[:-1], a[n].shape[-1] + 8), math.nan, dtype=dtype, device=DEV)
        wide[..., :a[n].shape[-1]] = a[n]
        odd[n] = wide[..., :a[n].shape[-1]]
    views["cut out"] = odd
    flat = {}
    for n in ("q", "k", "v"):
        store = torch.empty(a[n].numel() + 1, dtype=dtype, device=DEV)
        store[1:] = a[n].flatten()
        flat[n] = store[1:].view(a[n].shape)
    views["off by one"] = flat
    for name, view in views.items():
        got = _run({**a, **view})
        for n in want:
            # (the same kernels or their form for single elements: the same order of sums)
            assert torch.equal(got[n], want[n]), (name, n)
    one = a["k"][:, :, :1]
    got = _run({**a, "k": one.expand(-1, -1, H, -1)})
    _compare(got, {**a, "k": one.expand(-1, -1, H, -1)})
    # heads of odd width cut out of rows of whole vectors
    b = _inputs(1, 40, 1, 1, 21, 35, dtype, seed=41)
    wide = {}
    for n in ("q", "k", "v"):
        wide[n] = torch.full((*b[n].shape[:-1], 64), math.nan, dtype=dtype, device=DEV)[..., :b[n].shape[-1]]
        wide[n].copy_(b[n])
    _compare(_run({**b, **wide}), b)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_decays_at_their_ends(dtype):
    """No decay (a plain sum), decays that underflow within a chunk, and minus infinity (a memory of one token)."""
    a = _inputs(2, 140, 4, 2, 16, 24, dtype, seed=50)
    a["g"] = torch.tensor([0.0, -3.0, -200.0, -1e-4], device=DEV)
    _compare(_run(a), a)
    a["g"] = torch.full((4,), -math.inf, device=DEV)
    got = _run(a, grads=False)
    assert torch.isfinite(got["out"]).all()
    kv = a["k"].double().repeat_interleave(2, 2), a["v"].double().repeat_interleave(2, 2)
    want = (a["q"].double() * kv[0]).sum(-1, keepdim=True) * kv[1] * 16 ** -0.5
    A = (a["q"].double() * kv[0]).abs().sum(-1, keepdim=True) * kv[1].abs() * 16 ** -0.5
    u = 2 ** -8 if dtype == BF16 else 2 ** -24
    assert ((got["out"].double() - want).abs() <= u * want.abs() + (2.2 if dtype == BF16 else 40) * u * A).all()
    last = kv[0][:, -1, :, :, None] * kv[1][:, -1, :, None, :]
    assert torch.equal(got["last"], last.float())


def test_level_two_of_a_signature():
    """No decay, k = x_(t-1) - x_0 + dx / 2, v = dx: the last state is level 2 of the signature."""
    import pathsig_amd as ps
    B, L, d = 3, 400, 6
    x = _randn(B, L, d, seed=60, dtype=F32, scale=0.05).cumsum(1)
    dx = x[:, 1:] - x[:, :-1]
    k, v = (x[:, :-1] - x[:, :1] + dx / 2)[:, :, None], dx[:, :, None]
    _, last = ps.sequence.linear_attention(k, k, v, torch.zeros(1, device=DEV), return_state=True)
    want = ps.Signature(depth=2)(x)[:, d:].view(B, d, d)
    A = ref.attention_bound(_double(k), _double(k), _double(v), torch.zeros(1, dtype=torch.float64, device=DEV))["last"]
    # both sum L products in 32 bits, of increments that are themselves differences rounded in 32 bits
    assert ((last[:, 0] - want).double().abs() <= 2 * 2 ** -24 * (2 * L + 64) * A[:, 0]).all()


def test_gradients_against_differences():
    """The loss is linear in q, k, v and the state, one at a time: a difference over any distance is the derivative."""
    a = _inputs(2, 180, 4, 2, 24, 32, F32, seed=70)

    def loss(b):
        got = _run(b, grads=False)
        return float((got["out"].double() * a["do"].double()).sum() + (got["last"].double() * a["ds"].double()).sum())
    got = _run(a)
    bound = ref.attention_bound(*(_double(a[n]) for n in ("q", "k", "v", "g", "s0")), None, None, _double(a["do"]), _double(a["ds"]))
    for i, n in enumerate(("q", "k", "v", "s0")):
        d = _randn(*a[n].shape, seed=80 + i, dtype=F32)
        want = (loss({**a, n: a[n] + d}) - loss({**a, n: a[n] - d})) / 2
        size = float((bound["d" + n] * (d.double().abs() + a[n].double().abs())).sum())
        assert abs(float((got["d" + n].double() * d.double()).sum()) - want) <= 2 ** -24 * (2 * 180 + 32 + 64) * size, n
    for h in range(4):
        # central difference in the decay of one head: off by eps^2 / 6 times the third derivative, at most 180^3 A
        eps = 2.0 ** -13
        step = torch.zeros(4, device=DEV)
        step[h] = eps
        want = (loss({**a, "g": a["g"] + step}) - loss({**a, "g": a["g"] - step})) / (2 * eps)
        size = float((bound["out"][:, :, h] * a["do"][:, :, h].double().abs()).sum() + (bound["last"][:, h] * a["ds"][:, h].double().abs()).sum())
        memory = 3 / -float(a["g"][h])
        tol = 2 ** -24 * (2 * 180 + 32 + 64) * size / eps * 2 ** -4 + eps ** 2 * memory ** 2 * float(bound["dg"][h])
        assert abs(float(got["dg"][h]) - want) <= tol, h


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(1, 1, 1, 1, 1), (3, 4, 2, 24, 40), (2, 2, 2, 128, 128), (2, 3, 1, 72, 33), (1, 2, 1, 255, 7),
                                   (2, 2, 1, 64, 256), (5, 1, 1, 7, 130)])
def test_steps_follow_the_sequence(shape, dtype):
    """Token by token, the state in place: the values of the whole sequence."""
    from pathsig_amd import sequence
    B, H, Hkv, Dk, Dv = shape
    L = 9
    a = _inputs(B, L, H, Hkv, Dk, Dv, dtype, seed=90)
    state = a["s0"].clone()
    where = state.data_ptr()
    outs = []
    for t in range(L):
        version = state._version
        outs.append(sequence.linear_attention_step(a["q"][:, t], a["k"][:, t], a["v"][:, t], a["g"], state))
        assert state._version > version
    assert state.data_ptr() == where
    args = [_double(a[n]) for n in ("q", "k", "v", "g", "s0")]
    want, bound = ref.attention(*args), ref.attention_bound(*args)
    u = 2 ** -8 if dtype == BF16 else 2 ** -24
    got = torch.stack(outs, 1).double()
    assert ((got - want["out"]).abs() <= u * want["out"].abs() + 2 ** -24 * (2 * L + Dk + 64) * bound["out"]).all()
    assert ((state.double() - want["last"]).abs() <= 2 ** -24 * (2 * L + 64) * bound["last"]).all()


def test_steps_of_part_of_a_pool_leave_the_rest():
    from pathsig_amd import sequence
    pool = _randn(6, 2, 16, 24, seed=100, dtype=F32)
    before = pool.clone()
    q, k, v = (_randn(2, 2, n, seed=101 + n, dtype=F32) for n in (16, 16, 24))
    sequence.linear_attention_step(q, k[:, :1], v[:, :1], torch.tensor([-0.5, -0.1], device=DEV), pool[2:4])
    assert torch.equal(pool[:2], before[:2]) and torch.equal(pool[4:], before[4:])
    assert not torch.equal(pool[2:4], before[2:4])


def test_refusals_on_the_device():
    from pathsig_amd import sequence
    a = _inputs(2, 8, 2, 1, 8, 8, F32, seed=110)
    call = lambda **e: sequence.linear_attention(*({**a, **e}[n] for n in ("q", "k", "v", "g")), state={**a, **e}["s0"],  # noqa: E731
                                                 lengths=e.get("lengths"))
    for bad in (dict(q=a["q"].half()), dict(k=a["k"].bfloat16()), dict(g=a["g"].double()), dict(g=a["g"][:1]), dict(s0=a["s0"].double()),
                dict(s0=a["s0"][:1]), dict(k=a["k"][:, :4]), dict(lengths=torch.ones(3, device=DEV, dtype=torch.int32)),
                dict(lengths=torch.ones(2, device=DEV)), dict(lengths=torch.ones(2, dtype=torch.int32)), dict(k=a["k"].cpu())):
        with pytest.raises(RuntimeError):
            call(**bad)
    step = [a[n][:, 0] for n in ("q", "k", "v")]
    with pytest.raises(RuntimeError, match="in place"):
        sequence.linear_attention_step(*step, a["g"], a["s0"].transpose(2, 3))
    with pytest.raises(RuntimeError, match="no gradient"):
        sequence.linear_attention_step(step[0].requires_grad_(True), *step[1:], a["g"], a["s0"])
    with pytest.raises(RuntimeError):
        q = a["q"].clone().requires_grad_(True)
        out = sequence.linear_attention(q, a["k"], a["v"], a["g"])
        (grad,) = torch.autograd.grad(out.sum(), q, create_graph=True)
        torch.autograd.grad(grad.sum(), q)


def test_axes_of_one_and_decays_that_are_no_number():
    from pathsig_amd import sequence
    a = _inputs(2, 1, 2, 1, 8, 16, F32, seed=115)
    want = sequence.linear_attention(a["q"], a["k"], a["v"], a["g"])
    far = {n: torch.as_strided(a[n], a[n].shape, (a[n].stride(0), 2 ** 26, *a[n].stride()[2:])) for n in ("q", "k", "v")}
    assert torch.equal(sequence.linear_attention(far["q"], far["k"], far["v"], a["g"]), want)
    a["g"][1] = math.nan
    out, last = sequence.linear_attention(a["q"], a["k"], a["v"], a["g"], state=a["s0"], return_state=True)
    assert out[:, :, 1].isnan().all() and last[:, 1].isnan().all() and torch.isfinite(out[:, :, 0]).all()
    state = a["s0"].clone()
    sequence.linear_attention_step(a["q"][:, 0], a["k"][:, 0], a["v"][:, 0], a["g"], state)
    assert state[:, 1].isnan().all() and torch.isfinite(state[:, 0]).all()
    with torch.inference_mode():
        state = a["s0"].clone()
        sequence.linear_attention_step(a["q"][:, 0], a["k"][:, 0], a["v"][:, 0], a["g"], state)
    kept = state.clone()
    with torch.no_grad(), pytest.raises(RuntimeError, match="[Ii]nference"):
        sequence.linear_attention_step(a["q"][:, 0], a["k"][:, 0], a["v"][:, 0], a["g"], state)
    assert torch.equal(state[:, 0], kept[:, 0])
    with pytest.raises(RuntimeError):
        sequence.linear_attention(a["q"][..., :0], a["k"][..., :0], a["v"], a["g"])


def test_nothing_to_do():
    from pathsig_amd import sequence
    g = torch.tensor([-0.1, -0.2], device=DEV, requires_grad=True)
    for B, L in ((0, 5), (2, 0)):
        q, k, v = (torch.zeros(B, L, n, 8, device=DEV, requires_grad=True) for n in (2, 1, 1))
        s = _randn(B, 2, 8, 8, seed=120, dtype=F32).requires_grad_(True)
        out, last = sequence.linear_attention(q, k, v, g, state=s, return_state=True)
        assert out.shape == (B, L, 2, 8) and torch.equal(last, s)
        grads = torch.autograd.grad((out.sum() + (last * 3).sum(),), (q, k, v, g, s))
        assert torch.equal(grads[4], torch.full_like(s, 3.0)) and torch.equal(grads[3], torch.zeros_like(g))
    assert sequence.linear_attention_step(torch.zeros(0, 2, 8, device=DEV), torch.zeros(0, 1, 8, device=DEV), torch.zeros(0, 1, 8, device=DEV),
                                          g.detach(), torch.zeros(0, 2, 8, 8, device=DEV)).shape == (0, 2, 8)


def test_same_call_same_bits_on_another_stream():
    a = _inputs(2, 1500, 2, 1, 64, 64, BF16, seed=130)
    want = _run(a)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    results = []
    for s in streams:  # two calls at once
        with torch.cuda.stream(s):
            results.append(_run(a))
    torch.cuda.synchronize()
    for got in results:
        for n in want:
            assert torch.equal(got[n], want[n]), n


def test_captured_and_replayed():
    """A forward with its backward and steps in graphs, replayed on new inputs with eager work in between."""
    from pathsig_amd import sequence
    a = _inputs(2, 700, 2, 1, 32, 64, BF16, seed=140)
    leaves = {n: a[n].clone().requires_grad_(True) for n in ("q", "k", "v", "g", "s0")}

    def work():
        outs = sequence.linear_attention(*(leaves[n] for n in ("q", "k", "v", "g")), state=leaves["s0"], return_state=True)
        return [o.detach() for o in outs] + list(torch.autograd.grad(outs, list(leaves.values()), (a["do"], a["ds"])))

    state = a["s0"].clone()

    def step():
        return sequence.linear_attention_step(a["q"][:, 0], a["k"][:, 0], a["v"][:, 0], a["g"], state)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work(), step()
    torch.cuda.synchronize()
    graph, step_graph = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        results = work()
    with torch.cuda.graph(step_graph):
        answer = step()
    for i in range(4):
        fresh = _inputs(2, 700, 2, 1, 32, 64, BF16, seed=150 + i)
        with torch.no_grad():
            for n in leaves:
                leaves[n].copy_(fresh[n])
            a["q"].copy_(fresh["q"])
        graph.replay()
        eager = work()
        torch.cuda.synchronize()
        for x, y in zip(results, eager):
            assert torch.equal(x, y)
        kept = state.clone()
        step_graph.replay()
        want = sequence.linear_attention_step(a["q"][:, 0], a["k"][:, 0], a["v"][:, 0], a["g"], kept)
        assert torch.equal(answer, want) and torch.equal(state, kept)


def test_c_abi_by_itself():
    """Raw pointers, no torch operators: the forward keeps its workspace for the backward, or the backward works it out again."""
    from pathsig_amd import _load
    lib = _load.lib()
    B, L, H, Hkv, Dk, Dv = 2, 2600, 2, 1, 32, 48
    a = _inputs(B, L, H, Hkv, Dk, Dv, BF16, seed=160)
    c = _load.LinearAttentionCall(dtype=2, B=B, L=L, H=H, Hkv=Hkv, Dk=Dk, Dv=Dv, scale=Dk ** -0.5, learned_decay=1,
                                  log_decay=a["g"].data_ptr(), lengths=None)
    for n in ("q", "k", "v"):
        getattr(c, n + "_stride")[:] = a[n].stride()[:3]
    ref_c = ctypes.byref(c)
    stream = ctypes.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: None if t is None else t.data_ptr()  # noqa: E731
    size = lib.pathsig_linattn_forward_workspace(ref_c)
    ws = torch.empty(size, dtype=torch.uint8, device=DEV)
    out, last = torch.empty_like(a["do"]), torch.empty_like(a["s0"])
    assert lib.pathsig_linattn_forward(ref_c, p(a["q"]), p(a["k"]), p(a["v"]), p(a["s0"]), p(out), p(last), p(ws), size, stream) == 0
    back_size = lib.pathsig_linattn_backward_workspace(ref_c, 1)
    want = _run(a)
    assert torch.equal(out, want["out"]) and torch.equal(last, want["last"])
    for kept in (ws, None):
        back = torch.empty(back_size, dtype=torch.uint8, device=DEV)
        got = {n: torch.full_like(want[n], math.nan) for n in ("dq", "dk", "dv", "dg", "ds0")}
        rc = lib.pathsig_linattn_backward(ref_c, p(a["q"]), p(a["k"]), p(a["v"]), p(a["s0"]), p(kept), size if kept is not None else 0,
                                          p(a["do"]), p(a["ds"]), p(got["dq"]), p(got["dk"]), p(got["dv"]), p(got["dg"]), p(got["ds0"]),
                                          p(back), back_size, stream)
        assert rc == 0, lib.pathsig_last_error()
        for n in got:
            assert torch.equal(got[n], want[n]), n


def test_many_sequences_and_heads():
    """More blocks than the device takes at once; one head of sixty-four shares its keys with all."""
    a = _inputs(40, 70, 64, 1, 16, 16, BF16, seed=170)
    _compare(_run(a), a)


def test_offsets_past_32_bits():
    """A batch whose tensors hold more than 2^31 elements: the last sequence is answered like the same one alone."""
    from pathsig_amd import sequence
    B, L, H, D = 65, 32768, 8, 128
    g = torch.tensor([-0.01 * (h + 1) for h in range(H)], device=DEV)
    with torch.no_grad():
        q = torch.zeros(B, L, H, D, dtype=BF16, device=DEV)
        assert q.numel() > 2 ** 31
        last = _randn(1, L, H, D, seed=180, dtype=F32).bfloat16()
        q[-1:] = last
        out = sequence.linear_attention(q, q, q, g)
        want = sequence.linear_attention(last, last, last, g)
        # (one sequence alone is cut into pieces, whose states meet in another order)
        err = (out[-1:].float() - want.float())
        assert float(err.square().mean().sqrt()) <= 2 ** -7 * float(want.float().square().mean().sqrt())
        assert (out[:-1] == 0).all()


@pytest.mark.parametrize("Dk, Dv", [(18, 10), (64, 128), (128, 20), (128, 128), (256, 24), (256, 128)])
@pytest.mark.parametrize("L", [1, 2, 7, 32])
def test_scores_of_a_few_tokens_are_not_rounded_to_the_type(L, Dk, Dv):
    """bfloat16 answers and gradients of up to 32 tokens without a state are rounded once, at the end: half a step 2^-8 of the
    value.  With A as above, before that: scores in two terms, 2^-16 A; sums of up to 256 + 32 terms in 32 bits, 2^-15 A; powers
    of the decay, 2^-20 A: below 2^-14 A together.  (A score rounded to the type would be another 2^-8 |o| off where L is 1.)"""
    from pathsig_amd import sequence
    a = _inputs(3, L, 4, 4, Dk, Dv, BF16, seed=60 + L, state=False)
    leaves = [a[n].detach().requires_grad_(True) for n in ("q", "k", "v")]
    out = sequence.linear_attention(*leaves, a["g"])
    out.backward(a["do"])
    exact = [_double(a[n]) for n in ("q", "k", "v", "g")]
    do = _double(a["do"])
    want, size = ref.attention(*exact, do=do), ref.attention_bound(*exact, do=do)
    for name, got in (("out", out), ("q", leaves[0].grad), ("k", leaves[1].grad), ("v", leaves[2].grad)):
        key = name if name in want else "d" + name
        off = (got.detach().double() - want[key]).abs()
        assert bool((off <= 2.0 ** -8 * want[key].abs() + 2.0 ** -14 * size[key]).all()), (name, off.max().item())


def test_an_infinite_score_of_a_few_tokens_stays_infinite():
    from pathsig_amd import sequence
    q = torch.full((1, 2, 1, 8), 2.0 ** 127, dtype=BF16, device=DEV)
    v = torch.ones(1, 2, 1, 8, dtype=BF16, device=DEV)
    out = sequence.linear_attention(q, q, v, torch.zeros(1, dtype=F32, device=DEV))
    assert bool(torch.isposinf(out).all())
