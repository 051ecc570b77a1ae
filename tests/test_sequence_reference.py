"""The 64-bit formulas that the sequence operators are tested against: their gradients against differences, and linear attention
without decay against the second level of a signature."""
from __future__ import annotations

import torch

from oracle import tensor_oracle as TO
from tests import sequence_reference as ref


def _randn(*shape, seed):
    return torch.randn(*shape, dtype=torch.float64, generator=torch.Generator().manual_seed(seed))


def _difference(f, x, direction, eps=1e-5):
    return (f(x + eps * direction) - f(x - eps * direction)) / (2 * eps)


def test_attention_gradients_against_differences():
    B, L, H, Hkv, Dk, Dv = 2, 9, 4, 2, 3, 5
    args = {"q": _randn(B, L, H, Dk, seed=1), "k": _randn(B, L, Hkv, Dk, seed=2), "v": _randn(B, L, Hkv, Dv, seed=3),
            "g": -_randn(H, seed=4).abs(), "s0": _randn(B, H, Dk, Dv, seed=5)}
    lengths = torch.tensor([9, 4])
    do, ds = _randn(B, L, H, Dv, seed=6), _randn(B, H, Dk, Dv, seed=7)
    got = ref.attention(**args, lengths=lengths, do=do, ds=ds)
    for i, name in enumerate(args):
        direction = _randn(*args[name].shape, seed=20 + i)

        def loss(x):
            o = ref.attention(**{**args, name: x}, lengths=lengths)
            return float((o["out"] * do).sum() + (o["last"] * ds).sum())
        want = _difference(loss, args[name], direction)
        assert abs(float((got["d" + name] * direction).sum()) - want) < 1e-7 * max(1, abs(want)), name


def test_norm_gradients_against_differences():
    rows, C = 3, 7
    args = {n: _randn(rows, C, seed=i) for i, n in enumerate(("x", "gate", "residual"))}
    args.update({n: _randn(C, seed=10 + i) for i, n in enumerate(("weight", "scale", "next_weight"))})
    do, dn = _randn(rows, C, seed=30), _randn(rows, C, seed=31)
    for activation in ("silu", "sigmoid", "linear"):
        got, _ = ref.norms(**args, activation=activation, do=do, dn=dn)
        for i, name in enumerate(args):
            direction = _randn(*args[name].shape, seed=40 + i)

            def loss(x):
                o, _ = ref.norms(**{**args, name: x}, activation=activation)
                return float((o["out"] * do).sum() + (o["next"] * dn).sum())
            want = _difference(loss, args[name], direction)
            assert abs(float((got[name] * direction).sum()) - want) < 1e-6 * max(1, abs(want)), (activation, name)


def test_attention_without_decay_is_the_second_level_of_the_signature():
    B, L, d = 2, 12, 3
    x = _randn(B, L, d, seed=9).cumsum(1)
    dx = x[:, 1:] - x[:, :-1]
    k, v = (x[:, :-1] - x[:, :1] + dx / 2)[:, :, None], dx[:, :, None]
    last = ref.attention(k, k, v, torch.zeros(1, dtype=torch.float64))["last"]
    want = TO.signature(x, 2)[:, d:].reshape(B, d, d)
    assert float((last[:, 0] - want).abs().max()) < 1e-12
