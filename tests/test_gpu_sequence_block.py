"""The sequence operators together, as a model uses them: log-signatures of sliding windows, projected, through a block of linear
attention between its norms; trained, and streamed with the state carried from window to window."""
from __future__ import annotations

import pytest
import torch
from torch import nn

from tests.helpers import brownian_path

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.fixture(autouse=True)
def float32_by_default():
    """Tensors made here without a type are float32, whatever the tests before left as the default."""
    before = torch.get_default_dtype()
    torch.set_default_dtype(torch.float32)
    yield
    torch.set_default_dtype(before)




class Block(nn.Module):
    def __init__(self, C, H, Dk, Dv, learn_decay):
        super().__init__()
        from pathsig_amd import sequence
        self.shape = (H, Dk, Dv)
        self.before = sequence.NormBefore(channels=C)
        self.project = nn.Linear(C, H * (2 * Dk + 2 * Dv), bias=False, device=DEV)
        self.attend = sequence.LinearAttention(num_heads=H, learn_decay=learn_decay)
        self.heads = sequence.NormAfter(channels=Dv)
        self.join = nn.Linear(H * Dv, C, bias=False, device=DEV)
        self.after = sequence.NormAfter(channels=C, residual_scale=0.5, next_norm=True)

    def parts(self, x):
        H, Dk, Dv = self.shape
        return [t.unflatten(-1, (H, -1)) for t in
                self.project(self.before(x)).split((H * Dk, H * Dk, H * Dv, H * Dv), dim=-1)]

    def finish(self, x, heads, gate):
        return self.after(self.join(self.heads(heads, gate=gate).flatten(-2)), residual=x)

    def forward(self, x, state=None, lengths=None):
        q, k, v, gate = self.parts(x)
        out, last = self.attend(q, k, v, state=state, lengths=lengths, return_state=True)
        return (*self.finish(x, out, gate), last)

    def step(self, x, state):
        q, k, v, gate = self.parts(x)
        return self.finish(x, self.attend.step(q, k, v, state), gate)


def _features(B, L, d, depth, C, seed):
    import pathsig_amd as ps
    path = brownian_path(B, L, d, seed=seed).float().to(DEV).requires_grad_(True)
    starts = torch.arange(0, L - 31, 8, device=DEV)
    proj = ps.projections.lyndon(depth=depth, path_dim=d)
    logsig = ps.LogSignature(depth=depth, projection=proj, windows=torch.stack([starts, starts + 32], 1))(path)
    return path, logsig


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_trained(dtype):
    torch.manual_seed(1)
    B, C, H, Dk, Dv = 3, 96, 3, 16, 24
    path, logsig = _features(B, 900, 4, 3, C, seed=2)
    embed = nn.Linear(logsig.shape[-1], C, bias=False, device=DEV)
    block = Block(C, H, Dk, Dv, learn_decay=True)
    embed.to(dtype)
    for m in (block.before, block.project, block.heads, block.join, block.after):
        m.to(dtype)
    lengths = torch.tensor([logsig.shape[1], 0, 17], device=DEV)
    x = embed(logsig.to(dtype))
    out, normed, last = block(x, lengths=lengths)
    assert out.shape == normed.shape == x.shape and last.shape == (B, H, Dk, Dv)
    loss = normed.float().square().mean() + out.float().mean() + last.square().mean()
    leaves = [path, *embed.parameters(), *block.parameters()]
    grads = torch.autograd.grad(loss, leaves)
    for leaf, grad in zip(leaves, grads):
        assert grad.shape == leaf.shape and torch.isfinite(grad).all()
        assert float(grad.abs().max()) > 0
    # (what reaches the path of a sequence without tokens comes through the residual alone)
    assert float(grads[0][1].abs().max()) > 0


def test_gradient_of_the_whole_against_differences():
    torch.manual_seed(3)
    C, H, Dk, Dv = 40, 2, 8, 12
    block = Block(C, H, Dk, Dv, learn_decay=True)
    x = torch.randn(2, 70, C, device=DEV)
    up = torch.randn(2, 70, C, device=DEV) / 70

    def loss(x):
        out, normed, _ = block(x)
        return (out.double() * up).sum() + (normed.double() * up).sum()
    x.requires_grad_(True)
    (grad,) = torch.autograd.grad(loss(x), x)
    d = torch.randn(2, 70, C, device=DEV)
    d /= d.norm()
    eps = 2.0 ** -5
    with torch.no_grad():
        # Richardson: differences over eps and eps / 2, off by eps^4 of a function that is smooth over distances of one
        diff = [float(loss(x + e * d) - loss(x - e * d)) / (2 * e) for e in (eps, eps / 2)]
    want = (4 * diff[1] - diff[0]) / 3
    # 32-bit values of size one, some thousand of them with weights 1 / 70, over a distance of eps
    assert abs(float((grad * d).sum()) - want) < 70 ** -1 * (2 * 70 * C) ** 0.5 * 2 ** -20 / eps + 1e-2 * eps ** 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_streamed(dtype):
    """Prompt, then window by window: the values of the whole sequence."""
    torch.manual_seed(4)
    B, C, H, Dk, Dv, L, first = 2, 64, 4, 16, 16, 96, 70
    block = Block(C, H, Dk, Dv, learn_decay=False)
    for m in (block.before, block.project, block.heads, block.join, block.after):
        m.to(dtype)
    x = torch.randn(B, L, C, device=DEV).to(dtype)
    with torch.no_grad():
        out, normed, last = block(x)
        a, b, state = block(x[:, :first])
        outs, nexts = [a], [b]
        for t in range(first, L):
            o, n = block.step(x[:, t], state)
            outs.append(o[:, None])
            nexts.append(n[:, None])
    u = 2 ** -8 if dtype == torch.bfloat16 else 2 ** -20
    for got, want in ((torch.cat(outs, 1), out), (torch.cat(nexts, 1), normed), (state, last)):
        # both sides round each of about a dozen stages of the block in their type
        err = (got.double() - want.double()).square().mean().sqrt()
        assert float(err) <= 12 * u * float(want.double().square().mean().sqrt())


def test_state_dict_and_arguments():
    from pathsig_amd import sequence
    fixed, learned = sequence.LinearAttention(num_heads=4), sequence.LinearAttention(num_heads=4, learn_decay=True)
    assert set(fixed.state_dict()) == set(learned.state_dict()) == {"log_decay"}
    assert not list(fixed.parameters()) and [tuple(p.shape) for p in learned.parameters()] == [(4,)]
    learned.load_state_dict(fixed.state_dict())
    assert (fixed.log_decay < 0).all() and (fixed.log_decay[1:] > fixed.log_decay[:-1]).all()
    given = sequence.LinearAttention(num_heads=2, log_decay=[-0.5, 0.0], scale=1.0)
    assert given.log_decay.tolist() == [-0.5, 0.0]
    assert given.new_state(3, 4, 5).shape == (3, 2, 4, 5)
    for bad in (dict(num_heads=0), dict(num_heads=2, log_decay=[0.0]), dict(num_heads=2, decay_exponents=(0.0, 1.0))):
        with pytest.raises(ValueError):
            sequence.LinearAttention(**bad)
    with pytest.raises(ValueError):
        sequence.NormAfter(channels=8, activation="relu")
    assert set(sequence.NormAfter(channels=8, residual_scale=0.1, next_norm=True).state_dict()) == {"weight", "scale", "next_weight"}
    assert set(sequence.NormAfter(channels=8).state_dict()) == {"weight"}


def test_compiled_and_traced():
    """Fake tensors, opcheck and torch.compile see the operators as they are."""
    from pathsig_amd import sequence
    q = torch.randn(2, 40, 2, 16, device=DEV, requires_grad=True)
    g = torch.tensor([-0.1, -0.2], device=DEV)
    s = torch.randn(2, 2, 16, 16, device=DEV)
    tests = ("test_schema", "test_autograd_registration", "test_faketensor")
    torch.library.opcheck(torch.ops.pathsig.linear_attention.default, (q, q, q, g, s, None, 0.25, True), test_utils=tests)
    torch.library.opcheck(torch.ops.pathsig.linear_attention_step.default,
                          (q[:, 0].detach(), q[:, 0].detach(), q[:, 0].detach(), g, s.clone(), 0.25), test_utils=("test_schema", "test_faketensor"))
    x = torch.randn(6, 32, device=DEV, requires_grad=True)
    w = torch.randn(32, device=DEV, requires_grad=True)
    torch.library.opcheck(torch.ops.pathsig.norm_join.default, (x, w, x, x, w, w, 1e-6, 0, True), test_utils=tests)

    def f(q, x):
        out = sequence.linear_attention(q, q, q, g)
        return out.sum() + sequence.norm_after(x, w, gate=x, next_weight=w)[1].sum()
    want = torch.autograd.grad(f(q, x), (q, x))
    got = torch.autograd.grad(torch.compile(f, backend="aot_eager")(q, x), (q, x))
    for a, b in zip(got, want):
        assert torch.allclose(a, b, rtol=1e-5, atol=1e-5)
