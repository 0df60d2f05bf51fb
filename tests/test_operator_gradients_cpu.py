"""CPU: what has no derivative says so instead of passing for a constant. The launches are replaced by stand-ins: it is
what autograd is told that is tested."""
from __future__ import annotations

import pytest
import torch
import torch.autograd.forward_ad as fwd


@pytest.fixture
def stub(monkeypatch):
    import lsr.attention as A
    import lsr.grad as G
    monkeypatch.setattr(A, "_forward", lambda q, k, v, *how: (q.detach() * 2, q.new_zeros(q.shape[0], q.shape[2], q.shape[1])))
    monkeypatch.setattr(A, "_backward", lambda do, q, k, v, *how: (q.detach() * 3, k.detach() * 4, v.detach() * 5))
    monkeypatch.setattr(G, "_check_list", lambda ts, what: (list(ts), [], [], True))
    monkeypatch.setattr(G, "_norm", lambda ts, *rest: torch.stack([t.detach().square().sum() for t in ts]).sum().sqrt())
    return A, G


def qkv(**how):
    g = torch.Generator().manual_seed(0)
    return [torch.randn(1, 3, 2, 8, generator=g).requires_grad_(how.get("grad", False)) for _ in range(3)]


@pytest.mark.parametrize("which", [0, 1, 2])
@pytest.mark.parametrize("grad_mode", [True, False])
@pytest.mark.parametrize("name", ["attention", "attention_forward", "attention_backward", "grad_norm", "clip_grads"])
def test_forward_mode_is_refused(stub, name, grad_mode, which):
    A, G = stub
    with torch.set_grad_enabled(grad_mode), fwd.dual_level():
        ts = qkv()
        ts[which] = fwd.make_dual(ts[which], torch.ones_like(ts[which]))
        call = {"attention": lambda: A.attention(*ts), "attention_forward": lambda: A.attention_forward(*ts),
                "attention_backward": lambda: A.attention_backward(ts[0], *ts, ts[0], torch.zeros(1, 2, 3)),
                "grad_norm": lambda: G.grad_norm(ts), "clip_grads": lambda: G.clip_grads(ts, 1.0)}[name]
        with pytest.raises(NotImplementedError):
            call()
        # duals elsewhere are no concern of the call
        plain = qkv()
        assert torch.equal(A.attention(*plain), plain[0] * 2) and float(G.grad_norm(plain)) > 0


def test_a_gradient_that_is_not_there_raises(stub):
    _, G = stub
    ts = qkv(grad=True)
    loss = ts[0].square().sum() + G.grad_norm(ts)  # as a penalty beside a loss that has a gradient
    with pytest.raises(RuntimeError, match="grad_norm"):
        loss.backward()
    with torch.no_grad():
        quiet = G.grad_norm(ts)
    assert not quiet.requires_grad and torch.equal(quiet, G.grad_norm(ts).detach())
    assert not G.grad_norm(qkv()).requires_grad


def test_the_two_halves_lie_outside_autograd(stub):
    """As a program that joins them by hand calls them: the output is a leaf of its own."""
    A, _ = stub
    ts = qkv(grad=True)
    out, lse = A.attention_forward(*ts)
    assert not out.requires_grad and not lse.requires_grad
    out.requires_grad_(True).square().sum().backward()
    assert not any(g.requires_grad for g in A.attention_backward(out.grad, *ts, out, lse))


def test_attention_still_has_its_gradients(stub):
    A, _ = stub
    ts = qkv(grad=True)
    A.attention(*ts).sum().backward()
    assert all(torch.equal(t.grad, t.detach() * f) for t, f in zip(ts, (3, 4, 5)))
    with torch.no_grad():
        assert not A.attention(*ts).requires_grad
