"""Clipping writes through addresses: who relies on a tensor's version counter has to see it."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("view", ["whole", "transposed", "columns"])
def test_every_written_tensor_gets_a_new_version(view):
    from lsr import clip_grads
    form = {"whole": lambda t: t, "transposed": lambda t: t.t(), "columns": lambda t: t[:, 2:9]}[view]
    ts = [form(torch.ones(20, 30, device="cuda")) for _ in range(3)]
    outs = [form(torch.ones(20, 30, device="cuda")) for _ in range(3)]
    before = [t._version for t in ts + outs]
    clip_grads(ts, 1.0)
    assert all(t._version > v for t, v in zip(ts, before))
    before = [t._version for t in ts + outs]
    clip_grads(ts, 1.0, out=outs)
    assert [t._version for t in ts] == before[:3]  # read only
    assert all(t._version > v for t, v in zip(outs, before[3:]))
    with torch.inference_mode():
        clip_grads([torch.ones(5, device="cuda")], 1.0)  # has no counter


def test_a_value_saved_for_a_backward_pass_is_not_clipped_unnoticed():
    from lsr import clip_grads
    g = torch.ones(10, device="cuda")
    w = torch.ones(10, device="cuda", requires_grad=True)
    loss = (g * w).sum()
    clip_grads([g], 1.0)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()


def test_kronecker_factors_clipped_between_two_applications():
    """The dense operator of small factors is kept per version: after clipping it is formed anew. Both results are
    fp32-level (3xTF32, 2^-20 relative per product at most), over sums of terms of like size."""
    from lsr import clip_grads, kron
    g = torch.Generator(device="cuda").manual_seed(0)
    A, X, B = (torch.randn(s, device="cuda", generator=g) for s in ((8, 32, 32), (4096, 32, 32), (8, 32, 32)))
    kron._DENSE_CACHE.clear()
    first = kron.kron_apply(X, A, B)
    assert kron._DENSE_CACHE
    clip_grads([A], float(A.norm()) / 4)
    got, want = kron.kron_apply(X, A, B), first / 4
    assert float((got - want).norm() / want.norm()) < 1e-5
