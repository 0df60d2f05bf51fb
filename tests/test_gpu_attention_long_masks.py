"""Key masks of any length run on the tensor cores."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(n, m, h, kv, d, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda length, heads: torch.randn(1, length, heads, d, device="cuda", generator=gen).to(dtype)  # noqa: E731
    return normal(n, h), normal(m, kv), normal(m, kv), normal(n, h)


@pytest.mark.parametrize("n,h", [(3, 2), (300, 2), (1, 300)])
@pytest.mark.parametrize("m", [196608, 196609, 200000])
def test_masks_of_any_length_on_the_tensor_cores(m, n, h):
    """Bits for 196608 keys fit a block: with more the keys are dealt to several. The workspaces tell which kernels ran
    (the CUDA-core ones need none forward and a float per row backward). Bounds entry by entry, as for short sequences; the
    sums over m keys are of m / 128 tiles' sums of 128 terms, in fp32."""
    from lsr import _lib
    from lsr import attention as A
    kv, d, dtype = 1, 16, torch.bfloat16
    q, k, v, do = tensors(n, m, h, kv, d, dtype, m + n)
    mask = torch.rand(1, m, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.7
    mask[:, 1000:150000] = False
    mask[:, -5:] = True
    how = {"causal": True, "key_mask": mask}
    out, lse = A.attention_forward(q, k, v, **how)
    dq, dk, dv = A.attention_backward(do, q, k, v, out, lse, **how)
    args = A._pack(q, k, v, mask, True, None, out, lse, do, dq, dk, dv)
    lib = _lib.load()
    assert lib.lsr_attention_backward_workspace_bytes(args) > n * h * 4 + 16
    if m > 196608:
        assert lib.lsr_attention_forward_workspace_bytes(args) > 0
    # in 64 bits
    Q, DO, O = (t[0].double().transpose(0, 1) for t in (q, do, out))
    K, V = (t[0, :, 0].double() for t in (k, v))
    see = mask[0] & (torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n))
    x = (Q @ K.T) * d ** -0.5
    x = x.masked_fill(~see, float("-inf"))
    z = torch.logsumexp(x, -1)
    p = torch.exp(x - z[..., None])
    u, e = 2.0 ** -8, 2.0 ** -24
    terms = 256 + m / 128  # of a sum, one after the other
    assert float((lse[0].double() - z).abs().max()) <= 2.0 ** -18 + terms * e
    want = p @ V
    size = (p * (u + 2.0 ** -19 + terms * e)) @ V.abs()
    assert bool(((out[0].double().transpose(0, 1) - want).abs() <= size + u * (want.abs() + size)).all())
    p = torch.exp(x - lse[0].double()[..., None])
    ds = p * (DO @ V.T - (DO * O).sum(-1, keepdim=True)) * d ** -0.5
    part = p * d ** -0.5 * (DO.abs() @ V.T.abs() + (DO * O).abs().sum(-1, keepdim=True))
    eds = ds.abs() * (u + 2.0 ** -18 + terms * e) + part * 32 * e
    want, size = ds @ K, eds @ K.abs()
    assert bool(((dq[0].double().transpose(0, 1) - want).abs() <= size + u * (want.abs() + size)).all())
    rows = torch.arange(m, device="cuda") >= m - 4000  # the others' are as long again in memory
    for got, a, ea, b in ((dk, ds, eds, Q), (dv, p, p * (u + 2.0 ** -18 + terms * e), DO)):
        want = (a[:, :, rows].transpose(1, 2) @ b).sum(0)
        size = (ea[:, :, rows].transpose(1, 2) @ b.abs()).sum(0)
        assert bool(((got[0, rows, 0].double() - want).abs() <= size + u * (want.abs() + size) + 2.0 ** -130).all())
        assert not bool(got[0, ~mask[0], 0].any())
