"""Attention's gradients do not change their accuracy with the length of the sequence."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(n, m, h, kv, d, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda length, heads: torch.randn(1, length, heads, d, device="cuda", generator=gen).to(dtype)  # noqa: E731
    return normal(n, h), normal(m, kv), normal(m, kv), normal(n, h)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("longer", [513, 640])
def test_first_rows_of_a_causal_sequence_are_those_of_a_shorter_one(longer, d):
    """Queries up to 511 see the same keys in both, in the same tiles: their dq is the same bits."""
    from lsr import attention as A
    q, k, v, do = tensors(longer, longer, 40, 40, d, torch.bfloat16, longer)

    def dq(n):
        ts = [t[:, :n].contiguous() for t in (q, k, v, do)]
        out, lse = A.attention_forward(*ts[:3], causal=True)
        return A.attention_backward(ts[3], *ts[:3], out, lse, causal=True)[0]

    assert torch.equal(dq(longer)[:, :512], dq(512))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("n,m,causal,left", [(64, 64, True, 0), (128, 128, True, 0), (200, 200, True, 0), (700, 700, True, 0), (3000, 3000, True, 0),
                                             (300, 100, False, 0), (300, 140, True, 0), (900, 900, True, 700), (90, 900, False, 800)])
def test_score_gradients_of_rows_of_few_keys_are_not_rounded_once_only(n, m, causal, left, dtype):
    """dS enters its products in two 16-bit parts where rows see at most 128 keys: off by u^2 |dS|, u = eps / 2 (and fp16's
    spacing, 2^-38 of 2 max |dout| max |v|), beside the fp32 errors of the scores (see the other tests). With d the sum
    of that over a result's terms, rounding it leaves at most |rounding of the exact result| + 2 d: within d of a
    midpoint the two may round apart. One part alone adds about as much as the rounding itself: 1.4 times. The first 128
    rows that see a key, and the keys that they begin at. `left`: keys hidden before the first that is seen."""
    from lsr import attention as A
    q, k, v, do = tensors(n, m, 4, 2, 64, dtype, n + m)
    mask = torch.arange(m, device="cuda")[None] >= left if left else None
    how = {"causal": causal, "key_mask": mask}
    out, lse = A.attention_forward(q, k, v, **how)
    dq, dk, _ = A.attention_backward(do, q, k, v, out, lse, **how)
    Q, DO, O = (t[0].double().transpose(0, 1) for t in (q, do, out))
    K, V = (t[0].double().transpose(0, 1).repeat_interleave(2, 0) for t in (k, v))
    see = torch.arange(m, device="cuda")[None] >= left
    if causal:
        see = see & (torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n))
    see = see.expand(n, m)
    z = lse[0].double()[..., None]
    x = Q @ K.transpose(1, 2) * 0.125
    p = torch.where(see, torch.exp(x - z.masked_fill(torch.isneginf(z), 0.0)), torch.zeros_like(x))
    ds = p * (DO @ V.transpose(1, 2) - (DO * O).sum(-1, keepdim=True)) * 0.125
    e, u = 2.0 ** -24, torch.finfo(dtype).eps / 2
    part = 0.125 * p * (DO.abs() @ V.transpose(1, 2).abs() + (DO * O).abs().sum(-1, keepdim=True))
    rel = 68 * e * 0.125 * (Q.abs() @ K.transpose(1, 2).abs()) + 2.0 ** -21 + (x.abs() + z.nan_to_num(neginf=0).abs() + 4) * e
    low = 2.0 ** -38 * 2 * 0.125 * float(DO.norm(dim=-1).max() * V.norm(dim=-1).max()) if dtype == torch.float16 else 0.0
    eds = ds.abs() * (rel + u * u + 8 * e) + part * 72 * e + low * (p > 0)

    def check(got, want, d, name):
        own = (want.to(dtype).double() - want).norm()
        err, bound = float((got.double() - want).norm()), float(own + 2 * d.norm())
        assert err <= bound, (name, err / float(own), bound / float(own))

    first = max(0, left + n - m) if causal else 0
    rows = slice(first, min(n, first + 128))
    check(dq[0, rows].transpose(0, 1), (ds @ K)[:, rows], ((eds + min(m, 256) * e * ds.abs()) @ K.abs())[:, rows], "dq")
    if n <= 300:
        pairs = lambda t: t.reshape(2, 2, *t.shape[1:]).sum(1)  # noqa: E731
        keys = slice(left, min(m, 128 if not left else m))
        check(dk[0, keys].transpose(0, 1), pairs(ds.transpose(1, 2) @ Q)[:, keys],
              pairs((eds + 2 * n * e * ds.abs()).transpose(1, 2) @ Q.abs())[:, keys], "dk")
