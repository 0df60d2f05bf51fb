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
