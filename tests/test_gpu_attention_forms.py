"""Tensors of other strides give the bits of contiguous ones, and no wait of the tensor-core kernels has run out."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def odd(t):
    return torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(t.shape).copy_(t)


FORMS = {
    "odd address": odd,
    "by head": lambda t: t.transpose(1, 2).contiguous().transpose(1, 2),
    "wide rows": lambda t: torch.cat([t, t], -1)[..., :t.shape[3]],
    "entries apart": lambda t: t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0),
    "packed": lambda t: torch.stack([t, t, t], 2)[:, :, 1],
}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 128, 20, 65])
@pytest.mark.parametrize("form", FORMS)
def test_other_strides_same_bits(form, d, dtype):
    """One rule on type, head dimension and scale picks the kernels, whatever the strides: what those of the tensor
    cores cannot read in place is copied first. (Head dimensions that are no multiple of eight, and fp32, differ
    in how a tile is loaded alone.)"""
    from lsr import attention as A
    gen = torch.Generator(device="cuda").manual_seed(6)
    q, k, v, do = (torch.randn(2, 150, 3, d, device="cuda", generator=gen).to(dtype) for _ in range(4))
    mask = torch.rand(2, 150, device="cuda", generator=gen) < 0.8
    how = {"causal": True, "key_mask": mask}
    want = A.attention_forward(q, k, v, **how)
    want = want + A.attention_backward(do, q, k, v, *want, **how)
    f = FORMS[form]
    ts = [f(t) for t in (q, k, v)]
    how["key_mask"] = mask.t().contiguous().t()
    got = A.attention_forward(*ts, **how)
    got = got + A.attention_backward(f(do), *ts, f(got[0]), got[1], **how)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_an_expanded_batch_same_bits(dtype):
    from lsr import attention as A
    gen = torch.Generator(device="cuda").manual_seed(7)
    q, k, v, do = (torch.randn(1, 150, 3, 64, device="cuda", generator=gen).to(dtype).expand(3, -1, -1, -1) for _ in range(4))
    mask = (torch.rand(1, 150, device="cuda", generator=gen) < 0.8).expand(3, -1)
    got = A.attention_forward(q, k, v, key_mask=mask)
    got = got + A.attention_backward(do, q, k, v, *got, key_mask=mask)
    ts, m = [t.contiguous() for t in (q, k, v, do)], mask.contiguous()
    want = A.attention_forward(*ts[:3], key_mask=m)
    want = want + A.attention_backward(ts[3], *ts[:3], *want, key_mask=m)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


def test_no_wait_ran_out():
    """A wait that gives up leaves its code in the status word, and the outputs as they were allocated."""
    from lsr import _lib
    from lsr import attention as A
    _lib.device_status()
    gen = torch.Generator(device="cuda").manual_seed(8)
    for dtype in TYPES[:2]:
        for b, n, m, h, kv, d, causal, masked in ((1, 1, 1, 1, 1, 64, False, False), (2, 1, 5000, 8, 2, 128, True, True),
                                                  (1, 700, 700, 25, 25, 64, True, False), (3, 333, 1027, 6, 2, 80, False, True),
                                                  (1, 2000, 60, 4, 1, 64, False, True), (2, 1024, 1024, 40, 8, 128, True, True),
                                                  (2, 5, 0, 4, 2, 64, False, False), (1, 300, 40, 2, 1, 64, True, False)):
            q, do = (torch.randn(b, n, h, d, device="cuda", generator=gen).to(dtype) for _ in range(2))
            k, v = (torch.randn(b, m, kv, d, device="cuda", generator=gen).to(dtype) for _ in range(2))
            mask = torch.rand(b, m, device="cuda", generator=gen) < 0.4 if masked else None
            if masked and b > 1:
                mask[1] = False
            for _ in range(20):
                out, lse = A.attention_forward(q, k, v, causal=causal, key_mask=mask)
                A.attention_backward(do, q, k, v, out, lse, causal=causal, key_mask=mask)
    assert _lib.device_status() == 0


@pytest.mark.parametrize("dtype", TYPES)
def test_entries_of_a_batch_more_than_2_31_apart(dtype):
    from lsr import attention as A
    gen = torch.Generator(device="cuda").manual_seed(9)
    buf = torch.empty(2 ** 31 + 70000, dtype=dtype, device="cuda")
    far = [buf[o:].as_strided((2, 130, 2, 64), (2 ** 31, 128, 64, 1)) for o in (0, 16640, 33280)]
    near = [torch.randn(t.shape, device="cuda", generator=gen).to(dtype) for t in far]
    for t, x in zip(far, near):
        t.copy_(x)
    do = torch.randn(2, 130, 2, 64, device="cuda", generator=gen).to(dtype)
    got, want = [], []
    for ts, r in ((far, got), (near, want)):
        r += A.attention_forward(*ts, causal=True)
        r += A.attention_backward(do, *ts, *r, causal=True)
    assert all(torch.equal(x, y) for x, y in zip(got, want))


@pytest.mark.parametrize("more", [0, 1])
def test_a_grid_that_fills_the_gpu_is_not_split(more):
    """A block of two query tiles has an SM to itself: with one for each SM, keys dealt to two would only queue."""
    from lsr import _lib
    from lsr import attention as A
    h = torch.cuda.get_device_properties(0).multi_processor_count + more
    q, k = (torch.zeros(1, n, h, 64, device="cuda", dtype=torch.bfloat16) for n in (256, 1024))
    out, lse = A.attention_forward(q, k, k)
    assert _lib.load().lsr_attention_forward_workspace_bytes(A._pack(q, k, k, None, False, None, out, lse)) == 0
