"""Attention's backward pass where the size of dout, or the number of keys, takes dS to the ends of its type's range.

dS is rounded to 16 bits for the products that take it. In fp16 it is first brought to a size that its inputs allow: with
B = 2 max |dout_i| max |v_j| over the rows of a key head (at least the largest |dS|), 2^x B lies between 2^13 and 2^14, so
that no entry overflows and an entry of any size is off by at most max(u |dS|, 2^-25 2^-x) <= u |dS| + 2^-38 B, u = 2^-11.

Roundings of different entries have nothing to do with one another: an error within +-a has a variance of at most a^2 / 3 once
it is spread over that range, and the variance of a sum is the sum of its terms'. Over thousands of results the error's norm is
the root of the summed variances to within a few percent; 1.5 times that, beside what rounding the exact result itself
costs, is the bound here. The fp32 parts (scores, exponentials, sums: see the entry-by-entry bounds of the other tests)
are added in full."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def heads(t, kv):
    """[b, n, h, d] as [b, kv, h / kv, n, d] in 64 bits"""
    b, n, h, d = t.shape
    return t.double().permute(0, 2, 1, 3).reshape(b, kv, h // kv, n, d)


def back(t):
    b, kv, g, n, d = t.shape
    return t.reshape(b, kv * g, n, d).permute(0, 2, 1, 3)


def check(got, want, var, extra, name):
    assert bool(torch.isfinite(got).all()), name
    assert bool((want.abs() < 0.9 * torch.finfo(got.dtype).max).all()), "the case itself overflows"
    own = (want.to(got.dtype).double() - want).norm()
    err = (got.double() - want).norm()
    bound = 1.5 * (own + var.sum().sqrt()) + extra.norm()
    assert float(err) <= float(bound), (name, float(err / want.norm()), float(bound / want.norm()), float(own / want.norm()))


def run(q, k, v, do, causal=False, mask=None, scale=None):
    from lsr import attention as A
    b, n, h, d = q.shape
    m, kv = k.shape[1:3]
    out, lse = A.attention_forward(q, k, v, causal=causal, key_mask=mask, scale=scale)
    grads = A.attention_backward(do, q, k, v, out, lse, causal=causal, key_mask=mask, scale=scale)
    sc = d ** -0.5 if scale is None else scale
    if mask is not None:
        k, v = (t.masked_fill(~mask[:, :, None, None], 0.0) for t in (k, v))
    Q, K, V, O, DO = heads(q, kv), heads(k, kv), heads(v, kv), heads(out, kv), heads(do, kv)
    row = lse.double().reshape(b, kv, h // kv, n, 1)
    see = torch.ones(b, 1, 1, n, m, dtype=torch.bool, device="cuda")
    if causal:
        see &= torch.arange(m, device="cuda")[None] <= torch.arange(n, device="cuda")[:, None] + (m - n)
    if mask is not None:
        see = see & mask[:, None, None, None, :]
    s = sc * (Q @ K.transpose(-1, -2))
    p = torch.where(see, torch.exp(s - torch.where(torch.isneginf(row), torch.zeros_like(row), row)), torch.zeros_like(s))
    dp = DO @ V.transpose(-1, -2) - (DO * O).sum(-1, keepdim=True)
    ds = p * dp
    T = lambda x: x.transpose(-1, -2)  # noqa: E731
    u = torch.finfo(q.dtype).eps / 2
    if q.dtype == torch.float16:
        # (row norms as the kernel has them, so that a case near a power of two is no other case)
        B = 2 * DO.norm(dim=-1).amax((2, 3)) * V.norm(dim=-1).amax((2, 3))
        low = 2.0 ** -38 * B[:, :, None, None, None]
        lop = 2.0 ** -35  # p is taken times 2^10
    else:
        low, lop = 0.0, 0.0
    vds = ((u * ds) ** 2 + low ** 2 * (p > 0)) / 3
    vp = ((u * p) ** 2 + lop ** 2 * (p > 0)) / 3
    rel = (d + 4) * E * abs(sc) * (Q.abs() @ T(K.abs())) + 2.0 ** -21 + (s.abs() + row.nan_to_num(neginf=0).abs() + 4) * E
    eds = ds.abs() * (rel + 8 * E) + p * (d + 8) * E * (DO.abs() @ T(V.abs()) + (DO * O).abs().sum(-1, keepdim=True))
    g = h // kv
    sums = lambda x: x.sum(2, keepdim=True)  # noqa: E731
    check(grads[0], back(sc * (ds @ K)), sc * sc * (vds @ K ** 2), abs(sc) * (eds + m * E * ds.abs()) @ K.abs(), "dq")
    check(grads[1], back(sc * sums(T(ds) @ Q)), sc * sc * sums(T(vds) @ Q ** 2),
          abs(sc) * sums(T(eds + g * n * E * ds.abs()) @ Q.abs()), "dk")
    check(grads[2], back(sums(T(p) @ DO)), sums(T(vp) @ DO ** 2), sums(T(p * (rel + g * n * E)) @ DO.abs()), "dv")
    return grads


def tensors(b, n, m, h, kv, d, dtype, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(s, device="cuda", generator=gen)  # noqa: E731
    return normal(b, n, h, d).to(dtype), normal(b, m, kv, d).to(dtype), normal(b, m, kv, d).to(dtype), normal(b, n, h, d)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("size", [1e-4, 1e-2, 1.0, 300.0])
@pytest.mark.parametrize("n,m,h,kv,d,causal", [
    (2048, 8192, 1, 1, 64, False), (512, 4096, 2, 1, 64, False), (2048, 2048, 2, 2, 128, True), (64, 64, 8, 2, 64, True),
    (5, 6000, 2, 1, 64, True), (4000, 70, 2, 1, 80, False)])
def test_gradients_of_any_size(n, m, h, kv, d, causal, size, dtype):
    q, k, v, do = tensors(1, n, m, h, kv, d, dtype, n + m)
    run(q, k, v, (do * size).to(dtype), causal)


@pytest.mark.parametrize("n,m", [(64, 2), (5, 4), (700, 3)])
def test_fp16_score_gradients_past_the_type(n, m):
    """|dP| of about 64000 and probabilities of a third or a half: dS is past fp16's largest, its products are not."""
    q, k, v, do = tensors(2, n, m, 8, 4, 64, torch.float16, 5)
    run(q, k, (v * 8).half(), (do * 1000).half(), scale=2.0 ** -6)


def test_fp16_heads_and_entries_of_very_different_sizes():
    """A key head's size is that of its own heads and entry, with what the mask hides left out."""
    q, k, v, do = tensors(3, 300, 500, 6, 3, 64, torch.float16, 6)
    do *= torch.tensor([1.0, 2e-4, 30.0], device="cuda")[:, None, None, None]
    do *= torch.tensor([1.0, 0.1, 1e-3, 1e-3, 50.0, 5.0], device="cuda")[:, None]
    mask = torch.rand(3, 500, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.5
    mask[2, 40:] = False
    want = run(q, k, v, do.half(), True, mask)
    v2 = v.masked_fill(~mask[:, :, None, None], math.nan)
    v2[0, :, :, ::2] = torch.where(mask[0, :, None, None], v2[0, :, :, ::2], torch.full((), 60000.0, device="cuda", dtype=torch.float16))
    assert all(torch.equal(x, y) for x, y in zip(want, run(q, k, v2, do.half(), True, mask)))


@pytest.mark.parametrize("bad", [math.inf, math.nan])
def test_fp16_one_row_that_is_not_finite_leaves_the_others(bad):
    from lsr import attention as A
    q, k, v, do = tensors(1, 200, 300, 4, 2, 64, torch.float16, 7)
    do = (do * 1e-3).half()
    do[:, 17, 1] = 0.0
    out, lse = A.attention_forward(q, k, v)
    want = A.attention_backward(do, q, k, v, out, lse)
    do[:, 17, 1] = bad
    got = A.attention_backward(do, q, k, v, out, lse)
    rows = torch.arange(200, device="cuda") != 17
    assert torch.equal(got[0][:, rows], want[0][:, rows])
    assert torch.equal(got[1][:, :, 1], want[1][:, :, 1]) and torch.equal(got[2][:, :, 1], want[2][:, :, 1])


def test_fp16_nothing_but_zeros():
    q, k, v, do = tensors(1, 130, 140, 2, 1, 64, torch.float16, 8)
    for x, y in ((v, do.half() * 0), (v * 0, do.half())):
        grads = run(q, k, x, y)
        assert not bool(grads[0].any()) and not bool(grads[1].any())
