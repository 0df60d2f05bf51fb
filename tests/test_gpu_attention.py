"""Softmax attention and its gradients (lsr.attention) against the formulas in float64.

Tolerances are worked out entry by entry from the float64 result. With u = eps / 2 of the tensors'
type (its rounding of a value) and e = 2^-24:
* a score is a product of dim terms and its scaling in fp32, taken in any order: off by at most
  (dim + 4) e sum |q| |k| scale; the exponential turns that into a relative error of p, to which its
  own error (2^-21) and the rounding of its argument ((|s| + |lse| + 4) e) are added;
* p and ds are rounded to the type (16-bit types: u relative, or half the spacing of its smallest
  values) before they are multiplied; the sums over n terms are in fp32: n e of the sum of the terms' sizes;
* the result is rounded to the type."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import attention as oa

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def unit(dtype):
    return torch.finfo(dtype).eps / 2


def least(dtype):
    return torch.finfo(dtype).smallest_normal * unit(dtype)


def tensors(b, n, m, h, hk, d, dtype, seed=0, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*s):
        return torch.randn(s, device="cuda", generator=g)

    return ((normal(b, n, h, d) * spread).to(dtype), normal(b, m, hk, d).to(dtype), normal(b, m, hk, d).to(dtype),
            normal(b, n, h, d).to(dtype))


def f64(t):
    return t.detach().double().cpu().numpy()


def close(got, want, size, dtype, name):
    """|got - want| within `size`, and got's rounding to its type."""
    assert np.isfinite(f64(got)).all(), name
    tol = size + unit(dtype) * (np.abs(want) + size) + least(dtype)
    err = np.abs(f64(got) - want)
    assert (err <= tol).all(), (name, float((err / tol).max()), float(err.max()))


class Case:
    """A forward and a backward pass, checked."""

    def __init__(self, q, k, v, dout, causal=False, key_mask=None, scale=None):
        from lsr import attention as A
        self.how = {"causal": causal, "key_mask": key_mask, "scale": scale}
        self.out, self.lse = A.attention_forward(q, k, v, **self.how)
        self.grads = A.attention_backward(dout, q, k, v, self.out, self.lse, **self.how)
        dt, d, n, m, g = q.dtype, q.shape[3], q.shape[1], k.shape[1], q.shape[2] // k.shape[2]
        sc = d ** -0.5 if scale is None else scale
        mask = None if key_mask is None else key_mask.cpu().numpy()
        Q, K, V, DO = (f64(t) for t in (q, k, v, dout))
        want, lse, p = oa.forward(Q, K, V, sc, causal, mask)
        got_lse = self.lse.double().cpu().numpy()
        assert np.array_equal(np.isneginf(got_lse), np.isneginf(lse))
        fin = np.where(np.isneginf(lse), 0.0, lse)
        hf = oa.heads_first
        aQ, aK, aV, aDO = np.abs(hf(Q)), np.abs(oa._visible(K, mask, g)), np.abs(oa._visible(V, mask, g)), np.abs(hf(DO))
        score = abs(sc) * (aQ @ aK.transpose(0, 1, 3, 2))  # sum |q| |k| scale
        rel = (d + 4) * E * score + 2.0 ** -21 + (score + np.abs(fin)[..., None] + 4) * E
        # lse: the weighted mean of the scores' errors, and fp32's own rounding
        tol = (p * rel).sum(-1) + m * E + 4 * E * (np.abs(fin) + 1)
        assert (np.abs(np.where(np.isneginf(got_lse), 0.0, got_lse) - fin) <= tol).all()
        u, lo = (0.0, 0.0) if dt == torch.float32 else (unit(dt), least(dt))
        # p is rounded relative to its row's largest, which is at least 1 / m of the row's sum
        size = (p * (rel + u + (p * rel).sum(-1, keepdims=True) + 2 * m * E) + lo * m * (p.max(-1, keepdims=True))) @ aV
        close(self.out, want, size.transpose(0, 2, 1, 3), dt, "out")

        dq, dk, dv, p, ds = oa.backward(DO, Q, K, V, f64(self.out), self.lse.double().cpu().numpy(), sc, causal, mask)
        ep = p * rel  # of a probability
        parts = aDO @ aV.transpose(0, 1, 3, 2) + (aDO * np.abs(hf(f64(self.out)))).sum(-1, keepdims=True)
        eds = np.abs(ds) * rel + abs(sc) * p * (d + 4) * E * parts
        eds = eds + u * np.abs(ds) + abs(sc) * lo + 4 * E * np.abs(ds)
        ep = ep + u * p + lo * (p > 0)

        def shared(x):
            b, h, mm, dd = x.shape
            return x.reshape(b, h // g, g, mm, dd).sum(2).transpose(0, 2, 1, 3)

        t = lambda x: x.transpose(0, 1, 3, 2)  # noqa: E731
        close(self.grads[0], dq, ((eds + m * E * np.abs(ds)) @ aK).transpose(0, 2, 1, 3), dt, "dq")
        close(self.grads[1], dk, shared(t(eds + g * n * E * np.abs(ds)) @ aQ), dt, "dk")
        close(self.grads[2], dv, shared(t(ep + g * n * E * p) @ aDO), dt, "dv")


TYPES = [torch.bfloat16, torch.float16, torch.float32]
SHAPES = [  # b, n, m, h, hk, d
    (1, 1, 1, 1, 1, 64), (2, 1, 300, 4, 2, 64), (1, 300, 1, 2, 1, 64), (2, 128, 128, 2, 2, 64), (1, 129, 127, 3, 1, 64),
    (1, 257, 511, 2, 1, 128), (2, 65, 200, 2, 2, 80), (1, 200, 333, 4, 1, 8), (3, 31, 33, 1, 1, 128), (1, 640, 640, 2, 1, 64),
    (1, 100, 150, 2, 2, 20), (1, 70, 70, 1, 1, 1), (1, 130, 130, 2, 1, 127)]


@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_shapes_and_types(shape, dtype, causal):
    Case(*tensors(*shape, dtype, seed=sum(shape)), causal=causal)


@pytest.mark.parametrize("n,m,d,kv,causal,masked", [
    (400, 400, 64, 40, True, False), (260, 300, 128, 8, False, False), (300, 600, 64, 20, True, True),
    (600, 300, 128, 40, True, False), (257, 140, 80, 8, False, True)])
def test_many_heads(n, m, d, kv, causal, masked):
    """Enough blocks for every SM, lengths that end inside a tile and inside a pair of tiles."""
    q, k, v, do = tensors(2, n, m, 40, kv, d, torch.bfloat16, seed=n + d)
    mask = None
    if masked:
        mask = torch.arange(m, device="cuda") < torch.tensor([[m - 3], [m // 2]], device="cuda")
    Case(q, k, v, do, causal=causal, key_mask=mask)


@pytest.mark.parametrize("causal,masked", [(False, False), (True, True)])
@pytest.mark.parametrize("d", [64, 65, 96, 97, 128])
@pytest.mark.parametrize("b,n,m,h,kv", [(2, 300, 200, 40, 40), (1, 150, 260, 40, 8), (1, 100, 300, 16, 2), (1, 70, 300, 3, 1)])
def test_fp32_with_few_and_many_blocks(b, n, m, h, kv, d, causal, masked):
    """All divisions of a block's warps among rows and columns, and the widths of a tile."""
    q, k, v, do = tensors(b, n, m, h, kv, d, torch.float32, seed=n + d)
    mask = torch.arange(m, device="cuda").expand(b, m) < m - 37 if masked else None
    Case(q, k, v, do, causal=causal, key_mask=mask)


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("d", [65, 90, 127])
def test_16_bit_heads_of_odd_widths(dtype, d):
    Case(*tensors(1, 150, 260, 24, 8, d, dtype, seed=d), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("kind", ["right", "left", "holes", "empty entry", "one key", "far tiles"])
def test_key_masks(kind, causal, dtype):
    b, n, m = 3, 140, 390
    g = torch.Generator(device="cuda").manual_seed(5)
    j = torch.arange(m, device="cuda")
    mask = torch.ones(b, m, dtype=torch.bool, device="cuda")
    if kind == "right":
        mask = j < torch.tensor([[390], [129], [1]], device="cuda")
    elif kind == "left":
        mask = j >= torch.tensor([[0], [127], [300]], device="cuda")
    elif kind == "holes":
        mask = torch.rand(b, m, device="cuda", generator=g) < 0.5
    elif kind == "empty entry":
        mask[1] = False
    elif kind == "one key":
        mask = j == torch.tensor([[0], [200], [389]], device="cuda")
    else:
        mask = (j < 20) | (j > 380)
        mask = mask.expand(b, m)
    q, k, v, do = tensors(b, n, m, 4, 2, 64, dtype, seed=1)
    Case(q, k, v, do, causal=causal, key_mask=mask)
    # what the masked keys hold does not matter, not even to their own gradients' neighbours
    k2, v2 = (t.masked_fill(~mask[:, :, None, None], x) for t, x in ((k, math.nan), (v, math.inf)))
    from lsr import attention as A
    one = A.attention_forward(q, k, v, causal=causal, key_mask=mask)
    two = A.attention_forward(q, k2, v2, causal=causal, key_mask=mask)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    one = A.attention_backward(do, q, k, v, *one, causal=causal, key_mask=mask)
    two = A.attention_backward(do, q, k2, v2, *two, causal=causal, key_mask=mask)
    assert all(torch.equal(x, y) for x, y in zip(one, two))
    hidden = ~mask
    assert float(one[1][hidden].float().abs().sum()) == 0.0 and float(one[2][hidden].float().abs().sum()) == 0.0


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_before_the_first_key_are_empty(dtype):
    q, k, v, do = tensors(2, 300, 40, 2, 1, 64, dtype, seed=2)
    c = Case(q, k, v, do, causal=True)
    assert bool((c.out[:, :260] == 0).all()) and bool(torch.isneginf(c.lse[:, :, :260]).all())
    assert bool((c.grads[0][:, :260] == 0).all())


@pytest.mark.parametrize("dtype", TYPES[:2])
@pytest.mark.parametrize("n,m,h,hk,d,causal,masked", [(5, 1500, 2, 1, 64, True, False), (1500, 60, 4, 1, 64, False, False),
                                                      (3, 2000, 1, 1, 128, True, True), (1100, 130, 2, 2, 80, False, True)])
def test_few_rows_whose_steps_are_dealt_to_several_blocks(n, m, h, hk, d, causal, masked, dtype):
    mask = torch.arange(m, device="cuda")[None] % 7 != 3 if masked else None
    if masked and m > 1000:
        mask = mask & (torch.arange(m, device="cuda")[None] > 700)  # the first blocks' keys are all hidden
    Case(*tensors(1, n, m, h, hk, d, dtype, seed=n), causal=causal, key_mask=mask)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread", [0.0, 30.0])
def test_flat_and_peaked_rows(dtype, spread):
    """All scores 0, and scores of a few hundred that leave one key per row."""
    Case(*tensors(1, 150, 300, 2, 2, 64, dtype, seed=3, spread=spread), causal=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("scale", [-0.3, 0.0, 2.0])
def test_scales_of_either_sign(dtype, scale):
    Case(*tensors(1, 140, 150, 2, 1, 32, dtype, seed=14, spread=0.5), causal=True, scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
def test_scores_that_rise_and_fall_along_the_keys(dtype):
    """The running maximum moves at every tile, or only at the first."""
    q, k, v, do = tensors(1, 70, 900, 1, 1, 64, dtype, seed=4)
    ramp = torch.linspace(0, 4, 900, device="cuda")[None, :, None, None]
    q = q.abs()
    for r in (ramp, 4 - ramp):
        Case(q, (k * 0.1 + r).to(dtype), v, do)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("d", [64, 20, 128])
def test_strides(dtype, d):
    """The parts of one projection, [batch, heads, length, dim] transposed, misaligned and gapped tensors, a
    batch that is one tensor expanded: read in place or copied, the results are those of contiguous ones."""
    from lsr import attention as A
    b, n, h = 2, 150, 3
    g = torch.Generator(device="cuda").manual_seed(6)
    packed = torch.randn(b, n, 3 * h * d, device="cuda", generator=g).to(dtype)
    mask = torch.rand(n, b, device="cuda", generator=g).t() < 0.8
    base = packed.view(b, n, 3, h, d).unbind(2)

    def odd(t):
        buf = torch.empty(t.numel() + 1, dtype=dtype, device="cuda")[1:].view(t.shape)
        return buf.copy_(t)

    def by_head(t):
        return t.transpose(1, 2).contiguous().transpose(1, 2)

    def wide(t):
        return torch.cat([t, t], -1)[..., :d]

    def last(t):
        return t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)

    how = {"causal": True, "key_mask": mask.contiguous()}
    dout = torch.randn(b, n, h, d, device="cuda", generator=g).to(dtype)
    plain = [t.contiguous() for t in base]
    out, lse = A.attention_forward(*plain, **how)
    grads = A.attention_backward(dout, *plain, out, lse, **how)
    Case(*plain, dout, **how)
    for form in (lambda t: t, odd, by_head, wide, last):
        ts = [form(t) for t in base]
        Case(*ts, form(dout), causal=True, key_mask=mask)
    ts = [t[:1].expand(b, n, h, d) for t in plain]
    Case(*ts, dout, causal=True, key_mask=mask[:1].expand(b, n))
    del grads


@pytest.mark.parametrize("dtype", TYPES)
def test_autograd_matches_the_two_entry_points_and_sums_broadcast_keys(dtype):
    from lsr import attention as A
    q, k, v, do = tensors(2, 100, 120, 4, 2, 64, dtype, seed=8)
    leaves = [t.clone().requires_grad_(True) for t in (q, k[:1], v)]
    out = A.attention(leaves[0], leaves[1].expand_as(k), leaves[2], causal=True)
    out.backward(do)
    k = k[:1].expand_as(k)
    o, lse = A.attention_forward(q, k, v, causal=True)
    dq, dk, dv = A.attention_backward(do, q, k, v, o, lse, causal=True)
    assert torch.equal(out, o) and torch.equal(leaves[0].grad, dq) and torch.equal(leaves[2].grad, dv)
    assert torch.equal(leaves[1].grad, dk.sum(0, keepdim=True))
    with torch.no_grad():
        assert not A.attention(*leaves[:1], k, v, causal=True).requires_grad


def test_gradients_against_differences():
    """fp32, the derivative along a random direction: (f(x + t d) - f(x - t d)) / 2t with t = 2^-7. The cubic
    term is t^2 / 6 of the third derivative (bounded here by 60 |d|^3 of a sum of 40 * 64 outputs of size 1,
    far under 1e-2 of the first), rounding is 2^-23 of the sum's parts / 2t; 2 percent covers both."""
    from lsr import attention as A
    ts = tensors(1, 40, 50, 2, 1, 64, torch.float32, seed=9)
    mask = torch.rand(1, 50, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)) < 0.7
    how = {"causal": True, "key_mask": mask}
    q, k, v, do = ts
    out, lse = A.attention_forward(q, k, v, **how)
    grads = A.attention_backward(do, q, k, v, out, lse, **how)
    g = torch.Generator(device="cuda").manual_seed(2)
    for i, name in enumerate("qkv"):
        dirn = torch.randn(ts[i].shape, device="cuda", generator=g)
        f = []
        for t in (2.0 ** -7, -(2.0 ** -7)):
            x = list(ts[:3])
            x[i] = x[i] + t * dirn
            f.append(float((A.attention_forward(*x, **how)[0].double() * do.double()).sum()))
        want = (f[0] - f[1]) / 2.0 ** -6
        got = float((grads[i].double() * dirn.double()).sum())
        scale = float(grads[i].double().norm())
        assert abs(got - want) <= 0.02 * scale, (name, got, want, scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_same_bits_every_time_and_on_side_streams(dtype):
    from lsr import attention as A
    q, k, v, do = tensors(2, 500, 500, 8, 2, 64, dtype, seed=10)

    def all_of():
        o, lse = A.attention_forward(q, k, v, causal=True)
        return (o, lse) + tuple(A.attention_backward(do, q, k, v, o, lse, causal=True))

    first = all_of()
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(all_of())
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for other in got for x, y in zip(other, first))


def test_captured_and_replayed():
    from lsr import attention as A
    q, k, v, do = tensors(1, 200, 200, 4, 4, 64, torch.bfloat16, seed=11)
    A.attention_backward(do, q, k, v, *A.attention_forward(q, k, v, causal=True), causal=True)
    torch.cuda.synchronize()
    graphs, results = [], []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            o, lse = A.attention_forward(q, k, v, causal=True)
            results.append((o, lse) + tuple(A.attention_backward(do, q, k, v, o, lse, causal=True)))
        graphs.append(graph)
    q.mul_(0.5)
    want_o, want_lse = A.attention_forward(q, k, v, causal=True)
    want = (want_o, want_lse) + tuple(A.attention_backward(do, q, k, v, want_o, want_lse, causal=True))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(5):
        for graph, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                graph.replay()
    torch.cuda.synchronize()
    for r in results:
        assert all(torch.equal(x, y) for x, y in zip(r, want))


def test_a_thread_whose_first_call_this_is():
    """As an autograd worker's first backward pass: the thread has no CUDA context of its own yet."""
    import threading
    from lsr import attention as A
    q, k, v, do = tensors(1, 70, 70, 2, 2, 64, torch.bfloat16, seed=12)
    o, lse = A.attention_forward(q, k, v, causal=True)
    want = (o, lse) + tuple(A.attention_backward(do, q, k, v, o, lse, causal=True))
    torch.cuda.synchronize()
    got = []

    def work(backward_first):
        try:
            grads = A.attention_backward(do, q, k, v, o, lse, causal=True) if backward_first else ()
            got.append(tuple(A.attention_forward(q, k, v, causal=True)) + tuple(grads))
        except Exception as e:  # noqa: BLE001
            got.append(e)

    for first in (True, False):
        t = threading.Thread(target=work, args=(first,))
        t.start()
        t.join()
    torch.cuda.synchronize()
    for r in got:
        assert not isinstance(r, Exception), r
        assert all(torch.equal(x, y) for x, y in zip(r, want))


def test_nothing_to_do():
    from lsr import attention as A
    for b, n, m in ((0, 5, 5), (2, 0, 5), (2, 5, 0)):
        q, k, v, do = tensors(b, n, m, 2, 2, 64, torch.bfloat16)
        o, lse = A.attention_forward(q, k, v, causal=True)
        assert bool((o == 0).all()) and bool(torch.isneginf(lse).all())
        for x, y in zip(A.attention_backward(do, q, k, v, o, lse, causal=True), (q, k, v)):
            assert x.shape == y.shape and bool((x == 0).all())


def test_refusals():
    from lsr import attention as A
    q, k, v, do = tensors(2, 5, 6, 4, 2, 8, torch.bfloat16)
    out, lse = A.attention_forward(q, k, v)
    m = torch.ones(2, 6, dtype=torch.bool, device="cuda")
    for bad in ((q.float(), k, v, None), (q.double(), k.double(), v.double(), None), (q, k, v[:, :5], None), (q[0], k, v, None),
                (q, k[:1], v[:1], None), (q[:, :, :3], k, v, None), (q, k, v, m[:, :5]), (q, k, v, m.long()), (q, k, v, m.cpu()),
                (q, k.cpu(), v.cpu(), None), (q[..., :4], k, v, None)):
        with pytest.raises(ValueError):
            A.attention_forward(*bad[:3], key_mask=bad[3])
        with pytest.raises(ValueError):
            A.attention(*bad[:3], key_mask=bad[3])
    big = torch.zeros(1, 2, 1, 136, device="cuda", dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        A.attention(big, big, big)
    for bad in ((do[:1], out, lse), (do, out.float(), lse), (do, out, lse.double()), (do, out, lse[:, :, :2])):
        with pytest.raises(ValueError):
            A.attention_backward(bad[0], q, k, v, *bad[1:])
    x = q.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(A.attention(x, k, v).float().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.float().sum().backward()


def test_fp32_captured_and_replayed_among_other_launches():
    """The launch that takes dq starts before that of dk and dv has ended: what follows in the stream waits for both."""
    from lsr import attention as A
    q, k, v, do = tensors(2, 300, 300, 16, 4, 128, torch.float32, seed=15)
    out, lse = A.attention_forward(q, k, v, causal=True)
    want = A.attention_backward(do, q, k, v, out, lse, causal=True)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        copies = []
        for _ in range(3):
            copies.append([t.clone() for t in A.attention_backward(do, q, k, v, out, lse, causal=True)])
    for _ in range(10):
        for c in copies:
            for t in c:
                t.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for c in copies for x, y in zip(c, want))
    for _ in range(20):
        got = A.attention_backward(do, q, k, v, out, lse, causal=True)
        assert all(torch.equal(x.clone(), y) for x, y in zip(got, want))
