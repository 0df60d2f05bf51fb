"""CPU: whether two strided tensors share memory, and whether one repeats a place, against counting every byte."""
from __future__ import annotations

import random

import pytest
import torch


def places(t):
    at = torch.zeros(t.shape, dtype=torch.long)
    for k, (st, n) in enumerate(zip(t.stride(), t.shape)):
        at += (torch.arange(n) * st).view([-1 if j == k else 1 for j in range(t.dim())])
    first = (t.data_ptr() + at * t.element_size()).reshape(-1).tolist()
    return [a + b for a in first for b in range(t.element_size())]


def view(rng, buf):
    while True:
        dims = rng.randint(0, 3)
        shape = [rng.randint(1, 6) for _ in range(dims)]
        stride = [rng.choice((0, 1, 1, 2, 3, 4, 5, 6, 7, 10, 12, 15, 30)) for _ in range(dims)]
        span = 1 + sum(s * (n - 1) for s, n in zip(stride, shape))
        b = buf if rng.random() < 0.7 else buf.view(torch.bfloat16)
        if span <= b.numel():
            return b.as_strided(shape, stride, rng.randint(0, b.numel() - span))


@pytest.mark.parametrize("seed", range(8))
def test_sharing_against_every_byte(seed):
    from lsr import grad as G
    rng, buf = random.Random(seed), torch.zeros(200)
    for _ in range(400):
        a, b = view(rng, buf), view(rng, buf)
        x, y = places(a), places(b)
        assert G._share(a, b) == (not set(x).isdisjoint(y)), (a.shape, a.stride(), b.shape, b.stride())
        assert G._repeats(a) == (len(set(x)) < len(x)), (a.shape, a.stride())


def test_large_views_are_settled_at_once():
    from lsr import grad as G
    w = torch.empty(4800, 1600, device="meta").new_empty((4800, 1600), device="cpu")
    apart = [w[:, :800], w[:, 800:]], [w[::2], w[1::2]], [w.view(-1)[::2], w.view(-1)[1::4]], [w[:2400].t(), w[2400:].t()]
    for a, b in apart:
        assert not G._share(a, b) and not G._share(b, a)
    for a, b in ([w[:, :801], w[:, 800:]], [w, w[4799:]], [w.t()[5:], w[:, :6]], [w.view(-1)[::3], w.view(-1)[1::7]]):
        assert G._share(a, b) and G._share(b, a)
    assert not G._repeats(w[:, 3:]) and not G._repeats(w.t()[::3]) and G._repeats(w.as_strided((4000, 1600), (1599, 1)))


def test_lists_with_strided_outputs():
    from lsr import grad as G
    b, c = torch.zeros(12, 10), torch.zeros(12, 10)

    def flat(grads, outs, norm=None):
        return G._flatten(grads, outs, norm)

    for grads in ([b[:, :5], b[:, 3:]], [b, b[:, 3:5]], [b[:, 2], b[4]], [b[:1].expand(3, 10)]):
        with pytest.raises(ValueError):
            flat(grads, grads)
        with pytest.raises(ValueError):
            flat([torch.zeros(t.shape) for t in grads], grads)
        flat(grads, [torch.zeros(t.shape) for t in grads])  # only read
    with pytest.raises(ValueError):
        flat([b[:, :5], c[:, :5]], [c[:, 3:8], b[:, 5:]])
    with pytest.raises(ValueError):
        flat([b[:, :5]], [b[:, :5]], b.view(-1)[24:25])
    src, dst, back = flat([b[:, :5], c, b[:, 5:]], [b[:, :5], c, b[:, 5:]], b.new_zeros(()))
    assert src[1] is c and dst[1] is c and [o.data_ptr() for o, _ in back] == [b.data_ptr(), b[:, 5:].data_ptr()]


@pytest.mark.parametrize("seed", range(6))
def test_lists_against_every_byte(seed):
    from lsr import grad as G
    rng, buf = random.Random(100 + seed), torch.zeros(4000)
    for _ in range(150):
        if rng.random() < 0.5:  # slices of rows, most of them side by side
            w, at, ts = buf[:rng.randint(2, 9) * 40].view(-1, 40), 0, []
            while at < 36:
                n = rng.randint(1, 9)
                a = at if rng.random() < 0.95 else max(0, at - 1)
                ts.append(w[rng.randint(0, 1):, a:min(40, at + n)])
                at += n
            rng.shuffle(ts)
        else:
            ts = [view(rng, buf[rng.randint(0, 3000):][:300]) for _ in range(rng.randint(1, 4))]
        seen, want = set(), False
        for t in ts:
            p = places(t)
            want |= len(set(p)) < len(p) or not seen.isdisjoint(p)
            seen |= set(p)
        norm = buf[rng.randint(0, 3999):][:1] if rng.random() < 0.3 else None
        want |= norm is not None and not seen.isdisjoint(places(norm))
        try:
            G._check_shared(ts, ts, norm, set())
            got = False
        except ValueError:
            got = True
        assert got == want, [(t.shape, t.stride(), t.storage_offset()) for t in ts]


def test_a_matrix_cut_into_many_columns_is_looked_over_quickly():
    import time
    from lsr import grad as G
    cut = list(torch.zeros(64, 64 * 256).split(64, 1))
    t = time.perf_counter()
    G._check_shared(cut, cut, None, set())
    assert time.perf_counter() - t < 0.1  # 4 ms; 320 where every pair is compared
