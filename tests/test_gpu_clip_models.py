"""Norm and clipping of lists as long as a model's: several launches, several tables, every alignment.

Tolerances as derived for the short lists: the norm within 2 * 2^-24, an entry within its type's
half step (eps / 2, or half the spacing of its smallest values) and 5 * 2^-24 for the coefficient
and the product."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
LISTS = {
    "few large": [(3000, 2111), (5,), (0,), (1200, 901), (7, 4099)],  # 233 chunks of 32768
    "96": [(i % 37 + 1,) for i in range(95)] + [(70, 32768)],
    "97": [(i % 37 + 1,) for i in range(97)],
    "1024": [(i % 37 + 1,) for i in range(1024)],
    "1025": [(i % 37 + 1,) for i in range(1025)],
    "empty ones among": [(0,) if i % 3 else (i % 91 + 1,) for i in range(3000)],
    "96 and empty ones": [(i % 37 + 1,) for i in range(96)] + [(0,)] * 50,
    "50 among empty ones": [(0,) if i % 4 else (3000 * (i % 7) + 1,) for i in range(200)],
    "three tables": [(i % 37 + 1,) for i in range(2500)] + [(300, 1001)],
}


def make(shapes, dtype, seed):
    """Views of one buffer, side by side, so that most begin off 16-byte boundaries; and the buffer."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    sizes = [math.prod(s) for s in shapes]
    buf = torch.randn(sum(sizes), device="cuda", generator=g).to(dtype)
    return [t.view(s) for t, s in zip(buf.split(sizes), shapes)], buf


def norm_of(buf, p):
    x = buf.double().abs()
    return float(x.max() if p == math.inf else x.sum() if p == 1.0 else x.square().sum().sqrt())


def check_scaled(got, before, norm, bound):
    coef = min(1.0, bound / (norm + 1e-6))
    want = before.double() * coef
    u, tiny = torch.finfo(got.dtype).eps / 2, torch.finfo(got.dtype).smallest_normal * torch.finfo(got.dtype).eps / 2
    assert bool(((got.double() - want).abs() <= want.abs() * (u + 5 * E) + tiny).all())


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
def test_clip_in_place(name, dtype, p):
    from lsr import clip_grads, grad_norm
    ts, buf = make(LISTS[name], dtype, len(name))
    before, want = buf.clone(), norm_of(buf, p)
    got = clip_grads(ts, want * 2, p)  # within the bound: as it was
    assert abs(float(got) - want) <= 2 * E * want and torch.equal(buf, before)
    assert torch.equal(grad_norm(ts, p), got)
    got = clip_grads(ts, want / 3, p)
    assert abs(float(got) - want) <= 2 * E * want
    check_scaled(buf, before, want, want / 3)


@pytest.mark.parametrize("name", ["few large", "three tables"])
@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("shift", [0, 1, 3])
def test_clip_into_another_type_at_other_alignments(name, src, dst, shift):
    """shift: entries by which the outputs' places lie off the gradients'; where the two have no common
    16-byte boundary an entry is taken at a time."""
    from lsr import clip_grads
    ts, buf = make(LISTS[name], src, 3)
    before, want = buf.clone(), norm_of(buf, 2.0)
    room = torch.full((buf.numel() + 8,), math.nan, dtype=dst, device="cuda")
    whole = room[shift:shift + buf.numel()]
    outs = [o.view(t.shape) for o, t in zip(whole.split([t.numel() for t in ts]), ts)]
    for bound in (want / 3, want * 2):
        got = clip_grads(ts, bound, out=outs)
        assert abs(float(got) - want) <= 2 * E * want
        check_scaled(whole, before, want, bound)
        assert torch.equal(buf, before)
    assert bool(room[:shift].isnan().all()) and bool(room[shift + buf.numel():].isnan().all())


@pytest.mark.parametrize("name", ["few large", "three tables", "empty ones among"])
def test_a_norm_given_for_lists_of_several_launches(name):
    from lsr import clip_grads, grad_norm
    ts, buf = make(LISTS[name], torch.bfloat16, 5)
    before, want = buf.clone(), norm_of(buf, 2.0)
    whole = grad_norm(ts)
    kept = whole.clone()
    assert clip_grads(ts, want / 5, total_norm=whole) is whole and torch.equal(whole, kept)
    check_scaled(buf, before, want, want / 5)


def test_captured_in_place_over_several_tables():
    from lsr import clip_grads
    ts, buf = make(LISTS["three tables"], torch.float32, 7)
    clip_grads(ts, 1e30)
    before, want = buf.clone(), norm_of(buf, 2.0)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        norm = clip_grads(ts, want / 4)
    graph.replay()
    assert abs(float(norm) - want) <= 2 * E * want
    check_scaled(buf, before, want, want / 4)
    graph.replay()  # now within the bound, or over it by the rounding of the clipped entries alone
    assert abs(float(norm) - want / 4) <= 1e-5 * want


def test_a_tensor_of_more_than_2_31_entries():
    from lsr import clip_grads
    n = 2 ** 31 + 70001
    t = torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    at = torch.tensor([0, 1, 2 ** 31 - 1, 2 ** 31, n - 1], device="cuda")
    t[at] = torch.tensor([1.0, -2.0, 3.0, 4.0, -5.0], dtype=torch.bfloat16, device="cuda")
    want = 55.0 ** 0.5
    assert abs(float(clip_grads([t], want / 2)) - want) <= 2 * E * want
    check_scaled(t[at], torch.tensor([1.0, -2.0, 3.0, 4.0, -5.0], device="cuda"), want, want / 2)
    assert int(t.count_nonzero()) == 5
