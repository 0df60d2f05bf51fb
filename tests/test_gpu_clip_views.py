"""Clipping of views with gaps: outputs that share memory are refused, those that only interleave are not."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def base(rows=12, cols=10):
    return torch.arange(rows * cols, dtype=torch.float32, device="cuda").view(rows, cols) / 8


SHARING = {
    "columns": lambda b: [b[:, :5], b[:, 3:]],
    "columns and the whole": lambda b: [b, b[:, 3:5]],
    "rows and columns": lambda b: [b[2], b[:, 9]],
    "one element": lambda b: [b[:7, :4], b[6:, 3:]],
    "other strides": lambda b: [b.view(-1)[::3], b.view(-1)[1::7]],
    "in itself": lambda b: [b.as_strided((5, 4), (2, 1))],
    "expanded": lambda b: [b[:1].expand(4, 10)],
    "twice": lambda b: [b[:, :5], b[:, :5]],
    "other type": lambda b: [b[:, 4:6], b.view(torch.bfloat16)[:, 9:10]],
}
APART = {
    "columns": lambda b: [b[:, :5], b[:, 5:]],
    "rows": lambda b: [b[::2], b[1::2]],
    "transposed": lambda b: [b.t()[:5], b.t()[5:]],
    "every second row and column": lambda b: [b[::2, ::2], b[::2, 1::2], b[1::2, ::2], b[1::2, 1::2]],
    "a row and the rest": lambda b: [b[0], b[1:, 2:], b[1:, :2]],
    "other strides": lambda b: [b.view(-1)[::3], b.view(-1)[1::6]],
    "in itself apart": lambda b: [b.as_strided((2, 2), (3, 2))],
}


@pytest.mark.parametrize("name", SHARING)
def test_shared_memory_is_refused(name):
    from lsr import clip_grads
    b = base()
    keep = b.clone()
    views = SHARING[name](b)
    with pytest.raises(ValueError):
        clip_grads(views, 1.0)
    assert torch.equal(b, keep)
    with pytest.raises(ValueError):
        clip_grads([torch.ones(v.shape, device="cuda") for v in views], 1.0, out=views)
    assert torch.equal(b, keep)


@pytest.mark.parametrize("name", APART)
def test_what_only_interleaves_is_clipped(name):
    """Each entry: g times the coefficient, three fp32 roundings and the product's."""
    from lsr import clip_grads
    b = base()
    views = APART[name](b)
    before = [v.double() for v in views]
    norm = math.sqrt(sum(float(v.square().sum()) for v in before))
    got = clip_grads(views, norm / 4)
    assert abs(float(got) - norm) <= 2.0 ** -23 * norm
    for v, x in zip(views, before):
        want = x * (norm / 4 / (norm + 1e-6))
        assert bool(((v.double() - want).abs() <= want.abs() * 6 * 2.0 ** -24).all())


def test_an_output_over_a_gradient_or_the_given_norm_is_refused():
    from lsr import clip_grads
    b, c = base(), base()
    keep = b.clone()
    for grads, outs in (([b[:, :5], c[:, :5]], [c[:, 3:8], b[:, 5:]]), ([b[:, :5]], [b[:, 1:6]]), ([b[0], c], [b[:, 4], c])):
        outs = [o if o.shape == g.shape else o[:g.numel()] for g, o in zip(grads, outs)]
        grads = [g if o.shape == g.shape else g[:o.numel()] for g, o in zip(grads, outs)]
        with pytest.raises(ValueError):
            clip_grads(grads, 1.0, out=outs)
    assert torch.equal(b, keep)
    norm = b.view(-1)[17]
    with pytest.raises(ValueError):
        clip_grads([b[:, 5:9]], 1.0, total_norm=norm)
    assert clip_grads([b[:, :5]], 1e6, total_norm=norm) is norm


def test_overlapping_gradients_are_only_read():
    from lsr import clip_grads, grad_norm
    b = base()
    views = [b[:, :5], b[:, 3:]]
    want = math.sqrt(sum(float(v.double().square().sum()) for v in views))
    outs = [torch.empty_like(v, memory_format=torch.contiguous_format) for v in views]
    assert abs(float(grad_norm(views)) - want) <= 2.0 ** -23 * want
    assert abs(float(clip_grads(views, 2 * want, out=outs)) - want) <= 2.0 ** -23 * want
    assert all(torch.equal(o, v) for o, v in zip(outs, views))
