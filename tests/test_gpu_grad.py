"""Global gradient norm and clipping (lsr.grad) against float64.

Tolerances. The norm's sum is held in 64 bits (relative error far under 2^-24) and rounded once to
fp32: 2^-24 relative, doubled for the square root's own rounding. A clipped entry is g * coef with
coef off by its own three fp32 operations (4 * 2^-24 with the norm's) and the product's rounding
(2^-24), then rounded to the output type: u(type) = eps / 2, or half the spacing of its smallest values."""
from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle import grad as og

pytestmark = pytest.mark.gpu

U32 = 2.0 ** -24
TYPES = [torch.float32, torch.bfloat16, torch.float16]
INF = math.inf


def values(shapes, dtype, seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * scale).to(dtype) for s in shapes]


def f64(ts):
    return [t.double().cpu().numpy() for t in ts]


def check_scaled(got, want64, coef):
    u = torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(got.dtype).smallest_normal * u
    ref = np.asarray(want64, np.float64) * coef
    err = np.abs(got.double().cpu().numpy() - ref)
    assert (err <= np.abs(ref) * (u + 5 * U32) + tiny).all(), err.max()


LISTS = {
    "one entry": [(1,)],
    "odd sizes": [(3,), (65, 7), (1,), (0,), (129,), (5, 1, 13)],
    "over a chunk": [(40001,), (2, 32768), (32767,)],
    "many small": [(i % 37 + 1,) for i in range(1500)],  # more tensors than one launch takes
    "many chunks": [(3000, 2111), (5,), (1200, 901)],
}


@pytest.mark.parametrize("name", LISTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, INF])
def test_norm(name, dtype, p):
    from lsr import grad_norm
    ts = values(LISTS[name], dtype, seed=len(name))
    got = grad_norm(ts, p)
    assert got.dtype == torch.float32 and got.shape == () and got.is_cuda
    want = og.norm(f64(ts), p)
    assert abs(float(got) - want) <= 2 * U32 * want


def test_norm_of_mixed_types_and_misaligned_views():
    from lsr import grad_norm
    buf = {t: values([(70000,)], t, seed=3)[0] for t in TYPES}
    ts = [b[o:o + n] for b in buf.values() for o, n in ((1, 5), (7, 33000), (40003, 8), (50001, 17777))]
    want = og.norm(f64(ts), 2.0)
    assert abs(float(grad_norm(ts)) - want) <= 2 * U32 * want
    t = values([(33, 50)], torch.float32)[0]
    for view in (t.t(), t[:, 3:9], t[::2], t.t()[1::3]):  # permuted, gapped
        want = og.norm(f64([view]), 2.0)
        assert abs(float(grad_norm([view])) - want) <= 2 * U32 * want


def test_norm_of_nothing_and_of_extreme_values():
    from lsr import grad_norm
    assert float(grad_norm([])) == 0.0
    assert float(grad_norm([torch.empty(0, device="cuda")])) == 0.0
    for x in (1e30, 1e-30):  # squares of neither are fp32 numbers
        t = torch.full((1000,), x, device="cuda")
        want = og.norm(f64([t]), 2.0)
        assert abs(float(grad_norm([t])) - want) <= 2 * U32 * want
    for p in (1.0, 2.0, INF):
        t = torch.ones(5000, device="cuda")
        t[4321] = -INF
        assert float(grad_norm([t], p)) == INF
        t[77] = math.nan
        assert math.isnan(float(grad_norm([t, torch.ones(3, device="cuda")], p)))


def test_norm_is_the_same_bits_every_time():
    from lsr import grad_norm
    ts = values([(3001, 701), (17,), (999, 64)], torch.bfloat16)
    first = grad_norm(ts).clone()
    assert all(torch.equal(grad_norm(ts), first) for _ in range(10))


@pytest.mark.parametrize("src", TYPES)
@pytest.mark.parametrize("dst", TYPES)
@pytest.mark.parametrize("p", [1.0, 2.0, INF])
def test_clip_into_another_type(src, dst, p):
    from lsr import clip_grads
    ts = values(LISTS["odd sizes"] + LISTS["over a chunk"], src, seed=5)
    before = f64(ts)
    want = og.norm(before, p)
    for bound in (want / 3, want * 2):
        out = [torch.full(t.shape, math.nan, dtype=dst, device="cuda") for t in ts]
        got = clip_grads(ts, bound, p, out=out)
        assert abs(float(got) - want) <= 2 * U32 * want
        for o, b, t in zip(out, before, ts):
            check_scaled(o, b, og.coefficient(want, bound))
            assert np.array_equal(t.double().cpu().numpy(), b)  # read only


@pytest.mark.parametrize("dtype", TYPES)
def test_clip_in_place_leaves_what_lies_beside(dtype):
    from lsr import clip_grads
    buf = values([(100000,)], dtype, seed=7)[0]
    keep = buf.clone()
    spans = [(1, 6), (9, 33333), (40001, 40002), (40003, 99998)]
    ts = [buf[a:b] for a, b in spans]
    before = f64(ts)
    want = og.norm(before, 2.0)
    assert abs(float(clip_grads(ts, want / 7)) - want) <= 2 * U32 * want
    inside = torch.zeros(100000, dtype=torch.bool, device="cuda")
    for (a, b), x in zip(spans, before):
        check_scaled(buf[a:b], x, og.coefficient(want, want / 7))
        inside[a:b] = True
    assert torch.equal(buf[~inside], keep[~inside])
    at = buf.clone()
    clip_grads(ts, 1e6)  # within the bound: nothing changes
    assert torch.equal(buf, at)


def test_clip_of_views_and_given_norm():
    from lsr import clip_grads, grad_norm
    t = values([(33, 50)], torch.float32, seed=9)[0]
    for view in (t.t(), t[:, 3:9]):
        b = view.double().cpu().numpy()
        n = og.norm([b], 2.0)
        clip_grads([view], n / 3)
        check_scaled(view, b, og.coefficient(n, n / 3))
    a, c = values([(1000,), (77,)], torch.bfloat16, seed=11)
    before = f64([a, c])
    whole = grad_norm([a, c])
    assert clip_grads([a], 2.0, total_norm=whole) is whole
    clip_grads([c], 2.0, total_norm=whole)
    for x, b in zip((a, c), before):
        check_scaled(x, b, og.coefficient(og.norm(before, 2.0), 2.0))


def test_clip_by_norms_that_are_not_finite():
    from lsr import clip_grads, clip_grad_norm_
    t = torch.ones(1000, device="cuda")
    t[5] = INF
    out = [torch.empty_like(t)]
    assert float(clip_grads([t], 1.0, out=out)) == INF
    assert math.isnan(float(out[0][5])) and float(out[0].nan_to_num(0).abs().max()) == 0.0
    t[6] = math.nan
    clip_grads([t], 1.0, out=out)
    assert bool(out[0].isnan().all())
    p = torch.nn.Parameter(torch.zeros(1000, device="cuda"))
    p.grad = t.clone()
    with pytest.raises(RuntimeError):
        clip_grad_norm_([p], 1.0, error_if_nonfinite=True)
    assert torch.equal(p.grad.nan_to_num(7), t.nan_to_num(7))


def test_clip_grad_norm_of_a_model_as_torch_does():
    from lsr import MuonAdamW, clip_grad_norm_
    torch.manual_seed(0)
    model = torch.nn.Sequential(torch.nn.Linear(70, 33), torch.nn.Tanh(), torch.nn.Linear(33, 5)).cuda()
    model(torch.randn(64, 70, device="cuda")).square().sum().backward()
    ps = list(model.parameters())
    before = f64([p.grad for p in ps])
    n = og.norm(before, 2.0)
    got = clip_grad_norm_(iter(ps + [ps[0], torch.nn.Parameter(torch.zeros(3, device="cuda"))]), 0.5)
    assert abs(float(got) - n) <= 2 * U32 * n
    for p, b in zip(ps, before):
        check_scaled(p.grad, b, og.coefficient(n, 0.5))
    opt = MuonAdamW(list(model.bfloat16().named_parameters()), "batched", 1e-3, 0.95, 0.01, True, 5, 1e-7, "original", 8,
                    1e-4, (0.9, 0.95), 0.01, 0)
    for p in model.parameters():
        p.grad = torch.randn_like(p)
    before = f64([p.grad for p in model.parameters()])
    n = og.norm(before, 2.0)
    assert abs(float(opt.clip_grad_norm(0.25)) - n) <= 2 * U32 * n
    for p, b in zip(model.parameters(), before):
        check_scaled(p.grad, b, og.coefficient(n, 0.25))
    opt.muon_step()
    opt.adam_step()


def test_captured_and_on_two_streams():
    from lsr import clip_grads
    sets = [values([(1000, 333), (7,)], torch.float32, seed=s) for s in (1, 2)]
    outs = [[torch.empty_like(t) for t in ts] for ts in sets]
    clip_grads(sets[0], 1.0, out=outs[0])
    torch.cuda.synchronize()
    graphs, norms = [], []
    for ts, out in zip(sets, outs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            norms.append(clip_grads(ts, 1.0, out=out))
        graphs.append(g)
    streams = [torch.cuda.Stream() for _ in graphs]
    for round_ in range(3):
        for ts in sets:
            for t in ts:
                t.mul_(1.5)
        torch.cuda.synchronize()
        for _ in range(20):
            for g, s in zip(graphs, streams):
                with torch.cuda.stream(s):
                    g.replay()
        torch.cuda.synchronize()
        for ts, out, norm in zip(sets, outs, norms):
            want = og.norm(f64(ts), 2.0)
            assert abs(float(norm) - want) <= 2 * U32 * want
            for o, t in zip(out, ts):
                check_scaled(o, t.double().cpu().numpy(), og.coefficient(want, 1.0))


def test_refusals():
    from lsr import clip_grads, grad_norm
    a, b = torch.ones(10, device="cuda"), torch.ones(10, device="cuda")
    for bad in (lambda: grad_norm([a], 3.0), lambda: grad_norm([a.double()]), lambda: grad_norm([a, torch.ones(2)]),
                lambda: grad_norm([1.0]), lambda: clip_grads([a], -1.0), lambda: clip_grads([a], math.nan),
                lambda: clip_grads([a, a], 1.0), lambda: clip_grads([a[:6], a[5:]], 1.0),
                lambda: clip_grads([a[:5], a[5:]], 1.0, out=[a[5:], b[:5]]),
                lambda: clip_grads([a], 1.0, out=[b[:9]]), lambda: clip_grads([a], 1.0, out=[b, b]),
                lambda: clip_grads([a[:4]], 1.0, out=[a[2:6]]),
                lambda: clip_grads([torch.ones(1, device="cuda").expand(4)], 1.0),
                lambda: clip_grads([a], 1.0, total_norm=torch.ones(1)),
                lambda: grad_norm([torch.ones(3, device="cuda").to_sparse()])):
        with pytest.raises(ValueError):
            bad()
    assert torch.equal(a, torch.ones(10, device="cuda"))
