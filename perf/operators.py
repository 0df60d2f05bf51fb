"""The language-model training operators of lsr.grad and lsr.attention, as cases to time and compare.

    op "norm"   one norm over every gradient of a model                    lsr.grad_norm
    op "clip"   the same, and the gradients scaled and cast for the        lsr.clip_grads
                optimizer that takes them
    op "fwd"    softmax attention and its log-sum-exp                      lsr.attention.attention_forward
    op "bwd"    its gradients, probabilities recomputed from the           lsr.attention.attention_backward
                log-sum-exp
    op "train"  forward and backward through autograd                      lsr.attention.attention

Gradient cases are the parameter list of a GPT-2 shaped model: `e` columns, `layers` blocks, `vocab` rows of the
embedding. `flat` puts the gradients side by side in one buffer, as the bucket views of data-parallel training do.
Attention cases are [batch, length, heads, dim] with `kv` key heads; `packed` takes queries, keys and values as views of
one projection's output; `pad` shortens each batch entry's keys with a key mask, and `empty` leaves the last one none.
"""
import math
import sys
from pathlib import Path

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2}
ORDER = {"one": 1.0, "two": 2.0, "max": math.inf}  # of the norm


def _lsr():
    root = str(Path(__file__).resolve().parent.parent / "cuda-lsr_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    import lsr
    import lsr.attention
    return lsr


# ---------------------------------------------------------------------------
# Cases
# ---------------------------------------------------------------------------

def _grads(op, name, e, layers, vocab, dtype, to, p, flat, clipped):
    return {"name": name, "op": op, "e": e, "layers": layers, "vocab": vocab, "dtype": dtype, "to": to, "p": p, "flat": flat, "clipped": clipped}


def _attn(op, name, batch, q, k, heads, kv, dim, dtype, causal, packed=False, pad=False, empty=False):
    return {"name": name, "op": op, "batch": batch, "q": q, "k": k, "heads": heads, "kv": kv, "dim": dim, "dtype": dtype,
            "causal": causal, "packed": packed, "pad": pad, "empty": empty}


def listed():
    return [
        # the gradients of a two-layer test model in bucket views of odd sizes: a few launches, where latency counts
        _grads("norm", "norm small odd fp32", 65, 2, 211, "fp32", "fp32", "two", True, True),
        # every gradient of GPT-2-XL after its backward pass: one read of 3.1 GB
        _grads("norm", "norm gpt2-xl bf16", 1600, 48, 50257, "bf16", "bf16", "two", False, True),
        # a small fp16 model clipped by its largest entry, in views that start at odd places
        _grads("clip", "clip small odd fp16 max", 131, 4, 1031, "fp16", "fp16", "max", True, True),
        # GPT-2-large with gradients accumulated in fp32 and cast to the bf16 that the Muon step takes
        _grads("clip", "clip gpt2-large fp32 to bf16", 1280, 36, 50257, "fp32", "bf16", "two", True, True),
        # GPT-2-XL in bf16 at a norm under the bound: the common step, where nothing is to be clipped
        _grads("clip", "clip gpt2-xl bf16 within", 1600, 48, 50257, "bf16", "bf16", "two", True, False),
        # one micro-batch of the language-model driver at its default length
        _attn("fwd", "fwd gpt2-xl 512", 1, 512, 512, 25, 25, 64, "bf16", True, packed=True),
        # a few last tokens scored against long contexts of a padded batch
        _attn("fwd", "fwd 3 late rows padded fp16", 4, 3, 4097, 12, 4, 80, "fp16", True, pad=True),
        # a long document with shared key heads
        _attn("fwd", "fwd long 16384 kv 2", 1, 16384, 16384, 8, 2, 128, "bf16", True),
        # the backward pass of one micro-batch at the model's full 1024 positions
        _attn("bwd", "bwd gpt2-xl 1024", 1, 1024, 1024, 25, 25, 64, "bf16", True, packed=True),
        # keys of another length than the queries, padded, one entry of the batch a dummy without any key
        _attn("bwd", "bwd cross padded fp16", 3, 333, 1027, 6, 2, 80, "fp16", False, pad=True, empty=True),
        # a long document's backward pass with shared key heads
        _attn("bwd", "bwd long 8192 kv 4", 1, 8192, 8192, 16, 4, 128, "bf16", True),
        # the driver's small test model in fp32, forward and backward: a numerics check before a run
        _attn("train", "train small fp32", 2, 257, 257, 4, 4, 64, "fp32", True),
    ]


def _spread(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "clip", "fwd", "fwd", "bwd", "bwd", "train"))
    if op in ("norm", "clip"):
        dtype = rng.choice(("bf16", "bf16", "fp32", "fp16"))
        c = _grads(op, "", _spread(rng, 33, 1600), _spread(rng, 1, 48), _spread(rng, 100, 50257), dtype, rng.choice((dtype, "bf16")) if op == "clip" else dtype,
                   rng.choice(("two", "two", "two", "one", "max")), rng.random() < 0.5, rng.random() < 0.7)
    else:
        dtype = rng.choice(("bf16", "bf16", "bf16", "fp16", "fp16", "fp32"))
        kv = rng.choice((1, 2, 3, 4, 8))
        heads = kv * rng.choice((1, 1, 2, 4))
        # with one key alone the score has no gradient, and what is left of it is the rounding of 0
        least, longest = 1 if op == "fwd" else 8, 1500 if dtype == "fp32" else 8192
        same = rng.random() < 0.6
        k = _spread(rng, least, longest)
        q = k if same else _spread(rng, 1, longest)
        dim = rng.choice((64, 64, 128, 128, 32, 40, 80, 96))
        batch, causal = _spread(rng, 1, 8), rng.random() < 0.6
        most = {"fwd": 8 * 16384 ** 2, "bwd": 16 * 8192 ** 2, "train": 11 * 8192 ** 2}[op] * 128 // (1 if causal else 2)
        while batch * heads * q * k * dim > most:  # no more than the largest listed one
            batch, q, k = (batch - 1, q, k) if batch > 1 else (1, (q + 1) // 2, max(least, (k + 1) // 2))
        c = _attn(op, "", batch, q, k, heads, kv, dim, dtype, causal, packed=op != "train" and q == k and heads == kv and rng.random() < 0.5, pad=rng.random() < 0.3,
                  empty=batch > 1 and rng.random() < 0.15)
    del c["name"]
    return c


def _shapes(c):
    e, v = c["e"], c["vocab"]
    block = [(e,), (e,), (e, 3 * e), (3 * e,), (e, e), (e,), (e,), (e,), (e, 4 * e), (4 * e,), (4 * e, e), (e,)]
    return [(v, e), (1024, e)] + block * c["layers"] + [(e,), (e,)]


def _lengths(c):
    """Keys that each batch entry has."""
    b, k = c["batch"], c["k"]
    n = [max(1, k - i * k // (2 * b)) if c["pad"] else k for i in range(b)]
    if c["empty"]:
        n[-1] = 0
    return n


def _pairs(c):
    """Query-key pairs that are not masked, for one head."""
    q, k, total = c["q"], c["k"], 0
    for n in _lengths(c):
        if not c["causal"]:
            total += q * n
            continue
        # row i sees min(n, i + 1 + k - q) keys, none where that is negative
        first, last = max(0, q - k), min(q, max(0, n - 1 - k + q))
        total += (last - first) * (first + 1 + k - q + last + k - q) // 2 if last > first else 0
        total += (q - max(first, last)) * n
    return total


def work(c):
    if c["op"] in ("norm", "clip"):
        n = sum(math.prod(s) for s in _shapes(c))
        return {"bytes": n * SIZE[c["dtype"]] + 4 + (n * SIZE[c["to"]] if c["op"] == "clip" else 0), "flops": (2 if c["op"] == "norm" else 3) * n}
    qo, kv, rows = c["batch"] * c["q"] * c["heads"] * c["dim"], sum(_lengths(c)) * c["kv"] * c["dim"], c["batch"] * c["q"] * c["heads"]
    size, mask = SIZE[c["dtype"]], c["batch"] * c["k"] if c["pad"] or c["empty"] else 0
    out = 2 * c["batch"] * c["k"] * c["kv"] * c["dim"]
    products = {"fwd": 2, "bwd": 5, "train": 7}[c["op"]]
    moved = {"fwd": (2 * qo + 2 * kv) * size + 4 * rows, "bwd": (4 * qo + 2 * kv + out) * size + 4 * rows, "train": (4 * qo + 2 * kv + out) * size}[c["op"]]
    return {"bytes": moved + mask, "flops": products * 2 * _pairs(c) * c["heads"] * c["dim"]}


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _prepare_grads(c, gen):
    shapes, dt = _shapes(c), DTYPES[c["dtype"]]
    sizes = [math.prod(s) for s in shapes]
    total = sum(sizes)
    # layers differ by up to a hundred in scale; the norm is about 4 where it is to be clipped at 1, else about a third
    target = 4.0 if c["clipped"] else 0.33
    scale = (10.0 ** (-2.0 * torch.rand(len(sizes), generator=gen, device="cuda"))).double()
    n = torch.tensor(sizes, dtype=torch.float64, device="cuda")
    whole = {"one": (scale * n).sum() * 0.8, "two": (scale.square() * n).sum().sqrt(), "max": 5.0 * scale.max()}[c["p"]]
    # a bound on the sum of absolute values is one that grows with the model
    bound = 1e-3 * total if c["p"] == "one" else 1.0
    scale = (scale * (target * bound / whole)).float()
    if c["flat"]:
        buf = torch.empty(total, dtype=dt, device="cuda")
        grads = [t.view(s) for t, s in zip(buf.split(sizes), shapes)]
    else:
        buf = None
        grads = [torch.empty(s, dtype=dt, device="cuda") for s in shapes]
    for i, g in enumerate(grads):
        g.copy_(torch.randn(g.shape, generator=gen, device="cuda") * scale[i])
    st = {"case": c, "grads": grads, "buf": buf, "max_norm": bound}
    if c["op"] == "clip":
        st["whole"] = torch.empty(total, dtype=DTYPES[c["to"]], device="cuda")
        st["out"] = [t.view(s) for t, s in zip(st["whole"].split(sizes), shapes)]
    return st


def _prepare_attention(c, gen):
    b, q, k, h, kv, d, dt = c["batch"], c["q"], c["k"], c["heads"], c["kv"], c["dim"], DTYPES[c["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda")

    if c["packed"]:
        Q, K, V = normal(b, q, 3 * h * d).to(dt).view(b, q, 3, h, d).unbind(2)
    else:
        Q, K, V = normal(b, q, h, d).to(dt), normal(b, k, kv, d).to(dt), normal(b, k, kv, d).to(dt)
    mask = None
    if c["pad"] or c["empty"]:
        mask = torch.arange(k, device="cuda")[None, :] < torch.tensor(_lengths(c), device="cuda")[:, None]
    st = {"case": c, "q": Q, "k": K, "v": V, "mask": mask, "scale": d ** -0.5}
    if c["op"] in ("bwd", "train"):
        st["dout"] = normal(b, q, h, d).to(dt)
    if c["op"] == "bwd":  # what the forward pass of the same step left
        out, st["lse"] = _plain_forward(Q, K, V, mask, c["causal"], st["scale"])
        st["out"] = out.to(dt)
    if c["op"] == "train":
        st["leaves"] = [t.detach().clone().requires_grad_(True) for t in (Q, K, V)]
    return st


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return _prepare_grads(case, gen) if case["op"] in ("norm", "clip") else _prepare_attention(case, gen)


# ---------------------------------------------------------------------------
# Plain forms, in 32 bits
# ---------------------------------------------------------------------------

def _plain_norm(grads, p):
    if p == "max":
        return torch.stack([g.float().abs().amax() for g in grads]).amax()
    if p == "one":
        return torch.stack([g.float().abs().sum() for g in grads]).sum()
    return torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()


def _plain_clip(st):
    c = st["case"]
    norm = _plain_norm(st["grads"], c["p"])
    coef = (st["max_norm"] / (norm + 1e-6)).clamp(max=1.0)
    return {"norm": norm, "grads": torch.cat([(g.float() * coef).to(DTYPES[c["to"]]).reshape(-1) for g in st["grads"]])}


def _allowed(b, q, k, mask, causal, device):
    """[b or 1, 1, 1, q, k] truth values, None where every key is seen."""
    allow = None
    if causal:
        allow = (torch.arange(k, device=device)[None, :] <= torch.arange(q, device=device)[:, None] + (k - q))[None, None, None]
    if mask is not None:
        m = mask[:, None, None, None, :]
        allow = m if allow is None else allow & m
    return allow


def _by_head(t, kv):
    """[batch, length, heads, dim] as [batch, kv, heads / kv, length, dim] in 32 bits."""
    b, n, h, d = t.shape
    return t.float().permute(0, 2, 1, 3).reshape(b, kv, h // kv, n, d)


def _back(t, dtype):
    b, kv, g, n, d = t.shape
    return t.reshape(b, kv * g, n, d).permute(0, 2, 1, 3).to(dtype)


def _scores(qf, kf, mask, causal, scale):
    s = (qf @ kf.transpose(-1, -2)) * scale
    allow = _allowed(qf.shape[0], qf.shape[3], kf.shape[3], mask, causal, qf.device)
    return s if allow is None else s.masked_fill(~allow, -math.inf)


def _plain_forward(q, k, v, mask, causal, scale):
    kv = k.shape[2]
    s = _scores(_by_head(q, kv), _by_head(k, kv), mask, causal, scale)
    top = s.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)
    p = (s - top).exp()
    total = p.sum(-1, keepdim=True)
    out = torch.where(total > 0, (p @ _by_head(v, kv)) / total.clamp(min=1e-30), torch.zeros_like(total))
    lse = (total.log() + top).squeeze(-1)  # minus infinity where a row sees no key
    return _back(out, torch.float32), lse.reshape(q.shape[0], q.shape[2], q.shape[1])


def _plain_backward(dout, q, k, v, out, lse, mask, causal, scale):
    b, n, h, d = q.shape
    kv = k.shape[2]
    qf, kf, vf, of, df = (_by_head(t, kv) for t in (q, k, v, out, dout))
    row = lse.reshape(b, kv, h // kv, n, 1)
    row = torch.where(row == -math.inf, torch.full_like(row, math.inf), row)  # a row without keys: every probability 0
    p = (_scores(qf, kf, mask, causal, scale) - row).exp()
    dv = (p.transpose(-1, -2) @ df).sum(2, keepdim=True)
    ds = p * (df @ vf.transpose(-1, -2) - (df * of).sum(-1, keepdim=True)) * scale
    return ds @ kf, (ds.transpose(-1, -2) @ qf).sum(2, keepdim=True), dv


def _plain_attention(st):
    c = st["case"]
    dt, common = DTYPES[c["dtype"]], (st["mask"], c["causal"], st["scale"])
    if c["op"] == "bwd":
        out, lse = st["out"], st["lse"]
    else:
        out, lse = _plain_forward(st["q"], st["k"], st["v"], *common)
    if c["op"] == "fwd":
        return {"out": out.to(dt), "lse": lse}
    dq, dk, dv = _plain_backward(st["dout"], st["q"], st["k"], st["v"], out, lse, *common)
    grads = {"dq": _back(dq, dt), "dk": _back(dk, dt), "dv": _back(dv, dt)}
    return grads if c["op"] == "bwd" else {"out": out.to(dt), **grads}


# ---------------------------------------------------------------------------
# One pass
# ---------------------------------------------------------------------------

def _own_run(st):
    lsr = _lsr()
    c = st["case"]
    if c["op"] == "norm":
        return {"norm": lsr.grad_norm(st["grads"], norm_type=ORDER[c["p"]])}
    if c["op"] == "clip":
        return {"norm": lsr.clip_grads(st["grads"], st["max_norm"], norm_type=ORDER[c["p"]], out=st["out"]), "grads": st["whole"]}
    A, how = lsr.attention, {"causal": c["causal"], "scale": st["scale"], "key_mask": st["mask"]}
    if c["op"] == "fwd":
        out, lse = A.attention_forward(st["q"], st["k"], st["v"], **how)
        return {"out": out, "lse": lse}
    if c["op"] == "bwd":
        return dict(zip(("dq", "dk", "dv"), A.attention_backward(st["dout"], st["q"], st["k"], st["v"], st["out"], st["lse"], **how)))
    out = A.attention(*st["leaves"], **how)
    dq, dk, dv = torch.autograd.grad(out, st["leaves"], st["dout"])
    return {"out": out.detach(), "dq": dq, "dk": dk, "dv": dv}


def run(state):
    if own:
        return _own_run(state)
    if state["case"]["op"] == "norm":
        return {"norm": _plain_norm(state["grads"], state["case"]["p"])}
    return _plain_clip(state) if state["case"]["op"] == "clip" else _plain_attention(state)


# ---------------------------------------------------------------------------
# From the definitions, in 64 bits
# ---------------------------------------------------------------------------

def _exact_grads(c, st):
    total = torch.zeros((), dtype=torch.float64, device="cuda")
    for g in st["grads"]:
        a = g.double().abs()
        total = torch.maximum(total, a.max()) if c["p"] == "max" else total + (a if c["p"] == "one" else a * a).sum()
    norm = total.sqrt() if c["p"] == "two" else total
    if c["op"] == "norm":
        return {"norm": norm}
    coef = min(1.0, st["max_norm"] / (float(norm) + 1e-6))
    whole = torch.empty(sum(g.numel() for g in st["grads"]), dtype=torch.float64, device="cuda")
    at = 0
    for g in st["grads"]:
        whole[at:at + g.numel()] = g.reshape(-1).double() * coef
        at += g.numel()
    return {"norm": norm, "grads": whole}


def _exact_attention(c, st):
    b, q, k, h, kv, d = (c[n] for n in ("batch", "q", "k", "heads", "kv", "dim"))
    if 14 * b * h * q * k * d > 2e13:
        return None
    shape = {"device": "cuda", "dtype": torch.float64}
    out, lse = torch.zeros(b, q, h, d, **shape), torch.full((b, h, q), -math.inf, **shape)
    dq, dk, dv = torch.zeros(b, q, h, d, **shape), torch.zeros(b, k, kv, d, **shape), torch.zeros(b, k, kv, d, **shape)
    rows = max(1, min(q, 2 ** 28 // max(1, k)))
    for i, n in enumerate(_lengths(c)):
        if n == 0:
            continue
        for j in range(h):
            K, V = st["k"][i, :n, j // (h // kv)].double(), st["v"][i, :n, j // (h // kv)].double()
            for at in range(0, q, rows):
                Q = st["q"][i, at:at + rows, j].double()
                sees = torch.full((Q.shape[0],), n, device="cuda")
                if c["causal"]:
                    sees = torch.clamp(torch.arange(at, at + Q.shape[0], device="cuda") + 1 + k - q, min=0, max=n)
                hidden = torch.arange(n, device="cuda")[None, :] >= sees[:, None]
                x = (Q @ K.T).mul_(st["scale"]).masked_fill_(hidden, -math.inf)
                z = st["lse"][i, j, at:at + rows].double() if c["op"] == "bwd" else torch.logsumexp(x, 1)
                lse[i, j, at:at + rows] = z
                p = torch.exp_(x.sub_(torch.where(sees > 0, z, torch.zeros_like(z))[:, None]))
                o = st["out"][i, at:at + rows, j].double() if c["op"] == "bwd" else p @ V  # the backward pass is given the forward's
                out[i, at:at + rows, j] = o
                if c["op"] == "fwd":
                    continue
                do = st["dout"][i, at:at + rows, j].double()
                dv[i, :n, j // (h // kv)] += p.T @ do
                p.mul_((do @ V.T).sub_((do * o).sum(1, keepdim=True)))
                dq[i, at:at + rows, j] = (p @ K).mul_(st["scale"])
                dk[i, :n, j // (h // kv)] += (p.T @ Q).mul_(st["scale"])
    if c["op"] == "fwd":
        return {"out": out, "lse": lse}
    grads = {"dq": dq, "dk": dk, "dv": dv}
    return grads if c["op"] == "bwd" else {"out": out, **grads}


def exact(case, seed):
    st = prepare(case, seed)
    return _exact_grads(case, st) if case["op"] in ("norm", "clip") else _exact_attention(case, st)
