"""Global gradient norm and clipping over every tensor of a model, in liblsr's kernels.

* ``grad_norm(tensors, norm_type)``                   the norm of all tensors taken as one vector
* ``clip_grads(grads, max_norm, norm_type, out, total_norm)``
                                                      scaled by min(1, max_norm / (norm + 1e-6)), in
                                                      place or into ``out`` of another type
* ``clip_grad_norm_(parameters, max_norm, ...)``      the same on ``p.grad``, with the first four arguments
                                                      of ``torch.nn.utils.clip_grad_norm_`` (norms 1, 2
                                                      and inf, gradients on one device; no ``foreach``)

The tensors may mix fp32, bf16 and fp16 and any shapes; norms are fp32 device scalars, summed in 64
bits in one fixed order, and nothing waits for the device unless ``error_if_nonfinite`` is set. Every
tensor written gets a new version (autograd's check of saved values sees it; a graph's replay does not). The
list travels in the kernels' parameters, so a call can be captured into a CUDA graph. With gradients
sharded over ranks: ``grad_norm`` on each rank's own, the ranks' norms combined (for norm 2 the root
of the sum of squares), then ``clip_grads(..., total_norm=combined)``.

The reference trains unclipped (muon_lm_ddp.py:1367-1381). There is no CPU path: CPU tensors raise
``ValueError``.
"""
from __future__ import annotations

import math
from array import array

import torch
from torch.autograd.graph import increment_version

from . import _lib

_KINDS = {math.inf: 0, 1.0: 1, 2.0: 2}


# A model has hundreds of gradients: their properties are read by map over the unbound getters.
_ptr_of, _numel_of, _size_of, _is_contiguous = (torch.Tensor.data_ptr, torch.Tensor.numel, torch.Tensor.size,
                                                torch.Tensor.is_contiguous)
_device_of, _dtype_of = torch.Tensor.get_device, torch.Tensor.dtype.__get__


def _kind(norm_type) -> int:
    try:
        return _KINDS[float(norm_type)]
    except (KeyError, TypeError, ValueError):
        raise ValueError(f"norm_type must be 1, 2 or inf (got {norm_type!r})") from None


def _dense(t: torch.Tensor) -> bool:
    """Whether t's entries fill one range of memory, each place once."""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz != 1):
        if stride != want:
            return False
        want *= size
    return True


def _check_list(tensors, what: str):
    """(tensors, their addresses, element types, whether every one is contiguous)"""
    ts = [tensors] if isinstance(tensors, torch.Tensor) else list(tensors)
    try:
        dtypes, devices = list(map(_dtype_of, ts)), set(map(_device_of, ts))
        ptrs, whole = array("Q", map(_ptr_of, ts)), all(map(_is_contiguous, ts))
    except (TypeError, RuntimeError, NotImplementedError):  # no tensor, or one without plain memory (sparse, meta)
        raise ValueError(f"{what} must be dense tensors") from None
    if -1 in devices:
        raise ValueError(f"{what} must be CUDA tensors (liblsr has no CPU path)")
    if len(devices) > 1:
        raise ValueError(f"{what} must be on one device (got CUDA devices {sorted(devices)})")
    kinds = set(dtypes)
    if kinds - _lib.DTYPE_CODES.keys():
        raise ValueError(f"{what} must be fp32, bf16 or fp16 (got {kinds - _lib.DTYPE_CODES.keys()})")
    if len(kinds) == 1:
        codes = array("i", (_lib.DTYPE_CODES[dtypes[0]],)) * len(ts)
    else:
        codes = array("i", [_lib.DTYPE_CODES[t] for t in dtypes])
    return ts, ptrs, codes, whole


def _workspace(lib, count: int, like: torch.Tensor) -> torch.Tensor:
    # of this call alone: calls on several streams, or graphs captured here, share nothing
    return like.new_empty(lib.lsr_grad_workspace_bytes(count), dtype=torch.uint8)


def _address(a: array) -> int:
    return a.buffer_info()[0]


def _steps(t: torch.Tensor):
    """[(bytes, most)]: an entry of t lies at its address + sum of bytes * x, 0 <= x <= most, a pair per dimension."""
    size = t.element_size()
    return [(st * size, n - 1) for st, n in zip(t.stride(), t.shape) if n > 1]


def _reaches(steps, lo: int, hi: int) -> bool:
    """Whether a sum of bytes * x, 0 <= x <= most over all steps, lies in [lo, hi]. Where that is not settled within
    10000 trials (strides of no common order), yes."""
    merged: dict[int, int] = {}
    for c, n in steps:
        merged[c] = merged.get(c, 0) + n
    steps = sorted(merged.items(), reverse=True)
    rest, common = [0], [0]  # of the steps from k on: their largest sum, and what every sum is a multiple of
    for c, n in reversed(steps):
        rest.append(rest[-1] + c * n)
        common.append(math.gcd(common[-1], c))
    rest.reverse()
    common.reverse()
    left = 10000

    def search(k, lo, hi):
        nonlocal left
        if hi < 0 or lo > rest[k]:
            return False
        if lo <= 0:
            return True
        if k == len(steps) or hi // common[k] * common[k] < lo:
            return False
        left -= 1
        if left < 0:
            return True
        c, n = steps[k]
        return any(search(k + 1, lo - c * x, hi - c * x) for x in range(max(0, -((rest[k + 1] - lo) // c)), min(n, hi // c) + 1))

    return search(0, lo, hi)


def _share(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether an entry of a and one of b have a byte in common."""
    down = _steps(b)  # counted from b's last entry back
    apart = a.data_ptr() - b.data_ptr() - sum(c * n for c, n in down)
    return _reaches(_steps(a) + down, 1 - a.element_size() - apart, b.element_size() - 1 - apart)


def _repeats(t: torch.Tensor) -> bool:
    """Whether two entries of t have a byte in common."""
    size = t.element_size()
    steps, span = sorted(_steps(t)), size
    for c, n in steps:
        if c < span:
            break
        span += c * n
    else:
        return False
    # two different entries: x and y whose first difference is in step k, where it is 1 or more
    return any(_reaches([(c, n - 1)] + [(d, 2 * m) for d, m in steps[k + 1:]],
                        1 - size - c + sum(d * m for d, m in steps[k + 1:]), size - 1 - c + sum(d * m for d, m in steps[k + 1:]))
               for k, (c, n) in enumerate(steps))


def _check_shared(grads, outs, norm, checked) -> None:
    """ValueError where an output shares memory with another, itself, a gradient that it is not, or the norm; `checked`
    are the numbers of the pairs (gradient, output) that the library compares with one another by itself."""
    spans = []  # (first byte, end, written, compared by the library, tensor)

    def add(t, written, compared):
        at = t.data_ptr()
        spans.append((at, at + sum(c * n for c, n in _steps(t)) + t.element_size(), written, compared, t))

    for i, (g, o) in enumerate(zip(grads, outs)):
        if not o.numel():
            continue
        if i not in checked and _repeats(o):
            raise ValueError("an output's entries share memory (an expanded tensor, say): clip a copy of it")
        add(o, True, i in checked)
        if not (g is o or (g.data_ptr() == o.data_ptr() and g.stride() == o.stride() and g.dtype == o.dtype)):
            add(g, False, i in checked)
    if norm is not None:
        add(norm, False, False)
    spans.sort(key=lambda x: x[0])
    first, end = 0, 0
    for k in range(len(spans) + 1):  # runs of spans that overlap
        if k < len(spans) and spans[k][0] < end:
            end = max(end, spans[k][1])
            continue
        if any(_share(x[4], y[4]) for x, y in _meeting(_folded(spans[first:k]))
               if (x[2] or y[2]) and not (x[3] and y[3])):
            raise ValueError("an output shares memory with another output, a gradient or the norm: clip into copies")
        first, end = k, spans[k][1] if k < len(spans) else 0


def _folded(spans):
    """The spans, or where all are slices of rows equally far apart, their places within a row: slices that lie side by
    side then do not meet."""
    steps = [_steps(x[4]) for x in spans]
    rows = {max(s)[0] if s else 0 for s in steps}
    if len(rows) != 1 or 0 in rows:
        return spans
    row = rows.pop()
    at = [(x[0] - spans[0][0]) % row for x in spans]
    ends = [a + sum(c * n for c, n in s if c != row) + x[4].element_size() for a, s, x in zip(at, steps, spans)]
    if max(ends) > row:
        return spans
    return sorted(((a, e, *x[2:]) for a, e, x in zip(at, ends, spans)), key=lambda x: x[0])


def _meeting(spans):
    """The pairs of them that overlap; in order of their first bytes."""
    open_ = []
    for x in spans:
        open_ = [y for y in open_ if y[1] > x[0]]
        yield from ((x, y) for y in open_)
        open_.append(x)


def _flatten(ts, outs, norm):
    """(gradients, outputs, [(output, where its values are written first)]) that fill ranges of memory in one order."""
    direct = {i for i, (t, o) in enumerate(zip(ts, outs)) if _dense(t) and _dense(o) and t.stride() == o.stride()}
    _check_shared(ts, outs, norm, direct)
    src, dst, back = [], [], []
    for i, (t, o) in enumerate(zip(ts, outs)):
        if i in direct:
            src.append(t)
            dst.append(o)
            continue
        src.append(t.detach().contiguous())
        if o.is_contiguous():
            dst.append(o)
        else:
            dst.append(torch.empty(o.shape, dtype=o.dtype, device=o.device))
            back.append((o, dst[-1]))
    return src, dst, back


def grad_norm(tensors, norm_type: float = 2.0) -> torch.Tensor:
    """The norm (1, 2 or inf) over every entry of every tensor: a 0-d fp32 tensor on their device.

    It has no gradient: of tensors that autograd follows, the result raises RuntimeError where one is asked of it.
    """
    kind = _kind(norm_type)
    ts, *rest = _check_list(tensors, "tensors")
    if not ts:
        return torch.zeros(())
    return _lib.no_gradient("grad_norm", lambda: _norm(ts, *rest, kind), ts)


def _norm(ts, ptrs, dtypes, whole, kind) -> torch.Tensor:
    if not whole:
        ts = [t if _dense(t) else t.detach().contiguous() for t in ts]
        ptrs = array("Q", map(_ptr_of, ts))
    first = ts[0]
    lib = _lib.load()
    with _lib.on_device(first.device):
        norm = first.new_empty((), dtype=torch.float32)
        ws = _workspace(lib, len(ts), first)
        numel = array("q", map(_numel_of, ts))
        rc = lib.lsr_grad_norm(_address(ptrs), _address(numel), _address(dtypes), len(ts), kind, norm.data_ptr(),
                               ws.data_ptr(), ws.numel(), _lib.stream_handle(first.device))
    _lib.check(rc, "lsr_grad_norm")
    return norm


@torch.no_grad()
def clip_grads(grads, max_norm: float, norm_type: float = 2.0, out=None, total_norm: torch.Tensor | None = None) -> torch.Tensor:
    """Scale `grads` by min(1, max_norm / (norm + 1e-6)) and return the norm before it.

    In place when `out` is None; else out[i] = grads[i] * coefficient in out[i]'s type (same shapes,
    e.g. fp32 gradients to the bf16 that the Muon step takes), and out[i] may be grads[i] itself.
    Apart from that no output may share memory with another output or with a gradient (ValueError).
    `total_norm`: a 0-d fp32 device tensor, not part of an output, to be used instead of computing the norm.
    A NaN norm makes every entry NaN, an infinite one makes finite entries 0, as
    torch.nn.utils.clip_grad_norm_ does. Like that one it runs without a gradient of its own; forward-mode
    duals raise NotImplementedError.
    """
    kind = _kind(norm_type)
    max_norm = float(max_norm)
    if not max_norm >= 0.0:
        raise ValueError(f"max_norm must be at least 0 (got {max_norm})")
    src, pin, tin, whole = _check_list(grads, "grads")
    dst, pout, tout = src, pin, tin
    if out is not None:
        dst, pout, tout, same = _check_list(out, "out")
        whole = whole and same
        if list(map(_size_of, dst)) != list(map(_size_of, src)):
            raise ValueError("out must be one tensor of the same shape for each gradient")
    outs = dst
    if not src:
        return torch.zeros(()) if total_norm is None else total_norm
    _lib.refuse_duals("clip_grads", [*src, *dst] if total_norm is None else [*src, *dst, total_norm])
    first = src[0]
    dev = first.device
    if dst[0].get_device() != first.get_device():
        raise ValueError("out must be on the gradients' device")
    if total_norm is not None and (total_norm.dtype != torch.float32 or total_norm.device != dev or total_norm.numel() != 1):
        raise ValueError("total_norm must be one fp32 value on the gradients' device")
    back = []  # (output, dense tensor to copy into it)
    if not whole:
        src, dst, back = _flatten(src, dst, total_norm)
        pin, pout = array("Q", map(_ptr_of, src)), array("Q", map(_ptr_of, dst))
    lib = _lib.load()
    with _lib.on_device(dev):
        norm = first.new_empty((), dtype=torch.float32) if total_norm is None else total_norm
        ws = _workspace(lib, len(src), first) if total_norm is None else None
        numel = array("q", map(_numel_of, src))
        rc = lib.lsr_grad_clip(_address(pin), _address(pout), _address(numel), _address(tin), _address(tout), len(src),
                               kind, max_norm, int(total_norm is not None), norm.data_ptr(),
                               ws.data_ptr() if ws is not None else None, ws.numel() if ws is not None else 0,
                               _lib.stream_handle(dev))
        _lib.check(rc, "lsr_grad_clip")
        for o, t in back:
            o.copy_(t)
    # the kernels write through addresses: autograd, and whatever is kept for a tensor's version, is told here
    increment_version(outs)
    return norm


def clip_grad_norm_(parameters, max_norm: float, norm_type: float = 2.0, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Clip the gradients of `parameters` in place by their global norm and return it (0-d fp32).

    Parameters without a gradient are passed over; one listed twice counts once. With
    `error_if_nonfinite` the norm is read back first, and a NaN or infinite one raises RuntimeError
    with the gradients as they were.
    """
    ps = [parameters] if isinstance(parameters, torch.Tensor) else parameters
    grads = list({id(p): p.grad for p in ps if p.grad is not None}.values())
    if not error_if_nonfinite:
        return clip_grads(grads, max_norm, norm_type)
    norm = grad_norm(grads, norm_type)
    if not math.isfinite(float(norm)):
        raise RuntimeError(f"the gradients' norm of order {float(norm_type)} is {float(norm)}: they are not clipped")
    return clip_grads(grads, max_norm, norm_type, total_norm=norm) if grads else norm


__all__ = ["grad_norm", "clip_grads", "clip_grad_norm_"]
