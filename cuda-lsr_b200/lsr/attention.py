"""Softmax attention and its gradients, in liblsr's kernels.

* ``attention(q, k, v, causal, scale, key_mask)``            differentiable
* ``attention_forward(q, k, v, ...)``                        -> (out, lse)
* ``attention_backward(dout, q, k, v, out, lse, ...)``       -> (dq, dk, dv)

q is [batch, q_len, heads, dim], k and v [batch, kv_len, kv_heads, dim], heads a multiple of kv_heads
(query head h reads key head h // (heads // kv_heads)), dim 1..128; fp32, bf16 or fp16, all alike. Any
strides: entries of a head that are not contiguous are copied first, everything else is read in place
(the three parts of one projection's output, or [batch, heads, length, dim] tensors transposed).
``causal`` lets query i see keys up to i + kv_len - q_len, so that the last query sees the last key.
``key_mask`` is bool [batch, kv_len], True = seen; what the masked keys hold does not matter. A query
that sees no key has output 0, lse minus infinity and no gradient. lse is fp32 [batch, heads, q_len],
the natural logarithm. ``scale`` defaults to dim ** -0.5.

The backward pass computes the probabilities again from lse; memory grows with the lengths, not with
their product. Same inputs, same bits: nothing is summed in an order that varies. There is no dropout
and no second derivative. The reference leaves attention to its models' library
(muon_lm_ddp.py:752-822); there is no CPU path: CPU tensors raise ``ValueError``.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib

# lsr_attention_args (include/lsr.h): 8 ints, a float and its padding, 10 pointers, 25 strides
_ARGS = struct.Struct("=8if4x10Q25q")
_NONE = (0, 0, 0)


def _check(q, k, v, key_mask):
    for t, name in ((q, "q"), (k, "k"), (v, "v")):
        if not t.is_cuda:
            raise ValueError(f"{name} must be a CUDA tensor (liblsr has no CPU path)")
        if t.dim() != 4:
            raise ValueError(f"{name} must be [batch, length, heads, dim]")
    if q.dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"q must be fp32, bf16 or fp16 (got {q.dtype})")
    if k.dtype != q.dtype or v.dtype != q.dtype:
        raise ValueError(f"q, k and v must be of one type (got {q.dtype}, {k.dtype}, {v.dtype})")
    if k.device != q.device or v.device != q.device:
        raise ValueError("q, k and v must be on the same CUDA device")
    b, _, h, d = q.shape
    if k.shape != v.shape:
        raise ValueError(f"k and v must have one shape (got {tuple(k.shape)} and {tuple(v.shape)})")
    _, n, hk, dk = k.shape
    if k.shape[0] != b or dk != d:
        raise ValueError(f"k is {tuple(k.shape)}: batch {b} and dim {d} are q's")
    if not 1 <= d <= 128:
        raise ValueError(f"dim must be 1 to 128 (got {d})")
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"heads ({h}) must be a multiple of kv_heads ({hk})")
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != (b, n):
            raise ValueError(f"key_mask must be bool [{b}, {n}]")
        if key_mask.device != q.device:
            raise ValueError("key_mask must be on q's device")


def _read(t: torch.Tensor) -> torch.Tensor:
    return t if t.stride(3) == 1 or t.shape[3] == 1 else t.contiguous()


def _mask(m: torch.Tensor | None) -> torch.Tensor | None:
    return m if m is None or m.stride(1) == 1 or m.shape[1] <= 1 else m.contiguous()


def _pack(q, k, v, key_mask, causal, scale, out, lse, dout=None, dq=None, dk=None, dv=None) -> bytes:
    back = dout is not None
    ptr = [q.data_ptr(), k.data_ptr(), v.data_ptr(), key_mask.data_ptr() if key_mask is not None else 0,
           out.data_ptr(), lse.data_ptr()]
    ptr += [dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()] if back else [0, 0, 0, 0]
    strides = [s for t in (q, k, v, out) for s in t.stride()[:3]]
    strides += [s for t in (dout, dq, dk, dv) for s in t.stride()[:3]] if back else [0] * 12
    b, n, h, d = q.shape
    return _ARGS.pack(_lib.DTYPE_CODES[q.dtype], b, n, k.shape[1], h, k.shape[2], d, int(causal), scale, *ptr, *strides,
                      key_mask.stride(0) if key_mask is not None else 0)


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    # of this call alone: calls on several streams, or graphs captured here, share nothing
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _scale(scale, q) -> float:
    return float(q.shape[3]) ** -0.5 if scale is None else float(scale)


@torch.no_grad()
def attention_forward(q, k, v, *, causal: bool = False, scale: float | None = None, key_mask=None):
    """(out, lse): the attention of q over k and v, and the log-sum-exp of each query's scores."""
    _check(q, k, v, key_mask)
    q, k, v, key_mask = _read(q), _read(k), _read(v), _mask(key_mask)
    b, n, h, d = q.shape
    lib = _lib.load()
    with _lib.on_device(q.device):
        out = torch.empty((b, n, h, d), dtype=q.dtype, device=q.device)
        lse = torch.empty((b, h, n), dtype=torch.float32, device=q.device)
        args = _pack(q, k, v, key_mask, causal, _scale(scale, q), out, lse)
        nbytes = lib.lsr_attention_forward_workspace_bytes(args)
        ws = _workspace(nbytes, q.device)
        rc = lib.lsr_attention_forward(args, ws.data_ptr() if nbytes else None, nbytes, _lib.stream_handle(q.device))
    _lib.check(rc, "lsr_attention_forward")
    return out, lse


@torch.no_grad()
def attention_backward(dout, q, k, v, out, lse, *, causal: bool = False, scale: float | None = None, key_mask=None):
    """(dq, dk, dv) from the output's gradient and what attention_forward returned for the same arguments."""
    _check(q, k, v, key_mask)
    for t, name in ((dout, "dout"), (out, "out")):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must have q's shape, type and device")
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError("lse must be fp32 [batch, heads, q_len] on q's device")
    dout, q, k, v, out, key_mask = _read(dout), _read(q), _read(k), _read(v), _read(out), _mask(key_mask)
    lse = lse.contiguous()
    lib = _lib.load()
    with _lib.on_device(q.device):
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
        args = _pack(q, k, v, key_mask, causal, _scale(scale, q), out, lse, dout, dq, dk, dv)
        nbytes = lib.lsr_attention_backward_workspace_bytes(args)
        ws = _workspace(nbytes, q.device)
        rc = lib.lsr_attention_backward(args, ws.data_ptr() if nbytes else None, nbytes, _lib.stream_handle(q.device))
    _lib.check(rc, "lsr_attention_backward")
    return dq, dk, dv


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, causal, scale):
        out, lse = attention_forward(q, k, v, causal=causal, scale=scale, key_mask=key_mask)
        ctx.save_for_backward(q, k, v, key_mask, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, key_mask, out, lse = ctx.saved_tensors
        dq, dk, dv = attention_backward(dout, q, k, v, out, lse, causal=ctx.causal, scale=ctx.scale, key_mask=key_mask)
        return dq, dk, dv, None, None, None


def attention(q, k, v, *, causal: bool = False, scale: float | None = None, key_mask=None) -> torch.Tensor:
    """The attention of q over k and v, [batch, q_len, heads, dim]; gradients flow to q, k and v."""
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _Attention.apply(q, k, v, key_mask, bool(causal), scale)
    return attention_forward(q, k, v, causal=causal, scale=scale, key_mask=key_mask)[0]


__all__ = ["attention", "attention_forward", "attention_backward"]
