"""Softmax attention and its gradients, in liblsr's kernels.

* ``attention(q, k, v, causal, scale, key_mask)``            differentiable
* ``attention_forward(q, k, v, ...)``                        -> (out, lse)
* ``attention_backward(dout, q, k, v, out, lse, ...)``       -> (dq, dk, dv)

q is [batch, q_len, heads, dim], k and v [batch, kv_len, kv_heads, dim], heads a multiple of kv_heads
(query head h reads key head h // (heads // kv_heads)), dim 1..128; fp32, bf16 or fp16, all alike. Any
strides: the three parts of one projection's output or [batch, heads, length, dim] tensors transposed are
read in place; what is expanded, not on 16-byte boundaries or not contiguous within a head is copied first.
``causal`` lets query i see keys up to i + kv_len - q_len, so that the last query sees the last key.
``key_mask`` is bool [batch, kv_len], True = seen; what the masked keys hold does not matter, NaN included
(keys hidden by causality alone have to be finite: 0 times a NaN among them is a NaN). A query that sees
no key has output 0, lse minus infinity and no gradient. lse is fp32 [batch, heads, q_len], the natural
logarithm. ``scale`` defaults to dim ** -0.5.

Scores, exponentials and sums are fp32. With bf16 and fp16 tensors the probabilities and the scores' gradients are
rounded to that type for the products that take them, as the outputs are: results are off by up to 1.5 times what
rounding the exact ones makes (bf16 0.0024 relative, fp16 0.0003). fp32 tensors keep 32 bits throughout.

The backward pass computes the probabilities again from lse; memory grows with the lengths, not with
their product. Same inputs, same bits: nothing is summed in an order that varies. There is no dropout,
no second derivative and no forward-mode derivative (NotImplementedError). The two halves lie outside autograd: what
they return is cut off from the graph of their inputs. A captured backward pass wants no eager graph of the same leaves alive
(PyTorch adds to a leaf's gradient on the stream of the leaf's first graph). The reference leaves attention to its models' library
(muon_lm_ddp.py:752-822); there is no CPU path: CPU tensors raise ``ValueError``.
"""
from __future__ import annotations

import struct

import torch
from torch.autograd.function import once_differentiable

from . import _lib

# lsr_attention_args (include/lsr.h): 8 ints, a float and its padding, 10 pointers, 25 strides
_ARGS = struct.Struct("=8if4x10Q25q")
_NO_GRADS = ((0,) * 4, (0,) * 12)


def _check(q, k, v, key_mask):
    if not (q.is_cuda and k.is_cuda and v.is_cuda):
        raise ValueError("q, k and v must be CUDA tensors (liblsr has no CPU path)")
    qs, ks = q.shape, k.shape
    if len(qs) != 4 or len(ks) != 4:
        raise ValueError("q, k and v must be [batch, length, heads, dim]")
    dtype, device = q.dtype, q.get_device()
    if dtype not in _lib.DTYPE_CODES:
        raise ValueError(f"q must be fp32, bf16 or fp16 (got {dtype})")
    if k.dtype != dtype or v.dtype != dtype:
        raise ValueError(f"q, k and v must be of one type (got {dtype}, {k.dtype}, {v.dtype})")
    if k.get_device() != device or v.get_device() != device:
        raise ValueError("q, k and v must be on the same CUDA device")
    if v.shape != ks:
        raise ValueError(f"k and v must have one shape (got {tuple(ks)} and {tuple(v.shape)})")
    b, _, h, d = qs
    bk, n, hk, dk = ks
    if bk != b or dk != d:
        raise ValueError(f"k is {tuple(ks)}: batch {b} and dim {d} are q's")
    if not 1 <= d <= 128:
        raise ValueError(f"dim must be 1 to 128 (got {d})")
    if hk < 1 or h < 1 or h % hk:
        raise ValueError(f"heads ({h}) must be a multiple of kv_heads ({hk})")
    if key_mask is not None:
        if key_mask.dtype != torch.bool or key_mask.shape != (b, n):
            raise ValueError(f"key_mask must be bool [{b}, {n}]")
        if key_mask.get_device() != device:
            raise ValueError("key_mask must be on q's device")


def _read(t: torch.Tensor) -> torch.Tensor:
    """t, or a copy where its strides or address keep it from the kernels that dim and type allow."""
    if t.is_contiguous() and not t.data_ptr() & 15:
        return t
    *strides, last = t.stride()
    *sizes, d = t.shape
    good = last == 1 or d == 1
    if good and d % 8 == 0 and t.element_size() == 2:  # on the tensor cores, read by TMA
        good = not t.data_ptr() & 15 and all(st % 8 == 0 and st > 0 for st, sz in zip(strides, sizes) if sz != 1)
    return t if good else t.detach().clone(memory_format=torch.contiguous_format)


def _mask(m: torch.Tensor | None) -> torch.Tensor | None:
    return m if m is None or m.stride(1) == 1 or m.shape[1] <= 1 else m.contiguous()


def _pack(q, k, v, key_mask, causal, scale, out, lse, dout=None, dq=None, dk=None, dv=None) -> bytes:
    b, n, h, d = q.shape
    m, hk = k.shape[1:3]
    own = n * h * d, h * d, d  # strides of a contiguous tensor of q's shape
    back = _NO_GRADS
    if dout is not None:
        own_k = m * hk * d, hk * d, d
        back = ((dout.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr()), (*dout.stride()[:3], *own, *own_k, *own_k))
    return _ARGS.pack(
        _lib.DTYPE_CODES[q.dtype], b, n, m, h, hk, d, 1 if causal else 0, d ** -0.5 if scale is None else scale,
        q.data_ptr(), k.data_ptr(), v.data_ptr(), 0 if key_mask is None else key_mask.data_ptr(), out.data_ptr(),
        lse.data_ptr(), *back[0], *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], *out.stride()[:3], *back[1],
        0 if key_mask is None else key_mask.stride(0))


def _workspace(nbytes: int, device: torch.device) -> torch.Tensor | None:
    # of this call alone: calls on several streams, or graphs captured here, share nothing
    return torch.empty(nbytes, dtype=torch.uint8, device=device) if nbytes else None


def _forward(q, k, v, causal, scale, key_mask):
    _check(q, k, v, key_mask)
    q, k, v, key_mask = _read(q), _read(k), _read(v), _mask(key_mask)
    b, n, h, d = q.shape
    lib, dev = _lib.load(), q.device
    with _lib.on_device(dev):
        out = q.new_empty((b, n, h, d))
        lse = q.new_empty((b, h, n), dtype=torch.float32)
        args = _pack(q, k, v, key_mask, causal, scale, out, lse)
        nbytes = lib.lsr_attention_forward_workspace_bytes(args)
        ws = _workspace(nbytes, dev)
        rc = lib.lsr_attention_forward(args, ws.data_ptr() if nbytes else None, nbytes, _lib.stream_handle(dev))
    _lib.check(rc, "lsr_attention_forward")
    return out, lse


def attention_forward(q, k, v, *, causal: bool = False, scale: float | None = None, key_mask=None):
    """(out, lse): the attention of q over k and v, and the log-sum-exp of each query's scores, outside autograd."""
    _lib.refuse_duals("attention_forward", (q, k, v))
    return _forward(q, k, v, causal, scale, key_mask)


def _backward(dout, q, k, v, out, lse, causal, scale, key_mask):
    _check(q, k, v, key_mask)
    for t, name in ((dout, "dout"), (out, "out")):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise ValueError(f"{name} must have q's shape, type and device")
    if lse.shape != (q.shape[0], q.shape[2], q.shape[1]) or lse.dtype != torch.float32 or lse.device != q.device:
        raise ValueError("lse must be fp32 [batch, heads, q_len] on q's device")
    dout, q, k, v, out, key_mask = _read(dout), _read(q), _read(k), _read(v), _read(out), _mask(key_mask)
    lse = lse.contiguous()
    lib, dev = _lib.load(), q.device
    with _lib.on_device(dev):
        dq, dk, dv = q.new_empty(q.shape), k.new_empty(k.shape), k.new_empty(k.shape)
        args = _pack(q, k, v, key_mask, causal, scale, out, lse, dout, dq, dk, dv)
        nbytes = lib.lsr_attention_backward_workspace_bytes(args)
        ws = _workspace(nbytes, dev)
        rc = lib.lsr_attention_backward(args, ws.data_ptr() if nbytes else None, nbytes, _lib.stream_handle(dev))
    _lib.check(rc, "lsr_attention_backward")
    return dq, dk, dv


def attention_backward(dout, q, k, v, out, lse, *, causal: bool = False, scale: float | None = None, key_mask=None):
    """(dq, dk, dv) from the output's gradient and what attention_forward returned for the same arguments, outside autograd."""
    _lib.refuse_duals("attention_backward", (dout, q, k, v, out, lse))
    return _backward(dout, q, k, v, out, lse, causal, scale, key_mask)


class _Attention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, key_mask, causal, scale):
        out, lse = _forward(q, k, v, causal, scale, key_mask)
        ctx.save_for_backward(q, k, v, key_mask, out, lse)
        ctx.causal, ctx.scale = causal, scale
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        q, k, v, key_mask, out, lse = ctx.saved_tensors
        return *_backward(dout, q, k, v, out, lse, ctx.causal, ctx.scale, key_mask), None, None, None


def attention(q, k, v, *, causal: bool = False, scale: float | None = None, key_mask=None) -> torch.Tensor:
    """The attention of q over k and v, [batch, q_len, heads, dim]; gradients flow to q, k and v."""
    if _lib.differentiated((q, k, v)):
        return _Attention.apply(q, k, v, key_mask, bool(causal), scale)
    return _forward(q, k, v, causal, scale, key_mask)[0]


__all__ = ["attention", "attention_forward", "attention_backward"]
