"""CPU: argument checks of the gradient and attention operators (C ABI and Python), their oracles
against torch autograd, and the driver's adapter."""
from __future__ import annotations

import ctypes
import math
from array import array

import numpy as np
import pytest
import torch

from oracle import attention as oa
from oracle import grad as og


def _adr(a):
    return a.buffer_info()[0]


def test_grad_c_abi_rejects_bad_lists_before_any_device_work():
    from lsr import _lib
    lib = _lib.load()
    assert lib.lsr_grad_workspace_bytes(-1) == 0
    assert lib.lsr_grad_workspace_bytes(5000) > lib.lsr_grad_workspace_bytes(1) > 0
    ptr, n, t = array("Q", [4096, 8192]), array("q", [100, 100]), array("i", [0, 0])
    ws, norm = ctypes.create_string_buffer(1 << 20), ctypes.create_string_buffer(4)

    def norm_rc(ptr=ptr, n=n, t=t, count=2, kind=2, out=norm, nbytes=1 << 20):
        return lib.lsr_grad_norm(_adr(ptr), _adr(n), _adr(t), count, kind, out, ws, nbytes, None)

    assert norm_rc(kind=3) == -1 and norm_rc(count=-1) == -1 and norm_rc(out=None) == -1
    assert norm_rc(t=array("i", [0, 9])) == -1 and norm_rc(n=array("q", [1, -1])) == -1
    assert norm_rc(ptr=array("Q", [0, 8192])) == -1   # entries but no memory
    assert norm_rc(ptr=array("Q", [4098, 8192])) == -2  # not on its type's boundary
    assert norm_rc(nbytes=64) == -3

    def clip_rc(src, dst, n=n, t=t, u=t, bound=1.0):
        return lib.lsr_grad_clip(_adr(src), _adr(dst), _adr(n), _adr(t), _adr(u), 2, 2, bound, 0, norm, ws, 1 << 20, None)

    if not torch.cuda.is_available():  # past the checks there is no device here; made-up addresses go no further
        assert clip_rc(ptr, ptr) == -6 and clip_rc(ptr, array("Q", [16384, 32768])) == -6
        assert clip_rc(array("Q", [4096, 4496]), array("Q", [4096, 4496])) == -6  # side by side
    assert clip_rc(ptr, ptr, bound=-1.0) == -1 and clip_rc(ptr, ptr, bound=math.nan) == -1
    assert clip_rc(ptr, array("Q", [16384, 16384])) == -1      # two outputs in one place
    assert clip_rc(ptr, array("Q", [8192, 16384])) == -1       # an output over another's input
    assert clip_rc(ptr, array("Q", [4100, 16384])) == -1       # over its own input, but not in place
    assert clip_rc(ptr, ptr, u=array("i", [1, 0])) == -1       # in place with another type


def _args(dtype=1, b=2, n=3, m=4, h=6, hk=2, d=64, causal=1):
    from lsr.attention import _ARGS
    return _ARGS.pack(dtype, b, n, m, h, hk, d, causal, 0.5, *([4096] * 10), *([64] * 25))


def test_attention_c_abi_rejects_bad_arguments_before_any_device_work():
    from lsr import _lib
    lib = _lib.load()
    size = lib.lsr_attention_backward_workspace_bytes
    assert size(_args()) >= 2 * 6 * 3 * 4
    assert lib.lsr_attention_forward(None, None, 0, None) == -1
    for bad, rc in ((dict(dtype=3), -1), (dict(b=-1), -1), (dict(h=0), -1), (dict(d=0), -1), (dict(causal=2), -1),
                    (dict(hk=4), -2), (dict(d=129), -2), (dict(b=1 << 24), -2)):
        assert lib.lsr_attention_forward(_args(**bad), None, 0, None) == rc, bad
        assert lib.lsr_attention_backward(_args(**bad), 4096, 1 << 20, None) == rc, bad
        assert size(_args(**bad)) == 0
    assert lib.lsr_attention_backward(_args(), 4096, 16, None) == -3
    assert lib.lsr_attention_forward(_args(b=0), None, 0, None) == 0
    assert lib.lsr_attention_forward(_args(n=0), None, 0, None) == 0


def test_cpu_tensors_are_refused():
    import lsr
    from lsr import attention as A
    t = torch.zeros(1, 2, 3, 8)
    with pytest.raises(ValueError):
        A.attention(t, t, t)
    with pytest.raises(ValueError):
        lsr.grad_norm([t])
    with pytest.raises(ValueError):
        lsr.clip_grads([t], 1.0)
    p = torch.nn.Parameter(t)
    p.grad = t.clone()
    with pytest.raises(ValueError):
        lsr.clip_grad_norm_([p], 1.0)
    assert float(lsr.grad_norm([])) == 0.0 and float(lsr.clip_grad_norm_([torch.nn.Parameter(t)], 1.0)) == 0.0


@pytest.mark.parametrize("n,m,h,hk,causal,pad", [(5, 5, 4, 4, True, False), (3, 7, 4, 2, True, True), (6, 2, 3, 1, True, False),
                                                 (4, 9, 2, 2, False, True)])
def test_attention_oracle_against_autograd(n, m, h, hk, causal, pad):
    g = torch.Generator().manual_seed(n * m)
    q, k, v, do = (torch.randn(2, length, heads, 8, generator=g, dtype=torch.float64) for length, heads in
                   ((n, h), (m, hk), (m, hk), (n, h)))
    mask = None
    if pad:
        mask = torch.rand(2, m, generator=g) < 0.6
        mask[1] = False
    leaves = [t.clone().requires_grad_(True) for t in (q, k, v)]
    see = torch.from_numpy(oa.seen(2, n, m, causal, mask))
    K, V = (t.repeat_interleave(h // hk, 2).transpose(1, 2) for t in leaves[1:])
    s = (0.3 * leaves[0].transpose(1, 2) @ K.transpose(-1, -2)).masked_fill(~see, -1e300)
    p = torch.softmax(s, -1) * see  # rows that see nothing: zeros
    ref = (p @ V).transpose(1, 2)
    ref.backward(do)
    out, lse, pr = oa.forward(q.numpy(), k.numpy(), v.numpy(), 0.3, causal, mask)
    assert np.allclose(out, ref.detach().numpy(), atol=1e-12) and np.allclose(pr, p.detach().numpy(), atol=1e-12)
    assert np.array_equal(np.isneginf(lse), ~see.numpy().any(-1).repeat(h, 1))
    grads = oa.backward(do.numpy(), q.numpy(), k.numpy(), v.numpy(), out, lse, 0.3, causal, mask)[:3]
    for got, leaf in zip(grads, leaves):
        assert np.allclose(got, leaf.grad.numpy(), atol=1e-12)


def test_grad_oracle():
    assert og.norm([np.array([3.0]), np.array([[4.0]]), np.zeros(0)], 2.0) == 5.0
    assert og.norm([np.array([-3.0, 1.0])], np.inf) == 3.0 and og.norm([np.array([-3.0, 1.0])], 1.0) == 4.0
    assert og.coefficient(0.5, 1.0) == 1.0 and abs(og.coefficient(2.0, 1.0) - 0.5) < 1e-6
    assert og.coefficient(math.inf, 1.0) == 0.0 and math.isnan(og.coefficient(math.nan, 1.0))


def test_driver_flags_and_attention_adapter_refusals():
    from lsr import lm_driver as D
    a = D.build_parser().parse_args(["--muon-mode", "batched"])
    assert a.max_grad_norm == 0.0 and a.attention == "model"
    t = torch.zeros(1, 2, 3, 8)
    with pytest.raises(ValueError, match="attn_pdrop"):
        D._lsr_attention(torch.nn.Identity(), t, t, t, None, dropout=0.1)
    with pytest.raises(ValueError, match="sliding_window"):
        D._lsr_attention(torch.nn.Identity(), t, t, t, None, sliding_window=4)

    def causal_mask_function():
        pass

    def packed_mask_function():
        pass

    m = torch.ones(1, 3, dtype=torch.bool)
    assert D._lsr_attention_mask(mask_function=causal_mask_function, attention_mask=m, q_length=3) is m
    with pytest.raises(ValueError):
        D._lsr_attention_mask(mask_function=packed_mask_function, attention_mask=m)


@pytest.mark.parametrize("given", [0, 1])
def test_a_norm_inside_an_output_is_refused(given):
    from lsr import _lib
    lib = _lib.load()
    n, t = array("q", [100, 100]), array("i", [0, 0])
    ws = ctypes.create_string_buffer(1 << 20)

    def rc(src, dst, norm):
        src, dst = array("Q", src), array("Q", dst)
        return lib.lsr_grad_clip(_adr(src), _adr(dst), _adr(n), _adr(t), _adr(t), 2, 2, 1.0, given, norm, ws, 1 << 20, None)

    for at in (4096, 4096 + 396, 8192 + 4):
        assert rc([4096, 8192], [4096, 8192], at) == -1
        assert rc([16384, 32768], [4096, 8192], at) == -1
    if not given:  # the norm would be written over a gradient
        assert rc([4096, 8192], [16384, 32768], 4100) == -1
    if not torch.cuda.is_available():
        assert rc([4096, 8192], [4096, 8192], 4096 + 400) == -6
        if given:
            assert rc([4096, 8192], [16384, 32768], 4100) == -6  # a gradient's own entry, only read


@pytest.mark.parametrize("dtype,slot,off", [(1, 0, 1), (0, 1, 2), (2, 4, 1), (0, 4, 2), (1, 5, 2), (1, 6, 1), (0, 9, 2)])
def test_attention_tensors_off_their_entries_are_refused(dtype, slot, off):
    """slot: of q, k, v, key_mask, out, lse, dout, dq, dk, dv."""
    import struct
    from lsr import _lib
    lib = _lib.load()
    raw = bytearray(_args(dtype=dtype))
    at = 40 + 8 * slot
    assert struct.unpack_from("=Q", raw, at)[0] == 4096
    struct.pack_into("=Q", raw, at, 4096 + off)
    assert lib.lsr_attention_backward(bytes(raw), 1 << 20, 1 << 30, None) == -2
    assert lib.lsr_attention_forward(bytes(raw), 1 << 20, 1 << 30, None) == -2
