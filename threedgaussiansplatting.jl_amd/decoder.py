"""Operators of a learned decoder of rendered images over libtdgs.so: cross attention to an
encoder's states, with the gradient of each operand.

What a network that turns rendered features into images needs besides matrix products (an
appearance model of a photo collection, a refiner). The reference has no counterpart. Tensors are
float32, bfloat16 or float16 on the GPU; outputs and gradients are written into the tensors given,
on the current stream, without synchronisation. temp is scratch of the size its function's
*_temp() gives: with None a call allocates its own.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .core import check, dptr, lib, stream_ptr

DTYPES = {torch.float32: abi.TDGS_F32, torch.bfloat16: abi.TDGS_BF16, torch.float16: abi.TDGS_F16}


def _require(cond, message):
    if not cond:
        raise ValueError(message)


def _tensor(t, name, like):
    _require(isinstance(t, torch.Tensor) and t.is_cuda, f"{name} must be a tensor on the GPU")
    _require(t.device == like.device, f"{name} is on {t.device}, not on {like.device}")


# ------------------------------------------------------------------------------------
# Cross attention
# ------------------------------------------------------------------------------------

def _heads(t, name, shape, like):
    _tensor(t, name, like)
    _require(t.dtype == like.dtype, f"{name} is {t.dtype}, not {like.dtype}")
    _require(tuple(t.shape) == shape, f"{name} has shape {tuple(t.shape)}, not {shape}")
    s = t.stride()
    _require(s[3] == 1 or shape[3] <= 1, f"the last dimension of {name} must be contiguous")
    return abi.HeadsC(t.data_ptr(), s[0], s[1], s[2])


def _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask, temp):
    """The tdgs_attention of these tensors (v and out None: sizes only)."""
    _tensor(q, "q", q)
    _require(q.dtype in DTYPES, f"q is {q.dtype}: float32, bfloat16 and float16 are supported")
    _require(q.dim() == 4 and isinstance(k, torch.Tensor) and k.dim() == 4,
             "q and k must be (batch, length, heads, head_dim)")
    b, lq, h, d = q.shape
    kb, lk, hk = k.shape[:3]
    a = abi.AttentionC()
    a.dtype, a.batch, a.kv_batch, a.q_len, a.kv_len = DTYPES[q.dtype], b, kb, lq, lk
    a.heads, a.kv_heads, a.head_dim = h, hk, d
    a.scale = d ** -0.5 if scale is None else scale
    a.q = _heads(q, "q", (b, lq, h, d), q)
    a.k = _heads(k, "k", (kb, lk, hk, d), q)
    if v is not None:
        a.v = _heads(v, "v", (kb, lk, hk, d), q)
        a.out = _heads(out, "out", (b, lq, h, d), q)
    if kv_lengths is not None:
        _tensor(kv_lengths, "kv_lengths", q)
        _require(kv_lengths.dtype == torch.int32 and tuple(kv_lengths.shape) == (kb,) and kv_lengths.is_contiguous(),
                 f"kv_lengths must be {kb} contiguous int32 values")
        a.kv_lengths = kv_lengths.data_ptr()
    if kv_mask is not None:
        _tensor(kv_mask, "kv_mask", q)
        _require(kv_mask.dtype in (torch.bool, torch.uint8) and tuple(kv_mask.shape) == (kb, lk)
                 and (kv_mask.stride(1) == 1 or lk <= 1), f"kv_mask must be bool or uint8, ({kb}, {lk}), its rows contiguous")
        a.kv_mask, a.kv_mask_stride = kv_mask.data_ptr(), kv_mask.stride(0)
    if lse is not None:
        _tensor(lse, "lse", q)
        _require(lse.dtype == torch.float32 and tuple(lse.shape) == (b, h, lq) and lse.is_contiguous(),
                 f"lse must be contiguous float32, ({b}, {h}, {lq})")
        a.lse = lse.data_ptr()
    if temp is not None:
        _temp(temp, q)
        a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    return a


def _temp(temp, like):
    _tensor(temp, "temp", like)
    _require(temp.dtype == torch.uint8 and temp.is_contiguous(), "temp must be contiguous uint8")


def _own_temp(a, grad, like):
    n = lib().tdgs_cross_attention_temp_bytes(C.byref(a), grad)
    temp = torch.empty(max(n, 1), dtype=torch.uint8, device=like.device)
    a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    return temp


def cross_attention_temp(q, k, grad=False):
    """Scratch for cross_attention_ (with grad also cross_attention_grad_) on tensors of these sizes."""
    a = _attention(q, k, None, None, None, None, None, None, None)
    n = lib().tdgs_cross_attention_temp_bytes(C.byref(a), int(grad))
    return torch.empty(max(n, 1), dtype=torch.uint8, device=q.device)


def cross_attention_(out, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None, lse=None, temp=None):
    """out = softmax(scale q k^T) v over the allowed keys, per head (tdgs_cross_attention).

    q and out are (batch, q_len, heads, head_dim), k and v (kv_batch, kv_len, kv_heads, head_dim):
    kv_batch is batch, or 1 for one encoder's states shared by the batch; heads is a multiple of
    kv_heads, neighbouring heads sharing one. Any strides with the last dimension contiguous, head_dim
    up to 128, scale head_dim ** -0.5 by default. kv_lengths (kv_batch int32) allows each batch's first
    keys, kv_mask (kv_batch, kv_len; bool or uint8) single ones; k and v may hold anything where a key is not
    allowed. A query without allowed keys gets zeros. lse (batch, heads, q_len; float32), where given,
    receives the logarithm of each softmax's sum, which the gradient needs."""
    a = _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask, temp)
    if temp is None:
        temp = _own_temp(a, 0, q)
    check(lib().tdgs_cross_attention(stream_ptr(q.device), C.byref(a)))
    return out


def cross_attention_grad_(dq, dk, dv, dout, out, lse, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None,
                          temp=None):
    """The gradients of sum(dout * out) for cross_attention_'s operands (tdgs_cross_attention_grad), from
    its out and lse. dk and dv are summed over the heads, and batches, that share a key."""
    a = _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask, temp)
    _require(lse is not None, "the gradient needs the forward call's lse")
    if temp is None:
        temp = _own_temp(a, 1, q)
    g = abi.AttentionGradsC()
    g.dout = _heads(dout, "dout", tuple(q.shape), q)
    g.dq = _heads(dq, "dq", tuple(q.shape), q)
    g.dk = _heads(dk, "dk", tuple(k.shape), q)
    g.dv = _heads(dv, "dv", tuple(k.shape), q)
    check(lib().tdgs_cross_attention_grad(stream_ptr(q.device), C.byref(a), C.byref(g)))
    return dq, dk, dv
