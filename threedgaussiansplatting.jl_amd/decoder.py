"""Operators of a learned decoder of rendered images over libtdgs.so: cross attention to an
encoder's states, group norm with an activation (channels last) and embedding lookup, each with
its gradients.

What a network that turns rendered features into images needs besides matrix products (an
appearance model of a photo collection, a refiner, a codebook of Gaussian attributes). The reference has no counterpart. Tensors are
float32, bfloat16 or float16 on the GPU; outputs and gradients are written into the tensors given,
on the current stream, without synchronisation. temp is scratch of the size its function's
*_temp() gives: with None a call allocates its own.
"""
from __future__ import annotations

import ctypes as C

import torch

from . import abi
from .core import _handle, check, dptr, lib, stream_ptr

DTYPES = {torch.float32: abi.TDGS_F32, torch.bfloat16: abi.TDGS_BF16, torch.float16: abi.TDGS_F16}

ACTIVATIONS = {"identity": abi.TDGS_ACT_IDENTITY, "silu": abi.TDGS_ACT_SILU, "gelu": abi.TDGS_ACT_GELU,
               "relu": abi.TDGS_ACT_RELU}


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


def _new_temp(size, a, grad, like):
    return torch.empty(max(size(C.byref(a), int(grad)), 1), dtype=torch.uint8, device=like.device)


def cross_attention_temp(q, k, grad=False):
    """Scratch for cross_attention_ (with grad also cross_attention_grad_) on tensors of these sizes."""
    a = _attention(q, k, None, None, None, None, None, None, None)
    return _new_temp(lib().tdgs_cross_attention_temp_bytes, a, grad, q)


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
        temp = _new_temp(lib().tdgs_cross_attention_temp_bytes, a, False, q)
        a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    check(lib().tdgs_cross_attention(stream_ptr(q.device), C.byref(a)))
    return out


def cross_attention_grad_(dq, dk, dv, dout, out, lse, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None,
                          temp=None):
    """The gradients of sum(dout * out) for cross_attention_'s operands (tdgs_cross_attention_grad), from
    its out and lse. dk and dv are summed over the heads, and batches, that share a key."""
    a = _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask, temp)
    _require(lse is not None, "the gradient needs the forward call's lse")
    if temp is None:
        temp = _new_temp(lib().tdgs_cross_attention_temp_bytes, a, True, q)
        a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    g = abi.AttentionGradsC()
    g.dout = _heads(dout, "dout", tuple(q.shape), q)
    g.dq = _heads(dq, "dq", tuple(q.shape), q)
    g.dk = _heads(dk, "dk", tuple(k.shape), q)
    g.dv = _heads(dv, "dv", tuple(k.shape), q)
    check(lib().tdgs_cross_attention_grad(stream_ptr(q.device), C.byref(a), C.byref(g)))
    return dq, dk, dv


# ------------------------------------------------------------------------------------
# Group norm with an activation
# ------------------------------------------------------------------------------------

def _pixels(t, name, like):
    """The tdgs_pixels of a (n, .., channels) tensor whose middle dimensions are evenly strided."""
    _tensor(t, name, like)
    _require(t.dtype == like.dtype, f"{name} is {t.dtype}, not {like.dtype}")
    _require(t.shape == like.shape, f"{name} has shape {tuple(t.shape)}, not {tuple(like.shape)}")
    s, n = t.stride(), t.shape
    _require(s[-1] == 1 or n[-1] <= 1, f"the channels of {name} must be contiguous")
    step, count = 0, 1
    for i in range(t.dim() - 2, 0, -1):
        if n[i] > 1:
            _require(count == 1 or s[i] == step * count, f"the pixels of {name} must be evenly strided")
            if count == 1:
                step = s[i]
            count *= n[i]
    return abi.PixelsC(t.data_ptr(), s[0], step if count > 1 else n[-1])


def _norm(x, out, groups, weight, bias, eps, activation, stats, temp):
    _tensor(x, "x", x)
    _require(x.dtype in DTYPES, f"x is {x.dtype}: float32, bfloat16 and float16 are supported")
    _require(x.dim() >= 2, "x must be (n, .., channels)")
    _require(activation in ACTIVATIONS, f"activation {activation!r} is none of {', '.join(ACTIVATIONS)}")
    a = abi.NormC()
    n, c = x.shape[0], x.shape[-1]
    a.dtype = a.param_dtype = DTYPES[x.dtype]
    a.n, a.channels, a.groups, a.activation, a.eps = n, c, groups, ACTIVATIONS[activation], eps
    a.pixels = x.numel() // (n * c) if n * c else 0
    a.x = _pixels(x, "x", x)
    if out is not None:
        a.out = _pixels(out, "out", x)
    params = [p for p in (weight, bias) if p is not None]
    for p in params:
        _param(p, "weight and bias", x, params[0].dtype)
    if params:
        a.param_dtype = DTYPES[params[0].dtype]
    a.weight, a.bias = dptr(weight), dptr(bias)
    if stats is not None:
        _tensor(stats, "stats", x)
        _require(stats.dtype == torch.float32 and tuple(stats.shape) == (n, groups, 2) and stats.is_contiguous(),
                 f"stats must be contiguous float32, ({n}, {groups}, 2)")
        a.stats = stats.data_ptr()
    if temp is not None:
        _temp(temp, x)
        a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    return a


def _param(p, name, x, dtype):
    _tensor(p, name, x)
    _require(p.dtype == dtype and dtype in (torch.float32, x.dtype),
             f"{name} must be of one type, float32 or {x.dtype}")
    _require(tuple(p.shape) == (x.shape[-1],) and p.is_contiguous(), f"{name} must be {x.shape[-1]} contiguous values")


def group_norm_temp(x, groups, grad=False):
    """Scratch for group_norm_ (with grad also group_norm_grad_) on images of this size."""
    a = _norm(x, None, groups, None, None, 0.0, "identity", None, None)
    return _new_temp(lib().tdgs_group_norm_temp_bytes, a, grad, x)


def group_norm_(out, x, groups, weight=None, bias=None, *, eps=1e-5, activation="silu", stats=None, temp=None):
    """out = act(group norm of x * weight + bias), channels last (tdgs_group_norm).

    x and out are (n, .., channels): the dimensions between are the pixels, evenly strided, the
    channels contiguous; (width, height, channels) images as they are rendered, with a leading dimension. Mean and
    variance are taken per image and group of channels / groups neighbouring channels. weight and bias are
    float32 or of x's type; activation is identity, silu, gelu or relu. stats (n, groups, 2; float32),
    where given, receives mean and 1 / deviation, which the gradient needs. out may be x."""
    a = _norm(x, out, groups, weight, bias, eps, activation, stats, temp)
    if temp is None:
        temp = _new_temp(lib().tdgs_group_norm_temp_bytes, a, False, x)
        a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    check(lib().tdgs_group_norm(stream_ptr(x.device), C.byref(a)))
    return out


def group_norm_grad_(dx, dweight, dbias, dout, x, stats, groups, weight=None, bias=None, *, activation="silu",
                     temp=None):
    """The gradients of sum(dout * out) for group_norm_'s operands (tdgs_group_norm_grad), from its stats.
    dweight and dbias (of weight's and bias's type, float32 without them) may be None; dx may be dout."""
    _require(stats is not None, "the gradient needs the forward call's stats")
    a = _norm(x, None, groups, weight, bias, 0.0, activation, stats, temp)
    param = next((p.dtype for p in (weight, bias) if p is not None), torch.float32)
    a.param_dtype = DTYPES[param]
    g = abi.NormGradsC(_pixels(dout, "dout", x), _pixels(dx, "dx", x))
    for p, name in ((dweight, "dweight"), (dbias, "dbias")):
        if p is not None:
            _param(p, name, x, param)
    g.dweight, g.dbias = dptr(dweight), dptr(dbias)
    if temp is None:
        temp = _new_temp(lib().tdgs_group_norm_temp_bytes, a, True, x)
        a.temp, a.temp_bytes = temp.data_ptr(), temp.numel()
    check(lib().tdgs_group_norm_grad(stream_ptr(x.device), C.byref(a), C.byref(g)))
    return dx, dweight, dbias


# ------------------------------------------------------------------------------------
# Embedding
# ------------------------------------------------------------------------------------

def _tokens(tokens, like):
    _tensor(tokens, "tokens", like)
    _require(tokens.dtype in (torch.int32, torch.int64) and tokens.is_contiguous(),
             "tokens must be contiguous int32 or int64")
    return tokens.element_size()


def _rows(t, name, rows, dim, like):
    """(pointer, row stride) of a tensor of `rows` rows of dim contiguous elements."""
    _tensor(t, name, like)
    _require(t.dtype == like.dtype and t.dtype in DTYPES, f"{name} is {t.dtype}: one of float32, bfloat16 and float16")
    _require(t.dim() >= 2 and t.shape[-1] == dim and t.numel() == rows * dim,
             f"{name} has shape {tuple(t.shape)}, not {rows} rows of {dim}")
    if t.dim() > 2:
        _require(t.is_contiguous(), f"{name} must be contiguous, or two-dimensional")
        return t.data_ptr(), dim
    _require(t.stride(1) == 1 or dim <= 1, f"the rows of {name} must be contiguous")
    return t.data_ptr(), t.stride(0) if rows > 1 else dim


def embedding_lookup_(out, table, tokens, *, scale=1.0, ctx=None):
    """out[i] = scale table[tokens[i]] (tdgs_embedding_lookup). table is (vocab, dim), tokens int32 or int64
    of any shape, out their shape with dim behind. A token outside the table gives a row of zeros and an
    error at the next ctx_check of the context (by default the device's)."""
    size = _tokens(tokens, table)
    _require(table.dim() == 2, "table must be (vocab, dim)")
    vocab, dim = table.shape
    t, ts = _rows(table, "table", vocab, dim, table)
    o, os = _rows(out, "out", tokens.numel(), dim, table)
    check(lib().tdgs_embedding_lookup(_handle(ctx, table.device.index), stream_ptr(table.device), DTYPES[table.dtype], t,
                                      ts, vocab, dim, tokens.data_ptr(), size, tokens.numel(), scale, o, os))
    return out


def embedding_temp(table, tokens):
    """Scratch for embedding_grad_ with a table and tokens of these sizes."""
    n = lib().tdgs_embedding_grad_temp_bytes(tokens.numel(), table.shape[0], table.shape[1])
    return torch.empty(max(n, 1), dtype=torch.uint8, device=table.device)


def embedding_grad_(dtable, dout, tokens, *, scale=1.0, padding=None, temp=None, ctx=None):
    """dtable[v] = scale times the sum of the dout rows whose token is v, in 32 bits and in the tokens'
    order (tdgs_embedding_grad); every row is written. The token `padding` gives no gradient."""
    size = _tokens(tokens, dtable)
    _require(dtable.dim() == 2, "dtable must be (vocab, dim)")
    vocab, dim = dtable.shape
    t, ts = _rows(dtable, "dtable", vocab, dim, dtable)
    d, ds = _rows(dout, "dout", tokens.numel(), dim, dtable)
    if temp is None:
        temp = embedding_temp(dtable, tokens)
    _temp(temp, dtable)
    check(lib().tdgs_embedding_grad(_handle(ctx, dtable.device.index), stream_ptr(dtable.device), DTYPES[dtable.dtype], d,
                                    ds, tokens.data_ptr(), size, tokens.numel(), -1 if padding is None else padding,
                                    scale, t, ts, vocab, dim, temp.data_ptr(), temp.numel()))
    return dtable
