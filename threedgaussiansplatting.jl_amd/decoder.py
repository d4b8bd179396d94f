"""Operators of a learned decoder of rendered images over libtdgs.so: cross attention to an
encoder's states, group norm with an activation (channels last) and embedding lookup, each with
its gradients.

What a network that turns rendered features into images needs besides matrix products (an
appearance model of a photo collection, a refiner, a codebook of Gaussian attributes). The reference has no counterpart. Tensors are
float32, bfloat16 or float16 on the GPU; outputs and gradients are written into the tensors given,
on the current stream, without synchronisation. temp is scratch of the size its function's
*_temp() gives: with None a call allocates its own. cross_attention, group_norm and embedding are the
same operators as functions that torch can differentiate.
"""
from __future__ import annotations

import ctypes as C
import functools
import struct

import torch

from . import abi
from .core import _handle, check, dptr, lib

DTYPES = {torch.float32: abi.TDGS_F32, torch.bfloat16: abi.TDGS_BF16, torch.float16: abi.TDGS_F16}

ACTIVATIONS = {"identity": abi.TDGS_ACT_IDENTITY, "silu": abi.TDGS_ACT_SILU, "gelu": abi.TDGS_ACT_GELU,
               "relu": abi.TDGS_ACT_RELU}


# tdgs_attention, tdgs_attention_grads, tdgs_norm and tdgs_norm_grads (abi.AttentionC, ..) field by
# field: packing one takes a fifth of the time that filling the ctypes structure takes, which is most of
# what a call on a few queries costs.
_ATTENTION = struct.Struct("@8ifi" + 4 * "Pqqq" + "PPqPPN")
_ATTENTION_GRADS = struct.Struct("@" + 4 * "Pqqq")
_NORM = struct.Struct("@6ifiq" + 2 * "Pqq" + "PPPPN")
_NORM_GRADS = struct.Struct("@" + 2 * "Pqq" + "PP")
assert (_ATTENTION.size, _ATTENTION_GRADS.size, _NORM.size, _NORM_GRADS.size) == tuple(
    C.sizeof(t) for t in (abi.AttentionC, abi.AttentionGradsC, abi.NormC, abi.NormGradsC))


def _call(f, t, args, ctx=()):
    """f(*ctx, stream, *args) on t's device and its current stream: kernels are launched on the current device, whatever
    device a stream belongs to."""
    device = t.get_device()
    stream = torch._C._cuda_getCurrentRawStream(device)
    if device == torch._C._cuda_getDevice():
        check(f(*ctx, stream, *args))
    else:
        with torch.cuda.device(device):
            check(f(*ctx, stream, *args))


def _check_tensor(t, name, like):
    """Raises for anything but a tensor on like's device, which must be a GPU."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{name} must be a tensor on the GPU")
    if t.get_device() != like.get_device():
        raise ValueError(f"{name} is on {t.device}, not on {like.device}")


def _new_temp(size, packed, grad, like):
    return torch.empty(max(size(packed, int(grad)), 1), dtype=torch.uint8, device=like.device)


def _temp(temp, like):
    """(pointer, bytes) of the scratch."""
    _check_tensor(temp, "temp", like)
    if temp.dtype is not torch.uint8 or not temp.is_contiguous():
        raise ValueError("temp must be contiguous uint8")
    return temp.data_ptr(), temp.numel()


# ------------------------------------------------------------------------------------
# Cross attention
# ------------------------------------------------------------------------------------

def _heads(t, name, shape, like):
    """The fields of the tdgs_heads of t."""
    _check_tensor(t, name, like)
    if t.dtype is not like.dtype:
        raise ValueError(f"{name} is {t.dtype}, not {like.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    b, l, h, d = t.stride()
    if d != 1 and shape[3] > 1 and t.numel():
        raise ValueError(f"the last dimension of {name} must be contiguous")
    return t.data_ptr(), b, l, h


_NO_HEADS = (0, 0, 0, 0)


def _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask):
    """The fields of the tdgs_attention of these tensors, without the scratch (v and out None: sizes only)."""
    _check_tensor(q, "q", q)
    dtype = DTYPES.get(q.dtype)
    if dtype is None:
        raise ValueError(f"q is {q.dtype}: float32, bfloat16 and float16 are supported")
    if q.dim() != 4 or not isinstance(k, torch.Tensor) or k.dim() != 4:
        raise ValueError("q and k must be (batch, length, heads, head_dim)")
    shape, kv_shape = q.shape, k.shape
    b, lq, h, d = shape
    kb, lk, hk, kd = kv_shape
    if kd != d:
        raise ValueError(f"k has head dimension {kd}, not {d}")
    fields = (dtype, b, kb, lq, lk, h, hk, d, d ** -0.5 if scale is None and d else scale or 0.0, 0,
              *_heads(q, "q", shape, q), *_heads(k, "k", kv_shape, q))
    if v is None:
        return (*fields, *_NO_HEADS, *_NO_HEADS, 0, 0, 0, 0)
    lengths = mask = mask_stride = sums = 0
    if kv_lengths is not None:
        _check_tensor(kv_lengths, "kv_lengths", q)
        if kv_lengths.dtype is not torch.int32 or kv_lengths.shape != (kb,) or not kv_lengths.is_contiguous():
            raise ValueError(f"kv_lengths must be {kb} contiguous int32 values")
        lengths = kv_lengths.data_ptr()
    if kv_mask is not None:
        _check_tensor(kv_mask, "kv_mask", q)
        if (kv_mask.dtype not in (torch.bool, torch.uint8) or kv_mask.shape != (kb, lk)
                or (kv_mask.stride(1) != 1 and lk > 1)):
            raise ValueError(f"kv_mask must be bool or uint8, ({kb}, {lk}), its rows contiguous")
        mask, mask_stride = kv_mask.data_ptr(), kv_mask.stride(0)
    if lse is not None:
        _check_tensor(lse, "lse", q)
        if lse.dtype is not torch.float32 or lse.shape != (b, h, lq) or not lse.is_contiguous():
            raise ValueError(f"lse must be contiguous float32, ({b}, {h}, {lq})")
        sums = lse.data_ptr()
    return (*fields, *_heads(v, "v", kv_shape, q), *_heads(out, "out", shape, q), lengths, mask, mask_stride, sums)


def cross_attention_temp(q, k, grad=False):
    """Scratch for cross_attention_ (with grad also cross_attention_grad_) on tensors of these sizes."""
    a = _attention(q, k, None, None, None, None, None, None)
    return _new_temp(lib().tdgs_cross_attention_temp_bytes, _ATTENTION.pack(*a, 0, 0), grad, q)


def cross_attention_(out, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None, lse=None, temp=None):
    """out = softmax(scale q k^T) v over the allowed keys, per head (tdgs_cross_attention).

    q and out are (batch, q_len, heads, head_dim), k and v (kv_batch, kv_len, kv_heads, head_dim):
    kv_batch is batch, or 1 for one encoder's states shared by the batch; heads is a multiple of
    kv_heads, neighbouring heads sharing one. Any strides with the last dimension contiguous, head_dim
    up to 128, scale head_dim ** -0.5 by default. kv_lengths (kv_batch int32) allows each batch's first
    keys, kv_mask (kv_batch, kv_len; bool or uint8) single ones; k and v may hold anything where a key is not
    allowed. A query without allowed keys gets zeros. lse (batch, heads, q_len; float32), where given,
    receives the logarithm of each softmax's sum, which the gradient needs.

    With 16-bit types the weights are rounded to the type before their product with v where out has more than
    65536 elements, and keep twice its bits otherwise, so that a query's result may differ by 1.4 of its own
    rounding between a small call and a large one (tdgs_attention says it for the gradients)."""
    a = _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask)
    if temp is None:
        temp = cross_attention_temp(q, k)
    _call(lib().tdgs_cross_attention, q, (_ATTENTION.pack(*a, *_temp(temp, q)),))
    return out


def cross_attention_grad_(dq, dk, dv, dout, out, lse, q, k, v, *, scale=None, kv_lengths=None, kv_mask=None,
                          temp=None):
    """The gradients of sum(dout * out) for cross_attention_'s operands (tdgs_cross_attention_grad), from
    its out and lse. dk and dv are summed over the heads, and batches, that share a key; both may be None."""
    if lse is None:
        raise ValueError("the gradient needs the forward call's lse")
    a = _attention(q, k, v, out, lse, scale, kv_lengths, kv_mask)
    keys = _NO_HEADS * 2 if dk is None and dv is None else (*_heads(dk, "dk", k.shape, q), *_heads(dv, "dv", k.shape, q))
    g = (*_heads(dout, "dout", q.shape, q), *_heads(dq, "dq", q.shape, q), *keys)
    if temp is None:
        temp = cross_attention_temp(q, k, grad=True)
    _call(lib().tdgs_cross_attention_grad, q, (_ATTENTION.pack(*a, *_temp(temp, q)), _ATTENTION_GRADS.pack(*g)))
    return dq, dk, dv


# ------------------------------------------------------------------------------------
# Group norm with an activation
# ------------------------------------------------------------------------------------

def _pixel_step(s, n):
    """The stride between the pixels of a (n, .., channels) tensor of strides s and shape n, None where they are not evenly
    strided."""
    step, count = n[-1], 1
    for i in range(len(n) - 2, 0, -1):
        if n[i] > 1:
            if count == 1:
                step = s[i]
            elif s[i] != step * count:
                return None
            count *= n[i]
    return step


def _pixels(t, name, like):
    """The fields of the tdgs_pixels of a (n, .., channels) tensor whose middle dimensions are evenly strided."""
    _check_tensor(t, name, like)
    if t.dtype is not like.dtype:
        raise ValueError(f"{name} is {t.dtype}, not {like.dtype}")
    s, n = t.stride(), t.shape
    if n != like.shape:
        raise ValueError(f"{name} has shape {tuple(n)}, not {tuple(like.shape)}")
    if s[-1] != 1 and n[-1] > 1 and t.numel():
        raise ValueError(f"the channels of {name} must be contiguous")
    step = s[1] if len(n) == 3 else _pixel_step(s, n)
    if step is None:
        if t.numel():
            raise ValueError(f"the pixels of {name} must be evenly strided")
        step = n[-1]
    return t.data_ptr(), s[0], step


_NO_PIXELS = (0, 0, 0)


def _param(p, name, x, dtype):
    _check_tensor(p, name, x)
    if p.dtype is not dtype or (dtype is not torch.float32 and dtype is not x.dtype):
        raise ValueError(f"{name} must be of one type, float32 or {x.dtype}")
    if p.shape != (x.shape[-1],) or not p.is_contiguous():
        raise ValueError(f"{name} must be {x.shape[-1]} contiguous values")


def _norm(x, out, groups, weight, bias, eps, activation, stats):
    """The fields of the tdgs_norm of these tensors, without the scratch (out None: not written)."""
    _check_tensor(x, "x", x)
    dtype = DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"x is {x.dtype}: float32, bfloat16 and float16 are supported")
    if x.dim() < 2:
        raise ValueError("x must be (n, .., channels)")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r} is none of {', '.join(ACTIVATIONS)}")
    n, c = x.shape[0], x.shape[-1]
    first = weight if weight is not None else bias
    if first is not None:
        if weight is not None:
            _param(weight, "weight", x, first.dtype)
        if bias is not None:
            _param(bias, "bias", x, first.dtype)
    if stats is not None:
        _check_tensor(stats, "stats", x)
        if stats.dtype is not torch.float32 or stats.shape != (n, groups, 2) or not stats.is_contiguous():
            raise ValueError(f"stats must be contiguous float32, ({n}, {groups}, 2)")
    return (dtype, abi.TDGS_F32 if first is None else DTYPES[first.dtype], n, c, groups, act, eps, 0,
            x.numel() // (n * c) if n * c else 0, *_pixels(x, "x", x),
            *(_NO_PIXELS if out is None else _pixels(out, "out", x)), dptr(weight) or 0, dptr(bias) or 0,
            dptr(stats) or 0)


def group_norm_temp(x, groups, grad=False):
    """Scratch for group_norm_ (with grad also group_norm_grad_) on images of this size."""
    a = _norm(x, None, groups, None, None, 0.0, "identity", None)
    return _new_temp(lib().tdgs_group_norm_temp_bytes, _NORM.pack(*a, 0, 0), grad, x)


def group_norm_(out, x, groups, weight=None, bias=None, *, eps=1e-5, activation="silu", stats=None, temp=None):
    """out = act(group norm of x * weight + bias), channels last (tdgs_group_norm).

    x and out are (n, .., channels): the dimensions between are the pixels, evenly strided, the
    channels contiguous; (width, height, channels) images as they are rendered, with a leading dimension. Mean and
    variance are taken per image and group of channels / groups neighbouring channels. weight and bias are
    float32 or of x's type; activation is identity, silu, gelu or relu. stats (n, groups, 2; float32),
    where given, receives mean and 1 / deviation, which the gradient needs. out may be x."""
    a = _norm(x, out, groups, weight, bias, eps, activation, stats)
    if temp is None:
        temp = group_norm_temp(x, groups)
    _call(lib().tdgs_group_norm, x, (_NORM.pack(*a, *_temp(temp, x)),))
    return out


def group_norm_grad_(dx, dweight, dbias, dout, x, stats, groups, weight=None, bias=None, *, activation="silu",
                     temp=None):
    """The gradients of sum(dout * out) for group_norm_'s operands (tdgs_group_norm_grad), from its stats.
    dweight and dbias (of weight's and bias's type, float32 without them) may be None; dx may be dout."""
    if stats is None:
        raise ValueError("the gradient needs the forward call's stats")
    a = _norm(x, None, groups, weight, bias, 0.0, activation, stats)
    first = weight if weight is not None else bias
    for p, name in ((dweight, "dweight"), (dbias, "dbias")):
        if p is not None:
            _param(p, name, x, torch.float32 if first is None else first.dtype)
    g = (*_pixels(dout, "dout", x), *_pixels(dx, "dx", x), dptr(dweight) or 0, dptr(dbias) or 0)
    if temp is None:
        temp = group_norm_temp(x, groups, grad=True)
    _call(lib().tdgs_group_norm_grad, x, (_NORM.pack(*a, *_temp(temp, x)), _NORM_GRADS.pack(*g)))
    return dx, dweight, dbias


# ------------------------------------------------------------------------------------
# Embedding
# ------------------------------------------------------------------------------------

def _tokens(tokens, like):
    """The bytes of a token."""
    _check_tensor(tokens, "tokens", like)
    if (tokens.dtype is not torch.int32 and tokens.dtype is not torch.int64) or not tokens.is_contiguous():
        raise ValueError("tokens must be contiguous int32 or int64")
    return tokens.element_size()


def _table(t, name):
    """(vocab, dim, pointer, row stride)"""
    _check_tensor(t, name, t)
    if t.dtype not in DTYPES:
        raise ValueError(f"{name} is {t.dtype}: float32, bfloat16 and float16 are supported")
    if t.dim() != 2:
        raise ValueError(f"{name} must be (vocab, dim)")
    return (*t.shape, *_rows(t, name, *t.shape, t))


def _rows(t, name, rows, dim, like):
    """(pointer, row stride) of a tensor of `rows` rows of dim contiguous elements."""
    _check_tensor(t, name, like)
    if t.dtype is not like.dtype:
        raise ValueError(f"{name} is {t.dtype}, not {like.dtype}")
    if t.dim() < 2 or t.shape[-1] != dim or t.numel() != rows * dim:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {rows} rows of {dim}")
    if t.dim() > 2:
        if not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous, or two-dimensional")
        return t.data_ptr(), dim
    row, element = t.stride()
    if element != 1 and dim > 1 and rows:
        raise ValueError(f"the rows of {name} must be contiguous")
    return t.data_ptr(), row if rows > 1 else dim


def _check_padding(padding, vocab):
    # (counted from the end elsewhere: neither that nor "none" can be told from -1)
    if padding is not None and not 0 <= padding < vocab:
        raise ValueError(f"padding {padding} is no row of a table of {vocab}")


def embedding_lookup_(out, table, tokens, *, scale=1.0, ctx=None):
    """out[i] = scale table[tokens[i]] (tdgs_embedding_lookup). table is (vocab, dim), tokens int32 or int64
    of any shape, out their shape with dim behind. A token outside the table gives a row of zeros and an
    error at the next ctx_check of the context (by default the device's)."""
    vocab, dim, t, ts = _table(table, "table")
    size, n = _tokens(tokens, table), tokens.numel()
    o, os = _rows(out, "out", n, dim, table)
    _call(lib().tdgs_embedding_lookup, table,
          (DTYPES[table.dtype], t, ts, vocab, dim, tokens.data_ptr(), size, n, scale, o, os),
          (_handle(ctx, table.get_device()),))
    return out


def embedding_temp(table, tokens):
    """Scratch for embedding_grad_ with a table and tokens of these sizes."""
    n = lib().tdgs_embedding_grad_temp_bytes(tokens.numel(), table.shape[0], table.shape[1])
    return torch.empty(max(n, 1), dtype=torch.uint8, device=table.device)


def embedding_grad_(dtable, dout, tokens, *, scale=1.0, padding=None, temp=None, ctx=None):
    """dtable[v] = scale times the sum of the dout rows whose token is v, in 32 bits and in the tokens'
    order (tdgs_embedding_grad); every row is written. The token `padding`, a row of the table, gives no
    gradient (None: every token does)."""
    vocab, dim, t, ts = _table(dtable, "dtable")
    _check_padding(padding, vocab)
    size, n = _tokens(tokens, dtable), tokens.numel()
    d, ds = _rows(dout, "dout", n, dim, dtable)
    if temp is None:
        temp = embedding_temp(dtable, tokens)
    _call(lib().tdgs_embedding_grad, dtable,
          (DTYPES[dtable.dtype], d, ds, tokens.data_ptr(), size, n, -1 if padding is None else padding, scale, t, ts, vocab,
           dim, *_temp(temp, dtable)), (_handle(ctx, dtable.get_device()),))
    return dtable


# ------------------------------------------------------------------------------------
# As differentiable functions: once, their gradients have no kernels of their own
# ------------------------------------------------------------------------------------

def _rows_contiguous(t):
    """t, or a copy where its last dimension is not contiguous."""
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def _contiguous(t):
    return None if t is None else t.contiguous()


class _Refused(torch.autograd.Function):
    """The first n tensors as they are, as a function of the others that cannot be differentiated."""

    @staticmethod
    def forward(ctx, n, *tensors):
        return tensors[:n]

    @staticmethod
    def backward(ctx, *douts):
        raise RuntimeError("the gradients of the decoder operators cannot be differentiated again")


def _once(backward):
    """backward, whose gradients come from kernels, for a function that can be differentiated once: where torch builds
    a graph of the gradients, they hang on everything that they were made from, so that a second derivative
    raises. (once_differentiable refuses only what comes through dout, and takes them for constants otherwise.)"""
    @functools.wraps(backward)
    def wrapped(ctx, dout):
        with torch.no_grad():
            grads = backward(ctx, dout)
        made_from = [t for t in (dout, *ctx.saved_tensors) if t is not None and t.requires_grad] \
            if torch.is_grad_enabled() else ()
        if made_from:
            given = [g for g in grads if g is not None]
            refused = iter(_Refused.apply(len(given), *given, *made_from))
            grads = tuple(None if g is None else next(refused) for g in grads)
        return grads
    return wrapped


class _CrossAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, scale, kv_lengths, kv_mask):
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
        cross_attention_(out, q, k, v, scale=scale, kv_lengths=kv_lengths, kv_mask=kv_mask, lse=lse)
        ctx.save_for_backward(q, k, v, out, lse, kv_lengths, kv_mask)
        ctx.scale = scale
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        q, k, v, out, lse, kv_lengths, kv_mask = ctx.saved_tensors
        # (dq also leaves what dk and dv are computed from)
        wanted = (True, any(ctx.needs_input_grad[1:3]), any(ctx.needs_input_grad[1:3]))
        dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) if w else None
                      for t, w in zip((q, k, v), wanted))
        cross_attention_grad_(dq, dk, dv, dout.contiguous(), out, lse, q, k, v, scale=ctx.scale, kv_lengths=kv_lengths,
                              kv_mask=kv_mask)
        return dq, dk, dv, None, None, None


def cross_attention(q, k, v, *, scale=None, kv_lengths=None, kv_mask=None):
    """cross_attention_ as a differentiable function of q, k and v, all tensors of any strides."""
    return _CrossAttention.apply(_rows_contiguous(q), _rows_contiguous(k), _rows_contiguous(v), scale,
                                 _contiguous(kv_lengths), None if kv_mask is None else _rows_contiguous(kv_mask))


class _GroupNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, groups, eps, activation):
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        stats = torch.empty((x.shape[0], groups, 2), dtype=torch.float32, device=x.device)
        group_norm_(out, x, groups, weight, bias, eps=eps, activation=activation, stats=stats)
        ctx.save_for_backward(x, weight, bias, stats)
        ctx.groups, ctx.activation = groups, activation
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        x, weight, bias, stats = ctx.saved_tensors
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dweight, dbias = (torch.empty_like(p) if w else None for p, w in zip((weight, bias), ctx.needs_input_grad[1:3]))
        group_norm_grad_(dx, dweight, dbias, dout.contiguous(), x, stats, ctx.groups, weight, bias,
                         activation=ctx.activation)
        return dx, dweight, dbias, None, None, None


def group_norm(x, groups, weight=None, bias=None, *, eps=1e-5, activation="silu"):
    """group_norm_ as a differentiable function of x, weight and bias, all of any strides."""
    x = _rows_contiguous(x)
    if _pixel_step(x.stride(), x.shape) is None:
        x = x.contiguous()
    return _GroupNorm.apply(x, _contiguous(weight), _contiguous(bias), groups, eps, activation)


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, table, tokens, scale, padding):
        out = torch.empty((*tokens.shape, table.shape[1]), dtype=table.dtype, device=table.device)
        embedding_lookup_(out if out.dim() > 1 else out[None], table, tokens, scale=scale)
        ctx.save_for_backward(tokens)
        ctx.shape, ctx.scale, ctx.padding = table.shape, scale, padding
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        tokens, = ctx.saved_tensors
        dtable = torch.empty(ctx.shape, dtype=dout.dtype, device=dout.device)
        embedding_grad_(dtable, dout.reshape(-1, ctx.shape[1]).contiguous(), tokens, scale=ctx.scale, padding=ctx.padding)
        return dtable, None, None, None


def embedding(table, tokens, *, scale=1.0, padding=None):
    """embedding_lookup_ as a differentiable function of the table, it and the tokens of any strides; `padding` as in
    embedding_grad_."""
    _check_padding(padding, table.shape[0])
    return _Embedding.apply(_rows_contiguous(table), tokens.contiguous(), scale, padding)
