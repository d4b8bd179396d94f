"""Operators of a learned decoder of rendered images over libtdgs.so: cross attention to an
encoder's states, group norm with an activation (channels last), embedding lookup, linear layers with
bias, activation and residual, norms of queries and keys for each head with their rotation by position, and
dropout, each with its gradients.

What a network that turns rendered features into images needs (an appearance model of a photo collection, a
refiner, a codebook of Gaussian attributes). The reference has no counterpart. Tensors are
float32, bfloat16 or float16 on the GPU; outputs and gradients are written into the tensors given,
on the current stream, without synchronisation. temp is scratch of the size its function's
*_temp() gives: with None a call allocates its own. cross_attention, group_norm, embedding, linear, head_norm, rotate
and dropout are the same operators as functions that torch can differentiate.
"""
from __future__ import annotations

import ctypes as C
import functools
import math
import struct

import torch

from . import abi
from .core import _dev, _handle, check, dptr, lib

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
_LINEAR = struct.Struct("@2iq4i" + 5 * "Pq" + "PPN")
_LINEAR_GRADS = struct.Struct("@" + 3 * "Pq" + "P2i")
_HEAD_NORM = struct.Struct("@8if3i4i2iPPq" + 4 * "Pqqq" + "PPPN")
_HEAD_NORM_GRADS = struct.Struct("@" + 4 * "Pqqq" + "PP")
_DROPOUT = struct.Struct("@2i2qd2QP" + 3 * "Pq")
assert (_ATTENTION.size, _ATTENTION_GRADS.size, _NORM.size, _NORM_GRADS.size, _LINEAR.size, _LINEAR_GRADS.size,
        _HEAD_NORM.size, _HEAD_NORM_GRADS.size, _DROPOUT.size) == tuple(
    C.sizeof(t) for t in (abi.AttentionC, abi.AttentionGradsC, abi.NormC, abi.NormGradsC, abi.LinearC, abi.LinearGradsC,
                          abi.HeadNormC, abi.HeadNormGradsC, abi.DropoutC))


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
# Linear layers with bias, activation and residual
# ------------------------------------------------------------------------------------

def _even_rows(t):
    """The stride between the rows of a (.., n) tensor, None where they are not evenly strided."""
    n, s = t.shape, t.stride()
    if len(n) == 2:
        return s[0]
    step, count = n[-1], 1
    for i in range(len(n) - 2, -1, -1):
        if n[i] > 1:
            if count == 1:
                step = s[i]
            elif s[i] != step * count:
                return None
            count *= n[i]
    return step


def _matrix(t, name, shape, like, device):
    """(pointer, row stride) of a tensor of this shape, like's type and device, with evenly strided rows of contiguous
    elements."""
    # what is usual is looked at once: most of what a call on a few rows costs is this
    if isinstance(t, torch.Tensor) and len(shape) == 2 and t.shape == shape and t.dtype is like.dtype \
            and t.get_device() == device:
        row, element = t.stride()
        if element == 1 or shape[1] <= 1 or not t.numel():
            return t.data_ptr(), row
    _check_tensor(t, name, like)
    if t.dtype is not like.dtype:
        raise ValueError(f"{name} is {t.dtype}, not {like.dtype}")
    if t.shape != shape:
        raise ValueError(f"{name} has shape {tuple(t.shape)}, not {tuple(shape)}")
    cols = shape[-1]
    if cols > 1 and t.stride(-1) != 1 and t.numel():
        raise ValueError(f"the rows of {name} must be contiguous")
    step = _even_rows(t)
    if step is None:
        if t.numel():
            raise ValueError(f"the rows of {name} must be evenly strided")
        step = cols
    return t.data_ptr(), step


_NO_ROWS = (0, 0)


def _weight(w, name, like, shape=None):
    """(layout, pointer, row stride) of an (in, out) matrix that lies either way round."""
    if not isinstance(w, torch.Tensor) or w.get_device() != like.get_device():
        _check_tensor(w, name, like)
    if w.dtype is not like.dtype:
        raise ValueError(f"{name} is {w.dtype}, not {like.dtype}")
    if w.dim() != 2 or (shape is not None and w.shape != shape):
        raise ValueError(f"{name} has shape {tuple(w.shape)}, not {'(in, out)' if shape is None else tuple(shape)}")
    (rows, cols), (row, element) = w.shape, w.stride()
    if element == 1 or cols == 1:
        # (one column of a transposed matrix: rows of one element, or one row of them, whichever is contiguous)
        if cols > 1 or row != 1:
            return abi.TDGS_WEIGHT_IN_OUT, w.data_ptr(), row
    if row == 1 or rows == 1:
        return abi.TDGS_WEIGHT_OUT_IN, w.data_ptr(), element
    raise ValueError(f"the rows or the columns of {name} must be contiguous")


def _linear(x, weight, bias, activation, pre):
    """The fields of the tdgs_linear of these tensors up to out, those from pre to bias, the outputs' shape and the device."""
    if not isinstance(x, torch.Tensor) or not x.is_cuda:
        _check_tensor(x, "x", x)
    dtype = DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"x is {x.dtype}: float32, bfloat16 and float16 are supported")
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"activation {activation!r} is none of {', '.join(ACTIVATIONS)}")
    shape = x.shape
    if len(shape) < 1:
        raise ValueError("x must be (.., in)")
    device = x.get_device()
    layout, w, ws = _weight(weight, "weight", x)
    features, outputs = weight.shape
    if shape[-1] != features:
        raise ValueError(f"x has {shape[-1]} features, the weight {features}")
    xp, xs = _matrix(x, "x", shape, x, device)
    shape = (*shape[:-1], outputs)
    b = 0
    if bias is not None:
        if bias.dtype is not x.dtype or bias.shape != (outputs,) or bias.get_device() != device or not bias.is_contiguous():
            _check_vector(bias, "bias", outputs, x)
        b = bias.data_ptr()
    rows = x.numel() // features if features else 0
    return ((dtype, act, rows, features, outputs, layout, 0, xp, xs, w, ws),
            (*(_NO_ROWS if pre is None else _matrix(pre, "pre", shape, x, device)), b), shape, device)


def _check_vector(p, name, n, like):
    _check_tensor(p, name, like)
    if p.dtype is not like.dtype or p.shape != (n,) or not p.is_contiguous():
        raise ValueError(f"{name} must be {n} contiguous values of {like.dtype}")


def linear_temp(x, weight, grad=False):
    """Scratch for linear_ (with grad also linear_grad_, whatever its activation) on tensors of these sizes."""
    a, b, _, _ = _linear(x, weight, None, "silu", None)
    return _new_temp(lib().tdgs_linear_temp_bytes, _LINEAR.pack(*a, *_NO_ROWS, *_NO_ROWS, *b, 0, 0), grad, x)


def linear_(out, x, weight, bias=None, *, residual=None, activation="identity", pre=None, temp=None):
    """out = residual + act(x weight + bias) (tdgs_linear_forward).

    x is (.., in), weight (in, out), the others (.., out), all of one type, their rows contiguous and evenly strided; of the
    weight the rows or the columns are (the transpose of an (out, in) matrix is taken as it is). activation is identity,
    silu, gelu or relu. pre, where given, receives x weight + bias, which the gradient needs unless the activation is the
    identity. residual may be out; out and pre overlap nothing else."""
    a, b, shape, device = _linear(x, weight, bias, activation, pre)
    o = _matrix(out, "out", shape, x, device)
    r = _NO_ROWS if residual is None else _matrix(residual, "residual", shape, x, device)
    if temp is None:
        temp = _new_temp(lib().tdgs_linear_temp_bytes, _LINEAR.pack(*a, *o, *r, *b, 0, 0), False, x)
    _call(lib().tdgs_linear_forward, x, (_LINEAR.pack(*a, *o, *r, *b, *_temp(temp, x)),))
    return out


def linear_grad_(dx, dweight, dbias, dout, x, weight, *, activation="identity", pre=None, temp=None):
    """The gradients of sum(dout * out) for linear_'s x, weight and bias (tdgs_linear_grad), from its pre; any of them may
    be None. dweight lies either way round, whatever weight does. The residual's gradient is dout.

    With 16-bit types, silu and gelu, dout act'(pre) is rounded to the type for its two matrix products where it has more than
    65536 elements, and keeps twice its bits otherwise (tdgs_linear_grad); dbias is summed before that."""
    if pre is None and activation != "identity":
        raise ValueError("the gradient needs the forward call's pre")
    a, b, shape, device = _linear(x, weight, None, activation, pre)
    outputs = shape[-1]
    d = _matrix(dout, "dout", shape, x, device)
    g = _NO_ROWS if dx is None else _matrix(dx, "dx", x.shape, x, device)
    layout, w, ws = (0, 0, 0) if dweight is None else _weight(dweight, "dweight", x, weight.shape)
    db = 0
    if dbias is not None:
        _check_vector(dbias, "dbias", outputs, x)
        db = dbias.data_ptr()
    if temp is None:
        temp = _new_temp(lib().tdgs_linear_temp_bytes, _LINEAR.pack(*a, *_NO_ROWS, *_NO_ROWS, *b, 0, 0), True, x)
    _call(lib().tdgs_linear_grad, x, (_LINEAR.pack(*a, *_NO_ROWS, *_NO_ROWS, *b, *_temp(temp, x)),
                                      _LINEAR_GRADS.pack(*d, *g, w, ws, db, layout, 0)))
    return dx, dweight, dbias


# ------------------------------------------------------------------------------------
# Norms of queries and keys for each head, and their rotation by position
# ------------------------------------------------------------------------------------

_PAIRS = {"halves": abi.TDGS_PAIRS_HALVES, "interleaved": abi.TDGS_PAIRS_INTERLEAVED}
_POSITIONS = {torch.int32: abi.TDGS_POSITION_I32, torch.int64: abi.TDGS_POSITION_I64,
              torch.float32: abi.TDGS_POSITION_F32}


class Rotary:
    """The rotation of pairs of a head's elements by position on several axes (time, row, column, ..).

    sections holds the pairs of each axis, in order: pair j of an axis of n pairs turns by position * base ** (-j / n)
    radians, or by position * frequencies[pair] where these are given (one per pair of all sections). pairs
    says which elements are a pair: "halves", p and p + sum(sections), or "interleaved", 2 p and 2 p + 1. Elements of a head
    behind the pairs are not rotated."""

    def __init__(self, sections, *, base=10000.0, pairs="halves", frequencies=None, device=0):
        self.sections = tuple(int(s) for s in sections)
        if not 1 <= len(self.sections) <= 4 or min(self.sections) < 1:
            raise ValueError(f"sections {sections} are not one to four axes of one pair or more")
        if pairs not in _PAIRS:
            raise ValueError(f"pairs {pairs!r} are none of {', '.join(_PAIRS)}")
        if not base > 0:
            raise ValueError("the base must be positive")
        self.pairs, self.layout, self.axes = sum(self.sections), pairs, len(self.sections)
        if frequencies is None:
            frequencies = [base ** (-j / n) for n in self.sections for j in range(n)]
        f = torch.as_tensor(frequencies, dtype=torch.float64)
        if f.shape != (self.pairs,):
            raise ValueError(f"{tuple(f.shape)} frequencies of {self.pairs} pairs")
        # (a call asks this tensor for its address: a copy or an unpickled rotation has one of its own)
        self.turns = (f / (2 * math.pi)).to(_dev(device))
        self._fields = (self.pairs, _PAIRS[pairs], self.axes, *self.sections, *(0,) * (4 - self.axes))


def _head_norm(q, k, q_weight, k_weight, norm, eps, rotary, positions, inverse):
    """The fields of the tdgs_head_norm of these tensors up to q, and those of the weights."""
    if not isinstance(q, torch.Tensor) or not q.is_cuda:
        _check_tensor(q, "q", q)
    dtype = DTYPES.get(q.dtype)
    if dtype is None:
        raise ValueError(f"q is {q.dtype}: float32, bfloat16 and float16 are supported")
    if q.dim() != 4:
        raise ValueError("q must be (batch, length, heads, head_dim)")
    b, l, h, d = q.shape
    device = q.get_device()
    hk = 0
    if k is not None:
        if k.dim() != 4 or k.shape != (b, l, k.shape[2], d):
            raise ValueError(f"k has shape {tuple(k.shape)}, not ({b}, {l}, heads, {d})")
        hk = k.shape[2]
    first = q_weight if q_weight is not None else k_weight
    param, wq, wk = abi.TDGS_F32, 0, 0
    if first is not None:
        kind = first.dtype
        param = DTYPES.get(kind)
        if kind is not torch.float32 and kind is not q.dtype:
            raise ValueError(f"q_weight and k_weight must be of one type, float32 or {q.dtype}")
        if q_weight is not None:
            wq = _head_weight(q_weight, "q_weight", kind, d, q, device)
        if k_weight is not None:
            wk = _head_weight(k_weight, "k_weight", kind, d, q, device)
    if rotary is None:
        if positions is not None:
            raise ValueError("positions without a rotary")
        rotation, place = _NO_ROTATION, _NO_PLACE
    else:
        if not isinstance(positions, torch.Tensor) or not device == positions.get_device() == rotary.turns.get_device():
            _check_tensor(rotary.turns, "the rotary", q)
            _check_tensor(positions, "positions", q)
        kind = _POSITIONS.get(positions.dtype)
        if kind is None:
            raise ValueError(f"positions are {positions.dtype}: int32, int64 and float32 are supported")
        n, axes = positions.shape, rotary.axes
        batched = len(n) == 3
        if n != ((b, l, axes) if batched else (l, axes)) or not positions.is_contiguous():
            raise ValueError(f"positions must be contiguous, ({l}, {axes}) or ({b}, {l}, {axes})")
        rotation = rotary._fields
        place = (kind, rotary.turns.data_ptr(), positions.data_ptr(), l * axes if batched else 0)
    return ((dtype, param, b, l, h, hk, d, 1 if norm else 0, eps, *rotation, 1 if inverse else 0, *place), (wq, wk))


_NO_ROTATION, _NO_PLACE = (0,) * 7, (0,) * 4


def _head_weight(w, name, dtype, d, q, device):
    """The pointer of d contiguous values of a type."""
    if w.dtype is not dtype or w.shape != (d,) or w.get_device() != device or not w.is_contiguous():
        _check_tensor(w, name, q)
        raise ValueError(f"{name} must be {d} contiguous values of {dtype}")
    return w.data_ptr()


def _head_view(t, name, shape, like, device):
    """_heads, for which what is usual is looked at once."""
    if isinstance(t, torch.Tensor) and t.dtype is like.dtype and t.shape == shape and t.get_device() == device:
        b, l, h, d = t.stride()
        if d == 1:
            return t.data_ptr(), b, l, h
    return _heads(t, name, shape, like)


def _head_views(names, tensors, like):
    """The tdgs_heads fields of tensors like (q, k): k's may be missing."""
    q, k = like
    device = q.get_device()
    out = _head_view(tensors[0], names[0], q.shape, q, device)
    if k is None:
        if tensors[1] is not None:
            raise ValueError(f"{names[1]} without k")
        return (*out, *_NO_HEADS)
    return (*out, *_head_view(tensors[1], names[1], k.shape, q, device))


def head_norm_(q_out, k_out, q, k=None, q_weight=None, k_weight=None, *, eps=1e-6, rotary=None, positions=None):
    """Each head of q and k divided by the root of its mean square plus eps and multiplied by its weight; with a
    Rotary, rotated by position in the same pass (tdgs_head_norm_forward).

    q and k are (batch, length, heads, head_dim), of any strides with the last dimension contiguous, head_dim up to 256; k (and
    k_out) may be None. weights are head_dim values, float32 or of q's type; None: ones. positions are (length, axes) or
    (batch, length, axes), int32, int64 or float32; their angles are made in 64 bits, and what is left of them
    without whole turns is rounded to 2^-26 of a turn. q_out may be q and k_out k (the same strides too), and they overlap
    nothing else."""
    a, w = _head_norm(q, k, q_weight, k_weight, True, eps, rotary, positions, False)
    x = _head_views(("q", "k"), (q, k), (q, k))
    o = _head_views(("q_out", "k_out"), (q_out, k_out), (q, k))
    _call(lib().tdgs_head_norm_forward, q, (_HEAD_NORM.pack(*a, *x, *o, *w, 0, 0),))
    return q_out, k_out


def head_norm_temp(q, k=None):
    """Scratch for head_norm_grad_ on tensors of these sizes."""
    a, w = _head_norm(q, k, None, None, True, 0.0, None, None, False)
    n = lib().tdgs_head_norm_temp_bytes(_HEAD_NORM.pack(*a, *_NO_HEADS * 4, *w, 0, 0))
    return torch.empty(max(n, 1), dtype=torch.uint8, device=q.device)


def head_norm_grad_(dq, dk, dq_weight, dk_weight, dq_out, dk_out, q, k=None, q_weight=None, k_weight=None, *, eps=1e-6,
                    rotary=None, positions=None, temp=None):
    """The gradients of sum(dq_out * q_out) + sum(dk_out * k_out) for head_norm_'s operands (tdgs_head_norm_grad).
    dq_weight and dk_weight (of the weights' type, float32 without them) may be None; dq may be dq_out and dk dk_out."""
    a, w = _head_norm(q, k, q_weight, k_weight, True, eps, rotary, positions, False)
    x = _head_views(("q", "k"), (q, k), (q, k))
    first = q_weight if q_weight is not None else k_weight
    for p, name in ((dq_weight, "dq_weight"), (dk_weight, "dk_weight")):
        if p is not None:
            _check_tensor(p, name, q)
            dtype = torch.float32 if first is None else first.dtype
            if p.dtype is not dtype or p.shape != (q.shape[3],) or not p.is_contiguous():
                raise ValueError(f"{name} must be {q.shape[3]} contiguous values of {dtype}")
    g = (*_head_views(("dq_out", "dk_out"), (dq_out, dk_out), (q, k)), *_head_views(("dq", "dk"), (dq, dk), (q, k)))
    if temp is None:
        temp = head_norm_temp(q, k)
    _call(lib().tdgs_head_norm_grad, q, (_HEAD_NORM.pack(*a, *x, *_NO_HEADS * 2, *w, *_temp(temp, q)),
                                         _HEAD_NORM_GRADS.pack(*g, dptr(dq_weight) or 0, dptr(dk_weight) or 0)))
    return dq, dk, dq_weight, dk_weight


def rotate_(q_out, k_out, q, k, rotary, positions, *, inverse=False):
    """head_norm_'s rotation alone; the other way round with inverse, which is its gradient."""
    if rotary is None:
        raise ValueError("a rotation needs a Rotary")
    a, w = _head_norm(q, k, None, None, False, 0.0, rotary, positions, inverse)
    x = _head_views(("q", "k"), (q, k), (q, k))
    o = _head_views(("q_out", "k_out"), (q_out, k_out), (q, k))
    _call(lib().tdgs_head_norm_forward, q, (_HEAD_NORM.pack(*a, *x, *o, *w, 0, 0),))
    return q_out, k_out


# ------------------------------------------------------------------------------------
# Dropout
# ------------------------------------------------------------------------------------

def dropout_(out, x, p, seed, *, call=0, residual=None):
    """out = residual + x / (1 - p) where an element is kept, with probability 1 - p, and residual where it is dropped
    (tdgs_dropout_apply).

    Tensors are (.., n), their rows contiguous and evenly strided. Which elements are kept is a function of seed (64 bits), call and an
    element's place among x's, not of strides or type: the same call on dout, without a residual, is the gradient for x.
    call, a count that a program advances with every use, is a whole number, or an int64 tensor of one value on the GPU that
    the kernel reads (a captured call then takes another mask at each replay). out may be x or residual."""
    _check_tensor(x, "x", x)
    dtype = DTYPES.get(x.dtype)
    if dtype is None:
        raise ValueError(f"x is {x.dtype}: float32, bfloat16 and float16 are supported")
    if not 0 <= p <= 1:
        raise ValueError(f"dropout of {p}, which is no probability")
    if x.dim() == 0:
        raise ValueError("x must have a dimension")
    shape, device = x.shape, x.get_device()
    cols = shape[-1]
    number = device_call = 0
    if isinstance(call, torch.Tensor):
        _check_tensor(call, "call", x)
        if call.dtype is not torch.int64 or call.numel() != 1:
            raise ValueError("call must be a whole number or one int64 value")
        device_call = call.data_ptr()
    else:
        number = int(call) & (2 ** 64 - 1)
    r = _NO_ROWS if residual is None else _matrix(residual, "residual", shape, x, device)
    fields = (dtype, 0, x.numel() // cols if cols else 0, cols, p, int(seed) & (2 ** 64 - 1), number, device_call,
              *_matrix(x, "x", shape, x, device), *_matrix(out, "out", shape, x, device), *r)
    _call(lib().tdgs_dropout_apply, x, (_DROPOUT.pack(*fields),))
    return out


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
    def wrapped(ctx, *douts):
        with torch.no_grad():
            grads = backward(ctx, *douts)
        made_from = [t for t in (*douts, *ctx.saved_tensors) if t is not None and t.requires_grad] \
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


def _rows_even(t):
    """t, or a copy where its rows are not contiguous and evenly strided."""
    if t is None:
        return None
    t = _rows_contiguous(t)
    return t if _even_rows(t) is not None else t.contiguous()


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, activation):
        out = torch.empty((*x.shape[:-1], weight.shape[1]), dtype=x.dtype, device=x.device)
        pre = torch.empty_like(out) if activation != "identity" and any(ctx.needs_input_grad[:3]) else None
        linear_(out, x, weight, bias, residual=residual, activation=activation, pre=pre)
        ctx.save_for_backward(x, weight, pre)
        ctx.activation = activation
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        x, weight, pre = ctx.saved_tensors
        wants = ctx.needs_input_grad
        dx = torch.empty(x.shape, dtype=x.dtype, device=x.device) if wants[0] else None
        # (laid out as the weight is)
        dweight = torch.empty_strided(weight.shape, _dense(weight), dtype=x.dtype, device=x.device) if wants[1] else None
        dbias = torch.empty(weight.shape[1:], dtype=x.dtype, device=x.device) if wants[2] else None
        if any(wants[:3]):
            linear_grad_(dx, dweight, dbias, _rows_even(dout), x, weight, activation=ctx.activation, pre=pre)
        return dx, dweight, dbias, dout if wants[3] else None, None


def _dense(weight):
    """The strides of a dense matrix that lies as weight does."""
    rows, cols = weight.shape
    return (cols, 1) if weight.stride(1) == 1 else (1, rows)


def linear(x, weight, bias=None, *, residual=None, activation="identity"):
    """linear_ as a differentiable function of x, weight, bias and residual, all of any strides."""
    if weight.dim() == 2 and weight.stride(0) != 1:
        weight = _rows_contiguous(weight)
    return _Linear.apply(_rows_even(x), weight, _contiguous(bias), _rows_even(residual), activation)


class _HeadNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, eps, rotary, positions):
        outs = [None if x is None else torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k)]
        head_norm_(*outs, q, k, q_weight, k_weight, eps=eps, rotary=rotary, positions=positions)
        ctx.save_for_backward(q, k, q_weight, k_weight, positions)
        ctx.eps, ctx.rotary = eps, rotary
        ctx.set_materialize_grads(True)
        return outs[0] if k is None else tuple(outs)

    @staticmethod
    @_once
    def backward(ctx, *douts):
        q, k, q_weight, k_weight, positions = ctx.saved_tensors
        grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) if want else None
                 for x, want in zip((q, k, q_weight, k_weight), ctx.needs_input_grad)]
        # queries or keys of which nothing is wanted are left out of the call; weights are summed on the way to dx
        sides = [(torch.empty_like(d) if dx is None else dx, dw, d, x, w) for dx, dw, d, x, w in
                 zip(grads[:2], grads[2:], map(_rows_contiguous, douts), (q, k), (q_weight, k_weight))
                 if dx is not None or dw is not None]
        if sides:
            dx, dw, dout, x, w = zip(*sides, *[(None,) * 5] * (2 - len(sides)))
            head_norm_grad_(*dx, *dw, *dout, *x, *w, eps=ctx.eps, rotary=ctx.rotary, positions=positions)
        if k is None and grads[3] is not None:   # (a weight of no keys)
            grads[3].zero_()
        return *grads, None, None, None


def head_norm(q, k=None, q_weight=None, k_weight=None, *, eps=1e-6, rotary=None, positions=None):
    """head_norm_ as a differentiable function of q, k and their weights, all of any strides; returns q's result, or q's
    and k's."""
    return _HeadNorm.apply(_rows_contiguous(q), None if k is None else _rows_contiguous(k), _contiguous(q_weight),
                           _contiguous(k_weight), eps, rotary, _contiguous(positions))


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, rotary, positions, inverse):
        outs = [None if x is None else torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (q, k)]
        rotate_(*outs, q, k, rotary, positions, inverse=inverse)
        ctx.save_for_backward(positions)
        ctx.rotary, ctx.inverse = rotary, inverse
        ctx.set_materialize_grads(True)
        return outs[0] if k is None else tuple(outs)

    @staticmethod
    @_once
    def backward(ctx, *douts):
        positions, = ctx.saved_tensors
        grads = [torch.empty(d.shape, dtype=d.dtype, device=d.device) if want else None
                 for d, want in zip(douts, ctx.needs_input_grad)] + [None] * (2 - len(douts))
        sides = [(dx, d) for dx, d in zip(grads, map(_rows_contiguous, douts)) if dx is not None]
        if sides:
            dx, dout = zip(*sides, *[(None, None)] * (2 - len(sides)))
            rotate_(*dx, *dout, ctx.rotary, positions, inverse=not ctx.inverse)
        return *grads, None, None, None


def rotate(q, k, rotary, positions, *, inverse=False):
    """rotate_ as a differentiable function of q and k (k may be None), all of any strides."""
    return _Rotate.apply(_rows_contiguous(q), None if k is None else _rows_contiguous(k), rotary, _contiguous(positions),
                         inverse)


class _Dropout(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, p, seed, call):
        # (a call number on the device may move on before the gradient is asked for)
        call = call.clone() if isinstance(call, torch.Tensor) else call
        out = torch.empty(x.shape, dtype=x.dtype, device=x.device)
        dropout_(out, x, p, seed, call=call, residual=residual)
        ctx.p, ctx.seed, ctx.call = p, seed, call
        return out

    @staticmethod
    @_once
    def backward(ctx, dout):
        dx = None
        if ctx.needs_input_grad[0]:
            dx = torch.empty(dout.shape, dtype=dout.dtype, device=dout.device)
            dropout_(dx, _rows_even(dout), ctx.p, ctx.seed, call=ctx.call)
        return dx, dout if ctx.needs_input_grad[1] else None, None, None, None


def dropout(x, p, seed, *, call=0, residual=None):
    """dropout_ as a differentiable function of x and residual, of any strides."""
    return _Dropout.apply(_rows_even(x), _rows_even(residual), p, seed, call)
