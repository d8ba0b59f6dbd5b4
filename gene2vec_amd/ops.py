"""Tensor operators on the GPU: what a classifier over the gene embeddings
(``ggipnn.py``; the reference's src/GGIPNN.py) trains its table with.

    embedding_lookup       rows of a table by token, scaled; differentiable
    embedding_lookup_grad  the gradient of the table by itself
    global_norm            the 2-norm over a list of gradients
    clip_by_global_norm    the list scaled down to a norm; ``_`` at the end: in place

The names are those of the TF1 calls the reference's classifier is written in
(tf.nn.embedding_lookup, tf.global_norm, tf.clip_by_global_norm).

They run in ``libg2v.so`` on the tensors' own device and on torch's current
stream there, without synchronising; there is no CPU fallback.  Tensors that
another stream made are the caller's to wait for, and to ``record_stream``, as
with any torch operator.  Workspaces come from torch's allocator in each call,
so calls on several streams do not share any, and a call captured into a
``torch.cuda.graph`` keeps its own in the graph's pool.  The same inputs give
the same bits.  Wrong arguments raise ``ValueError`` before anything runs.

A backward pass is captured best on leaves that no live eager graph holds
(``del`` the loss of earlier steps, ``grad = None``): torch accumulates into a
leaf on the stream its eager graph was built on, and that ends a capture.
"""
from __future__ import annotations

import array
import ctypes as C
import functools
import math
from operator import attrgetter

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

_TYPES = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}
_FLT_MAX = torch.finfo(torch.float32).max


def _stream(index):
    return torch._C._cuda_getCurrentRawStream(index)


def _on_gpu(t, name):
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name} must be a tensor, not {type(t).__name__}")
    if not t.is_cuda or t.layout is not torch.strided:
        raise ValueError(f"{name} must be a dense tensor on the GPU (there is no CPU fallback)")


def _check_ids(ids, device):
    _on_gpu(ids, "ids")
    if ids.dtype not in _ID_BYTES:
        raise ValueError(f"ids must be int32 or int64, not {ids.dtype}")
    if ids.device != device:
        raise ValueError(f"ids are on {ids.device}, the rows on {device}")


def _check_options(scale, padding_idx, V, dtype):
    scale = float(scale)
    if not abs(scale) <= _FLT_MAX:
        raise ValueError(f"scale must be finite in fp32, not {scale}")
    if dtype not in _TYPES:
        raise ValueError(f"dtype must be float32, float16 or bfloat16, not {dtype}")
    if padding_idx is None:
        return scale, -1
    pad = int(padding_idx)
    if pad != padding_idx or not 0 <= pad < V:
        raise ValueError(f"padding_idx {padding_idx} is not in [0, {V})")
    return scale, pad


def _row_stride(t, V, D):
    """the row stride of the table, whose rows are contiguous"""
    s0, s1 = t.stride()
    if s1 != 1 and D > 1:
        raise ValueError("the elements of a row of params must be contiguous")
    if V == 1:
        return D
    if s0 < D:
        raise ValueError(f"the rows of params overlap (strides {t.stride()})")
    return s0


def _lookup(params, ids, ld, scale, dtype):
    V, D = params.shape
    index = params.device.index
    out = params.new_empty(ids.shape + (D,), dtype=dtype)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    N.check(N.lib().g2v_embed_lookup(
        index, params.data_ptr(), _TYPES[params.dtype], V, D, ld, ids.data_ptr(),
        _ID_BYTES[ids.dtype], ids.numel(), scale, out.data_ptr(), _TYPES[dtype], _stream(index)))
    return out


@functools.lru_cache(maxsize=256)
def _grad_workspace(n, V, D):
    nbytes = C.c_int64()
    N.check(N.lib().g2v_embed_grad_workspace(n, V, D, C.byref(nbytes)))
    return nbytes.value


def _lookup_grad(dy, ids, V, D, scale, pad, dtype):
    n = ids.numel()
    if not ids.is_contiguous():
        ids = ids.contiguous()
    if dy.dim() != 2:
        dy = dy.reshape(n, D)
    ld, s1 = dy.stride()
    if n <= 1:
        ld = D
    if (s1 != 1 and D > 1) or ld < D:  # a transposed or broadcast gradient
        dy = dy.contiguous()
        ld = D
    index = dy.device.index
    nbytes = _grad_workspace(n, V, D)
    grad = dy.new_empty((V, D), dtype=dtype)
    ws = dy.new_empty(nbytes, dtype=torch.uint8)
    N.check(N.lib().g2v_embed_grad(
        index, dy.data_ptr(), _TYPES[dy.dtype], ld, ids.data_ptr(), _ID_BYTES[ids.dtype], n, V, D,
        scale, pad, grad.data_ptr(), _TYPES[dtype], ws.data_ptr(), nbytes, _stream(index)))
    return grad


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, params, ids, ld, scale, pad, dtype):
        ctx.save_for_backward(ids)
        ctx.args = *params.shape, scale, pad, params.dtype
        return _lookup(params, ids, ld, scale, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        return _lookup_grad(dy, ids, *ctx.args), None, None, None, None, None


def embedding_lookup(params, ids, scale=1.0, padding_idx=None, dtype=None):
    """``scale * params[ids]``: a tensor of ``ids.shape + (D,)``.

    params       [V, D] float32, float16 or bfloat16; rows contiguous, any row
                 stride of at least D
    ids          int32 or int64 of any shape, up to 2^31 - 1 tokens; a token
                 outside [0, V) gets a zero row (-1: absent)
    scale        a number, applied in fp32
    padding_idx  a row that gets no gradient (it is looked up like the others)
    dtype        of the result; None: that of params.  One rounding from fp32

    Differentiable in params, once; the gradient is dense [V, D] in the type
    of params (``embedding_lookup_grad``).  ids that are not contiguous are
    copied.
    """
    _on_gpu(params, "params")
    if params.dim() != 2 or params.numel() == 0:
        raise ValueError(f"params must be a matrix [V, D], not {tuple(params.shape)}")
    if params.dtype not in _TYPES:
        raise ValueError(f"params must be float32, float16 or bfloat16, not {params.dtype}")
    V, D = params.shape
    ld = _row_stride(params, V, D)
    _check_ids(ids, params.device)
    if dtype is None:
        dtype = params.dtype
    scale, pad = _check_options(scale, padding_idx, V, dtype)
    if params.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(params, ids, ld, scale, pad, dtype)
    return _lookup(params, ids, ld, scale, dtype)


def embedding_lookup_grad(dy, ids, vocab_size, scale=1.0, padding_idx=None, dtype=None):
    """The gradient of ``embedding_lookup``'s table: ``[vocab_size, D]`` with
    row v = scale * the sum of ``dy[i]`` over ``ids[i] == v``.

    dy  ids.shape + (D,), float32, float16 or bfloat16, any strides (rows that
        are not contiguous are copied); dtype of the result: None = dy's.
    The sums are fp32 in a fixed order, without atomics, and rounded once.
    """
    _on_gpu(dy, "dy")
    _check_ids(ids, dy.device)
    if dy.dtype not in _TYPES:
        raise ValueError(f"dy must be float32, float16 or bfloat16, not {dy.dtype}")
    if dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape or dy.shape[-1] < 1:
        raise ValueError(f"dy {tuple(dy.shape)} does not hold a row for each of ids "
                         f"{tuple(ids.shape)}")
    V = int(vocab_size)
    if V != vocab_size or V < 1:
        raise ValueError(f"vocab_size must be a positive number, not {vocab_size}")
    dtype = dy.dtype if dtype is None else dtype
    scale, pad = _check_options(scale, padding_idx, V, dtype)
    return _lookup_grad(dy.detach(), ids, V, dy.shape[-1], scale, pad, dtype)


def _is_dense(t):
    """its elements fill one stretch of memory, each once, in whatever order"""
    if t.is_contiguous():
        return True
    want = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n != 1):
        if stride != want:
            return False
        want *= size
    return True


def _check_list(t_list, what):
    """the tensors of the list that are there, and their device"""
    t_list = list(t_list)
    there = [t for t in t_list if t is not None]
    if not there:
        raise ValueError(f"{what}: the list holds no tensor")
    for t in there:
        if not isinstance(t, torch.Tensor):
            raise ValueError(f"{what}: the list must hold tensors, not {type(t).__name__}")
    devices = set(map(attrgetter("device"), there))
    if (len(devices) > 1 or not there[0].is_cuda
            or set(map(attrgetter("layout"), there)) != {torch.strided}):
        for t in there:
            _on_gpu(t, what)
        raise ValueError(f"{what}: tensors on {sorted(map(str, devices))}")
    if not set(map(attrgetter("dtype"), there)) <= _TYPES.keys():
        raise ValueError(f"{what}: tensors must be float32, float16 or bfloat16, not "
                         f"{sorted({str(t.dtype) for t in there})}")
    if torch.is_grad_enabled() and any(map(attrgetter("requires_grad"), there)):
        raise ValueError(f"{what} is not differentiable: pass gradients, or call it under "
                         "no_grad()")
    if not all(map(torch.Tensor.is_contiguous, there)):
        for t in there:
            if not _is_dense(t):
                raise ValueError(f"{what}: the elements of a tensor must be dense in memory "
                                 f"(shape {tuple(t.shape)}, strides {t.stride()})")
    return t_list, there, devices.pop()


def _address(a):
    return a.buffer_info()[0]


def _pointers(tensors):
    return array.array("Q", map(torch.Tensor.data_ptr, tensors))


@functools.lru_cache(maxsize=256)
def _norm_workspace(n):
    nbytes = C.c_int64()
    N.check(N.lib().g2v_global_norm_workspace(n, C.byref(nbytes)))
    return nbytes.value


def _describe(there):
    numel = array.array("q", map(torch.Tensor.numel, there))
    types = array.array("i", [_TYPES[t.dtype] for t in there])
    norm = there[0].new_empty((), dtype=torch.float32)
    return numel, types, norm, there[0].new_empty(_norm_workspace(len(there)), dtype=torch.uint8)


def global_norm(t_list):
    """``sqrt(sum of squares)`` over every element of the tensors, as a 0-d
    float32 tensor on their device; ``None`` entries are left out.

    Tensors: float32, float16 or bfloat16, mixed as they come, of one device,
    dense in memory in any order of dimensions.  Squares and sums are fp64, so
    only a norm beyond fp32 itself overflows.  Not differentiable.
    """
    _, there, device = _check_list(t_list, "global_norm")
    src = _pointers(there)
    numel, types, norm, ws = _describe(there)
    N.check(N.lib().g2v_global_norm(device.index, _address(src), _address(numel), _address(types),
                                    len(there), norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                    _stream(device.index)))
    return norm


def _clip(there, outs, device, clip_norm):
    clip_norm = float(clip_norm)
    if not 0.0 < clip_norm < math.inf:
        raise ValueError(f"clip_norm must be positive and finite, not {clip_norm}")
    src = _pointers(there)
    dst = src if outs is there else _pointers(outs)
    numel, types, norm, ws = _describe(there)
    try:
        N.check(N.lib().g2v_clip_global_norm(
            device.index, _address(src), _address(dst), _address(numel), _address(types),
            len(there), clip_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(),
            _stream(device.index)))
    except N.G2VError as e:  # tensors that overlap
        raise (ValueError(str(e)) if e.code == N.G2V_EINVAL else e)
    return norm


def clip_by_global_norm(t_list, clip_norm, out=None):
    """``(list, norm)``: every tensor times ``clip_norm / max(norm, clip_norm)``,
    and the ``global_norm`` before it.

    out  None: new tensors; else a list of tensors of the same shapes, types
         and strides to write, apart from each other and from the inputs, or
         the input itself in its own place.  ``None`` entries stay ``None``.
    A norm that is not finite makes every element NaN, so that an overflow is
    not taken for a step of length zero.
    """
    t_list, there, device = _check_list(t_list, "clip_by_global_norm")
    if out is None:
        out = [None if t is None else torch.empty_like(t) for t in t_list]
        outs = [o for o in out if o is not None]
    else:
        out = list(out)
        if len(out) != len(t_list):
            raise ValueError(f"clip_by_global_norm: {len(out)} outputs for {len(t_list)} tensors")
        outs = [o for t, o in zip(t_list, out) if t is not None]
        for t, o in zip(there, outs):
            _on_gpu(o, "clip_by_global_norm: out")
            if (o.shape != t.shape or o.dtype != t.dtype or o.device != device
                    or not (o.is_contiguous() and t.is_contiguous() or o.stride() == t.stride())):
                raise ValueError("clip_by_global_norm: an output differs from its tensor in "
                                 "shape, type, strides or device")
            if o.requires_grad and torch.is_grad_enabled():
                raise ValueError("clip_by_global_norm: an output requires a gradient")
    norm = _clip(there, outs, device, clip_norm)
    torch.autograd.graph.increment_version(outs)
    return [None if t is None else o for t, o in zip(t_list, out)], norm


def clip_by_global_norm_(t_list, clip_norm):
    """``clip_by_global_norm`` in place; returns the norm before it."""
    _, there, device = _check_list(t_list, "clip_by_global_norm_")
    norm = _clip(there, there, device, clip_norm)
    torch.autograd.graph.increment_version(there)
    return norm
