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
import math

import torch
from torch.autograd.function import once_differentiable

from . import _native as N

_TYPES = {torch.float32: N.F32, torch.float16: N.F16, torch.bfloat16: N.BF16}
_ID_BYTES = {torch.int32: 4, torch.int64: 8}
_FLT_MAX = torch.finfo(torch.float32).max


def _refuse(cond, msg):
    if cond:
        raise ValueError(msg)


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def _workspace(nbytes, device):
    return torch.empty(max(nbytes, 16), dtype=torch.uint8, device=device)


def _on_gpu(t, name):
    _refuse(not isinstance(t, torch.Tensor), f"{name} must be a tensor, not {type(t).__name__}")
    _refuse(t.layout is not torch.strided or not t.is_cuda,
            f"{name} must be a dense tensor on the GPU (there is no CPU fallback)")


def _check_ids(ids, device):
    _on_gpu(ids, "ids")
    _refuse(ids.dtype not in _ID_BYTES, f"ids must be int32 or int64, not {ids.dtype}")
    _refuse(ids.device != device, f"ids are on {ids.device}, the rows on {device}")


def _check_options(scale, padding_idx, V, dtype):
    scale = float(scale)
    _refuse(not abs(scale) <= _FLT_MAX, f"scale must be finite in fp32, not {scale}")
    _refuse(dtype not in _TYPES, f"dtype must be float32, float16 or bfloat16, not {dtype}")
    if padding_idx is None:
        return scale, -1
    pad = int(padding_idx)
    _refuse(pad != padding_idx or not 0 <= pad < V, f"padding_idx {padding_idx} is not in [0, {V})")
    return scale, pad


def _row_stride(t, name):
    """the row stride of a matrix whose rows are contiguous"""
    V, D = t.shape
    _refuse(D > 1 and t.stride(1) != 1, f"the elements of a row of {name} must be contiguous")
    ld = t.stride(0) if V > 1 else D
    _refuse(ld < D, f"the rows of {name} overlap (strides {tuple(t.stride())})")
    return ld


def _lookup(params, ids, scale, dtype):
    V, D = params.shape
    out = torch.empty(ids.shape + (D,), dtype=dtype, device=params.device)
    ids = ids.contiguous()
    N.check(N.lib().g2v_embed_lookup(
        params.device.index, params.data_ptr(), _TYPES[params.dtype], V, D,
        _row_stride(params, "params"), ids.data_ptr(), _ID_BYTES[ids.dtype], ids.numel(), scale,
        out.data_ptr(), _TYPES[dtype], _stream(params.device)))
    return out


def _lookup_grad(dy, ids, V, D, scale, pad, dtype):
    ids = ids.contiguous()
    n = ids.numel()
    dy = dy.reshape(n, D)
    if (D > 1 and dy.stride(1) != 1) or (n > 1 and dy.stride(0) < D):
        dy = dy.contiguous()  # a transposed or broadcast gradient
    nbytes = C.c_int64()
    N.check(N.lib().g2v_embed_grad_workspace(n, V, D, C.byref(nbytes)))
    grad = torch.empty(V, D, dtype=dtype, device=dy.device)
    ws = _workspace(nbytes.value, dy.device)
    N.check(N.lib().g2v_embed_grad(
        dy.device.index, dy.data_ptr(), _TYPES[dy.dtype], dy.stride(0) if n > 1 else D,
        ids.data_ptr(), _ID_BYTES[ids.dtype], n, V, D, scale, pad, grad.data_ptr(), _TYPES[dtype],
        ws.data_ptr(), ws.numel(), _stream(dy.device)))
    return grad


class _EmbeddingLookup(torch.autograd.Function):
    @staticmethod
    def forward(ctx, params, ids, scale, pad, dtype):
        ctx.save_for_backward(ids)
        ctx.args = params.shape[0], params.shape[1], scale, pad, params.dtype
        return _lookup(params, ids, scale, dtype)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        ids, = ctx.saved_tensors
        V, D, scale, pad, dtype = ctx.args
        return _lookup_grad(dy, ids, V, D, scale, pad, dtype), None, None, None, None


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
    _refuse(params.dim() != 2 or params.numel() == 0,
            f"params must be a matrix [V, D], not {tuple(params.shape)}")
    _refuse(params.dtype not in _TYPES,
            f"params must be float32, float16 or bfloat16, not {params.dtype}")
    _row_stride(params, "params")
    _check_ids(ids, params.device)
    dtype = params.dtype if dtype is None else dtype
    scale, pad = _check_options(scale, padding_idx, params.shape[0], dtype)
    if params.requires_grad and torch.is_grad_enabled():
        return _EmbeddingLookup.apply(params, ids, scale, pad, dtype)
    return _lookup(params, ids, scale, dtype)


def embedding_lookup_grad(dy, ids, vocab_size, scale=1.0, padding_idx=None, dtype=None):
    """The gradient of ``embedding_lookup``'s table: ``[vocab_size, D]`` with
    row v = scale * the sum of ``dy[i]`` over ``ids[i] == v``.

    dy  ids.shape + (D,), float32, float16 or bfloat16, any strides (rows that
        are not contiguous are copied); dtype of the result: None = dy's.
    The sums are fp32 in a fixed order, without atomics, and rounded once.
    """
    _on_gpu(dy, "dy")
    _check_ids(ids, dy.device)
    _refuse(dy.dtype not in _TYPES, f"dy must be float32, float16 or bfloat16, not {dy.dtype}")
    _refuse(dy.dim() != ids.dim() + 1 or dy.shape[:-1] != ids.shape or dy.shape[-1] < 1,
            f"dy {tuple(dy.shape)} does not hold a row for each of ids {tuple(ids.shape)}")
    V = int(vocab_size)
    _refuse(V != vocab_size or V < 1, f"vocab_size must be a positive number, not {vocab_size}")
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
    _refuse(not there, f"{what}: the list holds no tensor")
    device = there[0].device if isinstance(there[0], torch.Tensor) else None
    grad = torch.is_grad_enabled()
    for t in there:
        if (not isinstance(t, torch.Tensor) or not t.is_cuda or t.device != device
                or t.dtype not in _TYPES or t.layout is not torch.strided
                or (grad and t.requires_grad) or not _is_dense(t)):
            _on_gpu(t, what)
            _refuse(t.device != device, f"{what}: tensors on {device} and {t.device}")
            _refuse(t.dtype not in _TYPES,
                    f"{what}: tensors must be float32, float16 or bfloat16, not {t.dtype}")
            _refuse(grad and t.requires_grad,
                    f"{what} is not differentiable: pass gradients, or call it under no_grad()")
            _refuse(True, f"{what}: the elements of a tensor must be dense in memory "
                          f"(shape {tuple(t.shape)}, strides {tuple(t.stride())})")
    return t_list, there, device


def _address(a):
    return a.buffer_info()[0]


def _pointers(tensors):
    return array.array("Q", [t.data_ptr() for t in tensors])


def _describe(there, device):
    numel = array.array("q", [t.numel() for t in there])
    types = array.array("i", [_TYPES[t.dtype] for t in there])
    nbytes = C.c_int64()
    N.check(N.lib().g2v_global_norm_workspace(len(there), C.byref(nbytes)))
    norm = torch.empty((), dtype=torch.float32, device=device)
    return numel, types, norm, _workspace(nbytes.value, device)


def global_norm(t_list):
    """``sqrt(sum of squares)`` over every element of the tensors, as a 0-d
    float32 tensor on their device; ``None`` entries are left out.

    Tensors: float32, float16 or bfloat16, mixed as they come, of one device,
    dense in memory in any order of dimensions.  Squares and sums are fp64, so
    only a norm beyond fp32 itself overflows.  Not differentiable.
    """
    _, there, device = _check_list(t_list, "global_norm")
    src = _pointers(there)
    numel, types, norm, ws = _describe(there, device)
    N.check(N.lib().g2v_global_norm(device.index, _address(src), _address(numel), _address(types),
                                    len(there), norm.data_ptr(), ws.data_ptr(), ws.numel(),
                                    _stream(device)))
    return norm


def _clip(there, outs, device, clip_norm):
    clip_norm = float(clip_norm)
    _refuse(not 0.0 < clip_norm < math.inf,
            f"clip_norm must be positive and finite, not {clip_norm}")
    src = _pointers(there)
    dst = src if outs is there else _pointers(outs)
    numel, types, norm, ws = _describe(there, device)
    try:
        N.check(N.lib().g2v_clip_global_norm(
            device.index, _address(src), _address(dst), _address(numel), _address(types),
            len(there), clip_norm, norm.data_ptr(), ws.data_ptr(), ws.numel(), _stream(device)))
    except N.G2VError as e:
        raise (ValueError(str(e)) if e.code == N.G2V_EINVAL else e)
    return norm


def _written(tensors):
    """autograd learns that they changed"""
    torch.autograd.graph.increment_version([t for t in tensors if not t.is_inference()])


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
        _refuse(len(out) != len(t_list),
                f"clip_by_global_norm: {len(out)} outputs for {len(t_list)} tensors")
        outs = []
        for t, o in zip(t_list, out):
            if t is None:
                continue
            _on_gpu(o, "clip_by_global_norm: out")
            _refuse(o.shape != t.shape or o.dtype != t.dtype or o.device != t.device
                    or not (o.is_contiguous() and t.is_contiguous() or o.stride() == t.stride()),
                    "clip_by_global_norm: an output differs from its tensor in shape, type, "
                    "strides or device")
            _refuse(torch.is_grad_enabled() and o.requires_grad,
                    "clip_by_global_norm: an output requires a gradient")
            outs.append(o)
    norm = _clip(there, outs, device, clip_norm)
    _written(outs)
    return [None if t is None else o for t, o in zip(t_list, out)], norm


def clip_by_global_norm_(t_list, clip_norm):
    """``clip_by_global_norm`` in place; returns the norm before it."""
    _, there, device = _check_list(t_list, "clip_by_global_norm_")
    norm = _clip(there, there, device, clip_norm)
    _written(there)
    return norm
