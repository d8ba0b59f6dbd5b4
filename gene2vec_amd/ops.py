"""Tensor operators on the GPU: what a classifier over the gene embeddings
(``ggipnn.py``; the reference's src/GGIPNN.py) trains its table with.

    embedding_lookup       rows of a table by token, scaled; differentiable
    embedding_lookup_grad  the gradient of the table by itself
    global_norm            the 2-norm over a list of gradients
    clip_by_global_norm    the list scaled down to a norm; ``_`` at the end: in place

They are torch operators too (``torch.ops.g2v``, which this module registers):
tracers, functional transforms and dispatch modes see them.

They run in ``libg2v.so`` on the tensors' own device and on torch's current
stream there, without synchronising; there is no CPU fallback.  Tensors that
another stream made are the caller's to wait for, and to ``record_stream``, as
with any torch operator.  Workspaces come from torch's allocator in each call,
so calls on several streams do not share any, and a call captured into a
``torch.cuda.graph`` keeps its own in the graph's pool.  The same inputs give
the same bits.  Tensors and values that do not fit raise ``ValueError``
(``TypeError``: what is no number) before anything runs, the library's own
errors ``_native.G2VError``.

A lookup in a table that requires its gradient is captured only while no graph
of that leaf, or of a leaf that the table was computed from, lives from the
default stream (``del`` the loss of earlier steps): torch accumulates on the
stream that graph was built on, and the default stream ends a capture, so the
call raises ``ValueError`` then.  A backward pass is captured together with its
lookup: one that was looked up before the capture, on another stream, is torch's
to run there, with the same end.
"""
from __future__ import annotations

import torch  # (its libraries, and its HIP runtime, come first)

from . import _native as N

N.lib()  # raises where libg2v.so is missing
try:
    from . import _g2v_torch as _x
except ImportError as e:
    raise N.NativeLibraryError(
        f"gene2vec_amd/_g2v_torch.so is missing or does not load ({e}): build it with "
        "`python -m gene2vec_amd.build`") from e
if (_x.abi_version() != N.ABI_VERSION
        or _x.torch_version() != torch.__version__.split("+")[0]):
    raise N.NativeLibraryError(
        f"_g2v_torch.so was built for libg2v's ABI {_x.abi_version()} and torch "
        f"{_x.torch_version()}, not {N.ABI_VERSION} and {torch.__version__}: "
        "`python -m gene2vec_amd.build --force`")


def embedding_lookup(params, ids, scale=1.0, padding_idx=None, dtype=None):
    """``scale * params[ids]``: a tensor of ``ids.shape + (D,)``.

    params       [V, D] float32, float16 or bfloat16; rows contiguous, any row
                 stride of at least D
    ids          int32 or int64 of any shape, up to 2^31 - 1 tokens; a token
                 outside [0, V) gets a zero row (-1: absent)
    scale        a number, applied in fp32
    padding_idx  a row that gets no gradient (it is looked up like the others)
    dtype        of the result; None: that of params.  One rounding from fp32

    Differentiable in params, once, and in forward mode; the gradient is dense
    [V, D] in the type of params (``embedding_lookup_grad``).  ids that are not
    contiguous are copied.
    """
    return _x.embedding_lookup(params, ids, scale, padding_idx, dtype)


def embedding_lookup_grad(dy, ids, vocab_size, scale=1.0, padding_idx=None, dtype=None):
    """The gradient of ``embedding_lookup``'s table: ``[vocab_size, D]`` with
    row v = scale * the sum of ``dy[i]`` over ``ids[i] == v``.

    dy  ids.shape + (D,), float32, float16 or bfloat16, any strides (rows that
        are not contiguous are copied); dtype of the result: None = dy's.
    The sums are fp32 in a fixed order, without atomics, and rounded once.
    Not differentiable, but for forward mode in dy: a dy that requires a gradient
    is refused in grad mode.
    """
    return _x.embedding_lookup_grad(dy, ids, vocab_size, scale, padding_idx, dtype)


def global_norm(t_list):
    """``sqrt(sum of squares)`` over every element of the tensors, as a 0-d
    float32 tensor on their device; ``None`` entries are left out.

    Tensors: float32, float16 or bfloat16, mixed as they come, of one device,
    dense in memory in any order of dimensions.  Squares and sums are fp64, so
    only a norm beyond fp32 itself overflows.  Not differentiable: a tensor that
    requires a gradient (in grad mode) or has a forward-mode tangent is refused.
    """
    return _x.global_norm(t_list)


def clip_by_global_norm(t_list, clip_norm, out=None):
    """``(list, norm)``: every tensor times ``clip_norm / max(norm, clip_norm)``,
    and the ``global_norm`` before it.

    out  None: new tensors; else a list of tensors of the same shapes, types
         and strides to write, apart from each other and from the inputs, or
         the input itself in its own place.  ``None`` entries stay ``None``.
    An element that is infinite or NaN makes every element NaN, so that an
    overflow is not taken for a step of length zero.  The factor is of the fp64
    norm: one that is finite but beyond fp32 is returned as infinity, and the
    tensors are clipped all the same.
    """
    return _x.clip_by_global_norm(t_list, clip_norm, out)


def clip_by_global_norm_(t_list, clip_norm):
    """``clip_by_global_norm`` in place; returns the norm before it."""
    return _x.clip_by_global_norm_(t_list, clip_norm)
