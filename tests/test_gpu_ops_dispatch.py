"""GPU: the tensor operators as torch's dispatcher sees them -- traced, under
functional transforms and dispatch modes.  Everything here is compared with the
eager call of the same operator on the same inputs, bit for bit: the kernels are
the same."""
import io

import pytest
import torch

from gene2vec_amd import ops

pytestmark = pytest.mark.gpu

V, D = 40, 12


def inputs(seed, n=50):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(V, D, device="cuda", generator=gen)
    ids = torch.randint(-1, V, (n,), device="cuda", generator=gen)
    return w, ids, torch.randn(n, D, device="cuda", generator=gen)


def clip_(dy, w):
    a, b = dy.clone(), w.clone()
    norm = ops.clip_by_global_norm_([a, None, b], 1.0)
    return a, b, norm


def clip_out(dy, w):
    outs = [torch.empty_like(dy), torch.empty_like(w)]
    _, norm = ops.clip_by_global_norm([dy, w], 1.0, out=outs)
    return outs[0], outs[1], norm


FORMS = {
    "lookup": lambda w, ids, dy: ops.embedding_lookup(w, ids, 1.5, 3),
    "lookup_2d": lambda w, ids, dy: ops.embedding_lookup(w, ids.view(5, 10).t()),
    "lookup_grad": lambda w, ids, dy: ops.embedding_lookup_grad(dy, ids, V, 0.5, 2),
    "norm": lambda w, ids, dy: ops.global_norm([dy, w]),
    "clip": lambda w, ids, dy: ops.clip_by_global_norm([dy, None, w], 1.0)[0][2],
    "clip_norm": lambda w, ids, dy: ops.clip_by_global_norm([dy, w], 1.0)[1],
    "clip_out": lambda w, ids, dy: clip_out(dy, w),
    "clip_": lambda w, ids, dy: clip_(dy, w),
}


def equal(a, b):
    a, b = (x if isinstance(x, tuple) else (x,) for x in (a, b))
    return len(a) == len(b) and all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize("form", FORMS)
def test_traced(form):
    f = FORMS[form]
    traced = torch.jit.trace(f, inputs(1))
    assert "g2v::" in str(traced.inlined_graph)
    buffer = io.BytesIO()
    torch.jit.save(traced, buffer)
    buffer.seek(0)
    loaded = torch.jit.load(buffer)
    for seed in (1, 2, 3):
        args = inputs(seed)
        # memory that a call would return unwritten does not hold its answer
        torch.full((4096,), float("nan"), device="cuda")
        assert equal(traced(*args), f(*args)) and equal(loaded(*args), f(*args))


def test_traced_lookup_is_differentiable_and_checks_its_inputs():
    w, ids, c = inputs(4)
    traced = torch.jit.trace(lambda w, ids: ops.embedding_lookup(w, ids, 2.0), (w, ids))
    w.requires_grad_(True)
    got, = torch.autograd.grad(traced(w, ids), w, c)
    assert torch.equal(got, ops.embedding_lookup_grad(c, ids, V, 2.0))
    for bad in ((w.double(), ids), (w, ids.float()), (w[:, ::2], ids), (w, ids.cpu()),
                (w.cpu(), ids.cpu())):
        with pytest.raises(Exception, match="must be|on cpu|contiguous|CPU"):
            traced(*bad)


@pytest.mark.parametrize("form", FORMS)
def test_dispatch_modes_see_the_operator(form):
    from torch.utils._python_dispatch import TorchDispatchMode
    seen = []

    class Watch(TorchDispatchMode):
        def __torch_dispatch__(self, func, types, args=(), kwargs=None):
            seen.append(func.name())
            return func(*args, **(kwargs or {}))

    args = inputs(5)
    want = FORMS[form](*args)
    with Watch():
        got = FORMS[form](*args)
    assert equal(got, want)
    assert any(name.startswith("g2v::") for name in seen), seen


def test_refusals_of_the_registered_operators():
    """called past the Python entries they check the same"""
    w, ids, dy = inputs(6)
    g = torch.ops.g2v
    for call in (lambda: g.embedding_lookup(w, ids.float(), 1.0, -1, torch.float32),
                 lambda: g.embedding_lookup(w, ids, 1.0, -1, torch.float64),
                 lambda: g.embedding_lookup(w, ids, 1.0, V, torch.float32),
                 lambda: g.embedding_lookup(w, ids, 1.0, -2, torch.float32),
                 lambda: g.embedding_lookup(w.t(), ids, 1.0, -1, torch.float32),
                 lambda: g.embedding_lookup_grad(dy, ids[:-1], V, 1.0, -1, torch.float32),
                 lambda: g.embedding_lookup_grad(dy, ids.cpu(), V, 1.0, -1, torch.float32),
                 lambda: g.embedding_lookup_grad(dy, ids, 0, 1.0, -1, torch.float32),
                 lambda: g.global_norm([w, dy.double()]), lambda: g.global_norm([]),
                 lambda: g.clip_by_global_norm([w], 0.0),
                 lambda: g.clip_by_global_norm_([w, w], 1.0),
                 lambda: g.clip_by_global_norm.out([w], 1.0, out=[dy]),
                 lambda: g.clip_by_global_norm.out([w], 1.0, out=[])):
        with pytest.raises((ValueError, NotImplementedError)):
            call()
