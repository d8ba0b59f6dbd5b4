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


# ---- forward-mode derivatives and functional transforms ----------------------------------
@pytest.mark.parametrize("requires_grad", [False, True])
def test_forward_mode(requires_grad):
    """the lookup is linear in its table, its gradient in dy: the tangent of the
    result is the operator of the tangent"""
    import torch.autograd.forward_ad as fwd
    w, ids, dy = inputs(7)
    tw, tdy = inputs(8)[::2]
    want = ops.embedding_lookup(tw, ids, 0.5), ops.embedding_lookup_grad(tdy, ids, V, 0.5, 3)
    w.requires_grad_(requires_grad)
    with fwd.dual_level():
        y = ops.embedding_lookup(fwd.make_dual(w, tw), ids, 0.5)
        assert y.requires_grad == requires_grad
        primal, tangent = fwd.unpack_dual(y)
        assert torch.equal(primal, ops.embedding_lookup(w, ids, 0.5))
        assert torch.equal(tangent, want[0])
        tangent = fwd.unpack_dual(ops.embedding_lookup_grad(fwd.make_dual(dy, tdy), ids, V, 0.5,
                                                            3)).tangent
        assert torch.equal(tangent, want[1])
        if requires_grad:  # forward over reverse
            g, = torch.autograd.grad(y, w, fwd.make_dual(dy, tdy))
            assert torch.equal(fwd.unpack_dual(g).tangent,
                               ops.embedding_lookup_grad(tdy, ids, V, 0.5))


def test_forward_mode_is_refused_where_there_is_no_derivative():
    import torch.autograd.forward_ad as fwd
    w, _, dy = inputs(9)
    kept = w.clone()
    with fwd.dual_level():
        dual = fwd.make_dual(w, torch.ones_like(w))
        for call in (lambda: ops.global_norm([dy, dual]),
                     lambda: ops.clip_by_global_norm([dual], 1.0),
                     lambda: ops.clip_by_global_norm([w], 1.0, out=[dual]),
                     lambda: ops.clip_by_global_norm_([dual], 1.0)):
            for guard in (torch.enable_grad, torch.no_grad):
                with guard(), pytest.raises(ValueError, match="tangent"):
                    call()
    assert torch.equal(w, kept)
    assert float(ops.global_norm([w])) > 0


def test_functional_transforms():
    w, ids, c = inputs(10)
    t = torch.randn_like(w)

    def f(w):
        return (ops.embedding_lookup(w, ids, 0.5, 3) * c).sum()

    want = ops.embedding_lookup_grad(c, ids, V, 0.5, 3)
    assert torch.equal(torch.func.grad(f)(w), want)
    y, dy = torch.func.jvp(lambda w: ops.embedding_lookup(w, ids, 2.0), (w,), (t,))
    assert torch.equal(y, ops.embedding_lookup(w, ids, 2.0))
    assert torch.equal(dy, ops.embedding_lookup(t, ids, 2.0))
    _, back = torch.func.vjp(lambda w: ops.embedding_lookup(w, ids, 2.0), w)
    assert torch.equal(back(c)[0], ops.embedding_lookup_grad(c, ids, V, 2.0))
    for a, b in zip(torch.func.vmap(lambda i: ops.embedding_lookup(w, i))(ids.view(5, 10)),
                    ids.view(5, 10)):
        assert torch.equal(a, ops.embedding_lookup(w, b))
    many = torch.stack([w, t])
    for a, b in zip(torch.func.vmap(lambda w: ops.embedding_lookup(w, ids))(many), many):
        assert torch.equal(a, ops.embedding_lookup(b, ids))
    per = torch.func.vmap(torch.func.grad(lambda w, i: (ops.embedding_lookup(w, i) * c[:10]).sum()),
                          (None, 0))(w, ids.view(5, 10))
    for a, b in zip(per, ids.view(5, 10)):
        assert torch.equal(a, ops.embedding_lookup_grad(c[:10], b, V))


def test_double_backward_is_refused():
    w, ids, c = inputs(11)
    w.requires_grad_(True)
    y = ops.embedding_lookup(w, ids)
    g, = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError, match="once, not twice"):
        g.sum().backward()
    # a gradient that nothing differentiable went into is a constant, as torch's own
    y = ops.embedding_lookup(w, ids)
    g, = torch.autograd.grad(y, w, c, create_graph=True)
    assert not g.requires_grad and torch.equal(g, ops.embedding_lookup_grad(c, ids, V))
    with pytest.raises(RuntimeError, match="once, not twice"):
        torch.func.grad(lambda a: torch.func.grad(
            lambda b: ops.embedding_lookup(b, ids).square().sum())(a).sum())(w.detach())


def test_an_undefined_gradient_is_zero():
    class Stop(torch.autograd.Function):
        @staticmethod
        def forward(ctx, y):
            return y.clone()

        @staticmethod
        def backward(ctx, dy):
            return None

    w, ids, _ = inputs(12)
    w = w.bfloat16().requires_grad_(True)
    g, = torch.autograd.grad(Stop.apply(ops.embedding_lookup(w, ids)).sum(), w)
    assert g.dtype == w.dtype and g.shape == w.shape and not g.any()


def test_the_gradient_refuses_a_dy_that_requires_one():
    _, ids, dy = inputs(13)
    want = ops.embedding_lookup_grad(dy, ids, V)
    dy.requires_grad_(True)
    with pytest.raises(ValueError, match="not differentiable"):
        ops.embedding_lookup_grad(dy, ids, V)
    with torch.no_grad():
        assert torch.equal(ops.embedding_lookup_grad(dy, ids, V), want)
    assert torch.equal(ops.embedding_lookup_grad(dy.detach(), ids, V), want)
    with pytest.raises(RuntimeError, match="once, not twice"):  # past the Python entry
        torch.ops.g2v.embedding_lookup_grad(dy, ids, V, 1.0, -1, torch.float32).sum().backward()


def test_whole_numbers_are_numbers():
    import numpy as np
    w, ids, dy = inputs(14)
    want = ops.embedding_lookup_grad(dy, ids, V, padding_idx=3)
    for three in (3, 3.0, np.int32(3), np.float32(3), torch.tensor(3)):
        for v in (V, float(V), np.int64(V)):
            assert torch.equal(ops.embedding_lookup_grad(dy, ids, v, padding_idx=three), want)
    for bad in ("3", b"3", [3], None):
        with pytest.raises(TypeError):
            ops.embedding_lookup_grad(dy, ids, bad)
        if bad is not None:
            with pytest.raises(TypeError):
                ops.embedding_lookup(w, ids, padding_idx=bad)
    for bad in (float("nan"), float("inf"), 10**30, 2.5):
        with pytest.raises(ValueError, match="whole"):
            ops.embedding_lookup_grad(dy, ids, bad)
