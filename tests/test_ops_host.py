"""Refusals of the tensor operators that need no GPU: the C entries check
their arguments before they touch the device, the Python layer before it calls
them, and the classifier's CPU path follows the same formulas."""
import ctypes as C

import numpy as np
import pytest
import torch

from gene2vec_amd import _native as N
from gene2vec_amd import ggipnn as G
from gene2vec_amd import ops

P = 0x10000  # a stand-in for a device address: refused calls never read it


def _lookup(**kw):
    a = dict(device=0, table=P, table_type=N.F32, V=10, D=4, ld=4, ids=P, id_bytes=8, n=3,
             scale=1.0, out=P, out_type=N.F32, stream=None)
    a.update(kw)
    return N.lib().g2v_embed_lookup(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(device=-1), N.G2V_EINVAL), (dict(table=None), N.G2V_EINVAL),
    (dict(table=P + 2), N.G2V_EINVAL), (dict(table_type=3), N.G2V_EINVAL),
    (dict(V=0), N.G2V_EINVAL), (dict(D=0), N.G2V_EINVAL), (dict(n=-1), N.G2V_EINVAL),
    (dict(ld=3), N.G2V_EINVAL), (dict(ids=None), N.G2V_EINVAL), (dict(ids=P + 4), N.G2V_EINVAL),
    (dict(id_bytes=2), N.G2V_EINVAL), (dict(out=None), N.G2V_EINVAL),
    (dict(out_type=-1), N.G2V_EINVAL), (dict(V=2**31), N.G2V_ERANGE), (dict(n=2**31), N.G2V_ERANGE),
    (dict(D=N.EMBED_MAX_DIM + 1, ld=N.EMBED_MAX_DIM + 1), N.G2V_ERANGE),
    (dict(ld=2**60), N.G2V_ERANGE)])
def test_lookup_refuses(kw, rc):
    assert _lookup(**kw) == rc
    assert b"g2v_embed_lookup" in N.lib().g2v_last_error()


def test_lookup_of_nothing_needs_no_device():
    assert _lookup(n=0, ids=None, out=None) == N.G2V_OK


def _grad(**kw):
    n, V, D = kw.get("n", 3), kw.get("V", 10), kw.get("D", 4)
    need = C.c_int64()
    N.lib().g2v_embed_grad_workspace(n, V, D, C.byref(need))
    a = dict(device=0, dy=P, dy_type=N.F32, dy_ld=4, ids=P, id_bytes=8, n=3, V=10, D=4, scale=1.0,
             padding_id=-1, grad=P, grad_type=N.F32, workspace=P, workspace_bytes=need.value,
             stream=None)
    a.update(kw)
    return N.lib().g2v_embed_grad(*a.values())


@pytest.mark.parametrize("kw,rc", [
    (dict(device=-1), N.G2V_EINVAL), (dict(dy=None), N.G2V_EINVAL), (dict(dy=P + 1), N.G2V_EINVAL),
    (dict(dy_ld=3), N.G2V_EINVAL), (dict(dy_type=9), N.G2V_EINVAL), (dict(V=0), N.G2V_EINVAL),
    (dict(V=2**31), N.G2V_ERANGE), (dict(n=2**31), N.G2V_ERANGE),
    (dict(id_bytes=0), N.G2V_EINVAL), (dict(ids=P + 4), N.G2V_EINVAL),
    (dict(grad=None), N.G2V_EINVAL), (dict(grad_type=7), N.G2V_EINVAL),
    (dict(padding_id=10), N.G2V_EINVAL), (dict(padding_id=-2), N.G2V_EINVAL)])
def test_grad_refuses(kw, rc):
    assert _grad(**kw) == rc
    assert b"g2v_embed_grad" in N.lib().g2v_last_error()


def test_workspaces_are_asked_for_and_checked():
    L = N.lib()
    b = C.c_int64(-1)
    assert L.g2v_embed_grad_workspace(5000, 1000, 64, C.byref(b)) == N.G2V_OK and b.value >= 0
    if b.value:
        assert _grad(n=5000, V=1000, D=64, dy_ld=64, workspace_bytes=b.value - 1) == N.G2V_EINVAL
        assert _grad(n=5000, V=1000, D=64, dy_ld=64, workspace=P + 8) == N.G2V_EINVAL
    for n in (0, 1, 64, 256, 257, 16384, 16385, 65536, 262145, 2**24, 2**31 - 1):
        for V in (1, 255, 256, 262144, 262145, 2**30, 2**30 + 1, 2**31 - 1):
            for D in (1, 200, 8193):
                assert L.g2v_embed_grad_workspace(n, V, D, C.byref(b)) == N.G2V_OK
                assert 4 * n + 8 * V <= b.value < 16 * n + 17 * V + n * D // 2 + 2**25
    assert L.g2v_embed_grad_workspace(-1, 10, 4, C.byref(b)) != N.G2V_OK
    assert L.g2v_embed_grad_workspace(3, 0, 4, C.byref(b)) == N.G2V_EINVAL
    assert L.g2v_embed_grad_workspace(3, 10, 4, None) == N.G2V_EINVAL
    assert L.g2v_global_norm_workspace(3, None) == N.G2V_EINVAL
    assert L.g2v_global_norm_workspace(-3, C.byref(b)) == N.G2V_EINVAL


def _list(ptrs, numel, types, dst=None, clip=None, norm=P, ws=P, short=0, device=0):
    L = N.lib()
    n = len(numel)
    need = C.c_int64()
    assert L.g2v_global_norm_workspace(n, C.byref(need)) == N.G2V_OK
    src = (C.c_void_p * n)(*ptrs)
    num = (C.c_int64 * n)(*numel)
    typ = (C.c_int32 * n)(*types)
    if clip is None:
        return L.g2v_global_norm(device, src, num, typ, n, norm, ws, need.value - short, None)
    out = (C.c_void_p * n)(*(ptrs if dst is None else dst))
    return L.g2v_clip_global_norm(device, src, out, num, typ, n, clip, norm, ws,
                                  need.value - short, None)


@pytest.mark.parametrize("a,kw,rc", [
    (([P], [4], [5]), {}, N.G2V_EINVAL), (([P + 2], [4], [N.F32]), {}, N.G2V_EINVAL),
    (([P + 1], [4], [N.BF16]), {}, N.G2V_EINVAL), (([None], [4], [N.F32]), {}, N.G2V_EINVAL),
    (([P], [-1], [N.F32]), {}, N.G2V_ERANGE), (([P], [2**41], [N.F32]), {}, N.G2V_ERANGE),
    (([P], [4], [N.F32]), dict(norm=None), N.G2V_EINVAL),
    (([P], [4], [N.F32]), dict(ws=None), N.G2V_EINVAL),
    (([P], [4], [N.F32]), dict(short=1), N.G2V_EINVAL),
    (([P], [4], [N.F32]), dict(device=-1), N.G2V_EINVAL)])
def test_norm_refuses(a, kw, rc):
    assert _list(*a, **kw) == rc
    assert _list(*a, clip=1.0, **kw) == rc


@pytest.mark.parametrize("clip", [0.0, -1.0, float("inf"), float("nan")])
def test_clip_refuses_the_bound(clip):
    assert _list([P], [4], [N.F32], clip=clip) == N.G2V_EINVAL


@pytest.mark.parametrize("ptrs,numel,dst", [
    ([P, P], [4, 4], None),                                  # the same tensor twice, in place
    ([P, P + 8], [4, 4], None),                              # two views that share elements
    ([P, P + 64], [4, 4], [P + 128, P + 136]),               # outputs that overlap
    ([P, P + 64], [4, 4], [P + 64, P + 128]),                # an output over another's input
    ([P], [4], [P + 4]),                                     # shifted by an element
    ([P, P + 256, P + 64], [100, 4, 4], [P + 512, P + 1024, P + 32])])
def test_clip_refuses_overlap(ptrs, numel, dst):
    assert _list(ptrs, numel, [N.F32] * len(ptrs), dst=dst, clip=1.0) == N.G2V_EINVAL
    assert b"overlap" in N.lib().g2v_last_error()


def test_python_layer_has_no_cpu_fallback():
    w, i = torch.zeros(4, 3), torch.zeros(2, dtype=torch.int64)
    for call in (lambda: ops.embedding_lookup(w, i),
                 lambda: ops.embedding_lookup_grad(torch.zeros(2, 3), i, 4),
                 lambda: ops.global_norm([w]), lambda: ops.clip_by_global_norm([w], 1.0),
                 lambda: ops.clip_by_global_norm_([w], 1.0)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for call in (lambda: ops.global_norm([]), lambda: ops.global_norm([None]),
                 lambda: ops.clip_by_global_norm_([], 1.0)):
        with pytest.raises(ValueError, match="no tensor"):
            call()
    with pytest.raises(ValueError, match="tensor"):
        ops.global_norm([1.0])
    with pytest.raises(ValueError, match="list of tensors"):
        ops.global_norm(w)
    with pytest.raises(ValueError, match="tensor"):
        ops.embedding_lookup(np.zeros((4, 3), np.float32), i)


def test_classifier_on_the_cpu_trains_its_table():
    gen = torch.Generator().manual_seed(3)
    emb = np.random.RandomState(0).randn(7, 4).astype(np.float32)
    frozen = G.build_model(7, emb, 4, "cpu", torch.Generator().manual_seed(3))
    assert not frozen.W.requires_grad
    model = G.build_model(7, emb, 4, "cpu", gen, train_embedding=True)
    x = torch.tensor([[0, 5], [5, 5], [2, 0]])
    loss = torch.nn.functional.cross_entropy(model(x, 1.0), torch.tensor([0, 1, 1]))
    loss.backward()
    assert model.W.grad.abs().sum(1).gt(0).tolist() == [True, False, True, False, False, True,
                                                        False]
    before = [p.grad.double().clone() for p in model.parameters()]
    norm = float(torch.sqrt(sum(g.square().sum() for g in before)))
    got = G.clip_gradients_(model.parameters(), norm / 4)
    # fp32: the norm and the factor round once, the product once more
    assert float(got) == pytest.approx(norm, rel=2**-24)
    for p, g in zip(model.parameters(), before):
        np.testing.assert_allclose(p.grad.double(), g / 4, rtol=3 * 2**-24, atol=1e-30)
    again = [p.grad.clone() for p in model.parameters()]
    G.clip_gradients_(model.parameters(), norm)
    assert all(torch.equal(p.grad, g) for p, g in zip(model.parameters(), again))
    model.W.grad[0, 0] = float("inf")
    G.clip_gradients_(model.parameters(), 1.0)
    assert all(p.grad.isnan().all() for p in model.parameters())
    with pytest.raises(ValueError):
        G.clip_gradients_(model.parameters(), 0.0)
