"""GPU: the GGIPNN classifier against itself on the CPU, frozen and trained."""
import math

import numpy as np
import pytest
import torch

from gene2vec_amd import ggipnn as G

pytestmark = pytest.mark.gpu

V, D = 60, 8


def model(device, trained, dtype=torch.float32):
    emb = np.random.RandomState(0).randn(V, D).astype(np.float32)
    m = G.build_model(V, emb, D, "cpu", torch.Generator().manual_seed(3), train_embedding=trained)
    return m.to(device, dtype)


def tokens(seed=0, n=40):
    return torch.from_numpy(np.random.RandomState(seed).randint(0, V, (n, 2)))


def close(a, b, dtype=torch.float32):
    """the same model on two devices: sums of at most 130 terms in four products
    one after the other, each off by at most 130 u of its absolute sum on either
    side, and absolute sums at most 8-fold the values (as the tests of the
    classifier's training steps bound them)"""
    scale = float(b.abs().max()) + 1e-12
    tol = 8 * 4 * 130 * 2 * torch.finfo(dtype).eps / 2
    assert float((a.detach().cpu().double() - b.detach().cpu().double()).abs().max()) <= tol * scale


class Keep1(torch.nn.Module):
    def __init__(self, inner):
        super().__init__()
        self.inner = inner

    def forward(self, x):
        return self.inner(x, 1.0)


def test_frozen_classifier_is_traced():
    m, x = model("cuda", False).eval(), tokens().cuda()
    traced = torch.jit.trace(Keep1(m), (x,))
    for seed in (0, 1, 2):
        x = tokens(seed).cuda()
        assert torch.equal(traced(x), m(x, 1.0))
        close(traced(x), model("cpu", False)(x.cpu(), 1.0))


def test_frozen_classifier_keeps_torch_indexing():
    """types, devices and signs of tokens as torch takes them, and every transform"""
    m, ref = model("cuda", False), model("cpu", False)
    x = tokens()
    x[0] = -1  # the last row
    for given in (x.cuda(), x.cuda().int(), x):  # tokens on the host too
        close(m(given, 1.0), ref(x, 1.0))
    close(m(x.cuda(), 1.0), ref(x % V, 1.0))
    m64, ref64 = model("cuda", False, torch.float64), model("cpu", False, torch.float64)
    close(m64(x.cuda(), 1.0), ref64(x, 1.0), torch.float64)
    t = torch.randn(V, D, device="cuda")

    def f(mod, x, w):
        return torch.func.functional_call(mod, {"W": w}, (x, 1.0))

    _, got = torch.func.jvp(lambda w: f(m, x.cuda(), w), (m.W.detach(),), (t,))
    _, want = torch.func.jvp(lambda w: f(ref, x, w), (ref.W.detach(),), (t.cpu(),))
    close(got, want)
    got = torch.func.vmap(lambda i: m(i, 1.0))(x.cuda().view(4, 10, 2))
    close(got.reshape(40, 2), ref(x, 1.0))
    got = torch.func.grad(lambda w: f(m, x.cuda(), w).square().sum())(m.W.detach())
    want = torch.func.grad(lambda w: f(ref, x, w).square().sum())(ref.W.detach())
    close(got, want)
    m.W.requires_grad_(True)  # by hand: twice differentiable, as any indexed tensor
    g, = torch.autograd.grad(m(x.cuda(), 1.0).square().sum(), m.W, create_graph=True)
    g.square().sum().backward()
    assert math.isfinite(float(m.W.grad.sum()))


def loss_and_grads(m, x):
    t = torch.arange(len(x), device=m.W.device) % 2
    loss = torch.nn.functional.cross_entropy(m(x, 1.0), t)
    return [loss.detach()] + list(torch.autograd.grad(loss, list(m.parameters())))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64])
@pytest.mark.parametrize("place", ["beside", "int32", "host"])
def test_trained_classifier_is_the_same_on_both_devices(dtype, place):
    """tokens outside the table among them"""
    x = tokens(5)
    x[0], x[1, 0], x[2, 1] = -1, V, 2**31 - 1
    given = {"beside": x.cuda(), "int32": x.cuda().int(), "host": x}[place]
    got = loss_and_grads(model("cuda", True, dtype), given)
    want = loss_and_grads(model("cpu", True, dtype), x)
    for a, b in zip(got, want):
        assert a.dtype == b.dtype
        close(a, b, dtype)


def test_trained_classifier_is_traced():
    m, x = model("cuda", True), tokens().cuda()
    traced = torch.jit.trace(Keep1(m), (x,))
    for seed in (0, 1, 2):
        x = tokens(seed).cuda()
        x[seed] = V
        assert torch.equal(traced(x), m(x, 1.0))
    g, = torch.autograd.grad(traced(x).square().sum(), m.W)
    w, = torch.autograd.grad(m(x, 1.0).square().sum(), m.W)
    assert torch.equal(g, w)
