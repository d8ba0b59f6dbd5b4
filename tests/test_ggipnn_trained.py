"""CPU: what the classifier makes of tokens outside its table."""
import numpy as np
import pytest
import torch

from gene2vec_amd import ggipnn as G

V, D = 9, 4


def model(trained, dtype=torch.float32):
    emb = np.random.RandomState(0).randn(V, D).astype(np.float32)
    return G.build_model(V, emb, D, "cpu", torch.Generator().manual_seed(3),
                         train_embedding=trained).to(dtype)


def test_frozen_table_is_indexed():
    m = model(False)
    x = torch.tensor([[-1, 2], [3, 4]])
    assert torch.equal(m(x, 1.0), m(x % V, 1.0))
    with pytest.raises(IndexError):
        m(torch.tensor([[V, 0]]), 1.0)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float64, torch.bfloat16])
@pytest.mark.parametrize("idt", [torch.int64, torch.int32])
def test_trained_table_has_zero_rows_for_other_tokens(dtype, idt):
    m = model(True, dtype)
    x = torch.tensor([[-1, 2], [V, 4], [2, 2**31 - 1], [2, 8]])
    ext = model(True, dtype)
    with torch.no_grad():  # the same with a row of zeros for them
        ext.W = torch.nn.Parameter(torch.cat([m.W, m.W.new_zeros(1, D)]))
    inside = torch.where((x >= 0) & (x < V), x, V)
    y, want = m(x.to(idt), 1.0), ext(inside, 1.0)
    assert y.dtype == dtype and torch.equal(y, want)
    c = torch.randn_like(y)
    g, = torch.autograd.grad(y, m.W, c)
    w, = torch.autograd.grad(want, ext.W, c)
    assert torch.equal(g, w[:V])
    assert g.abs().sum(1).gt(0).tolist() == [v in (2, 4, 8) for v in range(V)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16, torch.float64])
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_clipped_gradients_of_every_type(dtype, device):
    """factor and product round once each in fp32 (u = 2^-24; fp64: 2^-53), then
    the store (h = eps / 2 of the type): |err| <= (2 u + h) |x| (1 + 2^-8) + the
    half of the smallest subnormal"""
    gen = torch.Generator().manual_seed(1)
    m = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(s, dtype=dtype, device=device))
                                for s in ((300, 7), (40,), ())])
    for p in m:
        p.grad = torch.randn(p.shape, generator=gen).to(device, dtype)
    before = [p.grad.double().cpu().clone() for p in m]
    n = float(torch.sqrt(sum(g.square().sum() for g in before)))
    clip = n / 3.7
    got = G.clip_gradients_(m, clip)
    assert float(got) == pytest.approx(n, rel=2**-24 * (1 + 2**-8))
    i = torch.finfo(dtype)
    bound = (2 * (2**-53 if dtype == torch.float64 else 2**-24) + i.eps / 2) * (1 + 2**-8)
    for p, g in zip(m, before):
        want = g * (clip / n)
        # the norm's own sum in fp64: off by at most 2141 * 2^-53 of it
        tol = want.abs() * (bound + 2141 * 2**-53) + i.smallest_normal * i.eps / 2
        assert bool(((p.grad.double().cpu() - want).abs() <= tol).all())


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
def test_clipped_gradients_of_mixed_types(device):
    m = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros(3, dtype=t, device=device))
                                for t in (torch.float32, torch.float64, torch.bfloat16)])
    for p in m:
        p.grad = torch.full_like(p, 2.0)
    assert float(G.clip_gradients_(m, 3.0)) == 6.0
    assert all(torch.equal(p.grad, torch.ones_like(p)) for p in m)
