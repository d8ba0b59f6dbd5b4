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
