"""GPU: the lookup's gradient on both sides of the sizes where the length of its
pieces changes, against 64 bits.  The bound is that of any order of the sum: c
fp32 terms, the scale and the store (u = 2^-24, h = half a step of the type)
|err| <= 1.01 (c + 1) u S + h (|g| + 1.01 (c + 1) u S) + t, S = sum |x|."""
import numpy as np
import pytest
import torch

from gene2vec_amd import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("n,D", [(255, 16), (256, 16), (257, 16), (4095, 4096), (4096, 4096),
                                 (4097, 4096), (16383, 4096), (16385, 4096), (83886, 200),
                                 (83887, 200), (262143, 64), (262144, 64)])
@pytest.mark.parametrize("kind", ["zipf", "two"])
def test_sums_at_the_borders_of_the_piece_length(n, D, kind):
    V = 700
    rng = np.random.RandomState(n)
    ids = (np.exp(rng.rand(n) * np.log(V + 1)).astype(np.int64) - 1).clip(0, V - 1)
    if kind == "two":
        ids = rng.randint(0, 2, n) * (V - 1)
    ids = torch.from_numpy(ids).cuda()
    gen = torch.Generator(device="cuda").manual_seed(n)
    dy = torch.randn(n, D, device="cuda", generator=gen).bfloat16()
    g = ops.embedding_lookup_grad(dy, ids, V, dtype=torch.float32)
    assert torch.equal(g, ops.embedding_lookup_grad(dy, ids, V, dtype=torch.float32))
    u, h = 2.0**-24, 2.0**-24
    c = torch.bincount(ids, minlength=V).double()[:, None]
    order, lengths = torch.argsort(ids, stable=True), c[:, 0].long()
    for a in range(0, D, 512):
        x = dy[:, a:a + 512].double()
        ref = torch.segment_reduce(x[order], "sum", lengths=lengths, axis=0, initial=0)
        S = torch.segment_reduce(x[order].abs(), "sum", lengths=lengths, axis=0, initial=0)
        acc = 1.01 * (c + 1) * u * S
        err = (g[:, a:a + 512].double() - ref).abs()
        assert bool((err <= acc + h * (ref.abs() + acc) + 2.0**-150).all()), float(err.max())
