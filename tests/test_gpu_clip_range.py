"""GPU: clipping where the factor leaves fp32's normal numbers (a norm of more
than 2^126 times the bound), against 64 bits.

u = 2^-24, h = half a step of the type stored, t = half its smallest subnormal:
the factor and the product round once each to 24 bits, then the store; an fp32
result below the normal numbers rounds once more on its way there:
|err| <= (2 u + h)(1 + 2^-8) |x| + t + 2^-150."""
import math

import pytest
import torch

from gene2vec_amd import ggipnn as G
from gene2vec_amd import ops

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def check(outs, ts, clip):
    """powers of ten apart, the norm in units of the largest element: nothing
    overflows or falls below fp64"""
    top = max(float(t.double().abs().max()) for t in ts)
    n = top * math.sqrt(sum(float((t.double() / top).square().sum()) for t in ts))
    for o, t in zip(outs, ts):
        i = torch.finfo(t.dtype)
        want = t.double().cpu() * (clip / n)
        tol = (want.abs() * (2 * 2**-24 + i.eps / 2) * (1 + 2**-8)
               + i.smallest_normal * i.eps / 2 + 2.0**-150)
        err = (o.double().cpu() - want).abs()
        assert bool((err <= tol).all()), (float(err.max()), float(want.abs().max()))


def cases():
    gen = torch.Generator().manual_seed(2)
    big = torch.randn(9000, generator=gen).clamp(-3, 3) * 1e38
    small = torch.randn(31, generator=gen)
    yield [big], [1.0, 1e-5, 1e-20, 1e-36, 1e-40, 1e-300, 5e-324]
    yield [torch.full((4,), 3e38), small, big[:5].to(BF16)], [100.0, 1.0, 1e-10]
    yield [small * 1e-3, (small * 1e20).to(BF16)], [1e-18, 1e-19, 1e-30]
    yield [(small * 1e4).to(F16), small], [1e-33, 1e-36]


@pytest.mark.parametrize("case", range(4))
def test_factor_below_the_normal_numbers_on_the_cpu(case):
    ts, clips = list(cases())[case]
    for clip in clips:
        m = torch.nn.ParameterList([torch.nn.Parameter(torch.zeros_like(t)) for t in ts])
        for p, t in zip(m, ts):
            p.grad = t.clone()
        G.clip_gradients_(m, clip)
        check([p.grad for p in m], ts, clip)


@pytest.mark.gpu
@pytest.mark.parametrize("case", range(4))
def test_factor_below_the_normal_numbers(case):
    ts, clips = list(cases())[case]
    ts = [t.cuda() for t in ts]
    for clip in clips:
        outs, norm = ops.clip_by_global_norm(ts, clip)
        check(outs, ts, clip)
        same = [t.clone() for t in ts]
        assert torch.equal(ops.clip_by_global_norm_(same, clip), norm)
        assert all(torch.equal(a, b) for a, b in zip(same, outs))


@pytest.mark.gpu
def test_a_norm_beyond_fp32_is_returned_as_infinity_and_clipped():
    t = torch.full((5000,), 3e38, device="cuda")
    outs, norm = ops.clip_by_global_norm([t], 1.0)
    assert float(norm) == math.inf
    assert bool(outs[0].isfinite().all())
    check(outs, [t], 1.0)
    t[4999] = math.inf
    outs, norm = ops.clip_by_global_norm([t], 1.0)
    assert float(norm) == math.inf and bool(outs[0].isnan().all())
