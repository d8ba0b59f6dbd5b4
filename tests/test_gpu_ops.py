"""GPU: the tensor operators (embedding lookup and its gradient, global norm
and clipping) against their formulas in 64 bits.

Bounds, u = 2^-24 (half a step of fp32), h = half a step of the type stored
(finfo.eps / 2), t = half its smallest subnormal:
  lookup  one fp32 product and one rounding: |err| <= (u + h) |y| + t
  grad    a sum of c fp32 terms in any order is off by at most
          (c - 1) u sum|x| (1 + O(c u)), the scale and the store round once
          each: |err| <= (c + 1) u S + h (|g| + (c + 1) u S) + t, with
          S = |scale| sum|x|; 1.01 covers the second-order terms (c u < 2^-8)
  norm    fp64 throughout, rounded once: |err| <= u n (1 + 2^-20)
  clip    factor and product round once, then the store:
          |err| <= (2 u + h)(1 + 2^-20) |x| + t
"""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from gene2vec_amd import _native as N
from gene2vec_amd import ggipnn as G
from gene2vec_amd import ops

pytestmark = pytest.mark.gpu

U = 2.0**-24
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def half(t):
    return torch.finfo(t).eps / 2


def tiny(t):
    return float(torch.finfo(t).smallest_normal) * torch.finfo(t).eps / 2


def make_ids(kind, V, n, dtype, seed):
    rng = np.random.Generator(np.random.PCG64(seed))
    if kind == "zipf":
        ids = np.exp(rng.random(n) * math.log(V + 1)).astype(np.int64) - 1
        ids = rng.permutation(V)[ids.clip(0, V - 1)]
    elif kind == "same":
        ids = np.full(n, V - 1, np.int64)
    elif kind == "two":
        ids = np.where(rng.random(n) < 0.5, 0, V - 1)
    elif kind == "skew":  # half the tokens one row, a tenth its bucket's others
        u = rng.random(n)
        ids = np.where(u < 0.5, 7 % V, np.where(u < 0.6, rng.integers(0, V, n) // 256 * 256 + 7,
                                                rng.integers(0, V, n)))
        ids = ids.clip(0, V - 1)
    elif kind == "sorted":
        ids = np.sort(rng.integers(0, V, n))
    else:
        ids = rng.integers(0, V, n)
        if kind == "absent" and n:
            top = 2**31 - 1 if dtype == torch.int32 else 2**62
            far = np.array([-1, V, top, -top, -2**31] + ([2**32, -2**32] if dtype == torch.int64
                                                         else []))
            ids = np.where(rng.random(n) < 0.4, far[rng.integers(0, len(far), n)], ids)
    return torch.from_numpy(ids.astype(np.int64)).to(dtype)


def check_lookup(y, w, ids, scale, dtype):
    V, D = w.shape
    i = ids.long().cpu().reshape(-1)
    there = (i >= 0) & (i < V)
    ref = torch.where(there[:, None], w.double().cpu()[i.clamp(0, V - 1)] * scale, 0.0)
    assert y.dtype == dtype and tuple(y.shape) == tuple(ids.shape) + (D,)
    err = (y.double().cpu().reshape(-1, D) - ref).abs()
    s32 = float(np.float32(scale))  # the scale itself is held in fp32
    bound = (2 * U if s32 != scale else U) + half(dtype) * (1 + 4 * U)
    assert bool((err <= ref.abs() * bound + tiny(dtype)).all()), float(err.max())


def grad_reference(dy, ids, V, scale, pad):
    D = dy.shape[-1]
    i = ids.long().cpu().reshape(-1)
    x = dy.double().cpu().reshape(-1, D)
    there = (i >= 0) & (i < V)
    if pad is not None:
        there &= i != pad
    i, x = i[there], x[there]
    g = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i, x) * scale
    S = torch.zeros(V, D, dtype=torch.float64).index_add_(0, i, x.abs()) * abs(scale)
    c = torch.bincount(i, minlength=V).double()[:, None]
    return g, S, c


def check_grad(g, dy, ids, V, scale=1.0, pad=None):
    ref, S, c = grad_reference(dy, ids, V, scale, pad)
    assert tuple(g.shape) == tuple(ref.shape) and g.is_contiguous()
    h = half(g.dtype)
    extra = 1 if float(np.float32(scale)) != scale else 0  # the scale's own rounding
    acc = 1.01 * (c + 1 + extra) * U * S
    err = (g.double().cpu() - ref).abs()
    ok = err <= acc + h * (ref.abs() + acc) + tiny(g.dtype)
    assert bool(ok.all()), (int((~ok).sum()), float(err.max()))
    assert bool((g.cpu()[(c == 0).squeeze(1)] == 0).all())


# ---- lookup ------------------------------------------------------------------------------
@pytest.mark.parametrize("V,D,n,kind", [
    (1, 1, 1, "uniform"), (24447, 200, 1, "uniform"), (5, 3, 7, "absent"), (300, 7, 65, "zipf"),
    (1000, 8, 1000, "absent"), (777, 301, 999, "zipf"), (12472, 200, 256, "uniform"),
    (64, 4096, 33, "absent"), (50, 8193, 5, "uniform"), (2, 16, 100003, "same")])
@pytest.mark.parametrize("table,out", [(F32, F32), (BF16, BF16), (F16, F32), (F32, BF16),
                                       (BF16, F16), (F16, F16)])
def test_lookup(V, D, n, kind, table, out):
    gen = torch.Generator(device="cuda").manual_seed(V + D + n)
    w = torch.randn(V, D, device="cuda", generator=gen).to(table)
    for idt, scale in ((torch.int64, 1.0), (torch.int32, math.sqrt(D))):
        ids = make_ids(kind, V, n, idt, n).cuda()
        y = ops.embedding_lookup(w, ids, scale=scale, dtype=out)
        check_lookup(y, w, ids, scale, out)
    assert torch.equal(ops.embedding_lookup(w, torch.arange(V, device="cuda")), w)


def test_lookup_shapes_strides_and_nothing():
    base = torch.randn(40, 37, device="cuda")
    ids = torch.randint(0, 40, (6, 5, 4), device="cuda")
    for w in (base[:, 3:20], base[::3, 1:], base[7:8, :5], base[:, :1], base.t()[:, 5:6]):
        i = ids % w.shape[0]
        check_lookup(ops.embedding_lookup(w, i, 0.1), w, i, 0.1, F32)
        t = i.transpose(0, 2)
        check_lookup(ops.embedding_lookup(w, t), w, t, 1.0, F32)
    h = torch.randn(41 * 13 + 1, device="cuda").to(BF16)[1:].view(41, 13)  # 2-byte alignment
    i = ids % 41
    check_lookup(ops.embedding_lookup(h, i, 3.0, dtype=F32), h, i, 3.0, F32)
    assert ops.embedding_lookup(base, ids[:0]).shape == (0, 5, 4, 37)
    assert torch.equal(ops.embedding_lookup(base, ids[0, 0, 0]), base[ids[0, 0, 0]])


def test_lookup_keeps_special_values():
    w = torch.tensor([[math.inf, -math.inf, math.nan, -0.0]], device="cuda")
    y = ops.embedding_lookup(w, torch.tensor([0, -1], device="cuda"), 2.0).cpu()
    assert y[0, 0] == math.inf and y[0, 1] == -math.inf and y[0, 2].isnan()
    assert math.copysign(1, y[0, 3]) == -1 and bool((y[1] == 0).all())


@pytest.mark.parametrize("t", TYPES)
def test_subnormal_values_are_kept(t):
    i = torch.finfo(t)
    w = torch.tensor([[i.tiny / 2, -i.tiny / 4, i.tiny, i.smallest_normal * i.eps, i.max, i.min,
                       1.0, 0.0, -i.tiny / 8]] * 3, dtype=F32 if t == F32 else t, device="cuda")
    ids = torch.tensor([0, 1, 2, 2, 0], device="cuda")
    assert torch.equal(ops.embedding_lookup(w, ids), w[ids])
    g = ops.embedding_lookup_grad(w[ids[:3]], ids[:3], 4)  # one token a row: sums of one
    assert torch.equal(g[:3], w) and not g[3].any()
    out, _ = ops.clip_by_global_norm([w[:, :4].contiguous()], 1e9)
    assert torch.equal(out[0], w[:, :4])


# ---- the gradient ------------------------------------------------------------------------
GRAD = [(1, 1, 1, "uniform"), (1, 5, 200, "same"), (2, 3, 129, "two"), (10, 8, 0, "uniform"),
        (24447, 200, 1, "uniform"), (12472, 200, 256, "uniform"), (255, 9, 63, "zipf"),
        (256, 64, 64, "absent"), (257, 65, 65, "sorted"), (1000, 301, 1025, "zipf"),
        (24447, 200, 4096, "zipf"), (60000, 12, 5000, "absent"), (131, 1030, 777, "same"),
        (24447, 40, 70001, "zipf"), (300000, 4, 66000, "uniform"), (3, 130, 50000, "two"),
        (70000, 33, 300007, "zipf"), (512, 16, 262144, "absent"), (700, 4100, 500, "zipf"),
        (24447, 20, 70001, "skew"), (300000, 8, 70001, "skew"), (256, 16, 20000, "same"),
        (2, 64, 300000, "two"), (262144, 4, 40000, "skew"), (262145, 4, 40000, "skew"),
        (5000, 2, 1100000, "skew"), (24447, 16, 16384, "skew"), (24447, 16, 16385, "skew")]


@pytest.mark.parametrize("V,D,n,kind", GRAD)
@pytest.mark.parametrize("ty,tg", [(F32, F32), (BF16, F32), (BF16, BF16), (F16, F16)])
def test_grad(V, D, n, kind, ty, tg):
    gen = torch.Generator(device="cuda").manual_seed(V + D + n)
    dy = torch.randn(n, D, device="cuda", generator=gen).to(ty)
    idt = torch.int32 if (V + n) % 2 else torch.int64
    ids = make_ids(kind, V, n, idt, n + 1).cuda()
    g = ops.embedding_lookup_grad(dy, ids, V, dtype=tg)
    assert g.dtype == tg
    check_grad(g, dy, ids, V)
    assert torch.equal(g, ops.embedding_lookup_grad(dy, ids, V, dtype=tg))


@pytest.mark.parametrize("n", [5, 64, 65, 300, 9000, 70000, 140000])
def test_grad_scale_and_padding(n):
    V, D = 500, 24
    dy = torch.randn(n, D, device="cuda")
    ids = make_ids("zipf", V, n, torch.int64, n).cuda()
    hot = int(torch.bincount(ids.cpu()).argmax())
    for pad in (None, 0, hot, V - 1):
        for scale in (math.sqrt(D), -0.5, 0.0):
            g = ops.embedding_lookup_grad(dy, ids, V, scale, pad)
            check_grad(g, dy, ids, V, scale, pad)
            assert pad is None or not g[pad].any()


def test_grad_padding_hides_its_values():
    """NaN and infinity at padding and absent tokens reach no row"""
    ids = torch.tensor([3, 0, -1, 9, 3, 0], device="cuda")
    dy = torch.ones(6, 5, device="cuda")
    dy[[1, 5]], dy[2], dy[3] = math.nan, math.inf, -math.inf
    g = ops.embedding_lookup_grad(dy, ids, 9, padding_idx=0).cpu()
    want = torch.zeros(9, 5)
    want[3] = 2.0
    assert torch.equal(g, want)
    assert ops.embedding_lookup_grad(dy, ids, 9)[0].isnan().all()


@pytest.mark.parametrize("n", [100, 3000, 80000])
def test_grad_strides(n):
    V = 90
    ids = make_ids("zipf", V, 2 * n, torch.int32, 5).cuda().reshape(n, 2)
    wide = torch.randn(n, 2, 50, device="cuda")
    for dy in (wide, wide[:, :, 3:20], wide.flip(0), wide.transpose(0, 2).contiguous().transpose(
            0, 2), wide[:1].expand(n, 2, 50), wide[:, :, :1], torch.ones((), device="cuda").expand(
                n, 2, 6), wide.to(BF16)[:, :, 1:]):
        check_grad(ops.embedding_lookup_grad(dy, ids, V), dy, ids, V)
    t = ids.t()
    dy = wide.transpose(0, 1)
    check_grad(ops.embedding_lookup_grad(dy, t, V), dy, t, V)
    neg = torch._neg_view(wide)
    check_grad(ops.embedding_lookup_grad(neg.clone(), ids, V), -wide, ids, V)
    for call in (lambda: ops.embedding_lookup_grad(neg, ids, V), lambda: ops.global_norm([neg])):
        with pytest.raises(ValueError, match="negated"):
            call()


def test_offsets_past_32_bits():
    """a table, a gradient and activations of more than 2^31 elements"""
    V, D = 530000, 4100
    w = torch.zeros(V, D, dtype=BF16, device="cuda")
    ids = torch.tensor([V - 1, 0, 524288, V - 1, V - 2], device="cuda")
    w[ids[2:]] = torch.randn(3, D, device="cuda").to(BF16)
    y = ops.embedding_lookup(w, ids)
    assert torch.equal(y, w[ids])
    dy = torch.randn(5, D, device="cuda").to(BF16)
    g = ops.embedding_lookup_grad(dy, ids, V)
    rows = torch.tensor([0, 524288, V - 2, V - 1])
    local = torch.tensor([3, 0, 1, 3, 2], device="cuda")
    check_grad(g[rows.cuda()].contiguous(), dy, local, 4)
    g[rows.cuda()] = 0
    assert not any(bool(part.any()) for part in g.split(100000))
    del g
    many = torch.arange(V, device="cuda") % 7
    y = ops.embedding_lookup(w[:7], many)
    assert torch.equal(y[-1], w[(V - 1) % 7]) and not y[:, ::512].any()
    y.fill_(1)
    g = ops.embedding_lookup_grad(y, many, 8, dtype=F32)
    want = torch.bincount(many.cpu(), minlength=8).float()[:, None].expand(8, D)
    assert torch.equal(g.cpu(), want)  # whole numbers below 2^24: exact in any order


def test_more_rows_than_a_list_entry_holds():
    """over 2^30 rows the tokens are sorted without the packed lists"""
    V = 2**30 + 300
    for ids in ([], [V - 1, 3, 2**30 + 7, 3, 255, -1, V]):
        ids = torch.tensor(ids, dtype=torch.int64, device="cuda")
        dy = torch.arange(1.0, len(ids) + 1, device="cuda")[:, None].to(BF16)
        g = ops.embedding_lookup_grad(dy, ids, V)
        if len(ids):
            for row, want in ((V - 1, 1), (3, 6), (2**30 + 7, 3), (255, 5)):
                assert float(g[row]) == want
                g[row] = 0
        assert not any(bool(part.any()) for part in g.split(2**28))
        del g


# ---- autograd, streams, graphs -----------------------------------------------------------
def test_autograd_matches_formula_and_differences():
    V, D = 30, 6
    w = torch.randn(V, D, device="cuda", requires_grad=True)
    ids = torch.randint(-1, V, (8, 3), device="cuda")
    c = torch.randn(8, 3, D, device="cuda")
    y = ops.embedding_lookup(w, ids, scale=0.5, padding_idx=4)
    (y * c).sum().backward()
    check_grad(w.grad, c, ids, V, 0.5, 4)
    # the lookup is linear: a difference quotient over a whole step of 1 is the
    # derivative, up to the roundings of the 24 fp32 products and their sum
    with torch.no_grad():
        for v, d in ((0, 0), (7, 5), (29, 3)):
            e = torch.zeros_like(w)
            e[v, d] = 1.0
            f = [float((ops.embedding_lookup(w + s * e, ids, 0.5).double() * c).sum())
                 for s in (0.5, -0.5)]
            # each y is off by at most 2 u |y|, |y| <= 0.5 (|w| + 1)
            tol = 4 * U * float((0.5 * (w.abs().max() + 1) * c.abs()).sum())
            assert abs((f[0] - f[1]) - float(w.grad[v, d])) <= tol + 30 * U
    w.grad = None
    ops.embedding_lookup(w, ids, dtype=BF16).sum().backward()  # a broadcast gradient
    check_grad(w.grad, torch.ones(8, 3, D, device="cuda"), ids, V)
    y = ops.embedding_lookup(w, ids)
    g, = torch.autograd.grad(y.square().sum(), w, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()  # once only
    ids[0] = 0
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()  # the saved tokens changed


def test_two_lookups_of_one_table_accumulate():
    w = torch.randn(50, 16, device="cuda", requires_grad=True)
    a = torch.randint(0, 50, (40,), device="cuda")
    b = torch.randint(0, 50, (70,), device="cuda")
    ca, cb = torch.randn(40, 16, device="cuda"), torch.randn(70, 16, device="cuda")
    ((ops.embedding_lookup(w, a) * ca).sum() + (ops.embedding_lookup(w, b) * cb).sum()).backward()
    check_grad(w.grad, torch.cat([ca, cb]), torch.cat([a, b]), 50)


def test_inference_mode():
    w = torch.randn(20, 8, device="cuda", requires_grad=True)
    ids = torch.arange(20, device="cuda")
    with torch.inference_mode():
        y = ops.embedding_lookup(w, ids)
        outs, norm = ops.clip_by_global_norm([y], 0.1)
        ops.clip_by_global_norm_([y], 0.1)
        assert torch.equal(outs[0], y) and float(norm) > 0.1
    assert y.is_inference() and not y.requires_grad
    assert float(ops.global_norm([y])) > 0
    with pytest.raises(ValueError, match="inference"):
        ops.clip_by_global_norm_([y], 0.1)


def test_grad_modes_and_a_computed_table():
    w = torch.randn(20, 8, device="cuda")
    ids = torch.arange(6, device="cuda")
    assert not ops.embedding_lookup(w, ids).requires_grad
    w.requires_grad_(True)
    with torch.no_grad():
        assert not ops.embedding_lookup(w, ids).requires_grad
    y = ops.embedding_lookup(w * 2.0, ids)  # a table that is no leaf
    (g,) = torch.autograd.grad(y.sum(), w)
    want = torch.zeros(20, 8)
    want[:6] = 2.0
    assert torch.equal(g.cpu(), want)


@pytest.mark.parametrize("n", [200, 6000, 100000])
def test_on_another_stream(n):
    V, D = 3000, 64
    w = torch.randn(V, D, device="cuda")
    ids = make_ids("zipf", V, n, torch.int64, 3).cuda()
    dy = torch.randn(n, D, device="cuda")
    want = ops.embedding_lookup(w, ids), ops.embedding_lookup_grad(dy, ids, V)
    want += (ops.global_norm([dy, w]),)
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append((ops.embedding_lookup(w, ids), ops.embedding_lookup_grad(dy, ids, V),
                        ops.global_norm([dy, w])))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(x, y) for x, y in zip(g, want))


def test_two_threads_at_once():
    import threading
    V, D = 2000, 48
    table = torch.randn(V, D, device="cuda")
    work = [(make_ids("zipf", V, n, torch.int64, n).cuda(), torch.randn(n, D, device="cuda"))
            for n in (300, 20000, 5, 70000)]
    want = [ops.embedding_lookup_grad(dy, ids, V) for ids, dy in work]
    norms = [ops.global_norm([dy]) for _, dy in work]
    torch.cuda.synchronize()
    got, bad = {}, []

    def go(k):
        try:
            ids, dy = work[k]
            w = table.detach().requires_grad_(True)
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(20):
                    g, = torch.autograd.grad(ops.embedding_lookup(w, ids), w, dy)
                    out, norm = ops.clip_by_global_norm([g, dy], 1.0)
                    last = g, ops.global_norm([dy])
                torch.cuda.current_stream().synchronize()
            got[k] = last
        except BaseException as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=go, args=(k,)) for k in range(4)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    assert not bad, bad
    for k in range(4):
        assert torch.equal(got[k][0], want[k]) and torch.equal(got[k][1], norms[k])


@pytest.mark.parametrize("n", [100, 5000, 100000])
def test_captured_and_replayed(n):
    """two graphs of the same calls, replayed in turn with other inputs and
    eager calls in between"""
    V, D = 2000, 40
    w = torch.randn(V, D, device="cuda")
    state = []
    for k in range(2):
        ids = torch.zeros(n, dtype=torch.int64, device="cuda")
        dy = torch.zeros(n, D, device="cuda")
        g = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(g):
            y = ops.embedding_lookup(w, ids, 1.5)
            d = ops.embedding_lookup_grad(dy, ids, V, 1.5, k)
            clipped, norm = ops.clip_by_global_norm([d, dy], 0.5)
        state.append((g, ids, dy, y, d, clipped, norm))
    for r in range(4):
        for k, (g, ids, dy, *_) in enumerate(state):
            ids.copy_(make_ids(("zipf", "absent", "same", "uniform")[r], V, n, torch.int64,
                               10 * r + k))
            dy.normal_()
            g.replay()
        e = ops.embedding_lookup_grad(state[0][2], state[0][1], V, 1.5, 0)
        torch.cuda.synchronize()
        assert torch.equal(e, state[0][4])
        for k, (g, ids, dy, y, d, clipped, norm) in enumerate(state):
            assert torch.equal(y, ops.embedding_lookup(w, ids, 1.5))
            assert torch.equal(d, ops.embedding_lookup_grad(dy, ids, V, 1.5, k))
            want, wn = ops.clip_by_global_norm([d, dy], 0.5)
            assert torch.equal(norm, wn)
            assert all(torch.equal(a, b) for a, b in zip(clipped, want))


# ---- norm and clipping -------------------------------------------------------------------
def norm64(ts):
    return math.sqrt(sum(float(t.detach().cpu().double().square().sum()) for t in ts))


def check_clip(outs, ts, n, clip):
    f = clip / max(n, clip)
    for o, t in zip(outs, ts):
        assert o.dtype == t.dtype and o.shape == t.shape
        ref = t.detach().cpu().double() * f
        err = (o.cpu().double() - ref).abs()
        bound = ref.abs() * (2 * U + half(t.dtype)) * (1 + 2**-20) + tiny(t.dtype)
        assert bool((err <= bound).all()), float(err.max())


def tensors(sizes, types, seed=0, scale=1.0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=gen) * scale).to(types[k % len(types)])
            for k, s in enumerate(sizes)]


@pytest.mark.parametrize("sizes", [
    [()], [1], [0, 5, 0], [3, 0], [8191], [8192], [8193], [(12472, 200), (400, 100), 100, (10, 2)],
    [(k * 37) % 501 for k in range(300)], [1] * 129, [5] * 128, [2000003, 7, 1000001],
    [100] * 1000 + [300001]])
@pytest.mark.parametrize("types", [[F32], [BF16], [F16], [F32, BF16, F16]])
def test_norm_and_clip(sizes, types):
    ts = tensors(sizes, types, len(sizes))
    n = norm64(ts)
    got = ops.global_norm(ts)
    assert got.shape == () and got.dtype == F32
    assert abs(float(got) - n) <= n * U * (1 + 2**-20)
    for clip in (max(n, 1e-3) * 0.37, max(n, 1e-3) * 3):
        keep = [t.clone() for t in ts]
        outs, norm = ops.clip_by_global_norm(ts, clip)
        assert torch.equal(norm, got)
        check_clip(outs, ts, n, clip)
        assert all(torch.equal(a, b) for a, b in zip(ts, keep))
        into = [torch.empty_like(t) for t in ts]
        back, _ = ops.clip_by_global_norm(ts, clip, out=into)
        assert all(a is b for a, b in zip(back, into))
        assert all(torch.equal(a, b) for a, b in zip(into, outs))
        assert torch.equal(ops.clip_by_global_norm_(keep, clip), got)
        assert all(torch.equal(a, b) for a, b in zip(keep, outs))
        if clip > n:
            assert all(torch.equal(a, b) for a, b in zip(outs, ts))


def test_norm_of_odd_views():
    flat = torch.randn(100000, device="cuda").to(BF16)
    ts = [flat[1:8], flat[9:9000], flat[9001:50001].view(40, 1025).t(), flat[50003:]]
    n = norm64(ts)
    assert abs(float(ops.global_norm(ts)) - n) <= n * U * (1 + 2**-20)
    outs, _ = ops.clip_by_global_norm(ts, 1.0)
    check_clip(outs, ts, n, 1.0)
    kept = flat.clone()
    ops.clip_by_global_norm_(ts, 1.0)
    check_clip(ts, [kept[1:8], kept[9:9000], kept[9001:50001].view(40, 1025).t(), kept[50003:]],
               n, 1.0)
    for gap in (0, 8, 9000, 50001, 50002):
        assert flat[gap] == kept[gap]  # what lies between the views is left alone


def test_norm_range_and_special_values():
    big, small = torch.full((1000,), 1e30, device="cuda"), torch.full((7,), 1e-30, device="cuda")
    n = norm64([big])
    assert abs(float(ops.global_norm([big, small])) - n) <= n * U * (1 + 2**-20)
    n = norm64([small])
    assert abs(float(ops.global_norm([small])) - n) <= n * U * (1 + 2**-20)
    outs, _ = ops.clip_by_global_norm([big, small], 1.0)
    check_clip(outs, [big, small], norm64([big, small]), 1.0)
    zero = torch.zeros(50, device="cuda")
    zero[0] = -0.0
    outs, norm = ops.clip_by_global_norm([zero], 1.0)
    assert float(norm) == 0 and torch.equal(outs[0], zero)
    assert math.copysign(1, float(outs[0][0])) == -1
    top = torch.full((4,), 3e38, device="cuda")  # the norm is beyond fp32, the sum is not
    assert float(ops.global_norm([top])) == math.inf
    outs, _ = ops.clip_by_global_norm([top], 100.0)  # a factor of 1.7e-37: still normal
    check_clip(outs, [top], norm64([top]), 100.0)
    for bad in (math.inf, -math.inf, math.nan):
        x, y = torch.ones(9000, device="cuda"), torch.ones(3, device="cuda").to(F16)
        x[8999] = bad
        norm = ops.clip_by_global_norm_([y, x], 1.0)
        assert not math.isfinite(float(norm)) and x.isnan().all() and y.isnan().all()


def test_norm_past_32_bits():
    t = torch.zeros(2**31 + 4099, dtype=BF16, device="cuda")
    t[-1], t[2**31 - 1], t[2**31], t[0] = 3.0, 4.0, 12.0, 84.0
    assert float(ops.global_norm([t])) == 85.0  # exact: 9 + 16 + 144 + 7056 = 7225
    ops.clip_by_global_norm_([t], 42.5)
    assert [float(t[k]) for k in (-1, 2**31 - 1, 2**31, 0)] == [1.5, 2.0, 6.0, 42.0]
    t[-1] = t[2**31 - 1] = t[2**31] = t[0] = 0
    assert not any(bool(p.any()) for p in t.split(2**28))


def test_clip_tells_autograd_and_refuses():
    w = torch.randn(6, 4, device="cuda", requires_grad=True)
    (w.square().sum() / 2).backward()
    v = w.grad._version
    ops.clip_by_global_norm_([w.grad, None], 0.1)
    assert w.grad._version > v
    x, y = torch.ones(8, device="cuda"), torch.ones(8, device="cuda")
    outs, _ = ops.clip_by_global_norm([x, None, y], 1.0)
    assert outs[1] is None and len(outs) == 3
    with torch.no_grad():
        assert float(ops.global_norm([w])) > 0
    z = torch.ones(8, 8, device="cuda")
    for call in (
            lambda: ops.global_norm([w]), lambda: ops.clip_by_global_norm_([w], 1.0),
            lambda: ops.global_norm([x.double()]), lambda: ops.global_norm([x, x.cpu()]),
            lambda: ops.global_norm([z[:, :3]]), lambda: ops.global_norm([z[::2].t()]),
            lambda: ops.global_norm(z), lambda: ops.global_norm([x[:1].expand(8)]),
            lambda: ops.global_norm([x.to_sparse()]),
            lambda: ops.clip_by_global_norm_([x, x], 1.0),
            lambda: ops.clip_by_global_norm_([x, x[4:]], 1.0),
            lambda: ops.clip_by_global_norm([x, y], 1.0, out=[y, x]),
            lambda: ops.clip_by_global_norm([x], 1.0, out=[x[:4]]),
            lambda: ops.clip_by_global_norm([x], 1.0, out=[]),
            lambda: ops.clip_by_global_norm([x], 1.0, out=[y.to(BF16)]),
            lambda: ops.clip_by_global_norm([z], 1.0, out=[torch.ones(8, 8, device="cuda").t()]),
            lambda: ops.clip_by_global_norm([x], 0.0),
            lambda: ops.clip_by_global_norm([x], math.inf)):
        with pytest.raises(ValueError):
            call()
    assert torch.equal(x, torch.ones(8, device="cuda"))


def test_lookup_refuses():
    w = torch.randn(6, 4, device="cuda")
    i = torch.zeros(3, dtype=torch.int64, device="cuda")
    dy = torch.randn(3, 4, device="cuda")
    for call in (
            lambda: ops.embedding_lookup(w, i.cpu()), lambda: ops.embedding_lookup(w, i.short()),
            lambda: ops.embedding_lookup(w, i.float()), lambda: ops.embedding_lookup(w.double(), i),
            lambda: ops.embedding_lookup(w[0], i), lambda: ops.embedding_lookup(w[:0], i),
            lambda: ops.embedding_lookup(w[:, ::2], i), lambda: ops.embedding_lookup(w.t(), i),
            lambda: ops.embedding_lookup(w[:1].expand(6, 4), i),
            lambda: ops.embedding_lookup(w, i, math.inf), lambda: ops.embedding_lookup(w, i, 1e39),
            lambda: ops.embedding_lookup(w, i, padding_idx=6),
            lambda: ops.embedding_lookup(w, i, padding_idx=-1),
            lambda: ops.embedding_lookup(w, i, padding_idx=1.5),
            lambda: ops.embedding_lookup(w, i, dtype=torch.float64),
            lambda: ops.embedding_lookup_grad(dy[:2], i, 6),
            lambda: ops.embedding_lookup_grad(dy[:, :0], i, 6),
            lambda: ops.embedding_lookup_grad(dy.double(), i, 6),
            lambda: ops.embedding_lookup_grad(dy, i.cpu(), 6),
            lambda: ops.embedding_lookup_grad(dy, i, 0),
            lambda: ops.embedding_lookup_grad(dy, i, 6, dtype=torch.int32)):
        with pytest.raises(ValueError):
            call()


# ---- together, as the classifier trains ---------------------------------------------------
def _steps(device, dtype, steps, clip, native):
    """training steps of the classifier's model: the logits, gradients before
    and after clipping, and the norm of each; weights of the first step only
    (plain descent, so that the two sides stay comparable)"""
    gen = torch.Generator().manual_seed(5)
    rng = np.random.RandomState(2)
    V, D = 500, 20
    emb = rng.randn(V, D).astype(np.float32)
    model = G.build_model(V, emb, D, "cpu", gen, train_embedding=True).to(device, dtype)
    out = []
    for k in range(steps):
        x = torch.from_numpy(rng.randint(0, V, (128, 2))).to(device)
        x[:30] = 3  # a frequent gene
        t = torch.from_numpy(rng.randint(0, 2, 128)).to(device)
        logits = model(x, 1.0)
        loss = torch.nn.functional.cross_entropy(logits, t)
        model.zero_grad()
        loss.backward()
        before = [p.grad.clone() for p in model.parameters()]
        if native:
            norm = G.clip_gradients_(model.parameters(), clip)
        else:
            norm = torch.sqrt(sum(g.square().sum() for g in before))
            for p in model.parameters():
                p.grad.mul_(clip / norm.clamp(min=clip))
        out.append([logits.detach()] + before + [p.grad.clone() for p in model.parameters()]
                   + [norm])
        with torch.no_grad():
            for p in model.parameters():
                p -= 0.1 * p.grad
        del loss, logits
    return out


def test_classifier_step_against_64_bits():
    """lookup, backward and clipping together in fp32 against the same model in
    fp64 on the CPU.  Per value the chain is 5 products of inner length <= 100
    forward and as many backward: the running error of a dot product of length
    n is at most n u of its absolute sum, 10 stages of at most 130 terms each
    (128 rows, a bias, a scale) give 1300 u = 7.8e-5 of the magnitudes, taken
    here as those of the tensor's largest entry, times the 8-fold growth that
    absolute sums may have over values in 3 steps of descent."""
    got = _steps("cuda", F32, 3, 0.05, True)
    want = _steps("cpu", torch.float64, 3, 0.05, False)
    for g, w in zip(got, want):
        for a, b in zip(g, w):
            scale = float(b.abs().max()) + 1e-12
            assert float((a.cpu().double() - b).abs().max()) <= 8 * 1300 * U * scale


def test_classifier_trains_its_table_end_to_end(tmp_path):
    rng = np.random.RandomState(1)
    genes = [f"G{i}" for i in range(60)]
    for name, n in (("train", 600), ("valid", 10), ("test", 80)):
        a, b = rng.randint(0, 60, n), rng.randint(0, 60, n)
        (tmp_path / f"{name}_text.txt").write_text(
            "\n".join(f"{genes[i]} {genes[j]}" for i, j in zip(a, b)))
        (tmp_path / f"{name}_label.txt").write_text("\n".join(map(str, (a + b) % 2)))
    emb = tmp_path / "emb.txt"
    emb.write_text("".join(g + "\t" + "".join(f"{v} " for v in rng.randn(8)) + "\n" for g in genes))
    a = [G.train_and_auc(str(emb), str(tmp_path), seed=0, embedding_size=8, device="cuda",
                         train_embedding=t, clip_norm=c)
         for t, c in ((False, None), (True, None), (True, 0.5))]
    assert all(0.0 <= x <= 1.0 for x in a)


def test_captured_training_step():
    """forward, backward and clipping of a trained table in one graph"""
    V, D = 400, 16
    w = torch.randn(V, D, device="cuda", requires_grad=True)
    ids = torch.zeros(64, dtype=torch.int64, device="cuda")
    c = torch.randn(64, D, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):  # warm up away from the capture, keep no graph of it
        (ops.embedding_lookup(w, ids, 2.0) * c).sum().backward()
        w.grad = None
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grad, = torch.autograd.grad(ops.embedding_lookup(w, ids, 2.0), w, c)
        norm = ops.clip_by_global_norm_([grad], 1.0)
    for r in range(3):
        ids.copy_(make_ids("zipf", V, 64, torch.int64, r))
        g.replay()
        torch.cuda.synchronize()
        eager = ops.embedding_lookup_grad(c, ids, V, 2.0)
        assert torch.equal(norm, ops.clip_by_global_norm_([eager], 1.0))
        assert torch.equal(grad, eager)


def test_capture_beside_a_live_eager_graph_is_refused():
    w = torch.randn(30, 8, device="cuda", requires_grad=True)
    ids = torch.arange(10, device="cuda")
    x = torch.ones(4, device="cuda")
    live = ops.embedding_lookup(w, ids)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x += 1
        with pytest.raises(ValueError, match="alive"):
            ops.embedding_lookup(w, ids)
        with torch.no_grad():
            y = ops.embedding_lookup(w, ids)
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(x, torch.full_like(x, 2)) and torch.equal(y, w[:10])
    live.sum().backward()  # the eager graph is still good
    assert float(w.grad.sum()) == 80.0
    del live
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):  # a table that is no leaf, computed in the graph
        part, = torch.autograd.grad(ops.embedding_lookup(w * 2.0, ids).sum(), w)
    g.replay()
    torch.cuda.synchronize()
    assert float(part.sum()) == 160.0
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        both = ops.embedding_lookup(w, ids) + ops.embedding_lookup(w, ids)
        grad, = torch.autograd.grad(both.sum(), w)
    del both
    g.replay()
    torch.cuda.synchronize()
    assert float(grad.sum()) == 160.0


# ---- the C entries: exact buffers, any workspace contents --------------------------------
class Guarded:
    """nbytes of device memory at an offset of its element size from an aligned
    address, with sentinel bytes on both sides"""

    def __init__(self, nbytes, shift=0, fill=0x5A):
        self.whole = torch.full((nbytes + 4096,), fill, dtype=torch.uint8, device="cuda")
        self.at, self.n, self.fill = 2048 + shift, nbytes, fill
        self.inside = self.whole[self.at:self.at + nbytes]

    def ptr(self):
        return self.whole.data_ptr() + self.at

    def check(self):
        w = self.whole
        assert bool((w[:self.at] == self.fill).all())
        assert bool((w[self.at + self.n:] == self.fill).all())


CODE = {F32: N.F32, F16: N.F16, BF16: N.BF16}


@pytest.mark.parametrize("V,D,n,kind", [
    (1, 1, 1, "same"), (7, 3, 100, "zipf"), (300, 9, 257, "absent"), (999, 13, 5000, "skew"),
    (257, 200, 16384, "zipf"), (5000, 31, 16385, "zipf"), (2, 17, 40000, "two"),
    (24447, 5, 70001, "skew"), (262145, 1, 20000, "skew"), (40, 515, 3000, "same")])
@pytest.mark.parametrize("t", TYPES)
def test_c_entries_stay_inside_their_buffers(V, D, n, kind, t):
    L, st = N.lib(), torch.cuda.current_stream().cuda_stream
    size = torch.finfo(t).bits // 8
    w = torch.randn(V, D, device="cuda").to(t)
    dy = torch.randn(n, D, device="cuda").to(t)
    ids = make_ids(kind, V, n, torch.int32, V).cuda()
    out = Guarded(n * D * size, size)
    N.check(L.g2v_embed_lookup(0, w.data_ptr(), CODE[t], V, D, D, ids.data_ptr(), 4, n, 1.5,
                               out.ptr(), CODE[t], st))
    out.check()
    got = out.inside.clone().view(t).view(n, D)
    assert torch.equal(got, ops.embedding_lookup(w, ids, 1.5))
    need = C.c_int64()
    N.check(L.g2v_embed_grad_workspace(n, V, D, C.byref(need)))
    want = ops.embedding_lookup_grad(dy, ids, V, 1.5, 0)
    for fill in (0x00, 0x7F, 0xFF):
        ws, g = Guarded(need.value, 0, fill), Guarded(V * D * size, size, fill)
        N.check(L.g2v_embed_grad(0, dy.data_ptr(), CODE[t], D, ids.data_ptr(), 4, n, V, D, 1.5, 0,
                                 g.ptr(), CODE[t], ws.ptr(), need.value, st))
        ws.check()
        g.check()
        assert torch.equal(g.inside.clone().view(t).view(V, D), want)


@pytest.mark.parametrize("sizes", [[1], [5, 8191, 8192, 8193], [17] * 129, [1, 70001, 3] * 100])
def test_c_norm_and_clip_stay_inside_their_buffers(sizes):
    L, st = N.lib(), torch.cuda.current_stream().cuda_stream
    types = [TYPES[k % 3] for k in range(len(sizes))]
    ts = [torch.randn(s, device="cuda").to(t) for s, t in zip(sizes, types)]
    n = len(ts)
    outs = [Guarded(s * t.itemsize, t.itemsize) for s, t in zip(sizes, types)]
    src = (C.c_void_p * n)(*[t.data_ptr() for t in ts])
    dst = (C.c_void_p * n)(*[o.ptr() for o in outs])
    numel, codes = (C.c_int64 * n)(*sizes), (C.c_int32 * n)(*[CODE[t] for t in types])
    need = C.c_int64()
    N.check(L.g2v_global_norm_workspace(n, C.byref(need)))
    want, wn = ops.clip_by_global_norm(ts, 0.25)
    for fill in (0x00, 0x7F, 0xFF):
        ws, norm = Guarded(need.value, 0, fill), Guarded(4, 4, fill)
        N.check(L.g2v_global_norm(0, src, numel, codes, n, norm.ptr(), ws.ptr(), need.value, st))
        assert torch.equal(norm.inside.clone().view(F32)[0], wn)
        N.check(L.g2v_clip_global_norm(0, src, dst, numel, codes, n, 0.25, norm.ptr(), ws.ptr(),
                                       need.value, st))
        assert torch.equal(norm.inside.clone().view(F32)[0], wn)
        for g in (ws, norm, *outs):
            g.check()
        for o, x in zip(outs, want):
            assert torch.equal(o.inside.clone().view(x.dtype), x)


def test_saved_tensor_hooks_and_checkpoints():
    from torch.utils.checkpoint import checkpoint
    w = torch.randn(40, 6, device="cuda", requires_grad=True)
    ids = torch.randint(0, 40, (50,), device="cuda")
    c = torch.randn(50, 6, device="cuda")
    want = ops.embedding_lookup_grad(c, ids, 40)
    with torch.autograd.graph.save_on_cpu():
        y = ops.embedding_lookup(w, ids)
    assert torch.equal(torch.autograd.grad(y, w, c)[0], want)
    y = checkpoint(lambda a: ops.embedding_lookup(a, ids), w, use_reentrant=False)
    assert torch.equal(torch.autograd.grad(y, w, c)[0], want)
    y = ops.embedding_lookup(w, ids)
    for _ in range(2):  # the graph is kept
        assert torch.equal(torch.autograd.grad(y, w, c, retain_graph=True)[0], want)


def test_capture_beside_a_live_graph_of_a_side_stream():
    """a graph of the leaf that lives on a side stream is joined into the capture"""
    w = torch.randn(30, 8, device="cuda", requires_grad=True)
    ids = torch.arange(10, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        live = ops.embedding_lookup(w, ids)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        grad, = torch.autograd.grad(ops.embedding_lookup(w, ids, 3.0).sum(), w)
    for _ in range(2):
        g.replay()
        torch.cuda.synchronize()
        assert float(grad.sum()) == 240.0
    assert torch.equal(live.detach(), w.detach()[:10])
