"""The embedding and gradient operators as they are measured: the cases, their
inputs, the calls, and the same operators in plain torch.

    lookup  y[i] = scale * W[ids[i]], a zero row where ids[i] is outside [0, V)
    train   the lookup, and dW[v] = scale * sum of dy[i] over ids[i] == v (no
            row for padding_idx)
    norm    sqrt of the sum of squares over a list of gradients
    clip    the norm n, and every gradient times clip / max(n, clip)

``own`` False: plain torch, in 32 bits (the sum of squares in 64).  True: the
calls of ``gene2vec_amd.ops``.
"""
import math

import torch

own = False

DTYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16,
          "int32": torch.int32, "int64": torch.int64}
SIZE = {"fp32": 4, "bf16": 2, "fp16": 2, "int32": 4, "int64": 8}


def _lookup(name, kind, V, D, N, table, out, ids, scaled=True, absent=0.0, zipf=True, padding=-1):
    return {"name": name, "kind": kind, "V": V, "D": D, "N": N, "table": table, "out": out,
            "ids": ids, "scaled": scaled, "absent": absent, "zipf": zipf, "padding": padding}


def _grads(name, kind, tensors, elements, types, clip=0.3):
    return {"name": name, "kind": kind, "tensors": tensors, "elements": elements, "types": types,
            "clip": clip}


def listed():
    return [
        # one gene of the C2 vocabulary, as a server answers a single request
        _lookup("lookup_one", "lookup", 24447, 200, 1, "fp32", "fp32", "int64", scaled=False),
        # a batch of prompts at the C4 table's width, half precision throughout
        _lookup("lookup_prompt", "lookup", 60000, 512, 8192, "bf16", "bf16", "int64"),
        # an odd width and length, 5 % of the tokens out of vocabulary
        _lookup("lookup_odd", "lookup", 24447, 301, 9973, "fp16", "fp32", "int32", absent=0.05),
        # the largest: a generic language-model table and 64 Ki tokens
        _lookup("lookup_large", "lookup", 131072, 4096, 65536, "bf16", "bf16", "int64"),
        # the GGIPNN classifier's batch: 128 pairs over the 12,472 genes of its splits
        _lookup("train_classifier", "train", 12472, 200, 256, "fp32", "fp32", "int64",
                scaled=False, zipf=False),
        # a large batch of co-expression pairs at the C2 shape, frequent genes first
        _lookup("train_pairs", "train", 24447, 200, 65536, "fp32", "fp32", "int32",
                scaled=False),
        # fp32 table, bf16 activations, ragged length, padding inside the batch
        _lookup("train_mixed", "train", 60000, 512, 262147, "fp32", "bf16", "int64", absent=0.05,
                padding=0),
        # a wide bf16 table: most of the time is the dense gradient itself
        _lookup("train_wide", "train", 131072, 4096, 16384, "bf16", "bf16", "int64"),
        # the norm alone: 33 odd fp16 tensors
        _grads("norm_odd", "norm", 33, 1000003, "fp16"),
        # the norm alone: the gradients of a model of 10^9 parameters in bf16
        _grads("norm_large", "norm", 48, 1000000000, "bf16"),
        # the classifier's gradients: 8 small tensors and the embedding table's
        _grads("clip_classifier", "clip", 9, 0, "fp32"),
        # many tensors from scalars to millions of elements, two types
        _grads("clip_many", "clip", 600, 300000000, "mixed"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["lookup", "train", "norm", "clip"])
    if kind in ("norm", "clip"):
        tensors = _log(rng, 1, 700)
        c = _grads("", kind, tensors, max(tensors, _log(rng, 100, 300000000)),
                   rng.choice(["fp32", "bf16", "fp16", "mixed"]), rng.choice([0.01, 0.3, 2.0]))
    else:
        V, D, N = _log(rng, 2, 250000), _log(rng, 1, 8192), _log(rng, 1, 262144)
        while V * D > 1 << 28:
            V = max(2, V // 2)
        while N * D > 1 << 27:
            N = max(1, N // 2)
        c = _lookup("", kind, V, D, N, rng.choice(["fp32", "bf16", "fp16"]),
                    rng.choice(["fp32", "bf16", "fp16"]), rng.choice(["int32", "int64"]),
                    rng.random() < 0.5, rng.choice([0.0, 0.05]), rng.random() < 0.7,
                    rng.choice([-1, 0]))
    del c["name"]
    return c


def _sizes(case):
    """the elements of each gradient: the classifier's own, or a spread from 1
    to many times the mean that adds up to about case["elements"]"""
    if case["elements"] == 0:
        return [12472 * 200, 400 * 100, 100, 100 * 100, 100, 100 * 10, 10, 10 * 2, 2]
    n = case["tensors"]
    w = [math.exp(6.0 * ((k * 0.6180339887498949) % 1.0)) for k in range(n)]
    f = case["elements"] / sum(w)
    return [max(1, int(f * x)) for x in w]


def _types(case):
    t = case["types"]
    return [("fp32", "bf16")[k % 3 == 0] if t == "mixed" else t for k in range(len(_sizes(case)))]


def _scale(case):
    return math.sqrt(case["D"]) if case["scaled"] else 1.0


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)

    def rand(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    if case["kind"] in ("norm", "clip"):
        # one bucket per type, as data-parallel training keeps its gradients
        sizes, types = _sizes(case), _types(case)
        flat, outs, grads, clipped = {}, {}, [], []
        for t in sorted(set(types)):
            total = sum(n for n, x in zip(sizes, types) if x == t)
            flat[t] = torch.empty(total, device="cuda", dtype=DTYPES[t])
            outs[t] = torch.empty_like(flat[t])
            for a in range(0, total, 1 << 26):
                b = min(total, a + (1 << 26))
                flat[t][a:b] = 0.01 * rand(b - a)
        at = dict.fromkeys(flat, 0)
        for n, t in zip(sizes, types):
            grads.append(flat[t][at[t]:at[t] + n])
            clipped.append(outs[t][at[t]:at[t] + n])
            at[t] += n
        return {"case": case, "grads": grads, "clipped": clipped, "flat": outs, "source": flat,
                "clip": case["clip"] * 0.01 * math.sqrt(sum(sizes))}
    V, D, N = case["V"], case["D"], case["N"]
    table = torch.empty(V, D, device="cuda", dtype=DTYPES[case["table"]])
    step = max(1, (1 << 26) // D)
    for a in range(0, V, step):
        b = min(V, a + step)
        table[a:b] = rand(b - a, D) / math.sqrt(D)
    u = torch.rand(N, device="cuda", generator=gen, dtype=torch.float64)
    if case["zipf"]:  # P(id = r) = log((r + 2) / (r + 1)) / log(V + 1)
        ids = torch.exp(u * math.log(V + 1)).to(torch.int64) - 1
    else:
        ids = (u * V).to(torch.int64)
    ids = ids.clamp(0, V - 1)
    if case["absent"] > 0:
        gone = torch.rand(N, device="cuda", generator=gen) < case["absent"]
        ids = torch.where(gone, -1, ids)
    s = {"case": case, "table": table, "ids": ids.to(DTYPES[case["ids"]]), "scale": _scale(case),
         "out": DTYPES[case["out"]], "padding": case["padding"] if case["padding"] >= 0 else None}
    if case["kind"] == "train":
        table.requires_grad_(True)
        s["dy"] = rand(N, D).to(s["out"])
    return s


def _run_own(s):
    from gene2vec_amd import ops
    kind = s["case"]["kind"]
    if kind == "lookup":
        return ops.embedding_lookup(s["table"], s["ids"], scale=s["scale"], dtype=s["out"])
    if kind == "train":
        y = ops.embedding_lookup(s["table"], s["ids"], scale=s["scale"],
                                 padding_idx=s["padding"], dtype=s["out"])
        grad, = torch.autograd.grad(y, s["table"], s["dy"])
        return {"y": y, "grad": grad}
    if kind == "norm":
        return ops.global_norm(s["grads"])
    _, norm = ops.clip_by_global_norm(s["grads"], s["clip"], out=s["clipped"])
    return {"norm": norm, "clipped": s["flat"]}


def _plain_lookup(s):
    table = s["table"].detach()
    ids = s["ids"].to(torch.int64)
    there = (ids >= 0) & (ids < table.shape[0])
    at = torch.where(there, ids, 0)
    rows = table[at].to(torch.float32) * s["scale"]
    return torch.where(there[:, None], rows, 0.0).to(s["out"]), at, there


def _plain_norm(grads):
    total = torch.zeros((), device="cuda", dtype=torch.float64)
    for g in grads:
        x = g.to(torch.float32)
        total += (x * x).sum(dtype=torch.float64)
    return torch.sqrt(total).to(torch.float32)


def run(state):
    if own:
        return _run_own(state)
    s = state
    kind = s["case"]["kind"]
    if kind == "lookup":
        return _plain_lookup(s)[0]
    if kind == "train":
        y, at, there = _plain_lookup(s)
        if s["padding"] is not None:
            there = there & (at != s["padding"])
        dy = s["dy"].to(torch.float32) * s["scale"]
        grad = torch.zeros(s["table"].shape, device="cuda", dtype=torch.float32)
        grad.index_add_(0, at, torch.where(there[:, None], dy, 0.0))
        return {"y": y, "grad": grad.to(s["table"].dtype)}
    norm = _plain_norm(s["grads"])
    if kind == "norm":
        return norm
    factor = s["clip"] / torch.clamp(norm, min=s["clip"])
    for g, o in zip(s["grads"], s["clipped"]):
        o.copy_(g.to(torch.float32) * factor)
    return {"norm": norm, "clipped": s["flat"]}


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] in ("norm", "clip"):
        squares = 0.0
        for x in s["source"].values():
            for a in range(0, x.numel(), 1 << 27):
                part = x[a:a + (1 << 27)].double()
                squares += float(torch.dot(part, part))
        norm = math.sqrt(squares)
        if case["kind"] == "norm":
            return torch.tensor(norm, dtype=torch.float64)
        shrink = s["clip"] / max(norm, s["clip"])
        return {"norm": torch.tensor(norm, dtype=torch.float64),
                "clipped": {t: x.double() * shrink for t, x in s["source"].items()}}
    table, ids, scale = s["table"].detach().double(), s["ids"].long(), s["scale"]
    V, D = table.shape
    # the absent tokens take a row of zeros behind the table
    where = torch.where((ids < 0) | (ids >= V), V, ids)
    y = torch.cat([table, table.new_zeros(1, D)]).index_select(0, where).mul_(scale)
    if case["kind"] == "lookup":
        return y
    if s["padding"] is not None:
        where = torch.where(where == s["padding"], V, where)
    grad = torch.zeros(V + 1, D, dtype=torch.float64, device="cuda")
    for a in range(0, D, 512):  # columns apart: the sorted copies stay small
        grad[:, a:a + 512] = torch.zeros_like(grad[:, a:a + 512]).index_put_(
            (where,), s["dy"][:, a:a + 512].double(), accumulate=True)
    return {"y": y, "grad": grad[:V].mul_(scale)}


def _rows(case):
    """the distinct rows that the tokens are expected to name"""
    V, N = case["V"], case["N"]
    r = torch.arange(1, V + 1, dtype=torch.float64)
    p = torch.log1p(1 / r) / math.log(V + 1) if case["zipf"] else torch.full_like(r, 1 / V)
    return float((-torch.expm1(N * (1 - case["absent"]) * torch.log1p(-p.clamp(max=1 - 1e-12)))).sum())


def work(case):
    if case["kind"] in ("norm", "clip"):
        n = [a * SIZE[t] for a, t in zip(_sizes(case), _types(case))]
        elements = sum(_sizes(case))
        both = case["kind"] == "clip"
        return {"bytes": sum(n) * (2 if both else 1) + 4, "flops": elements * (3 if both else 2)}
    V, D, N = case["V"], case["D"], case["N"]
    w, o = SIZE[case["table"]], SIZE[case["out"]]
    there = N * (1 - case["absent"])
    got = {"bytes": N * SIZE[case["ids"]] + _rows(case) * D * w + N * D * o, "flops": there * D}
    if case["kind"] == "train":
        got["bytes"] += there * D * o + V * D * w
        got["flops"] += (there + _rows(case)) * D
    return got
