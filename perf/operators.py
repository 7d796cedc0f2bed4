"""Cases of the codebook, gradient-clipping and clipped-Adam operators.

Each case is one pass a training program makes: `run` computes it in its plain
form (elementary torch operations) or, where `own` is true, through
`cuda_rasterizer`. Sizes are those of the training scenes (1k, 50k, 500k, 1M
and at most 2M Gaussians of 3 + 3 + 4 + 1 + 16 floats, 16 SH coefficients) and
generic embedding tables.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
INDEX = {"i32": torch.int32, "i64": torch.int64}
SIZE = {"f32": 4, "bf16": 2, "f16": 2, "i32": 4, "i64": 8}
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8


def _package():
    root = os.path.join(os.getcwd(), "sar-3dgs_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from cuda_rasterizer import clipping, codebook
    return codebook, clipping


def listed():
    return [
        # SH rows of the smallest scene (1k Gaussians) from a 256-entry codebook: latency
        dict(name="lookup_1k", op="lookup", n=1000, d=16, codes=256, table="f32", rows="f32", index="i64", skew=2.0, none=0.0),
        # the 1M-Gaussian scene's SH rows from a half-size table, handed to the fp32 rasterizer
        dict(name="lookup_1m", op="lookup", n=1000000, d=16, codes=4096, table="bf16", rows="f32", index="i32", skew=3.0, none=0.01),
        # a generic embedding: a ragged batch of tokens, wide rows of an odd number of 16-byte pieces
        dict(name="lookup_wide", op="lookup", n=16381, d=1000, codes=50000, table="bf16", rows="bf16", index="i64", skew=2.0, none=0.02),
        # sorting the 50k scene's assignment once after a re-quantisation
        dict(name="sort_50k", op="sort", n=50000, codes=1024, index="i64", skew=2.0, none=0.0),
        # the 1M scene against the largest codebook
        dict(name="sort_1m", op="sort", n=1000000, codes=65536, index="i32", skew=1.0, none=0.01),
        # codebook gradient of the smallest scene: latency
        dict(name="grad_1k", op="grad", n=1000, d=16, codes=256, rows="f32", table="f32", index="i64", skew=2.0, none=0.0),
        # the 1M scene's SH gradient rows summed into 4096 codes, the most used code with about 6% of all rows
        dict(name="grad_1m", op="grad", n=1000000, d=16, codes=4096, rows="f32", table="f32", index="i32", skew=3.0, none=0.01),
        # gradient of a generic embedding table from 16-bit rows, most codes of it unused
        dict(name="grad_wide", op="grad", n=16381, d=1024, codes=32000, rows="bf16", table="f32", index="i64", skew=2.0, none=0.02),
        # the parameter gradients of the 50k scene, clipped
        dict(name="clip_50k", op="clip", tensors=5, total=50000 * 27, type="f32", ragged=0, norm=2.0, max_norm=1.0),
        # the gradients of a model of many ragged tensors in two types
        dict(name="clip_many", op="clip", tensors=160, total=200000000, type="bf16", ragged=1, norm=2.0, max_norm=1.0),
        # the 50k scene's training update: norm, clipping and Adam over its flat buffer
        dict(name="adam_50k", op="adam", n=50000, sh=16, step=100, max_norm=1.0),
        # the largest set that densification grows to
        dict(name="adam_2m", op="adam", n=2000000, sh=16, step=1000, max_norm=1.0),
    ]


def _log(rng, a, b):
    return int(round(math.exp(rng.uniform(math.log(a), math.log(b)))))


def draw(rng):
    op = rng.choice(["lookup", "sort", "grad", "clip", "adam"])
    if op in ("lookup", "grad"):
        d = _log(rng, 1, 64) if rng.random() < 0.5 else _log(rng, 64, 2048)
        n = _log(rng, 1, min(1000000, 16000000 // d))
        codes = _log(rng, 1, min(65536, 32000000 // d))
        t = rng.choice(["f32", "bf16", "f16"])
        f = rng.choice([t, "f32"])
        c = dict(op=op, n=n, d=d, codes=codes, index=rng.choice(["i32", "i64"]), skew=round(rng.uniform(1.0, 4.0), 2),
                 none=rng.choice([0.0, 0.01, 0.3]))
        c.update(dict(table=t, rows=f) if op == "lookup" else dict(rows=t, table=f))
        return c
    if op == "sort":
        return dict(op=op, n=_log(rng, 1, 1000000), codes=_log(rng, 1, 65536), index=rng.choice(["i32", "i64"]),
                    skew=round(rng.uniform(1.0, 4.0), 2), none=rng.choice([0.0, 0.01, 0.3]))
    if op == "clip":
        tensors = _log(rng, 1, 160)
        return dict(op=op, tensors=tensors, total=_log(rng, 10 * tensors, 100000000), type=rng.choice(["f32", "bf16", "f16"]),
                    ragged=rng.choice([0, 1]), norm=rng.choice([2.0, 2.0, math.inf]), max_norm=rng.choice([0.1, 1.0, 1e6]))
    return dict(op=op, n=_log(rng, 100, 2000000), sh=rng.choice([1, 4, 9, 16]), step=_log(rng, 1, 3000), max_norm=rng.choice([0.1, 1.0, 1e6]))


def _index(case, g):
    """Codes of n tokens, a few codes used far more than the others, some tokens without a code."""
    n, codes = case["n"], case["codes"]
    i = (torch.rand(n, generator=g, device="cuda", dtype=torch.float64) ** case["skew"] * codes).long().clamp_(max=codes - 1)
    i = torch.randperm(codes, generator=g, device="cuda")[i]
    i[torch.rand(n, generator=g, device="cuda") < case["none"]] = -1
    return i.to(INDEX[case["index"]])


def _lengths(case):
    """Elements of each tensor of a clip case: equal shares, or ragged ones of which every fourth is small and odd."""
    t, total = case["tensors"], case["total"]
    if not case["ragged"]:
        return [total // t + (k < total % t) for k in range(t)]
    small = [1 + (977 * k) % 4099 if k % 4 == 3 else 0 for k in range(t)]
    rest = max(0, total - sum(small))
    weight = [0 if s else 1 + (7 * k) % 13 for k, s in enumerate(small)]
    return [s or max(1, rest * w // max(1, sum(weight))) for s, w in zip(small, weight)]


def _parts(flat, lengths):
    at, got = 0, []
    for n in lengths:
        got.append(flat[at:at + n])
        at += n
    return got


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    s = dict(case=case)
    if case["op"] in ("lookup", "sort", "grad"):
        s["index"] = _index(case, g)
    if case["op"] == "lookup":
        s["table"] = randn(case["codes"], case["d"]).mul_(0.1).to(TYPES[case["table"]])
        s["scale"] = math.sqrt(case["d"])
    elif case["op"] == "grad":
        s["grad"] = randn(case["n"], case["d"]).mul_(1e-3).to(TYPES[case["rows"]])
        s["scale"] = math.sqrt(case["d"])
    elif case["op"] == "clip":
        # the gradients of each type in one flat buffer, as an all-reduce leaves them; a ragged list holds every
        # eighth tensor in 32 bits
        lengths = _lengths(case)
        kinds = ["f32" if case["ragged"] and k % 8 == 5 else case["type"] for k in range(len(lengths))]
        s["flat"], s["out"], s["grads"], s["outs"] = {}, {}, [None] * len(lengths), [None] * len(lengths)
        for kind in sorted(set(kinds)):
            at = [k for k, x in enumerate(kinds) if x == kind]
            size = [lengths[k] for k in at]
            flat = torch.empty(sum(size), dtype=TYPES[kind], device="cuda")
            flat.normal_(0.0, 1e-2, generator=g)
            out = torch.empty_like(flat)
            s["flat"][kind], s["out"][kind] = flat, out
            for k, x, y in zip(at, _parts(flat, size), _parts(out, size)):
                s["grads"][k], s["outs"][k] = x, y
    elif case["op"] == "adam":
        total = case["n"] * (4 + case["sh"])
        s["param"], s["grad"] = randn(total), randn(total).mul_(1e-2)
        s["m"], s["v"] = randn(total).mul_(1e-3), torch.rand(total, generator=g, device="cuda").mul_(1e-6)
        # means and opacity logits at lr, SH rows at lr / 100
        s["segments"] = [(3 * case["n"], 1e-3), (4 * case["n"], 1e-3), (total, 1e-5)]
    return s


def _keys(index, codes):
    i = index.long()
    return torch.where((i >= 0) & (i < codes), i, codes)


def _lookup(s):
    c = s["case"]
    i = _keys(s["index"], c["codes"])
    have = i < c["codes"]
    rows = s["table"].float()[torch.where(have, i, 0)] * s["scale"]
    return torch.where(have[:, None], rows, 0.0).to(TYPES[c["rows"]])


def _sort(s):
    keys, order = torch.sort(_keys(s["index"], s["case"]["codes"]), stable=True)
    offsets = torch.searchsorted(keys, torch.arange(s["case"]["codes"] + 1, device=keys.device))
    return order.int(), keys.int(), offsets.int()


def _grad(s):
    # 64-bit sums: the most used codes sum tens of thousands of rows
    c = s["case"]
    total = torch.zeros(c["codes"] + 1, c["d"], dtype=torch.float64, device="cuda")
    total.index_add_(0, _keys(s["index"], c["codes"]), s["grad"].double())
    return (total[:-1] * s["scale"]).to(TYPES[c["table"]])


def _norm(grads, kind):
    if kind == math.inf:
        return torch.stack([x.float().abs().max() for x in grads]).max().double()
    return torch.stack([x.double().square().sum() for x in grads]).sum().sqrt()


def _clip(s):
    c = s["case"]
    norm = _norm(s["grads"], c["norm"])
    coef = (c["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    [y.copy_(x.float() * coef) for x, y in zip(s["grads"], s["outs"])]
    return norm.float(), s["out"]


def _adam(s):
    c = s["case"]
    norm = _norm([s["grad"]], 2.0)
    g = s["grad"] * (c["max_norm"] / (norm + 1e-6)).clamp(max=1.0).float()
    s["m"].add_((g - s["m"]) * (1.0 - BETA1))
    s["v"].mul_(BETA2).add_(g * g * (1.0 - BETA2))
    move = s["m"] / (s["v"].sqrt() / math.sqrt(1.0 - BETA2 ** c["step"]) + EPS)
    ends = [0] + [e for e, _ in s["segments"]]
    [s["param"][a:b].sub_(move[a:b] * (lr / (1.0 - BETA1 ** c["step"]))) for a, b, (_, lr) in zip(ends, ends[1:], s["segments"])]
    return norm.float(), s["param"], s["m"], s["v"]


def _own(s):
    codebook, clipping = _package()
    c = s["case"]
    if c["op"] == "lookup":
        return codebook.lookup(s["table"], s["index"], scale=s["scale"], dtype=TYPES[c["rows"]])
    if c["op"] == "sort":
        return codebook.sort_by_code(s["index"], c["codes"])
    if c["op"] == "grad":
        return codebook.gradient(s["grad"], s["index"], c["codes"], scale=s["scale"], dtype=TYPES[c["table"]])
    if c["op"] == "clip":
        norm = clipping.clip_grads(s["grads"], c["max_norm"], norm_type=c["norm"], out=s["outs"])
        return norm, s["out"]
    norm = clipping.adam_step_clipped(s["param"], s["grad"], s["m"], s["v"], s["segments"], c["step"], c["max_norm"],
                                      betas=(BETA1, BETA2), eps=EPS)
    return norm, s["param"], s["m"], s["v"]


def run(state):
    if own:
        return _own(state)
    return {"lookup": _lookup, "sort": _sort, "grad": _grad, "clip": _clip, "adam": _adam}[state["case"]["op"]](state)


def work(case):
    op = case["op"]
    if op == "adam":
        total = case["n"] * (4 + case["sh"])
        return {"bytes": 28 * total, "flops": 18 * total}
    if op == "clip":
        lengths = _lengths(case)
        size = sum(n * (4 if case["ragged"] and k % 8 == 5 else SIZE[case["type"]]) for k, n in enumerate(lengths))
        return {"bytes": 2 * size, "flops": 3 * sum(lengths)}
    n, codes = case["n"], case["codes"]
    if op == "sort":
        return {"bytes": n * (SIZE[case["index"]] + 8) + 4 * (codes + 1), "flops": 0}
    used = min(n, codes) if op == "lookup" else codes
    return {"bytes": n * SIZE[case["index"]] + used * case["d"] * SIZE[case["table"]] + n * case["d"] * SIZE[case["rows"]],
            "flops": n * case["d"]}


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    host = lambda t: t.detach().cpu().double().numpy()  # noqa: E731
    if op in ("lookup", "sort", "grad"):
        index, codes = s["index"].cpu().numpy().astype(np.int64), case["codes"]
        valid = (index >= 0) & (index < codes)
    if op == "lookup":
        out = np.zeros((case["n"], case["d"]))
        out[valid] = host(s["table"])[index[valid]] * s["scale"]
        return out
    if op == "sort":
        keys = np.where(valid, index, codes)
        order = np.argsort(keys, kind="stable")
        counts = np.bincount(index[valid], minlength=codes)
        return order.astype(np.int32), keys[order].astype(np.int32), np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
    if op == "grad":
        grad = host(s["grad"])[valid]
        return np.stack([np.bincount(index[valid], weights=grad[:, j], minlength=codes) for j in range(case["d"])], axis=1) * s["scale"]
    if op == "clip":
        flats = list(s["flat"].values())
        if case["norm"] == math.inf:
            norm = max(float(x.abs().max()) for x in flats)
        else:
            norm = math.sqrt(math.fsum(float(torch.dot(p, p)) for x in flats for p in (q.double() for q in x.split(1 << 24))))
        coef = min(1.0, case["max_norm"] / (norm + 1e-6))
        return norm, {k: x.double() * coef for k, x in s["flat"].items()}
    g = s["grad"].double()
    norm = math.sqrt(float(torch.dot(g, g)))
    g *= min(1.0, case["max_norm"] / (norm + 1e-6))
    m = BETA1 * s["m"].double() + (1 - BETA1) * g
    v = BETA2 * s["v"].double() + (1 - BETA2) * g ** 2
    lr = torch.empty_like(g)
    at = 0
    for end, rate in s["segments"]:
        lr[at:end] = rate
        at = end
    t = case["step"]
    param = s["param"].double() - lr * (m / (1 - BETA1 ** t)) / ((v / (1 - BETA2 ** t)).sqrt() + EPS)
    return norm, param, m, v
