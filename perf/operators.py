"""The operators at the two ends of a graph model, as calls a user's program makes of them.

At the front a table of learned feature rows is looked up by node (or token) ids, and its gradient sums the rows of
equal ids.  At the back the scores over classes - or over all nodes, where links are predicted - become log
probabilities of given ids, entropies and the best alternatives, with the gradient for training.

Plain forms below are elementary torch operations in 32 bits, rounded once at the end; `exact` has the definitions in
64 bits.  Sizes are those of the benchmark's graphs (2^17 to 2^20 nodes, widths 64 to 128, 47 classes) and around them.
"""
from __future__ import annotations

import math
import os
import sys

import numpy as np
import torch

own = False

_DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def _api():
    pkg = os.path.join(os.getcwd(), "tr-spmm_zzx_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)
    import trspmm
    return trspmm


def listed():
    return [
        # a handful of nodes of a small graph, looked up on request: what a call costs before any work is done
        {"name": "lookup 64 of 4k F64 f16", "op": "lookup", "rows": 4096, "ids": 64, "F": 64, "table": "f16", "out": "f16",
         "scale": 1.0, "skew": False, "padding": False},
        # features of all nodes of a power-law graph by the popularity of what they refer to, table beyond the L2
        {"name": "lookup 1M of 1M F128 f16", "op": "lookup", "rows": 1 << 20, "ids": 1 << 20, "F": 128, "table": "f16",
         "out": "f16", "scale": 1.0, "skew": True, "padding": False},
        # fp32 master table, fp16 features for the product, a width that is a class count, padded id lists
        {"name": "lookup 300k of 50k F47 f32", "op": "lookup", "rows": 50021, "ids": 300007, "F": 47, "table": "f32",
         "out": "f16", "scale": 0.125, "skew": False, "padding": True},
        # the gradient of one small batch
        {"name": "grad 512 in 4k F64 f16", "op": "grad", "rows": 4096, "ids": 512, "F": 64, "table": "f16", "out": "f16",
         "scale": 1.0, "skew": False, "padding": False},
        # the gradient of the large lookup: most rows get little, the popular ones tens of thousands of sums
        {"name": "grad 1M in 1M F128 f16", "op": "grad", "rows": 1 << 20, "ids": 1 << 20, "F": 128, "table": "f16",
         "out": "f16", "scale": 1.0, "skew": True, "padding": False},
        # a training step of the lookup through autograd: rows out, gradient of the table back
        {"name": "train 200k of 50k F96 bf16", "op": "train", "rows": 50021, "ids": 200003, "F": 96, "table": "bf16",
         "out": "bf16", "scale": 9.75, "skew": False, "padding": True},
        # classify a few nodes of a small graph
        {"name": "classes 64x7 f16", "op": "classes", "n": 64, "C": 7, "type": "f16", "top": 1, "mask": "none", "scale": 1.0},
        # classify every node of a graph from fp32 logits, five alternatives each
        {"name": "classes 262k x47 f32 top5", "op": "classes", "n": 262144, "C": 47, "type": "f32", "top": 5, "mask": "none",
         "scale": 1.0},
        # one query scored against all nodes, eight best, with a temperature
        {"name": "classes 1x131k f16 top8", "op": "classes", "n": 1, "C": 1 << 17, "type": "f16", "top": 8, "mask": "none",
         "scale": 1.25},
        # link prediction with the known links of each query filtered out: a mask for every query, some leave nothing
        {"name": "classes 512x262k f16 masked", "op": "classes", "n": 512, "C": 1 << 18, "type": "f16", "top": 10,
         "mask": "full", "scale": 1.0},
        # training against all nodes: log probabilities and an entropy term, both with gradients, ragged rows
        {"name": "loss 4096x50k bf16", "op": "loss", "n": 4096, "C": 50021, "type": "bf16", "mask": "none", "scale": 1.0,
         "labelled": 1.0, "entropy": True},
        # the loss of a node classifier, a tenth of the nodes labelled
        {"name": "loss 262k x47 f16", "op": "loss", "n": 262144, "C": 47, "type": "f16", "mask": "none", "scale": 1.0,
         "labelled": 0.1, "entropy": False},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _width(rng):
    """Hidden sizes, other multiples of 8, and any number."""
    kind = rng.random()
    if kind < 0.4:
        return rng.choice((32, 64, 128, 256))
    if kind < 0.7:
        return 8 * _log_int(rng, 2, 64)
    return _log_int(rng, 5, 300)


def draw(rng):
    op = rng.choice(("lookup", "grad", "train", "classes", "classes", "loss"))
    if op in ("lookup", "grad", "train"):
        F = _width(rng)
        rows = _log_int(rng, 64, min(1 << 20, (1 << 27) // F) if op != "train" else min(1 << 18, (1 << 24) // F))
        ids = _log_int(rng, 1, min(1 << 20, (1 << 27) // F) if op != "train" else min(1 << 19, (1 << 25) // F))
        table = rng.choice(("f16", "f16", "bf16", "f32"))
        # an fp16 width of the fp32 tables' rows costs more bytes than the largest listed case where all are at their largest
        if table == "f32":
            rows, ids = max(rows // 2, 1), max(ids // 2, 1)
        return {"op": op, "rows": rows, "ids": ids, "F": F, "table": table,
                "out": rng.choice((table, table, "f16")) if op == "lookup" else table,
                "scale": rng.choice((1.0, 0.125, 9.75)), "skew": rng.random() < 0.5, "padding": rng.random() < 0.3}
    C = _log_int(rng, 2, 1 << 18)
    n = _log_int(rng, 1, min(1 << 18, ((1 << 27) if op == "loss" else (1 << 26)) // C))
    case = {"op": op, "n": n, "C": C, "type": rng.choice(("f16", "bf16", "f32")), "scale": rng.choice((1.0, 0.5, 1.25)),
            "mask": rng.choice(("none", "none", "class", "full"))}
    if op == "classes":
        return {**case, "top": rng.choice((0, 1, 5, 8, 16))}
    return {**case, "labelled": rng.choice((1.0, 1.0, 0.1)), "entropy": rng.random() < 0.5}


_MULTIPLIER = 1000003  # a prime, so that popular ids lie all over the table


def _ids(n, rows, skew, gen):
    u = torch.rand(n, generator=gen, device="cuda", dtype=torch.float64)
    if not skew:
        return (u * rows).long().clamp_(max=rows - 1)
    rank = torch.exp(u * math.log(rows)).long().clamp_(1, rows) - 1  # P(rank) ~ 1 / rank, as words and hubs have it
    return (rank * _MULTIPLIER) % rows


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def randn(shape, dtype, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    s = dict(case)
    if case["op"] in ("lookup", "grad", "train"):
        V, N, F = case["rows"], case["ids"], case["F"]
        s["idx"] = _ids(N, V, case["skew"], g)
        s["pad"] = None
        if case["padding"]:  # lists of ids filled up to a common length
            s["pad"] = 0
            s["idx"][torch.rand(N, generator=g, device="cuda") < 0.2] = 0
        if case["op"] != "grad":
            s["W"] = randn((V, F), _DT[case["table"]]).requires_grad_(case["op"] == "train")
        if case["op"] != "lookup":
            s["G"] = randn((N, F), _DT[case["out"]])
        return s
    n, C = case["n"], case["C"]
    # trained scores: a spread of a few units and, in most rows, one class ahead of the others
    x = torch.randn((n, C), generator=g, device="cuda").mul_(2.0)
    s["t"] = torch.randint(0, C, (n,), generator=g, device="cuda")
    x[torch.arange(n, device="cuda"), s["t"]] += 4.0 * torch.rand(n, generator=g, device="cuda")
    s["x"] = x.to(_DT[case["type"]])
    s["m"] = None
    if case["mask"] == "class":
        s["m"] = torch.rand(C, generator=g, device="cuda") < 0.9
    elif case["mask"] == "full":
        s["m"] = torch.rand((n, C), generator=g, device="cuda") < 0.9
        s["m"][7::61] = False  # queries for which nothing is left
    if case["op"] == "loss":
        s["t"][torch.rand(n, generator=g, device="cuda") >= case["labelled"]] = -1
        s["x"].requires_grad_()
        # the loss is a weighted mean over the rows; with fp16 scores it is scaled up, as gradients below 6e-8 would vanish
        unit = 256.0 if case["type"] == "f16" else 1.0 / n
        s["g_lp"] = -unit * torch.rand(n, generator=g, device="cuda")
        s["g_h"] = torch.full((n,), -0.01 * unit, device="cuda") if case["entropy"] else None
    return s


def _plain_lookup(s):
    y = s["W"].detach().float()[s["idx"]] * s["scale"]
    if s["pad"] is not None:
        y = y * (s["idx"] != s["pad"]).float()[:, None]
    return y.to(_DT[s["out"]])


def _plain_grad(s):
    G = s["G"].float()
    if s["pad"] is not None:
        G = G * (s["idx"] != s["pad"]).float()[:, None]
    acc = torch.zeros((s["rows"], s["F"]), device="cuda").index_add_(0, s["idx"], G)
    return (acc * s["scale"]).to(_DT[s["table"]])


def _plain_scores(s):
    x = s["x"].detach().float() * s["scale"]
    if s["m"] is not None:
        x = torch.where(s["m"], x, -math.inf)
    top = x.max(1, keepdim=True).values
    d = x - torch.where(top == -math.inf, 0.0, top)  # a row with nothing left stays at -inf
    e = torch.exp(d)
    S = e.sum(1, keepdim=True)
    log_S = torch.log(S)
    H = torch.where(S > 0, log_S - (e * d.clamp(min=-1e30)).sum(1, keepdim=True) / S.clamp(min=1.0), 0.0)
    return d, e, S, log_S, H


def _plain_logprobs(d, log_S, S, t):
    lp = d.gather(1, t.clamp(min=0)[:, None])
    lp = torch.where(S > 0, lp - log_S, -math.inf)[:, 0]
    return torch.where(t < 0, 0.0, lp)


def _plain_classes(s):
    d, e, S, log_S, H = _plain_scores(s)
    out = {"logprobs": _plain_logprobs(d, log_S, S, s["t"]), "entropy": H[:, 0]}
    if s["top"]:
        left, ids = s["x"].float(), []
        if s["m"] is not None:
            left = torch.where(s["m"], left, -math.inf)
        else:
            left = left.clone() if left is s["x"] else left
        for _ in range(min(s["top"], s["C"])):
            v, i = left.max(1)  # the first of equal ones
            ids.append(torch.where(v == -math.inf, -1, i))
            left.scatter_(1, i[:, None], -math.inf)
        ids += [torch.full_like(ids[0], -1)] * (s["top"] - len(ids))
        ids = torch.stack(ids, 1)
        lp = torch.where(ids < 0, -math.inf, d.gather(1, ids.clamp(min=0)) - log_S)
        out.update(top_logprobs=lp, top_ids=ids.to(torch.int32))
    return out


def _plain_loss(s):
    d, e, S, log_S, H = _plain_scores(s)
    out = {"logprobs": _plain_logprobs(d, log_S, S, s["t"]), "entropy": H[:, 0]}
    g = torch.where(s["t"] < 0, 0.0, s["g_lp"])[:, None]
    p = torch.where(S > 0, e / S.clamp(min=1.0), 0.0)
    w = g.expand_as(p)
    if s["g_h"] is not None:
        w = w + s["g_h"][:, None] * (d.clamp(min=-1e30) - log_S + H)
    dx = torch.where(p > 0, -p * w, 0.0)
    hit = torch.zeros_like(dx).scatter_(1, s["t"].clamp(min=0)[:, None], g)
    if s["m"] is not None:
        hit = torch.where(s["m"], hit, 0.0)
    out["grad"] = ((dx + hit) * s["scale"]).to(s["x"].dtype)
    return out


def run(s):
    if not own:
        if s["op"] == "lookup":
            return _plain_lookup(s)
        if s["op"] == "grad":
            return _plain_grad(s)
        if s["op"] == "train":
            return _plain_lookup(s), _plain_grad(s)
        return _plain_classes(s) if s["op"] == "classes" else _plain_loss(s)
    trspmm = _api()
    if s["op"] == "lookup":
        return trspmm.embedding(s["W"], s["idx"], scale=s["scale"], padding_id=s["pad"], out_dtype=_DT[s["out"]])
    if s["op"] == "grad":
        return trspmm.embedding_grad(s["G"], s["idx"], s["rows"], scale=s["scale"], padding_id=s["pad"])
    if s["op"] == "train":
        y = trspmm.embedding(s["W"], s["idx"], scale=s["scale"], padding_id=s["pad"])
        return y, torch.autograd.grad(y, s["W"], s["G"])[0]
    if s["op"] == "classes":
        r = trspmm.class_logprobs(s["x"], s["t"], top=s["top"], mask=s["m"], scale=s["scale"])
        out = {"logprobs": r.logprobs, "entropy": r.entropy}
        if s["top"]:
            out.update(top_logprobs=r.top_logprobs, top_ids=r.top_ids)
        return out
    r = trspmm.class_logprobs(s["x"], s["t"], mask=s["m"], scale=s["scale"], ignore_id=-1)
    if s["g_h"] is None:
        grad, = torch.autograd.grad(r.logprobs, s["x"], s["g_lp"])
    else:
        grad, = torch.autograd.grad((r.logprobs, r.entropy), s["x"], (s["g_lp"], s["g_h"]))
    return {"logprobs": r.logprobs, "entropy": r.entropy, "grad": grad}


def _distinct(case):
    """Expected number of table rows that the ids name."""
    V, N = case["rows"], case["ids"]
    if case["skew"] and V > 1:
        r = np.arange(1, V, dtype=np.float64)
        p = np.log1p(1.0 / r) / math.log(V)
    else:
        p = np.full(1, 1.0 / V)
    hit = -np.expm1(N * np.log1p(-np.minimum(p, 1.0 - 1e-12)))
    return float(hit.sum()) if hit.size > 1 or V == 1 else float(hit[0]) * V


def work(case):
    """Bytes: ids, each named table row and each gradient row once, each result once; scores, targets and masks once and
    the results once.  (The loss needs its scores once more only because they do not fit on the chip.)"""
    if case["op"] in ("lookup", "grad", "train"):
        V, N, F = case["rows"], case["ids"], case["F"]
        table, rows = F * _SIZE[case["table"]], F * _SIZE[case["out"]]
        fwd = 8 * N + _distinct(case) * table + N * rows
        bwd = 8 * N + N * rows + V * table
        return {"lookup": {"bytes": fwd, "flops": N * F}, "grad": {"bytes": bwd, "flops": N * F},
                "train": {"bytes": fwd + bwd - 8 * N, "flops": 2 * N * F}}[case["op"]]
    n, C = case["n"], case["C"]
    mask = {"none": 0, "class": C, "full": n * C}[case["mask"]]
    scores = n * C * _SIZE[case["type"]]
    if case["op"] == "classes":
        return {"bytes": scores + mask + 16 * n + 8 * n * case["top"], "flops": 6 * n * C}
    return {"bytes": 2 * scores + mask + 20 * n, "flops": 12 * n * C}


def exact(case, seed):
    s = prepare(case, seed)
    if s["op"] in ("lookup", "grad", "train"):
        idx, pad = s["idx"], s["pad"]
        keep = torch.ones_like(idx, dtype=torch.bool) if pad is None else idx != pad
        out = []
        if s["op"] != "grad":
            y = torch.zeros((idx.numel(), s["F"]), dtype=torch.float64, device="cuda")
            y[keep] = s["scale"] * s["W"].detach()[idx[keep]].double()
            out.append(y)
        if s["op"] != "lookup":
            acc = torch.zeros((s["rows"], s["F"]), dtype=torch.float64, device="cuda")
            acc.index_put_((idx[keep],), s["scale"] * s["G"][keep].double(), accumulate=True)
            out.append(acc)
        return out[0] if len(out) == 1 else tuple(out)
    n, C = s["n"], s["C"]
    step = max(1, (1 << 25) // C)
    parts = []
    for a in range(0, n, step):
        b = min(a + step, n)
        raw = s["x"].detach()[a:b].double()
        may = torch.isfinite(raw)
        if s["m"] is not None:
            may &= s["m"] if s["m"].dim() == 1 else s["m"][a:b]
        raw = raw.masked_fill(~may, -math.inf)
        z = raw * s["scale"]
        some = may.any(1)
        lse = torch.zeros(b - a, dtype=torch.float64, device="cuda")
        lse[some] = torch.logsumexp(z[some], 1)
        logp = z - lse[:, None]
        p = torch.exp(logp)
        finite_logp = logp.masked_fill(~may, 0.0)
        H = -(p * finite_logp).sum(1)
        t = s["t"][a:b]
        lp = logp[torch.arange(b - a, device="cuda"), t.clamp(min=0)].masked_fill(t < 0, 0.0)
        part = {"logprobs": lp, "entropy": H}
        if s["op"] == "classes" and s["top"]:
            order = torch.sort(raw, dim=1, descending=True, stable=True).indices[:, :s["top"]]
            if order.shape[1] < s["top"]:
                order = torch.nn.functional.pad(order, (0, s["top"] - order.shape[1]), value=-1)
            at = logp.gather(1, order.clamp(min=0)).masked_fill(order < 0, -math.inf)
            part.update(top_logprobs=at, top_ids=order.masked_fill(at == -math.inf, -1).to(torch.int32))
        if s["op"] == "loss":
            g = s["g_lp"][a:b].double().masked_fill(t < 0, 0.0)
            one = torch.zeros_like(p)
            one[torch.arange(b - a, device="cuda"), t.clamp(min=0)] = 1.0
            dz = g[:, None] * (one.masked_fill(~may, 0.0) - p)
            if s["g_h"] is not None:
                dz -= s["g_h"][a:b].double()[:, None] * p * (finite_logp + H[:, None])
            part["grad"] = s["scale"] * dz.masked_fill(~may, 0.0)
        parts.append(part)
    return {k: torch.cat([p[k] for p in parts]) for k in parts[0]}
