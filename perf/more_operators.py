"""More operators around the MoE block whose speed is measured, beside their
plain forms.

What a layer that is built from single operators (its shared expert has
adapters, or its router is trained) needs next to the router scores, norms
and adapters of `perf/operators.py`:

  proj           a dense projection with 4-bit weights in groups (INT4 with
                 16-bit scales and zero points, MXFP4) for a few rows, added
                 to a base where there is one
  proj_glu       the same for a gate|up projection, with the SwiGLU behind it
  sort           tokens to rows in expert order, weighted where the weights
                 are applied before the experts
  sort_grad      its gradient: of the tokens and of the weights
  combine_grad   the gradient of the way back (weighted rows and a gated
                 shared expert summed per token)
  scores_grad    the gradient of the router scores' weights, to the logits

`own` false computes them with elementary torch operations in 32 bits, `own`
true through the package's entry points.  Sizes follow
`grimoire_amd.configs` and the batch sizes of `perf/cases.py`.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"


def _proj(name, op, T, K, N, fmt, **kw):
    c = dict(op=op, T=T, K=K, N=N, fmt=fmt, group=32 if fmt == "mxfp4" else 128, zeros="none", x_bf16=False,
             y_bf16=False, base=False)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _sort(name, op, T, E, K, H, **kw):
    c = dict(op=op, T=T, E=E, K=K, H=H, weighted=False, x_bf16=False, rows_bf16=True, zipf=0.0, out=0.0)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _comb(name, T, K, H, **kw):
    c = dict(op="combine_grad", T=T, K=K, H=H, dy_bf16=False, rows_bf16=True, shared="none", gate=False, out=0.05)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _score(name, T, E, K, **kw):
    c = dict(op="scores_grad", T=T, E=E, K=K, score="softmax", normalize=True, scaling=1.0, bf16=False, masked=False,
             std=0.9)
    c.update(kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one sequence decoding: the shared expert's down projection, latency alone
        _proj("proj_1", "proj", 1, 768, 2048, "int4_f16"),
        # one sequence on a wide projection (an output head): every weight read once for one row
        _proj("proj_wide_1", "proj", 1, 7168, 32768, "int4", zeros="signed"),
        # eight sequences decoding: gate|up of a shared expert, rows of 2880 elements
        _proj("proj_glu_8", "proj_glu", 8, 2880, 5760, "mxfp4", x_bf16=True, y_bf16=True),
        # a draft of 32 tokens being verified: a shared expert's gate|up with zero points, in groups of 64
        _proj("proj_glu_32", "proj_glu", 32, 7168, 4096, "int4", group=64, zeros="asym", x_bf16=True),
        # two sequences decoding, weights applied before the experts: latency
        _sort("sort_2", "sort", 2, 128, 8, 2048, weighted=True),
        # a full prompt on 512 experts of skewed popularity
        _sort("sort_4096", "sort", 4096, 512, 10, 2048, x_bf16=True, zipf=1.2),
        # a small training batch on wide rows
        _sort("sort_grad_32", "sort_grad", 32, 256, 8, 7168),
        # a ragged batch with weights applied before the experts: their gradient too
        _sort("sort_grad_3001", "sort_grad", 3001, 128, 4, 2880, weighted=True, x_bf16=True),
        # a small batch, rows in full precision
        _comb("combine_grad_8", 8, 4, 2880, rows_bf16=False),
        # a full prompt behind ten experts a token and a gated shared expert
        _comb("combine_grad_4096", 4096, 10, 2048, shared="bf16", gate=True),
        # sigmoid scores of a draft-sized batch
        _score("scores_grad_64", 64, 256, 8, score="sigmoid", scaling=2.5, std=1.7),
        # a full prompt, probabilities over all 512 experts kept as they are
        _score("scores_grad_4096", 4096, 512, 10, normalize=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 0.5e15


def draw(rng):
    """A case of the same operators: any number of rows, sizes around and
    below the listed ones, every format and option."""
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["proj", "proj", "proj_glu", "sort", "sort_grad", "combine_grad", "scores_grad"])
        if op in ("proj", "proj_glu"):
            fmt = rng.choice(["int4", "int4", "int4_f16", "mxfp4"])
            group = 32 if fmt == "mxfp4" else rng.choice([32, 64, 128, 128, 256])
            zeros = "none" if fmt == "mxfp4" else rng.choice(["none", "asym", "signed"])
            glu = op == "proj_glu"
            N = _log(rng, 64, 32768)
            c = _proj("", op, _log(rng, 1, 128), group * _log(rng, max(1, 256 // group), 8192 // group),
                      N + N % 2 if glu else N, fmt, group=group, zeros=zeros, x_bf16=rng.random() < 0.5,
                      y_bf16=rng.random() < 0.5, base=not glu and rng.random() < 0.4)
            if c["N"] * c["K"] > 32768 * 7168:
                continue
        elif op in ("sort", "sort_grad"):
            K = rng.choice([1, 2, 4, 6, 8, 10])
            c = _sort("", op, _log(rng, 1, 8192), rng.randint(max(8, K), 512), K, 8 * _log(rng, 16, 1024),
                      weighted=rng.random() < 0.5, x_bf16=rng.random() < 0.5, rows_bf16=rng.random() < 0.7,
                      zipf=rng.choice([0.0, 1.1]), out=rng.choice([0.0, 0.1, 0.5]))
        elif op == "combine_grad":
            shared = rng.choice(["none", "bf16", "f32"])
            c = _comb("", _log(rng, 1, 8192), rng.choice([1, 2, 4, 5, 8, 10]), 8 * _log(rng, 16, 1024),
                      dy_bf16=rng.random() < 0.5, rows_bf16=rng.random() < 0.7, shared=shared,
                      gate=shared != "none" and rng.random() < 0.5, out=rng.choice([0.0, 0.05, 0.5]))
        else:
            K = rng.choice([1, 2, 4, 6, 8, 10, 16])
            # a single pick's weight, renormalised, is constant: no gradient
            c = _score("", _log(rng, 1, 8192), rng.randint(16, 512), K, score=rng.choice(["softmax", "sigmoid"]),
                       normalize=K > 1 and rng.random() < 0.5,
                       scaling=rng.choice([1.0, 2.5]), bf16=rng.random() < 0.3, masked=rng.random() < 0.3,
                       std=rng.choice([0.5, 0.9, 1.7]))
        if _cost(c) <= top:
            return c


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 16 + 3)


def _rn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _b16(t, yes):
    return t.bfloat16() if yes else t


def _proj_inputs(c, seed):
    g = _gen(seed)
    T, K, N, G = c["T"], c["K"], c["N"], c["K"] // c["group"]
    s = dict(payload=torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, generator=g, device=DEV), zeros=None)
    if c["fmt"] == "mxfp4":
        s["scales"] = torch.randint(127 - 8, 127 - 1, (N, G), dtype=torch.uint8, generator=g, device=DEV)
    else:
        sc = (_rn(g, N, G) * 0.02).abs()
        s["scales"] = sc.half() if c["fmt"] == "int4_f16" else sc.bfloat16()
        if c["zeros"] == "asym":
            s["zeros"] = torch.randint(4, 12, (N, G), dtype=torch.uint8, generator=g, device=DEV)
        elif c["zeros"] == "signed":
            s["zeros"] = torch.full((N, G), 255, dtype=torch.uint8, device=DEV)
    s["x"] = _b16(_rn(g, T, K), c["x_bf16"])
    s["base"] = _b16(_rn(g, T, N), c["y_bf16"]) if c["base"] else None
    return s


def _ids(g, c):
    """Routes of T tokens to K distinct experts, popularity as a power of the
    rank; a share of them (`out`) to experts that are not here: -1."""
    T, E, K = c["T"], c["E"], c["K"]
    pop = torch.arange(1, E + 1, device=DEV, dtype=torch.float32) ** -c["zipf"]
    pop = pop[torch.randperm(E, generator=g, device=DEV)]
    gumbel = -torch.log(-torch.log(torch.rand((T, E), generator=g, device=DEV).clamp(1e-7, 1 - 1e-7)))
    ids = torch.topk(torch.log(pop) + gumbel, K, dim=1).indices.int()
    ids[torch.rand((T, K), generator=g, device=DEV) < c["out"]] = -1
    return ids


def _order(ids, E):
    """Row of each route in expert order; routes of no expert behind them."""
    key = torch.where((ids >= 0) & (ids < E), ids, E).flatten()
    at = torch.argsort(key, stable=True)
    pos = torch.empty_like(at)
    pos[at] = torch.arange(at.numel(), device=DEV)
    return pos


def _weights(g, T, K):
    w = torch.rand((T, K), generator=g, device=DEV) + 0.05
    return w / w.sum(1, keepdim=True)


def _sort_inputs(c, seed):
    g = _gen(seed)
    T, K, H = c["T"], c["K"], c["H"]
    s = dict(ids=_ids(g, c), x=_b16(_rn(g, T, H), c["x_bf16"]), weight=_weights(g, T, K) if c["weighted"] else None)
    if c["op"] == "sort_grad":
        s["drows"] = _b16(_rn(g, T * K, H), c["rows_bf16"])
        live = (s["ids"] >= 0).flatten()
        s["inverse"] = torch.where(live, _order(s["ids"], c["E"]), -1).int()
    return s


def _comb_inputs(c, seed):
    g = _gen(seed)
    T, K, H = c["T"], c["K"], c["H"]
    s = dict(dy=_b16(_rn(g, T, H), c["dy_bf16"]), rows=_b16(_rn(g, T * K, H), c["rows_bf16"]),
             inverse=torch.randperm(T * K, generator=g, device=DEV).int(), weight=_weights(g, T, K), shared=None,
             gate=None)
    # routes whose expert is another rank's
    s["inverse"][torch.rand((T * K,), generator=g, device=DEV) < c["out"]] = -1
    if c["shared"] != "none":
        s["shared"] = _b16(_rn(g, T, H), c["shared"] == "bf16")
    if c["gate"]:
        s["gate"] = torch.sigmoid(_rn(g, T))
    return s


def _score_inputs(c, seed):
    g = _gen(seed)
    T, E, K = c["T"], c["E"], c["K"]
    l = _rn(g, T, E) * c["std"] + _rn(g, E) * 0.5
    out = torch.zeros((E,), dtype=torch.bool, device=DEV)
    if c["masked"]:
        # experts taken out of service; a token may be left with fewer than K
        out = torch.rand((E,), generator=g, device=DEV) < 0.3
        out[0] = False
        l[:, out] = -math.inf
    l = _b16(l, c["bf16"])
    # picks: the K largest under a balance bias
    val, ids = torch.topk(l.float() + _rn(g, E) * 0.3, K, dim=1)
    return dict(logits=l, ids=torch.where(val > -math.inf, ids, -1).int(), dw=_rn(g, T, K))


INPUTS = {"proj": _proj_inputs, "proj_glu": _proj_inputs, "sort": _sort_inputs, "sort_grad": _sort_inputs,
          "combine_grad": _comb_inputs, "scores_grad": _score_inputs}


def prepare(case, seed):
    c = case
    s = dict(c=c, **INPUTS[c["op"]](c, seed))
    T = c["T"]

    def empty(shape, b16=False, dtype=None):
        return torch.empty(shape, dtype=dtype or (torch.bfloat16 if b16 else torch.float32), device=DEV)
    if c["op"] in ("proj", "proj_glu"):
        s["y"] = empty((T, c["N"] if c["op"] == "proj" else c["N"] // 2), c["y_bf16"])
    elif c["op"] == "sort":
        # rows behind the last route's keep what they hold: zeros here
        s["rows"] = empty((T * c["K"], c["H"]), c["rows_bf16"]).zero_()
        s["counts"], s["offsets"] = (empty((c["E"],), dtype=torch.int32) for _ in range(2))
        s["inverse"] = empty((T * c["K"],), dtype=torch.int32)
    elif c["op"] == "sort_grad":
        s["dx"] = empty((T, c["H"]), c["x_bf16"])
        s["dweight"] = empty((T, c["K"])) if c["weighted"] else None
    elif c["op"] == "combine_grad":
        s["drows"] = torch.zeros_like(s["rows"])
        s["dweight"] = empty((T, c["K"]))
        s["dshared"] = torch.empty_like(s["shared"]) if s["shared"] is not None else None
        s["dgate"] = empty((T,)) if c["gate"] else None
    else:
        s["dlogits"] = torch.empty_like(s["logits"])
    if own:
        from grimoire_amd import _abi, ops, weights
        if c["op"] in ("proj", "proj_glu"):
            fmt = {"int4": _abi.FMT_INT4, "int4_f16": _abi.FMT_INT4_F16, "mxfp4": _abi.FMT_MXFP4}[c["fmt"]]
            w = weights.Weight(fmt, c["N"], c["K"], s["payload"], s["scales"], s["zeros"], c["K"] // c["group"])
            s["proj"] = ops.Projection4(w, T)
        elif c["op"] in ("sort", "sort_grad"):
            s["sort"] = ops.TokenSort(c["E"], c["K"], T, device=DEV)
        elif c["op"] == "scores_grad":
            s["scores"] = ops.RouteScores(score=c["score"], normalize=c["normalize"], scaling=c["scaling"])
        else:
            s["combine_grad"] = ops.combine_grad
    return s


# ------------------------------------------------------------------ one pass

def _own(s):
    op = s["c"]["op"]
    if op == "proj":
        s["proj"](s["x"], s["y"], base=s["base"])
        return {"y": s["y"]}
    if op == "proj_glu":
        s["proj"].swiglu(s["x"], s["y"])
        return {"y": s["y"]}
    if op == "sort":
        s["sort"](s["ids"], s["x"], s["rows"], s["counts"], s["offsets"], s["inverse"], weight=s["weight"])
        return {k: s[k] for k in ("rows", "counts", "offsets", "inverse")}
    if op == "sort_grad":
        s["sort"].grad(s["drows"], s["inverse"], s["dx"], x=s["x"] if s["weight"] is not None else None,
                       weight=s["weight"], dweight=s["dweight"])
        return {"dx": s["dx"], "dweight": s["dweight"]}
    if op == "combine_grad":
        s["combine_grad"](s["dy"], s["rows"], s["inverse"], s["weight"], s["drows"], s["dweight"], shared=s["shared"],
                          gate=s["gate"], dshared=s["dshared"], dgate=s["dgate"])
        return {k: s[k] for k in ("drows", "dweight", "dshared", "dgate")}
    s["scores"].grad(s["logits"], s["ids"], s["dw"], s["dlogits"])
    return {"dlogits": s["dlogits"]}


def _plain_proj(s):
    c = s["c"]
    T, K, N, G = c["T"], c["K"], c["N"], c["K"] // c["group"]
    q = torch.stack((s["payload"] & 15, s["payload"] >> 4), dim=2).view(N, G, c["group"]).float()
    if c["fmt"] == "mxfp4":
        # e2m1: a sign, two bits of exponent, one of mantissa
        sign, m = 1.0 - 2.0 * (q >= 8).float(), torch.where(q >= 8, q - 8.0, q)
        v = torch.where(m < 4, m * 0.5, torch.where(m < 6, m - 2.0, 2.0 * m - 8.0)) * sign
        scale = torch.exp2(s["scales"].float() - 127.0)
    else:
        z = 8.0 if c["fmt"] == "int4_f16" else 0.0
        if s["zeros"] is not None:
            z = s["zeros"].float()[:, :, None]
            # 255: the codes are signed
            q, z = torch.where(z == 255.0, q - 16.0 * (q >= 8).float(), q), torch.where(z == 255.0, 0.0, z)
        v, scale = q - z, s["scales"].float()
    y = s["x"].float() @ (v * scale[:, :, None]).view(N, K).T
    if s["base"] is not None:
        y = y + s["base"].float()
    if c["op"] == "proj_glu":
        gate, up = y[:, :N // 2], y[:, N // 2:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return {"y": _b16(y, c["y_bf16"])}


def _plain_sort(s):
    c = s["c"]
    T, E, K, H = c["T"], c["E"], c["K"], c["H"]
    pos, live = _order(s["ids"], E), s["ids"] >= 0
    counts = (s["ids"].flatten()[:, None] == torch.arange(E, device=DEV, dtype=torch.int32)).sum(0)
    v = s["x"].float()[:, None, :] * (live.float() if s["weight"] is None else live * s["weight"])[:, :, None]
    rows = torch.empty((T * K, H), device=DEV)
    rows[pos] = v.view(T * K, H)
    return {"rows": _b16(rows, c["rows_bf16"]), "counts": counts.int(),
            "offsets": (torch.cumsum(counts, 0) - counts).int(), "inverse": torch.where(live.flatten(), pos, -1).int()}


def _plain_sort_grad(s):
    c = s["c"]
    T, K, H = c["T"], c["K"], c["H"]
    inv = s["inverse"].long()
    v = s["drows"][inv.clamp(min=0)].float() * (inv >= 0).float()[:, None]
    v = v.view(T, K, H)
    if s["weight"] is None:
        return {"dx": _b16(v.sum(1), c["x_bf16"]), "dweight": None}
    return {"dx": _b16((v * s["weight"][:, :, None]).sum(1), c["x_bf16"]),
            "dweight": (v * s["x"].float()[:, None, :]).sum(2)}


def _plain_combine_grad(s):
    c = s["c"]
    T, K, H = c["T"], c["K"], c["H"]
    inv, live = s["inverse"].long(), s["inverse"] >= 0
    dy = s["dy"].float()
    v = s["rows"][inv.clamp(min=0)].float() * live.float()[:, None]
    buf = torch.zeros((T * K + 1, H), device=DEV)           # the last row: of routes without one
    buf[torch.where(live, inv, T * K)] = (dy[:, None, :] * s["weight"][:, :, None]).view(T * K, H)
    out = {"drows": _b16(buf[:T * K], c["rows_bf16"]), "dweight": (v.view(T, K, H) * dy[:, None, :]).sum(2),
           "dshared": None, "dgate": None}
    if s["shared"] is not None:
        out["dshared"] = _b16(dy if s["gate"] is None else dy * s["gate"][:, None], c["shared"] == "bf16")
        if s["gate"] is not None:
            out["dgate"] = (dy * s["shared"].float()).sum(1)
    return out


def _plain_scores_grad(s):
    c = s["c"]
    l, live = s["logits"].float(), s["ids"] >= 0
    at = s["ids"].clamp(min=0).long()
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True))
        p = e / e.sum(1, keepdim=True)
    else:
        p = 1.0 / (1.0 + torch.exp(-l))
    u = torch.where(live, p.gather(1, at), 0.0)
    dw = torch.where(live, s["dw"], 0.0) * c["scaling"]
    if c["normalize"]:
        z = u.sum(1, keepdim=True)
        du = (dw - (dw * u).sum(1, keepdim=True) / z) / z
    else:
        du = dw
    ds = torch.zeros_like(l).scatter_add_(1, at, torch.where(live, du, 0.0))
    d = p * (ds - (u * du).sum(1, keepdim=True)) if c["score"] == "softmax" else ds * p * (1.0 - p)
    return {"dlogits": _b16(d, c["bf16"])}


PLAIN = {"proj": _plain_proj, "proj_glu": _plain_proj, "sort": _plain_sort, "sort_grad": _plain_sort_grad,
         "combine_grad": _plain_combine_grad, "scores_grad": _plain_scores_grad}


def run(state):
    return _own(state) if own else PLAIN[state["c"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    T, K = c["T"], c["K"]
    if c["op"] in ("proj", "proj_glu"):
        N, G = c["N"], K // c["group"]
        out = N if c["op"] == "proj" else N // 2
        per = 1 if c["fmt"] == "mxfp4" else 2 + (c["zeros"] != "none")
        return {"bytes": N * K // 2 + N * G * per + T * K * (2 if c["x_bf16"] else 4) +
                T * (out + (N if c["base"] else 0)) * (2 if c["y_bf16"] else 4), "flops": 2 * T * K * N}
    if c["op"] == "scores_grad":
        E, b = c["E"], 2 if c["bf16"] else 4
        # renormalised or sigmoid weights depend on the picks alone
        read = T * E if c["score"] == "softmax" and not c["normalize"] else T * K
        return {"bytes": (read + T * E) * b + 8 * T * K, "flops": 10 * read}
    H, rb = c["H"], 2 if c["rows_bf16"] else 4
    live = T * K * (1.0 - c["out"])
    if c["op"] == "combine_grad":
        n = T * H * (2 if c["dy_bf16"] else 4) + live * H * 2 * rb + T * K * 12
        if c["shared"] != "none":
            n += T * H * (2 if c["shared"] == "bf16" else 4) * (2 if c["gate"] else 1) + (8 * T if c["gate"] else 0)
        return {"bytes": n, "flops": 3 * live * H}
    xb = 2 if c["x_bf16"] else 4
    n = T * H * xb + live * H * rb + T * K * 4
    if c["op"] == "sort":
        return {"bytes": n + T * K * 4 + 8 * c["E"] + (4 * T * K if c["weighted"] else 0), "flops": live * H}
    if c["weighted"]:
        n += T * H * xb + T * K * 8
    return {"bytes": n, "flops": (4 if c["weighted"] else 1) * live * H}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_proj(c, seed):
    s = _proj_inputs(c, seed)
    K, N, per = c["K"], c["N"], c["group"]
    codes = torch.empty((N, K), dtype=torch.int64, device=DEV)
    codes[:, 0::2] = s["payload"] % 16
    codes[:, 1::2] = s["payload"] // 16
    if c["fmt"] == "mxfp4":
        values = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6], dtype=torch.float64, device=DEV)
        w = torch.cat((values, -values))[codes]
        scale = torch.pow(2.0, s["scales"].double() - 127.0)
    else:
        scale = s["scales"].double()
        if s["zeros"] is None:
            w = (codes - (8 if c["fmt"] == "int4_f16" else 0)).double()
        else:
            z = torch.repeat_interleave(s["zeros"].long(), per, dim=1)
            w = torch.where(z == 255, (codes ^ 8) - 8, codes - z).double()
    w *= torch.repeat_interleave(scale, per, dim=1)
    y = torch.matmul(w, s["x"].double().T.contiguous()).T
    if c["op"] == "proj_glu":
        gate, up = y.chunk(2, dim=1)
        return {"y": torch.nn.functional.silu(gate) * up}
    return {"y": y if s["base"] is None else y + s["base"].double()}


def _exact_sort(c, seed):
    s = _sort_inputs(c, seed)
    T, E, K, H = c["T"], c["E"], c["K"], c["H"]
    ids = s["ids"].flatten()
    counts = torch.bincount(ids[ids >= 0].long(), minlength=E)
    routes = torch.argsort(ids, stable=True)[int((ids < 0).sum()):]     # those of an expert, by expert, in order
    inverse = torch.full_like(ids, -1)
    inverse[routes] = torch.arange(routes.numel(), dtype=torch.int32, device=DEV)
    rows = torch.zeros((T * K, H), dtype=torch.float64, device=DEV)
    rows[:routes.numel()] = s["x"].double()[torch.div(routes, K, rounding_mode="floor")]
    if c["weighted"]:
        rows[:routes.numel()] *= s["weight"].double().flatten()[routes, None]
    return {"rows": rows, "counts": counts.int(), "offsets": (counts.cumsum(0) - counts).int(), "inverse": inverse}


def _exact_sort_grad(c, seed):
    s = _sort_inputs(c, seed)
    T, K = c["T"], c["K"]
    x = s["x"].double().requires_grad_()
    w = (s["weight"].double() if c["weighted"] else torch.ones((T, K), dtype=torch.float64, device=DEV)).requires_grad_()
    r = torch.nonzero(s["inverse"] >= 0)[:, 0]
    rows = x[torch.div(r, K, rounding_mode="floor")] * w.flatten()[r, None]
    dx, dw = torch.autograd.grad(rows, (x, w), s["drows"][s["inverse"][r].long()].double())
    return {"dx": dx, "dweight": dw if c["weighted"] else None}


def _exact_combine_grad(c, seed):
    s = _comb_inputs(c, seed)
    T, K = c["T"], c["K"]
    leaf = {k: s[k].double().requires_grad_() for k in ("rows", "weight", "shared", "gate") if s[k] is not None}
    y = torch.zeros((T, c["H"]), dtype=torch.float64, device=DEV)
    for k in range(K):
        row = s["inverse"].view(T, K)[:, k].long()
        t = torch.nonzero(row >= 0)[:, 0]
        y = y.index_add(0, t, leaf["rows"][row[t]] * leaf["weight"][t, k][:, None])
    if "shared" in leaf:
        y = y + (leaf["shared"] * leaf["gate"][:, None] if "gate" in leaf else leaf["shared"])
    grads = dict(zip(leaf, torch.autograd.grad(y, list(leaf.values()), s["dy"].double())))
    return {"drows": grads["rows"], "dweight": grads["weight"], "dshared": grads.get("shared"),
            "dgate": grads.get("gate")}


def _exact_scores_grad(c, seed):
    s = _score_inputs(c, seed)
    l = s["logits"].double().requires_grad_()
    p = torch.softmax(l, 1) if c["score"] == "softmax" else torch.sigmoid(l)
    live = s["ids"] >= 0
    w = p.gather(1, s["ids"].long().clamp(min=0)).masked_fill(~live, 0.0)
    if c["normalize"]:
        w = w / w.sum(1, keepdim=True)
    return {"dlogits": torch.autograd.grad(w * c["scaling"], l, s["dw"].double().masked_fill(~live, 0.0))[0]}


EXACT = {"proj": _exact_proj, "proj_glu": _exact_proj, "sort": _exact_sort, "sort_grad": _exact_sort_grad,
         "combine_grad": _exact_combine_grad, "scores_grad": _exact_scores_grad}


def exact(case, seed):
    return EXACT[case["op"]](case, seed)
