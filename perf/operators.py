"""Operators around the MoE block whose speed is measured, beside their plain forms.

Five operators of one served block:

  route      router probabilities to experts: softmax over all experts or
             sigmoid, a selection bias, groups, top-k, renormalised weights
  norm       the norm after a dense block, its gate and residual scale, and
             the norm before the next block
  moe_norm   the same behind routed experts: their combine goes straight in
  lora_add   low-rank adapters of many requests added to a shared projection
  lora_glu   the same on a gate|up projection, with the SwiGLU behind it

`own` false computes them with elementary torch operations (32 bits, the
router's scores in 64: a choice between near-equal experts is a border),
`own` true through the package's entry points.  Sizes follow
`grimoire_amd.configs` and the batch sizes of `perf/cases.py`.
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
EPS = 1e-6


def _route(name, T, E, K, **kw):
    c = dict(op="route", T=T, E=E, K=K, score="softmax", bias=False, n_group=1, topk_group=1, top2=False,
             normalize=True, scaling=1.0, bf16=False, masked=False, std=0.9)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _norm(name, op, T, H, **kw):
    c = dict(op=op, T=T, H=H, K=0, x_bf16=False, post=True, gate="none", gate_bf16=False, sigmoid=False,
             rscale=1.0, bscale=1.0, shared=False, out_bf=True, out_f=True)
    c.update(kw)
    return dict(name=name, **c) if name else c


def _lora(name, op, T, K, N, slots, R, **kw):
    c = dict(op=op, T=T, K=K, N=N, slots=slots, R=R, x_bf16=False, y_bf16=False, order="mixed", runs=1, none=0.1)
    c.update(kw)
    return dict(name=name, **c) if name else c


def listed():
    return [
        # one sequence decoding on a layer of 128 experts: latency alone
        _route("route_1", 1, 128, 8),
        # a draft of 32 tokens on a large layer: sigmoid scores, balance bias, the 4 best of 8 groups
        _route("route_32_groups", 32, 256, 8, score="sigmoid", bias=True, n_group=8, topk_group=4, top2=True,
               scaling=2.5, std=1.7),
        # a full prompt on 512 experts: probabilities kept as they are, balance bias for the choice
        _route("route_4096", 4096, 512, 10, bias=True, normalize=False),
        # eight sequences decoding, rows of 2880 elements; a learned gate per channel
        _norm("norm_8", "norm", 8, 2880, gate="channel"),
        # a prompt through a wide dense block: elementwise sigmoid gate, scaled residual
        _norm("norm_4096", "norm", 4096, 7168, x_bf16=True, gate="full", gate_bf16=True, sigmoid=True,
              rscale=0.9, bscale=1.25),
        # a verified draft behind the experts of a large layer, shared expert beside them
        _norm("moe_norm_32", "moe_norm", 32, 7168, K=8, shared=True, bscale=2.5),
        # a ragged prompt behind the experts: ten a token, one gate a token
        _norm("moe_norm_3001", "moe_norm", 3001, 2048, K=10, shared=True, gate="row", sigmoid=True),
        # one sequence with an adapter on the shared expert's down projection
        _lora("lora_add_1", "lora_add", 1, 768, 2048, 16, 16, none=0.0),
        # 48 sequences of 32 adapters decoding together, in no order
        _lora("lora_add_48", "lora_add", 48, 2048, 7168, 32, 64),
        # prompt chunks of 9 requests, one behind the other
        _lora("lora_add_4096", "lora_add", 4096, 2048, 7168, 32, 64, x_bf16=True, y_bf16=True, order="runs", runs=9),
        # a draft of 32 tokens on a wide gate|up projection: 4 requests of 8 tokens
        _lora("lora_glu_32", "lora_glu", 32, 7168, 4096, 16, 32, order="runs", runs=4),
        # a ragged prompt on the gate|up projection, fp32 activations
        _lora("lora_glu_2001", "lora_glu", 2001, 2880, 5760, 8, 16, order="runs", runs=5),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _cost(c):
    w = work(c)
    return w["bytes"] / 4e12 + w["flops"] / 0.5e15


def draw(rng):
    """A case of the same five operators: any number of tokens, sizes around
    and below the listed ones, every option."""
    top = max(_cost(c) for c in listed())
    while True:
        op = rng.choice(["route", "norm", "moe_norm", "lora_add", "lora_glu"])
        if op == "route":
            T = _log(rng, 1, 8192)
            n_group = rng.choice([1, 1, 2, 4, 8, 16])
            E = n_group * rng.randint(max(1, 16 // n_group), 512 // n_group)
            topk_group = rng.randint(1, n_group)
            K = min(rng.choice([1, 2, 4, 6, 8, 10, 16]), topk_group * (E // n_group))
            c = _route("", T, E, K, score=rng.choice(["softmax", "sigmoid"]), bias=rng.random() < 0.6,
                       n_group=n_group, topk_group=topk_group, top2=rng.random() < 0.5,
                       normalize=rng.random() < 0.5, scaling=rng.choice([1.0, 2.5]), bf16=rng.random() < 0.3,
                       masked=rng.random() < 0.3, std=rng.choice([0.5, 0.9, 1.7]))
        elif op in ("norm", "moe_norm"):
            moe = op == "moe_norm"
            c = _norm("", op, _log(rng, 1, 8192), 4 * _log(rng, 32, 2048),
                      K=rng.choice([1, 2, 4, 5, 8, 10]) if moe else 0, x_bf16=not moe and rng.random() < 0.5,
                      post=rng.random() < 0.8, gate=rng.choice(["none", "channel", "row", "full"]),
                      gate_bf16=rng.random() < 0.5, sigmoid=rng.random() < 0.5, rscale=rng.choice([1.0, 0.9, 1.4]),
                      bscale=rng.choice([1.0, 0.22, 2.5]), shared=moe and rng.random() < 0.5,
                      out_bf=rng.random() < 0.7)
            c["out_f"] = rng.random() < 0.7 or not c["out_bf"]
        else:
            T = _log(rng, 1, 4096)
            N = 8 * _log(rng, 32, 896)
            c = _lora("", op, T, 8 * _log(rng, 32, 896), N, rng.randint(1, 48), 16 * rng.choice([1, 1, 2, 4, 8]),
                      x_bf16=rng.random() < 0.5, y_bf16=rng.random() < 0.5,
                      order="mixed" if T <= 256 and rng.random() < 0.6 else "runs", runs=rng.randint(1, 12),
                      none=rng.choice([0.0, 0.1, 0.5]))
        if _cost(c) <= top:
            return c


# ------------------------------------------------------------------ inputs

def _gen(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 16 + 1)


def _rn(g, *shape):
    return torch.randn(shape, generator=g, device=DEV)


def _route_inputs(c, seed):
    g = _gen(seed)
    T, E = c["T"], c["E"]
    # router logits of normed activations; experts differ in popularity
    l = _rn(g, T, E) * c["std"] + _rn(g, E) * 0.5
    if c["masked"]:
        # experts taken out of service, by -inf; at least one stays in each group
        out = torch.rand((E,), generator=g, device=DEV) < 0.15
        out[::max(1, E // c["n_group"])] = False
        l[:, out] = -math.inf
    l = l.bfloat16() if c["bf16"] else l
    b = _rn(g, E) * (0.3 / E if c["score"] == "softmax" else 0.05) if c["bias"] else None
    return dict(logits=l, bias=b)


def _norm_inputs(c, seed):
    g = _gen(seed)
    T, H, K = c["T"], c["H"], c["K"]
    s = dict(h=_rn(g, T, H) * 4.0, post_w=None, gate=None, shared=None)
    if c["op"] == "norm":
        x = _rn(g, T, H) * 0.7
        s["x"] = x.bfloat16() if c["x_bf16"] else x
    else:
        s["routed"] = _rn(g, T * K, H).bfloat16()
        s["inverse"] = torch.randperm(T * K, generator=g, device=DEV).int()
        rw = torch.rand((T, K), generator=g, device=DEV) + 0.05
        s["rw"] = rw / rw.sum(1, keepdim=True)
        # a few routes whose expert is another rank's
        s["inverse"][torch.rand((T * K,), generator=g, device=DEV) < 0.05] = -1
        if c["shared"]:
            s["shared"] = _rn(g, T, H) * 0.5
    if c["post"]:
        s["post_w"] = (_rn(g, H) * 0.1).bfloat16()
    s["pre_w"] = (_rn(g, H) * 0.1).bfloat16()
    if c["gate"] != "none":
        n = {"channel": (H,), "row": (T,), "full": (T, H)}[c["gate"]]
        gate = _rn(g, *n) if c["sigmoid"] else 0.3 + _rn(g, *n) * 0.1
        s["gate"] = gate.bfloat16() if c["gate_bf16"] else gate
    return s


def _lora_inputs(c, seed):
    g = _gen(seed)
    T, K, N, S, R = c["T"], c["K"], c["N"], c["slots"], c["R"]
    # ranks of the adapters in their slots: full, half, quarter, 8; what lies
    # past a rank is left from an earlier tenant and is not part of the adapter
    rank = torch.tensor([R, R // 2, R // 4, 8], dtype=torch.int32, device=DEV)
    rank = rank[torch.randint(0, 4, (S,), generator=g, device=DEV)]
    a = (_rn(g, S, R, K) / math.sqrt(K)).bfloat16()
    b = (_rn(g, S, N, R) * 0.1).bfloat16()
    scale = torch.rand((S,), generator=g, device=DEV) * 1.5 + 0.5
    if c["order"] == "runs":
        cut = torch.sort(torch.randint(0, T + 1, (c["runs"] - 1,), generator=g, device=DEV)).values
        run = torch.bucketize(torch.arange(T, device=DEV), cut, right=True)
        slot = torch.randint(0, S, (c["runs"],), generator=g, device=DEV)
        slot[torch.rand((c["runs"],), generator=g, device=DEV) < c["none"]] = -1
        slot = slot[run]
    else:
        slot = torch.randint(0, S, (T,), generator=g, device=DEV)
        slot[torch.rand((T,), generator=g, device=DEV) < c["none"]] = -1
    x, base = _rn(g, T, K), _rn(g, T, N)
    return dict(a=a, b=b, rank=rank, scale=scale, slot=slot.int(),
                x=x.bfloat16() if c["x_bf16"] else x, base=base.bfloat16() if c["y_bf16"] else base)


INPUTS = {"route": _route_inputs, "norm": _norm_inputs, "moe_norm": _norm_inputs, "lora_add": _lora_inputs,
          "lora_glu": _lora_inputs}


def prepare(case, seed):
    c = case
    s = dict(c=c, **INPUTS[c["op"]](c, seed))
    f32 = dict(device=DEV, dtype=torch.float32)
    b16 = dict(device=DEV, dtype=torch.bfloat16)
    T = c["T"]
    if c["op"] == "route":
        s["ids"] = torch.empty((T, c["K"]), dtype=torch.int32, device=DEV)
        s["w"] = torch.empty((T, c["K"]), **f32)
    elif c["op"] in ("norm", "moe_norm"):
        s["h_out"] = torch.empty((T, c["H"]), **f32)
        s["out"] = torch.empty((T, c["H"]), **f32) if c["out_f"] else None
        s["out_bf"] = torch.empty((T, c["H"]), **b16) if c["out_bf"] else None
    else:
        n = c["N"] if c["op"] == "lora_add" else c["N"] // 2
        s["y"] = torch.empty((T, n), **(b16 if c["y_bf16"] else f32))
    if own:
        from grimoire_amd import ops, weights
        if c["op"] == "route":
            s["params"] = ops.RouteScores(score=c["score"], bias=s["bias"], n_group=c["n_group"],
                                          topk_group=c["topk_group"], group_score="top2" if c["top2"] else "max",
                                          normalize=c["normalize"], scaling=c["scaling"])
        elif c["op"] in ("norm", "moe_norm"):
            s["norm"] = ops.BlockNorm(s["pre_w"], s["post_w"], eps=EPS, weight_offset=1.0, residual_scale=c["rscale"],
                                      block_scale=c["bscale"], gate=c["gate"], gate_sigmoid=c["sigmoid"])
        else:
            s["lora"] = ops.Lora(weights.LoraAdapters(s["a"], s["b"], s["rank"], s["scale"]), T)
    return s


# ------------------------------------------------------------------ one pass

def _own(s):
    c = s["c"]
    if c["op"] == "route":
        s["params"](s["logits"], s["ids"], s["w"])
        return {"ids": s["ids"], "weights": s["w"]}
    if c["op"] == "norm":
        s["norm"](s["h"], s["x"], s["h_out"], s["out"], s["out_bf"], gate=s["gate"])
        return {"h": s["h_out"], "out": s["out"], "out_bf": s["out_bf"]}
    if c["op"] == "moe_norm":
        s["norm"].moe(s["h"], s["routed"], s["inverse"], s["rw"], s["shared"], s["h_out"], s["out"], s["out_bf"],
                      gate=s["gate"])
        return {"h": s["h_out"], "out": s["out"], "out_bf": s["out_bf"]}
    if c["op"] == "lora_add":
        s["lora"].add(s["slot"], s["x"], s["y"], base=s["base"])
    else:
        s["lora"].swiglu(s["slot"], s["x"], s["base"], s["y"])
    return {"y": s["y"]}


def _plain_route(s):
    c = s["c"]
    T, E, K, G = c["T"], c["E"], c["K"], c["n_group"]
    l = s["logits"].double()
    live = l > -math.inf
    if c["score"] == "softmax":
        e = torch.exp(l - l.amax(1, keepdim=True))
        score = e / e.sum(1, keepdim=True)
    else:
        score = 1.0 / (1.0 + torch.exp(-l))
    sel = score if s["bias"] is None else score + s["bias"].double()
    sel = torch.where(live, sel, -math.inf)
    if G > 1:
        per = torch.sort(sel.view(T, G, E // G), dim=2, descending=True).values
        gs = per[:, :, 0]
        if c["top2"] and E // G > 1:
            gs = gs + torch.where(per[:, :, 1] > -math.inf, per[:, :, 1], 0.0)
        best = torch.sort(gs, dim=1, descending=True, stable=True).indices[:, :c["topk_group"]]
        keep = (best[:, None, :] == torch.arange(G, device=DEV)[None, :, None]).any(2)
        sel = torch.where(keep[:, :, None], sel.view(T, G, E // G), -math.inf).view(T, E)
    val, idx = torch.sort(sel, dim=1, descending=True, stable=True)
    val, idx = val[:, :K], idx[:, :K]
    ok = val > -math.inf
    w = torch.where(ok, score.gather(1, idx), 0.0)
    if c["normalize"]:
        t = w.sum(1, keepdim=True)
        w = torch.where(t > 0, w / t, 0.0)
    return {"ids": torch.where(ok, idx, -1).int(), "weights": (w * c["scaling"]).float()}


def _plain_norm(s):
    c = s["c"]
    if c["op"] == "norm":
        f = s["x"].float()
    else:
        inv = s["inverse"].view(c["T"], c["K"]).long()
        rows = s["routed"][inv.clamp(min=0)].float()
        f = (rows * torch.where(inv >= 0, s["rw"], 0.0)[:, :, None]).sum(1)
        if s["shared"] is not None:
            f = f + s["shared"]
    if s["post_w"] is not None:
        f = f * torch.rsqrt((f * f).mean(1, keepdim=True) + EPS) * (1.0 + s["post_w"].float())
    if s["gate"] is not None:
        gate = s["gate"].float()
        gate = 1.0 / (1.0 + torch.exp(-gate)) if c["sigmoid"] else gate
        f = f * (gate[:, None] if c["gate"] == "row" else gate)
    h = c["rscale"] * s["h"] + c["bscale"] * f
    out = h * torch.rsqrt((h * h).mean(1, keepdim=True) + EPS) * (1.0 + s["pre_w"].float())
    return {"h": h, "out": out if c["out_f"] else None, "out_bf": out.bfloat16() if c["out_bf"] else None}


def _plain_lora(s):
    c = s["c"]
    T, K, N, S, R = c["T"], c["K"], c["N"], c["slots"], c["R"]
    # every adapter's product for every row, those of other rows' adapters
    # and past the ranks struck out
    mine = s["slot"][:, None, None] == torch.arange(S, device=DEV)[None, :, None]
    mine = mine & (torch.arange(R, device=DEV)[None, :] < s["rank"][:, None])[None]
    low = (s["x"].float() @ s["a"].float().view(S * R, K).T).view(T, S, R) * s["scale"][None, :, None]
    low = torch.where(mine, low, 0.0).view(T, S * R)
    y = s["base"].float() + low @ s["b"].float().transpose(1, 2).reshape(S * R, N)
    if c["op"] == "lora_glu":
        gate, up = y[:, :N // 2], y[:, N // 2:]
        y = gate / (1.0 + torch.exp(-gate)) * up
    return {"y": y.bfloat16() if c["y_bf16"] else y}


PLAIN = {"route": _plain_route, "norm": _plain_norm, "moe_norm": _plain_norm, "lora_add": _plain_lora,
         "lora_glu": _plain_lora}


def run(state):
    return _own(state) if own else PLAIN[state["c"]["op"]](state)


# ------------------------------------------------------------------ what a pass cannot do without

def work(case):
    c = case
    T = c["T"]
    if c["op"] == "route":
        return {"bytes": T * c["E"] * (2 if c["bf16"] else 4) + (4 * c["E"] if c["bias"] else 0) + 8 * T * c["K"],
                "flops": 10 * T * c["E"]}
    if c["op"] in ("norm", "moe_norm"):
        H, K = c["H"], c["K"]
        n = 8 * T * H + (4 if c["out_f"] else 0) * T * H + (2 if c["out_bf"] else 0) * T * H
        n += T * K * (2 * H + 8) if K else T * H * (2 if c["x_bf16"] else 4)
        n += 4 * T * H if c["shared"] else 0
        n += {"none": 0, "channel": H, "row": T, "full": T * H}[c["gate"]] * (2 if c["gate_bf16"] else 4)
        return {"bytes": n + 4 * H, "flops": T * H * (2 * K + 12)}
    K, N, S, R = c["K"], c["N"], c["slots"], c["R"]
    # distinct adapters that the rows are expected to name, at the mean rank
    draws = T if c["order"] == "mixed" else min(c["runs"], T)
    used = S * (1 - (1 - (1 - c["none"]) / S) ** draws)
    r = (R + R // 2 + R // 4 + 8) / 4
    out = N if c["op"] == "lora_add" else N // 2
    yb = 2 if c["y_bf16"] else 4
    return {"bytes": T * K * (2 if c["x_bf16"] else 4) + T * (N + out) * yb + used * r * (K + N) * 2 + 4 * T,
            "flops": 2 * T * (1 - c["none"]) * r * (K + N)}


# ------------------------------------------------------------------ the definitions in 64 bits

def _exact_route(c, seed):
    s = _route_inputs(c, seed)
    T, E, K, G = c["T"], c["E"], c["K"], c["n_group"]
    l = s["logits"].double()
    p = torch.softmax(l, 1) if c["score"] == "softmax" else torch.sigmoid(l)
    sel = p + (s["bias"].double() if s["bias"] is not None else 0.0)
    sel = sel.masked_fill(torch.isneginf(l), -math.inf)
    if G > 1:
        groups = sel.unflatten(1, (G, E // G))
        if c["top2"] and E // G > 1:
            two = groups.topk(2, 2).values
            rated = two[..., 0] + two[..., 1].masked_fill(torch.isneginf(two[..., 1]), 0.0)
        else:
            rated = groups.amax(2)
        order = torch.argsort(rated, dim=1, descending=True, stable=True)
        drop = torch.ones_like(rated, dtype=torch.bool).scatter_(1, order[:, :c["topk_group"]], False)
        sel = groups.masked_fill(drop[..., None], -math.inf).flatten(1)
    ids = torch.argsort(sel, dim=1, descending=True, stable=True)[:, :K]
    gone = torch.isneginf(sel.gather(1, ids))
    w = p.gather(1, ids).masked_fill(gone, 0.0)
    if c["normalize"]:
        w = torch.nan_to_num(w / w.sum(1, keepdim=True))
    return {"ids": ids.int().masked_fill(gone, -1), "weights": w * c["scaling"]}


def _rms(v):
    return v / torch.sqrt(v.square().mean(-1, keepdim=True) + EPS)


def _exact_norm(c, seed):
    s = _norm_inputs(c, seed)
    T, K = c["T"], c["K"]
    if c["op"] == "norm":
        f = s["x"].double()
    else:
        f = torch.zeros((T, c["H"]), dtype=torch.float64, device=DEV)
        for k in range(K):
            row = s["inverse"].view(T, K)[:, k].long()
            t = torch.nonzero(row >= 0)[:, 0]
            f.index_add_(0, t, s["routed"][row[t]].double() * s["rw"][t, k].double()[:, None])
        if c["shared"]:
            f += s["shared"].double()
    if c["post"]:
        f = _rms(f) * (s["post_w"].double() + 1.0)
    if c["gate"] != "none":
        gate = torch.sigmoid(s["gate"].double()) if c["sigmoid"] else s["gate"].double()
        f = f * (gate.unsqueeze(1) if c["gate"] == "row" else gate)
    h = s["h"].double() * c["rscale"] + f * c["bscale"]
    out = _rms(h) * (s["pre_w"].double() + 1.0)
    return {"h": h, "out": out if c["out_f"] else None, "out_bf": out if c["out_bf"] else None}


def _exact_lora(c, seed):
    s = _lora_inputs(c, seed)
    y = s["base"].double()
    for a in torch.unique(s["slot"]).tolist():
        if a < 0:
            continue
        t, r = torch.where(s["slot"] == a)[0], int(s["rank"][a])
        low = s["x"][t].double() @ s["a"][a, :r].double().T
        y[t] += low @ s["b"][a, :, :r].double().T.contiguous() * s["scale"][a].double()
    if c["op"] == "lora_glu":
        gate, up = y.chunk(2, 1)
        y = torch.nn.functional.silu(gate) * up
    return {"y": y}


def exact(case, seed):
    return {"route": _exact_route, "norm": _exact_norm, "moe_norm": _exact_norm, "lora_add": _exact_lora,
            "lora_glu": _exact_lora}[case["op"]](case, seed)
