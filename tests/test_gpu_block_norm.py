"""The norms around a block (grimoire_block_norm, grimoire_moe_block_norm)
against the formulas in 64 bits.

Tolerances, u = 2^-24.  A row's sum of squares adds terms of one sign: at
most 32 in a thread, 6 across a wave, 16 across the waves, so it is off by
at most 55 u relative and its rsqrt by half of that plus 2 u; with the four
products behind it p is off by at most 34 u of |p|.  The combine's chain of
up to 17 terms is off by 17 u of the sum of their absolute values, a sigmoid
gate of |g| <= 6 by at most 14 u (1.45 |g| for the exponent, 2 each for exp2,
sum and reciprocal).  So h' is off by at most 72 u of
(|rs h| + |bs g| P), P the norm of the sum of absolute values, and o by the
same plus 34 u of itself.  A bf16 output adds half a step, 2^-8."""
import pytest
import torch

from grimoire_amd import _abi, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(T, H, K, seed, gate="none", gate_bf16=False, sigmoid=False, x_bf16=False, post=True, shared=False, rs=0.9,
         bs=1.25, offset=1.0, eps=1e-6):
    g = gen(seed)
    rn = lambda *s: torch.randn(s, generator=g)
    d = dict(T=T, H=H, K=K, gate_kind=gate, sigmoid=sigmoid, rs=rs, bs=bs, offset=offset, eps=eps, shared=None,
             gate=None, post=None)
    d["h"] = rn(T, H) * 3
    if K:
        R = max(1, T * K - T * K // 5)
        d["routed"] = rn(R, H).bfloat16()
        inv = torch.cat([torch.arange(R), torch.full((T * K - R,), -1)])[torch.randperm(T * K, generator=g)]
        d["inverse"] = inv.int()
        d["rw"] = torch.rand((T, K), generator=g) + 0.05
        if shared:
            d["shared"] = rn(T, H)
    else:
        x = rn(T, H)
        d["x"] = x.bfloat16() if x_bf16 else x
    if post:
        d["post"] = (rn(H) * 0.2).bfloat16()
    d["pre"] = (rn(H) * 0.2).bfloat16()
    if gate != "none":
        v = rn(*{"channel": (H,), "row": (T,), "full": (T, H)}[gate]).clamp(-6, 6)
        d["gate"] = v.bfloat16() if gate_bf16 else v
    return d


def want(d):
    """h', o and the magnitudes their tolerances are taken of, in fp64."""
    T, H, K = d["T"], d["H"], d["K"]
    if K:
        f, fa = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
        if d["shared"] is not None:
            f += d["shared"].double()
            fa += d["shared"].double().abs()
        for k in range(K):
            p = d["inverse"].view(T, K)[:, k].long()
            e = torch.where((p >= 0)[:, None], d["routed"][p.clamp(min=0)].double(), 0.0)
            f += d["rw"][:, k, None].double() * e
            fa += d["rw"][:, k, None].double() * e.abs()
    else:
        f = d["x"].double()
        fa = f.abs()
    c = 1.0
    if d["post"] is not None:
        c = torch.rsqrt(f.square().mean(1, keepdim=True) + d["eps"]) * (d["offset"] + d["post"].double())
    g = 1.0
    if d["gate"] is not None:
        g = d["gate"].double()
        g = torch.sigmoid(g) if d["sigmoid"] else g
        g = g[:, None] if d["gate_kind"] == "row" else g
    rs, bs = (float(torch.tensor(v, dtype=torch.float32)) for v in (d["rs"], d["bs"]))
    hh = rs * d["h"].double() + bs * g * c * f
    mag = (rs * d["h"].double()).abs() + (bs * g * c * fa).abs()
    hs = torch.rsqrt(hh.square().mean(1, keepdim=True) + d["eps"]) * (d["offset"] + d["pre"].double())
    return hh, mag, hh * hs, hs.abs()


def run(d, gpu, inplace=False, out=True, out_bf=True, x=None, stream=None):
    T, H = d["T"], d["H"]
    mv = lambda t: None if t is None else t.to(gpu)
    n = ops.BlockNorm(mv(d["pre"]), mv(d["post"]), eps=d["eps"], weight_offset=d["offset"], residual_scale=d["rs"],
                      block_scale=d["bs"], gate=d["gate_kind"], gate_sigmoid=d["sigmoid"])
    h = d["h"].to(gpu)
    ho = h if inplace else torch.full((T, H), float("nan"), device=gpu)
    o = torch.full((T, H), float("nan"), device=gpu) if out else None
    ob = torch.full((T, H), float("nan"), device=gpu, dtype=torch.bfloat16) if out_bf else None
    torch.cuda.synchronize()
    if d["K"]:
        n.moe(h, mv(d["routed"]), mv(d["inverse"]), mv(d["rw"]), mv(d["shared"]), ho, o, ob, gate=mv(d["gate"]),
              stream=stream)
    else:
        n(h, mv(d["x"]) if x is None else x, ho, o, ob, gate=mv(d["gate"]), stream=stream)
    torch.cuda.synchronize()
    return ho.cpu(), None if o is None else o.cpu(), None if ob is None else ob.cpu()


def check(d, gpu, **kw):
    h, o, ob = run(d, gpu, **kw)
    hh, mag, oo, hs = want(d)
    assert ((h.double() - hh).abs() <= 72 * U * mag).all()
    tol = 72 * U * mag * hs + 34 * U * oo.abs() + 1e-44
    if o is not None:
        assert ((o.double() - oo).abs() <= tol).all()
    if ob is not None:
        assert ((ob.double() - oo).abs() <= tol + oo.abs() * (2.0 ** -8 + U)).all()


# one chunk, odd numbers of chunks, each work-group size and its border
@pytest.mark.parametrize("T,H", [(1, 4), (3, 256), (2, 260), (8, 2880), (5, 1028), (3, 2052), (4, 4100), (33, 7168),
                                 (2, 8196), (2, 16388), (1, 32768)])
@pytest.mark.parametrize("bf16", [False, True])
def test_dense(gpu, T, H, bf16):
    print(f"block_norm T={T} H={H} bf16={bf16}", flush=True)
    check(make(T, H, 0, T + H, x_bf16=bf16, gate="channel", gate_bf16=bf16), gpu)
    check(make(T, H, 0, T + H, x_bf16=bf16, post=False, rs=1.0, bs=1.0), gpu, inplace=True)


@pytest.mark.parametrize("gate", ["none", "channel", "row", "full"])
@pytest.mark.parametrize("gate_bf16", [False, True])
@pytest.mark.parametrize("sigmoid", [False, True])
def test_gates(gpu, gate, gate_bf16, sigmoid):
    d = make(6, 516, 0, 1, gate=gate, gate_bf16=gate_bf16, sigmoid=sigmoid and gate != "none")
    check(d, gpu)
    check(make(6, 516, 3, 2, gate=gate, gate_bf16=gate_bf16, sigmoid=sigmoid and gate != "none"), gpu, inplace=True)


@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 8, 9, 10, 11, 16])
def test_experts(gpu, K):
    print(f"moe_block_norm K={K}", flush=True)
    check(make(13, 2048, K, K, shared=K % 2 == 0), gpu)
    check(make(2, 7168, K, K + 20, shared=K % 2 == 1, post=False, offset=0.0), gpu)


def test_no_rows_here(gpu):
    """Tokens whose every route is another rank's: f = 0 (or the shared
    expert alone), and rows past routed_rows are not read."""
    d = make(4, 512, 4, 7)
    d["inverse"][:] = -1
    d["inverse"][5] = d["routed"].shape[0]          # one past the end
    d["inverse"][6] = 2 ** 31 - 1
    h, o, _ = run(d, gpu)
    rs = torch.tensor(d["rs"], dtype=torch.float32)
    assert torch.equal(h, rs * d["h"])
    assert torch.isfinite(o).all()


def test_zero_and_special_rows(gpu):
    """A zero row stays zero (eps), a NaN or infinite row stays its own row's matter."""
    d = make(5, 1024, 0, 9, rs=1.0)
    d["x"][0] = 0
    d["h"][0] = 0
    d["x"][2, 7] = float("nan")
    d["x"][3, 1] = float("inf")
    h, o, ob = run(d, gpu)
    assert (h[0] == 0).all() and (o[0] == 0).all()
    assert torch.isnan(o[2]).all()
    assert not torch.isfinite(o[3, 1])
    hh, mag, oo, hs = want(d)
    for t in (1, 4):
        assert ((h[t].double() - hh[t]).abs() <= 72 * U * mag[t]).all()
        assert ((o[t].double() - oo[t]).abs() <= 72 * U * mag[t] * hs[t] + 34 * U * oo[t].abs()).all()


def test_outputs_chosen(gpu):
    d = make(3, 640, 0, 11)
    check(d, gpu, out=False)
    check(d, gpu, out_bf=False)
    check(d, gpu, out=False, out_bf=False)
    d["pre"] = None
    h, _, _ = run(d, gpu, out=False, out_bf=False)
    d["pre"] = torch.zeros(640).bfloat16()
    assert ((h.double() - want(d)[0]).abs() <= 72 * U * want(d)[1]).all()


def test_rows_apart_stream_and_graph(gpu):
    """x as columns of a wider projection, another stream, a captured call
    replayed on new inputs (in place: the residual moves on each replay)."""
    d = make(9, 384, 0, 13, x_bf16=True)
    wide = torch.full((9, 1000), float("nan"), dtype=torch.bfloat16, device=gpu)
    wide[:, 200:584] = d["x"].to(gpu)
    check(d, gpu, x=wide[:, 200:584])
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    check(d, gpu, x=wide[:, 200:584], stream=s)

    n = ops.BlockNorm(d["pre"].to(gpu), d["post"].to(gpu), residual_scale=0.5)
    h, x = d["h"].to(gpu), d["x"].to(gpu)
    o = torch.empty(9, 384, device=gpu)
    n(h.clone(), x, torch.empty_like(h), o)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        n(h, x, h, o)
    h.copy_(d["h"])
    he, oe = d["h"].to(gpu), torch.empty_like(o)
    for i in range(3):
        x.copy_(torch.randn(9, 384, generator=gen(50 + i)).bfloat16())
        g.replay()
        n(he, x, he, oe)
        torch.cuda.synchronize()
        assert torch.equal(h, he) and torch.equal(o, oe)


def test_python_refusals(gpu):
    d = make(4, 64, 0, 15)
    n = ops.BlockNorm(d["pre"].to(gpu), d["post"].to(gpu))
    h, x, o = d["h"].to(gpu), d["x"].to(gpu), torch.empty(4, 64, device=gpu)
    for bad in (dict(x=x[:, :32]), dict(x=x.double()), dict(x=x.t()), dict(h_out=o[:2]), dict(out=o.t()),
                dict(gate=o), dict(out_bf=o), dict(h=h.bfloat16())):
        kw = dict(h=h, x=x, h_out=o, out=None)
        kw.update(bad)
        with pytest.raises(_abi.GrimoireError):
            n(**kw)
    with pytest.raises(_abi.GrimoireError):
        n(h, x.cpu(), o)
    with pytest.raises(_abi.GrimoireError):
        ops.BlockNorm(None)(h, x, o, out=o.clone())
