"""Low-rank adapters beside a projection (grimoire_lora_add,
grimoire_lora_swiglu) against the formula in 64 bits.

Tolerances, u = 2^-23 (a step of the matrix core's fp32 sums, cut off or
rounded).  Products are exact (bf16 weights, fp32 activations in three exact
bf16 pieces).  z = A x: 32 steps inside an instruction, at most 3 K / 128 in
a wave's chain, 4 waves and 8 splits: off by (32 + 3 K / 128 + 12) u of
sum |a x|; the scale is one more step.  B z adds 16 + 3 R / 16 steps of
sum |b| |z|, base one.  silu(g) u: (2 |g| + 8) u of itself, and a change of g
moves it by at most 1.1 |u|.  A bf16 output adds half a step, 2^-8."""
import pytest
import torch

from grimoire_amd import _abi, ops, weights

pytestmark = pytest.mark.gpu
U = 2.0 ** -23


def gen(seed):
    return torch.Generator().manual_seed(seed)


def make(T, K, N, slots, R, seed, order="mixed", x_bf16=False, y_bf16=False, ranks=None):
    g = gen(seed)
    rn = lambda *s: torch.randn(s, generator=g)
    rank = torch.randint(0, R + 1, (slots,), generator=g) if ranks is None else torch.tensor(ranks)
    a, b = (rn(slots, R, K) / K ** 0.5).bfloat16(), (rn(slots, N, R) * 0.3).bfloat16()
    for s in range(slots):                  # past the rank lies anything
        a[s, rank[s]:] = float("nan")
        b[s, :, rank[s]:] = float("inf")
    if order == "mixed":
        slot = torch.randint(-1, slots, (T,), generator=g)
    elif order == "runs":
        cut = torch.sort(torch.randint(0, T + 1, (6,), generator=g)).values
        slot = torch.randint(-1, slots, (7,), generator=g)[torch.bucketize(torch.arange(T), cut, right=True)]
    else:
        slot = torch.full((T,), int(order))
    x, base = rn(T, K), rn(T, N)
    return dict(T=T, K=K, N=N, R=R, slots=slots, a=a, b=b, rank=rank.int(), slot=slot.int(),
                scale=torch.rand((slots,), generator=g) + 0.5, x=x.bfloat16() if x_bf16 else x,
                base=base.bfloat16() if y_bf16 else base)


def want(d):
    """base + delta in fp64, and the magnitude of delta's tolerance."""
    v, mag = d["base"].double(), torch.zeros(d["T"], d["N"], dtype=torch.float64)
    for s in range(d["slots"]):
        t, r = torch.where(d["slot"] == s)[0], int(d["rank"][s])
        if not len(t) or not r:
            continue
        x, a, b, c = d["x"][t].double(), d["a"][s, :r].double(), d["b"][s, :, :r].double(), float(d["scale"][s])
        v[t] += c * (x @ a.T) @ b.T
        mag[t] = c * (x.abs() @ a.abs().T) @ b.abs().T
    K, R = d["K"], d["R"]
    return v, (32 + 3 * K / 128 + 12 + 1 + 16 + 3 * R / 16 + 1) * U * mag + U * (d["base"].double().abs() + v.abs())


def want_glu(d):
    v, tol = want(d)
    I = d["N"] // 2
    g, u, tg, tu = v[:, :I], v[:, I:], tol[:, :I], tol[:, I:]
    s = g * torch.sigmoid(g)
    return s * u, 1.1 * tg * (u.abs() + tu) + s.abs() * tu + (2 * g.abs() + 8) * U * (s * u).abs() + 1e-30


def run(d, gpu, glu=False, y_bf16=False, inplace=False, lora=None, x=None, base=None, y=None, stream=None):
    mv = lambda t: t.to(gpu)
    if lora is None:
        lora = ops.Lora(weights.LoraAdapters(mv(d["a"]), mv(d["b"]), mv(d["rank"]), mv(d["scale"])), d["T"])
        lora.workspace.fill_(255)           # NaN: nothing of it may count
    x = mv(d["x"]) if x is None else x
    base = mv(d["base"]) if base is None else base
    if inplace:
        y = base
    elif y is None:
        y = torch.full((d["T"], d["N"] // 2 if glu else d["N"]), float("nan"), device=gpu,
                       dtype=torch.bfloat16 if y_bf16 else torch.float32)
    slot = mv(d["slot"])
    torch.cuda.synchronize()
    if glu:
        lora.swiglu(slot, x, base, y, stream=stream)
    else:
        lora.add(slot, x, y, base=None if inplace else base, stream=stream)
    torch.cuda.synchronize()
    return y.cpu()


def check(d, gpu, glu=False, y_bf16=False, **kw):
    y = run(d, gpu, glu, y_bf16, **kw)
    v, tol = want_glu(d) if glu else want(d)
    if y.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (v.abs() + tol)
    err = (y.double() - v).abs()
    assert (err <= tol).all(), float((err / tol).max())
    return y


SIZES = [(1, 768, 2048, 16, 16), (1, 8, 4, 1, 16), (2, 64, 8, 3, 32), (5, 72, 20, 2, 16), (16, 256, 64, 4, 48),
         (17, 520, 136, 40, 64), (33, 1000, 260, 5, 128), (100, 2048, 512, 32, 64), (48, 136, 40, 64, 256),
         (200, 7168, 96, 9, 16)]


@pytest.mark.parametrize("T,K,N,slots,R", SIZES)
@pytest.mark.parametrize("x_bf16", [False, True])
@pytest.mark.parametrize("y_bf16", [False, True])
def test_short_batches(gpu, T, K, N, slots, R, x_bf16, y_bf16):
    print(f"lora T={T} K={K} N={N} slots={slots} R={R}", flush=True)
    for order in ("mixed", "runs"):
        d = make(T, K, N, slots, R, T + K, order, x_bf16, y_bf16)
        check(d, gpu, y_bf16=y_bf16)
        check(d, gpu, inplace=True)
        check(d, gpu, y_bf16=not y_bf16)
    if N % 8 == 0:
        check(make(T, K, N, slots, R, T + N, "mixed", x_bf16, y_bf16), gpu, glu=True, y_bf16=y_bf16)
        check(make(T, K, N, slots, R, T + N, "runs", x_bf16, y_bf16), gpu, glu=True, y_bf16=not y_bf16)


@pytest.mark.parametrize("T,K,N,slots,R", [(513, 512, 136, 4, 16), (700, 264, 520, 12, 64), (1031, 136, 72, 3, 256),
                                           (2050, 64, 8, 30, 32), (512, 768, 264, 8, 128)])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_long_batches(gpu, T, K, N, slots, R, x_bf16):
    """Around and past the size where rows are taken as runs; mixed rows too."""
    print(f"lora T={T} K={K} N={N} slots={slots} R={R}", flush=True)
    for order in ("runs", "mixed", "0"):
        d = make(T, K, N, slots, R, T + K, order, x_bf16)
        check(d, gpu, inplace=order == "runs")
        check(d, gpu, glu=True)
    d = make(T, K, N, slots, R, 5, "runs", x_bf16, True)
    check(d, gpu, y_bf16=True)
    check(d, gpu, glu=True, y_bf16=True)


@pytest.mark.parametrize("T", [1, 40, 600])
def test_rows_without_adapter(gpu, T):
    """No adapter, a slot out of range, rank 0: base as it is, bit for bit
    (in place nothing is written); ranks past max_rank count as max_rank."""
    d = make(T, 128, 64, 3, 16, T, "-1")
    assert torch.equal(run(d, gpu), d["base"])
    for bad in (3, 2 ** 31 - 1, -2 ** 31):
        d["slot"][:] = bad
        assert torch.equal(run(d, gpu), d["base"])
        assert torch.equal(run(d, gpu, inplace=True), d["base"])
        check(d, gpu, glu=True)
    d = make(T, 128, 64, 3, 16, T, "1", ranks=[4, 0, 4])
    assert torch.equal(run(d, gpu), d["base"])
    d = make(T, 128, 64, 3, 16, T, "mixed", ranks=[16, 16, 16])
    full = run(d, gpu)
    d["rank"][:] = torch.tensor([17, 2 ** 31 - 1, 16])
    assert torch.equal(run(d, gpu), full)
    d["rank"][:] = -5
    assert torch.equal(run(d, gpu), d["base"])


@pytest.mark.parametrize("T,order", [(64, "mixed"), (700, "runs")])
def test_a_row_does_not_depend_on_the_others(gpu, T, order):
    """The same row alone among other adapters' rows gives the same bits, and
    a NaN or infinite row stays its own matter."""
    d = make(T, 512, 128, 6, 32, 3, order)
    y = run(d, gpu)
    e = dict(d, x=d["x"].clone(), slot=d["slot"].clone())
    keep = torch.arange(T) % 3 == 0
    e["slot"][~keep] = (e["slot"][~keep] + 2) % 6
    e["x"][1] = float("nan")
    e["x"][2] = float("inf")
    e["x"][4, 5] = 3.4e38
    z = run(e, gpu)
    assert torch.equal(y[keep], z[keep])
    assert torch.equal(run(d, gpu), y)
    # an adapter of NaNs is its own rows' matter too
    n = dict(d, a=d["a"].clone(), b=d["b"].clone(), scale=d["scale"].clone())
    n["a"][2], n["b"][2], n["scale"][2] = float("nan"), float("inf"), float("nan")
    z = run(n, gpu)
    assert torch.equal(y[d["slot"] != 2], z[d["slot"] != 2])


@pytest.mark.parametrize("T,K,N", [(1, 2048, 264), (1, 2056, 264), (7, 520, 2056), (16, 2048, 2048), (16, 64, 2056),
                                   (17, 64, 64)])
@pytest.mark.parametrize("R", [16, 32, 48, 64, 80])
def test_one_launch_and_two(gpu, T, K, N, R):
    """Around the sizes up to which a few rows take one launch."""
    for order, x_bf16, y_bf16 in (("mixed", False, False), ("mixed", True, True), ("runs", False, True)):
        d = make(T, K, N, 5, R, T + K + R, order, x_bf16, y_bf16)
        check(d, gpu, y_bf16=y_bf16)
        check(d, gpu, inplace=True)
        check(d, gpu, glu=True, y_bf16=not y_bf16)


def test_full_ranks_and_many_adapters_in_a_tile(gpu):
    """64 adapters in the 64 rows of a tile, each rank of the storage."""
    for R in (16, 32, 48, 64, 80, 128, 256):
        d = make(130, 72, 72, 64, R, R, ranks=[(7 * i) % R + 1 for i in range(64)])
        d["slot"] = torch.randperm(130, generator=gen(R)).remainder(64).int()
        check(d, gpu)
        check(d, gpu, glu=True)
        check(dict(d, slot=d["slot"].sort().values), gpu, inplace=True)


def test_large_and_tiny_values(gpu):
    """fp32 activations keep their 24 bits over the range: products that fit
    24 bits come out to the bit."""
    T, K, N = 20, 64, 16
    d = make(T, K, N, 2, 16, 8, "mixed", ranks=[16, 16])
    g = gen(1)
    d["a"] = torch.randint(-2, 3, (2, 16, K), generator=g).bfloat16()
    d["b"] = torch.zeros(2, N, 16).bfloat16()
    d["b"][:, torch.arange(16), torch.arange(16)] = 1.0
    d["scale"][:] = 1.0
    d["base"][:] = 0
    d["x"][:] = 0
    for t in range(T):          # one value of 24 bits a row, times -2 .. 2
        d["x"][t, (7 * t) % K] = float(2 ** 23 + 2 * t + 1) * 2.0 ** (8 * t - 120)
    v, _ = want(d)
    assert torch.equal(run(d, gpu).double(), v)


def test_rows_apart_stream_and_graphs(gpu):
    """Strided x, base and y whose other columns stay as they are; another
    stream; two captured graphs on one workspace, replayed in turn."""
    d = make(37, 128, 64, 4, 32, 21)
    x = torch.full((37, 200), float("nan"), device=gpu)
    x[:, 40:168] = d["x"].to(gpu)
    base = torch.full((37, 100), float("nan"), device=gpu)
    base[:, 4:68] = d["base"].to(gpu)
    wide = torch.full((37, 96), 7.0, device=gpu)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    y = check(d, gpu, x=x[:, 40:168], base=base[:, 4:68], y=wide[:, 8:72], stream=s)
    assert (wide[:, :8] == 7).all() and (wide[:, 72:] == 7).all()
    assert torch.equal(y, run(d, gpu))

    mv = lambda t: t.to(gpu)
    lora = ops.Lora(weights.LoraAdapters(mv(d["a"]), mv(d["b"]), mv(d["rank"]), mv(d["scale"])), 37)
    x, slot, base = mv(d["x"]), mv(d["slot"]), mv(d["base"])
    y1, h1 = torch.empty(37, 64, device=gpu), torch.empty(37, 32, device=gpu)
    lora.add(slot, x, y1, base=base)
    lora.swiglu(slot, x, base, h1)
    torch.cuda.synchronize()
    ga, gb = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(ga):
        lora.add(slot, x, y1, base=base)
    with torch.cuda.graph(gb):
        lora.swiglu(slot, x, base, h1)
    for i in range(3):
        e = make(37, 128, 64, 4, 32, 30 + i)
        x.copy_(e["x"])
        slot.copy_(e["slot"])
        ga.replay()
        gb.replay()
        torch.cuda.synchronize()
        e.update(a=d["a"], b=d["b"], rank=d["rank"], scale=d["scale"], base=d["base"])
        v, tol = want(e)
        assert ((y1.cpu().double() - v).abs() <= tol).all()
        v, tol = want_glu(e)
        assert ((h1.cpu().double() - v).abs() <= tol).all()


def test_loading_and_refusals(gpu):
    ad = weights.LoraAdapters.empty(3, 16, 64, 32, device=gpu)
    d = make(9, 64, 32, 3, 16, 40, ranks=[5, 16, 1])
    for s in range(3):
        r = int(d["rank"][s])
        ad.load(s, d["a"][s, :r].to(gpu), d["b"][s, :, :r].to(gpu), float(d["scale"][s]))
    lora = ops.Lora(ad, 9)
    check(d, gpu, lora=lora)
    slot, x, y = d["slot"].to(gpu), d["x"].to(gpu), d["base"].to(gpu)
    big = torch.zeros(10, 64, device=gpu)
    for bad in (dict(x=big), dict(x=x[:, :56]), dict(x=x.double()), dict(x=x.cpu()), dict(y=y[:, :28]), dict(y=y.t()),
                dict(row_slot=slot.long()), dict(row_slot=slot[:5]), dict(row_slot=slot.cpu()), dict(y=y.half())):
        kw = dict(row_slot=slot, x=x, y=y)
        kw.update(bad)
        with pytest.raises(_abi.GrimoireError):
            lora.add(**kw)
    with pytest.raises(_abi.GrimoireError):
        lora.swiglu(slot, x, y, y)


@pytest.mark.parametrize("slots", [2, 255, 256, 1000])
def test_many_slots(gpu, slots):
    """Tiles of dozens of adapters whose slots share most bits, short and
    long batches, the last slot and rows without one among them."""
    for T in (16, 64, 530):
        d = make(T, 64, 72, slots, 16, 60 + slots)
        d["slot"][: min(T, 12)] = torch.tensor([slots - 1, -1, slots - 2, 0, slots - 1, slots, slots // 2,
                                                slots // 2 - 1, -1, 1, 2**31 - 1, -2**31], dtype=torch.int32)
        e = dict(d, slot=torch.where((d["slot"] < 0) | (d["slot"] >= slots), -1, d["slot"]))
        ad = weights.LoraAdapters(*(d[k].to(gpu) for k in ("a", "b", "rank", "scale")))
        y = torch.full((T, 72), float("nan"), device=gpu)
        ops.Lora(ad, T).add(d["slot"].to(gpu), d["x"].to(gpu), y, base=d["base"].to(gpu))
        torch.cuda.synchronize()
        v, tol = want(e)
        assert ((y.cpu().double() - v).abs() <= tol).all()
