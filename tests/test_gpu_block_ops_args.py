"""Arguments of the block operators that have to be refused as such, and those
that must not be: shapes, one row far from the next, streams of other
devices, expert rows named by a view."""
import types

import pytest
import torch

from grimoire_amd import _abi, ops, weights

pytestmark = pytest.mark.gpu
T, H, K = 6, 64, 4


def test_shapes_and_streams(gpu):
    f = lambda *s: torch.zeros(*s, device=gpu)
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device=gpu)
    n = ops.BlockNorm(f(H).bfloat16())
    rows, inv, w = f(T * K, H).bfloat16(), i(T * K), f(T, K)
    lora = ops.Lora(weights.LoraAdapters.empty(2, 16, H, 32, device=gpu), T)
    there = types.SimpleNamespace(cuda_stream=0, device_index=f(1).get_device() + 1)
    calls = [lambda: n(f(H), f(H), f(H)), lambda: n(f(1, T, H), f(1, T, H), f(1, T, H)),
             lambda: n(f(T, H), f(T, H), f(T, H), stream=there),
             lambda: n.moe(f(T, H), rows[0], inv, w, None, f(T, H)),
             lambda: n.moe(f(T, H), rows, i(K, T).t(), w, None, f(T, H)),
             lambda: n.moe(f(T, H), rows, i(T, K + 1), w, None, f(T, H)),
             lambda: n.moe(f(T, H), rows, inv, w.view(-1), None, f(T, H)),
             lambda: lora.add(i(T), f(H), f(T, 32)), lambda: lora.add(i(1), f(()), f(1, 32)),
             lambda: lora.add(i(T), f(T, H), f(T, 32), stream=there),
             lambda: lora.add(i(T), f(T, H), f(T, 16).expand(T, 16).repeat(1, 2)[:, ::2]),
             lambda: ops.RouteScores()(f(T, 8), i(T, 2), f(T, 2), stream=there),
             lambda: ops.RouteScores()(f(8), i(T, 2), f(T, 2)), lambda: ops.RouteScores()(f(T, 8), i(2), f(2))]
    calls.append(lambda: ops.BlockNorm(f(H).bfloat16(), f(H + 4).bfloat16()))
    for c in calls:
        with pytest.raises(_abi.GrimoireError):
            c()
    for name in ("adapters", "workspace"):
        with pytest.raises(AttributeError):
            setattr(lora, name, None)


def test_one_row_of_a_larger_tensor(gpu):
    """The distance to a next row that is not there does not count."""
    g = torch.Generator().manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g).to(gpu)
    ad = weights.LoraAdapters.empty(1, 16, H, 32, device=gpu)
    ad.load(0, rn(3, H), rn(32, 3), 1.0)
    lora = ops.Lora(ad, 1)
    slot = torch.zeros(1, dtype=torch.int32, device=gpu)
    x, base = rn(1, H + 3)[:, :H], rn(1, 35)[:, :32]
    y, want = torch.empty(1, 35, device=gpu)[:, :32], torch.empty(1, 32, device=gpu)
    lora.add(slot, x, y, base=base)
    lora.add(slot, x.contiguous(), want, base=base.contiguous())
    n = ops.BlockNorm(rn(H).bfloat16())
    h, out, ref = rn(1, H), torch.empty(1, H, device=gpu), torch.empty(1, H, device=gpu)
    n(h, x, None, out)
    n(h, x.contiguous(), None, ref)
    torch.cuda.synchronize()
    assert torch.equal(y, want) and torch.equal(out, ref)


def test_inverse_by_token(gpu):
    g = torch.Generator().manual_seed(4)
    rn = lambda *s: torch.randn(*s, generator=g).to(gpu)
    n = ops.BlockNorm(rn(H).bfloat16(), rn(H).bfloat16())
    rows, w, h = rn(T * K, H).bfloat16(), rn(T, K), rn(T, H)
    inv = torch.randperm(T * K, generator=g).int().to(gpu)
    a, b = torch.empty(T, H, device=gpu), torch.empty(T, H, device=gpu)
    n.moe(h, rows, inv, w, None, a)
    n.moe(h, rows, inv.view(T, K), w, None, b)
    torch.cuda.synchronize()
    assert torch.equal(a, b)


def test_in_place_of_an_input(gpu):
    """Outputs in place of inputs of the same layout: h' over h, o over x, the
    bf16 o over a bf16 x, h' over the shared rows."""
    g = torch.Generator().manual_seed(5)
    for rows, width in ((T, H), (3, 2052), (300, 7168)):
        rn = lambda *s: torch.randn(*s, generator=g).to(gpu)
        for post in (None, rn(width).bfloat16()):
            n = ops.BlockNorm(rn(width).bfloat16(), post, block_scale=0.5)
            h, x, e = rn(rows, width), rn(rows, width), lambda: torch.empty(rows, width, device=gpu)
            xb, ob = x.bfloat16(), e().bfloat16()
            ho, o = e(), e()
            n(h, x, ho, o)
            h1, x1 = h.clone(), x.clone()
            n(h1, x1, h1, x1)
            n(h, xb, None, None, ob)
            n(h, xb, None, None, xb)
            routed, w = rn(rows * 2, width).bfloat16(), rn(rows, 2)
            inv = torch.arange(rows * 2, dtype=torch.int32, device=gpu)
            hm = e()
            n.moe(h, routed, inv, w, x, hm)
            x2 = x.clone()
            n.moe(h, routed, inv, w, x2, x2)
            torch.cuda.synchronize()
            assert torch.equal(h1, ho) and torch.equal(x1, o) and torch.equal(xb, ob) and torch.equal(x2, hm)


def test_two_streams_at_once(gpu):
    """One RouteScores, one BlockNorm and one set of adapters (with a
    workspace a stream) called from two streams in turn, many calls in
    flight: every result is that of the call alone."""
    g = torch.Generator().manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=g).to(gpu)
    rows, N, E = 80, 256, 64
    scores = ops.RouteScores("sigmoid", bias=rn(E), n_group=4, topk_group=2)
    norm = ops.BlockNorm(rn(H).bfloat16(), rn(H).bfloat16(), gate="row", gate_sigmoid=True)
    ad = weights.LoraAdapters.empty(5, 32, H, N, device=gpu)
    for s in range(5):
        ad.load(s, rn(7 * s + 1, H), rn(N, 7 * s + 1), 0.5)
    loras = [ops.Lora(ad, rows) for _ in range(2)]
    ins = [dict(l=rn(rows, E), h=rn(rows, H), x=rn(rows, H), gate=rn(rows), base=rn(rows, N),
                slot=torch.randint(-1, 5, (rows,), generator=g).int().to(gpu)) for _ in range(8)]

    def outs():
        return dict(ids=torch.empty(rows, K, dtype=torch.int32, device=gpu), w=torch.empty(rows, K, device=gpu),
                    h=torch.empty(rows, H, device=gpu), o=torch.empty(rows, H, device=gpu),
                    y=torch.empty(rows, N, device=gpu), s=torch.empty(rows, N // 2, device=gpu))

    def call(d, o, lora, stream):
        scores(d["l"], o["ids"], o["w"], stream=stream)
        norm(d["h"], d["x"], o["h"], o["o"], gate=d["gate"], stream=stream)
        lora.add(d["slot"], d["x"], o["y"], base=d["base"], stream=stream)
        lora.swiglu(d["slot"], d["x"], d["base"], o["s"], stream=stream)

    want = [outs() for _ in ins]
    for d, o in zip(ins, want):
        call(d, o, loras[0], None)
        torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[outs() for _ in ins] for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(len(ins)):
        for j, s in enumerate(streams):
            call(ins[(i + 3 * j) % len(ins)], got[j][(i + 3 * j) % len(ins)], loras[j], s)
    torch.cuda.synchronize()
    for j in range(2):
        for a, b in zip(got[j], want):
            for k in a:
                assert torch.equal(a[k], b[k]), (j, k)


def test_offsets_past_32_bits(gpu):
    """Rows 2^24 elements apart, slots of 2^25 elements: bytes and elements
    past 2^32.  Bit for bit what the same rows side by side give."""
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GiB of device memory")
    g = torch.Generator().manual_seed(7)
    rn = lambda *s: torch.randn(*s, generator=g).to(gpu)
    rows, apart, E, N = 260, 1 << 24, 64, 72
    far = torch.empty(rows, apart, device=gpu)                       # 16 GiB
    place = lambda v, at: far[:, at:at + v.shape[1]].copy_(v)
    scores, norm = ops.RouteScores(), ops.BlockNorm(rn(H).bfloat16(), rn(H).bfloat16())
    l, x, base, h = rn(rows, E), rn(rows, H), rn(rows, N), rn(rows, H)
    e = lambda *s: torch.empty(*s, device=gpu)
    i = lambda: torch.empty(rows, K, dtype=torch.int32, device=gpu)
    ids, w, o = [i(), i()], [e(rows, K), e(rows, K)], [e(rows, H), e(rows, H)]
    scores(l, ids[0], w[0])
    scores(place(l, 0), ids[1], w[1])
    norm(h, x, None, o[0])
    norm(h, place(x, 64), None, o[1])
    ad = weights.LoraAdapters.empty(3, 16, H, N, device=gpu)
    for s in range(3):
        ad.load(s, rn(16 - s, H), rn(N, 16 - s), 1.0)
    slot = torch.randint(-1, 3, (rows,), generator=g).int().to(gpu)
    y, t = e(rows, N), far[:, 256:256 + N]
    lora = ops.Lora(ad, rows)
    lora.add(slot, x, y, base=base)
    lora.add(slot, far[:, 64:64 + H], t, base=place(base, 128))
    torch.cuda.synchronize()
    assert torch.equal(ids[0], ids[1]) and torch.equal(w[0], w[1]) and torch.equal(o[0], o[1])
    assert torch.equal(t, y)
    del far, t

    wide, slots, R = 1 << 17, 68, 256                                # b: 4.25 GiB, its last slots past 2^31 elements
    ad = weights.LoraAdapters.empty(slots, R, H, wide, device=gpu)
    one = weights.LoraAdapters.empty(1, R, H, wide, device=gpu)
    a, b = rn(R, H), rn(wide, R)
    ad.load(slots - 1, a, b, 0.5)
    one.load(0, a, b, 0.5)
    x, base = rn(20, H), rn(20, wide)
    got, want = e(20, wide), e(20, wide)
    at = torch.full((20,), slots - 1, dtype=torch.int32, device=gpu)
    at[7] = -1
    ops.Lora(ad, 20).add(at, x, got, base=base)
    ops.Lora(one, 20).add(torch.where(at < 0, -1, 0).int(), x, want, base=base)
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(got[7], base[7]) and not torch.equal(got[8], base[8])

    rows, width = 300000, 7168                                       # h: 8 GiB
    h, x = torch.zeros(rows, width, device=gpu), torch.zeros(rows, width, dtype=torch.bfloat16, device=gpu)
    h[-3:], x[-3:] = rn(3, width), rn(3, width).bfloat16()
    norm = ops.BlockNorm(rn(width).bfloat16(), rn(width).bfloat16())
    # 300 rows: up to 256 a row's sum is spread over other threads
    small, out = e(300, width), torch.empty(rows, width, dtype=torch.bfloat16, device=gpu)
    sb = torch.empty(300, width, dtype=torch.bfloat16, device=gpu)
    norm(h[-300:].clone(), x[-300:], small, None, sb)
    norm(h, x, h, None, out)
    torch.cuda.synchronize()
    assert torch.equal(h[-300:], small) and torch.equal(out[-300:], sb) and not out[0].any()
