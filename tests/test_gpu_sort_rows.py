"""Tokens to rows in expert order with weights applied, and the gradients of the
ways there and back, against the formulas.

Tolerances, u = 2^-24 (a rounding of fp32).  rows and drows are one product,
rounded, then (bf16) rounded again: the same bits as torch's.  dx is a chain of
K steps: K u of sum |w r|.  dw and dgate sum H products: V ceil(H / (256 V))
steps in a thread's chain (V = 4 or 8 elements an access), 6 in a wave, 16 over
waves.  A bf16 output adds half a step, 2^-8."""
import pytest
import torch

from grimoire_amd import _abi, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def routes(T, E, K, seed, kind="mixed"):
    g = gen(seed)
    if kind == "one":
        return torch.full((T, K), E - 1, dtype=torch.int32)
    if kind == "none":
        return torch.full((T, K), -1, dtype=torch.int32)
    ids = torch.randint(0, E, (T, K), generator=g).int()
    if kind == "mixed":
        bad = torch.tensor([-1, E, -2 ** 31, 2 ** 31 - 1], dtype=torch.int32)[torch.randint(0, 4, (T, K), generator=g)]
        ids = torch.where(torch.rand((T, K), generator=g) < 0.2, bad, ids)
    return ids


def table(ids, E):
    flat = ids.flatten().long()
    live = (flat >= 0) & (flat < E)
    order = torch.argsort(torch.where(live, flat, E), stable=True)[:int(live.sum())]
    inv = torch.full_like(flat, -1)
    inv[order] = torch.arange(len(order))
    counts = torch.bincount(flat[live], minlength=E)
    return inv.int(), counts.int(), (counts.cumsum(0) - counts).int(), order


def b16(t, yes):
    return t.bfloat16() if yes else t


def data(T, H, K, seed, x_bf16=False):
    g = gen(seed)
    return b16(torch.randn((T, H), generator=g), x_bf16), torch.rand((T, K), generator=g) + 0.1


def sort(gpu, ids, x, E, rows_bf16, weight=None, perm=False, obj=None, **kw):
    T, K = ids.shape
    H = x.shape[1]
    obj = obj or ops.TokenSort(E, K, T, device=gpu)
    obj.workspace.fill_(255)
    rows = torch.full((T * K, H), 7.0, device=gpu, dtype=torch.bfloat16 if rows_bf16 else torch.float32)
    c, o = (torch.full((E,), -7, dtype=torch.int32, device=gpu) for _ in range(2))
    inv, pt = (torch.full((T * K,), -7, dtype=torch.int32, device=gpu) for _ in range(2))
    obj(ids.to(gpu), x.to(gpu), rows, c, o, inv, weight=None if weight is None else weight.to(gpu),
        perm_token=pt if perm else None, **kw)
    torch.cuda.synchronize()
    return rows.cpu(), c.cpu(), o.cpu(), inv.cpu(), pt.cpu()


def check_sort(got, ids, x, E, rows_bf16, weight=None, perm=False):
    T, K = ids.shape
    inv, counts, offsets, order = table(ids, E)
    rows, c, o, i, pt = got
    assert torch.equal(i, inv) and torch.equal(c, counts) and torch.equal(o, offsets)
    v = x.float()[order // K]
    if weight is not None:
        v = v * weight.flatten()[order, None]
    assert torch.equal(rows[:len(order)], b16(v, rows_bf16))
    assert bool((rows[len(order):] == 7.0).all())
    if perm:
        assert torch.equal(pt[:len(order)], (order // K).int()) and bool((pt[len(order):] == -7).all())


SIZES = [(1, 1, 1, 4), (1, 128, 8, 2048), (2, 16, 8, 132), (3, 512, 10, 24), (17, 5, 5, 260), (31, 64, 16, 1028),
         (64, 300, 4, 2880), (100, 128, 10, 512), (129, 512, 8, 40), (700, 128, 16, 64), (1500, 600, 6, 36),
         (5000, 64, 2, 8)]


@pytest.mark.parametrize("T,E,K,H", SIZES)
def test_sort(gpu, T, E, K, H):
    for n, kind in enumerate(("mixed", "all", "one", "none")):
        print(f"sort T={T} E={E} K={K} H={H} {kind}", flush=True)
        ids = routes(T, E, K, T + n, kind)
        for x_bf16, rows_bf16 in ((False, False), (False, True), (True, False), (True, True)):
            x, w = data(T, H, K, H + n, x_bf16)
            check_sort(sort(gpu, ids, x, E, rows_bf16), ids, x, E, rows_bf16)
            check_sort(sort(gpu, ids, x, E, rows_bf16, w, True), ids, x, E, rows_bf16, w, True)


def test_sort_no_tokens(gpu):
    obj = ops.TokenSort(300, 4, 8, device=gpu)
    c, o = (torch.full((300,), -7, dtype=torch.int32, device=gpu) for _ in range(2))
    i = dict(dtype=torch.int32, device=gpu)
    obj(torch.empty((0, 4), **i), torch.empty((0, 16), device=gpu), torch.empty((0, 16), device=gpu), c, o,
        torch.empty((0,), **i))
    torch.cuda.synchronize()
    assert not c.any() and not o.any()


def test_sort_many_experts(gpu):
    ids = routes(300, 5000, 4, 1, "mixed")
    x, w = data(300, 64, 4, 1)
    check_sort(sort(gpu, ids, x, 5000, True, w, True), ids, x, 5000, True, w, True)


def test_sort_keeps_what_is_not_finite(gpu):
    """Values are copied or multiplied as they are."""
    ids = routes(9, 12, 3, 2)
    x, w = data(9, 16, 3, 2)
    x[2, 3], x[4], x[5, 0], w[6, 1], w[7, 0] = float("inf"), NAN, -0.0, 0.0, float("inf")
    for weight in (None, w):
        rows = sort(gpu, ids, x, 12, False, weight)[0]
        _, _, _, order = table(ids, 12)
        v = x[order // 3] if weight is None else x[order // 3] * w.flatten()[order, None]
        torch.testing.assert_close(rows[:len(order)], v, rtol=0, atol=0, equal_nan=True)


@pytest.mark.parametrize("x_bf16", [False, True])
def test_rows_apart(gpu, x_bf16):
    """x, dx and dy in wider buffers, 8-byte aligned bf16: accessed by four."""
    T, E, K, H = 21, 40, 4, 264
    ids = routes(T, E, K, 3)
    x, w = data(T, H, K, 4, x_bf16)
    inv = table(ids, E)[0]
    for off, wide in ((4, H + 12), (8, H + 16)):
        buf = torch.full((T, wide), NAN, device=gpu, dtype=x.dtype)
        buf[:, off:off + H] = x.to(gpu)
        view = buf[:, off:off + H]
        T2, K2 = ids.shape
        obj = ops.TokenSort(E, K, T, device=gpu)
        got = sort_view(gpu, obj, ids, view, E, w)
        check_sort(got, ids, x, E, True, w)
        drows = b16(torch.randn((T * K, H), generator=gen(1)), True)
        out = torch.full((T, wide), 7.0, device=gpu, dtype=x.dtype)
        dw = torch.empty((T, K), device=gpu)
        obj.grad(drows.to(gpu), inv.to(gpu), out[:, off:off + H], x=view, weight=w.to(gpu), dweight=dw)
        torch.cuda.synchronize()
        check_sort_grad(out[:, off:off + H].cpu(), dw.cpu(), drows, inv.view(T, K), x, w)
        assert bool((out[:, :off] == 7.0).all()) and bool((out[:, off + H:] == 7.0).all())
        rows = b16(torch.randn((T * K, H), generator=gen(2)), True)
        check_combine(gpu, T, K, H, 11, dy=view, dy_cpu=x, rows=rows, inv=inv)


def sort_view(gpu, obj, ids, view, E, w):
    T, K = ids.shape
    rows = torch.full((T * K, view.shape[1]), 7.0, device=gpu, dtype=torch.bfloat16)
    c, o = (torch.empty((E,), dtype=torch.int32, device=gpu) for _ in range(2))
    inv = torch.empty((T, K), dtype=torch.int32, device=gpu)
    obj(ids.to(gpu), view, rows, c, o, inv, weight=w.to(gpu))
    torch.cuda.synchronize()
    return rows.cpu(), c.cpu(), o.cpu(), inv.cpu().flatten(), None


def dot_steps(H):
    return 8 * ((H + 2047) // 2048) + 4 * ((H + 1023) // 1024) + 6 + 16


def check_sort_grad(dx, dw, drows, inv, x=None, w=None):
    T, K = inv.shape
    live = (inv >= 0) & (inv < drows.shape[0])
    if drows.shape[0]:
        r = drows[inv.clamp(0, drows.shape[0] - 1).long()].double()
    else:
        r = torch.zeros((T, K, dx.shape[1]), dtype=torch.float64)
    r[~live] = 0.0
    ww = torch.ones((T, K)) if w is None else w
    t = r * ww.double()[:, :, None]
    v, tol = t.sum(1), K * U * t.abs().sum(1)
    if dx.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (v.abs() + tol)
    assert ((dx.double() - v).abs() <= tol).all()
    if w is not None:
        t = r * x.double()[:, None, :]
        assert ((dw.double() - t.sum(2)).abs() <= dot_steps(dx.shape[1]) * U * t.abs().sum(2)).all()
        assert bool((dw[~live] == 0).all())


def wild_inverse(T, K, R, seed):
    """Distinct rows, some routes without one: -1 and past the rows."""
    g = gen(seed)
    inv = torch.full((T * K,), -1, dtype=torch.int32)
    n = min(R, T * K)
    inv[torch.randperm(T * K, generator=g)[:n]] = torch.randperm(R, generator=g)[:n].int()
    bad = torch.tensor([-1, R, 2 ** 31 - 1, -2 ** 31], dtype=torch.int32)[torch.randint(0, 4, (T * K,), generator=g)]
    return torch.where(torch.rand((T * K,), generator=g) < 0.2, bad, inv)


GRAD = [(1, 1, 4), (1, 8, 7168), (2, 5, 132), (7, 16, 264), (32, 8, 7168), (65, 10, 1028), (300, 4, 2880), (301, 2, 40),
        (700, 9, 520)]


@pytest.mark.parametrize("T,K,H", GRAD)
def test_sort_grad(gpu, T, K, H):
    for R in (T * K, max(1, T * K // 2), 0):
        inv = wild_inverse(T, K, R, T + R)
        for x_bf16, rows_bf16, dx_bf16 in ((False, False, False), (False, True, True), (True, False, False),
                                           (True, True, True)):
            print(f"sort_grad T={T} K={K} H={H} R={R} {x_bf16} {rows_bf16}", flush=True)
            x, w = data(T, H, K, H, x_bf16)
            drows = b16(torch.randn((R, H), generator=gen(R)), rows_bf16)
            if R:                   # rows that no route names
                unnamed = torch.ones((R,), dtype=torch.bool)
                unnamed[inv[(inv >= 0) & (inv < R)].long()] = False
                drows[unnamed] = NAN
            obj = ops.TokenSort(8, K, T, device=gpu)
            for weighted in (False, True):
                dx = torch.full((T, H), NAN, device=gpu, dtype=torch.bfloat16 if dx_bf16 else torch.float32)
                dw = torch.full((T, K), NAN, device=gpu)
                kw = dict(x=x.to(gpu), weight=w.to(gpu), dweight=dw) if weighted else {}
                obj.grad(drows.to(gpu), inv.view(T, K).to(gpu), dx, **kw)
                torch.cuda.synchronize()
                check_sort_grad(dx.cpu(), dw.cpu(), drows, inv.view(T, K), x, w if weighted else None)


def check_combine(gpu, T, K, H, seed, dy=None, dy_cpu=None, rows=None, inv=None, dy_bf16=False, rows_bf16=True,
                  shared="none", gate=False, R=None):
    g = gen(seed)
    R = T * K if R is None else R
    if dy is None:
        dy_cpu = b16(torch.randn((T, H), generator=g), dy_bf16)
        dy = dy_cpu.to(gpu)
    if rows is None:
        rows = b16(torch.randn((R, H), generator=g), rows_bf16)
    inv = wild_inverse(T, K, R, seed) if inv is None else inv
    w = torch.rand((T, K), generator=g) + 0.1
    sh = None if shared == "none" else b16(torch.randn((T, H), generator=g), shared == "bf16")
    ga = torch.rand((T,), generator=g) if gate else None
    mv = lambda t: None if t is None else t.to(gpu)
    drows = torch.full_like(rows, 7.0).to(gpu)
    dw = torch.full((T, K), NAN, device=gpu)
    dsh = None if sh is None else torch.full_like(sh, NAN).to(gpu)
    dga = torch.full((T,), NAN, device=gpu) if gate else None
    live = ((inv >= 0) & (inv < R)).view(T, K)
    named = torch.zeros((R,), dtype=torch.bool)
    named[inv[live.flatten()].long()] = True
    rows = rows.clone()
    rows[~named] = NAN
    ops.combine_grad(dy, rows.to(gpu), inv.to(gpu), w.to(gpu), drows, dw, shared=mv(sh), gate=mv(ga), dshared=dsh, dgate=dga)
    torch.cuda.synchronize()
    r = torch.zeros((T, K, H), dtype=torch.float64)
    r[live] = rows[inv.view(T, K)[live].long()].double()
    y = dy_cpu.double()
    t = r * y[:, None, :]
    dwc = dw.cpu()
    assert ((dwc.double() - t.sum(2)).abs() <= dot_steps(H) * U * t.abs().sum(2)).all()
    assert bool((dwc[~live] == 0).all())
    want = torch.full_like(rows, 7.0)
    want[inv.view(T, K)[live].long()] = b16(dy_cpu.float()[:, None, :] * w[:, :, None], rows.dtype == torch.bfloat16)[live]
    assert torch.equal(drows.cpu(), want)
    if sh is not None:
        v = dy_cpu.float() if ga is None else dy_cpu.float() * ga[:, None]
        assert torch.equal(dsh.cpu(), b16(v, shared == "bf16"))
    if gate:
        t = y * sh.double()
        assert ((dga.cpu().double() - t.sum(1)).abs() <= dot_steps(H) * U * t.abs().sum(1)).all()


@pytest.mark.parametrize("T,K,H", GRAD)
def test_combine_grad(gpu, T, K, H):
    n = 0
    for dy_bf16 in (False, True):
        for rows_bf16 in (False, True):
            for shared, gate in (("none", False), ("bf16", False), ("f32", True), ("bf16", True)):
                for R in (T * K, max(1, T * K // 2), 0):
                    print(f"combine_grad T={T} K={K} H={H} R={R} {dy_bf16} {rows_bf16} {shared} {gate}", flush=True)
                    n += 1
                    check_combine(gpu, T, K, H, n, dy_bf16=dy_bf16, rows_bf16=rows_bf16, shared=shared, gate=gate, R=R)


def test_gradients_against_differences(gpu):
    """<d, gradient> against the change of a linear functional of the forward:
    sort and combine are linear in each argument, so a difference is exact up to
    rounding."""
    T, E, K, H = 24, 16, 4, 96
    ids = routes(T, E, K, 1)
    x, w = data(T, H, K, 1)
    g = torch.randn((T * K, H), generator=gen(3))
    inv = table(ids, E)[0]
    dx, dw = torch.empty((T, H), device=gpu), torch.empty((T, K), device=gpu)
    obj = ops.TokenSort(E, K, T, device=gpu)
    obj.grad(g.to(gpu), inv.to(gpu), dx, x=x.to(gpu), weight=w.to(gpu), dweight=dw)

    def loss(x, w):
        rows = sort(gpu, ids, x, E, False, w)[0].double()
        n = int((inv >= 0).sum())
        return float((rows[:n] * g[:n].double()).sum())
    a, b = torch.randn((T, H), generator=gen(4)), torch.randn((T, K), generator=gen(5))
    size = float((x.abs().sum() * 4))
    assert abs(loss(x + a, w) - loss(x, w) - float((a.double() * dx.cpu().double()).sum())) <= 64 * U * size
    assert abs(loss(x, w + b) - loss(x, w) - float((b.double() * dw.cpu().double()).sum())) <= 64 * U * size


def test_other_stream_and_graph(gpu):
    """All three captured into one graph and replayed with new routes, eager calls
    between the replays."""
    T, E, K, H = 40, 64, 8, 512
    i32 = dict(dtype=torch.int32, device=gpu)
    obj, eager = ops.TokenSort(E, K, T, device=gpu), ops.TokenSort(E, K, T, device=gpu)
    ids, x, w = torch.zeros((T, K), **i32), torch.empty((T, H), device=gpu), torch.empty((T, K), device=gpu)

    def outs():
        return [torch.zeros((T * K, H), device=gpu), torch.empty((E,), **i32), torch.empty((E,), **i32),
                torch.empty((T * K,), **i32), torch.empty((T, H), device=gpu), torch.empty((T, K), device=gpu),
                torch.zeros((T * K, H), device=gpu), torch.empty((T, K), device=gpu)]

    def step(o, s, stream=None):
        s(ids, x, *o[:4], weight=w, stream=stream)
        s.grad(o[0], o[3], o[4], x=x, weight=w, dweight=o[5], stream=stream)
        ops.combine_grad(x, o[0], o[3], w, o[6], o[7], stream=stream)
    a, b = outs(), outs()

    def fill(seed):
        d = data(T, H, K, seed)
        ids.copy_(routes(T, E, K, seed, "all"))
        x.copy_(d[0])
        w.copy_(d[1])
    fill(0)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    step(a, obj, side)
    side.synchronize()
    step(b, eager)
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(a, b))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(a, obj)
    for seed in (1, 2, 3):
        fill(seed)
        graph.replay()
        torch.cuda.synchronize()
        step(b, eager)
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(a, b))


def test_offsets_past_32_bits(gpu):
    """Rows past 2^31 elements."""
    T, E, K, H = 40000, 8, 8, 7168
    assert T * K * H > 2 ** 31
    g = torch.Generator(device=gpu).manual_seed(1)
    ids = torch.stack([torch.arange(E, device=gpu)] * T).int().contiguous()
    x = torch.randn((T, H), device=gpu, generator=g).bfloat16()
    rows = torch.empty((T * K, H), device=gpu, dtype=torch.bfloat16)
    i32 = dict(dtype=torch.int32, device=gpu)
    c, o, inv = torch.empty((E,), **i32), torch.empty((E,), **i32), torch.empty((T, K), **i32)
    obj = ops.TokenSort(E, K, T, device=gpu)
    obj(ids, x, rows, c, o, inv)
    for e in range(E):
        assert torch.equal(rows[e * T:(e + 1) * T], x)
    dx = torch.empty((T, H), device=gpu)
    obj.grad(rows, inv, dx)
    assert torch.equal(dx, 8 * x.float())
    w, drows, dw = torch.full((T, K), 0.5, device=gpu), torch.zeros_like(rows), torch.empty((T, K), device=gpu)
    ops.combine_grad(x, rows, inv, w, drows, dw)
    assert torch.equal(drows[-T:], (x.float() * 0.5).bfloat16()) and torch.equal(dw[:, 0], dw[:, 7])


def test_rows_far_apart(gpu):
    """Rows of x, dx and dy whose offsets pass 32 bits."""
    T, E, K, H, S = 40, 16, 4, 264, 1 << 26
    assert (T - 1) * S > 2 ** 31
    ids = routes(T, E, K, 3)
    x, w = data(T, H, K, 4)
    inv = table(ids, E)[0]
    view, dx = (torch.empty(((T - 1) * S + H,), device=gpu).as_strided((T, H), (S, 1)) for _ in range(2))
    view.copy_(x)
    obj = ops.TokenSort(E, K, T, device=gpu)
    check_sort(sort_view(gpu, obj, ids, view, E, w), ids, x, E, True, w)
    drows = torch.randn((T * K, H), generator=gen(1))
    dw = torch.empty((T, K), device=gpu)
    obj.grad(drows.to(gpu), inv.to(gpu), dx, x=view, weight=w.to(gpu), dweight=dw)
    torch.cuda.synchronize()
    check_sort_grad(dx.cpu(), dw.cpu(), drows, inv.view(T, K), x, w)
    check_combine(gpu, T, K, H, 11, dy=view, dy_cpu=x, inv=inv)


def test_host_refusals_on_the_gpu_objects(gpu):
    T, E, K, H = 4, 8, 2, 16
    obj = ops.TokenSort(E, K, T, device=gpu)
    i32 = dict(dtype=torch.int32, device=gpu)
    ids, x, w = torch.zeros((T, K), **i32), torch.zeros((T, H), device=gpu), torch.zeros((T, K), device=gpu)
    rows, c, o, inv = torch.zeros((T * K, H), device=gpu), torch.zeros((E,), **i32), torch.zeros((E,), **i32), \
        torch.zeros((T * K,), **i32)
    for args, kw in (((ids.long(), x, rows, c, o, inv), {}), ((ids, x.half(), rows, c, o, inv), {}),
                     ((ids, x, rows[:4], c, o, inv), {}), ((ids, x, rows, c[:4], o, inv), {}),
                     ((ids, x, rows, c, o, inv[:4]), {}), ((ids, x, rows, c, o, inv), dict(weight=w[:, :1])),
                     ((ids.cpu(), x, rows, c, o, inv), {}), ((ids, x.cpu(), rows, c, o, inv), {}),
                     ((ids, x, rows, c, c, inv), {}), ((ids, rows[:T], rows, c, o, inv), {}),
                     ((ids, torch.zeros((5, H), device=gpu), rows, c, o, inv), {}),
                     ((ids, x[:, :6].contiguous(), rows[:, :6].contiguous(), c, o, inv), {})):
        with pytest.raises(_abi.GrimoireError):
            obj(*args, **kw)
    dx, dw = torch.zeros((T, H), device=gpu), torch.zeros((T, K), device=gpu)
    for args, kw in (((rows, inv, dx), dict(weight=w)), ((rows, inv, dx), dict(weight=w, x=x)),
                     ((rows, inv, rows[:T]), {}), ((rows, inv.cpu(), dx), {}), ((rows[:, :8], inv, dx), {}),
                     ((rows, inv, dx), dict(weight=w, x=x, dweight=w))):
        with pytest.raises(_abi.GrimoireError):
            obj.grad(*args, **kw)
    dr = torch.zeros_like(rows)
    for args, kw in (((x, rows, inv, w, rows, dw), {}), ((x, rows, inv, w, dr.bfloat16(), dw), {}),
                     ((x, rows, inv, w, dr, w), {}), ((x, rows, inv, w, dr, dw), dict(shared=x)),
                     ((x, rows, inv, w, dr, dw), dict(shared=dx, dshared=torch.zeros_like(dx), gate=w[:, 0].contiguous())),
                     ((x, rows, inv, w, dr, dw), dict(gate=w[:, 0].contiguous(), dgate=w[:, 1].contiguous())),
                     ((x, rows, inv, w, dr, dw), dict(shared=dx, dshared=x))):
        with pytest.raises(_abi.GrimoireError):
            ops.combine_grad(*args, **kw)
