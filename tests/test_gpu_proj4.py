"""Dense 4-bit projections (grimoire_proj4, grimoire_proj4_swiglu) against the
formula in 64 bits.

Tolerances, u = 2^-23 (a step of the matrix core's fp32 sums, cut off or
rounded).  Products are exact: codes in bf16, fp32 activations in three exact
bf16 pieces.  INT4: a group's sum of (16 + q) x and of x, each 32 steps inside
an instruction and 4 of a chain, two steps to take 16 + z times the sum of x
off, one for the scale, then at most K / 32 groups, 16 waves, 3 pieces:
(42 + K / 32 + 19) u of sum |s| (16 + q + 16 + z) |x|.  MXFP4: 32 steps in an
instruction, K / 32 in the chain, waves and pieces: (32 + K / 32 + 19) u of
sum |w x|.  base is one step more.  silu(g) u: (2 |g| + 8) u of itself, and a
change of g moves it by at most 1.1 |u|.  A bf16 output adds half a step,
2^-8."""
import ctypes as C

import pytest
import torch

from grimoire_amd import _abi, ops
from grimoire_amd.weights import Weight
from helpers import dequant

pytestmark = pytest.mark.gpu
U = 2.0 ** -23

FMTS = {"int4": _abi.FMT_INT4, "int4_f16": _abi.FMT_INT4_F16, "mxfp4": _abi.FMT_MXFP4}
KINDS = [("int4", "none"), ("int4", "asym"), ("int4", "signed"), ("int4", "mixed"), ("int4_f16", "none"),
         ("int4_f16", "mixed"), ("mxfp4", "none")]


def make_weight(fmt, zeros, N, K, group, seed, pad=0):
    """pad: bytes between the rows (and, MXFP4, scales), of any value."""
    g = torch.Generator().manual_seed(seed)
    G = K // (32 if fmt == "mxfp4" else group)
    payload = torch.randint(0, 256, (N, K // 2 + pad), dtype=torch.uint8, generator=g)
    if fmt == "mxfp4":
        sc = torch.randint(118, 130, (N, G + pad), dtype=torch.uint8, generator=g)
        sc[:, G:] = 255
        return Weight(_abi.FMT_MXFP4, N, K, payload, sc, None, G + pad)
    s = torch.randn((N, G), generator=g) * 0.1
    z = None
    if zeros == "asym":
        z = torch.randint(0, 17, (N, G), dtype=torch.uint8, generator=g)
    elif zeros == "signed":
        z = torch.full((N, G), 255, dtype=torch.uint8)
    elif zeros == "mixed":
        z = torch.tensor([0, 1, 8, 15, 16, 100, 254, 255], dtype=torch.uint8)[torch.randint(0, 8, (N, G), generator=g)]
    return Weight(FMTS[fmt], N, K, payload, (s.half() if fmt == "int4_f16" else s.bfloat16()).view(torch.int16), z, G)


def reference(w, x, base=None, glu=False):
    """The outputs in fp64 and their tolerance."""
    N, K = w.N, w.K
    x = x.double()
    W = dequant(w)[:, :K].double()
    v = x @ W.T
    if w.fmt == _abi.FMT_MXFP4:
        tol = (32 + K / 32 + 19) * U * (x.abs() @ W.abs().T)
    else:
        G = w.row_scales
        q = torch.stack((w.payload[:, :K // 2] & 15, w.payload[:, :K // 2] >> 4), dim=2).view(N, G, K // G).double()
        z = w.zeros.double() if w.zeros is not None else torch.full((N, G), 8.0 if w.fmt == _abi.FMT_INT4_F16 else 0.0).double()
        signed = z == 255                    # codes xor 8, zero point 8
        z = torch.where(signed, 8.0, z)
        q = torch.where(signed[:, :, None], (q + 8) % 16, q)
        raw = w.scales.view(torch.int16)
        s = (raw.view(torch.bfloat16) if w.fmt == _abi.FMT_INT4 else raw.view(torch.float16)).double()
        mag = ((32 + q + z[:, :, None]) * s.abs()[:, :, None]).view(N, K)
        tol = (42 + K / 32 + 19) * U * (x.abs() @ mag.T)
    if base is not None:
        v = v + base.double()
        tol = tol + U * (v.abs() + base.double().abs())
    if glu:
        g, up, tg, tu = v[:, :N // 2], v[:, N // 2:], tol[:, :N // 2], tol[:, N // 2:]
        s = g * torch.sigmoid(g)
        v = s * up
        tol = 1.1 * tg * (up.abs() + tu) + s.abs() * tu + (2 * g.abs() + 8) * U * v.abs() + 1e-30
    return v, tol


def check(y, v, tol):
    if y.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (v.abs() + tol)
    err = (y.cpu().double() - v).abs()
    assert (err <= tol).all(), float((err / tol).max())


def run(gpu, w, x, y_bf16=False, base=None, glu=False, **kw):
    proj = ops.Projection4(w.to(gpu), x.shape[0])
    y = torch.full((x.shape[0], w.N // 2 if glu else w.N), float("nan"), device=gpu,
                   dtype=torch.bfloat16 if y_bf16 else torch.float32)
    xg = x.to(gpu)
    if glu:
        proj.swiglu(xg, y, **kw)
    else:
        proj(xg, y, base=None if base is None else base.to(gpu), **kw)
    torch.cuda.synchronize()
    return y


def rows(T, K, seed, b16=False):
    x = torch.randn((T, K), generator=torch.Generator().manual_seed(seed))
    return x.bfloat16() if b16 else x


SIZES = [(1, 32, 16), (1, 64, 1), (2, 96, 18), (3, 768, 512), (5, 160, 34), (6, 2048, 100), (11, 2880, 64),
         (16, 288, 50), (17, 1056, 40), (33, 7168, 24), (64, 512, 130), (130, 256, 20), (1, 16384, 8), (40, 4128, 6)]


@pytest.mark.parametrize("fmt,zeros", KINDS)
@pytest.mark.parametrize("T,K,N", SIZES)
def test_sizes(gpu, T, K, N, fmt, zeros):
    for group in (32,) if fmt == "mxfp4" else (32, 64, 128, 256):
        if K % group:
            continue
        w = make_weight(fmt, zeros, N, K, group, T + K + group)
        for x_bf16 in (False, True):
            print(f"proj4 {fmt} {zeros} T={T} K={K} N={N} group={group} bf16={x_bf16}", flush=True)
            x = rows(T, K, K + group, x_bf16)
            check(run(gpu, w, x, y_bf16=not x_bf16), *reference(w, x))
            if N % 2 == 0:
                check(run(gpu, w, x, y_bf16=x_bf16, glu=True), *reference(w, x, glu=True))


@pytest.mark.parametrize("fmt,zeros", [("int4", "mixed"), ("mxfp4", "none")])
@pytest.mark.parametrize("T", [1, 7, 20])
def test_base(gpu, fmt, zeros, T):
    """A base of either type; in place, which gives the same bits."""
    w = make_weight(fmt, zeros, 97, 416, 32, T)
    for x_bf16 in (False, True):
        x = rows(T, 416, T, x_bf16)
        for b16 in (False, True):
            base = rows(T, 97, 5, b16)
            want = reference(w, x, base)
            check(run(gpu, w, x, base=base), *want)
            y = run(gpu, w, x, base=base, y_bf16=b16)
            check(y, *want)
            proj, z = ops.Projection4(w.to(gpu), T), base.to(gpu).clone()
            proj(x.to(gpu), z, base=z)
            assert torch.equal(z, y)


def test_positive_rows(gpu):
    """Activations of one sign: the sums that the zero points take off are large."""
    w = make_weight("int4", "asym", 40, 2048, 128, 3)
    x = rows(4, 2048, 3).abs() + 1.0
    check(run(gpu, w, x), *reference(w, x))


@pytest.mark.parametrize("fmt,zeros", [("int4", "mixed"), ("mxfp4", "none")])
@pytest.mark.parametrize("glu", [False, True])
def test_rows_apart(gpu, fmt, zeros, glu):
    """Padded weight rows, rows of x, y and base in wider buffers, y at an
    address of one element's alignment; what lies between stays as it was."""
    T, K, N = 9, 352, 38
    w = make_weight(fmt, zeros, N, K, 32, 8, pad=16 if fmt == "mxfp4" else 0)
    if fmt != "mxfp4":
        pay = torch.full((N, K // 2 + 16), 0xAB, dtype=torch.uint8)
        pay[:, :K // 2] = w.payload
        w = Weight(w.fmt, N, K, pay, w.scales, w.zeros, w.row_scales)
    x = rows(T, K, 1)
    width = N // 2 if glu else N
    xb = torch.full((T, K + 24), float("nan"), device=gpu)
    xb[:, 8:8 + K] = x.to(gpu)
    buf = torch.full((T, 2 * width + 3), 7.0, device=gpu)
    proj = ops.Projection4(w.to(gpu), T)
    if glu:
        proj.swiglu(xb[:, 8:8 + K], buf[:, 1:1 + width])
        check(buf[:, 1:1 + width], *reference(w, x, glu=True))
        rest = (buf[:, :1], buf[:, 1 + width:])
    else:
        base = rows(T, N, 2)
        buf[:, 1 + N:1 + 2 * N] = base.to(gpu)
        proj(xb[:, 8:8 + K], buf[:, 1:1 + N], base=buf[:, 1 + N:1 + 2 * N])
        check(buf[:, 1:1 + N], *reference(w, x, base))
        assert torch.equal(buf[:, 1 + N:1 + 2 * N].cpu(), base)
        rest = (buf[:, :1], buf[:, 1 + 2 * N:])
    assert all(bool((r == 7.0).all()) for r in rest)


@pytest.mark.parametrize("fmt,zeros", [("int4", "asym"), ("mxfp4", "none")])
@pytest.mark.parametrize("x_bf16", [False, True])
def test_row_that_is_not_finite(gpu, fmt, zeros, x_bf16):
    """Infinities and NaN stay in their own rows, whose outputs are not finite."""
    w = make_weight(fmt, zeros, 48, 256, 64, 4)
    x = rows(20, 256, 6, x_bf16)
    clean = run(gpu, w, x)
    bad = x.clone()
    bad[3, 17], bad[19, 255] = float("inf"), float("nan")
    y = run(gpu, w, bad)
    keep = [t for t in range(20) if t not in (3, 19)]
    assert torch.equal(y[keep], clean[keep])
    assert not torch.isfinite(y[19]).any()
    hit = dequant(w)[:, 17] != 0
    assert not torch.isfinite(y[3].cpu()[hit]).any()


@pytest.mark.parametrize("x_bf16", [False, True])
def test_large_rows(gpu, x_bf16):
    """Rows up to 5e33 with the zero points farthest from the codes: (16 + q + 16 + z)
    times a group's sum stays a number."""
    w = make_weight("int4", "mixed", 64, 512, 128, 4)
    x = rows(5, 512, 6, x_bf16).clamp(-4, 4) * 1.2e33
    check(run(gpu, w, x), *reference(w, x))


@pytest.mark.parametrize("x_bf16", [False, True])
def test_rows_far_apart(gpu, x_bf16):
    """Rows of x, y and base whose offsets pass 32 bits."""
    T, K, N, S = 40, 256, 48, 1 << 26
    w = make_weight("int4", "asym", N, K, 64, 4)
    x, base = rows(T, K, 6, x_bf16), rows(T, N, 7)
    xg = torch.empty(((T - 1) * S + K,), device=gpu, dtype=x.dtype).as_strided((T, K), (S, 1))
    y = torch.empty(((T - 1) * S + N,), device=gpu).as_strided((T, N), (S, 1))
    bg = torch.empty(((T - 1) * S + N,), device=gpu).as_strided((T, N), (S, 1))
    assert (T - 1) * S > 2 ** 31
    xg.copy_(x)
    bg.copy_(base)
    ops.Projection4(w.to(gpu), T)(xg, y, base=bg)
    check(y, *reference(w, x, base))


def test_zero_and_extreme_scales(gpu):
    """Scales of 0, the smallest and the largest; MXFP4's 2^-127 and 2^127, and
    its NaN in the rows and groups that have it."""
    w = make_weight("int4", "asym", 16, 128, 64, 4)
    s = torch.tensor([0.0, 1e-38, 3e38 / 16 / 1024, -2.0]).bfloat16()
    w.scales.copy_(s[torch.arange(32) % 4].view(16, 2).view(torch.int16))
    x = rows(3, 128, 6) / 16
    check(run(gpu, w, x), *reference(w, x))
    m = make_weight("mxfp4", "none", 16, 64, 32, 4)
    m.scales[:] = 127
    m.scales[0], m.scales[1], m.scales[2, 1] = 1, 250, 255
    x = rows(3, 64, 6)
    y = run(gpu, m, x).cpu()
    v, tol = reference(m, x)
    ok = [n for n in range(16) if n != 2]
    check(y[:, ok], v[:, ok], tol[:, ok] + 2.0 ** -126)
    assert torch.isnan(y[:, 2]).all()


@pytest.mark.parametrize("code", [0, 1])
def test_smallest_scales(gpu, code):
    """MXFP4's scales of 2^-127 and 2^-126: weights below bf16's and fp32's normal
    numbers, large rows."""
    m = make_weight("mxfp4", "none", 16, 64, 32, 4)
    for x_bf16 in (False, True):
        x = rows(3, 64, 6, x_bf16) * 1e30
        m.scales[:] = code + 100
        v, tol = reference(m, x)
        m.scales[:] = code
        check(run(gpu, m, x), v * 2.0 ** -100, tol * 2.0 ** -100)


def test_no_rows(gpu):
    w = make_weight("int4", "asym", 16, 64, 32, 1)
    proj = ops.Projection4(w.to(gpu), 4)
    proj(torch.empty((0, 64), device=gpu), torch.empty((0, 16), device=gpu))
    torch.cuda.synchronize()


@pytest.mark.parametrize("T,fmt", [(1, "int4"), (12, "mxfp4"), (40, "int4")])
def test_other_stream_and_graph(gpu, T, fmt):
    """On another stream; captured and replayed with new rows, eager calls of the
    same object between the replays."""
    K, N = 1024, 272
    w = make_weight(fmt, "asym", N, K, 128, 9)
    proj = ops.Projection4(w.to(gpu), T)
    x, y, e = torch.empty((T, K), device=gpu), torch.empty((T, N), device=gpu), torch.empty((T, N), device=gpu)
    x.copy_(rows(T, K, 0))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    proj(x, y, stream=side)
    side.synchronize()
    check(y, *reference(w, x.cpu()))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        proj(x, y)
    for seed in (1, 2, 3):
        x.copy_(rows(T, K, seed))
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        proj(x, e)
        torch.cuda.synchronize()
        assert torch.equal(y, e)
        check(y, *reference(w, x.cpu()))


def test_two_at_once(gpu):
    """Two projections on two streams, again and again the same bits."""
    a, b = (make_weight(f, "asym", 2048, 2048, 128, s) for f, s in (("int4", 1), ("mxfp4", 2)))
    pa, pb = ops.Projection4(a.to(gpu), 3), ops.Projection4(b.to(gpu), 20)
    xa, xb = rows(3, 2048, 1).to(gpu), rows(20, 2048, 2).to(gpu)
    ya, yb = torch.empty((3, 2048), device=gpu), torch.empty((20, 2048), device=gpu)
    pa(xa, ya)
    pb(xb, yb)
    sa, sb = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    za, zb = torch.empty_like(ya), torch.empty_like(yb)
    for _ in range(10):
        pa(xa, za, stream=sa)
        pb(xb, zb, stream=sb)
    torch.cuda.synchronize()
    assert torch.equal(za, ya) and torch.equal(zb, yb)


def test_rows_do_not_depend_on_the_batch(gpu):
    """A bf16 row's outputs are the same alone and in a batch of up to 16."""
    w = make_weight("int4", "asym", 80, 1536, 128, 5)
    x = rows(16, 1536, 5, True)
    y = run(gpu, w, x)
    for t in (0, 7, 15):
        v, tol = reference(w, x[t:t + 1])
        check(run(gpu, w, x[t:t + 1]), v, tol)
        check(y[t:t + 1], v, tol)


def test_weight_past_4_gib(gpu):
    """Payload, scale and zero offsets past 32 bits; the first and last rows."""
    N, K, g = 600_000, 16384, 32
    gen = torch.Generator(device=gpu).manual_seed(1)
    pay = torch.randint(0, 256, (N, K // 2), dtype=torch.uint8, device=gpu, generator=gen)
    sc = torch.rand((N, K // g), device=gpu, generator=gen).bfloat16().view(torch.int16)
    z = torch.randint(0, 16, (N, K // g), dtype=torch.uint8, device=gpu, generator=gen)
    x = rows(2, K, 3)
    y = torch.empty((2, N), device=gpu)
    ops.Projection4(Weight(_abi.FMT_INT4, N, K, pay, sc, z, K // g), 2)(x.to(gpu), y)
    torch.cuda.synchronize()
    for lo in (0, N - 40):
        part = Weight(_abi.FMT_INT4, 40, K, pay[lo:lo + 40].cpu(), sc[lo:lo + 40].cpu(), z[lo:lo + 40].cpu(), K // g)
        check(y[:, lo:lo + 40], *reference(part, x))


def test_host_refusals_on_the_gpu_objects(gpu):
    w = make_weight("int4", "asym", 16, 64, 32, 1).to(gpu)
    proj = ops.Projection4(w, 4)
    x, y = torch.zeros((4, 64), device=gpu), torch.zeros((4, 16), device=gpu)
    for args, kw in (((x.half(), y), {}), ((x[:, :32], y), {}), ((x, y[:, :8]), {}), ((x, y.half()), {}),
                     ((x.cpu(), y), {}), ((x, y.cpu()), {}), ((x.T.contiguous().T, y), {}),
                     ((x, y), dict(base=y.cpu())), ((x, y), dict(base=y[:2])),
                     ((torch.zeros((5, 64), device=gpu), torch.zeros((5, 16), device=gpu)), {})):
        with pytest.raises(_abi.GrimoireError):
            proj(*args, **kw)
    with pytest.raises(_abi.GrimoireError):
        proj(x.view(-1)[1:65].view(1, 64), y[:1])
    with pytest.raises(_abi.GrimoireError):
        proj.swiglu(x, y)
    for bad in (Weight(_abi.FMT_INT8, 16, 64, w.payload, w.scales, None, 1),
                Weight(w.fmt, 16, 64, w.payload, w.scales.float(), w.zeros, 2),
                Weight(w.fmt, 16, 64, w.payload, w.scales[:8], w.zeros, 2),
                Weight(w.fmt, 16, 64, w.payload, w.scales.view(torch.float16), w.zeros, 2),
                Weight(_abi.FMT_INT4_F16, 16, 64, w.payload, w.scales.view(torch.bfloat16), w.zeros, 2),
                Weight(w.fmt, 16, 64, w.payload.cpu(), w.scales, w.zeros, 2)):
        with pytest.raises(_abi.GrimoireError):
            ops.Projection4(bad, 4)
    shared = torch.zeros((8, 64), device=gpu)
    with pytest.raises(_abi.GrimoireError):
        proj(shared[:4], shared[:4, :16])                                             # output inside x
    lib = _abi.lib()
    assert lib.grimoire_proj4(None, C.byref(proj.struct), x.data_ptr(), 0, 64, None, 0, 0, w.payload.data_ptr(), 0, 16, 4,
                              *proj._ws) == _abi.ERR_ARG
    assert lib.grimoire_proj4(None, C.byref(proj.struct), x.data_ptr(), 0, 64, None, 0, 0, y.data_ptr(), 0, 16, 4, None,
                              0) == _abi.ERR_WORKSPACE
