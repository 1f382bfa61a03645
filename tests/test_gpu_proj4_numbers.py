"""What the dense 4-bit projections do with numbers at the edges; weights, formula
and tolerances of test_gpu_proj4."""
import pytest
import torch

from helpers import dequant
from test_gpu_proj4 import check, make_weight, reference, rows, run

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def with_infinities(T, K, seed, b16):
    """Rows 0, 3, 6 ...: one infinity, two of a sign, two of both signs, a NaN."""
    x = rows(T, K, seed, b16)
    for n, t in enumerate(range(0, T, 3)):
        x[t, (37 * n) % K] = INF if n % 2 else -INF
        if n % 4 == 1:
            x[t, (37 * n + 8) % K] = INF
        if n % 4 == 2:
            x[t, (37 * n + K // 2) % K] = INF
        if n % 4 == 3:
            x[t, (37 * n + 1) % K] = NAN
    return x


SIZES = [(1, 96, 34), (4, 2048, 40), (9, 320, 20), (20, 416, 48), (16, 7168, 24), (33, 1024, 18)]


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("b16", [False, True])
def test_infinities_with_mxfp4(gpu, T, K, N, b16):
    """As the formula has them, in 64 bits: x of either type, K whole or in parts."""
    w = make_weight("mxfp4", "none", N, K, 32, T)
    x = with_infinities(T, K, T, b16)
    v, tol = reference(w, x)
    fin = torch.isfinite(x).all(1)
    y = run(gpu, w, x)
    if fin.any():
        check(y[fin.to(gpu)], v[fin], tol[fin])
    torch.testing.assert_close(y.cpu().double()[~fin], v[~fin], rtol=0, atol=0, equal_nan=True)
    assert torch.isinf(v[~fin]).any() and torch.isnan(v[~fin]).any()


@pytest.mark.parametrize("T,K,N", SIZES)
@pytest.mark.parametrize("b16", [False, True])
def test_infinities_with_int4(gpu, T, K, N, b16):
    """Rows with one are NaN throughout, the others as they are without."""
    for fmt, zeros in (("int4", "asym"), ("int4_f16", "none")):
        w = make_weight(fmt, zeros, N, K, 32, T)
        x = with_infinities(T, K, T, b16)
        fin = torch.isfinite(x).all(1)
        y = run(gpu, w, x)
        assert torch.isnan(y.cpu()[~fin]).all()
        assert torch.equal(y.cpu()[fin], run(gpu, w, torch.where(fin[:, None], x, torch.ones_like(x))).cpu()[fin])


@pytest.mark.parametrize("b16", [False, True])
def test_swiglu_of_an_infinity(gpu, b16):
    """MXFP4: silu(g) u as the formula has it, g / (1 + e^-g) u."""
    w = make_weight("mxfp4", "none", 64, 96, 32, 2)
    x = rows(5, 96, 2, b16)
    x[2, 40], x[4, 7] = INF, -INF
    y = run(gpu, w, x, glu=True).cpu()
    p = x.double() @ dequant(w)[:, :96].double().T
    g, u = p[:, :32], p[:, 32:]
    v = g / (1 + torch.exp(-g)) * u
    for t in (2, 4):
        torch.testing.assert_close(y[t].double(), v[t], rtol=0, atol=0, equal_nan=True)
    ok = [0, 1, 3]
    want, tol = reference(w, x[ok], glu=True)
    check(y[ok], want, tol)


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("b16", [False, True])
def test_codes_at_their_zero_point(gpu, group, b16):
    """The formula has 0: what is left is rounding of sums of (16 + q) x and x."""
    w = make_weight("int4", "asym", 32, 1024, group, 7)
    w.zeros.clamp_(max=15)
    code = w.zeros.repeat_interleave(group // 2, dim=1)
    w.payload.copy_(code | code << 4)
    x = rows(6, 1024, 7, b16) + 2.0
    v, tol = reference(w, x)
    assert not v.any()
    check(run(gpu, w, x), v, tol)


@pytest.mark.parametrize("b16", [False, True])
def test_largest_scales_of_mxfp4(gpu, b16):
    """Scale byte 252 with every code, 254 with codes up to 1."""
    w = make_weight("mxfp4", "none", 48, 128, 32, 9)
    w.scales.fill_(252)
    x = rows(5, 128, 9, b16) * 2.0 ** -30
    check(run(gpu, w, x), *reference(w, x))
    w.scales.fill_(254)
    codes = torch.tensor([0, 1, 2, 8, 9, 10], dtype=torch.uint8)
    w.payload.copy_(codes[(w.payload % 6).long()] | codes[(w.payload // 6 % 6).long()] << 4)
    assert dequant(w).abs().max() <= 2.0 ** 127
    check(run(gpu, w, x), *reference(w, x))


@pytest.mark.parametrize("b16,most", [(True, 16), (False, 4)])
def test_rows_alone_and_in_a_batch(gpu, b16, most):
    """The same bits where x of a whole row stays in the LDS for either, as K is
    shared out alike then (wider rows: header)."""
    for fmt in ("int4", "mxfp4"):
        w = make_weight(fmt, "asym", 80, 1536, 128, 5)
        x = rows(most, 1536, 5, b16)
        y = run(gpu, w, x)
        for t in (0, 1, most - 1):
            assert torch.equal(run(gpu, w, x[t:t + 1]), y[t:t + 1])
