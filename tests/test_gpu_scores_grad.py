"""The gradient of the router scores (grimoire_moe_router_scores_grad) against
autograd of their definition in 64 bits.

Tolerance, u = 2^-24.  A score's relative error: the difference l - m rounded
(|l - m| u, at most R u with R the row's spread, 2 |l| of a sigmoid), exp and a
division of a few steps, a sum of 8 + 6 steps; the sums over picks 6 steps more;
products and differences a few: (R + 64) u of s (|du| + sum u |du|), where |du|
of renormalised weights is (|g| + sum p |g|) / Z.  A bf16 output adds half a
step, 2^-8.  An exponential below 2^-126, the smallest normal number, may be 0:
the score s is then off by at most 2^-126 (its divisor, the sum of all, is at
least 1), which s (du - sum u du) multiplies by at most |du| + sum u |du|; a
result below 2^-126 may be 0 as well: 2^-126 (1 + |du| + sum u |du|) more."""
import math

import pytest
import torch

from grimoire_amd import _abi, ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
NAN, INF = float("nan"), float("inf")


def case(T, E, K, seed, bf16=False, std=1.5):
    g = torch.Generator().manual_seed(seed)
    l = torch.randn((T, E), generator=g) * std + torch.randn((E,), generator=g)
    l = l.bfloat16() if bf16 else l
    ids = torch.topk(l.float() + torch.randn((E,), generator=g), K, dim=1).indices.int()
    return l, ids, torch.randn((T, K), generator=g)


def want(l, ids, dw, score, normalize, scaling):
    x = l.double().nan_to_num(nan=-INF, posinf=3.402823466e+38, neginf=-INF).requires_grad_()
    E = l.shape[1]
    live = (ids >= 0) & (ids < E)
    at = ids.clamp(0, E - 1).long()
    s = torch.softmax(x, 1) if score == "softmax" else torch.sigmoid(x)
    s = torch.where(torch.isnan(s), 0.0, s)          # a row without an expert
    u = s.gather(1, at).masked_fill(~live, 0.0)
    g = dw.double().masked_fill(~live, 0.0) * scaling
    z = u.sum(1, keepdim=True)
    w = u / torch.where(z > 0, z, 1.0) if normalize else u
    # 1 - s of a sigmoid near 1 is s of -x: autograd of sigmoid forms the difference
    ds = torch.autograd.grad((w * g).sum(), s, retain_graph=True)[0]
    d = ds * s * torch.sigmoid(-x) if score == "sigmoid" else torch.autograd.grad((w * g).sum(), x)[0]
    d = d.detach().nan_to_num(0.0)
    with torch.no_grad():
        fin = torch.where(torch.isfinite(x), x, 0.0)
        R = (fin.amax(1, keepdim=True) - fin.amin(1, keepdim=True)) + 2 * fin.abs().amax(1, keepdim=True)
        du = g.abs()
        if normalize:
            zz = torch.where(z > 0, z, 1.0)
            du = (g.abs() + (u * g.abs()).sum(1, keepdim=True) / zz) / zz
        dense = torch.zeros_like(s).scatter_add_(1, at, du.masked_fill(~live, 0.0))
        if score == "softmax":
            by = dense + (u * du).sum(1, keepdim=True)
            mag = s * by
        else:
            by = dense
            mag = s * torch.sigmoid(-x) * by
    return d, (R.clamp(max=400.0) + 64) * U * mag + 2.0 ** -126 * (1 + by)


def run(gpu, l, ids, dw, score="softmax", normalize=True, scaling=1.0, inplace=False, **kw):
    sc = ops.RouteScores(score, normalize=normalize, scaling=scaling)
    lg = l.to(gpu)
    out = lg if inplace else torch.full_like(lg, NAN)
    sc.grad(lg, ids.to(gpu), dw.to(gpu), out, **kw)
    torch.cuda.synchronize()
    return out.cpu()


def check(out, d, tol):
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (d.abs() + tol)
    err = (out.double() - d).abs()
    assert (err <= tol).all(), float((err / tol).max())


FORMS = [(s, n) for s in ("softmax", "sigmoid") for n in (False, True)]


@pytest.mark.parametrize("T,E,K", [(1, 1, 1), (1, 128, 8), (3, 64, 4), (5, 65, 16), (32, 256, 8), (33, 100, 1),
                                   (130, 512, 10), (9, 511, 16), (4, 16, 16)])
@pytest.mark.parametrize("score,normalize", FORMS)
def test_sizes(gpu, T, E, K, score, normalize):
    for bf16 in (False, True):
        print(f"scores_grad T={T} E={E} K={K} {score} {normalize} {bf16}", flush=True)
        l, ids, dw = case(T, E, K, T + E, bf16)
        ref = want(l, ids, dw, score, normalize, 2.5)
        out = run(gpu, l, ids, dw, score, normalize, 2.5)
        check(out, *ref)
        assert torch.equal(run(gpu, l, ids, dw, score, normalize, 2.5, inplace=True), out)


@pytest.mark.parametrize("score,normalize", FORMS)
def test_empty_slots_and_repeats(gpu, score, normalize):
    """Slots without an expert (also out of range), a row of none, an expert
    picked twice; infinite gradients of empty slots do not count."""
    l, ids, dw = case(12, 48, 6, 5)
    ids[0] = -1
    ids[1, 3:] = -1
    ids[2, 1], ids[3, 2], ids[4, 0] = 48, 2 ** 31 - 1, -2 ** 31
    ids[5] = ids[5, 0]
    ids[6, 4] = ids[6, 1]
    dw[0], dw[1, 5], dw[2, 1] = NAN, INF, NAN
    ref = want(l, ids, dw, score, normalize, 1.0)
    out = run(gpu, l, ids, dw, score, normalize)
    check(out, *ref)
    assert not out[0].any()


@pytest.mark.parametrize("score,normalize", FORMS)
def test_experts_out_and_far_logits(gpu, score, normalize):
    """-inf and NaN logits are out, +inf is the largest finite one; scores that
    vanish, rows of one value."""
    l, ids, dw = case(10, 80, 4, 6, std=30.0)
    l[0, ids[0, 0].long()] = -INF
    l[1, 5], l[2, ids[2, 1].long()], l[3, 7] = NAN, NAN, -3.4e38
    l[4] = 0.25
    l[5] = -INF
    l[6, ids[6, 2].long()] = INF
    l[7] *= 1e-30
    out = run(gpu, l, ids, dw, score, normalize)
    assert torch.isfinite(out).all()
    d, tol = want(l, ids, dw, score, normalize, 1.0)
    keep = [t for t in range(10) if t not in (3, 6)]         # spreads no fp32 step can count
    check(out[keep], d[keep], tol[keep])
    assert not out[5].any()
    assert out[0, ids[0, 0].long()] == 0 and out[2, ids[2, 1].long()] == 0 and out[1, 5] == 0


def test_renormalised_softmax_leaves_the_rest_at_zero(gpu):
    l, ids, dw = case(20, 200, 8, 7)
    out = run(gpu, l, ids, dw)
    picked = torch.zeros((20, 200), dtype=torch.bool).scatter_(1, ids.long(), True)
    assert not out[~picked].any() and out[picked].any()


def test_against_differences(gpu):
    """A central difference of the scores' own weights (choice held by keeping the
    step small) along a random direction."""
    for score, normalize in FORMS:
        l, _, dw = case(16, 64, 4, 8)
        sc = ops.RouteScores(score, normalize=normalize, scaling=1.5)
        ids, w = torch.empty((16, 4), dtype=torch.int32, device=gpu), torch.empty((16, 4), device=gpu)

        def weights(x):
            sc(x.float().to(gpu).contiguous(), ids, w)
            torch.cuda.synchronize()
            return ids.cpu().clone(), w.cpu().double()
        base = weights(l)[0]
        v = torch.randn((16, 64), generator=torch.Generator().manual_seed(9)).double()
        out = run(gpu, l, base, dw, score, normalize, 1.5).double()
        h = 2.0 ** -10
        up, wu = weights(l.double() + h * v)
        dn, wd = weights(l.double() - h * v)
        same = (up == base).all(1) & (dn == base).all(1)
        assert same.sum() >= 8
        num = ((wu - wd) * dw.double()).sum(1) / (2 * h)
        # h^2 / 6 of a third derivative (a weight's is below 4 |v|^3 times it), fp32 weights over 2 h
        size = dw.double().abs().sum(1) * 1.5
        tol = size * (h * h / 6 * 4 * v.abs().amax(1) ** 3 * 8 + 2 * U * 16 / (2 * h)) + 2.0 ** -18 * size
        assert ((num - (out * v).sum(1)).abs() <= tol)[same].all()


@pytest.mark.parametrize("bf16", [False, True])
def test_rows_apart(gpu, bf16):
    l, ids, dw = case(11, 70, 5, 3, bf16)
    for score, normalize in FORMS:
        buf = torch.full((11, 101), NAN, device=gpu, dtype=l.dtype)
        out = torch.full((11, 83), 7.0, device=gpu, dtype=l.dtype)
        buf[:, 3:73] = l.to(gpu)
        sc = ops.RouteScores(score, normalize=normalize)
        sc.grad(buf[:, 3:73], ids.to(gpu), dw.to(gpu), out[:, 5:75])
        torch.cuda.synchronize()
        assert torch.equal(out[:, 5:75].cpu(), run(gpu, l, ids, dw, score, normalize))
        assert bool((out[:, :5] == 7.0).all()) and bool((out[:, 75:] == 7.0).all())


def test_bias_and_groups_have_no_gradient(gpu):
    l, _, dw = case(16, 64, 4, 4)
    bias = torch.randn((64,), generator=torch.Generator().manual_seed(1)).to(gpu) * 0.1
    sc = ops.RouteScores("sigmoid", bias=bias, n_group=8, topk_group=4, group_score="top2", scaling=2.0)
    ids, w, d = torch.empty((16, 4), dtype=torch.int32, device=gpu), torch.empty((16, 4), device=gpu), \
        torch.empty((16, 64), device=gpu)
    lg = l.to(gpu)
    sc(lg, ids, w)
    sc.grad(lg, ids, dw.to(gpu), d)
    torch.cuda.synchronize()
    check(d.cpu(), *want(l, ids.cpu(), dw, "sigmoid", True, 2.0))


def test_other_stream_and_graph(gpu):
    l, ids, dw = case(64, 128, 8, 2)
    sc = ops.RouteScores("softmax", normalize=False)
    lg, ig, dg = l.to(gpu), ids.to(gpu), dw.to(gpu)
    out, e = torch.empty_like(lg), torch.empty_like(lg)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    sc.grad(lg, ig, dg, out, stream=side)
    side.synchronize()
    check(out.cpu(), *want(l, ids, dw, "softmax", False, 1.0))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        sc.grad(lg, ig, dg, out)
    for seed in (3, 4, 5):
        n = case(64, 128, 8, seed)
        for a, b in zip((lg, ig, dg), n):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        sc.grad(lg, ig, dg, e)
        torch.cuda.synchronize()
        assert torch.equal(out, e)


def test_host_refusals_on_the_gpu_objects(gpu):
    l, ids, dw = (t.to(gpu) for t in case(4, 32, 4, 1))
    sc, d = ops.RouteScores(), torch.empty((4, 32), device=gpu)
    for args in ((l, ids.long(), dw, d), (l, ids, dw[:, :2], d), (l, ids, dw, d.bfloat16()), (l, ids, dw, d.cpu()),
                 (l.half(), ids, dw, d), (l, ids.cpu(), dw, d), (l, ids, dw, d[:, :16]), (l.cpu(), ids, dw, d)):
        with pytest.raises(_abi.GrimoireError):
            sc.grad(*args)
    buf = torch.zeros((8, 32), device=gpu)
    with pytest.raises(_abi.GrimoireError):
        sc.grad(buf[:4], ids, dw, buf[1:5])
