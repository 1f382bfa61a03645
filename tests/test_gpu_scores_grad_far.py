"""The gradient of renormalised router scores where every pick's logit is far
below zero, and of infinite logits, against 64 bits.

With p_k = e^ls(l_k) / sum_j e^ls(l_j), ls the logarithm of a sigmoid (softmax:
the logit itself), s the sigmoid and g_k = scaling * dweight_k:
  dlogits_k = p_k (1 - s_k) (g_k - sum_j p_j g_j)     (softmax: without 1 - s_k).

Tolerance, u = 2^-24, R the spread of min(l, 0) (softmax: l) over the picks, at
most 104 (what is further away has an exponential of 0).  The difference of two of them is rounded: R u of its exponential, which is off by 4 u
itself; 1 / (1 + e^-|l|) 5 u; their product 1: (R + 10) u.  A sum over lanes 6
more, a division 1: p (2 R + 27) u.  sum p g: 8 u more, relative to sum p |g|.
1 - s 10 u, g, a difference and two products 4: (4 R + 80) u of
p (1 - s) (|g| + sum p |g|).  An exponential below 2^-126 may be 0, where what it
is divided by is at least 1/2, and so may a result: 2^-124 (1 + |g| + sum |g|).
A bf16 output adds half a step, 2^-8.  Nothing here is divided by the sum of the
scores."""
import pytest
import torch

from grimoire_amd import ops

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
INF = float("inf")


def want(l, ids, dw, score, scaling):
    x = l.double()
    at = ids.long()
    pl, g = x.gather(1, at), dw.double() * scaling
    flat = pl.clamp(max=0.0) if score == "sigmoid" else pl
    p = torch.softmax(torch.nn.functional.logsigmoid(pl) if score == "sigmoid" else pl, 1)
    f = torch.sigmoid(-pl) if score == "sigmoid" else torch.ones_like(pl)
    S = lambda t: (p * t).sum(1, keepdim=True)
    d = p * f * (g - S(g))
    R = (flat.amax(1, keepdim=True) - flat.amin(1, keepdim=True)).clamp(max=104.0)
    tol = (4 * R + 80) * U * p * f * (g.abs() + S(g.abs())) + 2.0 ** -124 * (1 + g.abs() + g.abs().sum(1, keepdim=True))
    out = lambda v: torch.zeros_like(x).scatter_add_(1, at, v)
    return out(d), out(tol)


def run(gpu, l, ids, dw, score, normalize=True, scaling=1.0):
    lg = l.to(gpu)
    out = torch.full_like(lg, float("nan"))
    ops.RouteScores(score, normalize=normalize, scaling=scaling).grad(lg, ids.to(gpu), dw.to(gpu), out)
    torch.cuda.synchronize()
    return out.cpu()


def check(out, d, tol):
    if out.dtype == torch.bfloat16:
        tol = tol + 2.0 ** -8 * (d.abs() + tol)
    err = (out.double() - d).abs()
    assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


def picks(T, E, K, g):
    return torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).int()


LEVELS = [0.0, -60.0, -84.0, -86.0, -87.0, -87.4, -88.5, -90.0, -104.0, -120.0, -300.0, -700.0]


@pytest.mark.parametrize("score", ["sigmoid", "softmax"])
@pytest.mark.parametrize("level", LEVELS)
def test_far_logits(gpu, score, level):
    """All of a token's logits near one level, large gradients."""
    for n, (T, E, K) in enumerate([(1, 16, 1), (3, 8, 2), (40, 64, 4), (33, 300, 8), (9, 512, 16)]):
        g = torch.Generator().manual_seed(n)
        for bf16 in (False, True):
            print(f"far {score} level={level} T={T} E={E} K={K} bf16={bf16}", flush=True)
            l = level + torch.randn((T, E), generator=g) * 1.5
            l = l.bfloat16() if bf16 else l
            ids, dw = picks(T, E, K, g), torch.randn((T, K), generator=g) * 50
            out = run(gpu, l, ids, dw, score, scaling=2.5)
            check(out, *want(l, ids, dw, score, 2.5))
            if K > 1:
                assert bool(out.any(1).all())


def test_values_worked_out_by_hand(gpu):
    """Sigmoids this far down are e^l: p is the softmax of the picks, 1 - s is 1."""
    l = torch.tensor([[-86.0, -86.2, -86.4], [-87.0, -87.0, -500.0], [-90.0, -91.0, -90.0], [-86.0, -87.2, -600.0]])
    ids = torch.tensor([[0, 1, 2]] * 4, dtype=torch.int32)
    dw = torch.tensor([[50.0, -200.0, 0.5], [12.0, -12.0, 0.0], [1.0, -2.0, 0.5], [20.0, -20.0, 0.0]])
    d = torch.tensor([[38.394, -50.799, 12.405], [6.0, -6.0, 0.0], [0.2860, -0.3609, 0.0749], [7.1158, -7.1158, 0.0]])
    assert (run(gpu, l, ids, dw, "sigmoid") - d).abs().max() <= 1e-3


def test_picks_far_apart(gpu):
    """Ordinary picks beside far ones, in either order; experts that are out."""
    g = torch.Generator().manual_seed(3)
    T, E, K = 64, 96, 6
    l = torch.randn((T, E), generator=g)
    l = torch.where(torch.rand((T, E), generator=g) < 0.5, l - 95.0, l)
    l = torch.where(torch.rand((T, E), generator=g) < 0.1, l + 120.0, l)
    ids, dw = picks(T, E, K, g), torch.randn((T, K), generator=g) * 30
    check(run(gpu, l, ids, dw, "sigmoid", scaling=1.5), *want(l, ids, dw, "sigmoid", 1.5))
    far = l - 130.0
    far[torch.rand((T, E), generator=g) < 0.1] = -INF
    far.scatter_(1, ids[:, :1].long(), -100.0)              # a token keeps one expert
    check(run(gpu, far, ids, dw, "sigmoid"), *want(far.clamp(min=-3e38), ids, dw, "sigmoid", 1.0))


@pytest.mark.parametrize("level", [0.0, -85.0, -87.0, -90.0, -110.0])
def test_against_differences_of_the_forward(gpu, level):
    """Along a random direction, the forward's weights of both sides.  Logits and
    steps are multiples of 2^-12, so both sides are exact.  A weight's third
    derivative along the step is at most 3 w D^3, D = 2 max |step| = 2^-8: a third
    of it, w D^3 = 2^-24 w, is what the difference is off by; the fp32 weights u
    each."""
    T, E, K = 32, 64, 4
    g = torch.Generator().manual_seed(int(-level))
    l = level + torch.randint(-4096, 4097, (T, E), generator=g) / 4096.0
    step = torch.randint(-8, 9, (T, E), generator=g) / 4096.0
    dw = torch.randn((T, K), generator=g)
    sc = ops.RouteScores("sigmoid", scaling=1.5)
    ids, w = torch.empty((T, K), dtype=torch.int32, device=gpu), torch.empty((T, K), device=gpu)

    def weights(x):
        sc(x.to(gpu), ids, w)
        torch.cuda.synchronize()
        return ids.cpu().clone(), w.cpu().double()
    base, w0 = weights(l)
    up, wu = weights(l + step)
    dn, wd = weights(l - step)
    same = (up == base).all(1) & (dn == base).all(1)
    assert same.sum() >= 16
    out = run(gpu, l, base, dw, "sigmoid", scaling=1.5).double()
    _, tol = want(l, base, dw, "sigmoid", 1.5)
    size = (dw.double().abs() * w0).sum(1)
    num = (dw.double() * (wu - wd)).sum(1)
    part = (out * 2 * step.double()).sum(1)
    bound = size * 1.01 * (2.0 ** -24 + 2 * U) + (tol * 2 * step.double().abs()).sum(1)
    assert ((num - part).abs() <= bound)[same].all()
    assert bool((part.abs() > 4 * bound)[same].any())


def test_where_the_forward_has_no_weights(gpu):
    """Every pick's sigmoid 0 in 64 bits: the forward's weights are 0, the gradient
    too; on this side of that border both are there."""
    l = torch.tensor([[-709.0, -709.5, -709.7, -800.0], [-710.0, -711.0, -712.0, -800.0], [-3e38] * 4, [-INF] * 4])
    sc = ops.RouteScores("sigmoid")
    ids, w = torch.empty((4, 3), dtype=torch.int32, device=gpu), torch.empty((4, 3), device=gpu)
    sc(l.to(gpu), ids, w)
    torch.cuda.synchronize()
    dw = torch.tensor([[1.0, -2.0, 3.0]] * 4)
    out = run(gpu, l, ids.cpu().clamp(min=0), dw, "sigmoid")
    assert bool(w[0].all()) and not w[1:].any()
    assert bool(out[0, :3].all()) and not out[1:].any() and out[0, 3] == 0


@pytest.mark.parametrize("normalize", [False, True])
def test_infinite_logits(gpu, normalize):
    """+inf counts as the largest finite logit.  Softmax: its score is 1, every other
    0, and the whole row's gradient 0, picked or not (renormalised: if picked).  Sigmoid: 1 - s is 0 there, and
    the other picks' are those beside a score of 1."""
    g = torch.Generator().manual_seed(8)
    T, E, K = 12, 80, 4
    l, ids, dw = torch.randn((T, E), generator=g), picks(T, E, K, g), torch.randn((T, K), generator=g)
    for picked in (True, False):
        at = ids[:, 1:2].long() if picked else torch.tensor([[next(e for e in range(E) if e not in r)] for r in ids.tolist()])
        hot = l.scatter(1, at, INF)
        out = run(gpu, hot, ids, dw, "softmax", normalize)
        if picked or not normalize:
            assert not out.any()
        else:                                               # the picks alone
            check(out, *want(l, ids, dw, "softmax", 1.0))
        out = run(gpu, hot, ids, dw, "sigmoid", normalize)
        assert not out.gather(1, at).any()
        one = l.scatter(1, at, 200.0)
        assert torch.equal(out, run(gpu, one, ids, dw, "sigmoid", normalize))
        if normalize:
            check(out, *want(one, ids, dw, "sigmoid", 1.0))
