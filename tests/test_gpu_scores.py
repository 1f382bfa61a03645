"""Router scores (grimoire_moe_router_scores) against the definition in 64
bits, token by token: the same experts in the same order, and the weights to
half a step of fp32 (the kernel computes them in fp64 and rounds once)."""
import math

import pytest
import torch

from grimoire_amd import ops

pytestmark = pytest.mark.gpu


def want(logits, K, score="softmax", bias=None, n_group=1, topk_group=1, group_score="max", normalize=True,
         scaling=1.0):
    """The definition, in Python floats (64 bits)."""
    T, E = logits.shape
    ids = torch.full((T, K), -1, dtype=torch.int32)
    ws = torch.zeros((T, K), dtype=torch.float64)
    big = torch.finfo(torch.float32).max
    b = [0.0] * E if bias is None else bias.double().tolist()
    for t, row in enumerate(logits.double().tolist()):
        row = [-math.inf if math.isnan(l) else min(l, big) for l in row]
        top = max(row)
        if score == "softmax":
            ex = [math.exp(l - top) if l > -math.inf else 0.0 for l in row]
            z = math.fsum(ex)
            s = [v / z if z > 0 else 0.0 for v in ex]
        else:
            # below -745 the value is under the smallest double: 0
            s = [1.0 / (1.0 + math.exp(-l)) if l > -700.0 else math.exp(max(l, -1e6)) for l in row]
        sel = [s[e] + b[e] if row[e] > -math.inf else -math.inf for e in range(E)]
        sel = [-math.inf if math.isnan(v) else v for v in sel]
        live = [e for e in range(E) if sel[e] > -math.inf]
        if n_group > 1:
            gs = E // n_group
            rated = []
            for g in range(n_group):
                v = sorted((sel[e] for e in live if e // gs == g), reverse=True)
                r = -math.inf if not v else v[0] + (v[1] if group_score == "top2" and len(v) > 1 else 0.0)
                rated.append((-r, g))
            kept = {g for _, g in sorted(rated)[:topk_group]}
            live = [e for e in live if e // gs in kept]
        pick = sorted(live, key=lambda e: (-sel[e], e))[:K]
        w = [s[e] for e in pick]
        if normalize:
            z = math.fsum(w)
            w = [v / z if z > 0 else 0.0 for v in w]
        for i, e in enumerate(pick):
            ids[t, i], ws[t, i] = e, w[i] * float(torch.tensor(scaling, dtype=torch.float32))
    return ids, ws


def run(gpu, logits, K, bias=None, stream=None, **kw):
    T = logits.shape[0]
    ids = torch.full((T, K), -7, dtype=torch.int32, device=gpu)
    w = torch.full((T, K), float("nan"), device=gpu)
    r = ops.RouteScores(bias=None if bias is None else bias.to(gpu), **kw)
    r(logits if logits.is_cuda else logits.to(gpu), ids, w, stream=stream)
    torch.cuda.synchronize()
    return ids.cpu(), w.cpu()


def check(gpu, logits, K, bias=None, **kw):
    ids, w = run(gpu, logits, K, bias, **kw)
    wi, ww = want(logits.cpu(), K, bias=bias, **kw)
    assert torch.equal(ids, wi)
    # one rounding to fp32 (2^-24 relative, 2^-150 below the normal range)
    # of a value off by a few steps of fp64
    assert ((w.double() - ww).abs() <= ww.abs() * (2.0 ** -24 + 1e-13) + 2.0 ** -149).all()
    return ids, w


def rand(T, E, seed, std=1.2):
    return torch.randn(T, E, generator=torch.Generator().manual_seed(seed)) * std


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("T,E,K", [(1, 128, 8), (1, 1, 1), (5, 3, 3), (33, 64, 16), (7, 65, 5), (6, 130, 10),
                                   (9, 300, 7), (70, 512, 16), (2, 511, 4)])
def test_scores(gpu, T, E, K, score):
    print(f"scores T={T} E={E} K={K} {score}", flush=True)
    l = rand(T, E, T + E)
    b = rand(1, E, 3, 0.05)[0]
    check(gpu, l, K, score=score)
    check(gpu, l, K, b, score=score, normalize=False, scaling=2.5)
    check(gpu, l.bfloat16(), K, b, score=score)


@pytest.mark.parametrize("group_score", ["max", "top2"])
@pytest.mark.parametrize("E,G,kept,K", [(256, 8, 4, 8), (60, 3, 1, 7), (495, 33, 20, 16), (64, 64, 10, 10),
                                        (510, 5, 2, 16), (30, 2, 2, 4), (63, 7, 3, 6), (512, 17 - 1, 5, 16)])
def test_groups(gpu, E, G, kept, K, group_score):
    print(f"groups E={E} G={G} kept={kept} K={K} {group_score}", flush=True)
    l, b = rand(19, E, E + G), rand(1, E, 5, 0.05)[0]
    for score in ("softmax", "sigmoid"):
        check(gpu, l, K, b, score=score, n_group=G, topk_group=kept, group_score=group_score)
    out = torch.rand(19, E, generator=torch.Generator().manual_seed(1)) < 0.9
    l[out] = -math.inf                     # groups with one expert left, and with none
    check(gpu, l, K, b, score="sigmoid", n_group=G, topk_group=kept, group_score=group_score)


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_ties_and_borders(gpu, score):
    """Equal logits go to the lower index; logits one fp32 step apart, whose
    fp32 scores round together, keep their order."""
    l = rand(64, 200, 4).round()
    check(gpu, l, 12, score=score)
    check(gpu, l, 9, score=score, n_group=10, topk_group=3, group_score="top2")
    check(gpu, torch.zeros(3, 512), 16, score=score)              # more ties than lanes
    check(gpu, torch.zeros(3, 512), 16, score=score, n_group=64, topk_group=9)
    near = torch.full((4, 96), 0.75)
    near[:, 50] = torch.nextafter(near[0, 0], torch.tensor(1.0))
    near[:, 20] = torch.nextafter(near[0, 0], torch.tensor(0.0))
    ids, _ = check(gpu, near, 2, score=score)
    assert ids[0].tolist() == [50, 0]


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
def test_masks_and_special_values(gpu, score):
    l = rand(12, 70, 6)
    l[0] = -math.inf                       # nothing left
    l[1, 3:] = -math.inf                   # fewer than K left
    l[2, ::2] = float("nan")
    l[3] = float("nan")
    l[4, 5] = math.inf
    l[5, :] = torch.finfo(torch.float32).min    # the type's lowest value is a number
    l[6, 10:] = torch.finfo(torch.float32).min
    l[7, 9] = l[7, 4] = math.inf
    l[8] = 300.0
    l[9] = -300.0 - torch.arange(70.0)
    check(gpu, l, 8, score=score)
    check(gpu, l, 8, score=score, normalize=False)
    b = rand(1, 70, 8, 0.1)[0]
    b[1], b[2], b[3] = math.inf, -math.inf, float("nan")
    check(gpu, l, 8, b, score=score)
    check(gpu, l, 8, b, score=score, n_group=7, topk_group=2)


def test_rows_apart_streams_and_graph(gpu):
    """Rows with a stride, another stream, and a captured call replayed on new logits."""
    wide = rand(40, 300, 9).to(gpu)
    view = wide[:, 37:37 + 201]
    assert not view.is_contiguous()
    check(gpu, view, 6)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    ids, w = run(gpu, view, 6, stream=s)
    assert torch.equal(ids, want(view.cpu(), 6)[0])

    l = rand(9, 128, 10).to(gpu)
    ids = torch.empty(9, 8, dtype=torch.int32, device=gpu)
    w = torch.empty(9, 8, device=gpu)
    r = ops.RouteScores()
    r(l, ids, w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        r(l, ids, w)
    for i in range(3):
        new = rand(9, 128, 20 + i)
        l.copy_(new)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(ids.cpu(), want(new, 8)[0])


def test_many_tokens(gpu):
    """A full prompt: routes and bits do not depend on a token's place."""
    l = rand(4099, 256, 11)
    l[4098] = l[0]
    b = rand(1, 256, 12, 0.002)[0]
    ids, w = run(gpu, l, 8, b, normalize=False)
    wi, _ = want(l[::131], 8, bias=b, normalize=False)
    assert torch.equal(ids[::131], wi)
    assert torch.equal(ids[4098], ids[0]) and torch.equal(w[4098], w[0])
