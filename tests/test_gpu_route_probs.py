"""GRIM_ROUTE_PROBS in the whole layer: the forward's routes are those of the
definition in 64 bits on the layer's own logits, and its outputs those of the
CPU oracle on the routes it reports, in every regime and format."""
import ctypes as C

import pytest
import torch

from grimoire_amd import _abi, configs, ops
from oracle import oracle as O
from tests.helpers import assert_close
from tests.test_gpu_scores import want

pytestmark = pytest.mark.gpu

CASES = [  # regime, name, T, E, K, H, I, fmt, n_group, topk_group, shared
    (0, "one", 1, 64, 6, 512, 256, "int4", 1, 1, False),
    (1, "slots", 4, 64, 6, 512, 256, "mxfp4", 0, 0, False),
    (7, "one_launch", 1, 32, 4, 512, 256, "int4", 8, 3, False),
    (3, "stages", 5, 64, 8, 512, 256, "int8", 4, 2, True),
    (2, "gemm", 70, 32, 4, 512, 256, "int8", 1, 1, True),
    (2, "gemm_mx", 40, 32, 4, 512, 256, "mxfp4", 1, 1, False),
    (4, "grouped", 12, 64, 8, 512, 512, "mxfp4", 8, 3, False),
    (5, "grouped_valu", 12, 64, 8, 512, 512, "int4", 1, 1, False),
    (0, "wreg", 60, 32, 4, 512, 256, "bf16", 1, 1, False),
    (0, "prompt", 520, 32, 4, 512, 256, "int8", 4, 2, False),
    # the split-K router leaves two partial sums: the scores kernel adds them
    (0, "split_router", 4200, 64, 4, 512, 128, "int8", 1, 1, False),
]


def layer(c, gpu):
    regime, name, T, E, K, H, I, fmt, G, kept, shared = c
    cfg = configs.Config(name, T, H, E, K, I, fmt, route=_abi.ROUTE_PROBS, shared=shared, n_group=G, topk_group=kept,
                         scaling=2.5, bias_std=1e-2)
    wl = configs.make_workload(cfg, "cpu", seed=T + E)
    wl.layer.norm_topk = T % 2 == 0
    return cfg, wl


@pytest.mark.parametrize("c", CASES, ids=[c[1] for c in CASES])
def test_forward(gpu, c):
    print(f"probs {c}", flush=True)
    cfg, wl = layer(c, gpu)
    T, E, K = cfg.T, cfg.E, cfg.K
    bias = wl.route_bias.to(gpu)
    Lg = wl.layer.to(gpu)
    fwd = ops.MoeForward(Lg, T, configs.route_params(cfg, bias), c[0])
    y = torch.full((T, cfg.H), float("nan"), device=gpu)
    oe = torch.full((T, K), -7, dtype=torch.int32, device=gpu)
    ow = torch.full((T, K), float("nan"), device=gpu)
    fwd(wl.x.to(gpu), y, oe, ow)
    torch.cuda.synchronize()
    oe, ow = oe.cpu(), ow.cpu()
    logits = O.router_logits(wl.layer.router, wl.x)
    kw = dict(bias=wl.route_bias, n_group=max(1, cfg.n_group), topk_group=cfg.topk_group, scaling=cfg.scaling,
              normalize=wl.layer.norm_topk)
    # the device's logits may be 1e-4 from the oracle's (the router's own
    # tolerance): tokens whose choice that could move are left out
    we, ww = want(logits, K, **kw)
    noise = torch.rand(3, T, E, generator=torch.Generator().manual_seed(1)) * 2e-4 - 1e-4
    sure = torch.stack([(want(logits + n, K, **kw)[0] == we).all(1) for n in noise]).all(0)
    assert sure.float().mean() > 0.5
    assert torch.equal(oe[sure], we[sure])
    assert ((ow.double() - ww)[sure].abs() <= 1e-3 * ww[sure].abs()).all()
    gate = None
    assert_close(y.cpu(), O.moe_forward(wl.layer.struct(), oe, ow, gate, wl.x), what=cfg.name)


def test_shards_sum_to_the_layer(gpu):
    c = (0, "shards", 9, 32, 4, 512, 256, "mxfp4", 1, 1, False)
    cfg, wl = layer(c, gpu)
    bias, x = wl.route_bias.to(gpu), wl.x.to(gpu)
    rp = configs.route_params(cfg, bias)
    whole = torch.empty(cfg.T, cfg.H, device=gpu)
    ops.MoeForward(wl.layer.to(gpu), cfg.T, rp, 3)(x, whole)
    total = torch.zeros_like(whole)
    for b in (0, 16):
        part = torch.empty_like(whole)
        ops.MoeForward(wl.layer.shard(b, 16).to(gpu), cfg.T, rp, 1).shard(x, part, b, 16)
        total += part
    torch.cuda.synchronize()
    assert_close(total.cpu(), whole.cpu(), what="shards")


def test_refusals(gpu):
    c = (1, "refuse", 2, 32, 4, 512, 256, "int4", 1, 1, False)
    cfg, wl = layer(c, gpu)
    x, y = wl.x.to(gpu), torch.empty(cfg.T, cfg.H, device=gpu)
    rp = configs.route_params(cfg, wl.route_bias.to(gpu))
    fwd = ops.MoeForward(wl.layer.to(gpu), cfg.T, rp, 1)
    with pytest.raises(_abi.GrimoireError):
        fwd.stage(fwd.STAGE_ROUTER, x, y)
    for n_group, kept in ((-1, 1), (5, 1), (32, 3), (4, 0), (4, 5)):
        bad = _abi.RouteParams(mode=_abi.ROUTE_PROBS, n_group=n_group, topk_group=kept, scaling=1.0)
        with pytest.raises(_abi.GrimoireError):
            ops.MoeForward(fwd.L, cfg.T, bad, 0)(x, y)
    bad = _abi.RouteParams(mode=4, scaling=1.0)
    with pytest.raises(_abi.GrimoireError):
        ops.MoeForward(fwd.L, cfg.T, bad, 0)(x, y)


@pytest.mark.parametrize("c", CASES, ids=[c[1] for c in CASES])
def test_too_few_experts_left(gpu, c):
    """The bias takes experts out of service until fewer than K are left: the
    free slots hold expert -1 and weight 0, and add nothing in any regime."""
    print(f"probs, few left {c}", flush=True)
    cfg, wl = layer((*c[:8], 1, 1, c[10]), gpu)
    T, E, K = cfg.T, cfg.E, cfg.K
    bias = torch.full((E,), float("-inf"))
    left = torch.randperm(E, generator=torch.Generator().manual_seed(E))[:K - 1]
    bias[left] = 0.0
    Lg, dbias = wl.layer.to(gpu), bias.to(gpu)
    fwd = ops.MoeForward(Lg, T, configs.route_params(cfg, dbias), c[0])
    y = torch.full((T, cfg.H), float("nan"), device=gpu)
    oe = torch.full((T, K), -7, dtype=torch.int32, device=gpu)
    ow = torch.full((T, K), float("nan"), device=gpu)
    fwd(wl.x.to(gpu), y, oe, ow)
    torch.cuda.synchronize()
    oe, ow = oe.cpu(), ow.cpu()
    assert (oe[:, -1] == -1).all() and (ow[:, -1] == 0).all()
    assert torch.equal(oe[:, :-1].sort(1).values, left.int().sort().values.expand(T, K - 1))
    ids, w = oe.clone(), ow
    ids[:, -1] = int(left[0])                    # the oracle's stand-in, of weight 0
    assert_close(y.cpu(), O.moe_forward(wl.layer.struct(), ids, w, None, wl.x), what=cfg.name)


def test_without_a_workspace(gpu):
    """The library's own scratch serves this mode as the caller's does."""
    for regime, T in ((0, 3), (1, 2), (7, 1), (2, 40)):
        cfg, wl = layer((regime, "noalloc", T, 32, 4, 512, 256, "int8", 4, 2, False), gpu)
        bias = wl.route_bias.to(gpu)
        rp = configs.route_params(cfg, bias)
        Lg, x = wl.layer.to(gpu), wl.x.to(gpu)
        y0, y1 = torch.empty(T, cfg.H, device=gpu), torch.full((T, cfg.H), float("nan"), device=gpu)
        fwd = ops.MoeForward(Lg, T, rp, regime)
        fwd(x, y0)
        r = _abi.lib().grimoire_moe_forward_noalloc(None, C.byref(fwd.struct), C.byref(rp), None, x.data_ptr(),
                                                    y1.data_ptr(), T, None, None, regime)
        assert r == 0, _abi.lib().grimoire_moe_last_error().decode()
        torch.cuda.synchronize()
        assert torch.equal(y0, y1)
