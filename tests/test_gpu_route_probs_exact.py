"""GRIM_ROUTE_PROBS in the whole layer on logits that every order of their
sum forms exactly: activations and router weights are small integers (the
latter times 2^-5), so all partial sums are integers below 2^24 in that unit
and nothing rounds.  The forward's routes then are those of the definition in
64 bits for every token, ties and all, and its weights are off by their one
rounding to fp32."""
import pytest
import torch

from grimoire_amd import configs, ops
from tests.test_gpu_route_probs import CASES, layer
from tests.test_gpu_scores import want

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("c", CASES, ids=[c[1] for c in CASES])
def test_routes(gpu, c, bias):
    print(f"probs, exact logits {c} bias={bias}", flush=True)
    cfg, wl = layer(c, gpu)
    T, E, K, H = cfg.T, cfg.E, cfg.K, cfg.H
    g = torch.Generator().manual_seed(T + K)
    x = torch.randint(-2, 3, (T, H), generator=g).float()
    wl.layer.router = torch.randint(-4, 5, (E, H), generator=g).float() / 32
    b = wl.route_bias if bias else None
    db = b.to(gpu) if bias else None                 # its address is in the route's parameters
    fwd = ops.MoeForward(wl.layer.to(gpu), T, configs.route_params(cfg, db), c[0])
    y = torch.empty(T, H, device=gpu)
    oe = torch.full((T, K), -7, dtype=torch.int32, device=gpu)
    ow = torch.full((T, K), float("nan"), device=gpu)
    fwd(x.to(gpu), y, oe, ow)
    torch.cuda.synchronize()
    logits = (x.double() @ wl.layer.router.double().T).float()
    we, ww = want(logits, K, bias=b, n_group=max(1, cfg.n_group), topk_group=cfg.topk_group, scaling=cfg.scaling,
                  normalize=wl.layer.norm_topk)
    assert torch.equal(oe.cpu(), we)
    # one rounding to fp32 of a value off by a few steps of fp64
    assert ((ow.cpu().double() - ww).abs() <= ww.abs() * (2.0 ** -24 + 1e-13) + 2.0 ** -149).all()
