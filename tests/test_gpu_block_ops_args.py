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
    for c in calls:
        with pytest.raises(_abi.GrimoireError):
            c()


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
