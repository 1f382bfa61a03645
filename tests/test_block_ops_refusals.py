"""Host-side refusals of the block operators' entry points: nothing here
reaches a kernel (the pointers are not memory)."""
import ctypes as C

import pytest
import torch

from grimoire_amd import _abi, ops, weights

OK, SHAPE, ARG = 0, _abi.ERR_SHAPE, _abi.ERR_ARG
A = 1 << 12   # an aligned address nothing is read from


def scores(n_experts=64, top_k=8, row_stride=None, logits=A, ids=A, w=A, tokens=2, null=False, **kw):
    p = _abi.ScoreParams(score=0, n_group=1, topk_group=1, group_score=0, normalize=1, scaling=1.0)
    for k, v in kw.items():
        setattr(p, k, v)
    return _abi.lib().grimoire_moe_router_scores(None, None if null else C.byref(p), logits, 0,
                                                 n_experts if row_stride is None else row_stride, tokens, n_experts,
                                                 top_k, ids, w)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), OK), (dict(tokens=0, logits=None), OK), (dict(tokens=-1), OK),
    (dict(logits=None), ARG), (dict(ids=None), ARG), (dict(w=None), ARG), (dict(null=True), ARG), (dict(score=2), ARG),
    (dict(n_experts=0, row_stride=1), SHAPE), (dict(n_experts=513), SHAPE), (dict(top_k=0), SHAPE),
    (dict(top_k=17), SHAPE), (dict(n_experts=4, top_k=5), SHAPE), (dict(row_stride=63), SHAPE),
    (dict(n_group=-1), SHAPE), (dict(n_group=7, topk_group=1), SHAPE), (dict(n_group=8, topk_group=0), SHAPE),
    (dict(n_group=8, topk_group=9), SHAPE), (dict(n_group=16, topk_group=1), SHAPE),
    (dict(n_group=8, topk_group=1, group_score=2), ARG),
    (dict(n_experts=130, n_group=65, topk_group=65, top_k=1), SHAPE)])
def test_scores(kw, status):
    assert scores(**kw) == status


def norm(h=A, x=A, h_out=A, out=A, out_bf=None, tokens=2, hidden=64, x_stride=None, gate=None, gate_bf16=0, x_bf16=0,
         **kw):
    p = _abi.BlockNormParams(post_weight=A, pre_weight=A, weight_offset=1.0, eps=1e-6, residual_scale=1.0,
                             block_scale=1.0, gate_kind=0, gate_sigmoid=0)
    for k, v in kw.items():
        setattr(p, k, v)
    return _abi.lib().grimoire_block_norm(None, C.byref(p), gate, gate_bf16, h, x, x_bf16,
                                          hidden if x_stride is None else x_stride, h_out, out, out_bf, tokens, hidden)


def moe_norm(routed=A, rows=9, inverse=A, rw=A, shared=None, top_k=4, hidden=64, tokens=2):
    p = _abi.BlockNormParams(post_weight=A, pre_weight=A, weight_offset=1.0, eps=1e-6, residual_scale=1.0,
                             block_scale=1.0, gate_kind=0, gate_sigmoid=0)
    return _abi.lib().grimoire_moe_block_norm(None, C.byref(p), None, 0, A, routed, rows, inverse, rw, shared, A, A,
                                              None, tokens, top_k, hidden)


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), OK), (dict(tokens=0, h=None), OK), (dict(h=None), ARG), (dict(x=None), ARG),
    (dict(hidden=66), SHAPE), (dict(hidden=0), SHAPE), (dict(hidden=32772), SHAPE), (dict(x_stride=60), SHAPE),
    (dict(x_stride=66), SHAPE), (dict(h_out=None, out=None), ARG), (dict(pre_weight=None), ARG),
    (dict(gate_kind=4, gate=A), ARG), (dict(gate_kind=1), ARG), (dict(gate=A), ARG), (dict(h=A + 4), ARG),
    (dict(x=A + 8), ARG), (dict(x=A + 4, x_bf16=1), ARG), (dict(out=A + 8), ARG), (dict(out_bf=A + 4), ARG),
    (dict(h_out=A + 4), ARG), (dict(post_weight=A + 4), ARG), (dict(gate_kind=1, gate=A + 8), ARG),
    (dict(gate_kind=3, gate=A + 4, gate_bf16=1), ARG), (dict(gate_kind=2, gate=A + 2), ARG)])
def test_block_norm(kw, status):
    assert norm(**kw) == status


@pytest.mark.parametrize("kw,status", [
    (dict(tokens=0), OK), (dict(routed=None), ARG), (dict(inverse=None), ARG), (dict(rw=None), ARG),
    (dict(top_k=0), SHAPE), (dict(top_k=17), SHAPE), (dict(rows=-1), SHAPE), (dict(hidden=2), SHAPE),
    (dict(routed=A + 4), ARG), (dict(shared=A + 4), ARG)])
def test_moe_block_norm(kw, status):
    assert moe_norm(**kw) == status


def lora(glu=False, rows=3, slot=A, x=A, x_bf16=0, x_stride=64, base=A, base_bf16=0, base_stride=32, y=2 * A, y_bf16=0,
         y_stride=None, ws=A, ws_bytes=1 << 20, **kw):
    L = _abi.Lora(K=64, N=32, slots=4, max_rank=16, a=A, b=A, rank=A, scale=A)
    for k, v in kw.items():
        setattr(L, k, v)
    fn = _abi.lib().grimoire_lora_swiglu if glu else _abi.lib().grimoire_lora_add
    return fn(None, C.byref(L), slot, x, x_bf16, x_stride, base, base_bf16, base_stride, y, y_bf16,
              (16 if glu else 32) if y_stride is None else y_stride, rows, ws, ws_bytes)


@pytest.mark.parametrize("kw,status", [
    (dict(rows=0), OK), (dict(rows=0, x=None), OK), (dict(slot=None), ARG), (dict(x=None), ARG), (dict(base=None), ARG),
    (dict(y=None), ARG), (dict(a=None), ARG), (dict(b=None), ARG), (dict(rank=None), ARG), (dict(scale=None), ARG),
    (dict(K=0), SHAPE), (dict(K=60), SHAPE), (dict(N=30), SHAPE), (dict(N=0), SHAPE), (dict(slots=0), SHAPE),
    (dict(max_rank=0), SHAPE), (dict(max_rank=24), SHAPE), (dict(max_rank=272), SHAPE), (dict(x_stride=56), SHAPE),
    (dict(x_stride=68), SHAPE), (dict(base_stride=28), SHAPE), (dict(base_stride=34), SHAPE),
    (dict(y_stride=28), SHAPE), (dict(y_stride=33), SHAPE), (dict(x=A + 8), ARG), (dict(base=A + 8), ARG),
    (dict(base=A + 4, base_bf16=1), ARG), (dict(y=A + 8), ARG), (dict(a=A + 8), ARG), (dict(b=A + 2), ARG),
    (dict(y=A, y_bf16=1), ARG), (dict(y=A, y_stride=36), ARG), (dict(glu=True, y=A), ARG),
    (dict(glu=True, N=36, base_stride=36), SHAPE), (dict(glu=True, y_stride=12), SHAPE),
    (dict(x_stride=(1 << 24) + 8), SHAPE), (dict(base_stride=(1 << 24) + 4), SHAPE),
    (dict(y_stride=(1 << 24) + 4), SHAPE), (dict(K=1 << 22, x_stride=1 << 22, max_rank=256), SHAPE),
    (dict(N=1 << 22, base_stride=1 << 22, y_stride=1 << 22, max_rank=256), SHAPE),
    (dict(ws=None), _abi.ERR_WORKSPACE), (dict(ws_bytes=3 * 16 * 4 - 1), _abi.ERR_WORKSPACE), (dict(ws=A + 4), ARG)])
def test_lora(kw, status):
    assert lora(**kw) == status


def test_lora_workspace_grows_with_rows():
    """One size holds every shorter batch, those that split K among them."""
    for K in (8, 64, 2048, 7168):
        L = _abi.Lora(K=K, N=32, slots=4, max_rank=32)
        n = [_abi.lib().grimoire_lora_workspace_bytes(C.byref(L), r) for r in (1, 16, 511, 512, 513, 700, 5000, 9000)]
        assert n == sorted(n) and n[0] >= 32 * 4
    assert _abi.lib().grimoire_lora_workspace_bytes(None, 5) == 0
    assert _abi.lib().grimoire_lora_workspace_bytes(C.byref(L), 0) == 0


def test_lora_adapters_shapes():
    ad = weights.LoraAdapters.empty(3, 16, 64, 32, device="cpu")
    ad.load(1, torch.ones(5, 64), torch.ones(32, 5), 0.5)
    assert ad.rank.tolist() == [0, 5, 0] and float(ad.a.sum()) == 5 * 64 and float(ad.b[1, :, 5:].sum()) == 0
    for bad in (dict(slot=3), dict(slot=-1), dict(a=torch.ones(17, 64), b=torch.ones(32, 17)),
                dict(a=torch.ones(5, 63)), dict(b=torch.ones(32, 6))):
        kw = dict(slot=0, a=torch.ones(5, 64), b=torch.ones(32, 5), scale=1.0)
        kw.update(bad)
        with pytest.raises(_abi.GrimoireError):
            ad.load(**kw)
    with pytest.raises(_abi.GrimoireError):
        weights.LoraAdapters(ad.a, ad.b[:, :, :8], ad.rank, ad.scale)
    with pytest.raises(_abi.GrimoireError):
        weights.LoraAdapters(ad.a.float(), ad.b, ad.rank, ad.scale)
    with pytest.raises(_abi.GrimoireError):
        ops.Lora(ad, 4)


def test_cpu_tensors_and_bad_names():
    with pytest.raises(_abi.GrimoireError):
        ops.RouteScores()(torch.zeros(2, 8), torch.zeros(2, 2, dtype=torch.int32), torch.zeros(2, 2))
    with pytest.raises(_abi.GrimoireError):
        ops.RouteScores(score="relu")
    with pytest.raises(_abi.GrimoireError):
        ops.RouteScores(bias=torch.zeros(8))
    with pytest.raises(_abi.GrimoireError):
        ops.BlockNorm(None)(torch.zeros(2, 8), torch.zeros(2, 8), torch.zeros(2, 8))
    with pytest.raises(_abi.GrimoireError):
        ops.BlockNorm(None, gate="head")


M = 1 << 20   # arguments that lie apart


@pytest.mark.parametrize("kw", [
    dict(ids=M, w=2 * M, logits=M), dict(ids=M, w=2 * M, logits=2 * M + 60), dict(ids=M, w=M + 60, logits=4 * M),
    dict(ids=M, w=2 * M, logits=M - 256)])
def test_scores_overlap(kw):
    assert scores(**kw) == ARG


@pytest.mark.parametrize("kw", [
    dict(h_out=M + 16), dict(out=M + 256), dict(out=2 * M - 16), dict(out_bf=2 * M), dict(out=3 * M),
    dict(out_bf=3 * M + 256), dict(x=3 * M + 256, x_stride=128), dict(x=3 * M + 256, x_stride=128, x_bf16=1),
    dict(x=3 * M, x_stride=128), dict(gate_kind=3, gate=3 * M, gate_bf16=1), dict(gate_kind=2, gate=3 * M + 16),
    dict(gate_kind=1, gate=4 * M + 256)])
def test_block_norm_overlap(kw):
    args = dict(h=M, x=2 * M, h_out=3 * M, out=4 * M, out_bf=None)
    args.update(kw)
    assert norm(**args) == ARG


@pytest.mark.parametrize("kw", [dict(routed=4 * M + 496), dict(inverse=4 * M + 508), dict(rw=4 * M), dict(rw=5 * M + 8),
                                dict(shared=4 * M + 256), dict(h=5 * M - 256)])
def test_moe_block_norm_overlap(kw):
    p = _abi.BlockNormParams(pre_weight=A, eps=1e-6)
    a = dict(h=M, routed=2 * M, inverse=3 * M, rw=3 * M + 64, shared=None)
    a.update(kw)
    assert _abi.lib().grimoire_moe_block_norm(None, C.byref(p), None, 0, a["h"], a["routed"], 9, a["inverse"], a["rw"],
                                              a["shared"], 4 * M, None, 5 * M, 2, 4, 64) == ARG


@pytest.mark.parametrize("kw", [
    dict(y=M), dict(y=M + 256), dict(y=M - 64), dict(y=2 * M + 64), dict(y=2 * M, base_stride=64, y_stride=36),
    dict(glu=True, y=2 * M + 64), dict(y=2 * M + 112, base_stride=64, y_stride=64),
    dict(y=M + 128, x_stride=96, y_stride=96), dict(y=M + 240, x_stride=96, y_stride=96),
    dict(y=M, y_bf16=1, x_bf16=1), dict(y=2 * M, y_bf16=1)])
def test_lora_overlap(kw):
    args = dict(x=M, base=2 * M, y=3 * M)
    args.update(kw)
    assert lora(**args) == ARG


def test_lora_adapters_load_bits():
    """bf16 bits held as int16 are loaded as what they stand for."""
    ad = weights.LoraAdapters.empty(2, 16, 64, 32, device="cpu")
    a, b = torch.randn(3, 64).bfloat16(), torch.randn(32, 3).bfloat16()
    ad.load(1, a.view(torch.int16), b.view(torch.int16), 1.0)
    assert torch.equal(ad.a[1, :3], a) and torch.equal(ad.b[1, :, :3], b)
    bits = weights.LoraAdapters(ad.a.view(torch.int16), ad.b.view(torch.int16), ad.rank, ad.scale)
    bits.load(0, a.float(), b, 1.0)
    assert torch.equal(ad.a[0, :3], a) and torch.equal(ad.b[0, :, :3], b)
    for bad in (torch.ones(3, 64, dtype=torch.int32), torch.ones(64), torch.ones(3, 64, dtype=torch.int8)):
        with pytest.raises(_abi.GrimoireError):
            ad.load(0, bad, b, 1.0)


def test_what_an_operator_was_made_for_stays():
    """The structs hold addresses: the tensors behind them are not swapped."""
    ad = weights.LoraAdapters.empty(2, 16, 64, 32, device="cpu")
    assert (ad.slots, ad.max_rank, ad.K, ad.N) == (2, 16, 64, 32)
    for obj, names in ((ad, ("a", "b", "rank", "scale", "K", "N", "slots", "max_rank")), (ops.RouteScores(), ("bias",)),
                       (ops.BlockNorm(None), ("pre_weight", "post_weight", "gate"))):
        for n in names:
            with pytest.raises(AttributeError):
                setattr(obj, n, getattr(obj, n))
    with pytest.raises(_abi.GrimoireError):
        weights.LoraAdapters(ad.a[0], ad.b, ad.rank, ad.scale)
    with pytest.raises(_abi.GrimoireError):
        weights.LoraAdapters(ad.a, ad.b[0], ad.rank, ad.scale)
