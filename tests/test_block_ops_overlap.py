"""Outputs of the block operators that share memory with an argument which
other rows' work reads are refused: one at the same address, with the same
width, is no argument that an output may take the place of.  Host checks
only: what is not refused would reach a launch."""
import ctypes as C
import os

import pytest

from grimoire_amd import _abi

pytestmark = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="made-up device addresses: no GPU may see them")

ARG = _abi.ERR_ARG
M = 1 << 20   # arguments that lie apart


def launched(status):
    """Past every check: the launch found no GPU."""
    return status > 0


def norm(T=3, H=64, gate=None, gate_kind=0, gate_bf16=0, moe=False, K=2, rows=7, **kw):
    a = dict(h=M, x=2 * M, h_out=3 * M, out=4 * M, out_bf=5 * M, routed=6 * M, inverse=7 * M, rw=8 * M, shared=9 * M,
             post=10 * M, pre=11 * M, x_bf16=0)
    a.update(kw)
    p = _abi.BlockNormParams(post_weight=a["post"], pre_weight=a["pre"], weight_offset=1.0, eps=1e-6,
                             residual_scale=1.0, block_scale=1.0, gate_kind=gate_kind)
    if moe:
        return _abi.lib().grimoire_moe_block_norm(None, C.byref(p), gate, gate_bf16, a["h"], a["routed"], rows,
                                                  a["inverse"], a["rw"], a["shared"], a["h_out"], a["out"],
                                                  a["out_bf"], T, K, H)
    return _abi.lib().grimoire_block_norm(None, C.byref(p), gate, gate_bf16, a["h"], a["x"], a["x_bf16"], H,
                                          a["h_out"], a["out"], a["out_bf"], T, H)


CHANNEL, ROW, FULL = _abi.GATE_CHANNEL, _abi.GATE_ROW, _abi.GATE_FULL


@pytest.mark.parametrize("kw", [
    dict(gate=3 * M, gate_kind=CHANNEL), dict(gate=4 * M, gate_kind=CHANNEL),
    dict(gate=5 * M, gate_kind=CHANNEL, gate_bf16=1), dict(gate=3 * M, gate_kind=ROW, T=64),
    dict(gate=5 * M, gate_kind=ROW, gate_bf16=1, T=64), dict(gate=3 * M + 256, gate_kind=CHANNEL)])
@pytest.mark.parametrize("moe", [False, True])
def test_gate_of_many_rows(kw, moe):
    assert norm(moe=moe, **kw) == ARG


@pytest.mark.parametrize("kw", [
    dict(T=16, K=4, rw=3 * M), dict(T=16, K=4, rw=4 * M), dict(T=16, K=4, inverse=3 * M),
    dict(T=16, K=4, inverse=4 * M), dict(T=32, K=4, inverse=5 * M),          # T K = H (H / 2 beside the bf16 rows)
    dict(rows=1, routed=5 * M), dict(rows=2, routed=3 * M), dict(rows=2, routed=4 * M), dict(T=1, rows=2, routed=3 * M),
    dict(T=1, K=4, H=4, rw=3 * M)])
def test_routes_and_expert_rows(kw):
    assert norm(moe=True, **kw) == ARG


@pytest.mark.parametrize("kw", [
    dict(h_out=M), dict(out=M), dict(x=4 * M), dict(x=5 * M, x_bf16=1), dict(gate=4 * M, gate_kind=FULL),
    dict(gate=5 * M, gate_kind=FULL, gate_bf16=1), dict(moe=True, shared=3 * M), dict(moe=True, h_out=M, shared=4 * M),
    dict(T=1, gate=3 * M, gate_kind=CHANNEL), dict(moe=True, T=1, rows=1, routed=5 * M),
    dict(gate=3 * M + 768, gate_kind=CHANNEL), dict()])
def test_in_place_stays(kw):
    """h, x, shared and a full gate of an output's own layout; what one row alone
    reads."""
    assert launched(norm(**kw))


@pytest.mark.parametrize("kw", [dict(post=3 * M), dict(post=4 * M + 704), dict(pre=5 * M), dict(pre=3 * M - 64),
                                dict(pre=4 * M + 8), dict(T=1, pre=5 * M), dict(T=1, post=5 * M)])
@pytest.mark.parametrize("moe", [False, True])
def test_norm_weights(kw, moe):
    assert norm(moe=moe, **kw) == ARG
    assert launched(norm(moe=moe, post=None)) and launched(norm(moe=moe, pre=None, out=None, out_bf=None))
    assert launched(norm(moe=moe, post=11 * M, pre=3 * M + 768))


def scores(bias=3 * M, E=64, K=8, T=2, logits=M, ids=2 * M, w=2 * M + 4096):
    p = _abi.ScoreParams(score=0, n_group=1, topk_group=1, group_score=0, normalize=1, scaling=1.0, bias=bias)
    return _abi.lib().grimoire_moe_router_scores(None, C.byref(p), logits, 0, E, T, E, K, ids, w)


@pytest.mark.parametrize("kw", [dict(bias=2 * M), dict(bias=2 * M - 252), dict(bias=2 * M + 60), dict(bias=2 * M + 4096)])
def test_scores_bias(kw):
    assert scores(**kw) == ARG
    assert launched(scores()) and launched(scores(bias=None)) and launched(scores(bias=2 * M + 64))


LORA = dict(x=M, base=2 * M, y=3 * M, slot=4 * M, a=5 * M, b=6 * M, rank=7 * M, scale=8 * M, ws=9 * M)
LORA_BYTES = dict(slot=3 * 4, a=4 * 16 * 64 * 2, b=4 * 32 * 16 * 2, rank=4 * 4, scale=4 * 4)


def lora(glu=False, rows=3, **kw):
    a = dict(LORA, **kw)
    L = _abi.Lora(K=64, N=32, slots=4, max_rank=16, a=a["a"], b=a["b"], rank=a["rank"], scale=a["scale"])
    need = _abi.lib().grimoire_lora_workspace_bytes(C.byref(L), rows)
    fn = _abi.lib().grimoire_lora_swiglu if glu else _abi.lib().grimoire_lora_add
    return fn(None, C.byref(L), a["slot"], a["x"], 0, 64, a["base"], 0, 32, a["y"], 0, 16 if glu else 32, rows,
              a["ws"], need)


@pytest.mark.parametrize("name", list(LORA_BYTES))
@pytest.mark.parametrize("glu", [False, True])
def test_adapter_output(name, glu):
    """An output over the adapters, their ranks and scales or the rows' slots."""
    y, n = LORA["y"], 3 * (16 if glu else 32) * 4
    last = LORA_BYTES[name]
    for at in (y, y + n - 16, y - last // 16 * 16 + (16 if last % 16 == 0 else 0)):
        assert lora(glu, **{name: at}) == ARG
        # in place it is an output all the same
        assert glu or lora(base=y, **{name: at}) == ARG
    for at in (y + n, y - (last + 15) // 16 * 16):
        assert launched(lora(glu, **{name: at}))
    assert launched(lora(glu)) and (glu or launched(lora(base=y)))


@pytest.mark.parametrize("name,n", [("x", 3 * 64 * 4), ("base", 3 * 32 * 4), ("y", 3 * 16 * 4), *LORA_BYTES.items()])
@pytest.mark.parametrize("glu", [False, True])
def test_adapter_workspace(name, n, glu):
    """The workspace apart from everything: z is written while x, the slots,
    the adapters and ranks are read, and read while y is written."""
    L = _abi.Lora(K=64, N=32, slots=4, max_rank=16)
    need = int(_abi.lib().grimoire_lora_workspace_bytes(C.byref(L), 3))
    at, n = LORA[name], (n + 15) // 16 * 16
    for ws in (at, at + n - 16, at - need + 16):
        assert lora(glu, ws=ws) == ARG
    if name != "y" or glu:
        for ws in (at + n, at - need):
            assert launched(lora(glu, ws=ws))
    assert glu or lora(base=LORA["y"], ws=LORA["y"]) == ARG
