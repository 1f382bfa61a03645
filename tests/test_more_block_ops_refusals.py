"""What the 4-bit projections, the sorted rows, their gradients and the router
scores' gradient refuse, on the host, before anything is launched.  CPU only:
addresses are made up and no call here reaches a kernel."""
import ctypes as C

import pytest

from grimoire_amd import _abi

A = 1 << 20           # addresses 16 MiB apart
P = [A + (i << 24) for i in range(16)]
SHAPE, ARG, FORMAT, WS = _abi.ERR_SHAPE, _abi.ERR_ARG, _abi.ERR_FORMAT, _abi.ERR_WORKSPACE


def weight(**kw):
    d = dict(fmt=_abi.FMT_INT4, N=64, K=256, row_scales=2, row_bytes=128, payload=P[0], scales=P[1], zeros=P[2])
    d.update(kw)
    return _abi.QuantWeight(**d)


def proj(w=None, **kw):
    d = dict(x=P[3], x16=0, xs=256, base=None, b16=0, bs=0, y=P[4], y16=0, ys=64, rows=4, ws=P[6], n=1 << 24)
    d.update(kw)
    w = weight() if w is None else w
    return _abi.lib().grimoire_proj4(None, C.byref(w), d["x"], d["x16"], d["xs"], d["base"], d["b16"], d["bs"], d["y"],
                                     d["y16"], d["ys"], d["rows"], d["ws"], d["n"])


def glu(w=None, **kw):
    d = dict(x=P[3], xs=256, h=P[4], hs=32, rows=4, ws=P[6], n=1 << 24)
    d.update(kw)
    w = weight() if w is None else w
    return _abi.lib().grimoire_proj4_swiglu(None, C.byref(w), d["x"], 0, d["xs"], d["h"], 0, d["hs"], d["rows"], d["ws"],
                                            d["n"])


@pytest.mark.parametrize("w,status", [
    (dict(fmt=_abi.FMT_INT8), FORMAT), (dict(fmt=_abi.FMT_BF16), FORMAT), (dict(fmt=99), FORMAT),
    (dict(payload=None), ARG), (dict(scales=None), ARG), (dict(payload=P[0] + 8), ARG), (dict(scales=P[1] + 1), ARG),
    (dict(N=0), SHAPE), (dict(N=-1), SHAPE), (dict(K=0), SHAPE), (dict(K=240, row_bytes=128, row_scales=2), SHAPE),
    (dict(row_bytes=112), SHAPE), (dict(row_bytes=136), SHAPE), (dict(row_scales=3), SHAPE), (dict(row_scales=16), SHAPE),
    (dict(fmt=_abi.FMT_MXFP4, row_scales=7), SHAPE)])
def test_weights(w, status):
    assert proj(weight(**w)) == status
    assert glu(weight(**w)) == status


@pytest.mark.parametrize("kw,status", [
    (dict(x=None), ARG), (dict(y=None), ARG), (dict(xs=248), SHAPE), (dict(xs=260), SHAPE), (dict(xs=1 << 29), SHAPE),
    (dict(ys=63), SHAPE), (dict(ys=-64), SHAPE), (dict(ys=1 << 29), SHAPE), (dict(base=P[5], bs=60), SHAPE),
    (dict(x=P[3] + 8), ARG), (dict(y=P[4] + 2), ARG), (dict(base=P[5] + 1, bs=64), ARG),
    (dict(y=P[3]), ARG), (dict(y=P[0]), ARG), (dict(y=P[1]), ARG), (dict(y=P[2]), ARG),
    (dict(base=P[4], bs=128), ARG), (dict(base=P[4], bs=64, b16=1), ARG), (dict(base=P[4] + 4, bs=64), ARG),
    (dict(x=P[4] + 512, y=P[4]), ARG), (dict(ws=None), WS), (dict(n=1024), WS), (dict(ws=P[6] + 8), ARG),
    (dict(ws=P[3]), ARG), (dict(ws=P[4]), ARG), (dict(ws=P[0]), ARG), (dict(ws=P[2]), ARG), (dict(base=P[6], bs=64), ARG)])
def test_projection_arguments(kw, status):
    assert proj(**kw) == status


@pytest.mark.parametrize("w", [dict(K=512, row_bytes=256, row_scales=1), dict(row_scales=0), dict(row_scales=-1),
                               dict(K=1024, row_bytes=512, row_scales=2)])
def test_groups_that_there_are_not(w):
    assert proj(weight(**w), xs=1024) == SHAPE
    assert glu(weight(**w), xs=1024) == SHAPE


def test_projection_no_rows_and_odd_glu():
    assert proj(rows=0, x=None, y=None) == 0
    assert glu(weight(N=63)) == SHAPE
    assert glu(hs=31) == SHAPE
    assert glu(h=P[3]) == ARG
    assert _abi.lib().grimoire_proj4(None, None, P[3], 0, 256, None, 0, 0, P[4], 0, 64, 4, P[6], 1 << 24) == ARG
    assert _abi.lib().grimoire_proj4_workspace_bytes(None, 4) == 0
    w = weight()
    n = [_abi.lib().grimoire_proj4_workspace_bytes(C.byref(w), r) for r in (-1, 0, 1, 4, 64, 65, 1 << 20)]
    assert n[0] == n[1] == 0 and 0 < n[2] < n[3] < n[4] == n[5] == n[6]
    assert proj(n=n[3], y=None) == ARG and proj(n=n[3] - 1) == WS


def test_more_rows_than_a_launch_takes():
    assert proj(rows=(1 << 18) + 1) == SHAPE and glu(rows=(1 << 18) + 1) == SHAPE
    assert proj(rows=1 << 18, n=1 << 62, ws=None) == WS


def sort(**kw):
    d = dict(ids=P[0], x=P[1], x16=0, xs=64, w=P[2], rows=P[3], r16=1, c=P[4], o=P[5], inv=P[6], pt=None, T=16, H=64, E=8,
             K=4, ws=P[7], n=1 << 20)
    d.update(kw)
    return _abi.lib().grimoire_moe_sort_rows(None, d["ids"], d["x"], d["x16"], d["xs"], d["w"], d["rows"], d["r16"], d["c"],
                                             d["o"], d["inv"], d["pt"], d["T"], d["H"], d["E"], d["K"], d["ws"], d["n"])


@pytest.mark.parametrize("kw,status", [
    (dict(ids=None), ARG), (dict(x=None), ARG), (dict(rows=None), ARG), (dict(c=None), ARG), (dict(o=None), ARG),
    (dict(inv=None), ARG), (dict(ws=None), WS), (dict(n=8), WS), (dict(E=0), SHAPE), (dict(E=20000), SHAPE),
    (dict(K=0), SHAPE), (dict(K=17), SHAPE), (dict(H=62), SHAPE), (dict(H=0), SHAPE), (dict(xs=60), SHAPE),
    (dict(xs=66), SHAPE), (dict(T=1 << 30, K=16), SHAPE), (dict(x=P[1] + 8), ARG), (dict(rows=P[3] + 4), ARG),
    (dict(rows=P[1]), ARG), (dict(rows=P[0]), ARG), (dict(rows=P[2]), ARG), (dict(c=P[5]), ARG), (dict(inv=P[0]), ARG),
    (dict(pt=P[6]), ARG), (dict(pt=P[3]), ARG), (dict(ws=P[1]), ARG), (dict(ws=P[3]), ARG), (dict(ws=P[7] + 2), ARG),
    (dict(T=0, c=P[5]), ARG)])
def test_sort_arguments(kw, status):
    assert sort(**kw) == status


def sort_grad(**kw):
    d = dict(dr=P[0], r16=1, n=64, inv=P[1], w=P[2], x=P[3], x16=0, xs=64, dx=P[4], d16=0, ds=64, dw=P[5], T=16, K=4, H=64)
    d.update(kw)
    return _abi.lib().grimoire_moe_sort_rows_grad(None, d["dr"], d["r16"], d["n"], d["inv"], d["w"], d["x"], d["x16"],
                                                  d["xs"], d["dx"], d["d16"], d["ds"], d["dw"], d["T"], d["K"], d["H"])


@pytest.mark.parametrize("kw,status", [
    (dict(dr=None), ARG), (dict(inv=None), ARG), (dict(dx=None), ARG), (dict(w=None), ARG), (dict(x=None), ARG),
    (dict(dw=None), ARG), (dict(w=None, x=None), ARG), (dict(n=-1), SHAPE), (dict(n=1 << 31), SHAPE), (dict(K=17), SHAPE),
    (dict(K=0), SHAPE), (dict(H=66), SHAPE), (dict(ds=60), SHAPE), (dict(ds=66), SHAPE), (dict(xs=62), SHAPE),
    (dict(dr=P[0] + 4), ARG), (dict(dx=P[4] + 8), ARG), (dict(x=P[3] + 8), ARG), (dict(dx=P[0]), ARG), (dict(dx=P[3]), ARG),
    (dict(dw=P[2]), ARG), (dict(dw=P[1]), ARG), (dict(dw=P[4]), ARG)])
def test_sort_grad_arguments(kw, status):
    assert sort_grad(**kw) == status


def combine(**kw):
    d = dict(dy=P[0], y16=0, ys=64, rows=P[1], r16=1, n=64, inv=P[2], w=P[3], dr=P[4], dw=P[5], sh=P[6], s16=0, g=P[7],
             ds=P[8], dg=P[9], T=16, K=4, H=64)
    d.update(kw)
    return _abi.lib().grimoire_moe_combine_grad(None, d["dy"], d["y16"], d["ys"], d["rows"], d["r16"], d["n"], d["inv"],
                                                d["w"], d["dr"], d["dw"], d["sh"], d["s16"], d["g"], d["ds"], d["dg"],
                                                d["T"], d["K"], d["H"])


@pytest.mark.parametrize("kw,status", [
    (dict(dy=None), ARG), (dict(rows=None), ARG), (dict(dr=None), ARG), (dict(inv=None), ARG), (dict(w=None), ARG),
    (dict(dw=None), ARG), (dict(ds=None), ARG), (dict(sh=None), ARG), (dict(dg=None), ARG), (dict(g=None), ARG),
    (dict(sh=None, ds=None), ARG), (dict(n=-1), SHAPE), (dict(K=17), SHAPE), (dict(H=2), SHAPE), (dict(ys=62), SHAPE),
    (dict(dy=P[0] + 8), ARG), (dict(rows=P[1] + 4), ARG), (dict(dr=P[4] + 4), ARG), (dict(ds=P[8] + 8), ARG),
    (dict(dr=P[1]), ARG), (dict(dr=P[0]), ARG), (dict(ds=P[6]), ARG), (dict(dw=P[3]), ARG), (dict(dg=P[7]), ARG),
    (dict(dg=P[5]), ARG)])
def test_combine_grad_arguments(kw, status):
    assert combine(**kw) == status


def scores(**kw):
    d = dict(l=P[0], b16=0, s=64, e=P[1], dw=P[2], d=P[3], ds=64, T=16, E=64, K=4, score=0)
    d.update(kw)
    p = _abi.ScoreParams(d["score"], 1, 1, 0, 1, 1.0, None)
    return _abi.lib().grimoire_moe_router_scores_grad(None, C.byref(p), d["l"], d["b16"], d["s"], d["e"], d["dw"], d["d"],
                                                      d["ds"], d["T"], d["E"], d["K"])


@pytest.mark.parametrize("kw,status", [
    (dict(l=None), ARG), (dict(e=None), ARG), (dict(dw=None), ARG), (dict(d=None), ARG), (dict(score=2), ARG),
    (dict(E=0), SHAPE), (dict(E=513, s=520, ds=520), SHAPE), (dict(K=0), SHAPE), (dict(K=17), SHAPE),
    (dict(E=3, K=4), SHAPE), (dict(s=63), SHAPE), (dict(ds=63), SHAPE), (dict(s=1 << 29), SHAPE), (dict(d=P[0] + 4), ARG),
    (dict(d=P[0], ds=72), ARG), (dict(d=P[1]), ARG), (dict(d=P[2]), ARG)])
def test_scores_grad_arguments(kw, status):
    assert scores(**kw) == status


def test_no_tokens():
    assert scores(T=0, l=None) == 0 and combine(T=0, dy=None) == 0 and sort_grad(T=0, dx=None) == 0


def test_more_tokens_than_a_launch_takes():
    n = (1 << 23) + 1
    assert sort(T=n, K=1, n=1 << 62) == SHAPE and sort_grad(T=n, K=1) == SHAPE and combine(T=n, K=1) == SHAPE
    assert scores(T=(1 << 24) + 1) == SHAPE
