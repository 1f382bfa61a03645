"""Sorted rows and 4-bit projections on both sides of the sizes where they change
their way of working.  Tolerances: those of test_gpu_sort_rows.py and
test_gpu_proj4.py."""
import pytest
import torch

from grimoire_amd import ops
from test_gpu_proj4 import check, make_weight, reference, rows, run
from test_gpu_sort_rows import check_combine, check_sort, check_sort_grad, data, routes, sort

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,E,K,H", [
    (1024, 16, 8, 8), (1025, 16, 8, 8),            # 8192 routes
    (512, 2048, 16, 8), (512, 2049, 16, 8),        # 2048 experts
    (1170, 64, 7, 20), (8192, 40, 1, 4), (4096, 2048, 2, 4), (4097, 2048, 2, 4),
    (8192, 100, 8, 4), (8193, 100, 8, 4),          # 65536 routes
    (12288, 100, 8, 4), (12289, 100, 8, 4),        # 98304
    (418, 30, 8, 8), (420, 30, 8, 8), (223, 30, 16, 8), (225, 30, 16, 8), (2022, 30, 1, 8), (2023, 30, 1, 8),
    (65536, 7, 1, 4), (65537, 7, 1, 4), (9001, 2048, 16, 4)])
def test_sort_sizes(gpu, T, E, K, H):
    for n, kind in enumerate(("mixed", "one")):
        ids = routes(T, E, K, T + n, kind)
        x, w = data(T, H, K, H + n)
        check_sort(sort(gpu, ids, x, E, True), ids, x, E, True)
        check_sort(sort(gpu, ids, x, E, False, w, True), ids, x, E, False, w, True)


@pytest.mark.parametrize("K", [1, 2, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 16])
@pytest.mark.parametrize("T", [64, 65])
def test_combine_slots(gpu, T, K):
    check_combine(gpu, T, K, 260, K, shared="bf16", gate=True)
    check_combine(gpu, T, K, 1032, K, dy_bf16=True, rows_bf16=False)


@pytest.mark.parametrize("T", [1, 3, 100, 255, 256, 257, 511, 512])
@pytest.mark.parametrize("H", [4, 1028, 7168])
def test_sort_grad_columns(gpu, T, H):
    """Columns shared out (without weights), larger work-groups (with)."""
    K = 5
    inv = torch.randperm(T * K, generator=torch.Generator().manual_seed(T)).int().view(T, K)
    x, w = data(T, H, K, H)
    drows = torch.randn((T * K, H), generator=torch.Generator().manual_seed(H)).bfloat16()
    obj = ops.TokenSort(8, K, T, device=gpu)
    for weighted in (False, True):
        dx, dw = torch.full((T, H), float("nan"), device=gpu), torch.full((T, K), float("nan"), device=gpu)
        kw = dict(x=x.to(gpu), weight=w.to(gpu), dweight=dw) if weighted else {}
        obj.grad(drows.to(gpu), inv.to(gpu), dx, **kw)
        torch.cuda.synchronize()
        check_sort_grad(dx.cpu(), dw.cpu(), drows, inv, x, w if weighted else None)


@pytest.mark.parametrize("T,E,K", [(6, 16, 4), (1100, 16, 8), (9000, 16, 8)])
def test_sort_two_at_once(gpu, T, E, K):
    """Two objects on two streams, again and again the same bits."""
    i32 = dict(dtype=torch.int32, device=gpu)
    objs, args, want, streams = [], [], [], []
    for s in (1, 2):
        x, w = data(T, 64, K, s)
        objs.append(ops.TokenSort(E, K, T, device=gpu))
        args.append([routes(T, E, K, s, "all").to(gpu), x.to(gpu), torch.zeros((T * K, 64), device=gpu),
                     torch.zeros(E, **i32), torch.zeros(E, **i32), torch.zeros((T, K), **i32), w.to(gpu)])
        objs[-1](*args[-1])
        want.append([t.clone() for t in args[-1]])
        streams.append(torch.cuda.Stream())
    torch.cuda.synchronize()
    for a in args:
        for t in a[2:6]:
            t.fill_(-9)
    torch.cuda.synchronize()
    for _ in range(10):
        for o, a, st in zip(objs, args, streams):
            o(*a, stream=st)
    torch.cuda.synchronize()
    for a, w in zip(args, want):
        assert all(torch.equal(p, q) for p, q in zip(a, w))


@pytest.mark.parametrize("fmt,zeros", [("int4", "mixed"), ("mxfp4", "none")])
@pytest.mark.parametrize("T,K,N", [
    (3, 96, 70003),          # more tiles than work-groups: x stays
    (2, 640, 20010),
    (20, 2048, 5002),        # x in several turns
    (9, 5152, 34),           # parts of K of unequal length
    (24, 4096, 600), (70, 2880, 130), (1000, 128, 50), (6, 14336, 20), (48, 7168, 40)])
def test_projection_sizes(gpu, T, K, N, fmt, zeros):
    w = make_weight(fmt, zeros, N, K, 32, T + K)
    for x_bf16 in (False, True):
        print(f"proj4 {fmt} T={T} K={K} N={N} bf16={x_bf16}", flush=True)
        x, base = rows(T, K, K, x_bf16), rows(T, N, 3)
        check(run(gpu, w, x, base=base, y_bf16=x_bf16), *reference(w, x, base))
        if N % 2 == 0:
            check(run(gpu, w, x, glu=True), *reference(w, x, glu=True))
        del x, base


def test_projection_in_place_over_parts_of_k(gpu):
    """base is y where a second launch sums."""
    w = make_weight("int4", "asym", 40, 7168, 128, 1)
    x, base = rows(40, 7168, 1), rows(40, 40, 2)
    want = run(gpu, w, x, base=base)
    proj, z = ops.Projection4(w.to(gpu), 40), base.to(gpu).clone()
    proj(x.to(gpu), z, base=z)
    assert torch.equal(z, want)
    check(z, *reference(w, x, base))


def test_projection_with_a_larger_workspace(gpu):
    """An object for many rows gives a few the same bits as one made for them."""
    w = make_weight("mxfp4", "none", 40, 7168, 32, 1)
    x = rows(6, 7168, 1)
    want = run(gpu, w, x)
    proj, y = ops.Projection4(w.to(gpu), 500), torch.empty((6, 40), device=gpu)
    proj.workspace.fill_(255)
    proj(x.to(gpu), y)
    assert torch.equal(y, want)
