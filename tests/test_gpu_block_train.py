"""The operators around the experts together.  Served: a layer whose shared
expert is two 4-bit projections with their requests' adapters and whose tokens
are sorted by TokenSort.  Trained: scores -> sorted rows -> expert products ->
combine with a gated shared expert, and all of it backwards, against autograd in
64 bits; as a graph too, replayed with new inputs.

Tolerances of the training step, u = 2^-24 (a rounding of fp32): forward weights
of the scores have 2 (|l - max| + 2) u of two exponentials (differences up to 10
here), E additions and a few more: 64 u.  A product over n terms: n u of the sum
of their absolute values, whatever its order.  So, with A = |W| of the chosen
experts and sums over what an index is summed over:
  y:   (H + K + 68) u of |w| A |x| (+ |gate shared|)
  dx:  (D + K + 68) u of |w| A^T |g|
  dw:  (H + D + 4) u of |g| A |x|             =: e
  dlogits: dw_s/dl_e = w_s (d_se - w_e / S) f_e, f = 1 (softmax) or 1 - sigmoid,
       with the signs taken off: that times (e_s + 80 u |dw_s|)."""
import pytest
import torch

import test_gpu_block_run as served
from grimoire_amd import ops, weights
from test_gpu_block_run import E, H, I, K, SI, Layer

pytestmark = pytest.mark.gpu
U = 2.0 ** -24


class Layer4(Layer):
    """The shared expert in 4 bits, tokens sorted by TokenSort."""

    def __init__(self, gpu, make):
        super().__init__(gpu)
        self.sgu, self.sdn = make(2 * SI, H, 3).to(gpu), make(H, SI, 4).to(gpu)
        n = served.T
        self.up, self.down = ops.Projection4(self.sgu, n), ops.Projection4(self.sdn, n)
        self.sort = ops.TokenSort(E, K, n, device=gpu)

    def step(self):
        self.before(self.h, self.attn, self.h, self.x, self.xb)
        ops.router_logits(self.router, self.x, self.logits)
        self.scores(self.logits, self.ids, self.w)
        n = served.T
        self.sort(self.ids, self.x, self.xperm, self.counts, self.offsets, self.inverse)
        ops.grouped_gemm(self.gu, 2 * I, True, self.xperm, self.pair, self.offsets, self.counts, E, n * K)
        ops.grouped_gemm(self.dn, H, False, self.pair, self.rows, self.offsets, self.counts, E, n * K, a_pair=True,
                         out_bf16=True)
        self.up(self.xb, self.sv)
        self.lora[0].swiglu(self.slot, self.xb, self.sv, self.sh)
        self.down(self.sh, self.shared)
        self.lora[1].add(self.slot, self.sh, self.shared)
        self.after.moe(self.h, self.rows, self.inverse, self.w, self.shared, self.h2, self.out, self.out_bf,
                       gate=self.gate)


MAKE = {"int4": lambda n, k, s: weights.make_gptq_int4(n, k, group=64, seed=s),
        "mxfp4": lambda n, k, s: weights.make_mxfp4(n, k, exp_lo=-7, exp_hi=-5, seed=s)}


@pytest.mark.parametrize("fmt", ["int4", "mxfp4"])
@pytest.mark.parametrize("n", [1, 5, 40])
def test_served_layer(gpu, monkeypatch, fmt, n):
    monkeypatch.setattr(served, "T", n)
    L = Layer4(gpu, MAKE[fmt])
    L.load(1)
    h0 = L.h.clone()
    L.step()
    served.check(L, h0)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.step()
    for seed in (2, 3, 4):
        L.load(seed)
        h0 = L.h.clone()
        g.replay()
        served.check(L, h0)
        got = [t.clone() for t in (L.h2, L.out, L.out_bf, L.ids, L.w)]
        L.load(seed)
        L.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, (L.h2, L.out, L.out_bf, L.ids, L.w)))


class Train:
    """One step of a block of T tokens: experts W [E][D][H], a gated shared
    output; `first`: weights are applied to the rows before the experts."""

    def __init__(self, gpu, score, first, T=37, E=16, K=4, H=96, D=80, scaling=1.5):
        self.dims, self.first, self.scaling, self.score = (T, E, K, H, D), first, scaling, score
        f, i = (dict(device=gpu, dtype=t) for t in (torch.float32, torch.int32))
        self.W = (torch.randn((E, D, H), generator=torch.Generator().manual_seed(5)) * 0.2).to(gpu)
        self.scores = ops.RouteScores(score=score, scaling=scaling)
        self.sort = ops.TokenSort(E, K, T, device=gpu)
        self.x, self.g, self.logits = torch.empty(T, H, **f), torch.empty(T, D, **f), torch.empty(T, E, **f)
        self.shared, self.gate = torch.empty(T, D, **f), torch.empty(T, **f)
        self.ids, self.w, self.inv = torch.empty(T, K, **i), torch.empty(T, K, **f), torch.empty(T, K, **i)
        self.one = torch.ones(T, K, **f)
        self.counts, self.offsets = torch.empty(E, **i), torch.empty(E, **i)
        self.rows, self.out = torch.empty(T * K, H, **f), torch.empty(T * K, D, **f)
        self.y, self.dx, self.dlogits = torch.empty(T, D, **f), torch.empty(T, H, **f), torch.empty(T, E, **f)
        self.dout, self.dw = torch.empty(T * K, D, **f), torch.empty(T, K, **f)
        self.spare = torch.empty(T, K, **f)
        self.dshared, self.dgate = torch.empty(T, D, **f), torch.empty(T, **f)
        self.at = torch.arange(T * K, **i)

    def load(self, seed):
        g = torch.Generator().manual_seed(seed)
        for t in (self.x, self.g, self.logits, self.shared, self.gate):
            t.copy_(torch.randn(t.shape, generator=g))

    def forward(self):
        T, E, K, H, D = self.dims
        self.sort(self.ids, self.x, self.rows, self.counts, self.offsets, self.inv, weight=self.w if self.first else None)
        expert = torch.searchsorted(self.offsets + self.counts, self.at, right=True)
        self.We = self.W[expert]
        self.out.copy_((self.We * self.rows[:, None, :]).sum(2))
        ops.launch_moe_unpermute(self.out, self.inv, self.one if self.first else self.w, self.y, T, K, D)
        self.y.add_(self.gate[:, None] * self.shared)

    def step(self):
        self.scores(self.logits, self.ids, self.w)
        self.forward()
        ops.combine_grad(self.g, self.out, self.inv, self.one if self.first else self.w, self.dout,
                         self.spare if self.first else self.dw, shared=self.shared, gate=self.gate,
                         dshared=self.dshared, dgate=self.dgate)
        drows = (self.We * self.dout[:, :, None]).sum(1)
        extra = dict(x=self.x, weight=self.w, dweight=self.dw) if self.first else {}
        self.sort.grad(drows, self.inv, self.dx, **extra)
        self.scores.grad(self.logits, self.ids, self.dw, self.dlogits)

    results = property(lambda self: [t.clone() for t in (self.y, self.dx, self.dw, self.dlogits, self.dshared, self.dgate)])

    def check(self):
        torch.cuda.synchronize()
        T, E, K, H, D = self.dims
        ids = self.ids.cpu().long()
        x, l, sh, ga = (t.cpu().double().requires_grad_() for t in (self.x, self.logits, self.shared, self.gate))
        p = l.gather(1, ids)
        sig = torch.sigmoid(l)
        p = p.softmax(1) if self.score == "softmax" else sig.gather(1, ids) / sig.gather(1, ids).sum(1, keepdim=True)
        w = self.scaling * p
        w.retain_grad()
        We, g = self.W.cpu().double()[ids], self.g.cpu().double()
        y = (w[:, :, None] * (We * x[:, None, None, :]).sum(3)).sum(1) + ga[:, None] * sh
        (y * g).sum().backward()
        A, w0 = We.abs(), w.detach()
        xa, ga_, gs = x.detach().abs(), g.abs(), (ga[:, None] * sh).detach().abs()
        up = (A * xa[:, None, None, :]).sum(3)
        near = lambda got, want, tol: self._near(got.cpu().double(), want.detach(), tol)
        near(self.y, y, (H + K + 68) * U * ((w0[:, :, None] * up).sum(1) + gs))
        near(self.dx, x.grad, (D + K + 68) * U * (w0[:, :, None] * (A * ga_[:, None, :, None]).sum(2)).sum(1))
        e = (H + D + 4) * U * (ga_[:, None, :] * up).sum(2)
        near(self.dw, w.grad, e)
        each = e + 80 * U * w.grad.abs()
        f = torch.ones_like(w0) if self.score == "softmax" else 1 - sig.detach().gather(1, ids)
        jac = w0[:, :, None] * (torch.eye(K).double() + w0[:, None, :] / self.scaling) * f[:, None, :]
        near(self.dlogits, l.grad, torch.zeros_like(l).detach().scatter(1, ids, (jac * each[:, :, None]).sum(1)))
        near(self.dshared, sh.grad, U * sh.grad.abs())
        near(self.dgate, ga.grad, (D + 4) * U * (ga_ * sh.detach().abs()).sum(1))

    @staticmethod
    def _near(got, want, tol):
        err = (got - want).abs()
        assert (err <= tol).all(), float((err / tol.clamp_min(1e-300)).max())


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("first", [False, True])
def test_training_step(gpu, score, first):
    """Eagerly, and as a graph while the eager results live."""
    t = Train(gpu, score, first)
    for seed in (1, 2):
        t.load(seed)
        t.step()
        t.check()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        t.step()
    for seed in (3, 4, 5):
        t.load(seed)
        graph.replay()
        t.check()
        got = t.results
        t.load(seed)
        t.step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, t.results))


@pytest.mark.parametrize("T", [1, 3])
def test_small_steps(gpu, T):
    t = Train(gpu, "softmax", False, T=T, E=5, K=5, H=8, D=4)
    t.load(1)
    t.step()
    t.check()


def test_two_graphs_share_a_workspace(gpu):
    """Two captured calls of one TokenSort and of one Projection4, replayed one
    after the other, each with its own arguments."""
    T, N = 50, 48
    sort = ops.TokenSort(16, 4, T, device=gpu)
    proj = ops.Projection4(MAKE["int4"](N, 7168, 1).to(gpu), T)
    i32 = dict(dtype=torch.int32, device=gpu)

    def args(seed):
        g = torch.Generator().manual_seed(seed)
        return dict(ids=torch.randint(0, 16, (T, 4), generator=g).int().to(gpu),
                    x=torch.randn((T, 7168), generator=g).to(gpu), rows=torch.empty((T * 4, 7168), device=gpu),
                    counts=torch.empty(16, **i32), offsets=torch.empty(16, **i32), inverse=torch.empty((T, 4), **i32),
                    y=torch.empty((T, N), device=gpu))

    def call(a):
        sort(*(a[k] for k in ("ids", "x", "rows", "counts", "offsets", "inverse")))
        proj(a["x"], a["y"])
    both, graphs = [args(1), args(2)], []
    for a in both:
        call(a)
    torch.cuda.synchronize()
    want = [[a[k].clone() for k in ("rows", "counts", "offsets", "inverse", "y")] for a in both]
    for a in both:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            call(a)
    for _ in range(3):
        for a in both:
            for k in ("rows", "counts", "offsets", "inverse", "y"):
                a[k].fill_(-3)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, w in zip(both, want):
            assert all(torch.equal(a[k], v) for k, v in zip(("rows", "counts", "offsets", "inverse", "y"), w))


def test_combine_gradient_against_differences(gpu):
    """The combine is linear in its rows, weights and shared rows: what a step
    along a direction changes is the gradient's product with it, up to rounding:
    (K + 2) u of each output's terms for the two forward passes, in sums of 64
    bits; the gradients' own errors, D u of their terms, beside it."""
    T, K, D = 21, 3, 132
    g = torch.Generator().manual_seed(9)
    rn = lambda *s: torch.randn(s, generator=g)
    rows, w, sh, ga, dy = rn(T * K, D), rn(T, K), rn(T, D), rn(T), rn(T, D)
    inv = torch.randperm(T * K, generator=g).int().view(T, K)
    c = [t.to(gpu) for t in (dy, rows, inv, w, sh, ga)]
    dr, dw, ds, dg = (torch.empty_like(t) for t in (c[1], c[3], c[4], c[5]))
    ops.combine_grad(*c[:4], dr, dw, shared=c[4], gate=c[5], dshared=ds, dgate=dg)

    def loss(rows, w, sh, ga):
        y = torch.empty((T, D), device=gpu)
        ops.launch_moe_unpermute(rows.to(gpu), c[2], w.to(gpu), y, T, K, D)
        return float(((y.cpu().double() + ga.double()[:, None] * sh.double()) * dy.double()).sum())
    at, grads = [rows, w, sh, ga], [dr, dw, ds, dg]
    for n, grad in enumerate(grads):
        step = rn(*at[n].shape)
        moved = [t + step if m == n else t for m, t in enumerate(at)]
        exact = moved[n].double() - at[n].double()              # the step as fp32 takes it
        diff = loss(*moved) - loss(*at)
        size = sum(float(((a[0][inv.long()].abs() * a[1].abs()[:, :, None]).sum(1) * dy.abs()).sum())
                   + float((a[2].abs() * a[3].abs()[:, None] * dy.abs()).sum()) for a in (moved, at))
        part = float((grad.cpu().double() * exact).sum())
        terms = float((dy.abs()[:, None, :] * (rows[inv.long()].abs() + w.abs()[:, :, None] + 1.0)).sum()) \
            + float((dy.abs() * (sh.abs() + ga.abs()[:, None])).sum())
        assert abs(diff - part) <= (K + 2) * U * size + (D + 2) * U * terms * float(exact.abs().max())
