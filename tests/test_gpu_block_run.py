"""The operators around the MoE block together, as a served layer runs them:
the norms before the block -> router logits -> scores -> dispatch -> expert
products, beside them the shared expert with its requests' adapters (gate|up
+ SwiGLU, down) -> combine, norm, gate, residual, next norm.  Checked against
the same in 64 bits on the routes the router chose, eagerly and as a graph
replayed on new inputs.

Tolerance: every stage's output is within a half step of bf16 (2^-8) of its
own: the normed input, the routed h, the shared h, the expert rows and the
shared expert's two projections.  A product passes a relative change of its
input on as it is, silu(g) u as at most about 2.1 times (g and u both
change), so f is off by at most (2.1 + 1 + 1 + 2.1 + 1) 2^-8 = 2.9e-2 of the
norms of its two summands, and the norms pass that on."""
import pytest
import torch

from grimoire_amd import ops, weights
from tests.helpers import dequant

pytestmark = pytest.mark.gpu
T, H, E, K, I, SI, REQ = 96, 512, 16, 4, 256, 256, 5


class Layer:
    """The weights of one layer and the buffers of a batch of T rows."""

    def __init__(self, gpu):
        g = torch.Generator().manual_seed(77)
        rn = lambda *s: torch.randn(s, generator=g)
        self.gu = weights.make_bf16(E * 2 * I, H, seed=1).to(gpu)
        self.dn = weights.make_bf16(E * H, I, seed=2).to(gpu)
        self.sgu = weights.make_bf16(2 * SI, H, seed=3).to(gpu)
        self.sdn = weights.make_bf16(H, SI, seed=4).to(gpu)
        self.router = (rn(E, H) * 0.05).to(gpu)
        w = [(rn(H) * 0.1).bfloat16().to(gpu) for _ in range(4)]
        self.before = ops.BlockNorm(w[0], w[1], residual_scale=0.9)
        self.after = ops.BlockNorm(w[2], w[3], block_scale=0.5, gate="row", gate_sigmoid=True)
        self.scores = ops.RouteScores(bias=(rn(E) * 0.01).to(gpu), n_group=4, topk_group=2, scaling=1.5)
        ads = []
        for n, k in ((2 * SI, H), (H, SI)):
            ad = weights.LoraAdapters.empty(4, 32, k, n, device=gpu)
            for s, r in enumerate((32, 7, 16, 1)):
                ad.load(s, (rn(r, k) / k ** 0.5).to(gpu), (rn(n, r) * 0.2).to(gpu), 1.0 + 0.25 * s)
            ads.append(ad)
        self.ads = ads
        self.lora = [ops.Lora(a, T) for a in ads]
        f32, b16, i32 = (dict(device=gpu, dtype=d) for d in (torch.float32, torch.bfloat16, torch.int32))
        self.h, self.attn = torch.empty(T, H, **f32), torch.empty(T, H, **f32)
        self.slot, self.gate = torch.empty(T, **i32), torch.empty(T, **f32)
        self.x, self.xb = torch.empty(T, H, **f32), torch.empty(T, H, **b16)
        self.logits = torch.empty(T, E, **f32)
        self.ids, self.w = torch.empty(T, K, **i32), torch.empty(T, K, **f32)
        self.xperm = torch.empty(T * K, H, **b16)
        self.counts, self.offsets = torch.empty(E, **i32), torch.empty(E, **i32)
        self.inverse = torch.empty(T * K, **i32)
        self.ws = torch.empty(ops.route_workspace_bytes(T, K, E), dtype=torch.uint8, device=gpu)
        self.pair = torch.empty(T * K, 2, I, **b16)
        self.rows = torch.empty(T * K, H, **b16)
        self.all, self.zero = torch.full((1,), T, **i32), torch.zeros(1, **i32)
        self.sv, self.sh = torch.empty(T, 2 * SI, **f32), torch.empty(T, SI, **b16)
        self.shared = torch.empty(T, H, **f32)
        self.h2, self.out = torch.empty(T, H, **f32), torch.empty(T, H, **f32)
        self.out_bf = torch.empty(T, H, **b16)

    def load(self, seed):
        g = torch.Generator().manual_seed(seed)
        rn = lambda *s: torch.randn(s, generator=g)
        self.h.copy_(rn(T, H) * 2)
        self.attn.copy_(rn(T, H))
        self.gate.copy_(rn(T))
        self.slot.copy_(torch.randint(-1, 4, (REQ,), generator=g)[torch.arange(T) * REQ // T])

    def step(self):
        self.before(self.h, self.attn, self.h, self.x, self.xb)
        ops.router_logits(self.router, self.x, self.logits)
        self.scores(self.logits, self.ids, self.w)
        ops.launch_moe_route_grouped(self.x, self.ids, self.xperm, None, self.counts, self.offsets, self.inverse,
                                     None, None, 0, T, H, E, 128, K, workspace=self.ws)
        ops.grouped_gemm(self.gu, 2 * I, True, self.xperm, self.pair, self.offsets, self.counts, E, T * K)
        ops.grouped_gemm(self.dn, H, False, self.pair, self.rows, self.offsets, self.counts, E, T * K, a_pair=True,
                         out_bf16=True)
        ops.grouped_gemm(self.sgu, 2 * SI, False, self.xb, self.sv, self.zero, self.all, 1, T)
        self.lora[0].swiglu(self.slot, self.xb, self.sv, self.sh)
        ops.grouped_gemm(self.sdn, H, False, self.sh, self.shared, self.zero, self.all, 1, T)
        self.lora[1].add(self.slot, self.sh, self.shared)
        self.after.moe(self.h, self.rows, self.inverse, self.w, self.shared, self.h2, self.out, self.out_bf,
                       gate=self.gate)

    def want(self, h, ids, w):
        """h', o and f's scale from the inputs loaded, in fp64."""
        d = lambda t: t.double()
        rms = lambda v: v * torch.rsqrt(v.square().mean(1, keepdim=True) + 1e-6)
        nw = lambda t: 1.0 + t.double()
        h = 0.9 * d(h) + rms(d(self.attn)) * nw(self.before.post_weight)
        x = rms(h) * nw(self.before.pre_weight)
        silu = torch.nn.functional.silu
        gu, dn = d(dequant(self.gu)).view(E, 2 * I, H), d(dequant(self.dn)).view(E, H, I)
        f = torch.zeros(T, H, dtype=torch.float64, device=h.device)
        for e in range(E):
            t, k = torch.where(ids == e)
            v = x[t] @ gu[e].T.contiguous()
            f.index_add_(0, t, (silu(v[:, :I]) * v[:, I:]) @ dn[e].T.contiguous() * d(w)[t, k][:, None])

        def adapted(v, base, ad):
            out = v @ d(dequant(base)).T.contiguous()
            for s in range(4):
                t, r = torch.where(self.slot == s)[0], int(ad.rank[s])
                low = v[t] @ d(ad.a[s, :r]).T.contiguous()
                out[t] += float(ad.scale[s]) * low @ d(ad.b[s, :, :r]).T.contiguous()
            return out
        v = adapted(x, self.sgu, self.ads[0])
        f = f + adapted(silu(v[:, :SI]) * v[:, SI:], self.sdn, self.ads[1])
        p = rms(f) * nw(self.after.post_weight)
        hh = h + 0.5 * torch.sigmoid(d(self.gate))[:, None] * p
        return h, hh, rms(hh) * nw(self.after.pre_weight)


def check(L, h0):
    torch.cuda.synchronize()
    h, hh, out = L.want(h0, L.ids, L.w)
    norm = torch.linalg.norm
    assert norm(L.h.double() - h) <= 1e-5 * norm(h)
    assert norm((L.h2.double() - L.h.double()) - (hh - h)) <= 2.9e-2 * norm(hh - h)
    assert norm(L.out.double() - out) <= 2.9e-2 * norm(out)
    assert norm(L.out_bf.double() - out) <= 3.4e-2 * norm(out)
    assert int((L.ids < 0).sum()) == 0
    total = L.w.double().sum(1)
    assert ((total - 1.5).abs() < 1e-5).all()


def test_layer_eager_and_replayed(gpu):
    L = Layer(gpu)
    for seed in (1, 2):
        L.load(seed)
        h0 = L.h.clone()
        L.step()
        check(L, h0)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        L.step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        L.step()
    for seed in (3, 4, 5):
        L.load(seed)
        h0 = L.h.clone()
        g.replay()
        check(L, h0)
        got = [t.clone() for t in (L.h2, L.out, L.out_bf, L.ids, L.w)]
        L.load(seed)
        L.step()
        torch.cuda.synchronize()
        for a, b in zip(got, (L.h2, L.out, L.out_bf, L.ids, L.w)):
            assert torch.equal(a, b)
