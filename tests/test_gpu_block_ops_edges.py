"""The block operators at the edges of what their arguments may be."""
import pytest
import torch

from grimoire_amd import ops, weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("T,H,shared", [(1, 64, False), (5, 260, True), (300, 512, False)])
def test_no_expert_rows(gpu, T, H, shared):
    """A rank that got no routes: the expert rows are an empty tensor, whose
    address is null; every route is another rank's."""
    g = torch.Generator().manual_seed(T)
    rn = lambda *s: torch.randn(*s, generator=g).to(gpu)
    n = ops.BlockNorm(rn(H).bfloat16(), rn(H).bfloat16(), block_scale=0.5)
    h, w, sh = rn(T, H), rn(T, 4), rn(T, H) if shared else None
    inv = torch.full((T * 4,), -1, dtype=torch.int32, device=gpu)
    inv[::3] = 0                                     # past the rows there are
    got = [torch.full((T, H), float("nan"), device=gpu) for _ in range(2)]
    ref = [torch.full((T, H), float("nan"), device=gpu) for _ in range(2)]
    none = torch.empty(0, H, dtype=torch.bfloat16, device=gpu)
    assert none.data_ptr() == 0
    n.moe(h, none, inv, w, sh, *got)
    n.moe(h, torch.full((1, H), float("nan"), device=gpu).bfloat16(), torch.full_like(inv, -1), w, sh, *ref)
    torch.cuda.synchronize()
    assert torch.equal(got[0], ref[0]) and torch.equal(got[1], ref[1])
    assert torch.isfinite(got[1]).all()
    if not shared:
        assert torch.equal(got[0], h)
