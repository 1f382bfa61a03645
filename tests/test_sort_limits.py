"""The limits of the sort's experts and slots, where an object of it is made: CPU
only, nothing is allocated or launched."""
import pytest

from grimoire_amd import _abi, ops

NOT_THERE = [(8, 0, 4), (8, -1, 4), (8, 17, 4), (0, 2, 4), (-3, 2, 4), (16385, 2, 4), (8, 2, -1)]


@pytest.mark.parametrize("E,K,T", NOT_THERE)
def test_refused_where_it_is_made(E, K, T):
    assert _abi.lib().grimoire_moe_sort_workspace_bytes(T, K, E) == 0
    with pytest.raises(_abi.GrimoireError, match="num_experts=.*top_k=.*max_tokens="):
        ops.TokenSort(E, K, T)


@pytest.mark.parametrize("E,K,T", [(1, 1, 0), (16384, 16, 1), (8, 16, 1 << 23)])
def test_workspaces_of_the_limits(E, K, T):
    """A count of each expert for every 256 routes, and a few words."""
    n = _abi.lib().grimoire_moe_sort_workspace_bytes(T, K, E)
    assert n >= 4 * E * max(1, (T * K + 255) // 256)
