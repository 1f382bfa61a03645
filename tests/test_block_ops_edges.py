"""The block operators' arguments that look wrong and are not: host checks
only, what is accepted would reach a launch."""
import os

import pytest

from tests.test_block_ops_overlap import ARG, launched, norm

no_gpu = pytest.mark.skipif(os.path.exists("/dev/kfd"), reason="made-up device addresses: no GPU may see them")


@no_gpu
def test_no_expert_rows():
    """No rows, no memory: a rank without routes.  Rows without memory are
    still refused."""
    assert launched(norm(moe=True, routed=None, rows=0))
    assert norm(moe=True, routed=None, rows=1) == ARG
    assert norm(moe=True, inverse=None, rows=0) == ARG and norm(moe=True, rw=None, rows=0) == ARG
