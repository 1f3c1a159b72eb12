"""What the transformer blocks' operators take and refuse at the edges of their documented arguments."""
import pytest
import torch

import block_ops_reference as ref
from vita_amd import _lib as L
from vita_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16]


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


@pytest.mark.parametrize("H,Hk", [(0, 2), (2, 0), (0, 0)])
def test_norm_rope_without_heads_is_refused(H, Hk):
    """(It left the other side's result unwritten.)"""
    q, k = torch.zeros(2, 3, H, 8, device=DEV), torch.zeros(2, 3, Hk, 8, device=DEV)
    rope = ref.rope_table(3, 1, 8).to(DEV)
    for call in (lambda: ops.qk_norm_rope(q, k, rope), lambda: ops.qk_norm_rope_bwd(q, k, q, k, rope)):
        with pytest.raises(L.VitaHipError, match="needs a head"):
            call()
