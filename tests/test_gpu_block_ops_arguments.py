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


def _off(t):
    """The same numbers one element behind a 16-byte border, as a slice of a flat buffer of parameters has them."""
    return torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)[1:].view(t.shape).copy_(t)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M", [5, 70])
def test_gated_parameters_off_the_borders(dtype, M):
    g = torch.Generator().manual_seed(M)
    x, w, b, dh = _randn(g, M, 16, dtype=dtype), _randn(g, 48, 16, dtype=dtype), _randn(g, 48), _randn(g, M, 24, dtype=dtype)
    h, saved = ops.gated_linear(x, w, b, need_saved=True)
    assert torch.equal(ops.gated_linear(x, w, _off(b)), h)
    want = ops.gated_linear_bwd(dh, x, w, b, saved=saved)
    got = ops.gated_linear_bwd(dh, x, w, _off(b), saved=_off(saved) if saved is not None else None)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_backward_of_a_part_of_a_batch(dtype):
    """Row statistics sliced out of a batch's (3 heads x 5 fp32 rows of 8 bytes: the second batch row starts off the 16-byte borders)."""
    g = torch.Generator().manual_seed(2)
    q, k, v, do = (_randn(g, 3, 5, 3, 16, dtype=dtype) for _ in range(4))
    o, stats = ops.attention(q, k, v, need_lse=True)
    want = ops.attention_bwd(do, q, k, v, o, stats)
    for part in (slice(1, 3), slice(1, 2)):
        got = ops.attention_bwd(*(t[part] for t in (do, q, k, v, o, stats)))
        assert all(torch.equal(p, q[part]) for p, q in zip(got[:3], want[:3]))


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_parameters_off_the_borders(dtype):
    g = torch.Generator().manual_seed(3)
    q, k = _randn(g, 2, 3, 4, 24, dtype=dtype), _randn(g, 2, 3, 2, 24, dtype=dtype)
    rope, w = ref.rope_table(3, 1, 24).to(DEV), {n: _randn(g, 24) for n in ("q_weight", "q_bias", "k_weight", "k_bias")}
    want = ops.qk_norm_rope(q, k, rope, **w)
    got = ops.qk_norm_rope(q, k, _off(rope), **{n: _off(t) for n, t in w.items()})
    assert all(torch.equal(p, q) for p, q in zip(got, want))
