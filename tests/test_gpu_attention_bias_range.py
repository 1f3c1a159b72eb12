"""ops.attention's learned bias over its whole range: large entries, entries that no pair of tokens meets, and every radius up to the largest
with many query heads to a key head, against the 64-bit forms and bounds of tests/block_ops_reference.py."""
import pytest
import torch

import block_ops_reference as ref
from vita_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16]


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


def _check(q, k, v, g, **kw):
    o, stats = ops.attention(q, k, v, need_lse=True, **kw)
    do = _randn(g, *q.shape, dtype=q.dtype)
    got = (o, None, *ops.attention_bwd(do, q, k, v, o, stats, **kw))
    want = ref.attention(q, k, v, do=do, **kw)
    # The bounds are relative: they do not count probabilities of exp(-100) and the like, which fp32 flushes to zero.  Such a P is off by at
    # most 2^-126; with |dP|, |delta| <= c = D max|dO| max|v| its dS = P (dP - delta) by 2^-126 2 c and its own flush of 2^-126; a result adds
    # at most B H Sq Sk of either, each times an element of q, k, v or dO (and |scale| < 1) or 1.
    m = max(1.0, *(t.abs().max().item() for t in (q, k, v, do)))
    B, Sq, H, D = q.shape
    flush = 2.0 ** -126 * (2 * D * m * m + 1) * B * H * Sq * k.shape[1] * m
    for i, n in enumerate(("o", "lse", "dq", "dk", "dv", "dtable")):
        if n != "lse":
            ref.assert_close(got[i], want[2 * i], want[2 * i + 1] + flush, n)


# ---- large entries ----------------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("value", [100.0, 1000.0])
@pytest.mark.parametrize("Sq,Sk", [(17, 17), (33, 33), (33, 80), (150, 150), (1, 70)])
def test_large_bias(dtype, causal, value, Sq, Sk):
    """exp(value) is beyond fp32; the softmax does not depend on a constant.  By distance: everywhere, beyond the radius, inside it."""
    g = torch.Generator().manual_seed(Sq + Sk)
    for R in (3, 64):
        for hidden in ([0, 1, 2, 3], [0, 3], [1, 2]):
            q, k, v = _randn(g, 2, Sq, 4, 32, dtype=dtype), _randn(g, 2, Sk, 2, 32, dtype=dtype), _randn(g, 2, Sk, 2, 32, dtype=dtype)
            table = _randn(g, 4, 4, dtype=dtype)
            table[hidden] += value
            buckets = torch.randint(1, 3, (2 * R + 1,), generator=g, dtype=torch.int32)
            buckets[0], buckets[-1] = 0, 3
            _check(q, k, v, g, causal=causal, table=table, buckets=buckets.to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("entry", ["nan", "inf", "outside"])
@pytest.mark.parametrize("Sq,Sk", [(17, 17), (33, 80), (150, 150)])
def test_entries_of_distances_that_no_pair_has(dtype, entry, Sq, Sk):
    g = torch.Generator().manual_seed(Sq)
    R = Sk + 60
    q, k, v = _randn(g, 2, Sq, 2, 32, dtype=dtype), _randn(g, 2, Sk, 2, 32, dtype=dtype), _randn(g, 2, Sk, 2, 32, dtype=dtype)
    table = _randn(g, 4, 2, dtype=dtype)
    table[3] = float(entry) if entry != "outside" else 0.0
    buckets = torch.randint(0, 3, (2 * R + 1,), generator=g, dtype=torch.int32)
    far = torch.arange(-R, R + 1)
    buckets[(far <= -Sk) | (far > Sq - 1)] = 9 if entry == "outside" else 3
    _check(q, k, v, g, table=table, buckets=buckets.to(DEV))


# ---- the radius -------------------------------------------------------------------------------------------------------------------
def _radius(dtype, R, Sq, Sk, H, Hk, D):
    g = torch.Generator().manual_seed(R + Sq)
    q, k, v = _randn(g, 2, Sq, H, D, dtype=dtype), _randn(g, 2, Sk, Hk, D, dtype=dtype), _randn(g, 2, Sk, Hk, D, dtype=dtype)
    bias = dict(table=_randn(g, 32, H, dtype=dtype), buckets=torch.randint(0, 32, (2 * R + 1,), generator=g, dtype=torch.int32).to(DEV))
    pad = torch.zeros(2, Sk, dtype=torch.bool)
    pad[1, Sk // 3:] = True
    _check(q, k, v, g, causal=R % 2 == 0, key_pad=pad.to(DEV), **bias)


@pytest.mark.parametrize("R", [240, 241, 243, 244, 256, 1024])
@pytest.mark.parametrize("Sq", [1, 17, 32, 70])
@pytest.mark.parametrize("Sk", [64, 300])
@pytest.mark.parametrize("D", [96, 128])
def test_backward_at_every_radius(R, Sq, Sk, D):
    _radius(torch.float32, R, min(Sq, Sk), Sk, 2, 2, D)


@pytest.mark.parametrize("dtype,G", [(torch.float32, 4), (torch.float32, 8), (torch.float32, 12), (torch.float32, 32), (torch.bfloat16, 16), (torch.bfloat16, 64)])
@pytest.mark.parametrize("R", [128, 432, 664, 1024])
@pytest.mark.parametrize("D", [64, 128])
def test_packed_heads_at_every_radius(dtype, G, R, D):
    """Few rows of many query heads to a key head: one of 300 and of 129 keys."""
    _radius(dtype, R, 1, 300, G, 1, D)
    _radius(dtype, R, max(1, 64 // G), 129, 2 * G, 2, D)
