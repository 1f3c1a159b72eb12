"""ops.attention and its backward pass where whole runs of keys are padded (in front, in holes, behind), against the 64-bit forms and bounds
of tests/block_ops_reference.py."""
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
    for i, n in enumerate(("o", "lse", "dq", "dk", "dv", "dtable")):
        if n == "lse" or (n == "dtable" and kw.get("table") is None):
            continue
        ref.assert_close(got[i], want[2 * i], want[2 * i + 1], n)


# the keys that a batch row has, by ranges (None: up to the last one): padded in front by one word of 64 and by parts of it, holes of a
# word and across words, padded behind, two keys, none
LIVE = [[(64, None)], [(70, None)], [(192, None)], [(0, 60), (128, None)], [(0, 50), (200, None)], [(0, 90)], [(100, 101), (255, 256)], []]


def _live(Sk):
    pad = torch.ones(len(LIVE), Sk, dtype=torch.bool)
    for b, runs in enumerate(LIVE):
        for lo, hi in runs:
            pad[b, lo:hi] = False
    return pad.to(DEV)


def _runs_of_padded_keys(dtype, causal, R, Sq, Sk, H, Hk, D):
    g = torch.Generator().manual_seed(Sq + Sk + D)
    B = len(LIVE)
    q, k, v = _randn(g, B, Sq, H, D, dtype=dtype), _randn(g, B, Sk, Hk, D, dtype=dtype), _randn(g, B, Sk, Hk, D, dtype=dtype)
    bias = {}
    if R is not None:
        bias = dict(table=_randn(g, 16, H, dtype=dtype), buckets=torch.randint(0, 16, (2 * R + 1,), generator=g, dtype=torch.int32).to(DEV))
    _check(q, k, v, g, key_pad=_live(Sk), causal=causal, **bias)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("R", [None, 9])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("Sq,Sk", [(1, 300), (20, 300), (200, 300), (300, 300)])
def test_runs_of_padded_keys(dtype, causal, R, D, Sq, Sk):
    _runs_of_padded_keys(dtype, causal, R, Sq, Sk, 2, 1, D)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal,R", [(False, None), (True, 9)])
def test_runs_of_padded_keys_many_heads(dtype, causal, R):
    """Enough rows that workgroups of 4 x 32 rows run (fewer take the form whose waves share out the other axis)."""
    _runs_of_padded_keys(dtype, causal, R, 200, 300, 16, 16, 32)


@pytest.mark.parametrize("causal,R", [(False, 9), (True, None)])
def test_runs_of_padded_keys_long_uneven_rows(causal, R):
    """fp32, 512 tokens and as many workgroups as there are CUs: rows of unequal length take the shared form here too."""
    _runs_of_padded_keys(torch.float32, causal, R, 512, 512, 8, 8, 16)
