"""The size queries of the transformer blocks' operators, which run before any check: 0 for what the call itself refuses."""
import ctypes as C

import pytest

from vita_amd import _lib as L


def _attention(**change):
    a = L.AttentionArgs()
    a.dtype, a.B, a.H, a.Hk, a.Sq, a.Sk, a.D, a.scale = L.DT_F32, 2, 4, 2, 1, 10000, 64, 0.125
    a.table = a.buckets = a.dtable = 1 << 20
    a.radius, a.num_buckets = 16, 8
    for n, v in change.items():
        setattr(a, n, v)
    return a


def test_attention_sizes():
    lib = L.load()
    assert lib.vita_attention_workspace_bytes(C.byref(_attention())) > 0 and lib.vita_attention_bwd_workspace_bytes(C.byref(_attention())) > 0


@pytest.mark.parametrize("change", [dict(Hk=0), dict(Hk=-2), dict(Hk=3), dict(Hk=8), dict(H=0), dict(H=-4), dict(B=0), dict(B=-1), dict(Sq=0), dict(Sq=-1),
                                    dict(Sk=-1), dict(D=0), dict(D=-8), dict(D=20), dict(D=136), dict(radius=-1), dict(radius=1025), dict(radius=1 << 30),
                                    dict(table=None, radius=-1), dict(dtable=None, radius=-1), dict(Sq=1 << 29), dict(Sk=2147483647)], ids=str)
def test_attention_sizes_of_refused_calls(change):
    lib = L.load()
    for query in (lib.vita_attention_workspace_bytes, lib.vita_attention_bwd_workspace_bytes):
        assert query(C.byref(_attention(**change))) == 0
        assert query(None) == 0
