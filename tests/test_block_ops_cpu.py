"""The transformer blocks' operators without a GPU: what the C entry points and the Python layer refuse, and the bucket ids."""
import ctypes as C

import pytest
import torch

from vita_amd import _lib as L
from vita_amd import ops


def _norm_rope():
    a = L.NormRopeArgs()
    a.dtype, a.norm, a.B, a.S, a.D, a.eps = L.DT_BF16, L.NORM_LAYER, 2, 3, 64, 1e-5
    a.rope, a.rope_rows, a.rope_heads = 1 << 20, 8, 1
    for s in (a.q, a.k):
        s.x = s.y = s.dy = 1 << 20
        s.H = 4
    return a


@pytest.mark.parametrize("change,text", [(dict(dtype=7), "dtype"), (dict(norm=2), "norm"), (dict(D=3), "shape"), (dict(D=258), "shape"), (dict(D=0), "shape"),
                                         (dict(B=-1), "shape"), (dict(rope=None), "rotation table"), (dict(rope_rows=2), "3 tokens"),
                                         (dict(rope_heads=2), "2 heads"), (dict(rope=4 + (1 << 20)), "8-byte"), (dict(B=1 << 28, S=4), "2\\^31"),
                                         (dict(positions=1 << 20, ld_positions=2), "ld_positions")])
def test_norm_rope_refuses(change, text):
    lib = L.load()
    a = _norm_rope()
    for n, v in change.items():
        setattr(a, n, v)
    for call in (lambda: lib.vita_qk_norm_rope(C.byref(a), None), lambda: lib.vita_qk_norm_rope_bwd(C.byref(a), None, 0, None)):
        assert call() == -1
        with pytest.raises(L.VitaHipError, match=text):
            L.check(-1, "call")


def test_norm_rope_refuses_tensors_and_workspace():
    lib = L.load()
    for side in ("q", "k"):
        for field, value, text in (("x", None, "null"), ("y", None, "null"), ("x", 1 + (1 << 20), "misaligned"), ("H", 0, "head counts")):
            a = _norm_rope()
            setattr(getattr(a, side), field, value)
            assert lib.vita_qk_norm_rope(C.byref(a), None) == -1 and text in lib.vita_last_error().decode()
    a = _norm_rope()
    a.k.dy = None
    assert lib.vita_qk_norm_rope_bwd(C.byref(a), None, 0, None) == -1
    a = _norm_rope()
    need = lib.vita_qk_norm_rope_bwd_workspace_bytes(C.byref(a))
    assert need > 0 and lib.vita_qk_norm_rope_bwd(C.byref(a), 1 << 20, need - 1, None) == -3
    assert lib.vita_qk_norm_rope_bwd(C.byref(a), (1 << 20) + 8, need, None) == -3 and "aligned" in lib.vita_last_error().decode()
    assert lib.vita_qk_norm_rope(None, None) == -1
    a.B = 0
    assert lib.vita_qk_norm_rope(C.byref(a), None) == 0


def _attention():
    a = L.AttentionArgs()
    a.dtype, a.B, a.H, a.Hk, a.Sq, a.Sk, a.D, a.scale = L.DT_BF16, 2, 4, 2, 40, 50, 64, 0.125
    for n in ("q", "k", "v", "o", "dout", "dq", "dk", "dv"):
        setattr(a, n, 1 << 20)
        setattr(a, n + "_sb", 64 * 4 * 64)
        setattr(a, n + "_ss", 64 * 4)
        setattr(a, n + "_sh", 64)
    a.stats = 1 << 20
    return a


@pytest.mark.parametrize("change,text", [(dict(dtype=2), "dtype"), (dict(H=0), "shape"), (dict(Sq=-1), "shape"), (dict(Hk=3), "4 query heads over 3"),
                                         (dict(D=20), "head dimension 20"), (dict(D=136), "head dimension"), (dict(D=0), "head dimension"),
                                         (dict(q=None), "non-null"), (dict(v=8 + (1 << 20)), "aligned"), (dict(k_ss=60), "strides"),
                                         (dict(o_sh=4), "strides"), (dict(k_ss=1 << 23), "2\\^23"), (dict(q_ss=-64), "2\\^23"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
                                         (dict(key_pad=1 << 20, ld_pad=49), "ld_pad"), (dict(table=1 << 20, buckets=None), "bias"),
                                         (dict(table=1 << 20, buckets=1 << 20, radius=1025, num_buckets=4), "radius 1025"),
                                         (dict(table=1 << 20, buckets=1 << 20, radius=-1, num_buckets=4), "radius"),
                                         (dict(table=1 << 20, buckets=1 << 20, radius=3, num_buckets=0), "0 buckets"), (dict(Sq=1 << 29), "too long")])
def test_attention_refuses(change, text):
    lib = L.load()
    a = _attention()
    for n, v in change.items():
        setattr(a, n, v)
    for call in (lambda: lib.vita_attention(C.byref(a), None, 0, None), lambda: lib.vita_attention_bwd(C.byref(a), None, 0, None)):
        assert call() == -1
        with pytest.raises(L.VitaHipError, match=text):
            L.check(-1, "call")


def test_attention_bwd_refuses():
    lib = L.load()
    for change in (dict(stats=None), dict(stats=8 + (1 << 20)), dict(dout=None), dict(dq_ss=3), dict(dk=None), dict(dv=2 + (1 << 20)), dict(dtable=1 << 20)):
        a = _attention()
        for n, v in change.items():
            setattr(a, n, v)
        assert lib.vita_attention_bwd(C.byref(a), None, 0, None) == -1, change
    a = _attention()
    need = lib.vita_attention_bwd_workspace_bytes(C.byref(a))
    assert need >= 2 * 4 * 40 * 4 and lib.vita_attention_bwd(C.byref(a), 1 << 20, need - 1, None) == -3
    # one token over a long cache: the key axis is split, and the parts need room
    a.Sq, a.Sk = 1, 10000
    assert lib.vita_attention_workspace_bytes(C.byref(a)) > 0 and lib.vita_attention(C.byref(a), None, 0, None) == -3
    a.B = 0
    assert lib.vita_attention(C.byref(a), None, 0, None) == 0 and lib.vita_attention_workspace_bytes(C.byref(a)) == 0
    assert lib.vita_attention(None, None, 0, None) == -1


def _gated():
    a = L.GatedArgs()
    a.dtype, a.act, a.M, a.F, a.K = L.DT_BF16, L.ACT_SILU, 5, 64, 32
    a.x = a.w = a.h = a.dh = a.dx = a.dw = 1 << 20
    a.ldx = a.ldw = a.ld_dx = a.ld_dw = 32
    a.ldh = a.ld_dh = 64
    return a


@pytest.mark.parametrize("change,text", [(dict(dtype=5), "dtype"), (dict(act=L.ACT_NONE), "activation"), (dict(act=6), "activation"), (dict(F=60), "multiples of 8"),
                                         (dict(K=4), "multiples of 8"), (dict(M=-1), "shape"), (dict(x=None), "rows"), (dict(ldx=24), "rows"), (dict(ldw=36), "rows"),
                                         (dict(w=8 + (1 << 20)), "rows"), (dict(b=4 + (1 << 20)), "b must"), (dict(z=1 << 20, ldz=64), "bad z")])
def test_gated_refuses(change, text):
    lib = L.load()
    a = _gated()
    for n, v in change.items():
        setattr(a, n, v)
    for call in (lambda: lib.vita_gated_linear(C.byref(a), None, 0, None), lambda: lib.vita_gated_linear_bwd(C.byref(a), None, 0, None)):
        assert call() == -1
        with pytest.raises(L.VitaHipError, match=text):
            L.check(-1, "call")


def test_gated_refuses_outputs_and_workspace():
    lib = L.load()
    a = _gated()
    a.h = None
    assert lib.vita_gated_linear(C.byref(a), None, 0, None) == -1
    for change in (dict(dh=None), dict(ld_dh=32), dict(ld_dx=8), dict(dw=4 + (1 << 20)), dict(M=0)):
        a = _gated()
        for n, v in change.items():
            setattr(a, n, v)
        assert lib.vita_gated_linear_bwd(C.byref(a), None, 0, None) == -1, change
    a = _gated()
    need = lib.vita_gated_linear_bwd_workspace_bytes(C.byref(a))
    assert need > 0 and lib.vita_gated_linear_bwd(C.byref(a), 1 << 20, need - 1, None) == -3
    a.M = 0
    assert lib.vita_gated_linear(C.byref(a), None, 0, None) == 0


def test_no_cpu_path_and_shapes():
    q = torch.zeros(2, 3, 4, 16)
    rope = torch.zeros(3, 8, 2)
    for call in (lambda: ops.qk_norm_rope(q, q, rope), lambda: ops.attention(q, q, q), lambda: ops.gated_linear(q[0, 0], q[0, 0])):
        with pytest.raises(L.VitaHipError, match="on the GPU"):
            call()


def test_struct_layouts_match_the_header(tmp_path):
    import os
    import subprocess
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    names = {"vita_norm_rope_side": L.NormRopeSide, "vita_norm_rope_args": L.NormRopeArgs, "vita_attention_args": L.AttentionArgs, "vita_gated_args": L.GatedArgs}
    src = '#include <stdio.h>\n#include <stddef.h>\n#include "vita_hip.h"\nint main(void){'
    want = []
    for n, s in names.items():
        src += f'printf("%zu\\n", sizeof({n}));'
        want.append(C.sizeof(s))
        for f, _ in s._fields_:
            src += f'printf("%zu\\n", offsetof({n}, {f}));'
            want.append(getattr(s, f).offset)
    (tmp_path / "s.c").write_text(src + "return 0;}\n")
    subprocess.run(["gcc", "-std=c99", "-Wall", "-Werror", "-I", os.path.join(root, "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    assert [int(x) for x in subprocess.run([str(tmp_path / "s")], check=True, capture_output=True, text=True).stdout.split()] == want


def test_relative_buckets():
    b = ops.relative_buckets(32, 128)
    assert b.dtype == torch.int32 and b.shape == (257,)
    assert b[128] == 0 and b[127] == 1 and b[129] == 17 and b[128 - 7] == 7 and b[0] == 15 and b[256] == 31 and b[128 + 8] == 16 + 8
    behind, ahead = b[:129].flip(0), b[129:] - 16
    assert (behind[1:] >= behind[:-1]).all() and (behind[1:] == ahead).all()
    c = ops.relative_buckets(8, 16, bidirectional=False)
    assert (c[16:] == 0).all() and c[15] == 1 and c[0] == 7
    for bad in ((2, 10), (7, 10), (8, 2)):
        with pytest.raises(ValueError):
            ops.relative_buckets(*bad)


def _apart(*a, **k):
    try:
        ops._apart("out", *a, **k)
        return True
    except L.VitaHipError:
        return False


def test_outputs_apart_from_inputs():
    for x, i in ((torch.zeros(2, 5, 3, 4, 8), 2), (torch.zeros(2, 5, 4, 3, 8), 3), (torch.zeros(3, 1, 3, 4, 8), 2), (torch.zeros(1, 1, 3, 4, 8), 2)):
        q, k, v = x.unbind(i)                                         # slices of a packed projection, whole or by heads
        assert _apart(q, k, v) and _apart(k, q, v) and not _apart(q, q) and not _apart(q, k, q[..., :4, :]) and _apart(q, q, but=(q,))
        assert _apart(q, None, torch.zeros(2, 5, 4, 8), k[:0])
    x = torch.zeros(2, 5, 3, 4, 8)
    assert not _apart(x[:, :, 0], x[:, :, 0, 1:]) and _apart(x[:, :, 0, :2], x[:, :, 0, 2:]) and not _apart(x[:, 1:, 0], x[:, :-1, 0])
    assert not _apart(x[:, :, 0], x[:, :, 0, :2], but=(x[:, :, 0, :2],))
    z = torch.zeros(40, 64)
    assert _apart(z[:, :40], z[:, 40:]) and not _apart(z[:, :40], z[:, 39:]) and not _apart(z[1:], z[:-1]) and _apart(z[:20], z[20:])


def test_outputs_do_not_overlap_themselves():
    like = torch.zeros(1)
    for good in (torch.zeros(2, 5, 4, 8), torch.zeros(5, 2, 4, 8).transpose(0, 1), torch.zeros(2, 4, 5, 8).transpose(1, 2), torch.zeros(2, 5, 4, 3, 8)[:, :, :, 1]):
        assert ops._out(good, "out", (2, 5, 4, 8), like) is good
    for strides in ((40, 8, 8, 1), (160, 32, 4, 1), (160, 16, 8, 1), (0, 32, 8, 1), (160, 32, 8, 0), (640, 128, 16, 2)):
        with pytest.raises(L.VitaHipError, match="overlap"):
            ops._out(torch.zeros(4000).as_strided((2, 5, 4, 8), strides), "out", (2, 5, 4, 8), like)
