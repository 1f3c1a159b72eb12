"""The transformer blocks' operators on the GPU (ops.qk_norm_rope, ops.attention, ops.gated_linear and their backward passes) against
plain 64-bit forms, with the elementwise bounds of tests/block_ops_reference.py; the calls as a run, on other streams and in graphs."""
import math

import pytest
import torch

import block_ops_reference as ref
from vita_amd import _lib as L
from vita_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
TYPES = [torch.float32, torch.bfloat16]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _randn(g, *shape, scale=1.0, dtype=torch.float32):
    return (torch.randn(*shape, generator=g) * scale).to(dtype).to(DEV)


# ---- norms + rotation -----------------------------------------------------------------------------------------------------------
def _norm_rope_case(g, B, S, H, Hk, D, dtype, norm, dealt, bias=True, T=None, packed=True):
    if packed:
        qkv = _randn(g, B, S, H + 2 * Hk, D, dtype=dtype)
        q, k = qkv[:, :, :H], qkv[:, :, H:H + Hk]
    else:
        q, k = _randn(g, B, S, H, D, dtype=dtype), _randn(g, B, S, Hk, D, dtype=dtype)
    p = {n: (1 if n.endswith("weight") else 0) + _randn(g, D, scale=0.3) for n in ("q_weight", "q_bias", "k_weight", "k_bias")}
    if not bias:
        p["q_bias"] = p["k_bias"] = None
    rope = ref.rope_table(T or S, H if dealt else 1, D).to(DEV)
    return q, k, rope, p, dict(norm=norm)


def _check_norm_rope(q, k, rope, p, kw, positions=None, eps=1e-5, g=None):
    qo, ko = ops.qk_norm_rope(q, k, rope, positions=positions, eps=eps, **p, **kw)
    dq, dk = _randn(g, *q.shape, dtype=q.dtype), _randn(g, *k.shape, dtype=q.dtype)
    grads = ops.qk_norm_rope_bwd(dq, dk, q, k, rope, positions=positions, eps=eps, **p, **kw)
    for n, x, y, dy, dx, dw, db in (("q", q, qo, dq, grads[0], grads[2], grads[3]), ("k", k, ko, dk, grads[1], grads[4], grads[5])):
        r = ref.norm_rope(x, rope, p[n + "_weight"], p[n + "_bias"], kw["norm"], eps, positions, dy)
        ref.assert_close(y, r[0], r[1], n)
        ref.assert_close(dx, r[2], r[3], "d" + n)
        for got, want, bound, what in ((dw, r[4], r[5], "weight"), (db, r[6], r[7], "bias")):
            if p[f"{n}_{what}"] is None:
                assert got is None
            else:
                ref.assert_close(got, want, bound, f"d{n}_{what}")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("norm", ["layer", "rms"])
@pytest.mark.parametrize("B,S,H,Hk,D,dealt", [(1, 1, 1, 1, 2, False), (3, 17, 8, 8, 64, True), (2, 5, 6, 2, 24, False), (1, 129, 4, 1, 128, False),
                                              (2, 3, 3, 3, 10, True), (1, 7, 2, 2, 256, False), (25, 1, 4, 2, 72, False), (2, 33, 5, 5, 30, False)])
def test_norm_rope(dtype, norm, B, S, H, Hk, D, dealt):
    g = _gen(B * 1000 + S * 10 + D)
    q, k, rope, p, kw = _norm_rope_case(g, B, S, H, Hk, D, dtype, norm, dealt, bias=norm == "layer")
    _check_norm_rope(q, k, rope, p, kw, g=g)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_positions(dtype):
    g = _gen(3)
    q, k, rope, p, kw = _norm_rope_case(g, 4, 6, 4, 2, 32, dtype, "layer", False, T=50)
    _check_norm_rope(q, k, rope, p, kw, positions=torch.randint(0, 50, (4, 6), generator=g).to(DEV), g=g)       # each token anywhere, twice the same too
    _check_norm_rope(q, k, rope, p, kw, positions=torch.randint(0, 50, (6,), generator=g).to(DEV), g=g)
    _check_norm_rope(q, k, rope, p, kw, positions=torch.randint(0, 50, (1, 6), generator=g).to(DEV).expand(4, 6), g=g)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_position_outside_the_table_is_nan(dtype):
    g = _gen(4)
    q, k, rope, p, kw = _norm_rope_case(g, 2, 4, 2, 2, 16, dtype, "layer", False)
    pos = torch.tensor([[0, 1, 4, 3], [-1, 1, 2, 3]], device=DEV)
    qo, ko = ops.qk_norm_rope(q, k, rope, positions=pos, **p, **kw)
    bad = torch.tensor([[0, 0, 1, 0], [1, 0, 0, 0]], dtype=torch.bool, device=DEV)
    for y in (qo, ko):
        assert torch.equal(torch.isnan(y).all(-1).all(-1), bad) and torch.equal(torch.isnan(y).any(-1).any(-1), bad)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_rope_layouts_and_in_place(dtype):
    g = _gen(5)
    q, k, rope, p, kw = _norm_rope_case(g, 2, 9, 4, 2, 40, dtype, "rms", False, bias=False)
    want = ops.qk_norm_rope(q.contiguous(), k.contiguous(), rope, **p, **kw)
    for a, b in ((q.transpose(1, 2).contiguous().transpose(1, 2), k.transpose(0, 1).contiguous().transpose(0, 1)),     # head-major, token-major
                 (q.transpose(2, 3).contiguous().transpose(2, 3), k)):                                                  # head dimension not contiguous
        got = ops.qk_norm_rope(a, b, rope, **p, **kw)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    odd = torch.zeros(2 * 9 * 4 * 40 + 1, dtype=dtype, device=DEV)[1:].view(2, 9, 4, 40).copy_(q)                       # rows off the 16-byte borders
    assert torch.equal(ops.qk_norm_rope(odd, k, rope, **p, **kw)[0], want[0])
    a, b = q.contiguous().clone(), k.contiguous().clone()
    got = ops.qk_norm_rope(a, b, rope, out=(a, b), **p, **kw)
    assert got[0] is a and torch.equal(a, want[0]) and torch.equal(b, want[1])
    dq, dk = _randn(g, *q.shape, dtype=dtype), _randn(g, *k.shape, dtype=dtype)
    plain = ops.qk_norm_rope_bwd(dq, dk, q, k, rope, **p, **kw)
    here = ops.qk_norm_rope_bwd(dq, dk, q, k, rope, out=(dq, dk), **p, **kw)
    assert all(x is None and y is None or torch.equal(x, y) for x, y in zip(plain, here))


def test_norm_rope_same_bits_every_time():
    g = _gen(6)
    q, k, rope, p, kw = _norm_rope_case(g, 7, 300, 8, 8, 64, torch.float32, "layer", True)
    dq, dk = _randn(g, *q.shape), _randn(g, *k.shape)
    a = ops.qk_norm_rope_bwd(dq, dk, q, k, rope, **p, **kw)
    for _ in range(3):
        assert all(torch.equal(x, y) for x, y in zip(a, ops.qk_norm_rope_bwd(dq, dk, q, k, rope, **p, **kw)))


def test_norm_rope_offsets_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 20 GiB of GPU memory")
    far = (1 << 32) + 64                                              # elements between the two batch rows
    g = _gen(7)
    buf = torch.zeros(far + 4096, dtype=torch.bfloat16, device=DEV)
    q = buf.as_strided((2, 3, 2, 32), (far, 64, 32, 1))
    q.copy_(_randn(g, 2, 3, 2, 32, dtype=torch.bfloat16))
    rope = ref.rope_table(3, 1, 32).to(DEV)
    near = q.contiguous().clone()
    got = ops.qk_norm_rope(q, near, rope, out=(q, torch.empty_like(near)))                   # the far one in place
    assert torch.equal(got[0], got[1])
    d = _randn(g, 2, 3, 2, 32, dtype=torch.bfloat16)
    a, b = ops.qk_norm_rope_bwd(d, d, q, got[1], rope)[:2]
    assert torch.equal(a, b)


# ---- attention ------------------------------------------------------------------------------------------------------------------
def _attention_case(g, B, Sq, Sk, H, Hk, D, dtype, pad, R, nb=16):
    q, k, v = _randn(g, B, Sq, H, D, dtype=dtype), _randn(g, B, Sk, Hk, D, dtype=dtype), _randn(g, B, Sk, Hk, D, dtype=dtype)
    kw = {}
    if pad is not None:
        m = torch.rand(B, Sk, generator=g) < pad
        if B > 1:
            m[B // 2] = True                                          # a row of the batch without any key
        kw["key_pad"] = m.to(DEV)
    if R is not None:
        kw["table"] = _randn(g, nb, H, dtype=dtype)
        kw["buckets"] = torch.randint(0, nb, (2 * R + 1,), generator=g, dtype=torch.int32).to(DEV)
    return q, k, v, kw


def _lse(stats):
    """log sum exp in 64 bits from the row statistics: m ln 2 - ln r, -inf for a row without keys."""
    m, r = stats[..., 0].double().cpu(), stats[..., 1].double().cpu()
    return torch.where(r == 0, -math.inf, m * math.log(2) - torch.log(torch.where(r == 0, 1.0, r)))


def _check_attention(q, k, v, kw, g, names=("o", "lse", "dq", "dk", "dv", "dtable")):
    o, stats = ops.attention(q, k, v, need_lse=True, **kw)
    do = _randn(g, *q.shape, dtype=q.dtype)
    got = (o, _lse(stats), *ops.attention_bwd(do, q, k, v, o, stats, **kw))
    want = ref.attention(q, k, v, do=do, **kw)
    for i, n in enumerate(names):
        if n == "-":
            continue
        if n == "dtable" and "table" not in kw:
            assert got[i] is None
            continue
        ref.assert_close(got[i], want[2 * i], want[2 * i + 1], n)


# (B, Sq, Sk, H, Hk, D): one token, tiles' borders, odd lengths, shared key heads, fewer and more queries than keys
SHAPES = [(1, 1, 1, 1, 1, 8), (2, 17, 17, 8, 8, 64), (3, 1, 40, 4, 2, 32), (2, 1, 333, 8, 2, 64), (1, 33, 65, 2, 1, 24), (2, 64, 64, 2, 2, 40),
          (1, 129, 130, 2, 2, 128), (1, 31, 257, 4, 1, 96), (1, 150, 70, 2, 2, 72), (1, 97, 97, 3, 3, 104), (5, 16, 16, 4, 4, 32), (1, 5, 200, 24, 2, 16)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention(dtype, causal, shape):
    g = _gen(sum(shape))
    q, k, v, kw = _attention_case(g, *shape, dtype, None, None)
    _check_attention(q, k, v, dict(kw, causal=causal), g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("causal", [False, True])
@pytest.mark.parametrize("pad,R", [(0.3, None), (None, 5), (0.5, 0), (0.9, 40)])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_attention_masks_and_bias(dtype, causal, pad, R, shape):
    g = _gen(sum(shape) + 7)
    q, k, v, kw = _attention_case(g, *shape, dtype, pad, R)
    _check_attention(q, k, v, dict(kw, causal=causal, scale=0.7 / math.sqrt(shape[-1])), g)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_padded_keys_may_hold_anything(dtype):
    g = _gen(11)
    for Sq, Sk, H, Hk in ((1, 300, 4, 2), (40, 150, 2, 2), (17, 17, 4, 4)):
        q, k, v, kw = _attention_case(g, 3, Sq, Sk, H, Hk, 32, dtype, 0.4, 9)
        o, lse = ops.attention(q, k, v, need_lse=True, **kw)
        do = _randn(g, *q.shape, dtype=dtype)
        want = (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, **kw))
        bad = kw["key_pad"][..., None, None]
        for junk in (math.nan, math.inf, -math.inf):
            k2, v2 = torch.where(bad, junk, k), torch.where(bad, junk, v)
            o, lse = ops.attention(q, k2, v2, need_lse=True, **kw)
            got = (o, lse, *ops.attention_bwd(do, q, k2, v2, o, lse, **kw))
            assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert (want[0][1] == 0).all() and (want[1][1] == 0).all() and all((t[1] == 0).all() for t in want[2:5])


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_far_tiles_of_the_bias(dtype):
    """Distances on both sides far outside the radius, so that whole tiles share one bucket, and with a small radius inside one tile."""
    g = _gen(12)
    for R in (1, 33, 128):
        q, k, v, kw = _attention_case(g, 1, 400, 400, 2, 1, 16, dtype, None, R, nb=7)
        _check_attention(q, k, v, kw, g)
        _check_attention(q, k, v, dict(kw, causal=True), g)
        q, k, v, kw = _attention_case(g, 2, 1, 700, 2, 1, 16, dtype, 0.2, R, nb=7)
        _check_attention(q, k, v, kw, g)


def test_attention_bucket_outside_the_table_is_nan():
    g = _gen(13)
    q, k, v, kw = _attention_case(g, 1, 4, 4, 2, 2, 16, torch.float32, None, 3, nb=4)
    kw["buckets"][3] = 4                                              # distance 0
    assert torch.isnan(ops.attention(q, k, v, **kw)).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_large_scores(dtype):
    """Scores of several hundred: the running maximum has to carry every tile, early ones outweighed by later ones and the other way."""
    g = _gen(14)
    q, k, v, kw = _attention_case(g, 1, 40, 500, 2, 2, 32, dtype, None, None)
    ramp = torch.linspace(-3, 3, 500, device=DEV)[None, :, None, None]
    for kk in (k * 6, (q.float().mean() + ramp * 4).to(dtype).expand_as(k).contiguous(), (-ramp * 4).to(dtype).expand_as(k).contiguous()):
        _check_attention(q * 4, kk, v, {}, g)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("low", ["lowest", "-inf"])
def test_attention_masks_in_the_table(dtype, low):
    """Buckets that hide their keys: by the type's lowest value (a row with nothing else averages its keys, as the formula does) and by
    -inf (such a row gives zeros), for whole tiles and inside them."""
    g = _gen(19)
    for Sq, Sk, R in ((40, 300, 3), (1, 300, 20), (150, 150, 60), (17, 17, 16)):
        q, k, v, kw = _attention_case(g, 2, Sq, Sk, 2, 1, 32, dtype, None, R, nb=4)
        value = torch.finfo(dtype).min if low == "lowest" else -math.inf
        for hidden in ([1], [0, 1, 2], [0, 1, 2, 3]):
            table = kw["table"].clone()
            table[hidden] = value
            _check_attention(q, k, v, dict(kw, table=table), g, names=("o", "-", "dq", "dk", "dv", "dtable"))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_layouts(dtype):
    g = _gen(15)
    for B, Sq, Sk, H, Hk in ((2, 40, 70, 4, 2), (3, 1, 200, 4, 2), (2, 17, 17, 2, 2)):
        q, k, v, kw = _attention_case(g, B, Sq, Sk, H, Hk, 24, dtype, 0.3, 6)
        o, lse = ops.attention(q, k, v, need_lse=True, **kw)
        do = _randn(g, *q.shape, dtype=dtype)
        want = (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, **kw))
        head_major = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)                # noqa: E731
        off = lambda t: torch.zeros(t.numel() + 3, dtype=dtype, device=DEV)[3:].view(t.shape).copy_(t)   # noqa: E731
        kv = torch.stack([k, v], 2)                                                          # (B, Sk, 2, Hk, D)
        for a, b, c in ((head_major(q), head_major(k), head_major(v)), (q, kv[:, :, 0], kv[:, :, 1]), (off(q), off(k), off(v)),
                        (q.transpose(2, 3).contiguous().transpose(2, 3), k, v)):
            out = head_major(torch.empty_like(q))
            assert ops.attention(a, b, c, out=out, need_lse=True, **kw)[0] is out
            grads = (torch.full_like(kv, 7.0), head_major(torch.empty_like(q)))
            got = (out, lse, *ops.attention_bwd(do, a, b, c, out, lse, out=(grads[1], grads[0][:, :, 0], grads[0][:, :, 1]), **kw))
            assert all(torch.equal(x, y) for x, y in zip(got, want))
        wide = torch.zeros(B, 2 * Sk, dtype=torch.bool, device=DEV)
        wide[:, :Sk] = kw["key_pad"]
        plain = ops.attention(q, k, v, **kw)
        assert torch.equal(ops.attention(q, k, v, **dict(kw, key_pad=wide[:, :Sk])), plain)
        assert torch.equal(ops.attention(q, k, v, **dict(kw, key_pad=kw["key_pad"].to(torch.uint8) * 200)), plain)
        ref_o = ref.attention(q, k, v, **kw)
        ref.assert_close(plain, ref_o[0], ref_o[1], "without statistics")
        one = kw["key_pad"][:1].expand(B, Sk)                                                # one mask for the batch
        assert torch.equal(ops.attention(q, k, v, **dict(kw, key_pad=one)), ops.attention(q, k, v, **dict(kw, key_pad=one.contiguous())))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_no_keys_no_queries(dtype):
    g = _gen(16)
    q, k, v, kw = _attention_case(g, 2, 3, 0, 2, 2, 16, dtype, None, 2)
    o, lse = ops.attention(q, k, v, need_lse=True, **kw)
    assert (o == 0).all() and (lse == 0).all()
    assert all((t == 0).all() for t in ops.attention_bwd(o, q, k, v, o, lse, **kw))
    o, lse = ops.attention(k, q, q, need_lse=True, **kw)
    assert o.shape == k.shape and lse.numel() == 0
    assert all((t == 0).all() for t in ops.attention_bwd(o, k, q, q, o, lse, **kw))


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_same_bits_every_time(dtype):
    g = _gen(17)
    q, k, v, kw = _attention_case(g, 3, 200, 333, 4, 2, 64, dtype, 0.2, 20)
    do = _randn(g, *q.shape, dtype=dtype)
    first = None
    for _ in range(3):
        o, lse = ops.attention(q, k, v, need_lse=True, **kw)
        got = (o, lse, *ops.attention_bwd(do, q, k, v, o, lse, **kw))
        first = first or got
        assert all(torch.equal(a, b) for a, b in zip(first, got))


def test_attention_offsets_past_32_bits():
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 30 GiB of GPU memory")
    far = (1 << 32) + 128                                             # elements between the batch rows of a long cache
    g = _gen(18)
    buf = torch.zeros(far + (1 << 16), dtype=torch.bfloat16, device=DEV)
    view = lambda off: buf.as_strided((2, 200, 2, 32), (far, 128, 32, 1), off)               # noqa: E731
    k, v = view(0), view(64)
    k.copy_(_randn(g, 2, 200, 2, 32, dtype=torch.bfloat16))
    v.copy_(_randn(g, 2, 200, 2, 32, dtype=torch.bfloat16))
    for Sq in (1, 40):
        q = _randn(g, 2, Sq, 4, 32, dtype=torch.bfloat16)
        do = _randn(g, *q.shape, dtype=torch.bfloat16)
        res = []
        for a, b in ((k, v), (k.contiguous(), v.contiguous())):
            o, lse = ops.attention(q, a, b, need_lse=True)
            res.append((o, lse, *ops.attention_bwd(do, q, a, b, o, lse)[:3]))
        assert all(torch.equal(x, y) for x, y in zip(*res))


# ---- gated feed-forward product ---------------------------------------------------------------------------------------------------
def _gated_case(g, M, K, F, dtype, bias):
    x, w = _randn(g, M, K, dtype=dtype), _randn(g, 2 * F, K, scale=K ** -0.5, dtype=dtype)
    return x, w, _randn(g, 2 * F, scale=0.5) if bias else None


def _check_gated(x, w, b, act, g):
    h, saved = ops.gated_linear(x, w, b, act, need_saved=True)
    dh = _randn(g, *h.shape, dtype=x.dtype)
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, b, act, saved)
    r = ref.gated(x, w, b, act, dh)
    ref.assert_close(h, r[0], r[1], "h")
    ref.assert_close(dx, r[2], r[3], "dx")
    ref.assert_close(dw, r[4], r[5], "dw")
    if b is None:
        assert db is None
    else:
        ref.assert_close(db, r[6], r[7], "db")
    assert torch.equal(ops.gated_linear(x, w, b, act), h)
    again = ops.gated_linear_bwd(dh, x, w, b, act, saved)
    assert torch.equal(dx, again[0]) and torch.equal(dw, again[1]) and (db is None or torch.equal(db, again[2]))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("M,K,F", [(1, 8, 8), (1, 512, 64), (5, 64, 200), (17, 40, 24), (25, 512, 136), (33, 72, 72), (64, 128, 128), (129, 200, 264), (300, 96, 520)])
def test_gated(dtype, M, K, F):
    g = _gen(M + K + F)
    _check_gated(*_gated_case(g, M, K, F, dtype, True), "silu", g)
    _check_gated(*_gated_case(g, M, K, F, dtype, False), "gelu_tanh", g)


@pytest.mark.parametrize("M,K,F,act", [(2049, 72, 2816, "silu"), (2300, 40, 2568, "gelu_tanh"), (2100, 264, 2720, "mish"),       # the product's tiles fill the chip
                                       (12289, 1000, 40, "silu"),                                                             # dx's do
                                       (40, 1000, 6152, "gelu"), (77, 1032, 6400, "silu")])                                   # dw's do
def test_gated_wide(M, K, F, act):
    g = _gen(M + F)
    _check_gated(*_gated_case(g, M, K, F, torch.bfloat16, M != 2300), act, g)


@pytest.mark.parametrize("M,K,F", [(1, 8, 8), (2, 48, 88), (34, 48, 96), (64, 128, 1024)])
def test_gated_few_rows_gradients(M, K, F):
    """bf16: dz reaches dx and dw nearly whole, what is left is their own rounding."""
    g = _gen(M + K)
    x, w, b = _gated_case(g, M, K, F, torch.bfloat16, True)
    dh = _randn(g, M, F, dtype=torch.bfloat16)
    dx, dw, db = ops.gated_linear_bwd(dh, x, w, b, "silu")
    r = ref.gated(x, w, b, "silu", dh, parts=2)
    ref.assert_close(dx, r[2], r[3], "dx")
    ref.assert_close(dw, r[4], r[5], "dw")
    ref.assert_close(db, r[6], r[7], "db")


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["relu", "gelu", "gelu_tanh", "silu", "mish"])
def test_gated_activations(dtype, act):
    g = _gen(21)
    x, w, b = _gated_case(g, 70, 64, 48, dtype, True)
    if act == "relu":                                                 # keep the gate away from the corner, where an error of z flips the slope
        gate = (x.double() @ w[:48].double().t() + b[:48].double()).abs().amin(0)
        w, b = w.clone(), b.clone()
        b[:48] += torch.where(gate < 1e-3, 20.0, 0.0)
    _check_gated(x, w, b, act, g)
    _check_gated(x * 20, w, b, "silu" if act == "relu" else act, g)   # far into both tails


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_layouts_and_parts(dtype):
    g = _gen(22)
    x, w, b = _gated_case(g, 37, 48, 40, dtype, True)
    h, saved = ops.gated_linear(x, w, b, "silu", need_saved=True)
    dh = _randn(g, *h.shape, dtype=dtype)
    want = ops.gated_linear_bwd(dh, x, w, b, "silu", saved)
    wide = torch.full((37, 64), 5.0, dtype=dtype, device=DEV)
    wide[:, 8:56] = x
    off = torch.zeros(x.numel() + 1, dtype=dtype, device=DEV)[1:].view(x.shape).copy_(x)
    for a, ww in ((wide[:, 8:56], w), (off, w), (x.t().contiguous().t(), w.t().contiguous().t()), (x[:1].expand(37, 48), w)):
        out = torch.full((37, 48), 3.0, dtype=dtype, device=DEV)
        got = ops.gated_linear(a, ww, b, "silu", out=out[:, :40])
        assert torch.equal(got, h) if a.stride(0) else torch.equal(got, h[:1].expand(37, 40))
        assert (out[:, 40:] == 3).all()
        if a.stride(0):
            assert all(torch.equal(p, q) for p, q in zip(ops.gated_linear_bwd(dh, a, ww, b, "silu", saved), want))
    part = ops.gated_linear_bwd(dh, x, w, b, "silu", saved, need_dx=False, need_db=False)
    assert part[0] is None and part[2] is None and torch.equal(part[1], want[1])
    part = ops.gated_linear_bwd(dh, x, w, b, "silu", saved, need_dw=False)
    assert part[1] is None and torch.equal(part[0], want[0]) and torch.equal(part[2], want[2])
    empty = ops.gated_linear_bwd(dh[:0], x[:0], w, b, "silu", saved[:0] if saved is not None else None)
    assert empty[0].shape == (0, 48) and (empty[1] == 0).all() and (empty[2] == 0).all()


# ---- together ---------------------------------------------------------------------------------------------------------------------
def _block(qkv, wts, rope, table, buckets, key_pad, w1, b1, w2):
    """norms + rotation, attention with the bias, gated feed-forward: as a block runs them."""
    B, S, n, D = qkv.shape
    H = n // 3
    q, k = ops.qk_norm_rope(qkv[:, :, :H], qkv[:, :, H:2 * H], rope, **wts)
    o = ops.attention(q, k, qkv[:, :, 2 * H:], table=table, buckets=buckets, key_pad=key_pad)
    return ops.gated_linear(o.reshape(B * S, H * D), w1, b1, "gelu_tanh") @ w2


def _block_inputs(g, B, S, H, D, F):
    wts = {n: (1 if n.endswith("weight") else 0) + _randn(g, D, scale=0.2) for n in ("q_weight", "q_bias", "k_weight", "k_bias")}
    pad = torch.zeros(B, S, dtype=torch.bool, device=DEV)
    pad[0, S // 2:] = True
    return (_randn(g, B, S, 3 * H, D), wts, ref.rope_table(S, H, D).to(DEV), _randn(g, 8, H), ops.relative_buckets(8, 12, device=DEV), pad,
            _randn(g, 2 * F, H * D, scale=(H * D) ** -0.5), _randn(g, 2 * F, scale=0.1), _randn(g, F, H * D, scale=F ** -0.5))


def test_block_gradients_against_differences():
    """The gradients that autograd carries through the run against central differences, in 64 bits, of its plain form."""
    g = _gen(31)
    args = _block_inputs(g, 2, 9, 2, 16, 24)
    qkv, wts, rope, table, buckets, pad, w1, b1, w2 = args
    leaves = [qkv, *wts.values(), table, w1, b1]
    leaves = [t.clone().requires_grad_() for t in leaves]
    out = _block(leaves[0], dict(zip(wts, leaves[1:5])), rope, leaves[5], buckets, pad, leaves[6], leaves[7], w2)
    head = _randn(g, *out.shape)
    out.backward(head)

    buckets, rope = args[4], args[2]

    def plain(x):
        qkv, qw, qb, kw_, kb, table, w1, b1 = x
        q, k = (ref.norm_rope(qkv_, rope, w, b, "layer", 1e-5, None)[0] for qkv_, w, b in ((qkv[:, :, :2], qw, qb), (qkv[:, :, 2:4], kw_, kb)))
        o = _attention64(q, k, qkv[:, :, 4:], table, buckets.cpu().long(), pad.cpu())
        z = o.reshape(18, 32) @ w1.t() + b1
        a, _ = ref.act_and_slope(z[:, :24], "gelu_tanh")
        return ((a * z[:, 24:]) @ w2.double().cpu() * head.double().cpu()).sum()

    x = [t.detach().double().cpu() for t in leaves]
    for i, t in enumerate(x):
        d = torch.randn(t.shape, generator=g, dtype=torch.float64)
        step = 1e-5
        hi, lo = (plain([y + s * step * d if j == i else y for j, y in enumerate(x)]) for s in (1, -1))
        want = ((hi - lo) / (2 * step)).item()
        got = (leaves[i].grad.double().cpu() * d).sum().item()
        # fp32 through three operators of at most 32-long sums: 1e-4 of the terms' size, far over (n + 2) u of each
        assert abs(got - want) <= 1e-4 * (leaves[i].grad.double().cpu() * d).abs().sum().item() + 1e-6, i


def _attention64(q, k, v, table, buckets, pad):
    B, S, H, D = q.shape
    s = torch.einsum("bihd,bjhd->bhij", q, k) * D ** -0.5
    R = buckets.numel() // 2
    dist = (torch.arange(S)[None] - torch.arange(S)[:, None]).clamp(-R, R) + R
    s = (s + table[buckets[dist]].permute(2, 0, 1)).masked_fill(pad[:, None, None], -math.inf)
    return torch.einsum("bhij,bjhd->bihd", torch.softmax(s, -1), v)


def test_block_on_another_stream_and_in_a_graph():
    g = _gen(32)
    args = list(_block_inputs(g, 3, 17, 4, 32, 64))
    want = _block(*args)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _block(*args)
    side.synchronize()
    assert torch.equal(got, want)

    def step(qkv, do, dh):
        q, k = ops.qk_norm_rope(qkv[:, :, :4], qkv[:, :, 4:8], args[2], **args[1])
        kw = dict(table=args[3], buckets=args[4], key_pad=args[5])
        o, lse = ops.attention(q, k, qkv[:, :, 8:], need_lse=True, **kw)
        x = o.view(51, 128)
        h, z = ops.gated_linear(x, args[6], args[7], "silu", need_saved=True)
        dx, dw, db = ops.gated_linear_bwd(dh, x, args[6], args[7], "silu", z)
        dq, dk, dv, dt = ops.attention_bwd(dx.view_as(o), q, k, qkv[:, :, 8:], o, lse, **kw)
        return (h, dx, dw, db, dv, dt, *ops.qk_norm_rope_bwd(dq, dk, qkv[:, :, :4], qkv[:, :, 4:8], args[2], **args[1]))

    static = [args[0].clone(), None, _randn(g, 51, 64)]
    graphs = []
    with torch.cuda.stream(side):
        step(*static)
        side.synchronize()
        for _ in range(2):                                            # two graphs of the same calls, replayed beside each other
            gr = torch.cuda.CUDAGraph()
            with torch.cuda.graph(gr, stream=side):
                res = step(*static)
            graphs.append((gr, res))
    torch.cuda.synchronize()
    for i in range(4):
        static[0].copy_(_randn(g, 3, 17, 12, 32))
        static[2].copy_(_randn(g, 51, 64))
        want = step(*static)                                          # eager work between the replays
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for s, (gr, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                gr.replay()
        torch.cuda.synchronize()
        for _, res in graphs:
            assert all(torch.equal(a, b) for a, b in zip(res, want)), i


def test_autograd_gives_the_backward_calls_results():
    g = _gen(33)
    q, k, v, kw = _attention_case(g, 2, 19, 19, 2, 1, 16, torch.bfloat16, 0.2, 4)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, kw["table"])]
    o = ops.attention(*leaves[:3], table=leaves[3], buckets=kw["buckets"], key_pad=kw["key_pad"])
    do = _randn(g, *o.shape, dtype=o.dtype)
    o.backward(do)
    o2, lse = ops.attention(q, k, v, need_lse=True, **kw)
    for t, d in zip(leaves, ops.attention_bwd(do, q, k, v, o2, lse, **kw)):
        assert torch.equal(t.grad, d)
    x, w, b = _gated_case(g, 9, 16, 16, torch.float32, True)
    leaves = [t.clone().requires_grad_() for t in (x, w, b)]
    h = ops.gated_linear(*leaves, "mish")
    dh = _randn(g, *h.shape)
    h.backward(dh.t().contiguous().t())                               # a gradient of another layout
    saved = ops.gated_linear(x, w, b, "mish", need_saved=True)[1]
    for t, d in zip(leaves, ops.gated_linear_bwd(dh, x, w, b, "mish", saved)):
        assert torch.equal(t.grad, d)
    with pytest.raises(L.VitaHipError, match="out="):
        ops.attention(q.clone().requires_grad_(), k, v, out=torch.empty_like(q))


def test_outputs_that_share_memory_are_refused():
    x = torch.zeros(2, 40, 3, 4, 16, device=DEV)
    q, k, v = x.unbind(2)
    rope = ref.rope_table(40, 1, 16).to(DEV)
    ops.qk_norm_rope(q, k, rope, out=(q, k))                          # in place in the packed projection
    o, stats = ops.attention(q, k, v, need_lse=True)
    d = torch.zeros_like(o)
    new = [torch.empty_like(o) for _ in range(3)]
    ops.attention_bwd(d, q, k, v, o, stats, out=new)
    for call in (lambda: ops.qk_norm_rope(q, k, rope, out=(k, q)), lambda: ops.qk_norm_rope(q, k, rope, out=(new[0], new[0])),
                 lambda: ops.qk_norm_rope_bwd(d, new[0], q, k, rope, out=(new[0], new[1])),
                 lambda: ops.attention(q, k, v, out=q), lambda: ops.attention(q, k, v, out=v),
                 lambda: ops.attention_bwd(d, q, k, v, o, stats, out=(new[0], new[1], new[1])),
                 lambda: ops.attention_bwd(d, q, k, v, o, stats, out=(d, new[1], new[2])),
                 lambda: ops.gated_linear(d.view(-1, 64)[:, :16], torch.zeros(32, 16, device=DEV), out=d.view(-1, 64)[:, 8:24])):
        with pytest.raises(L.VitaHipError, match="shares memory"):
            call()
