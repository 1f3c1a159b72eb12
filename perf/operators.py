"""The transformer block's operators, measured: norms of queries and keys with the rotation in the same pass, softmax attention with a
learned relative position bias by buckets, and the gated feed-forward product, each with its backward pass.

Sizes: the transformer action encoder (512 wide, 8 heads of 64, 17 tokens: a CLS token and 16 action steps; 128 rows a training batch,
25 rows when serving) and generic longer and wider ones.  A case's fields: `op`, `dtype` of activations, `train` (forward and backward)
and the operator's sizes."""
import math

import torch

own = False

DEV = "cuda"
DT = {"f32": torch.float32, "bf16": torch.bfloat16}


# ---- cases -------------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # norms of queries and keys + rotation
        # one new token for each of 25 environments, every row at a position of its own: latency
        dict(name="norm_rope_token_f32", op="norm_rope", dtype="f32", train=False, B=25, S=1, H=8, G=1, D=64, norm="layer", dealt=True, T=256),
        # a training batch of the transformer action encoder (LayerNorm over a head, rotation dealt to the heads in order)
        dict(name="norm_rope_encoder_train_f32", op="norm_rope", dtype="f32", train=True, B=128, S=17, H=8, G=1, D=64, norm="layer", dealt=True, T=17),
        # long sequences of odd length, 32 query heads over 8 key heads, root-mean-square norm: training, memory-bound
        dict(name="norm_rope_long_train_bf16", op="norm_rope", dtype="bf16", train=True, B=2, S=8191, H=32, G=4, D=128, norm="rms", dealt=False, T=8192),
        # attention
        # the encoder's 17 tokens when serving 25 rows: latency
        dict(name="attention_encoder_serve_f32", op="attention", dtype="f32", train=False, B=25, Sq=17, Sk=17, H=8, G=1, D=64, causal=False, pad=False, R=16, buckets=32),
        # a training batch of the encoder
        dict(name="attention_encoder_train_f32", op="attention", dtype="f32", train=True, B=128, Sq=17, Sk=17, H=8, G=1, D=64, causal=False, pad=True, R=16, buckets=32),
        # one new token a row over a long cache, 32 query heads over 8 key heads, rows of unequal length: memory-bound
        dict(name="attention_token_bf16", op="attention", dtype="bf16", train=False, B=25, Sq=1, Sk=4097, H=32, G=4, D=128, causal=True, pad=True, R=0, buckets=0),
        # mid-size training in 32 bits with padded rows and the bias: matrix-bound at the 32-bit rate
        dict(name="attention_mid_train_f32", op="attention", dtype="f32", train=True, B=4, Sq=1000, Sk=1000, H=8, G=1, D=64, causal=False, pad=True, R=128, buckets=32),
        # a long causal training sequence of odd length with the bias: matrix-bound
        dict(name="attention_long_train_bf16", op="attention", dtype="bf16", train=True, B=2, Sq=4095, Sk=4095, H=16, G=1, D=128, causal=True, pad=False, R=128, buckets=32),
        # gated feed-forward product
        # the encoder's feed-forward when serving 25 rows of one token
        dict(name="gated_token_f32", op="gated", dtype="f32", train=False, M=25, K=512, F=2048, act="gelu_tanh", bias=True),
        # the same for a wide bf16 block: bound by reading the weights once
        dict(name="gated_token_bf16", op="gated", dtype="bf16", train=False, M=25, K=2048, F=8192, act="silu", bias=False),
        # a training batch of the encoder: 128 x 17 tokens
        dict(name="gated_encoder_train_f32", op="gated", dtype="f32", train=True, M=2176, K=512, F=2048, act="gelu_tanh", bias=True),
        # a wide bf16 block in training, an odd number of tokens: the largest, matrix-bound
        dict(name="gated_wide_train_bf16", op="gated", dtype="bf16", train=True, M=8191, K=2048, F=8192, act="silu", bias=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm_rope", "attention", "attention", "gated"])
    dtype, train = rng.choice(["f32", "bf16"]), rng.random() < 0.5
    if op == "norm_rope":
        G, D = rng.choice([1, 1, 2, 4]), 8 * rng.randint(2, 16)
        H = G * rng.choice([1, 2, 3, 8])
        S = _log(rng, 1, 8192)
        B = _log(rng, 1, max(1, min(512, 67_000_000 // (S * H * D * (2 if dtype == "f32" else 1)))))
        return dict(op=op, dtype=dtype, train=train, B=B, S=S, H=H, G=G, D=D, norm=rng.choice(["layer", "rms"]), dealt=G == 1 and rng.random() < 0.5,
                    T=S + rng.randint(0, 64))
    if op == "attention":
        G, D = rng.choice([1, 1, 2, 4]), 8 * rng.randint(2, 16)
        H = G * rng.choice([1, 2, 3, 8])
        most = 100_000_000 if dtype == "f32" else 500_000_000
        kind = rng.choice(["token", "self", "self", "cross"])
        if kind == "token":
            Sq, Sk, train = 1, _log(rng, 1, 16384), False
        elif kind == "self":
            Sq = Sk = _log(rng, 1, 4095)
        else:
            Sk = _log(rng, 16, 4095)
            Sq = rng.randint(1, Sk)
        H = min(H, max(1, most // (Sq * Sk)) // G * G or G)
        B = _log(rng, 1, max(1, min(256, most // (Sq * Sk * H), 60_000_000 // (max(Sq, Sk) * H * D))))
        R = rng.choice([0, 16, 128])
        return dict(op=op, dtype=dtype, train=train, B=B, Sq=Sq, Sk=Sk, H=H, G=G, D=D, causal=rng.random() < 0.5, pad=rng.random() < 0.5, R=R,
                    buckets=32 if R else 0)
    K, F = 8 * _log(rng, 4, 256), 8 * _log(rng, 4, 1024)
    most = (137_000_000_000 if dtype == "bf16" else 9_000_000_000) // (K * F)
    return dict(op=op, dtype=dtype, train=train, M=_log(rng, 1, max(1, min(16384, most))), K=K, F=F, act=rng.choice(["gelu_tanh", "silu"]),
                bias=rng.random() < 0.5)


# ---- inputs ------------------------------------------------------------------------------------------------------------------
def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(int(seed))
    dt = DT[case["dtype"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(*shape, generator=g, device=DEV) * scale).to(dtype)

    s = {"case": case}
    if case["op"] == "norm_rope":
        B, S, H, D, T = case["B"], case["S"], case["H"], case["D"], case["T"]
        Hk = H // case["G"]
        qkv = normal(B, S, H + 2 * Hk, D)                       # what the projection writes: queries, keys and values of a token together
        s["q"], s["k"] = qkv[:, :, :H], qkv[:, :, H:H + Hk]
        for n in ("q", "k"):
            s[n + "_weight"] = 1.0 + normal(D, scale=0.1, dtype=torch.float32)
            s[n + "_bias"] = normal(D, scale=0.1, dtype=torch.float32) if case["norm"] == "layer" else None
        n = H * D if case["dealt"] else D                       # dealt: head h turns with frequencies h * D / 2 ... of the full width
        theta = 10000.0 ** (-torch.arange(0, n, 2, device=DEV, dtype=torch.float64) / n)
        angle = torch.arange(T, device=DEV, dtype=torch.float64)[:, None] * theta[None]
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float()
        s["positions"] = (torch.arange(S, device=DEV)[None] + torch.randint(0, T - S + 1, (B, 1), generator=g, device=DEV)) if T > S else None
        if case["train"]:
            s["dq"], s["dk"] = normal(B, S, H, D), normal(B, S, Hk, D)
    elif case["op"] == "attention":
        B, Sq, Sk, H, D = case["B"], case["Sq"], case["Sk"], case["H"], case["D"]
        Hk = H // case["G"]
        s["q"], s["k"], s["v"] = normal(B, Sq, H, D), normal(B, Sk, Hk, D), normal(B, Sk, Hk, D)
        s["table"] = s["buckets"] = s["key_pad"] = None
        if case["R"]:
            s["table"] = normal(case["buckets"], H)
            s["buckets"] = _log_buckets(case["R"], case["buckets"])
        if case["pad"]:
            length = torch.randint(1, Sk + 1, (B, 1), generator=g, device=DEV)
            if B > 2:
                length[B // 2] = 0                              # a row of the batch with no key at all
            s["key_pad"] = torch.arange(Sk, device=DEV)[None] >= length
        if case["train"]:
            s["do"] = normal(B, Sq, H, D)
    else:
        M, K, F = case["M"], case["K"], case["F"]
        s["x"] = normal(M, K)
        s["w"] = normal(2 * F, K, scale=K ** -0.5)              # rows 0 .. F - 1: gate, F .. 2 F - 1: up
        s["b"] = normal(2 * F, scale=0.1, dtype=torch.float32) if case["bias"] else None
        if case["train"]:
            s["dh"] = normal(M, F)
    return s


def _log_buckets(R, n):
    """Bucket of each distance -R .. R (key position - query position): half the buckets for keys behind, half for keys ahead; the first
    half of each exact, the rest in equal steps of the logarithm up to R."""
    d = torch.arange(-R, R + 1, dtype=torch.float64)
    half = n // 2
    exact = half // 2
    far = exact + (torch.log(d.abs().clamp(min=1) / exact) / math.log(R / exact) * (half - exact) + 1e-9).floor().clamp(max=half - exact - 1)
    return (torch.where(d.abs() < exact, d.abs(), far) + half * (d > 0)).to(torch.int32).to(DEV)


# ---- one pass ----------------------------------------------------------------------------------------------------------------
def run(s):
    c = s["case"]
    if own:
        from vita_amd import ops
        if c["op"] == "norm_rope":
            kw = dict(q_weight=s["q_weight"], q_bias=s["q_bias"], k_weight=s["k_weight"], k_bias=s["k_bias"], norm=c["norm"], positions=s["positions"])
            q, k = ops.qk_norm_rope(s["q"], s["k"], s["rope"], **kw)
            out = {"q": q, "k": k}
            if c["train"]:
                out["grads"] = ops.qk_norm_rope_bwd(s["dq"], s["dk"], s["q"], s["k"], s["rope"], **kw)
            return out
        if c["op"] == "attention":
            kw = dict(causal=c["causal"], key_pad=s["key_pad"], table=s["table"], buckets=s["buckets"])
            if not c["train"]:
                return {"o": ops.attention(s["q"], s["k"], s["v"], **kw)}
            o, lse = ops.attention(s["q"], s["k"], s["v"], need_lse=True, **kw)
            return {"o": o, "grads": ops.attention_bwd(s["do"], s["q"], s["k"], s["v"], o, lse, **kw)}
        if not c["train"]:
            return {"h": ops.gated_linear(s["x"], s["w"], s["b"], c["act"])}
        h, saved = ops.gated_linear(s["x"], s["w"], s["b"], c["act"], need_saved=True)
        return {"h": h, "grads": ops.gated_linear_bwd(s["dh"], s["x"], s["w"], s["b"], c["act"], saved)}
    return {"norm_rope": _norm_rope, "attention": _attention, "gated": _gated}[c["op"]](s, c)


# ---- plain forms -------------------------------------------------------------------------------------------------------------
EPS = 1e-5


def _turn(x, cos, sin):
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack([a * cos - b * sin, b * cos + a * sin], -1).flatten(-2)


def _rope_rows(s, c, heads):
    rope = s["rope"] if s["positions"] is None else s["rope"][s["positions"]]     # ([B,] S, F, 2)
    rope = rope[:c["S"]] if s["positions"] is None else rope
    rope = rope.unflatten(-2, (heads if c["dealt"] else 1, c["D"] // 2))
    return rope[..., 0], rope[..., 1]


def _normed(x, c):
    mean = x.mean(-1, keepdim=True) if c["norm"] == "layer" else 0.0
    r = ((x - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()
    return (x - mean) * r, r


def _norm_rope_one(s, c, n):
    x = s[n].float()
    cos, sin = _rope_rows(s, c, x.shape[2])
    y, r = _normed(x, c)
    w, b = s[n + "_weight"], s[n + "_bias"]
    out = _turn(y * w + b if b is not None else y * w, cos, sin).to(s[n].dtype)
    if not c["train"]:
        return out, ()
    d = _turn(s["d" + n].float(), cos, -sin)                    # the rotation's transpose
    e = d * w
    centre = e.mean(-1, keepdim=True) if c["norm"] == "layer" else 0.0
    dx = r * (e - centre - y * (e * y).mean(-1, keepdim=True))
    return out, (dx.to(s[n].dtype), (d * y).sum((0, 1, 2)), d.sum((0, 1, 2)) if b is not None else None)


def _norm_rope(s, c):
    q, gq = _norm_rope_one(s, c, "q")
    k, gk = _norm_rope_one(s, c, "k")
    out = {"q": q, "k": k}
    if c["train"]:
        out["grads"] = (gq[0], gk[0], gq[1], gq[2], gk[1], gk[2])
    return out


def _attention(s, c):
    B, Sq, Sk, H, G, D = c["B"], c["Sq"], c["Sk"], c["H"], c["G"], c["D"]
    dt, scale = s["q"].dtype, c["D"] ** -0.5
    q = s["q"].float().transpose(1, 2)                                            # (B, H, Sq, D)
    k, v = (s[n].float().transpose(1, 2).repeat_interleave(G, 1).contiguous() for n in ("k", "v"))
    p = torch.matmul(q, k.transpose(2, 3)) * scale
    dist = torch.arange(Sk, device=DEV)[None] - (torch.arange(Sq, device=DEV)[:, None] + (Sk - Sq))
    if s["table"] is not None:
        p += s["table"].float()[s["buckets"].long()[dist.clamp(-c["R"], c["R"]) + c["R"]]].permute(2, 0, 1)
    if c["causal"]:
        p.masked_fill_(dist > 0, -math.inf)
    if s["key_pad"] is not None:
        p.masked_fill_(s["key_pad"][:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = (p - torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    p /= torch.where(total == 0, 1.0, total)                                      # a row with no key gives zeros
    out = {"o": torch.matmul(p, v).transpose(1, 2).to(dt).contiguous()}
    if not c["train"]:
        return out
    do = s["do"].float().transpose(1, 2).contiguous()
    dv = torch.matmul(p.transpose(2, 3), do)
    ds = torch.matmul(do, v.transpose(2, 3))
    ds = p * (ds - (p * ds).sum(-1, keepdim=True))
    dq = torch.matmul(ds, k) * scale
    dk = torch.matmul(ds.transpose(2, 3), q.contiguous()) * scale
    dk, dv = (t.unflatten(1, (H // G, G)).sum(2).transpose(1, 2).to(dt).contiguous() for t in (dk, dv))
    dtable = None
    if s["table"] is not None:
        # sums along the diagonals: row i of the flipped matrix shifted right by i, then over rows; then into the buckets
        t = torch.nn.functional.pad(ds.sum(0).flip(1), (0, Sq)).flatten(1)[:, :Sq * (Sk + Sq - 1)].view(H, Sq, Sk + Sq - 1).sum(1)
        far = torch.arange(Sk + Sq - 1, device=DEV) - (Sq - 1) - (Sk - Sq)
        at = s["buckets"].long()[far.clamp(-c["R"], c["R"]) + c["R"]]
        dtable = torch.zeros(c["buckets"], H, dtype=torch.float64, device=DEV).index_add_(0, at, t.t().double()).to(dt)
    out["grads"] = (dq.transpose(1, 2).to(dt).contiguous(), dk, dv, dtable)
    return out


def _act(g, act):
    if act == "silu":
        sg = 1.0 / (1.0 + torch.exp(-g))
        return g * sg, sg * (1.0 + g * (1.0 - sg))
    inner = math.sqrt(2.0 / math.pi) * (g + 0.044715 * g * g * g)
    th = torch.tanh(inner)
    return 0.5 * g * (1.0 + th), 0.5 * (1.0 + th) + 0.5 * g * (1.0 - th * th) * math.sqrt(2.0 / math.pi) * (1.0 + 3 * 0.044715 * g * g)


def _gated(s, c):
    F, dt = c["F"], s["x"].dtype
    x, w = s["x"].float(), s["w"].float()
    z = torch.matmul(x, w.t())
    if s["b"] is not None:
        z = z + s["b"]
    a, da = _act(z[:, :F], c["act"])
    u = z[:, F:]
    out = {"h": (a * u).to(dt)}
    if c["train"]:
        dh = s["dh"].float()
        dz = torch.cat([dh * u * da, dh * a], 1)
        out["grads"] = (torch.matmul(dz, w).to(dt), torch.matmul(dz.t(), x).to(dt), dz.sum(0) if s["b"] is not None else None)
    return out


# ---- what a pass cannot do without ---------------------------------------------------------------------------------------------
def work(case):
    e = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "norm_rope":
        n = case["B"] * case["S"] * (case["H"] + case["H"] // case["G"]) * case["D"]
        rope = case["B"] * case["S"] * (case["H"] if case["dealt"] else 1) * case["D"] * 4 if case["T"] > case["S"] else case["S"] * case["D"] * 4
        return {"bytes": n * e * (5 if case["train"] else 2) + min(rope, case["T"] * case["D"] * 4 * (case["H"] if case["dealt"] else 1)),
                "flops": n * (20 if case["train"] else 8)}
    if case["op"] == "attention":
        B, Sq, Sk, H, G, D = (case[n] for n in ("B", "Sq", "Sk", "H", "G", "D"))
        pairs = Sq * Sk
        if case["causal"]:                                       # query i sees keys 0 .. i + Sk - Sq
            lo = max(0, Sk - Sq)
            first = max(0, Sq - Sk)
            rows = Sq - first
            pairs = rows * (lo + 1) + rows * (rows - 1) // 2
        if case["pad"]:
            pairs //= 2                                          # lengths are even over 1 .. Sk
        q, kv = B * Sq * H * D, B * Sk * (H // G) * D // (2 if case["pad"] else 1)
        both = 2 * B * H * pairs * D
        # forward: two products; backward: the gradients of the four operands of those two
        return {"bytes": e * ((2 * q + 2 * kv) + (4 * q + 4 * kv if case["train"] else 0)), "flops": both * (6 if case["train"] else 2)}
    M, K, F = case["M"], case["K"], case["F"]
    fwd = M * K + 2 * F * K + M * F
    bwd = M * F + M * K + 2 * F * K + M * K + 2 * F * K
    return {"bytes": e * (fwd + (bwd if case["train"] else 0)), "flops": 4 * M * F * K * (3 if case["train"] else 1)}


# ---- the definitions in 64 bits ------------------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    c = case

    def wide(t):
        return None if t is None else t.double()

    def norm_rope(n):
        x, w, b = wide(s[n]), wide(s[n + "_weight"]), wide(s[n + "_bias"])
        B, S, h, D = x.shape
        at = s["positions"] if s["positions"] is not None else torch.arange(S, device=DEV)[None].expand(B, S)
        turn = torch.view_as_complex(wide(s["rope"]))[at].view(B, S, -1, D // 2)
        mu = x.mean(-1, keepdim=True) if c["norm"] == "layer" else torch.zeros_like(x[..., :1])
        sd = torch.sqrt(((x - mu) ** 2).sum(-1, keepdim=True) / D + EPS)
        y = (x - mu) / sd
        t = y * w + (0 if b is None else b)
        out = torch.view_as_real(torch.view_as_complex(t.reshape(B, S, h, D // 2, 2)) * turn).reshape(B, S, h, D)
        if not c["train"]:
            return out, None
        d = torch.view_as_real(torch.view_as_complex(wide(s["d" + n]).reshape(B, S, h, D // 2, 2)) * turn.conj()).reshape(B, S, h, D)
        e = d * w
        proj = (e * y).sum(-1, keepdim=True) / D
        mid = e.sum(-1, keepdim=True) / D if c["norm"] == "layer" else 0
        return out, ((e - mid - y * proj) / sd, torch.einsum("bshd,bshd->d", d, y), None if b is None else d.sum((0, 1, 2)))

    if c["op"] == "norm_rope":
        (q, gq), (k, gk) = norm_rope("q"), norm_rope("k")
        out = {"q": q, "k": k}
        if c["train"]:
            out["grads"] = (gq[0], gk[0], gq[1], gq[2], gk[1], gk[2])
        return out
    if c["op"] == "attention":
        B, Sq, Sk, H, G, D, R = (c[n] for n in ("B", "Sq", "Sk", "H", "G", "D", "R"))
        if B * H > 4096:
            return None
        dist = torch.arange(Sk, device=DEV)[None] - torch.arange(Sk - Sq, Sk, device=DEV)[:, None]
        at = s["buckets"].long()[dist.clamp(-R, R) + R] if R else None
        o = torch.zeros(B, Sq, H, D, dtype=torch.float64, device=DEV)
        train = c["train"]
        dq, dk, dv = (torch.zeros(t.shape, dtype=torch.float64, device=DEV) for t in (s["q"], s["k"], s["v"])) if train else (None,) * 3
        dt = torch.zeros(c["buckets"], H, dtype=torch.float64, device=DEV) if train and R else None
        for h in range(H):
            per = torch.zeros(Sq, Sk, dtype=torch.float64, device=DEV) if dt is not None else None
            for b in range(B):
                q, k, v = wide(s["q"][b, :, h]), wide(s["k"][b, :, h // G]), wide(s["v"][b, :, h // G])
                sc = q @ k.t() / math.sqrt(D)
                if R:
                    sc = sc + wide(s["table"])[:, h][at]
                seen = torch.ones(Sq, Sk, dtype=torch.bool, device=DEV)
                if c["causal"]:
                    seen &= dist <= 0
                if s["key_pad"] is not None:
                    seen &= ~s["key_pad"][b][None]
                sc = torch.where(seen, sc, -math.inf)
                p = torch.softmax(sc, -1).nan_to_num(0.0)         # a row with no key: zeros
                o[b, :, h] = p @ v
                if train:
                    g = wide(s["do"][b, :, h])
                    dv[b, :, h // G] += p.t() @ g
                    dp = g @ v.t()
                    ds = p * (dp - (g * o[b, :, h]).sum(-1, keepdim=True))
                    dq[b, :, h] = ds @ k / math.sqrt(D)
                    dk[b, :, h // G] += ds.t() @ q / math.sqrt(D)
                    if per is not None:
                        per += ds
            if per is not None:
                dt[:, h] = torch.bincount(at.flatten(), weights=per.flatten(), minlength=c["buckets"])
        return {"o": o, "grads": (dq, dk, dv, dt)} if train else {"o": o}
    x, w, b = wide(s["x"]), wide(s["w"]), wide(s["b"])
    gate, up = (x @ half.t() for half in w.chunk(2))
    if b is not None:
        gate, up = gate + b[:c["F"]], up + b[c["F"]:]
    gate.requires_grad_(c["train"])
    if c["act"] == "silu":
        a = gate * torch.sigmoid(gate)
    else:
        a = 0.5 * gate * (1 + torch.tanh(math.sqrt(2 / math.pi) * (gate + 0.044715 * gate ** 3)))
    out = {"h": (a * up).detach()}
    if c["train"]:
        dh = wide(s["dh"])
        dg, = torch.autograd.grad(a, gate, dh * up)
        du = dh * a.detach()
        out["grads"] = (dg @ w[:c["F"]] + du @ w[c["F"]:], torch.cat([dg.t() @ x, du.t() @ x]), torch.cat([dg.sum(0), du.sum(0)]) if b is not None else None)
    return out
