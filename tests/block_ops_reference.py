"""Plain 64-bit forms of the transformer blocks' operators (ops.qk_norm_rope, ops.attention, ops.gated_linear) with their gradients, and
elementwise bounds on what fp32 arithmetic and the roundings to the call's type may add.

u = 2^-24 is fp32's half step, ut the half step of the call's type (2^-24 or 2^-8).  A sum of n products in fp32, in any order, is off by at
most (n + 2) u sum |a b|; exp2 / rcp / sqrt of the hardware are counted as 2 u each."""
import math

import torch

U = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def assert_close(got, want, bound, what=""):
    """|got - want| <= bound elementwise, with NaN and infinities at the same places."""
    got, want, bound = got.detach().double().cpu(), want.double().cpu(), bound.double().cpu()
    assert got.shape == want.shape, f"{what}: {tuple(got.shape)} against {tuple(want.shape)}"
    fine = torch.isfinite(want)
    assert torch.equal(torch.isnan(got), torch.isnan(want)), f"{what}: NaN at other places"
    off = (got - want).abs()[fine] - bound.expand_as(want)[fine]
    assert off.numel() == 0 or off.max().item() <= 0, f"{what}: {off.max().item():.3g} over the bound, which is {bound.expand_as(want)[fine].flatten()[off.argmax()].item():.3g}"


# ---- norms of queries and keys + rotation -------------------------------------------------------------------------------------
def rope_table(positions, heads, D, base=10000.0):
    n = heads * D
    theta = base ** (-torch.arange(0, n, 2, dtype=torch.float64) / n)
    a = torch.arange(positions, dtype=torch.float64)[:, None] * theta[None]
    return torch.stack([a.cos(), a.sin()], -1).float()


def norm_rope(x, rope, weight, bias, norm, eps, positions, dy=None):
    """One side.  Returns (y, bound_y) and, with dy, also (dx, bound, dw, bound, db, bound)."""
    ut = half_step(x.dtype)
    x64, rope = x.double().cpu(), rope.double().cpu()
    B, S, H, D = x64.shape
    at = positions.cpu().expand(B, S) if positions is not None else torch.arange(S).expand(B, S)
    cs = rope[at].view(B, S, -1, D // 2, 2)
    c, s = cs[..., 0], cs[..., 1]
    w = weight.double().cpu() if weight is not None else torch.ones(D, dtype=torch.float64)
    b = bias.double().cpu() if bias is not None else torch.zeros(D, dtype=torch.float64)
    mean = x64.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(x64[..., :1])
    xc = x64 - mean
    r = 1.0 / torch.sqrt((xc * xc).mean(-1, keepdim=True) + eps)
    n = xc * r
    # x - mean: the mean is off by (D + 2) u mean|x|; r by (D + 8) u and what the shifted mean adds to the variance (second order)
    en = (D + 4) * U * x64.abs().mean(-1, keepdim=True) * r * (1 if norm == "layer" else 0) + n.abs() * (D + 12) * U

    def turn(v, sign=1.0):
        p = v.unflatten(-1, (D // 2, 2))
        return torch.stack([p[..., 0] * c - sign * p[..., 1] * s, p[..., 1] * c + sign * p[..., 0] * s], -1).flatten(-2)

    def turn_abs(v):
        p = v.unflatten(-1, (D // 2, 2))
        return torch.stack([p[..., 0] * c.abs() + p[..., 1] * s.abs(), p[..., 1] * c.abs() + p[..., 0] * s.abs()], -1).flatten(-2)

    t = n * w + b
    y = turn(t)
    by = turn_abs(en * w.abs() + 2 * U * (t.abs() + (n * w).abs())) + 4 * U * turn_abs(t.abs()) + ut * y.abs()
    if dy is None:
        return y, by * (1 + 2 * ut)
    g = dy.double().cpu()
    d = turn(g, -1.0)
    ed = 3 * U * turn_abs(g.abs())
    e = d * w
    ee = ed * w.abs() + U * e.abs()
    em = e.mean(-1, keepdim=True) if norm == "layer" else torch.zeros_like(mean)
    proj = (e * n).mean(-1, keepdim=True)
    dx = r * (e - em - n * proj)
    mean_abs = e.abs().mean(-1, keepdim=True)
    proj_abs = (e * n).abs().mean(-1, keepdim=True)
    eproj = (ee * n.abs() + e.abs() * en).mean(-1, keepdim=True) + (D + 4) * U * proj_abs
    bdx = r * (ee + (ee.mean(-1, keepdim=True) + (D + 4) * U * mean_abs) + en * proj.abs() + n.abs() * eproj + 4 * U * (e.abs() + mean_abs + n.abs() * proj_abs)) \
        + (D + 12) * U * dx.abs() + ut * dx.abs()
    rows = B * S * H
    dw, db = (d * n).sum((0, 1, 2)), d.sum((0, 1, 2))
    bdw = (ed * n.abs() + d.abs() * en).sum((0, 1, 2)) + (rows + 2) * U * (d * n).abs().sum((0, 1, 2))
    bdb = ed.sum((0, 1, 2)) + (rows + 2) * U * d.abs().sum((0, 1, 2))
    return y, by * (1 + 2 * ut), dx, bdx * (1 + 2 * ut), dw, bdw, db, bdb


# ---- attention ----------------------------------------------------------------------------------------------------------------
def attention(q, k, v, scale=None, causal=False, key_pad=None, table=None, buckets=None, do=None):
    """(o, bound, lse, bound) and, with do, (dq, bound), (dk, bound), (dv, bound), (dtable, bound) behind them."""
    dt = q.dtype
    ut = half_step(dt)
    up = ut if dt == torch.bfloat16 else 0.0            # P and dS are rounded to bf16 for the products that read them
    q64, k64, v64 = (t.double().cpu().transpose(1, 2) for t in (q, k, v))
    B, H, Sq, D = q64.shape
    Hk, Sk = k64.shape[1], k64.shape[2]
    G = H // Hk
    scale = D ** -0.5 if scale is None else scale
    seen = torch.ones(B, 1, Sq, Sk, dtype=torch.bool)
    dist = torch.arange(Sk)[None] - (torch.arange(Sq)[:, None] + Sk - Sq)
    if causal:
        seen = seen & (dist <= 0)
    if key_pad is not None:
        pad = key_pad.cpu().bool()
        seen = seen & ~pad[:, None, None]
        k64, v64 = (torch.where(pad[:, None, :, None], 0.0, t) for t in (k64, v64))
    k64, v64 = k64.repeat_interleave(G, 1), v64.repeat_interleave(G, 1)
    s = q64 @ k64.transpose(2, 3) * scale
    es = (D + 4) * U * (q64.abs() @ k64.abs().transpose(2, 3)) * abs(scale)
    if table is not None:
        R = buckets.numel() // 2
        idx = buckets.cpu().long()[dist.clamp(-R, R) + R]
        bias = table.double().cpu()[idx].permute(2, 0, 1)
        s = s + bias
        es = es + 3 * U * (bias.abs() + s.abs())
    s = torch.where(seen, s, -math.inf)
    top = s.amax(-1, keepdim=True) if Sk else torch.full((B, H, Sq, 1), -math.inf, dtype=torch.float64)
    safe = torch.where(top == -math.inf, 0.0, top)
    p = torch.exp(s - safe)
    tot = p.sum(-1, keepdim=True)
    p = p / torch.where(tot == 0, 1.0, tot)
    lse = torch.where(tot == 0, -math.inf, safe + torch.log(torch.where(tot == 0, 1.0, tot)))[..., 0]
    # exponents are formed times log2 e: their argument is off by es and two roundings of its size; a probability relative to its sum
    ea = es.masked_fill(~seen.expand_as(es), 0.0) + 4 * U * torch.where(seen, (s - safe).abs() + safe.abs(), 0.0).nan_to_num(0.0, 0.0, 0.0)
    # a mask of the type's lowest value: where a row has other keys its probability is exactly 0, else every score is that value exactly
    ea = torch.where((p == 0) | (safe.abs() > 1e30), 0.0, ea)
    worst = ea.amax(-1, keepdim=True) if Sk else torch.zeros(B, H, Sq, 1, dtype=torch.float64)
    rp = (ea + worst + (Sk + 16) * U) * 1.01
    o = p @ v64
    bo = (p * (rp + up)) @ v64.abs() + (Sk + 8) * U * (p @ v64.abs())
    eo = bo
    bo = (bo + ut * o.abs()) * (1 + 2 * ut)
    out = [o.transpose(1, 2), bo.transpose(1, 2), lse, (worst[..., 0] + (Sk + 24) * U * (1 + lse.abs().nan_to_num(0.0, 0.0, 0.0)))]
    if do is None:
        return out
    g = do.double().cpu().transpose(1, 2)
    dv = p.transpose(2, 3) @ g
    bdv = (p * (rp + 4 * U + up)).transpose(2, 3) @ g.abs() + (G * Sq + 8) * U * (p.transpose(2, 3) @ g.abs())
    dp = g @ v64.transpose(2, 3)
    edp = (D + 4) * U * (g.abs() @ v64.abs().transpose(2, 3))
    delta = (g * o).sum(-1, keepdim=True)
    edelta = (g.abs() * (eo + ut * o.abs())).sum(-1, keepdim=True) * (1 + 2 * ut) + (D + 4) * U * (g * o).abs().sum(-1, keepdim=True)
    ds = p * (dp - delta)
    eds = p * (edp + edelta) + (rp + 6 * U) * ds.abs() + 2 * U * p * (dp.abs() + delta.abs())
    eds = eds * 1.01
    dq, dk = ds @ k64 * scale, ds.transpose(2, 3) @ q64 * scale
    bdq = ((eds + (up + (Sk + 8) * U) * ds.abs()) @ k64.abs()) * abs(scale)
    bdk = ((eds + (up + (G * Sq + 8) * U) * ds.abs()).transpose(2, 3) @ q64.abs()) * abs(scale)

    def shared(t):
        return t.unflatten(1, (Hk, G)).sum(2)

    dk, bdk, dv, bdv = shared(dk), shared(bdk), shared(dv), shared(bdv)
    for t, b in ((dq, bdq), (dk, bdk), (dv, bdv)):
        out += [t.transpose(1, 2), ((b * 1.02 + ut * t.abs()) * (1 + 2 * ut)).transpose(1, 2)]
    if table is not None:
        n = table.shape[0]
        dt_, bt = torch.zeros(n, H, dtype=torch.float64), torch.zeros(n, H, dtype=torch.float64)
        dt_.index_add_(0, idx.flatten(), ds.sum(0).flatten(1).t())
        bt.index_add_(0, idx.flatten(), (eds * 1.02 + (B * Sq * Sk + 8) * U * ds.abs()).sum(0).flatten(1).t())
        out += [dt_, (bt + ut * dt_.abs()) * (1 + 2 * ut)]
    return out


# ---- gated feed-forward product -------------------------------------------------------------------------------------------------
def act_and_slope(g, act):
    """act(g), act'(g) in 64 bits, and bounds on |act'| and |act''| for what an error of g does."""
    if act == "relu":
        return g.clamp(min=0), (g > 0).double()
    if act == "gelu":
        cdf = 0.5 * (1 + torch.erf(g / math.sqrt(2)))
        return g * cdf, cdf + g * torch.exp(-g * g / 2) / math.sqrt(2 * math.pi)
    if act == "gelu_tanh":
        a = math.sqrt(2 / math.pi)
        th = torch.tanh(a * (g + 0.044715 * g ** 3))
        return 0.5 * g * (1 + th), 0.5 * (1 + th) + 0.5 * g * (1 - th * th) * a * (1 + 3 * 0.044715 * g * g)
    if act == "silu":
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    sp = torch.nn.functional.softplus(g)
    th = torch.tanh(sp)
    return g * th, th + g * torch.sigmoid(g) * (1 - th * th)


def gated(x, w, b, act, dh=None, parts=1):
    """(h, bound) and, with dh, (dx, bound), (dw, bound), (db, bound) behind them.  The slopes of the smooth activations are at most 1.2
    and their second derivatives at most 1.2; the kernels' activations and slopes are counted with 1e-6 of max(1, |g|) of their own.
    parts: the numbers of x's type that dz goes into the products as; the second rounds what the first left, so together they miss ut^2."""
    ut = half_step(x.dtype)
    up = ut ** parts if x.dtype == torch.bfloat16 else 0.0
    x64, w64 = x.double().cpu(), w.double().cpu()
    M, K = x64.shape
    F = w64.shape[0] // 2
    z = x64 @ w64.t()
    ez = (K + 4) * U * (x64.abs() @ w64.abs().t())
    if b is not None:
        z = z + b.double().cpu()
        ez = ez + U * (z.abs() + b.double().cpu().abs())
    g, u, eg, eu = z[:, :F], z[:, F:], ez[:, :F], ez[:, F:]
    a, da = act_and_slope(g, act)
    ea = 1.2 * eg + 1e-6 * g.abs().clamp(min=1)
    eda = 1.2 * eg + 1e-6 * g.abs().clamp(min=1)
    h = a * u
    out = [h, ((ea * u.abs() + (a.abs() + ea) * eu + 2 * U * h.abs()) + ut * h.abs()) * (1 + 2 * ut)]
    if dh is None:
        return out
    d = dh.double().cpu()
    dz = torch.cat([d * u * da, d * a], 1)
    edz = torch.cat([d.abs() * (eu * da.abs() + u.abs() * eda + eu * eda), d.abs() * ea], 1) + 4 * U * dz.abs()
    dx, dw, db = dz @ w64, dz.t() @ x64, dz.sum(0)
    bx = (edz + (up + (2 * F + 4) * U) * dz.abs()) @ w64.abs()
    bw = (edz + (up + (M + 4) * U) * dz.abs()).t() @ x64.abs()
    bb = (edz + (M + 4) * U * dz.abs()).sum(0)
    for t, e in ((dx, bx), (dw, bw)):
        out += [t, (e * 1.01 + ut * t.abs()) * (1 + 2 * ut)]
    return out + [db, bb * 1.01]
