"""Every form of the transformer blocks' operators captured into a graph, forward and backward, and replayed on new inputs with eager work between
the replays: the same bits as the eager calls."""
import pytest
import torch

import block_ops_reference as ref
from vita_amd import ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def _attention(g, dtype, B, Sq, Sk, H, Hk, D, R, causal):
    pad = torch.zeros(B, Sk, dtype=torch.bool)
    for b in range(B):
        pad[b, :(b * 70) % Sk] = True                                 # padded in front
    kw = dict(causal=causal, key_pad=pad.to(DEV))
    if R is not None:
        kw |= dict(table=torch.randn(8, H, generator=g).to(dtype).to(DEV), buckets=torch.randint(0, 8, (2 * R + 1,), generator=g, dtype=torch.int32).to(DEV))

    def step(q, k, v, do):
        o, stats = ops.attention(q, k, v, need_lse=True, **kw)
        return [ops.attention(q, k, v, **kw), o, stats, *ops.attention_bwd(do, q, k, v, o, stats, **kw)]
    return step, [(B, Sq, H, D), (B, Sk, Hk, D), (B, Sk, Hk, D), (B, Sq, H, D)]


def _gated(g, dtype, M, K, F):
    w, b = (torch.randn(2 * F, K, generator=g) * K ** -0.5).to(dtype).to(DEV), torch.randn(2 * F, generator=g).to(DEV)

    def step(x, dh):
        h, saved = ops.gated_linear(x, w, b, need_saved=True)
        return [h, *ops.gated_linear_bwd(dh, x, w, b, saved=saved)]
    return step, [(M, K), (M, F)]


def _norm_rope(g, dtype, B, S, H, Hk, D):
    rope, p = ref.rope_table(S, 1, D).to(DEV), {n: torch.randn(D, generator=g).to(DEV) for n in ("q_weight", "q_bias", "k_weight", "k_bias")}

    def step(q, k, dq, dk):
        return [*ops.qk_norm_rope(q, k, rope, **p), *ops.qk_norm_rope_bwd(dq, dk, q, k, rope, **p)]
    return step, [(B, S, H, D), (B, S, Hk, D)] * 2


FORMS = {
    "one wave": (_attention, 3, 17, 17, 4, 2, 64, 9, False), "split keys": (_attention, 2, 1, 4000, 8, 2, 64, None, True),
    "packed heads": (_attention, 2, 1, 300, 32, 1, 128, 1024, False), "shared keys": (_attention, 3, 200, 300, 2, 1, 128, 33, True),
    "rows": (_attention, 8, 200, 300, 16, 16, 32, 9, True), "wide dq": (_attention, 2, 20, 100, 2, 2, 128, 1024, False),
    "few gated rows": (_gated, 5, 64, 200), "gated rows": (_gated, 300, 96, 520), "gated tiles": (_gated, 2300, 40, 2568),
    "norms": (_norm_rope, 5, 130, 6, 2, 72),
}


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("form", FORMS)
def test_captured_and_replayed(form, dtype):
    make, *sizes = FORMS[form]
    g = torch.Generator().manual_seed(len(form))
    step, shapes = make(g, dtype, *sizes)

    def fresh():
        return [torch.randn(*s, generator=g).to(dtype).to(DEV) for s in shapes]

    static = fresh()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(*static)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        res = step(*static)
    for i in range(3):
        for t, n in zip(static, fresh()):
            t.copy_(n)
        want = step(*static)                                          # eager work between the replays
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(res, want)), i
