"""The transformer blocks on the library's kernels under torch.autocast."""
import copy

import pytest
import torch

from vita_amd import encoders, ops

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_gated_product_takes_autocast_type(monkeypatch):
    """Under autocast the gated product runs in bf16, as the Linear layers beside it do."""
    torch.manual_seed(6)
    blk = encoders.TransformerBlock(64, 8, rope_max_seq_length=17, gated=True, rel_buckets=8, kernels=True)
    want = copy.deepcopy(blk).double()
    blk = blk.to(DEV)
    seen = []
    call = ops.gated_linear
    monkeypatch.setattr(ops, "gated_linear", lambda x, w, b, act: (seen.append((x.dtype, w.dtype, b.dtype)), call(x, w, b, act))[1])
    x = torch.randn(5, 17, 64)
    a, a64 = x.to(DEV).requires_grad_(True), x.double().requires_grad_(True)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = blk(a)
    y64 = want(a64)
    assert seen == [(torch.bfloat16, torch.bfloat16, torch.float32)]
    y.float().square().sum().backward()
    y64.square().sum().backward()
    # one block: 6 roundings to bf16 (2^-8 each) in a row, doubled by the norms between them: 0.05 of the largest value
    for got, ref in ((y, y64), (a.grad, a64.grad), *((p.grad, q.grad) for p, q in zip(blk.parameters(), want.parameters()))):
        assert (got.double().cpu() - ref).abs().max().item() <= 0.05 * ref.abs().max().item()
    blk(a)
    assert seen[1:] == [(torch.float32,) * 3]


def test_gated_product_keeps_its_type_under_float16():
    torch.manual_seed(7)
    mlp = encoders._GatedMlp(32, 48, kernels=True).to(DEV)
    x = torch.randn(3, 5, 32, device=DEV)
    with torch.autocast("cuda", dtype=torch.float16):
        y = mlp(x)
    want = mlp(x)
    assert ops.gated_linear(x.view(15, 32), mlp.fc1.weight, mlp.fc1.bias, "gelu_tanh").abs().max().item() <= 4
    # fc2 alone runs in float16: its operands' and its result's roundings of 2^-11, on values of at most 4
    assert y.dtype == torch.float16 and (y.float() - want).abs().max().item() <= 3 * 2.0 ** -11 * (mlp.fc2.weight.abs().sum(1).max() * 4).item()
