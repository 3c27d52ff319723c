"""The bf16 copies of fp32 weights (fused_encoder.bf16_shadow) follow the tensor, its version and its layout. On the CPU,
with the cast itself in torch."""
import importlib

import pytest
import torch


@pytest.fixture
def fe(monkeypatch):
    fe = importlib.import_module("sparsify_amd.fused_encoder")       # (the package re-exports the function of that name)

    def cast(src, out=None):
        assert src.is_contiguous()
        return src.bfloat16() if out is None else out.copy_(src)

    monkeypatch.setattr(fe.ops, "cast_bf16", cast)
    monkeypatch.setattr(fe, "_shadows", {})
    return fe


def test_a_transpose_is_not_its_base(fe):
    W = torch.nn.Parameter(torch.randn(8, 8))
    for t in (W, W.t(), W, W.detach().t(), W.detach(), W):
        assert torch.equal(fe.bf16_shadow(t), t.detach().bfloat16())
    assert fe.peek_bf16_shadow(W) is not None and fe.peek_bf16_shadow(W.t()) is None
    assert fe.shadow_is_current(W) and not fe.shadow_is_current(W.t())


@pytest.mark.parametrize("grad", [False, True])
def test_views_of_one_size_at_one_address(fe, grad):
    B = torch.randn(64, 16, requires_grad=grad)
    views = [B[:32], B[::2], B.view(32, 32)[:, :16], B[:32]]
    for v in views + views[::-1]:
        assert torch.equal(fe.bf16_shadow(v), v.detach().bfloat16())


def test_the_copy_is_kept_until_the_weight_changes(fe):
    W = torch.nn.Parameter(torch.randn(4, 6))
    first = fe.bf16_shadow(W)
    fe.bf16_shadow(W[:2]), fe.bf16_shadow(W.t())                     # views leave W's copy where it is
    assert fe.bf16_shadow(W) is first and fe.bf16_shadow(W.detach()) is first
    with torch.no_grad():
        W.mul_(2)
    assert not fe.shadow_is_current(W)
    assert torch.equal(fe.bf16_shadow(W), W.detach().bfloat16())
    new = (W * 3).detach().bfloat16()
    fe.register_bf16_shadow(W, new)
    assert fe.bf16_shadow(W) is new
    del W
    assert not fe._shadows


def test_a_weight_transposed_in_place(fe):
    W = torch.randn(8, 8)
    fe.bf16_shadow(W)
    W.t_()
    assert torch.equal(fe.bf16_shadow(W), W.bfloat16())
