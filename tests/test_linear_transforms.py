"""fused_linear and the 8-bit checkpoints under forward-mode differentiation and torch.jit.trace, on the CPU, with the
products themselves in torch: what matters is which way the call takes."""
import importlib

import pytest
import torch
import torch.autograd.forward_ad as forward_ad


@pytest.fixture
def linear(monkeypatch):
    from sparsify_amd import fused_linear
    fl = importlib.import_module("sparsify_amd.fused_linear")        # (the package re-exports the function of that name)

    def product(x, W, bias=None, residual=None, activation="none", out_dtype=None, keep_z=None, keep_x=None):
        out = torch.empty(x.shape[0], W.shape[0])
        # behind torch's back, as a kernel writes it
        out.numpy()[:] = x.detach().numpy() @ W.detach().numpy().T
        return out, None, None

    monkeypatch.setattr(fl.ops, "linear", product)
    monkeypatch.setattr(fl, "_operands", lambda x, W: (x, W))
    return fused_linear


def test_a_tangent_is_refused(linear):
    x, W, b, r = torch.randn(3, 4), torch.randn(5, 4), torch.randn(5), torch.randn(3, 5)
    with forward_ad.dual_level():
        assert torch.allclose(linear(x, W), x @ W.T, atol=1e-5)      # no input carries one
        for i in range(4):
            args = [x, W, b, r]
            args[i] = forward_ad.make_dual(args[i], torch.ones_like(args[i]))
            with pytest.raises(NotImplementedError):
                linear(*args[:3], residual=args[3])
    assert torch.allclose(linear(x, W), x @ W.T, atol=1e-5)


@pytest.mark.parametrize("grad", [False, True])
def test_a_traced_call_computes(linear, grad):
    W = torch.randn(5, 4, requires_grad=grad)
    traced = torch.jit.trace(lambda a, w: linear(a, w), (torch.randn(3, 4), W), check_trace=False)
    for seed in range(3):
        x = torch.randn(3, 4, generator=torch.Generator().manual_seed(seed))
        assert torch.allclose(traced(x, W), x @ W.T, atol=1e-5)


def test_checkpoints_are_not_traced():
    from sparsify_amd import Checkpoint8, checkpoint8
    x = torch.randn(3, 8)
    c = Checkpoint8(torch.zeros(33, 16, dtype=torch.uint8), "int8", (3, 8), torch.float32)
    for f in (lambda a: checkpoint8(a).restore(), lambda a: a + c.restore()):
        with pytest.raises(RuntimeError, match="cannot be traced"):
            torch.jit.trace(f, (x,), check_trace=False)
