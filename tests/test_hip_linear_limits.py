"""fused_linear and the 8-bit checkpoints where a caller comes near a limit. Tolerances as in test_hip_linear.py."""
import math

import pytest
import torch

from test_hip_linear import TINY, assert_within, backward64, forward64, make

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------ one operand copied, the other as it is
FAR = (1 << 22) + 4


def far_rows(t, size=FAR):
    """t's rows `size` elements apart, NaN in front of and behind each."""
    N, D = t.shape
    big = torch.empty(N * size, dtype=t.dtype, device="cuda")
    rows = big.view(N, size)
    rows[:, : D + 64] = math.nan
    rows[:, 4 : 4 + D] = t.cuda()
    return rows[:, 4 : 4 + D]


def framed(t):
    """t's rows one after another (stride D), NaN in front of the first and behind the last."""
    N, D = t.shape
    flat = torch.full(((N + 2) * D + 64,), math.nan, dtype=t.dtype, device="cuda")
    flat[D : D + N * D] = t.cuda().reshape(-1)
    return flat[D : D + N * D].view(N, D)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("N,D,M", [(330, 201, 150), (400, 204, 40), (70, 1003, 90), (64, 2050, 33)])
@pytest.mark.parametrize("far", ["x", "W"])
def test_one_operand_with_rows_far_apart(device, dtype, N, D, M, far):
    """Only the operand whose rows lie 2^22 elements apart is copied (fp32): the other is read up to its last element and no
    further, whatever follows, a NaN of the next token or of the memory behind the tensor. The same bits as from dense rows."""
    from sparsify_amd import fused_linear
    x, W, b, _ = make(N, D, M, dtype, D)
    want, tol, _, _ = forward64(x, W, b, None, "silu", dtype)
    xc, Wc = (far_rows(x), framed(W)) if far == "x" else (framed(x), far_rows(W))
    g = torch.randn(N, M, generator=torch.Generator().manual_seed(D)).to(dtype).cuda()
    outs = []
    for pair in ((x.cuda(), W.cuda()), (xc, Wc)):
        ts = [t.detach().requires_grad_() for t in (*pair, b.cuda())]
        y = fused_linear(*ts, activation="silu")
        outs.append((y.detach(), *torch.autograd.grad(y, ts, g)))
    assert_within(outs[1][0], want, tol, "y")
    for a, c in zip(*outs):
        assert torch.equal(a, c)
    x[7] = math.nan                                 # of one token: the others are as before
    got = fused_linear(far_rows(x) if far == "x" else framed(x), Wc, b.cuda(), activation="silu")
    keep = torch.arange(N, device="cuda") != 7
    assert torch.isnan(got[7]).all() and torch.equal(got[keep], outs[0][0][keep])


# ------------------------------------------------------------------ fp32 weights under bf16 autocast
def autocast_linear(*args, **kw):
    from sparsify_amd import fused_linear
    with torch.autocast("cuda", dtype=torch.bfloat16):
        return fused_linear(*args, **kw)


def assert_autocast_step(x, W, g):
    """One step of fp32 x and W under autocast: the product of their bf16 values, gradients from bf16 operands with g (bf16)
    as it is, fp32 results. W: the tensor or view itself, gradients taken at it."""
    xi = x.detach().requires_grad_()
    y = autocast_linear(xi, W)
    xb, Wb = x.detach().cpu().bfloat16(), W.detach().cpu().bfloat16()
    want, tol, _, _ = forward64(xb, Wb, None, None, "none", torch.bfloat16)
    assert_within(y.detach(), want, tol, "y")
    dx, dW = torch.autograd.grad(y, [xi, W], g)
    ref = backward64(xb, Wb, None, "none", g.cpu(), want, xb, torch.float32, torch.bfloat16, 0.0)
    assert_within(dx, *ref["x"], "dx")
    want, mag = g.cpu().double().T @ xb.double(), g.cpu().double().abs().T @ xb.double().abs()
    assert_within(dW, want, (x.shape[0] + 4) * 2.0**-23 * mag + 2.0**-24 * want.abs() + TINY, "dW")


def test_weights_at_one_address(device):
    """A weight, its transpose, and two views of one size: each by its own values, forward and gradients, in any order."""
    gen = torch.Generator().manual_seed(1)
    W = (torch.randn(96, 96, generator=gen) / 10).cuda().requires_grad_()
    x = torch.randn(130, 96, generator=gen).cuda()
    g = {m: torch.randn(130, m, generator=gen).bfloat16().cuda() for m in (96, 48)}
    views = [W, W.t(), W[:48], W[::2], W.t()[:48], W]
    for v in views + views[::-1]:
        assert_autocast_step(x, v, g[v.shape[0]])
