"""fused_linear and the 8-bit checkpoints where a caller comes near a limit. Tolerances as in test_hip_linear.py."""
import math

import pytest
import torch

from test_hip_linear import assert_within, forward64, make

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
