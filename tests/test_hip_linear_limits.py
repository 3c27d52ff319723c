"""fused_linear and the 8-bit checkpoints where a caller comes near a limit. Tolerances as in test_hip_linear.py."""
import math

import pytest
import torch

from test_hip_linear import TINY, assert_within, backward64, cuda, forward64, make

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


def autocast_inputs(seed, N=130, D=260, M=70):
    x, W, b, r = make(N, D, M, torch.float32, seed, res=torch.float32)
    g = torch.randn(N, M, generator=torch.Generator().manual_seed(seed)).cuda()
    return [t.requires_grad_() for t in cuda(x, W, b, r)], g


def autocast_step(ts, g):
    y = autocast_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint="e4m3")
    return (y.detach(), *torch.autograd.grad(y, ts, g))


def test_captured_autocast_steps_read_the_weight_of_each_replay(device):
    """fp32 parameters under autocast in two captured graphs, the parameters changed between replays; an eager call between
    capture and first replay, and between replays, sees its own weights too."""
    want = {s: autocast_step(*autocast_inputs(s)) for s in range(5)}
    graphs = []
    for seed in range(2):
        ts, g = autocast_inputs(seed)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            autocast_step(ts, g)                    # (the eager call before leaves nothing that the capture takes up)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = autocast_step(ts, g)
        for a, c in zip(autocast_step(ts, g), want[seed]):
            assert torch.equal(a, c)
        graphs.append((graph, ts, g, outs))
    for seed in (2, 3, 4):
        new, ng = autocast_inputs(seed)
        for graph, ts, g, outs in graphs:
            with torch.no_grad():
                for t, n in zip(ts, new):
                    t.copy_(n)
                g.copy_(ng)
            graph.replay()
        torch.cuda.synchronize()
        for _, ts, g, outs in graphs:
            for a, c in zip(outs, want[seed]):
                assert torch.equal(a, c)
            for a, c in zip(autocast_step(ts, g), want[seed]):
                assert torch.equal(a, c)


def test_a_graph_that_changes_its_weight(device):
    """Training inside a graph: every replay moves W, whose version the host never sees. An eager call reads the new W."""
    ts, g = autocast_inputs(3)

    def train():
        y = autocast_linear(*ts[:3], residual=ts[3])
        (dW,) = torch.autograd.grad(y, ts[1:2], g)
        with torch.no_grad():
            ts[1].sub_(dW)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        train()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        train()
    for _ in range(3):
        autocast_step(ts, g)
        before = ts[1].detach().clone()
        graph.replay()
        fresh = [t.detach().clone().requires_grad_() for t in ts]
        assert not torch.equal(fresh[1], before)
        for a, c in zip(autocast_step(ts, g), autocast_step(fresh, g)):
            assert torch.equal(a, c)


def test_autocast_steps_on_two_streams(device):
    """Two streams that share a weight, changed in place between rounds: neither reads what the other has not written yet."""
    (x, W, b, r), g = autocast_inputs(4, 300, 700, 90)
    other, _ = autocast_inputs(5, 300, 700, 90)
    values = [W.detach().clone(), other[1].detach().clone()]
    want = []
    for v in values:
        want.append(autocast_step([x, v.clone().requires_grad_(), b, r], g))
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(6):
        for st in streams:
            torch.cuda.current_stream().wait_stream(st)
        with torch.no_grad():
            W.copy_(values[i % 2])
        for j, st in enumerate(streams if i % 4 < 2 else streams[::-1]):
            st.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(st):
                if j == 0:
                    torch.cuda._sleep(10_000_000)   # the first stream is behind the second by some milliseconds
                got.append((i % 2, autocast_step([x, W, b, r], g)))
    torch.cuda.synchronize()
    for i, outs in got:
        for a, c in zip(outs, want[i]):
            assert torch.equal(a, c)


def test_a_weight_changed_behind_its_version(device):
    ts, g = autocast_inputs(6)
    autocast_step(ts, g)
    ts[1].data.mul_(0.5)                            # (.data has a version counter of its own)
    fresh = [t.detach().clone().requires_grad_() for t in ts]
    for a, c in zip(autocast_step(ts, g), autocast_step(fresh, g)):
        assert torch.equal(a, c)


def test_a_weight_that_changes_between_forward_and_backward(device):
    """dx reads the bf16 copy of the forward, dW no weight: the gradients are those at the forward's weight."""
    ts, g = autocast_inputs(7)
    want = autocast_step(ts, g)
    y = autocast_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint="e4m3")
    with torch.no_grad():
        ts[1].zero_()
    for a, c in zip(torch.autograd.grad(y, ts, g), want[1:]):
        assert torch.equal(a, c)


def test_a_traced_call_launches_the_kernels(device):
    from sparsify_amd import fused_linear
    x, W, b, r = cuda(*make(40, 72, 56, torch.bfloat16, 2, res=torch.float32))

    def f(x, W, b, r):
        return fused_linear(x, W, b, residual=r, activation="silu")

    traced = torch.jit.trace(f, (x, W, b, r), check_trace=False)
    for seed in (3, 4):
        args = cuda(*make(40, 72, 56, torch.bfloat16, seed, res=torch.float32))
        assert torch.equal(traced(*args), f(*args))


# ------------------------------------------------------------------ values near the largest
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_finite_values_restore_as_finite_ones(device, fmt, dtype):
    """Groups whose largest value is 2^127 and up. Codes under the scale that keeps it; where the nearest one stands for 2^128,
    the one below it: off by at most a step, 2^122, instead of half of one (int8), or by 2^-4 of the value (e4m3)."""
    from sparsify_amd import checkpoint8
    from test_hip_linear import codes64
    most = torch.finfo(dtype).max
    edges = [1.0, 1.5, 1.75, 1.765625, 1.875, 1.9296875, 1.9375, 1.9765625, 1.984375, 1.9921875]
    tops = torch.tensor([e * 2.0**127 for e in edges] + [most], dtype=torch.float64).to(dtype)
    assert torch.isfinite(tops).all()
    x = torch.randn(64, tops.numel(), generator=torch.Generator().manual_seed(0)).double()
    x = (x / x.abs().amax(0) * 2.0**126).to(dtype)
    x[5], x[40] = tops, -tops
    x[6] = torch.nextafter(tops.float(), torch.zeros(())).to(dtype)
    x[6] = torch.where(torch.isfinite(x[6]), x[6], tops)
    want = codes64(x, fmt)
    last = 63 * 2.0**122 if fmt == "int8" else 240 * 2.0**120
    want = torch.where(want.abs() >= 2.0**128, torch.sign(want) * last, want)
    for keep_sign in (False, True):
        c = checkpoint8(x.cuda(), fmt, keep_sign=keep_sign)
        for kept in (torch.float32, torch.bfloat16):
            got = c.restore(kept)
            assert torch.isfinite(got).all()
            pick = torch.ones_like(want, dtype=torch.bool) if not keep_sign else want != 0
            assert torch.equal(got.double().cpu()[pick], want[pick])
    off = (want - x.double()).abs()
    bound = 2.0**-4 * x.double().abs() + 2.0**-13 * 2.0**127 if fmt == "e4m3" else torch.full_like(off, 2.0**122)
    assert (off <= bound).all()


def test_kept_pre_activation_near_the_largest(device):
    """The product's own codes of z: an identity's values as they come."""
    from sparsify_amd import ops
    top = torch.finfo(torch.float32).max
    x = torch.tensor([top, -top, 2.0**127, 1.9375 * 2.0**127, 1.0, 0.0, -3e38, 3.3e38]).repeat(64, 8).cuda()
    W = torch.eye(64, device="cuda")
    for fmt in ("int8", "e4m3"):
        for kernel_rows in (64, 130):               # the few-rows kernel's way over fp32, and codes in the epilogue
            xi = x.repeat(3, 1)[:kernel_rows]
            _, z, _ = ops.linear(xi, W, activation="silu", keep_z=fmt)
            got = ops.checkpoint8_restore(z, fmt, kernel_rows, 64, torch.float32)
            want = ops.checkpoint8_restore(ops.checkpoint8_save(xi, fmt), fmt, kernel_rows, 64, torch.float32)
            assert torch.isfinite(got).all() and torch.equal(got, want)


# ------------------------------------------------------------------ few rows, on both sides of the rules' borders
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D,M", [(1024, 4095), (2048, 4097), (2050, 6000), (520, 8192), (1536, 8200), (4096, 2047), (48, 9001)])
def test_few_rows_of_any_width(device, monkeypatch, D, M, dtype):
    from sparsify_amd import ops
    for N in (1, 4, 8, 9, 16, 17, 24, 32, 33, 64):
        x, W, b, r = make(N, D, M, dtype, D + N, res=dtype)
        want, tol, z, ez = forward64(x, W, b, r, "silu", dtype)
        xc, Wc, bc, rc = cuda(x, W, b, r)
        for kernel in ("few", None):
            monkeypatch.setenv("SPHIP_LINEAR", kernel) if kernel else monkeypatch.delenv("SPHIP_LINEAR")
            y, zk, _ = ops.linear(xc, Wc, bc, rc, "silu", keep_z=torch.float32)
            assert_within(y, want, tol, f"y {N} {kernel}")
            assert_within(zk, z, ez + 2.0**-24 * z.abs() + TINY, f"z {N} {kernel}")
