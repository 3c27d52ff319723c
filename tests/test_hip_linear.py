"""fused_linear (act(x W^T + b) + r, its gradients) and the 8-bit checkpoints, against their definitions in 64 bits on the
same inputs. Tolerances are elementwise bounds from the operations' roundings:
  * a sum of K fp32 terms: K + 4 additions, each off by at most 2^-23 of the sum of magnitudes;
  * the activations' polynomials: 4e-7 (1 + |z|) on a value, 1e-6 on a slope (both below 1.13 in slope);
  * a rounding to bf16 2^-8 of the value, to fp32 2^-24; dz is rounded once to the product's dtype before it is used."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

HALF = {torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}
ACTS = ["none", "relu", "gelu", "silu"]
TINY = 2.0**-126


def act64(z, act):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[act]()


def slope64(z, act):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "silu": lambda: s + z * s * (1 - s),
            "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[act]()


def codes64(x, fmt, keep_sign=False):
    """The values an 8-bit checkpoint of x (N, D) stands for, in 64 bits, value by value from the definition."""
    out = []
    for rows in x.double().split(32):
        top = rows.abs().amax(0)
        e = torch.full_like(top, -126.0 if fmt == "int8" else -117.0)
        most = 127.0 if fmt == "int8" else 448.0
        while True:                                       # the smallest exponent that keeps the group's maximum
            over = torch.isfinite(top) & (top / torch.exp2(e) > most)
            if not over.any():
                break
            e = e + over
        q = rows / torch.exp2(e)
        if fmt == "int8":
            k = torch.round(q)
            least = 1.0
        else:
            step = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0**-6))) - 3)
            k = torch.round(q / step) * step
            least = 2.0**-9
        if keep_sign:
            k = torch.where((k == 0) & (q != 0), torch.sign(q) * least, k)
        out.append(torch.where(torch.isfinite(top), k * torch.exp2(e), torch.full_like(k, math.nan)))
    return torch.cat(out) if out else x.double()


def make(N, D, M, dtype, seed, bias=True, res=None):
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp(0.5 * torch.randn(D, generator=g)) * torch.where(torch.rand(D, generator=g) < 0.05, 20.0, 1.0)
    x = (torch.randn(N, D, generator=g) * scale + 0.3 * scale).to(dtype)
    W = (torch.randn(M, D, generator=g) / (scale * D**0.5)).to(dtype)
    b = torch.randn(M, generator=g).to(dtype) * 0.5 if bias else None
    r = None if res is None else torch.randn(N, M, generator=g).to(res)
    return x, W, b, r


def cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


def forward64(x, W, b, r, act, out_dtype):
    """(y, elementwise bound, z, bound of z)"""
    xd, Wd = x.double(), W.double()
    K = x.shape[1]
    z = xd @ Wd.T
    mag = xd.abs() @ Wd.abs().T
    if b is not None:
        z, mag = z + b.double(), mag + b.double().abs()
    ez = (K + 4) * 2.0**-23 * mag
    y = act64(z, act)
    tol = 1.13 * ez + (4e-7 * (1 + z.abs()) if act in ("gelu", "silu") else 0)
    if r is not None:
        y = y + r.double()
        tol = tol + 2.0**-24 * (y.abs() + r.double().abs())
    return y, tol + HALF[out_dtype] * (y.abs() + tol) + TINY, z, ez


def assert_within(got, want, tol, what=""):
    got = got.double().cpu()
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), (f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst {float(((got - want).abs() / tol).nan_to_num(math.inf).max()):.3g} "
                           f"times the bound at {tuple(int(i) for i in bad.nonzero()[0])}")


SHAPES = [(1, 64, 64), (1, 1, 1), (2, 7, 3), (3, 129, 65), (16, 256, 1000), (17, 513, 40), (31, 64, 257), (33, 1000, 96),
          (64, 2048, 128), (100, 72, 200), (128, 128, 128), (129, 96, 129), (257, 255, 511), (300, 4096, 640), (1003, 769, 450)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D,M", SHAPES)
def test_forward(device, N, D, M, dtype):
    from sparsify_amd import fused_linear
    for i, act in enumerate(ACTS):
        res = [None, dtype, torch.float32, None][(i + N) % 4]
        x, W, b, r = make(N, D, M, dtype, N + D + M + i, bias=(i + M) % 3 != 0, res=res)
        out_dtype = dtype if res is None else torch.promote_types(dtype, res)
        y, tol, _, _ = forward64(x, W, b, r, act, out_dtype)
        xc, Wc, bc, rc = cuda(x, W, b, r)
        got = fused_linear(xc, Wc, bc, residual=rc, activation=act)
        assert got.dtype == out_dtype and got.shape == (N, M)
        assert_within(got, y, tol, f"{act} {N}x{D}x{M}")


def test_forward_takes_leading_dims_strides_and_odd_addresses(device):
    from sparsify_amd import fused_linear
    for dtype in (torch.bfloat16, torch.float32):
        x, W, b, r = make(6 * 11, 200, 130, dtype, 5, res=dtype)
        y, tol, _, _ = forward64(x, W, b, r, "silu", dtype)
        xc, Wc, bc, rc = cuda(x, W, b, r)
        wide = torch.full((66, 407), float("nan"), dtype=dtype, device="cuda")
        wide[:, 3:203] = xc                                # rows at odd addresses, NaN between them
        wideW = torch.full((130, 333), float("nan"), dtype=dtype, device="cuda")
        wideW[:, 1:201] = Wc
        wideR = torch.full((66, 301), float("nan"), dtype=dtype, device="cuda")
        wideR[:, 5:135] = rc
        base = fused_linear(xc, Wc, bc, residual=rc, activation="silu")
        assert_within(base, y, tol)
        for xi in (xc, wide[:, 3:203], xc.t().contiguous().t()):
            for wi in (Wc, wideW[:, 1:201], Wc.t().contiguous().t()):
                got = fused_linear(xi, wi, bc, residual=wideR[:, 5:135], activation="silu")
                assert torch.equal(got, base)
        got = fused_linear(xc.reshape(6, 11, 200), Wc, bc, residual=rc.reshape(6, 11, 130), activation="silu")
        assert got.shape == (6, 11, 130) and torch.equal(got.reshape(66, 130), base)
        one = fused_linear(xc[7], Wc, bc, residual=rc[7], activation="silu")          # a single token without a batch dim
        assert one.shape == (130,)
        assert_within(one, y[7], tol[7])


def test_forward_writes_its_rows_only(device):
    """The C entry point with row strides wider than the rows: what lies between and behind them stays."""
    from sparsify_amd import _lib
    lib = _lib.load()
    for dtype in (torch.bfloat16, torch.float32):
        for N, D, M in ((5, 40, 33), (200, 64, 129), (1, 512, 64)):
            x, W, b, _ = make(N, D, M, dtype, 1)
            xc, Wc, bc = cuda(x, W, b)
            out = torch.full((N + 2, M + 5), 7.0, dtype=dtype, device="cuda")
            z = torch.full((N + 2, M + 3), 7.0, device="cuda")
            dt = _lib.BF16 if dtype == torch.bfloat16 else _lib.F32
            nws = lib.sphip_linear_workspace_bytes(dt, _lib.F32, N, D, M, 0)
            ws = torch.empty(max(nws, 16), dtype=torch.uint8, device="cuda")
            _lib.check(lib.sphip_linear(xc.data_ptr(), D, Wc.data_ptr(), D, dt, bc.data_ptr(), dt, 1, None, 0, 0,
                                        out[1:].data_ptr(), dt, M + 5, z[1:].data_ptr(), _lib.F32, None, M + 3, None, None,
                                        0, 0, N, D, M, ws.data_ptr(), nws, torch.cuda.current_stream().cuda_stream), "sphip_linear")
            y, tol, zz, ez = forward64(x, W, b, None, "relu", dtype)
            assert_within(out[1:N + 1, :M], y, tol)
            assert_within(z[1:N + 1, :M], zz, ez + HALF[torch.float32] * zz.abs() + TINY)
            for t, m in ((out, M), (z, M)):
                assert (t[0] == 7).all() and (t[N + 1] == 7).all() and (t[:, m:] == 7).all()


@pytest.mark.parametrize("act", ACTS)
def test_forward_infinities_and_nan_stay_in_their_rows(device, act):
    from sparsify_amd import fused_linear
    for dtype in (torch.bfloat16, torch.float32):
        x, W, b, _ = make(70, 96, 80, dtype, 3)
        xc, Wc, bc = cuda(x, W, b)
        clean = fused_linear(xc, Wc, bc, activation=act)
        xb = xc.clone()
        xb[9, 5], xb[40, 95] = float("nan"), float("inf")
        got = fused_linear(xb, Wc, bc, activation=act)
        rows = torch.ones(70, dtype=torch.bool, device="cuda")
        rows[9] = rows[40] = False
        assert torch.equal(got[rows], clean[rows])
        assert torch.isnan(got[9]).all()
        z = torch.where(Wc[:, 95] > 0, math.inf, -math.inf).double()
        want = {"none": z, "relu": z.clamp(min=0), "gelu": z, "silu": z}[act]
        pos = z > 0
        assert torch.equal(got[40][pos].double(), want[pos])
        big = torch.full((2, 4), 1e30, device="cuda", dtype=dtype)         # saturated activations
        got = fused_linear(big, torch.eye(4, device="cuda", dtype=dtype), activation=act)
        assert torch.equal(got, big)
        got = fused_linear(-big, torch.eye(4, device="cuda", dtype=dtype), activation=act)
        assert torch.equal(got, -big if act == "none" else torch.zeros_like(big))


# ------------------------------------------------------------------ 8-bit checkpoints
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D", [(1, 1), (1, 768), (31, 15), (32, 16), (33, 17), (64, 100), (95, 257), (256, 768), (1000, 1111), (5, 4099)])
def test_checkpoint_is_the_nearest_code(device, N, D, dtype, fmt):
    from sparsify_amd import checkpoint8
    for keep_sign in (False, True):
        x = make(N, D, 1, dtype, N + D)[0]
        g = torch.Generator().manual_seed(N)
        x[torch.rand(N, D, generator=g) < 0.1] = 0
        x[torch.rand(N, D, generator=g) < 0.05] *= 1e-6
        if D > 3:
            x[:, 2] = 0                                             # a feature that is all zeros
            x[:, 3] = (x[:, 3].double() * 2.0**-118).to(dtype)      # under the smallest scale
        c = checkpoint8(x.cuda(), fmt, keep_sign=keep_sign)
        got = c.restore()
        assert got.dtype == dtype and got.shape == x.shape
        want = codes64(x, fmt, keep_sign)
        assert torch.equal(got.double().cpu(), want)
        assert torch.equal(c.restore(torch.float32).double().cpu(), want)
        assert torch.equal(c.restore(torch.bfloat16).double().cpu(), want)
        assert c.nbytes < 1.07 * max(N, 31) * (D + 16) + 2000
        if keep_sign:
            assert torch.equal(torch.sign(got).cpu(), torch.sign(x))
        half = 0.5 / 63.5 if fmt == "int8" else 2.0**-4             # the stated error: of the group's maximum / of the value
        for lo in range(0, N, 32):
            top = x[lo:lo + 32].double().abs().amax(0)
            # e4m3 near zero: half a step is 2^-10 2^e, and 2^e < top / 224 < top 2^-7.8: below 2^-4 top 2^-13
            ref = top if fmt == "int8" else torch.maximum(x[lo:lo + 32].double().abs(), top * 2.0**-13)
            slack = 2.0 if keep_sign else 1.0
            assert ((want[lo:lo + 32] - x[lo:lo + 32].double()).abs() <= slack * half * ref + 2.0**-126).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_checkpoint_ties_and_range_ends(device, fmt):
    """Values half way between codes go to the even one; the largest code is reached and not passed; every exponent."""
    from sparsify_amd import checkpoint8
    if fmt == "int8":
        col = torch.cat([torch.arange(-127, 128) / 1.0, torch.arange(-126, 127) + 0.5, torch.tensor([127.0, -127.0])])
    else:
        table = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).float()
        col = torch.cat([table, (table[1:] + table[:-1]) / 2, -table])
    n = -(-col.numel() // 31)
    x = torch.zeros(n * 32)
    top = 127.0 if fmt == "int8" else 448.0
    for i in range(n):                                           # every group's maximum is the format's largest code
        x[32 * i] = top
        part = col[31 * i:31 * (i + 1)]
        x[32 * i + 1:32 * i + 1 + part.numel()] = part
    exps = list(range(-116, 119, 6)) + [118]
    x = torch.stack([x * 2.0**e for e in exps] + [x * (1 + 2.0**-20)], 1)
    want = codes64(x, fmt)
    got = checkpoint8(x.cuda(), fmt).restore()
    assert torch.equal(got.double().cpu(), want)
    assert (got[::32, 2].cpu() == top * 2.0**exps[2]).all()


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_checkpoint_keeps_nan_and_infinities_in_their_group(device, fmt):
    from sparsify_amd import checkpoint8
    for dtype in (torch.bfloat16, torch.float32):
        x = make(100, 50, 1, dtype, 0)[0]
        clean = checkpoint8(x.cuda(), fmt).restore()
        x[40, 7], x[99, 8], x[0, 49] = float("nan"), float("inf"), -float("inf")
        got = checkpoint8(x.cuda(), fmt).restore()
        bad = torch.zeros(100, 50, dtype=torch.bool, device="cuda")
        bad[32:64, 7] = bad[96:, 8] = bad[:32, 49] = True
        assert torch.isnan(got[bad]).all() and torch.equal(got[~bad], clean[~bad])


def test_checkpoint_takes_strided_rows_and_leading_dims(device):
    from sparsify_amd import checkpoint8
    x = make(77, 90, 1, torch.bfloat16, 2)[0].cuda()
    base = checkpoint8(x, "int8").restore()
    wide = torch.full((77, 201), float("nan"), dtype=torch.bfloat16, device="cuda")
    wide[:, 11:101] = x
    assert torch.equal(checkpoint8(wide[:, 11:101], "int8").restore(), base)
    assert torch.equal(checkpoint8(x.t().contiguous().t(), "int8").restore(), base)
    c = checkpoint8(x.reshape(7, 11, 90), "int8")
    assert c.restore().shape == (7, 11, 90) and torch.equal(c.restore().reshape(77, 90), base)
    e = checkpoint8(x[:0], "e4m3")
    assert e.restore().shape == (0, 90)


# ------------------------------------------------------------------ gradients
def backward64(x, W, b, act, g, zhat, xhat, in_dtype, compute, ez):
    """Gradients from the definition at the kept values, and elementwise bounds."""
    gd, Wd, xd = g.double(), W.double(), xhat.double()
    dz = gd * slope64(zhat, act)
    # the slope's own error and, where z is kept as it is, what z's error does to it (|act''| <= 0.8)
    edz = gd.abs() * ((1e-6 + 0.8 * ez) if act in ("gelu", "silu") else 0.0)
    rdz = edz + (HALF[compute] * dz.abs() if act != "none" or g.dtype != compute else 0.0)
    N, M = dz.shape
    out = {}
    dx = dz @ Wd
    t = rdz @ Wd.abs() + (M + 4) * 2.0**-23 * (dz.abs() @ Wd.abs())
    out["x"] = dx, t + HALF[in_dtype] * (dx.abs() + t) + TINY
    dW = dz.T @ xd
    t = rdz.T @ xd.abs() + (N + 4) * 2.0**-23 * (dz.abs().T @ xd.abs())
    out["W"] = dW, t + HALF[W.dtype] * (dW.abs() + t) + TINY
    if b is not None:
        db = dz.sum(0)
        t = edz.sum(0) + (N + 4) * 2.0**-24 * dz.abs().sum(0)
        out["b"] = db, t + HALF[b.dtype] * (db.abs() + t) + TINY
    return out


GRAD_SHAPES = [(1, 64, 64), (2, 7, 3), (17, 130, 65), (33, 64, 257), (64, 96, 100), (130, 200, 129), (300, 257, 140), (1003, 129, 200)]


@pytest.mark.parametrize("fmt", [None, "int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D,M", GRAD_SHAPES)
def test_backward(device, N, D, M, dtype, fmt):
    """The kept z is read back from the forward's own outputs (its codes are exact functions of it), so that a code that
    falls to the other side of a tie is no error of the gradient."""
    from sparsify_amd import ops
    from sparsify_amd.checkpoint8 import checkpoint8
    from sparsify_amd.fused_linear import fused_linear
    for i, act in enumerate(ACTS):
        res = [None, dtype, torch.float32, None][(i + N + M) % 4]
        x, W, b, r = make(N, D, M, dtype, N + D + M + i, bias=(i + N) % 3 != 0, res=res)
        leaves = [None if t is None else t.requires_grad_() for t in cuda(x, W, b, r)]
        xc, Wc, bc, rc = leaves
        y = fused_linear(xc, Wc, bc, residual=rc, activation=act, checkpoint=fmt)
        want_y, tol, z, _ = forward64(x, W, b, r, act, y.dtype)
        assert_within(y.detach(), want_y, tol, f"y {act}")
        g = torch.randn(N, M, generator=torch.Generator().manual_seed(i)).to(y.dtype)
        grads = torch.autograd.grad(y, [t for t in leaves if t is not None], g.cuda())
        # what the backward kept
        args = (xc.detach(), Wc.detach(), None if bc is None else bc.detach(), None if rc is None else rc.detach(), act)
        zk = ops.linear(*args, keep_z=torch.float32 if fmt else dtype)[1]
        zhat = zk.double().cpu()
        if fmt:
            _, zc, xcodes = ops.linear(*args, keep_z=fmt, keep_x=fmt)
            zhat = ops.checkpoint8_restore(zc, fmt, N, M, torch.float32).double().cpu()
            assert torch.equal(zhat, codes64(zk.cpu(), fmt, act == "relu"))
            assert torch.equal(xcodes[:, :D], checkpoint8(xc, fmt).data[:, :D])
            if act == "relu":
                assert torch.equal(torch.sign(zhat), torch.sign(zk.double().cpu()))
        xhat = codes64(x, fmt) if fmt else x
        want = backward64(x, W, b, act, g, zhat, xhat, dtype, dtype, 0.0)
        names = [n for n, t in zip("xWbr", leaves) if t is not None]
        for n, got in zip(names, grads):
            if n == "r":
                assert got.dtype == rc.dtype and torch.equal(got.cpu(), g.to(rc.dtype))
            else:
                assert got.dtype == dtype
                assert_within(got, *want[n], f"d{n} {act} {N}x{D}x{M}")


@pytest.mark.parametrize("act", ["none", "gelu", "silu"])
@pytest.mark.parametrize("fmt", [None, "int8"])
def test_gradient_against_differences(device, act, fmt):
    """Directional derivatives of the fp32 op itself. x holds whole numbers up to 100, which "int8" keeps exactly; the
    second difference of a smooth activation is below 0.8 |dz|^2, sums are off by K 2^-23."""
    from sparsify_amd import fused_linear
    g = torch.Generator().manual_seed(0)
    N, D, M = 48, 40, 36
    x = torch.randint(-100, 101, (N, D), generator=g).float()
    x[::32] = 100.0
    W = torch.randn(M, D, generator=g) / 300
    b = torch.randn(M, generator=g)
    r = torch.randn(N, M, generator=g)
    c = torch.randn(N, M, generator=g)
    x, W, b, r, c = cuda(x, W, b, r, c)
    leaves = [t.clone().requires_grad_() for t in (x, W, b, r)]
    y = fused_linear(*leaves[:3], residual=leaves[3], activation=act, checkpoint=fmt)
    grads = torch.autograd.grad(y, leaves, c)

    def f(ts):
        return (fused_linear(*ts[:3], residual=ts[3], activation=act).double() * c.double()).sum()

    h = 2.0**-6
    for i, t in enumerate((x, W, b, r)):
        v = torch.randn(t.shape, generator=g).cuda() / (300 if i == 1 else 1)
        if i == 0 and fmt:
            continue                                           # z is in 8 bits: dx is the gradient at the restored z
        ts = [x, W, b, r]
        up, dn = list(ts), list(ts)
        up[i], dn[i] = t + h * v, t - h * v
        num = (f(up) - f(dn)) / (2 * h)
        # what each argument's direction does to z, and the 8-bit z's error of 1/127 of its group's maximum
        dz = {0: lambda: v @ W.t(), 1: lambda: x @ v.t(), 2: lambda: v.expand(N, M), 3: lambda: torch.zeros(N, M).cuda()}[i]().double()
        z = x.double() @ W.double().t() + b.double()
        trunc = 0.8 / 6 * 8 * h * h * (dz.abs() ** 3 * c.abs()).sum() if act != "none" else 0.0
        noise = (D + 4) * 2.0**-23 * ((x.abs() @ W.abs().t() + b.abs() + r.abs()).double() * c.abs()).sum() / h
        kept = 0.8 / 127 * (z.abs().max() * dz.abs() * c.abs()).sum() if fmt and act != "none" else 0.0
        got = (grads[i].double() * v.double()).sum()
        assert abs(float(got - num)) <= float(trunc + noise + kept) + 1e-3, (i, float(got), float(num))


@pytest.mark.parametrize("N,D,M", [(256, 64, 256), (300, 128, 520), (1000, 192, 704), (64, 1024, 136), (257, 256, 255), (1030, 320, 1000),
                                   (2048, 128, 257), (1, 64, 64), (129, 129, 129), (700, 77, 1001), (33, 1000, 3)])
@pytest.mark.parametrize("kernel", ["64", "128", "256", "few"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_every_product_kernel(device, monkeypatch, N, D, M, kernel, dtype):
    """Each of the product's kernels on small and ragged shapes (SPHIP_LINEAR): forward, and both gradient products with
    their K-strided operands, packed or as they are, split over K and whole, against the definition."""
    from sparsify_amd import ops
    if kernel == "few" and N > 64:
        N = N % 64 + 1                                 # (the kernel for few rows)
    monkeypatch.setenv("SPHIP_LINEAR", kernel)
    ops._linear_bytes.cache_clear(), ops._linear_backward_bytes.cache_clear()
    try:
        for i, (act, fmt) in enumerate([("none", "int8"), ("gelu", None), ("relu", "e4m3"), ("silu", "int8")]):
            res = [None, torch.float32, dtype, None][i]
            x, W, b, r = make(N, D, M, dtype, N + i, bias=i != 1, res=res)
            out_dtype = dtype if res is None else torch.promote_types(dtype, res)
            xc, Wc, bc, rc = cuda(x, W, b, r)
            y, zk, _ = ops.linear(xc, Wc, bc, rc, act, keep_z=torch.float32)
            want, tol, z, ez = forward64(x, W, b, r, act, out_dtype)
            assert_within(y, want, tol, f"y {act}")
            assert_within(zk, z, ez + HALF[torch.float32] * z.abs() + TINY, f"z {act}")
            _, zq, xq = ops.linear(xc, Wc, bc, rc, act, keep_z=fmt or dtype, keep_x=fmt)
            zhat = ops.checkpoint8_restore(zq, fmt, N, M, torch.float32) if fmt else zq
            g = torch.randn(N, M, generator=torch.Generator().manual_seed(i)).to(out_dtype)
            dx, dW, db = ops.linear_backward(g.cuda(), Wc, zq, xq if fmt else xc, act, z_fmt=fmt, x_fmt=fmt,
                                             dx_dtype=dtype, dw_dtype=dtype, db_dtype=dtype)
            ref = backward64(x, W, torch.zeros(M, dtype=dtype), act, g, zhat.double().cpu(),
                             codes64(x, fmt) if fmt else x, dtype, dtype, 0.0)
            for n, got in (("x", dx), ("W", dW), ("b", db)):
                assert_within(got, *ref[n], f"d{n} {act} {N}x{D}x{M}")
    finally:
        monkeypatch.undo()
        ops._linear_bytes.cache_clear(), ops._linear_backward_bytes.cache_clear()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
def test_kept_z_near_the_largest_value(device, fmt, dtype):
    """ReLU's slopes, 0 or 1, and the sums of up to 64 of them are whole numbers: exact."""
    from sparsify_amd import ops
    z = torch.tensor([3.0e38, -3.0e38, 1.8e38, -1.0, 0.0, 2.0**-100, 1.7e38, -1.7e38]).repeat(64, 8).to(dtype).cuda()
    q = ops.checkpoint8_save(z, fmt, True)
    g = torch.ones(64, 64, dtype=dtype, device="cuda")
    W, x = torch.eye(64, dtype=dtype, device="cuda"), torch.ones(64, 64, dtype=dtype, device="cuda")
    dx, dW, db = ops.linear_backward(g, W, q, x, "relu", z_fmt=fmt, dx_dtype=dtype, dw_dtype=dtype, db_dtype=dtype)
    want = (z > 0).to(dtype)
    assert torch.equal(dx, want)
    assert torch.equal(db, want.sum(0)) and torch.equal(dW, want.T @ x)


@pytest.mark.parametrize("N,D,M", [(300, 72, 88), (70, 1000, 328), (513, 200, 520)])
@pytest.mark.parametrize("kernel", ["64", "128", "256", "few"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_nothing_behind_a_row_is_multiplied(device, monkeypatch, N, D, M, kernel, dtype):
    """Rows that are whole 16-byte pieces but no whole number of K steps, inside larger tensors of NaN."""
    from sparsify_amd import ops
    if kernel == "few":
        N = N % 64 + 1
    monkeypatch.setenv("SPHIP_LINEAR", kernel)
    ops._linear_bytes.cache_clear(), ops._linear_backward_bytes.cache_clear()

    def framed(t, left):
        big = torch.full((t.shape[0] + 2, t.shape[1] + left + 24), math.nan, dtype=t.dtype, device="cuda")
        big[1:-1, left : left + t.shape[1]] = t.cuda()
        return big[1:-1, left : left + t.shape[1]]

    try:
        x, W, _, _ = make(N, D, M, dtype, 5, bias=False)
        g = torch.randn(N, M, generator=torch.Generator().manual_seed(6)).to(dtype)
        for left in (16, 3):                              # on 16-byte boundaries, and off them
            xc, Wc, gc = framed(x, left), framed(W, left), framed(g, left)
            y, _, _ = ops.linear(xc, Wc)
            want, tol, _, _ = forward64(x, W, None, None, "none", dtype)
            assert_within(y, want, tol, f"y {left}")
            dx, dW, db = ops.linear_backward(gc, Wc, None, xc, "none", dx_dtype=dtype, dw_dtype=dtype, db_dtype=dtype)
            ref = backward64(x, W, torch.zeros(M, dtype=dtype), "none", g, torch.zeros(N, M).double(), x, dtype, dtype, 0.0)
            for n, got in (("x", dx), ("W", dW), ("b", db)):
                assert_within(got, *ref[n], f"d{n} {left}")
            dx, dW, _ = ops.linear_backward(gc, Wc, None, xc, "none", dx_dtype=dtype, dw_dtype=dtype)
            for n, got in (("x", dx), ("W", dW)):
                assert_within(got, *ref[n], f"d{n} alone {left}")
    finally:
        monkeypatch.undo()
        ops._linear_bytes.cache_clear(), ops._linear_backward_bytes.cache_clear()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [40, 770, 2048, 3001])
@pytest.mark.parametrize("N", [1, 9, 16, 17, 32, 33, 64])
def test_few_rows_of_a_wide_layer(device, monkeypatch, N, D, dtype):
    """The kernel for few rows with 32 rows of W per workgroup (M from 8161 on), forced and as it is chosen."""
    from sparsify_amd import ops
    M = 8197
    x, W, b, r = make(N, D, M, dtype, D + N, res=torch.float32)
    want, tol, z, ez = forward64(x, W, b, r, "gelu", torch.float32)
    xc, Wc, bc, rc = cuda(x, W, b, r)
    try:
        for kernel in ("few", None):
            if kernel:
                monkeypatch.setenv("SPHIP_LINEAR", kernel)
            else:
                monkeypatch.undo()
            ops._linear_bytes.cache_clear()
            y, zk, _ = ops.linear(xc, Wc, bc, rc, "gelu", keep_z=torch.float32)
            assert_within(y, want, tol, f"y {kernel}")
            assert_within(zk, z, ez + HALF[torch.float32] * z.abs() + TINY, f"z {kernel}")
            _, zq, _ = ops.linear(xc, Wc, bc, rc, "gelu", keep_z="int8")
            assert torch.equal(ops.checkpoint8_restore(zq, "int8", N, M, torch.float32).double().cpu(), codes64(zk.cpu(), "int8"))
    finally:
        monkeypatch.undo()
        ops._linear_bytes.cache_clear()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("fmt", [None, "e4m3"])
def test_rows_far_apart(device, dtype, fmt):
    """Rows 2^22 elements apart lie behind a tile's descriptor: copied first, the same bits as from dense rows."""
    from sparsify_amd import fused_linear
    x, W, b, _ = make(130, 200, 72, dtype, 3)
    ld = (1 << 22) + 8

    def far(t):
        big = torch.empty(t.shape[0], ld, dtype=dtype, device="cuda")
        big[:, :8], big[:, 8 + t.shape[1] : 64 + t.shape[1]] = math.nan, math.nan
        big[:, 8 : 8 + t.shape[1]] = t.cuda()
        return big[:, 8 : 8 + t.shape[1]]

    g = torch.randn(130, 72, device="cuda").to(dtype)
    outs = []
    for xi, wi in ((x.cuda(), W.cuda()), (far(x), W.cuda()), (x.cuda(), far(W)), (far(x), far(W))):
        ts = [t.detach().requires_grad_() for t in (xi, wi, b.cuda())]
        y = fused_linear(*ts, activation="gelu", checkpoint=fmt)
        outs.append((y.detach(), *torch.autograd.grad(y, ts, g)))
    for o in outs[1:]:
        for a, c in zip(o, outs[0]):
            assert torch.equal(a, c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N", [3, 20, 70])
def test_longest_rows(device, dtype, N):
    """2^22 - 65 features, the most that is taken, on either side; sums of -1, 0 and 1 are whole numbers below 2^24: exact."""
    from sparsify_amd import ops
    most, few = (1 << 22) - 65, 5
    gen = torch.Generator("cuda").manual_seed(N)
    a, b = (torch.randint(-1, 2, (n, most), device="cuda", generator=gen).to(dtype) for n in (N, few))
    want = torch.stack([(a.float() * r.float()).sum(1, dtype=torch.float64) for r in b], 1)
    y, _, _ = ops.linear(a, b, out_dtype=torch.float32)                            # K = most
    assert torch.equal(y.double(), want)
    W = b.t().contiguous()                                                         # (most, few)
    dx, _, _ = ops.linear_backward(a, W, None, None, dx_dtype=torch.float32)       # K = most, W's columns
    assert torch.equal(dx.double(), want)
    x = torch.randint(-1, 2, (N, few), device="cuda", generator=gen).to(dtype)
    _, dW, db = ops.linear_backward(a, W, None, x, dw_dtype=torch.float32, db_dtype=torch.float32)
    assert torch.equal(db.double(), a.sum(0, dtype=torch.float64))
    assert torch.equal(dW.double(), torch.stack([(a.float() * c[:, None].float()).sum(0, dtype=torch.float64) for c in x.t()], 1))


def test_only_the_asked_gradients_and_reuse(device):
    from sparsify_amd import checkpoint8, fused_linear
    x, W, b, r = cuda(*make(200, 96, 64, torch.bfloat16, 4, res=torch.float32))
    full = [t.clone().requires_grad_() for t in (x, W, b, r)]
    y = fused_linear(*full[:3], residual=full[3], activation="gelu", checkpoint="int8")
    g = torch.randn_like(y)
    want = torch.autograd.grad(y, full, g, retain_graph=True)
    again = torch.autograd.grad(y, full, g)                      # nothing was consumed
    for a, c in zip(want, again):
        assert torch.equal(a, c)
    for i in range(4):
        ts = [t.clone().requires_grad_(j == i) for j, t in enumerate((x, W, b, r))]
        y = fused_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint="int8")
        (got,) = torch.autograd.grad(y, [ts[i]], g)
        assert torch.equal(got, want[i]), i
    c = checkpoint8(x, "int8")                                   # a checkpoint that exists already
    ts = [t.clone().requires_grad_() for t in (x, W, b, r)]
    y = fused_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint=c)
    for a, t in zip(torch.autograd.grad(y, ts, g), want):
        assert torch.equal(a, t)
    y = fused_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint="int8")
    loss = (y * y).sum()                                         # a broadcast incoming gradient, then its gradient refused
    (dx,) = torch.autograd.grad(y.sum(), [ts[0]], retain_graph=True)
    assert torch.isfinite(dx).all()
    with pytest.raises(RuntimeError):
        (d,) = torch.autograd.grad(loss, [ts[0]], create_graph=True)
        d.sum().backward()


def test_autocast_and_master_weights(device):
    """fp32 parameters under bf16 autocast: the product runs on bf16 copies, gradients come back in fp32, unrounded."""
    from sparsify_amd import fused_linear
    x, W, b, _ = make(100, 72, 48, torch.float32, 9)
    xc, Wc, bc = [t.cuda().requires_grad_() for t in (x, W, b)]
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = fused_linear(xc, Wc, bc, activation="none", checkpoint="e4m3")
    assert y.dtype == torch.bfloat16
    xb, Wb = x.bfloat16(), W.bfloat16()
    want, tol, _, _ = forward64(xb, Wb, b, None, "none", torch.bfloat16)
    assert_within(y.detach(), want, tol)
    g = torch.randn(100, 48, generator=torch.Generator().manual_seed(1)).bfloat16()
    dx, dW, db = torch.autograd.grad(y, [xc, Wc, bc], g.cuda())
    assert dx.dtype == dW.dtype == db.dtype == torch.float32
    ref = backward64(xb, Wb, b, "none", g, want, codes64(xb, "e4m3"), torch.float32, torch.bfloat16, 0.0)
    assert_within(dx, *ref["x"])
    dW64 = g.double().T @ codes64(xb, "e4m3")
    assert_within(dW, dW64, 104 * 2.0**-23 * (g.double().abs().T @ codes64(xb, "e4m3").abs()) + TINY)
    assert_within(db, *ref["b"])


def test_empty_batch(device):
    from sparsify_amd import fused_linear
    W, b = torch.randn(5, 8, device="cuda", requires_grad=True), torch.randn(5, device="cuda", requires_grad=True)
    x = torch.zeros(2, 0, 8, device="cuda", requires_grad=True)
    for fmt in (None, "int8"):
        y = fused_linear(x, W, b, activation="gelu", checkpoint=fmt)
        assert y.shape == (2, 0, 5)
        dx, dW, db = torch.autograd.grad(y, [x, W, b], torch.zeros_like(y))
        assert dx.shape == x.shape and not dW.any() and not db.any()


def test_empty_batch_with_an_expanded_gradient(device):
    """The gradient of a sum is one value, expanded: strides of zero, also where there are no rows."""
    from sparsify_amd import fused_linear
    for lead in ((0,), (3,), (2, 0), (2, 5)):
        ts = [t.requires_grad_() for t in cuda(torch.randn(*lead, 40), torch.randn(24, 40), torch.randn(24))]
        for fmt in (None, "int8"):
            y = fused_linear(*ts, activation="silu", checkpoint=fmt)
            got = torch.autograd.grad(y.sum(), ts)
            want = torch.autograd.grad(fused_linear(*ts, activation="silu", checkpoint=fmt), ts, torch.ones_like(y))
            for a, c, t in zip(got, want, ts):
                assert a.shape == t.shape and torch.equal(a, c)


def test_masked_rows_of_a_padded_batch(device):
    """Rows behind the last sequence (zero gradient) add nothing to dW and db and get a zero dx, whatever finite values
    they hold; whole groups of 32 of them may hold anything that "none" or "relu" passes on."""
    from sparsify_amd import fused_linear
    x, W, b, _ = cuda(*make(96, 64, 48, torch.bfloat16, 6))
    g = torch.randn(96, 48, device="cuda").bfloat16()
    g[64:] = 0
    for fmt in (None, "int8", "e4m3"):
        outs = []
        for fill in (0.0, 1e4):
            xi = x.clone()
            xi[64:] = fill
            ts = [t.clone().requires_grad_() for t in (xi, W, b)]
            y = fused_linear(*ts, activation="silu", checkpoint=fmt)
            outs.append(torch.autograd.grad(y, ts, g))
        for a, c in zip(*outs):
            assert torch.equal(a, c)
        assert not outs[0][0][64:].any()


# ------------------------------------------------------------------ streams and graphs
def test_two_streams_at_once(device):
    from sparsify_amd import fused_linear
    sets = [cuda(*make(300, 700, 90, torch.bfloat16, s, res=torch.float32)) for s in range(2)]

    def step(x, W, b, r):
        ts = [t.detach().clone().requires_grad_() for t in (x, W, b, r)]
        y = fused_linear(*ts[:3], residual=ts[3], activation="silu", checkpoint="int8")
        return (y.detach(), *torch.autograd.grad(y, ts, torch.ones_like(y)))

    want = [step(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for _ in range(5):
        for st, s in zip(streams, sets):
            with torch.cuda.stream(st):
                got.append(step(*s))
    torch.cuda.synchronize()
    for i, outs in enumerate(got):
        for a, c in zip(outs, want[i % 2]):
            assert torch.equal(a, c)


def test_captured_steps_replay(device):
    """Forward and gradients of two captured graphs (they share no scratch), replayed between eager calls."""
    from sparsify_amd import fused_linear
    graphs = []
    side = torch.cuda.Stream()

    def step(ts, g):
        y = fused_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint="e4m3")
        return (y.detach(), *torch.autograd.grad(y, ts, g))

    def inputs(seed):
        ts = [t.requires_grad_() for t in cuda(*make(130, 1500, 70, torch.bfloat16, seed, res=torch.bfloat16))]
        return ts, torch.randn(130, 70, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).bfloat16()

    for seed in range(2):
        ts, g = inputs(seed)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            step(ts, g)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs = step(ts, g)
        graphs.append((graph, ts, g, outs))
    for seed in (5, 6, 7):
        for graph, ts, g, outs in graphs:
            new, ng = inputs(seed)
            with torch.no_grad():
                for t, n in zip(ts, new):
                    t.copy_(n)
                g.copy_(ng)
        other = torch.cuda.Stream()
        other.wait_stream(torch.cuda.current_stream())
        graphs[0][0].replay()
        with torch.cuda.stream(other):
            graphs[1][0].replay()
        torch.cuda.current_stream().wait_stream(other)
        want = step(*inputs(seed))
        torch.cuda.synchronize()
        for _, _, _, outs in graphs:
            for a, c in zip(outs, want):
                assert torch.equal(a, c)


def test_same_bits_every_time(device):
    from sparsify_amd import fused_linear
    x, W, b, r = cuda(*make(777, 900, 200, torch.bfloat16, 8, res=torch.bfloat16))
    first = None
    for _ in range(4):
        ts = [t.clone().requires_grad_() for t in (x, W, b, r)]
        y = fused_linear(*ts[:3], residual=ts[3], activation="gelu", checkpoint="int8")
        outs = (y.detach(), *torch.autograd.grad(y, ts, torch.full_like(y, 0.25)))
        first = first or outs
        for a, c in zip(outs, first):
            assert torch.equal(a, c)


# ------------------------------------------------------------------ offsets past 32 bits
def test_more_than_two_to_the_31_elements(device):
    from sparsify_amd import checkpoint8, fused_linear
    N, D, M = 70000, 64, 32768
    g = torch.Generator("cuda").manual_seed(0)
    x = torch.randn(N, D, device="cuda", generator=g).bfloat16()
    W = (torch.randn(M, D, device="cuda", generator=g) / 8).bfloat16()
    y = fused_linear(x, W, activation="relu")
    pick = torch.cat([torch.arange(3), torch.arange(65530, 65540), torch.arange(N - 40, N)]).cuda()
    want, tol, _, _ = forward64(x[pick].cpu(), W.cpu(), None, None, "relu", torch.bfloat16)
    assert_within(y[pick], want, tol)
    c = checkpoint8(y, "int8")
    back = c.restore()
    lo = N // 32 * 32 - 64
    assert torch.equal(back[lo:].double().cpu(), codes64(y[lo:].cpu(), "int8"))
    del back, c
    # the same matrix as an incoming gradient: dW and dx contract over and along its rows
    xr, Wr = x.clone().requires_grad_(), W.clone().requires_grad_()
    out = fused_linear(xr, Wr, checkpoint="e4m3")
    gy = y.clamp_(max=1.0)
    keep = torch.zeros(N, dtype=torch.bool, device="cuda")
    keep[pick] = True
    gy[~keep] = 0
    dx, dW = torch.autograd.grad(out, [xr, Wr], gy)
    gp = gy[pick].double().cpu()
    assert not dx[~keep].any()
    wd = W.double().cpu()
    t = (M + 4) * 2.0**-23 * (gp.abs() @ wd.abs())
    assert_within(dx[pick], gp @ wd, t + 2.0**-8 * ((gp @ wd).abs() + t) + TINY)
    xs = torch.cat([codes64(x[i // 32 * 32:i // 32 * 32 + 32].cpu(), "e4m3")[i % 32][None] for i in pick.tolist()])
    t = 200 * 2.0**-23 * (gp.abs().T @ xs.abs())
    assert_within(dW, gp.T @ xs, t + 2.0**-8 * ((gp.T @ xs).abs() + t) + TINY)
