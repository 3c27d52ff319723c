"""What fused_linear, the 8-bit checkpoints and their C entry points refuse, before anything is launched (no GPU needed:
shapes, types, strides, alignments and workspaces are checked on the host)."""
import pytest
import torch

EINVAL, EUNSUPPORTED, EWORKSPACE = 1, 2, 4
F32, BF16, INT8, E4M3 = 0, 1, 16, 17
P = 1 << 20                      # an address that is aligned and never read


def lib():
    from sparsify_amd import _lib
    return _lib.load()


def linear(**kw):
    a = dict(x=P, ldx=64, W=P, ldw=64, dtype=BF16, bias=None, bias_dtype=0, act=0, res=None, res_dtype=0, ldr=0, out=P,
             out_dtype=BF16, ldo=32, z=None, z_kind=0, z_scales=None, ldz=0, xc=None, xs=None, x_fmt=0, ldq=0, N=80, D=64, M=32,
             ws=None, nws=0)
    assert set(kw) <= set(a)
    return lib().sphip_linear(*{**a, **kw}.values(), None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(x=None), EINVAL, b"null"), (dict(W=None), EINVAL, b"null"), (dict(out=None), EINVAL, b"null"),
    (dict(dtype=2), EINVAL, b"dtype"), (dict(out_dtype=-1), EINVAL, b"dtype"), (dict(bias=P, bias_dtype=7), EINVAL, b"dtype"),
    (dict(act=4), EINVAL, b"activation"), (dict(act=-1), EINVAL, b"activation"),
    (dict(N=0), EINVAL, b"empty"), (dict(D=0), EINVAL, b"empty"), (dict(M=-3), EINVAL, b"empty"),
    (dict(N=1 << 31), EUNSUPPORTED, b"int32"), (dict(ldx=63), EINVAL, b"stride"), (dict(ldw=10), EINVAL, b"stride"),
    (dict(ldo=31), EINVAL, b"stride"), (dict(res=P, ldr=31), EINVAL, b"stride"), (dict(z=P, ldz=8), EINVAL, b"stride"),
    (dict(x=P + 1), EINVAL, b"aligned"), (dict(out=P + 2, out_dtype=F32), EINVAL, b"aligned"),
    (dict(bias=P + 1, bias_dtype=BF16), EINVAL, b"aligned"), (dict(D=4096, ldx=4096, ldw=4096), EWORKSPACE, b"workspace"),
    (dict(D=4096, ldx=4096, ldw=4096, ws=P + 4, nws=1 << 30), EWORKSPACE, b"aligned"),
    (dict(z=P, z_kind=9, ldz=32), EINVAL, b"dtype"), (dict(z=P, z_kind=INT8, ldz=32), EINVAL, b"codes"),
    (dict(z=P, z_kind=E4M3, z_scales=P, ldz=40), EINVAL, b"codes"), (dict(z=P + 8, z_kind=INT8, z_scales=P, ldz=32), EINVAL, b"codes"),
    (dict(z=P, z_kind=INT8, z_scales=P, ldz=32, D=4096, ldx=4096, ldw=4096), EWORKSPACE, b"workspace"), (dict(xc=P, x_fmt=BF16), EINVAL, b"dtype"),
    (dict(xc=P, x_fmt=INT8, ldq=64), EINVAL, b"codes"), (dict(xc=P, xs=P, x_fmt=INT8, ldq=48), EINVAL, b"codes")])
def test_linear_entry(kw, status, word):
    assert linear(**kw) == status and word in lib().sphip_last_error()


def backward(**kw):
    a = dict(g=P, g_dtype=BF16, ldg=32, W=P, ldw=64, dtype=BF16, act=0, z=None, z_kind=0, z_scales=None, ldz=0, x=P, x_kind=BF16,
             x_scales=None, ldx=64, dx=P, dx_dtype=BF16, lddx=64, dW=P, dw_dtype=BF16, lddw=64, db=None, db_dtype=0, N=8, D=64, M=32,
             ws=None, nws=0)
    assert set(kw) <= set(a)
    return lib().sphip_linear_backward(*{**a, **kw}.values(), None)


@pytest.mark.parametrize("kw,status,word", [
    (dict(g=None), EINVAL, b"null"), (dict(W=None), EINVAL, b"null"), (dict(x=None), EINVAL, b"null"),
    (dict(dx=None, dW=None), EINVAL, b"null"), (dict(dtype=5), EINVAL, b"dtype"), (dict(g_dtype=INT8), EINVAL, b"dtype"),
    (dict(db=P, db_dtype=3), EINVAL, b"dtype"), (dict(act=4), EINVAL, b"activation"), (dict(act=2), EINVAL, b"needs z"),
    (dict(act=2, z=P, z_kind=5, ldz=32), EINVAL, b"needs z"), (dict(act=2, z=P, z_kind=F32, ldz=31), EINVAL, b"stride"),
    (dict(act=1, z=P, z_kind=INT8, ldz=32), EINVAL, b"codes"), (dict(act=1, z=P, z_kind=INT8, z_scales=P, ldz=40), EINVAL, b"codes"),
    (dict(x_kind=F32), EINVAL, b"product's type"), (dict(x_kind=18), EINVAL, b"product's type"), (dict(x_kind=E4M3), EINVAL, b"codes"),
    (dict(x_kind=INT8, x_scales=P, ldx=72), EINVAL, b"codes"), (dict(x=P + 4, x_kind=INT8, x_scales=P), EINVAL, b"codes"),
    (dict(ldg=31), EINVAL, b"stride"), (dict(ldw=63), EINVAL, b"stride"), (dict(lddx=63), EINVAL, b"stride"),
    (dict(ldx=63), EINVAL, b"stride"), (dict(lddw=1), EINVAL, b"stride"), (dict(dx=P + 1), EINVAL, b"aligned"),
    (dict(g=P + 2, g_dtype=F32), EINVAL, b"aligned"), (dict(N=0), EINVAL, b"empty"), (dict(M=1 << 31, ldg=1 << 31), EUNSUPPORTED, b"int32"),
    (dict(), EWORKSPACE, b"workspace"), (dict(ws=P + 8, nws=1 << 30), EWORKSPACE, b"aligned"),
    (dict(dx=None, dW=None, db=P, db_dtype=F32), EWORKSPACE, b"workspace")])
def test_backward_entry(kw, status, word):
    assert backward(**kw) == status and word in lib().sphip_last_error()


def test_workspace_queries():
    L = lib()
    assert L.sphip_linear_workspace_bytes(BF16, 0, 0, 8, 8, 0) == 0 and L.sphip_linear_workspace_bytes(9, 0, 8, 8, 8, 0) == 0
    assert (L.sphip_linear_workspace_bytes(BF16, INT8, 80, 4096, 32, 0)
            >= L.sphip_linear_workspace_bytes(BF16, F32, 80, 4096, 32, 0) + 80 * 32 * 4)
    assert L.sphip_linear_workspace_bytes(BF16, INT8, 80, 64, 32, 0) == 0 and L.sphip_linear_workspace_bytes(BF16, F32, 8, 4096, 32, 0) == 0
    assert L.sphip_linear_backward_workspace_bytes(BF16, INT8, 0, 0, 1, 64, 64, 32, 3) == 2 * 32 * 4
    assert L.sphip_linear_backward_workspace_bytes(F32, F32, 1, 1, 1, 8, -1, 32, 0) == 0
    # copies: of the operands that are named, of both where rows are no whole 16-byte pieces
    for odd, rows in [(0, 0), (1, 80), (2, 40), (3, 120)]:
        assert L.sphip_linear_workspace_bytes(BF16, F32, 80, 72, 40, odd) == rows * 128 * 2
        assert L.sphip_linear_workspace_bytes(BF16, F32, 80, 71, 40, odd) == 120 * 128 * 2
        want = L.sphip_linear_backward_workspace_bytes(F32, F32, 1, 1, 0, 64, 64, 64, 0)
        assert L.sphip_linear_backward_workspace_bytes(F32, F32, 1, 1, 0, 64, 64, 64, odd) == want + 64 * 64 * 4 * bin(odd).count("1")


def test_longest_rows():
    most = (1 << 22) - 65
    assert linear(D=most, ldx=most, ldw=most) == EWORKSPACE
    for kw in (dict(D=most + 1, ldx=most + 1, ldw=most + 1), dict(M=most + 1, ldo=most + 1)):
        assert linear(**kw) == EUNSUPPORTED and b"2^22" in lib().sphip_last_error()
    for kw in (dict(D=most + 1, ldx=most + 1, ldw=most + 1, lddx=most + 1, lddw=most + 1), dict(M=most + 1, ldg=most + 1)):
        assert backward(**kw) == EUNSUPPORTED and b"2^22" in lib().sphip_last_error()


def test_more_work_than_a_launch_holds():
    N = (1 << 31) - 300
    assert linear(N=N, M=4096, ldo=4096) == EUNSUPPORTED and b"grid" in lib().sphip_last_error()
    L = lib()
    assert L.sphip_checkpoint8_save(P, BF16, 64, INT8, 0, P, P, 64, N, 64, None) == EUNSUPPORTED and b"grid" in L.sphip_last_error()
    assert L.sphip_checkpoint8_restore(P, P, 256, INT8, P, BF16, 256, N, 256, None) == EUNSUPPORTED and b"grid" in L.sphip_last_error()
    nws = L.sphip_linear_backward_workspace_bytes(BF16, BF16, 0, 0, 1, N, 64, 32, 0)
    assert backward(N=N, dx=None, dW=None, db=P, db_dtype=F32, ws=P, nws=nws) == EUNSUPPORTED and b"grid" in L.sphip_last_error()


def test_checkpoint_entries():
    L = lib()

    def save(x=P, dtype=BF16, ldx=64, fmt=INT8, keep=0, codes=P, scales=P, ldq=64, N=8, D=64):
        return L.sphip_checkpoint8_save(x, dtype, ldx, fmt, keep, codes, scales, ldq, N, D, None)

    for kw in [dict(x=None), dict(codes=None), dict(scales=None), dict(dtype=3), dict(fmt=1), dict(fmt=18), dict(ldx=63), dict(ldq=48),
               dict(ldq=72), dict(codes=P + 8), dict(scales=P + 1), dict(N=0), dict(D=0), dict(x=P + 1), dict(N=1 << 31)]:
        assert save(**kw) == EINVAL, kw

    def restore(codes=P, scales=P, ldq=64, fmt=E4M3, out=P, dtype=F32, ldo=64, N=8, D=64):
        return L.sphip_checkpoint8_restore(codes, scales, ldq, fmt, out, dtype, ldo, N, D, None)

    for kw in [dict(out=None), dict(codes=None), dict(scales=None), dict(dtype=2), dict(fmt=0), dict(ldo=63), dict(ldq=80, D=81),
               dict(out=P + 2), dict(N=-1)]:
        assert restore(**kw) == EINVAL, kw


def test_python_surface_refuses_on_the_host():
    from sparsify_amd import Checkpoint8, checkpoint8, fused_linear
    x, W = torch.randn(4, 8), torch.randn(5, 8)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_linear(x, W)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        fused_linear(x.requires_grad_(), W, checkpoint="int8")
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        checkpoint8(x)
    with pytest.raises(ValueError, match="Unknown activation"):
        fused_linear(x, W, activation="tanh")
    with pytest.raises(ValueError, match="8-bit format"):
        fused_linear(x, W, checkpoint="e5m2")
    with pytest.raises(ValueError, match="8-bit format"):
        checkpoint8(x, "int4")
    with pytest.raises(ValueError, match="does not go with weight"):
        fused_linear(x, torch.randn(5, 9))
    with pytest.raises(ValueError, match="does not go with weight"):
        fused_linear(x, torch.randn(0, 8))
    with pytest.raises(ValueError, match="bias"):
        fused_linear(x, W, torch.randn(4))
    with pytest.raises(ValueError, match="residual"):
        fused_linear(x, W, residual=torch.randn(5))
    with pytest.raises(ValueError, match="scalar"):
        checkpoint8(torch.tensor(1.0))
    c = Checkpoint8(torch.zeros(33, 16, dtype=torch.uint8), "int8", (3, 8), torch.float32)
    assert c.rows == 3 and c.columns == 8 and c.nbytes == 33 * 16
    with pytest.raises(ValueError, match="checkpoint holds"):
        fused_linear(x, W, checkpoint=c)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        c.restore()


def test_the_training_switch():
    from sparsify_amd import SparseCoderConfig, TrainConfig
    assert TrainConfig(sae=SparseCoderConfig()).checkpoint_8bit is None
    assert TrainConfig(sae=SparseCoderConfig(), checkpoint_8bit="int8").checkpoint_8bit == "int8"
    with pytest.raises(ValueError, match="checkpoint_8bit"):
        TrainConfig(sae=SparseCoderConfig(), checkpoint_8bit="fp8")
    with pytest.raises(ValueError, match="shard_latents"):
        TrainConfig(sae=SparseCoderConfig(), checkpoint_8bit="int8", shard_latents=True)


def test_a_gradient_of_x_needs_the_weight_in_the_products_type(monkeypatch):
    from sparsify_amd import ops
    monkeypatch.setattr(ops, "_rows", lambda t, name, shape=None, like=None: (P, t.shape[1], ops._dt(t)))
    g, W = torch.zeros(4, 5), torch.zeros(5, 8)
    with pytest.raises(ValueError, match="products in torch.bfloat16 with a weight of torch.float32"):
        ops.linear_backward(g, W, None, None, dx_dtype=torch.float32, dtype=torch.bfloat16)


def test_the_workspace_follows_the_forced_kernel(monkeypatch):
    """SPHIP_LINEAR set to something else between two calls of one shape: each passes what the library asks for now."""
    from sparsify_amd import ops
    sizes = []
    monkeypatch.setattr(ops, "_rows", lambda t, name, shape=None, like=None: (P, t.shape[1], ops._dt(t)))
    monkeypatch.setattr(ops, "_scratch", lambda t, nbytes: sizes.append(nbytes))
    monkeypatch.setattr(ops, "_call", lambda *args: None)
    N, D, M = 64, 4096, 136
    x, W, g = (torch.zeros(s, dtype=torch.bfloat16) for s in ((N, D), (M, D), (N, M)))
    seen = set()
    for kernel in ("64", "128", "few", "256", "64"):
        monkeypatch.setenv("SPHIP_LINEAR", kernel)
        ops.linear(x, W)
        ops.linear_backward(g, W, None, x, dx_dtype=torch.bfloat16, dw_dtype=torch.bfloat16)
        want = (lib().sphip_linear_workspace_bytes(BF16, 0, N, D, M, 0),
                lib().sphip_linear_backward_workspace_bytes(BF16, BF16, 1, 1, 0, N, D, M, 0))
        assert tuple(sizes[-2:]) == want, kernel
        seen.add(want)
    assert len(seen) >= 3
