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
             out_dtype=BF16, ldo=32, z=None, z_dtype=0, ldz=0, N=8, D=64, M=32, ws=None, nws=0)
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
    (dict(D=4096, ldx=4096, ldw=4096, ws=P + 4, nws=1 << 30), EWORKSPACE, b"aligned")])
def test_linear_entry(kw, status, word):
    assert linear(**kw) == status and word in lib().sphip_last_error()


def test_gradient_entries():
    L = lib()

    def preact(g=P, g_dtype=BF16, ldg=32, z=None, kind=0, sc=None, ldz=0, act=0, dz=P, dz_dtype=BF16, lddz=32, db=None, db_dtype=0,
               N=8, M=32, ws=None, nws=0):
        return L.sphip_linear_grad_preact(g, g_dtype, ldg, z, kind, sc, ldz, act, dz, dz_dtype, lddz, db, db_dtype, N, M, ws, nws, None)

    for kw, st in [(dict(g=None), EINVAL), (dict(dz=None), EINVAL), (dict(act=9), EINVAL), (dict(act=2), EINVAL),
                   (dict(act=2, z=P, kind=5, ldz=32), EINVAL), (dict(act=2, z=P, kind=INT8, ldz=32), EINVAL),
                   (dict(act=2, z=P, kind=INT8, sc=P, ldz=40), EINVAL), (dict(act=2, z=P, kind=F32, ldz=31), EINVAL),
                   (dict(lddz=33), EINVAL), (dict(lddz=28), EINVAL), (dict(ldg=8), EINVAL), (dict(dz=P + 8), EINVAL),
                   (dict(N=0), EINVAL), (dict(db=P, db_dtype=F32), EWORKSPACE), (dict(db=P, db_dtype=3), EINVAL)]:
        assert preact(**kw) == st, kw

    def gin(dz=P, lddz=32, W=P, ldw=64, dtype=BF16, dx=P, dx_dtype=BF16, lddx=64, N=8, D=64, M=32, ws=None, nws=0):
        return L.sphip_linear_grad_input(dz, lddz, W, ldw, dtype, dx, dx_dtype, lddx, N, D, M, ws, nws, None)

    for kw, st in [(dict(dz=None), EINVAL), (dict(W=None), EINVAL), (dict(dx=None), EINVAL), (dict(dtype=16), EINVAL),
                   (dict(lddz=31), EINVAL), (dict(ldw=63), EINVAL), (dict(lddx=63), EINVAL), (dict(M=0), EINVAL),
                   (dict(D=1 << 31, ldw=1 << 31, lddx=1 << 31), EUNSUPPORTED), (dict(dx=P + 1), EINVAL),
                   (dict(M=4096, lddz=4096), EWORKSPACE)]:
        assert gin(**kw) == st, kw

    def gw(dz=P, lddz=32, dtype=BF16, x=P, sc=None, kind=BF16, ldx=64, dW=P, dw_dtype=BF16, lddw=64, N=8, D=64, M=32, ws=None, nws=0):
        return L.sphip_linear_grad_weight(dz, lddz, dtype, x, sc, kind, ldx, dW, dw_dtype, lddw, N, D, M, ws, nws, None)

    for kw, st in [(dict(dz=None), EINVAL), (dict(x=None), EINVAL), (dict(dW=None), EINVAL), (dict(kind=F32), EINVAL),
                   (dict(kind=INT8), EINVAL), (dict(kind=E4M3, sc=P, ldx=72), EINVAL), (dict(kind=INT8, sc=P + 4), EINVAL),
                   (dict(kind=18, sc=P), EINVAL), (dict(lddz=1), EINVAL), (dict(ldx=63), EINVAL), (dict(lddw=63), EINVAL),
                   (dict(N=0), EINVAL), (dict(N=1 << 20), EWORKSPACE)]:
        assert gw(**kw) == st, kw
    assert L.sphip_linear_workspace_bytes(0, 8, 8) == 0 and L.sphip_linear_workspace_bytes(8, -1, 8) == 0
    assert L.sphip_linear_grad_weight_workspace_bytes(1 << 20, 64, 32) > 0


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
    codes, scales = torch.zeros(32, 16, dtype=torch.uint8), torch.zeros(1, 16, dtype=torch.uint8)
    c = Checkpoint8(codes, scales, "int8", (3, 8), torch.float32)
    assert c.rows == 3 and c.columns == 8 and c.nbytes == 33 * 16
    with pytest.raises(ValueError, match="checkpoint holds"):
        fused_linear(x, W, checkpoint=c)
    with pytest.raises(RuntimeError, match="no CPU fallback"):
        c.restore()
