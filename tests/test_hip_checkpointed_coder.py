"""SparseCoder.checkpoint: a (skip-)transcoder's step with its input kept once, in 8 bits, for the encoder's and W_skip's
gradients, next to the same step with the input kept as it is."""
import copy

import pytest
import torch

pytestmark = pytest.mark.gpu


def grid_input(N, D, dtype, seed=0):
    """Values an int8 checkpoint keeps exactly: whole numbers up to 127 times one power of two per feature."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randint(-100, 101, (N, D), generator=g).float()
    x[::32] = 127.0
    return (x * torch.exp2(torch.randint(-8, -4, (D,), generator=g).float())).to(dtype).cuda()


def coder(D, M, k, skip=True, transcode=True, **kw):
    from sparsify_amd import SparseCoder, SparseCoderConfig
    torch.manual_seed(0)
    sae = SparseCoder(D, SparseCoderConfig(num_latents=M, k=k, transcode=transcode, skip_connection=skip, **kw)).cuda()
    g = torch.Generator().manual_seed(1)
    with torch.no_grad():
        if transcode:
            sae.W_dec.copy_(torch.randn(M, D, generator=g) / D**0.5)
        if skip:
            sae.W_skip.copy_(torch.randn(D, D, generator=g) / D**0.5)
        sae.b_dec.copy_(torch.randn(D, generator=g) * 0.1)
    return sae


def step(sae, x, y=None, **kw):
    sae.zero_grad(set_to_none=True)
    out = sae(x, y, **kw)
    (out.fvu + out.auxk_loss / 32 + out.multi_topk_fvu / 8).backward()
    return out, {n: p.grad.clone() for n, p in sae.named_parameters()}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("N,D,M,k", [(256, 64, 512, 8), (301, 96, 1000, 16), (33, 128, 256, 4)])
def test_encoder_gradients_are_those_of_the_restored_input(device, N, D, M, k, dtype):
    """On an input the 8 bits hold exactly, the autoencoder's step is the ordinary one: the same forward, and the encoder's
    gradient from the same rows (bit for bit where the ordinary step reads bf16 rows too)."""
    sae = coder(D, M, k, skip=False, transcode=False)
    x = grid_input(N, D, dtype)
    want_out, want = step(sae, x)
    kept = copy.deepcopy(sae)
    kept.checkpoint = "int8"
    got_out, got = step(kept, x)
    assert torch.equal(got_out.sae_out, want_out.sae_out) and torch.equal(got_out.latent_indices, want_out.latent_indices)
    for n in want:
        if dtype == torch.bfloat16 or n != "encoder.weight":
            assert torch.equal(got[n], want[n]), n
        else:
            # rows x - b_dec in fp32 there, rows x and the shift apart here: k N terms of 2^-23 each
            bound = want["encoder.weight"].abs().max() * N * 2.0**-20
            assert (got[n] - want[n]).abs().max() <= bound, n


@pytest.mark.parametrize("fmt", ["int8", "e4m3"])
@pytest.mark.parametrize("N,D,M,k", [(300, 96, 1000, 16), (64, 80, 512, 8)])
def test_skip_transcoder_against_the_formulas(device, N, D, M, k, fmt):
    """W_skip.grad = g^T x^ and encoder.weight.grad = the selected rows' g_a x^, x^ the restored input, in 64 bits from the
    step's own dL/dsae_out and activations' gradients; sae_out = the decode plus the unrounded product."""
    from sparsify_amd import checkpoint8
    sae = coder(D, M, k)
    sae.checkpoint = fmt
    g = torch.Generator().manual_seed(2)
    x = (torch.randn(N, D, generator=g) * torch.exp(torch.randn(D, generator=g))).cuda()
    y = torch.randn(N, D, generator=g).cuda()
    out, grads = step(sae, x, y)
    xhat = checkpoint8(x, fmt).restore().double()
    xb, Wb = x.bfloat16().double(), sae.W_skip.detach().bfloat16().double()
    dec = sae.decode(out.latent_acts, out.latent_indices).detach().double()
    want = dec + xb @ Wb.T
    tol = (D + 4) * 2.0**-23 * (xb.abs() @ Wb.abs().T) + 2.0**-22 * (want.abs() + dec.abs())
    assert ((out.sae_out.detach().double() - want).abs() <= tol).all()
    tv = (y.double() - y.double().mean(0)).pow(2).sum()
    go = 2 * (out.sae_out.detach().double() - y.double()) / tv                   # dL/dsae_out of the FVU
    dW = go.T @ xhat
    # g in fp32 from the step (2^-20 of it), rounded to bf16 for the product (2^-8), sums of N terms
    tol = (2.0**-8 + 2.0**-20 + (N + 4) * 2.0**-23) * (go.abs().T @ xhat.abs()) + 2.0**-24 * dW.abs()
    assert ((grads["W_skip"].double() - dW).abs() <= tol).all()
    ga = (go[:, None, :] * sae.W_dec.detach().double()[out.latent_indices]).sum(-1) * (out.latent_acts > 0)
    mag = (go.abs()[:, None, :] * sae.W_dec.detach().double().abs()[out.latent_indices]).sum(-1)
    We = torch.zeros(M, D, dtype=torch.float64, device="cuda")
    err = torch.zeros_like(We)
    for s in range(k):
        We.index_add_(0, out.latent_indices[:, s], ga[:, s, None] * xhat)
        err.index_add_(0, out.latent_indices[:, s], (mag[:, s, None] * (D + 8) * 2.0**-20 + 2.0**-8 * ga[:, s, None].abs()) * xhat.abs())
    assert ((grads["encoder.weight"].double() - We).abs() <= err + N * 2.0**-23 * err + 1e-30).all()


def test_input_is_kept_once_and_in_8_bits(device):
    """What the graph of a skip transcoder's forward holds of its input, by the tensors saved for the backward."""
    N, D, M, k = 1024, 256, 1024, 8

    def saved(sae, x):
        held = {}

        def pack(t):
            held[t.data_ptr()] = t.numel() * t.element_size()
            return t

        with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
            out = sae(x, torch.randn_like(x))
        params = {p.data_ptr() for p in sae.parameters()}
        total = sum(b for p, b in held.items() if p not in params)
        del out
        return total

    sae = coder(D, M, k)
    x = torch.randn(N, D, device="cuda").bfloat16()
    plain = saved(sae, x)
    sae.checkpoint = "int8"
    kept = saved(sae, x)
    # the bf16 rows (once for both products: they are the caller's tensor) give way to a byte per value and a scale per 32
    assert plain - kept >= N * D * 2 - N * D * 33 // 32 - (1 << 16)
    with torch.no_grad():
        assert sae._keep(x) is None


@pytest.mark.parametrize("kw", [dict(), dict(multi_topk=True), dict(transcode=False, skip=False), dict(activation="groupmax")])
def test_every_variant_steps(device, kw):
    """AuxK, multi-top-k, groupmax, an autoencoder: the loss with the kept input is the ordinary one up to the skip product's
    missing rounding, every gradient is there and close."""
    N, D, M, k = 512, 64, 512, 8
    sae = coder(D, M, k, **kw)
    x = grid_input(N, D, torch.bfloat16, 3)
    y = torch.randn(N, D, device="cuda")
    mask = torch.zeros(M, dtype=torch.bool, device="cuda")
    mask[::3] = True
    args = {} if kw.get("activation") == "groupmax" else dict(dead_mask=mask)
    want_out, want = step(sae, x, y if sae.cfg.transcode else None, **args)
    kept = copy.deepcopy(sae)
    kept.checkpoint = "int8"
    out, got = step(kept, x, y if sae.cfg.transcode else None, **args)
    # the skip product's rounding: 2^-9 of it per element, so the loss moves by less than 2^-7 of itself
    assert abs(float(out.fvu) - float(want_out.fvu)) <= 2.0**-7 * float(want_out.fvu)
    for n in want:
        a, b = got[n].double(), want[n].double()
        assert float((a - b).norm()) <= 2.0**-6 * float(b.norm()) + 1e-12, n


def test_trainer_switch(device, tmp_path):
    from sparsify_amd import SparseCoderConfig, TrainConfig
    from sparsify_amd.trainer import Trainer

    class Source:
        widths = {"h0": 64}

        def __len__(self):
            return 4

        def __iter__(self):
            for i in range(4):
                x = torch.randn(256, 64, device="cuda", generator=torch.Generator("cuda").manual_seed(i))
                yield {"h0": (x, x.flip(-1))}

    for opt in ("signsgd", "signum"):
        cfg = TrainConfig(sae=SparseCoderConfig(num_latents=512, k=8, transcode=True, skip_connection=True), optimizer=opt, lr=1e-3,
                          save_dir=str(tmp_path), save_every=10**9, checkpoint_8bit="e4m3")
        tr = Trainer(cfg, Source(), device="cuda")
        sae = tr.saes["h0"]
        assert sae.checkpoint == "e4m3"
        before = {n: p.detach().clone() for n, p in sae.named_parameters()}
        for b in Source():
            tr.train_micro_batch(b)
        torch.cuda.synchronize()
        for n, p in sae.named_parameters():
            assert torch.isfinite(p).all() and not torch.equal(p, before[n]), n


def test_mismatched_checkpoint_is_refused(device):
    from sparsify_amd import checkpoint8, fused_encoder
    sae = coder(64, 256, 4)
    x = torch.randn(32, 64, device="cuda")
    with pytest.raises(ValueError, match="checkpoint holds"):
        sae.encode(x, kept=checkpoint8(x[:16], "int8"))
    with pytest.raises(ValueError, match="checkpoint holds"):
        fused_encoder(x, sae.encoder.weight, sae.encoder.bias, 4, "topk", kept=checkpoint8(x[:, :32], "int8"))
