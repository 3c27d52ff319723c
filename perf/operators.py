"""The dense side of a sparse coder's training step, measured: a product with its epilogue (the skip path
of a transcoder), the 8-bit checkpoint of an activation, and the product's gradients from that checkpoint.

  linear      y = act(x W^T + b) + r, one rounding at the end
  checkpoint  groups of 32 consecutive tokens of one feature share a power-of-two scale; a value is kept
              as an 8-bit integer ("int8") or an 8-bit float of 4 exponent bits ("e4m3") and restored
  grad        the same product in training: y, and from dL/dy the gradients of x, W, b and r. The
              product keeps x and (where the activation needs it) z = x W^T + b as such checkpoints:
              dz = g act'(z^), dx = dz W, dW = dz^T x^, db = sum_n dz, dr = g

Plain forms compute in 32 bits and round once at the end."""
import math

import torch

own = False

GROUP = 32                     # tokens that share a scale
DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # the skip product of a transcoder at d = 4096, one token at a time: W is read once, nothing else counts
        dict(name="linear_token", op="linear", N=1, D=4096, M=4096, dtype="bf16", act="none", bias=False, res="f32"),
        # a handful of tokens (a steering probe's batch) through a wide layer
        dict(name="linear_few", op="linear", N=24, D=2048, M=8192, dtype="bf16", act="gelu", bias=True, res="none"),
        # sizes nothing divides: a ragged batch, an odd number of features
        dict(name="linear_ragged", op="linear", N=1003, D=769, M=2050, dtype="bf16", act="silu", bias=True, res="same"),
        # the headline batch and width: 16384 tokens, d = 4096, onto the fp32 reconstruction
        dict(name="linear_batch", op="linear", N=16384, D=4096, M=4096, dtype="bf16", act="gelu", bias=True, res="f32"),
        # the exact-fp32 path (no autocast), at the encoder test's width
        dict(name="linear_f32", op="linear", N=2048, D=1024, M=1024, dtype="f32", act="relu", bias=True, res="none"),
        # a small model's activations in fp32: launch-bound
        dict(name="checkpoint_small", op="checkpoint", N=256, D=768, dtype="f32", fmt="int8"),
        # the default batch (32 x 2048 tokens) at d = 4096: one stream through HBM
        dict(name="checkpoint_batch", op="checkpoint", N=65536, D=4096, dtype="bf16", fmt="int8"),
        # a last group of 9 tokens, rows that start at odd addresses
        dict(name="checkpoint_ragged", op="checkpoint", N=5001, D=1111, dtype="bf16", fmt="e4m3"),
        # d = 768, one short sequence: every product is smaller than the chip
        dict(name="grad_small", op="grad", N=256, D=768, M=768, dtype="bf16", act="gelu", bias=True, res="none", fmt="int8"),
        # the skip connection of a transcoder in training at the headline batch
        dict(name="grad_batch", op="grad", N=16384, D=4096, M=4096, dtype="bf16", act="none", bias=False, res="f32", fmt="int8"),
        # odd sizes everywhere, activation and residual
        dict(name="grad_ragged", op="grad", N=4099, D=1001, M=1500, dtype="bf16", act="silu", bias=True, res="same", fmt="e4m3"),
        # the exact-fp32 path in training
        dict(name="grad_f32", op="grad", N=2048, D=512, M=512, dtype="f32", act="none", bias=True, res="none", fmt="e4m3"),
    ]


def draw(rng):
    def size(lo, hi):
        n = round(math.exp(rng.uniform(math.log(lo), math.log(hi))))
        step = rng.choice((1, 1, 2, 8, 64))          # half of them of no particular divisor
        return min(hi, max(lo, n // step * step if n >= step else n))

    op = rng.choice(("linear", "checkpoint", "grad"))
    dtype = rng.choice(("bf16", "bf16", "f32"))
    fmt = rng.choice(("int8", "e4m3"))
    if op == "checkpoint":
        D = size(64, 8192)
        return dict(op=op, N=size(1, min(65536, (1 << 28) // D)), D=D, dtype=dtype, fmt=fmt)
    D, M = size(64, 8192), size(64, 8192)
    flops = (5.4e11 if dtype == "bf16" else 3e10) if op == "linear" else (1.6e12 if dtype == "bf16" else 3e10) / 3
    case = dict(op=op, N=size(1, max(2, min(16384, int(flops / (2 * D * M))))), D=D, M=M, dtype=dtype,
                act=rng.choice(("none", "relu", "gelu", "silu")), bias=rng.random() < 0.6,
                res=rng.choice(("none", "same", "f32")))
    if op == "grad":
        # in fp32 an activation's derivative is taken at z as it is (no 8-bit copy of z)
        case["fmt"] = fmt if dtype == "bf16" or case["act"] == "none" else "none"
        if dtype == "f32" and case["act"] == "relu":
            case["act"] = "silu"                     # smooth: a step at 0 in fp32 is decided by the order of a sum
    return case


def work(case):
    N, D = case["N"], case["D"]
    es = 2 if case["dtype"] == "bf16" else 4
    if case["op"] == "checkpoint":
        codes = N * D + -(-N // GROUP) * D
        return {"bytes": 2 * N * D * es + 2 * codes, "flops": 2 * N * D}
    M = case["M"]
    rs = 0 if case["res"] == "none" else 4 if case["res"] == "f32" else es
    os_ = 4 if case["res"] == "f32" else es
    fwd = N * D * es + M * D * es + (M * es if case["bias"] else 0) + N * M * rs + N * M * os_
    if case["op"] == "linear":
        return {"bytes": fwd, "flops": 2 * N * D * M}
    kept = (N * D if case["fmt"] != "none" else N * D * es)
    if case["act"] != "none":
        kept += N * M if case["fmt"] != "none" else N * M * es
    back = N * M * os_ + N * D * es + M * D * es + (M * es if case["bias"] else 0)
    return {"bytes": fwd + back + 2 * kept, "flops": 6 * N * D * M}


# ------------------------------------------------------------------ inputs
def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev)
    gen.manual_seed(seed)
    N, D = case["N"], case["D"]
    dt = DTYPES[case["dtype"]]

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device=dev)

    # a residual stream: every feature with its own scale and offset, one in 128 of them large
    scale = torch.exp(0.5 * randn(D)) * (1 + 29 * (torch.rand(D, generator=gen, device=dev) < 1 / 128))
    x = torch.addcmul(0.3 * scale, randn(N, D), scale).to(dt)
    state = {"case": dict(case), "x": x}
    if case["op"] == "checkpoint":
        return state
    M = case["M"]
    state["W"] = (randn(M, D) / (scale * math.sqrt(D))).to(dt)
    state["b"] = (0.2 * randn(M)).to(dt) if case["bias"] else None
    state["r"] = None if case["res"] == "none" else randn(N, M).to(torch.float32 if case["res"] == "f32" else dt)
    if case["op"] == "grad":
        state["g"] = (randn(N, M) / N).to(torch.float32 if case["res"] == "f32" else dt)
        for name in ("x", "W", "b", "r"):            # leaves, as a training program holds them
            if state[name] is not None:
                state[name].requires_grad_(True)
    return state


# ------------------------------------------------------------------ plain forms
def _act(z, act):
    if act == "none":
        return z
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))


def _slope(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))


def _round_trip(x, fmt, keep_sign=False):
    """The values an 8-bit checkpoint of x (N, D), fp32, stands for."""
    N, D = x.shape
    G = -(-N // GROUP)
    padded = torch.zeros(G * GROUP, D, dtype=torch.float32, device=x.device)
    padded[:N] = x
    groups = padded.view(G, GROUP, D)
    top = groups.abs().amax(1, keepdim=True)
    mant, expo = torch.frexp(top)                    # top = mant 2^expo, mant in [1/2, 1)
    # the smallest scale that keeps the largest value at 127 (int8) or 448 (e4m3)
    if fmt == "int8":
        e = expo - 7 + (mant > 127 / 128).to(expo.dtype)
    else:
        e = expo - 9 + (mant > 0.875).to(expo.dtype)
    e = torch.where(top > 0, e, torch.full_like(e, -126)).clamp(min=-126)
    q = torch.ldexp(groups, -e)
    code = torch.round(q) if fmt == "int8" else q.to(torch.float8_e4m3fn).float()
    if keep_sign:
        least = 1.0 if fmt == "int8" else 2.0 ** -9
        code = torch.where((code == 0) & (q != 0), torch.sign(q) * least, code)
    return torch.ldexp(code, e).view(G * GROUP, D)[:N]


def run(state):
    c = state["case"]
    x, act = state["x"], c.get("act")
    if own:
        import sparsify_amd

        if c["op"] == "checkpoint":
            return {"restored": sparsify_amd.checkpoint8(x, c["fmt"]).restore()}
        W, b, r = state["W"], state["b"], state["r"]
        if c["op"] == "linear":
            return {"y": sparsify_amd.fused_linear(x, W, b, residual=r, activation=act)}
        y = sparsify_amd.fused_linear(x, W, b, residual=r, activation=act,
                                      checkpoint=None if c["fmt"] == "none" else c["fmt"])
        leaves = {"dx": x, "dW": W, "db": b, "dr": r}
        leaves = {k: t for k, t in leaves.items() if t is not None}
        grads = torch.autograd.grad(y, list(leaves.values()), state["g"])
        return {"y": y.detach(), **dict(zip(leaves, grads))}

    with torch.no_grad():
        xf = x.float()
        if c["op"] == "checkpoint":
            return {"restored": _round_trip(xf, c["fmt"]).to(x.dtype)}
        W, b, r = state["W"], state["b"], state["r"]
        Wf = W.float()
        z = xf @ Wf.T
        if b is not None:
            z = z + b.float()
        y = _act(z, act)
        if r is not None:
            y = y + r.float()
        y = y.to(torch.float32 if c["res"] == "f32" else x.dtype)
        if c["op"] == "linear":
            return {"y": y}
        g = state["g"].float()
        if act == "none":
            dz = g
        elif c["fmt"] == "none":
            dz = g * _slope(z, act)
        else:
            dz = g * _slope(_round_trip(z, c["fmt"], keep_sign=act == "relu"), act)
        kept = xf if c["fmt"] == "none" else _round_trip(xf, c["fmt"])
        out = {"y": y, "dx": (dz @ Wf).to(x.dtype), "dW": (dz.T @ kept).to(W.dtype)}
        if b is not None:
            out["db"] = dz.sum(0).to(b.dtype)
        if r is not None:
            out["dr"] = state["g"].to(r.dtype)
        return out


# ------------------------------------------------------------------ from the definition, in 64 bits
def _code_values(v, fmt, keep_sign):
    """v (N, D) in 64 bits -> the nearest value of the 8-bit format under its group's scale."""
    parts = []
    for rows in v.split(GROUP):
        top = rows.abs().max(0).values
        most = 127.0 if fmt == "int8" else 448.0
        need = top.clamp(min=2.0 ** -200) / most
        e = torch.ceil(torch.log2(need))
        e = torch.where(torch.exp2(e - 1) >= need, e - 1, e)          # log2 may round either way
        e = torch.where(torch.exp2(e) < need, e + 1, e).clamp(min=-126.0)
        q = rows / torch.exp2(e)
        if fmt == "int8":
            step = torch.ones_like(q)
        else:                                                        # 3 bits below the leading one, from 2^-6 down fixed steps
            lead = torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6)))
            step = torch.exp2(lead - 3)
        k = torch.round(q / step) * step
        if keep_sign:
            k = torch.where((k == 0) & (q != 0), torch.sign(q) * (1.0 if fmt == "int8" else 2.0 ** -9), k)
        parts.append(k * torch.exp2(e))
    return torch.cat(parts)


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        x = s["x"].double()
        if case["op"] == "checkpoint":
            return {"restored": _code_values(x, case["fmt"], False)}
        W, act = s["W"].double(), case["act"]
        z = torch.mm(x, W.t().contiguous())
        if s["b"] is not None:
            z += s["b"].double()
        value = {"none": lambda t: t, "relu": lambda t: t.clamp(min=0), "silu": lambda t: t * torch.sigmoid(t),
                 "gelu": lambda t: t * torch.special.ndtr(t)}[act](z)
        y = value if s["r"] is None else value + s["r"].double()
        if case["op"] == "linear":
            return {"y": y}
        kept = x if case["fmt"] == "none" else _code_values(x, case["fmt"], False)
        dz = s["g"].double()
        if act != "none":
            at = z if case["fmt"] == "none" else _code_values(z, case["fmt"], act == "relu")
            sig = torch.sigmoid(at)
            dz = dz * {"relu": lambda: (at > 0).double(), "silu": lambda: sig + at * sig * (1 - sig),
                       "gelu": lambda: torch.special.ndtr(at) + at * torch.exp(-at * at / 2) / math.sqrt(2 * math.pi)}[act]()
        out = {"y": y, "dx": torch.mm(dz, W), "dW": torch.mm(dz.t().contiguous(), kept)}
        if s["b"] is not None:
            out["db"] = dz.sum(0)
        if s["r"] is not None:
            out["dr"] = s["g"].double()
        return out
