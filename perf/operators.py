"""Cases of the 8-bit training operators: LayerNorm with its backward pass, activations whose input is kept in 8 bits for the
backward pass, the matrix product of 8-bit operands with a power-of-two scale for each block of 128, and the weight gradient
taken from an 8-bit activation.

8-bit format (both sides): a row of C values is cut into blocks of 128 (the last one padded with zeros); a block holds e4m3
codes and one exponent E, the smallest with max |x| <= 448 * 2^E; a code stands for code * 2^E.  `q` is [rows, 128 * blocks]
float8_e4m3fn, `scale` is uint8 [blocks, rows rounded up to 16] with E + 127 (weights: one exponent for 128 rows x 128 columns,
`scale` is [blocks, row blocks])."""
import math

import torch

own = False

DEVICE = "cuda"


# ------------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # SD 2.1's 8 x 8 level at network batch 8: the smallest LayerNorm of a training step, launch latency counts
        dict(name="ln 512x1280", op="layernorm", rows=512, cols=1280, x="fp16", both=True, residual=True),
        # SD 2.1's 64 x 64 level at network batch 8: the largest row count, narrow rows
        dict(name="ln 32768x320", op="layernorm", rows=32768, cols=320, x="fp16", both=True, residual=True),
        # SAM ViT-H's fp32 residual stream, four images: the backward pass alone
        dict(name="ln bwd 16384x1280 fp32", op="layernorm", rows=16384, cols=1280, x="fp32", both=False, residual=True),
        # eight prompts of 77 tokens: a ragged row count, the LayerNorm's input kept in 8 bits
        dict(name="ln bwd 616x1024 fp8", op="layernorm", rows=616, cols=1024, x="fp8", both=False, residual=False),
        # SD 2.1's feed-forward at the 8 x 8 level, forward: value * gelu(gate), the input kept in 8 bits
        dict(name="geglu save 512x5120", op="activation", rows=512, cols=5120, act="geglu", use=False, fp8=False),
        # SAM ViT-H's MLP, forward: both the output (the next product's operand) and the input in 8 bits
        dict(name="gelu save 16384x5120", op="activation", rows=16384, cols=5120, act="gelu", use=False, fp8=True),
        # SD 2.1's feed-forward at the 64 x 64 level, backward from the 8-bit input
        dict(name="geglu use 32768x1280", op="activation", rows=32768, cols=1280, act="geglu", use=True, fp8=False),
        # the text keys and values of one SD 2.1 block: few, ragged rows against a wide weight
        dict(name="gemm 616x2560x1024", op="gemm", rows=616, n=2560, k=1024, act="none", bias=False, residual=False),
        # an attention output projection at the 32 x 32 level: bias and residual in the epilogue
        dict(name="gemm 8192x640x640", op="gemm", rows=8192, n=640, k=640, act="none", bias=True, residual=True),
        # SAM ViT-H mlp.lin1, four images: the largest product
        dict(name="gemm 16384x5120x1280", op="gemm", rows=16384, n=5120, k=1280, act="gelu", bias=True, residual=False),
        # weight gradient of the text projection: a small output
        dict(name="wgrad 616x1280x1024", op="wgrad", rows=616, n=1280, k=1024),
        # weight gradient of SAM ViT-H mlp.lin2, four images
        dict(name="wgrad 16384x1280x5120", op="wgrad", rows=16384, n=1280, k=5120),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _width(rng, lo, hi):
    """A width: a multiple of 128, of 8, or any number."""
    v = _log(rng, lo, hi)
    step = rng.choice((128, 8, 1))
    return max(lo, v // step * step)


def draw(rng):
    op = rng.choice(("layernorm", "activation", "gemm", "wgrad"))
    if op == "layernorm":
        cols = _width(rng, 8, 4096)
        rows = _log(rng, 1, min(32768, 32768 * 640 // cols))
        x = rng.choice(("fp16", "fp32", "fp8"))
        return dict(op=op, rows=rows, cols=cols, x=x, both=x != "fp8" and rng.random() < 0.5, residual=rng.random() < 0.5)
    if op == "activation":
        cols = _width(rng, 16, 5120)
        act = rng.choice(("gelu", "silu", "geglu"))
        rows = _log(rng, 1, min(32768, 16384 * 2560 // cols))
        use = rng.random() < 0.5
        return dict(op=op, rows=rows, cols=cols, act=act, use=use, fp8=act != "geglu" and not use and rng.random() < 0.5)
    n, k = _width(rng, 8, 5120), _width(rng, 32, 5120)
    rows = _log(rng, 1, min(32768, 16384 * 5120 * 1280 // (n * k)))
    if op == "wgrad":
        return dict(op=op, rows=rows, n=n, k=k)
    return dict(op=op, rows=rows, n=n, k=k, act=rng.choice(("none", "silu", "gelu")), bias=rng.random() < 0.5, residual=rng.random() < 0.3)


def work(case):
    M = case["rows"]
    if case["op"] == "layernorm":
        C = case["cols"]
        sx = {"fp16": 2, "fp32": 4, "fp8": 1 + 1 / 128}[case["x"]]
        so = 4 if case["x"] == "fp32" else 2
        fwd = M * C * 2 + 8 * C + 8 * M if case["both"] else 8 * M           # y and the affine; or the statistics read
        bwd = M * C * (2 + sx + so + (so if case["residual"] else 0)) + 12 * C
        return dict(bytes=fwd + bwd, flops=M * C * (20 if case["both"] else 12))
    if case["op"] == "activation":
        H, g = case["cols"], 2 if case["act"] == "geglu" else 1
        if case["use"]:
            return dict(bytes=M * H * (2 + g * (1 + 1 / 128) + 2 * g), flops=30 * M * H)
        return dict(bytes=M * H * (2 * g + g * (1 + 1 / 128) + ((1 + 1 / 128) if case["fp8"] else 2)), flops=20 * M * H)
    N, K = case["n"], case["k"]
    if case["op"] == "wgrad":
        return dict(bytes=2 * M * N + M * K * (1 + 1 / 128) + 4 * N * K + 4 * N, flops=2 * M * N * K)
    return dict(bytes=(M + N) * K + M * K / 128 + N * K / 16384 + 2 * M * N * (2 if case["residual"] else 1) + (4 * N if case["bias"] else 0),
                flops=2 * M * N * K)


# ---------------------------------------------------------------------------------------------------------------- inputs
def _pow2(e):
    """2^e for whole e, exactly, from the bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _blocks(x):
    """fp32 [R, C] -> [R, blocks, 128], padded with zeros."""
    R, C = x.shape
    nb = -(-C // 128)
    if nb * 128 != C:
        x = torch.nn.functional.pad(x, (0, nb * 128 - C))
    return x.view(R, nb, 128)


def _exponent(amax):
    f, e = torch.frexp(amax)
    e = e - 9 + (f > 0.875).to(e.dtype)
    return torch.where(amax > 0, e, torch.zeros_like(e)).clamp(-100, 120)


def _quantize(x):
    """fp32 [R, C] -> (codes [R, 128 * blocks], exponents [R, blocks])."""
    v = _blocks(x)
    e = _exponent(v.abs().amax(-1))
    q = (v * _pow2(-e)[..., None]).to(torch.float8_e4m3fn)
    return q.view(x.shape[0], -1), e


def _scale_rows(e):
    """Exponents [R, blocks] -> the stored form, uint8 [blocks, R rounded up to 16]."""
    R, nb = e.shape
    s = torch.full((nb, -(-R // 16) * 16), 127, dtype=torch.uint8, device=e.device)
    s[:, :R] = (e + 127).to(torch.uint8).t()
    return s


def _quantize_weight(w):
    """fp32 [N, K] -> (codes [N, 128 * blocks], uint8 [blocks, row blocks])."""
    N, K = w.shape
    nb, rb = -(-K // 128), -(-N // 128)
    v = torch.nn.functional.pad(w, (0, nb * 128 - K, 0, rb * 128 - N)).view(rb, 128, nb, 128)
    e = _exponent(v.abs().amax((1, 3)))
    q = (v * _pow2(-e)[:, None, :, None]).to(torch.float8_e4m3fn)
    return q.view(rb * 128, nb * 128)[:N].contiguous(), (e + 127).to(torch.uint8).t().contiguous()


def _activations(g, M, C):
    """Rows of a transformer's stream: unequal rows, a few strong channels."""
    x = torch.randn(M, C, generator=g, device=DEVICE)
    x *= 0.5 + torch.rand(M, 1, generator=g, device=DEVICE)
    ch = torch.rand(C, generator=g, device=DEVICE)
    x *= torch.where(ch > 0.98, 6.0, 1.0)
    return x + 0.1 * torch.randn(C, generator=g, device=DEVICE)


def prepare(case, seed):
    g = torch.Generator(device=DEVICE).manual_seed(seed)
    M = case["rows"]
    s = dict(case=case)
    if case["op"] == "layernorm":
        C = case["cols"]
        x = _activations(g, M, C)
        s["gamma"] = 1 + 0.2 * torch.randn(C, generator=g, device=DEVICE)
        s["beta"] = 0.1 * torch.randn(C, generator=g, device=DEVICE)
        s["dy"] = (0.02 * torch.randn(M, C, generator=g, device=DEVICE)).half()
        out = torch.float32 if case["x"] == "fp32" else torch.float16
        s["residual"] = (0.02 * torch.randn(M, C, generator=g, device=DEVICE)).to(out) if case["residual"] else None
        s["x"] = x.to(out)
        if not case["both"]:                                     # the statistics that the forward pass left
            xd = s["x"].double()
            var, mean = torch.var_mean(xd, -1, correction=0)
            s["stats"] = torch.stack([mean, (var + 1e-5).rsqrt()], -1).float()
        if case["x"] == "fp8":
            s["x"], e = _quantize(x)
            s["x_scale"] = _scale_rows(e)
        return s
    if case["op"] == "activation":
        H, w = case["cols"], case["cols"] * (2 if case["act"] == "geglu" else 1)
        z = (1.5 * _activations(g, M, w)).half()
        if case["use"]:
            s["z"], e = _quantize(z.float().view(-1, H))         # geglu: the two halves of a row are rows of their own
            s["z_scale"] = _scale_rows(e)
            s["dh"] = (0.02 * torch.randn(M, H, generator=g, device=DEVICE)).half()
        else:
            s["z"] = z
        return s
    N, K = case["n"], case["k"]
    s["x"], e = _quantize(_activations(g, M, K))
    s["x_scale"] = _scale_rows(e)
    if case["op"] == "wgrad":
        s["dy"] = (0.02 * torch.randn(M, N, generator=g, device=DEVICE)).half()
        return s
    s["w"], s["w_scale"] = _quantize_weight(torch.randn(N, K, generator=g, device=DEVICE) * K ** -0.5)
    s["bias"] = 0.1 * torch.randn(N, generator=g, device=DEVICE) if case["bias"] else None
    s["residual"] = torch.randn(M, N, generator=g, device=DEVICE).half() if case["residual"] else None
    return s


# ----------------------------------------------------------------------------------------------------------- plain forms
def _decode(q, scale, C):
    """Codes and stored exponents of rows -> fp32 [R, C]."""
    R = q.shape[0]
    e = scale[:, :R].t().to(torch.int32) - 127
    return (q.float().view(R, -1, 128) * _pow2(e)[..., None]).view(R, -1)[:, :C]


def _decode_weight(q, scale, K):
    N = q.shape[0]
    f = _pow2(scale.t().to(torch.int32) - 127).repeat_interleave(128, 0)[:N].repeat_interleave(128, 1)
    return (q.float() * f)[:, :K]


def _phi(x):
    """The normal distribution function and its density."""
    return 0.5 * (1 + torch.erf(x * 0.7071067811865476)), torch.exp(-0.5 * x * x) * 0.3989422804014327


def _layernorm(s):
    c, C = s["case"], s["case"]["cols"]
    x = _decode(s["x"], s["x_scale"], C) if c["x"] == "fp8" else s["x"].float()
    out = {}
    if c["both"]:
        mean = x.mean(-1, keepdim=True)
        rstd = ((x - mean).square().mean(-1, keepdim=True) + 1e-5).rsqrt()
        out["y"] = ((x - mean) * rstd * s["gamma"] + s["beta"]).half()
        out["stats"] = torch.cat([mean, rstd], -1)
    else:
        mean, rstd = s["stats"][:, :1], s["stats"][:, 1:]
    dy = s["dy"].float()
    xh = (x - mean) * rstd
    g = dy * s["gamma"]
    dx = rstd * (g - g.mean(-1, keepdim=True) - xh * (g * xh).mean(-1, keepdim=True))
    if s["residual"] is not None:
        dx = dx + s["residual"].float()
    out["dx"] = dx if c["x"] == "fp32" else dx.half()
    out["dgamma"], out["dbeta"] = (dy * xh).sum(0), dy.sum(0)
    return out


def _activation(s):
    c, H = s["case"], s["case"]["cols"]
    if c["use"]:
        z = _decode(s["z"], s["z_scale"], H)
        dh = s["dh"].float()
        if c["act"] == "silu":
            sg = torch.sigmoid(z)
            return (dh * sg * (1 + z * (1 - sg))).half()
        if c["act"] == "gelu":
            P, p = _phi(z)
            return (dh * (P + z * p)).half()
        z = z.view(-1, 2, H)
        P, p = _phi(z[:, 1])
        return torch.cat([dh * z[:, 1] * P, dh * z[:, 0] * (P + z[:, 1] * p)], -1).half()
    z = s["z"].float()
    q, e = _quantize(z.view(-1, H))
    if c["act"] == "geglu":
        v, gate = z.chunk(2, -1)
        h = v * gate * _phi(gate)[0]
    elif c["act"] == "silu":
        h = z * torch.sigmoid(z)
    else:
        h = z * _phi(z)[0]
    out = dict(saved=q, saved_scale=_scale_rows(e)[:, :e.shape[0]])
    if c["fp8"]:
        hq, he = _quantize(h)
        return dict(h=hq, h_scale=_scale_rows(he)[:, :he.shape[0]], **out)
    return dict(h=h.half(), **out)


def _gemm(s):
    c = s["case"]
    v = _decode(s["x"], s["x_scale"], c["k"]) @ _decode_weight(s["w"], s["w_scale"], c["k"]).t()
    if s["bias"] is not None:
        v = v + s["bias"]
    if c["act"] == "silu":
        v = v * torch.sigmoid(v)
    elif c["act"] == "gelu":
        v = v * _phi(v)[0]
    if s["residual"] is not None:
        v = v + s["residual"].float()
    return v.half()


def _wgrad(s):
    dy = s["dy"].float()
    return dict(dw=dy.t().contiguous() @ _decode(s["x"], s["x_scale"], s["case"]["k"]), db=dy.sum(0))


def run(state):
    c, s = state["case"], state
    if not own:
        return {"layernorm": _layernorm, "activation": _activation, "gemm": _gemm, "wgrad": _wgrad}[c["op"]](s)
    from editanything_amd import ops
    if c["op"] == "layernorm":
        out = {}
        x = ops.Fp8Tensor(s["x"], s["x_scale"], c["cols"]) if c["x"] == "fp8" else s["x"]
        stats = s.get("stats")
        if c["both"]:
            out["y"], stats = ops.layernorm_train(x, s["gamma"], s["beta"])
            out["stats"] = stats
        out["dx"], out["dgamma"], out["dbeta"] = ops.layernorm_backward(s["dy"], x, stats, s["gamma"], residual=s["residual"])
        return out
    if c["op"] == "activation":
        act = {"gelu": ops.ACT_GELU, "silu": ops.ACT_SILU, "geglu": ops.ACT_GEGLU}[c["act"]]
        if c["use"]:
            return ops.activation_fp8_backward(s["dh"], ops.Fp8Tensor(s["z"], s["z_scale"], c["cols"]), act)
        h, saved = ops.activation_fp8(s["z"], act, fp8=c["fp8"])
        out = dict(saved=saved.q, saved_scale=saved.scale[:, :saved.rows])
        if c["fp8"]:
            return dict(h=h.q, h_scale=h.scale[:, :h.rows], **out)
        return dict(h=h, **out)
    x = ops.Fp8Tensor(s["x"], s["x_scale"], c["k"])
    if c["op"] == "wgrad":
        dw, db = ops.gemm_fp8_wgrad(s["dy"], x)
        return dict(dw=dw, db=db)
    act = {"none": ops.ACT_NONE, "silu": ops.ACT_SILU, "gelu": ops.ACT_GELU}[c["act"]]
    return ops.gemm_fp8(x, ops.Fp8Tensor(s["w"], s["w_scale"], c["k"]), bias=s["bias"], act=act, residual=s["residual"])


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _e4m3_rows(x):
    """fp64 [R, C] -> (values of the codes, exponents): the exponent by counting up from a low one, the code by rounding to
    the format's step (2^-3 of the leading power of two, 2^-9 at least), ties to even."""
    R, C = x.shape
    nb = -(-C // 128)
    v = torch.zeros(R, nb * 128, dtype=torch.float64, device=x.device)
    v[:, :C] = x
    v = v.view(R, nb, 128)
    top = v.abs().max(-1).values
    e = torch.ceil(torch.log2(top.clamp_min(1e-300) / 448.0))
    e = torch.where(448.0 * torch.exp2(e - 1) >= top, e - 1, e)
    e = torch.where(448.0 * torch.exp2(e) < top, e + 1, e)
    e = torch.where(top > 0, e, torch.zeros_like(e)).clamp(-100, 120)
    u = v / torch.exp2(e)[..., None]
    step = torch.exp2(torch.floor(torch.log2(u.abs().clamp_min(2.0 ** -6))) - 3)
    return (torch.round(u / step) * step).view(R, -1), e


def _value(q, scale, C):
    R, nb = q.shape[0], q.shape[1] // 128
    f = torch.exp2(scale.double() - 127.0)
    f = f[:, :R].t()
    return torch.stack([q[:, b * 128:(b + 1) * 128].double() * f[:, b:b + 1] for b in range(nb)], 1).view(R, -1)[:, :C]


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "layernorm":
        C = case["cols"]
        x = _value(s["x"], s["x_scale"], C) if case["x"] == "fp8" else s["x"].double()
        out = {}
        gamma, beta, dy = s["gamma"].double(), s["beta"].double(), s["dy"].double()
        if case["both"]:
            mu = x.sum(1) / C
            sd = (((x - mu[:, None]) ** 2).sum(1) / C + 1e-5).sqrt()
            out["stats"] = torch.stack([mu, 1 / sd], 1)
        else:
            mu, sd = s["stats"][:, 0].double(), 1 / s["stats"][:, 1].double()
        n = (x - mu[:, None]) / sd[:, None]
        if case["both"]:
            out["y"] = n * gamma + beta
        g = dy * gamma
        dx = (g - (g.sum(1) / C)[:, None] - n * ((g * n).sum(1) / C)[:, None]) / sd[:, None]
        out["dx"] = dx if s["residual"] is None else dx + s["residual"].double()
        out["dgamma"], out["dbeta"] = (dy * n).sum(0), dy.sum(0)
        return out
    if case["op"] == "activation":
        H = case["cols"]
        gelu = lambda t: 0.5 * t * torch.erfc(-t / math.sqrt(2.0))  # noqa: E731
        slope = lambda t: 0.5 * torch.erfc(-t / math.sqrt(2.0)) + t * torch.exp(-t * t / 2) / math.sqrt(2 * math.pi)  # noqa: E731
        if case["use"]:
            z, dh = _value(s["z"], s["z_scale"], H), s["dh"].double()
            if case["act"] == "gelu":
                return dh * slope(z)
            if case["act"] == "silu":
                t = torch.exp(-z)
                return dh * (1 / (1 + t) + z * t / (1 + t) ** 2)
            v, t = z[0::2], z[1::2]
            return torch.cat([dh * gelu(t), dh * v * slope(t)], 1)
        z = s["z"].double()
        q, e = _e4m3_rows(z.view(-1, H))
        out = dict(saved=q, saved_scale=None)
        h = z[:, :H] * gelu(z[:, H:]) if case["act"] == "geglu" else gelu(z) if case["act"] == "gelu" else z / (1 + torch.exp(-z))
        if case["fp8"]:
            out["h"], out["h_scale"] = _e4m3_rows(h)[0], None
        else:
            out["h"] = h
        return out
    x = _value(s["x"], s["x_scale"], case["k"])
    if case["op"] == "wgrad":
        dy = s["dy"].double()
        return dict(dw=(x.t().contiguous() @ dy).t(), db=dy.sum(0))
    K, N = case["k"], case["n"]
    w = s["w"].double()
    for b in range(s["w_scale"].shape[0]):
        f = torch.exp2(s["w_scale"][b].double() - 127)[torch.arange(N, device=w.device) // 128]
        w[:, b * 128:(b + 1) * 128] *= f[:, None]
    v = x @ w[:, :K].t().contiguous()
    if s["bias"] is not None:
        v = v + s["bias"].double()
    if case["act"] == "gelu":
        v = 0.5 * v * torch.erfc(-v / math.sqrt(2.0))
    elif case["act"] == "silu":
        v = v / (1 + torch.exp(-v))
    return v if s["residual"] is None else v + s["residual"].double()
