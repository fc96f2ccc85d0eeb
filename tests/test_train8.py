"""The 8-bit training operators (ops.quantize_fp8 ... ops.gemm_fp8_wgrad): every kernel through the C entries on the CPU emulation and
on the GPU against a plain evaluation in 64 bits, the refusals, and the public functions on the GPU (streams, graphs, a whole block).

Tolerances count roundings: u16 = 2^-11 is half a step of fp16, u32 = 2^-24 of fp32; a sum of n fp32 terms in any order is off by at most
n u32 sum |terms| (2 n u32 where the matrix unit may truncate instead of rounding)."""
import ctypes
import math

import numpy as np
import pytest
import torch

from editanything_amd import _lib as L
from editanything_amd import ops
from emu_util import epilogue, ptr

U16, U32 = 2.0 ** -11, 2.0 ** -24
TINY16 = 2.0 ** -25                        # half of fp16's smallest step
SILU, GELU, GEGLU = L.ACT_SILU, L.ACT_GELU, L.ACT_GEGLU
erf = np.vectorize(math.erf, otypes=[np.float64])


# ------------------------------------------------------------------------------------------------- the format, in 64 bits
def _code_values():
    v = []
    for c in range(127):
        e, m = c >> 3, c & 7
        v.append(m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7))
    return np.array(v)


CODES = _code_values()


def encode(u):
    """|u| <= 448 -> codes: the nearest, ties to the even code; not finite -> 0x7f."""
    a = np.abs(np.where(np.isfinite(u), u, 0.0))
    hi = np.clip(np.searchsorted(CODES, a), 0, 126)
    lo = np.clip(hi - 1, 0, 126)
    dl, dh = a - CODES[lo], CODES[hi] - a
    c = np.where(dl < dh, lo, np.where(dh < dl, hi, np.where(lo % 2 == 0, lo, hi)))
    return np.where(np.isfinite(u), c | np.where(np.signbit(u), 128, 0), 0x7F).astype(np.uint8)


def decode(c):
    c = c.astype(np.int64)
    v = np.append(CODES, np.nan)[c & 127]
    return np.where(c & 128, -v, v)


def exponent(top):
    e = 0
    if top > 0:
        e = math.frexp(top)[1] - 12
        while 448.0 * 2.0 ** e < top:
            e += 1
    return min(max(e, -100), 120)


def blocks_of(x):
    R, C = x.shape
    nb = -(-C // 128)
    v = np.zeros((R, nb * 128))
    v[:, :C] = x
    return v.reshape(R, nb, 128)


def quantize(x):
    """-> (codes [R, Kp], exponents [nb, R])."""
    v = blocks_of(x.astype(np.float64))
    top = np.abs(np.where(np.isfinite(v), v, 0)).max(-1)
    e = np.vectorize(exponent, otypes=[np.int64])(top)
    with np.errstate(invalid="ignore"):
        q = encode(v / 2.0 ** e[..., None])
    return q.reshape(x.shape[0], -1), e.T


def quantize_weight(w):
    N, K = w.shape
    nb, rb = -(-K // 128), -(-N // 128)
    e = np.zeros((nb, rb), np.int64)
    q = np.zeros((N, nb * 128), np.uint8)
    for b in range(nb):
        for r in range(rb):
            blk = w[r * 128:(r + 1) * 128, b * 128:(b + 1) * 128].astype(np.float64)
            e[b, r] = exponent(np.abs(blk).max())
            q[r * 128:r * 128 + blk.shape[0], b * 128:b * 128 + blk.shape[1]] = encode(blk / 2.0 ** e[b, r])
    return q, e


def pack_scales(e):
    s = np.full((e.shape[0], (e.shape[1] + 15) // 16 * 16), 255, np.uint8)      # (behind the last row: NaN, must not matter)
    s[:, :e.shape[1]] = e + 127
    return s


def values(q, e, C):
    R = q.shape[0]
    return (decode(q).reshape(R, -1, 128) * 2.0 ** e.T[..., None]).reshape(R, -1)[:, :C]


def rows(seed, R, C, dtype, scale=1.0):
    """Rows with unequal sizes, a strong column, and (from 3 rows on) a row of zeros."""
    g = np.random.default_rng(seed)
    x = g.standard_normal((R, C)) * (0.25 + 2 * g.random((R, 1))) * scale
    x[:, C // 2] *= 20
    if R > 2:
        x[1] = 0
    return x.astype(dtype)


SHAPES = [(1, 1), (1, 128), (3, 8), (17, 320), (16, 640), (5, 77), (2, 129), (33, 1280), (19, 1000)]


# ------------------------------------------------------------------------------------------------------------ quantisation
def special_rows(dtype):
    x = np.zeros((7, 300), dtype)
    x[0, :128] = 448.0                                        # exactly the largest code
    x[0, 128:256] = np.nextafter(dtype(448.0), dtype(1000))   # just above: the next exponent
    x[1, 5] = np.inf
    x[1, 6] = -np.inf
    x[1, 7] = np.nan
    x[1, 8] = 3.0
    x[2, :] = np.nan
    x[3, 0] = np.finfo(dtype).max
    x[3, 1] = -np.finfo(dtype).max
    x[3, 130] = np.finfo(dtype).tiny
    x[4, 0] = np.finfo(dtype).smallest_subnormal
    x[5, :128] = np.linspace(-448, 448, 128)                  # ties and steps of every octave
    x[5, 128:256] = 2.0 ** -np.arange(128).clip(0, 20)
    x[5, 256:] = np.arange(44) * 0.5 + 0.25
    x[6, :] = -0.0
    return x


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("shape", SHAPES + ["special"])
def test_quantize_rows_bit_for_bit(kb, shape, dtype):
    x = special_rows(dtype) if shape == "special" else rows(1, *shape, dtype)
    R, C = x.shape
    nb = -(-C // 128)
    q, s = kb.up(np.full((R + 1, nb * 128), 0x55, np.uint8)), kb.up(np.full((nb, (R + 15) // 16 * 16), 0x55, np.uint8))
    assert kb.lib.ea_quantize_fp8(ptr(x), int(dtype is np.float32), ptr(q), ptr(s), R, C, kb.stream) == 0
    want, e = quantize(x)
    got, gs = kb.down(q), kb.down(s)
    assert (gs[:, :R] == e + 127).all()
    nan = want & 127 == 127
    assert (got[:R] == want)[~nan].all() and (got[:R][nan] & 127 == 127).all()
    assert (got[R] == 0x55).all(), "nothing behind the last row is written"
    assert (gs[:, R:] == 0x55).all()
    out = kb.zeros((R, C), np.float32)
    assert kb.lib.ea_dequantize_fp8(ptr(q), ptr(s), 1, ptr(out), 1, R, C, kb.stream) == 0
    with np.errstate(over="ignore"):           # (fp32's largest value rounds up to the code 256 at 2^120: 2^128 is infinite in fp32)
        ref = values(want, e, C).astype(np.float32)
    assert np.array_equal(kb.down(out), ref, equal_nan=True)


def test_blocks_below_the_smallest_exponent_read_as_zero_or_less(kb):
    x = np.zeros((2, 128), np.float32)
    x[0, 0], x[0, 1], x[1, 0] = 2.0 ** -95, 2.0 ** -108, 2.0 ** -120
    q, s = kb.zeros((2, 128), np.uint8), kb.zeros((1, 16), np.uint8)
    assert kb.lib.ea_quantize_fp8(ptr(x), 1, ptr(q), ptr(s), 2, 128, kb.stream) == 0
    want, e = quantize(x)
    assert (kb.down(q) == want).all() and (kb.down(s)[:, :2] == e + 127).all() and e[0, 1] == -100


@pytest.mark.parametrize("dtype", [np.float16, np.float32])
@pytest.mark.parametrize("N,K", [(1, 1), (128, 128), (130, 320), (77, 1000), (256, 257)])
def test_quantize_weight_bit_for_bit(kb, N, K, dtype):
    w = rows(2, N, K, dtype)
    nb = -(-K // 128)
    q, s = kb.zeros((N, nb * 128), np.uint8), kb.zeros((nb, -(-N // 128)), np.uint8)
    assert kb.lib.ea_quantize_fp8_weight(ptr(w), int(dtype is np.float32), ptr(q), ptr(s), N, K, kb.stream) == 0
    want, e = quantize_weight(w)
    assert (kb.down(q) == want).all() and (kb.down(s) == e + 127).all()
    out = kb.zeros((N, K), np.float16)
    assert kb.lib.ea_dequantize_fp8(ptr(q), ptr(s), 128, ptr(out), 0, N, K, kb.stream) == 0
    f = np.repeat(np.repeat(2.0 ** e.T, 128, 0)[:N], 128, 1)
    assert np.array_equal(kb.down(out), (decode(want) * f)[:, :K].astype(np.float16))


def test_a_transposed_weight_quantises_to_the_same_values(kb):
    w = rows(3, 200, 300, np.float32)
    a, ea = quantize_weight(w)
    b, eb = quantize_weight(np.ascontiguousarray(w.T))
    q, s = kb.zeros((300, 256), np.uint8), kb.zeros((2, 3), np.uint8)
    wt = np.ascontiguousarray(w.T)
    assert kb.lib.ea_quantize_fp8_weight(ptr(wt), 1, ptr(q), ptr(s), 300, 200, kb.stream) == 0
    assert (kb.down(q) == b).all() and (kb.down(s) == eb + 127).all() and (ea == eb.T).all()
    assert (a[:, :300] == b[:, :200].T).all()


# -------------------------------------------------------------------------------------------------------------- activations
def act64(z, act):
    """f(z), f'(z) of the single-input functions."""
    if act == SILU:
        with np.errstate(over="ignore"):
            s = 1 / (1 + np.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    P = 0.5 * (1 + erf(z / math.sqrt(2)))
    return z * P, P + z * np.exp(-z * z / 2) / math.sqrt(2 * math.pi)


ACT_ABS = 2e-6        # the GELU's own bound is 5.1e-7 (ea_platform.h); a slope adds x phi(x) <= 0.25 at fp32 exp accuracy (a few u32)


@pytest.mark.parametrize("fp8", [0, 1])
@pytest.mark.parametrize("act", [SILU, GELU, GEGLU])
@pytest.mark.parametrize("M,H", [(1, 1), (3, 128), (17, 320), (5, 77), (18, 1000), (2, 648)])
def test_activation_save(kb, M, H, act, fp8):
    g = 2 if act == GEGLU else 1
    z = rows(4, M, g * H, np.float16, 1.5)
    nb = -(-H // 128)
    zq, zs = kb.zeros((M * g, nb * 128), np.uint8), kb.zeros((nb, (M * g + 15) // 16 * 16), np.uint8)
    h = kb.up(np.full((M + 1, H), 7, np.float16))
    hq, hs = kb.zeros((M, nb * 128), np.uint8), kb.zeros((nb, (M + 15) // 16 * 16), np.uint8)
    assert kb.lib.ea_activation_fp8(ptr(z), act, None if fp8 else ptr(h), ptr(hq) if fp8 else None, ptr(hs) if fp8 else None, ptr(zq), ptr(zs), M,
                                    H, kb.stream) == 0
    want, e = quantize(z.reshape(M * g, H))
    assert (kb.down(zq) == want).all() and (kb.down(zs)[:, :M * g] == e + 127).all()
    z64 = z.astype(np.float64)
    v = z64[:, :H] if g == 2 else 1.0
    ref = v * act64(z64[:, H:] if g == 2 else z64, GELU if g == 2 else act)[0]
    tol = ACT_ABS * np.maximum(np.abs(v), 1) + 4 * U32 * np.abs(ref)
    if fp8:
        got = values(kb.down(hq), kb.down(hs)[:, :M].astype(np.int64) - 127, H)
        top = np.abs(blocks_of(ref)).max(-1, keepdims=True)
        # half a step of a code: 2^-4 of the value, or half of the smallest step 2^-9 * 2^E with 2^E <= 2 top / 448 (the next exponent may be taken)
        err = 2.0 ** -4 * np.abs(blocks_of(ref)) + 2.0 ** -10 * 2 * top / 448
        assert (np.abs(got - ref) <= err.reshape(M, -1)[:, :H] + 2 * tol).all()
        assert not kb.down(hq)[:, H:].any(), "the padding stays zero codes"
    else:
        assert (np.abs(kb.down(h)[:M] - ref) <= U16 * np.abs(ref) + TINY16 + tol).all()
        assert (kb.down(h)[M] == 7).all()


@pytest.mark.parametrize("act", [SILU, GELU, GEGLU])
@pytest.mark.parametrize("M,H", [(1, 1), (3, 128), (17, 320), (5, 77), (18, 1000)])
def test_activation_backward(kb, M, H, act):
    g = 2 if act == GEGLU else 1
    q, e = quantize(rows(5, M * g, H, np.float32, 1.5))
    dh = rows(6, M, H, np.float16, 0.05)
    z = values(q, e, H).reshape(M, g, H)
    dz = kb.zeros((M, g * H), np.float16)
    assert kb.lib.ea_activation_fp8_bwd(ptr(dh), ptr(q), ptr(pack_scales(e)), act, ptr(dz), M, H, kb.stream) == 0
    d = dh.astype(np.float64)
    if g == 2:
        f, s = act64(z[:, 1], GELU)
        ref = np.concatenate([d * f, d * z[:, 0] * s], 1)
        mag = np.concatenate([np.abs(d) * np.maximum(np.abs(z[:, 1]), 1), np.abs(d * z[:, 0])], 1)
    else:
        ref = d * act64(z[:, 0], act)[1]
        mag = np.abs(d) * np.maximum(np.abs(z[:, 0]), 1)      # (SiLU's slope: s's error enters times z)
    assert (np.abs(kb.down(dz) - ref) <= U16 * np.abs(ref) + TINY16 + ACT_ABS * mag + 8 * U32 * np.abs(ref)).all()
    if g == 1:                                               # the slope against differences of the function
        h = 1e-4
        num = (act64(z[:, 0] + h, act)[0] - act64(z[:, 0] - h, act)[0]) / (2 * h)
        assert (np.abs(kb.down(dz) - d * num) <= U16 * np.abs(ref) + TINY16 + (ACT_ABS + 1e-7) * mag + 8 * U32 * np.abs(ref)).all()


def test_activation_extremes(kb):
    """The ends of fp16, infinities and NaN: finite in, finite out; NaN stays NaN."""
    z = np.zeros((1, 128), np.float16)
    z[0, :8] = [65504, -65504, 30000, -12, 6.1e-5, -6e-8, 88.9, -88.9]
    z[0, 8] = np.nan
    for act in (SILU, GELU):
        h, zq, zs = kb.zeros((1, 128), np.float16), kb.zeros((1, 128), np.uint8), kb.zeros((1, 16), np.uint8)
        assert kb.lib.ea_activation_fp8(ptr(z), act, ptr(h), None, None, ptr(zq), ptr(zs), 1, 128, kb.stream) == 0
        got = kb.down(h).astype(np.float64)[0]
        ref = act64(z.astype(np.float64), act)[0][0]
        assert np.isnan(got[8]) and (np.abs(got[:8] - ref[:8]) <= U16 * np.abs(ref[:8]) + 1e-6).all() and not got[9:].any()
        dh, dz = np.ones((1, 128), np.float16), kb.zeros((1, 128), np.float16)
        assert kb.lib.ea_activation_fp8_bwd(ptr(dh), ptr(zq), ptr(zs), act, ptr(dz), 1, 128, kb.stream) == 0
        got = kb.down(dz).astype(np.float64)[0]
        assert np.isnan(got[8]) and np.isfinite(got[:8]).all() and (np.abs(got[9:] - 0.5) <= U16).all()


# ---------------------------------------------------------------------------------------------------------------- LayerNorm
def ln_stats(x, eps):
    mu = x.mean(1)
    return mu, 1 / np.sqrt(((x - mu[:, None]) ** 2).mean(1) + eps)


LN_SHAPES = [(1, 1), (1, 8), (5, 320), (70, 320), (9, 384), (6, 392), (37, 640), (5, 1280), (3, 1288), (2, 2560), (3, 2568), (2, 4096), (3, 77),
             (5, 513), (2, 1537), (2, 4095), (521, 40)]


@pytest.mark.parametrize("fp8", [0, 1])
@pytest.mark.parametrize("in_f32", [0, 1])
@pytest.mark.parametrize("M,C", LN_SHAPES)
def test_layernorm_train(kb, M, C, in_f32, fp8):
    x = rows(7, M, C, np.float32 if in_f32 else np.float16) + (np.float32 if in_f32 else np.float16)(0.5)
    gn = np.random.default_rng(8)
    gamma, beta = gn.standard_normal(C).astype(np.float32), gn.standard_normal(C).astype(np.float32)
    nb = -(-C // 128)
    y, q, s = kb.up(np.full((M + 1, C), 7, np.float16)), kb.zeros((M, nb * 128), np.uint8), kb.zeros((nb, (M + 15) // 16 * 16), np.uint8)
    st = kb.zeros((M, 2), np.float32)
    eps = 1e-5
    assert kb.lib.ea_layernorm_train(ptr(x), in_f32, ptr(gamma), ptr(beta), eps, None if fp8 else ptr(y), ptr(q) if fp8 else None,
                                     ptr(s) if fp8 else None, ptr(st), M, C, kb.stream) == 0
    x64 = x.astype(np.float64)
    mu, r = ln_stats(x64, eps)
    got = kb.down(st).astype(np.float64)
    # the mean's sum: C u32 sum |x| / C; the centred squares inherit it.  1 / sigma: half of the variance's relative error, + a few roundings
    emu = (C + 2) * U32 * np.abs(x64).mean(1)
    var = 1 / r ** 2
    erel = (0.5 * ((C + 4) * U32 * (var - eps) + 2 * emu * np.sqrt(var) + emu ** 2) / var) + 8 * U32
    assert (np.abs(got[:, 0] - mu) <= emu + U32 * np.abs(mu)).all() and (np.abs(got[:, 1] - r) <= erel * r).all()
    n = (x64 - mu[:, None]) * r[:, None]
    ref = n * gamma + beta
    en = emu[:, None] * r[:, None] + np.abs(n) * (erel[:, None] + 4 * U32)
    tol = en * np.abs(gamma) + 4 * U32 * (np.abs(ref) + np.abs(beta))
    if fp8:
        v = values(kb.down(q), kb.down(s)[:, :M].astype(np.int64) - 127, C)
        top = np.abs(blocks_of(ref)).max(-1, keepdims=True)
        err = (2.0 ** -4 * np.abs(blocks_of(ref)) + 2.0 ** -10 * 2 * top / 448).reshape(M, -1)[:, :C]
        assert (np.abs(v - ref) <= err + 2 * tol).all()
        assert not kb.down(q)[:, C:].any()
    else:
        assert (np.abs(kb.down(y)[:M] - ref) <= U16 * np.abs(ref) + TINY16 + tol).all()
        assert (kb.down(y)[M] == 7).all()


@pytest.mark.parametrize("launches", [1, 2])
@pytest.mark.parametrize("kind,res", [(0, 0), (0, 1), (1, 0), (1, 1), (2, 0), (2, 1)])
@pytest.mark.parametrize("M,C", LN_SHAPES)
def test_layernorm_backward(kb, M, C, kind, res, launches):
    force(kb, 100 + launches)
    x = rows(9, M, C, np.float32 if kind else np.float16)
    gn = np.random.default_rng(10)
    gamma = (1 + 0.3 * gn.standard_normal(C)).astype(np.float32)
    dy = (0.1 * gn.standard_normal((M, C))).astype(np.float16)
    out = np.float32 if kind == 1 else np.float16
    residual = (0.1 * gn.standard_normal((M, C))).astype(out) if res else None
    xs = None
    x64 = x.astype(np.float64)
    mu, r = ln_stats(x64, 1e-5)
    if kind == 2:
        q, e = quantize(x)
        x, xs, x64 = q, pack_scales(e), values(q, e, C)
    st = np.stack([mu, r], 1).astype(np.float32)
    dx, dg, db = kb.up(np.full((M + 1, C), 7, out)), kb.zeros((C,), np.float32), kb.zeros((C,), np.float32)
    nbytes = kb.lib.ea_layernorm_bwd_workspace_bytes(M, C)
    assert (nbytes > 0) == (launches == 2)
    ws = kb.zeros((nbytes // 4,), np.float32) if nbytes else None
    args = (ptr(dy), ptr(x), kind, ptr(xs), ptr(st), ptr(gamma), ptr(residual), ptr(dx), ptr(dg), ptr(db), M, C)
    if nbytes:
        assert kb.lib.ea_layernorm_bwd(*args, ptr(ws), nbytes - 1, kb.stream) == kb.lib.ea_layernorm_bwd(*args, None, nbytes, kb.stream) == -4
    assert kb.lib.ea_layernorm_bwd(*args, ptr(ws), nbytes, kb.stream) == 0
    mu, r = st.astype(np.float64).T
    n = (x64 - mu[:, None]) * r[:, None]
    d = dy.astype(np.float64)
    g = d * gamma
    ref = r[:, None] * (g - g.mean(1, keepdims=True) - n * (g * n).mean(1, keepdims=True)) + (0 if residual is None else residual.astype(np.float64))
    # the row sums are off by C u32 of their absolute means; everything else by a few roundings of the terms
    s1, s2 = np.abs(g).mean(1, keepdims=True), np.abs(g * n).mean(1, keepdims=True)
    nerr = U32 * r[:, None] * (np.abs(x64) + np.abs(mu[:, None])) + 2 * U32 * np.abs(n)
    tol = r[:, None] * ((C + 6) * U32 * (s1 + np.abs(n) * s2) + 6 * U32 * np.abs(g) + nerr * s2 + np.abs(n) * (np.abs(g) * nerr).mean(1, keepdims=True))
    got = kb.down(dx)
    assert (got[M] == 7).all()
    # (C = 1 in 8 bits: sigma = sqrt(eps) blows the decoding error up to 77577, which rounds to fp16's infinity from 65520 on)
    over = (np.abs(ref) >= 65520) & (kind != 1)
    assert np.isinf(got[:M][over]).all()
    err = np.abs(np.where(over, 0, got[:M]) - np.where(over, 0, ref))
    assert (err <= (U32 if kind == 1 else U16) * np.abs(ref) + (0 if kind == 1 else TINY16) + 1.01 * tol + 4 * U32 * np.abs(ref)).all()
    dg, db = kb.down(dg).astype(np.float64), kb.down(db).astype(np.float64)
    assert (np.abs(dg - (d * n).sum(0)) <= (M + 4) * U32 * np.abs(d * n).sum(0) + (np.abs(d) * nerr).sum(0) + 1e-30).all()
    assert (np.abs(db - d.sum(0)) <= (M + 2) * U32 * np.abs(d).sum(0)).all()


def test_layernorm_gradients_against_differences():
    """The formula that the kernels are held to, against central differences of the loss sum(w * LayerNorm(x)) in 64 bits."""
    g = np.random.default_rng(11)
    x, w, gamma, beta = g.standard_normal((3, 10)), g.standard_normal((3, 10)), g.standard_normal(10), g.standard_normal(10)

    def loss(x, gamma, beta):
        mu, r = ln_stats(x, 1e-5)
        return (w * ((x - mu[:, None]) * r[:, None] * gamma + beta)).sum()
    mu, r = ln_stats(x, 1e-5)
    n = (x - mu[:, None]) * r[:, None]
    k = w * gamma
    dx = r[:, None] * (k - k.mean(1, keepdims=True) - n * (k * n).mean(1, keepdims=True))
    h = 1e-6

    def diff(f, a):
        out = np.zeros_like(a)
        for i in np.ndindex(a.shape):
            p, m = a.copy(), a.copy()
            p[i] += h
            m[i] -= h
            out[i] = (f(p) - f(m)) / (2 * h)
        return out
    assert np.abs(diff(lambda v: loss(v, gamma, beta), x) - dx).max() < 1e-7
    assert np.abs(diff(lambda v: loss(x, v, beta), gamma) - (w * n).sum(0)).max() < 1e-7
    assert np.abs(diff(lambda v: loss(x, gamma, v), beta) - w.sum(0)).max() < 1e-7


# --------------------------------------------------------------------------------------------------------------- the product
def gemm_case(M, N, K, seed=12):
    aq, ae = quantize(rows(seed, M, K, np.float32))
    wq, we = quantize_weight(rows(seed + 1, N, K, np.float32, 0.1))
    a = values(aq, ae, K)
    w = (decode(wq) * np.repeat(np.repeat(2.0 ** we.T, 128, 0)[:N], 128, 1))[:, :K]
    return aq, pack_scales(ae), wq, (we + 127).astype(np.uint8), a @ w.T, np.abs(a) @ np.abs(w).T


def force(kb, kernel):
    """Pin one of gemm_fp8's kernels (0: the launch rule's own choice)."""
    if kernel:
        assert L.set_tuning(kb.lib, variant=kernel) == 0


KERNELS = [0, 101, 102, 103, 104]

# The matrix unit adds 8 neighbouring products of 8-bit operands before they meet the fp32 accumulator, each product cut towards zero at
# 2^-13 of the power of two of the eight's largest (measured: beside 256, seven products of 256 * 2^-13 all count and seven of
# 256 * 2^-14 all vanish, whatever their sign; products of other eights and the accumulator lose nothing).  So an eight is off by at
# most 7 * 2^-13 of its largest product, and a sum by that share of its sum of magnitudes.
UNIT = 7 * 2.0 ** -13

GEMM_SHAPES = [(1, 1, 1), (1, 128, 128), (16, 8, 130), (70, 100, 300), (128, 256, 256), (130, 72, 640), (33, 7, 77), (200, 264, 200)]


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("form", ["plain", "bias gelu fp32", "bias silu residual", "residual32 scale"])
@pytest.mark.parametrize("M,N,K", GEMM_SHAPES)
def test_gemm_fp8(kb, M, N, K, form, kernel):
    if kb.name == "emu" and kernel and (M, N) not in ((1, 1), (70, 100), (130, 72)):
        pytest.skip("every kernel at three shapes on the emulation, at all of them on the GPU")
    force(kb, kernel)
    aq, sa, wq, sw, ref, mag = gemm_case(M, N, K)
    g = np.random.default_rng(13)
    f32out = "fp32" in form
    out = kb.up(np.full((M + 1, N), 7, np.float32 if f32out else np.float16))
    bias = g.standard_normal(N).astype(np.float32) if "bias" in form else None
    res = g.standard_normal((M, N)).astype(np.float16) if "residual" in form and "32" not in form else None
    res32 = g.standard_normal((M, N)).astype(np.float32) if "residual32" in form else None
    act = GELU if "gelu" in form else SILU if "silu" in form else 0
    scale = 0.5 if "scale" in form else 1.0
    e = epilogue(out, bias=bias, act=act, scale=scale, residual=res, residual32=res32)
    assert kb.lib.ea_gemm_fp8(ptr(aq), ptr(sa), ptr(wq), ptr(sw), M, N, K, ctypes.byref(e), kb.stream) == 0
    v = ref + (0 if bias is None else bias.astype(np.float64))
    err = (2 * (K + 2) * U32 + UNIT) * mag + U32 * np.abs(v)
    if act:
        err = 1.13 * err + ACT_ABS + 4 * U32 * np.abs(v)           # (neither slope exceeds 1.13)
        v = act64(v, act)[0]
    v = scale * v + (0 if res is None else res.astype(np.float64)) + (0 if res32 is None else res32.astype(np.float64))
    got = kb.down(out)
    assert (got[M] == 7).all()
    assert (np.abs(got[:M] - v) <= scale * err + (2 * U32 if f32out else U16) * np.abs(v) + TINY16 + 4 * U32 * np.abs(v)).all()


@pytest.mark.parametrize("kernel", KERNELS)
@pytest.mark.parametrize("M,N,K", GEMM_SHAPES + [(300, 520, 512), (257, 300, 1300), (17, 24, 8450)])
def test_gemm_fp8_whole_numbers_exactly(kb, M, N, K, kernel):
    """Whole numbers up to 8 under per-block powers of two: every product and sum is a whole number of small steps that fp32 and the
    matrix unit hold, so the result has to be exact -- each row, column, block and scale in its place."""
    g = np.random.default_rng(19)
    nb = -(-K // 128)
    a, w = np.zeros((M, nb * 128)), np.zeros((N, nb * 128))
    a[:, :K], w[:, :K] = g.integers(-8, 9, (M, K)), g.integers(-8, 9, (N, K))
    ea, ew = g.integers(-2, 3, (nb, M)), g.integers(-1, 2, (nb, -(-N // 128)))
    aq, wq = encode(a), encode(w)
    out = kb.up(np.full((M + 1, N), 7, np.float32))
    force(kb, kernel)
    assert kb.lib.ea_gemm_fp8(ptr(aq), ptr(pack_scales(ea)), ptr(wq), ptr((ew + 127).astype(np.uint8)), M, N, K, ctypes.byref(epilogue(out)),
                              kb.stream) == 0
    ref = values(aq, ea, K) @ (decode(wq) * np.repeat(np.repeat(2.0 ** ew.T, 128, 0)[:N], 128, 1))[:, :K].T
    got = kb.down(out)
    assert np.array_equal(got[:M], ref) and (got[M] == 7).all()


def test_gemm_fp8_exponents_and_nan(kb):
    """Exponents far apart in one row and in one weight; a NaN code reaches its own row only."""
    M, N, K = 20, 24, 384
    a, w = rows(14, M, K, np.float32), rows(15, N, K, np.float32)
    a[:, :128] *= 2.0 ** 40
    a[:, 256:] *= 2.0 ** -40
    w[:, :128] *= 2.0 ** -38
    w[:, 256:] *= 2.0 ** 41
    aq, ae = quantize(a)
    wq, we = quantize_weight(w)
    aq[3, 200] = 0x7F
    av, wv = values(aq, ae, K), decode(wq) * np.repeat(2.0 ** we.T, 128, 1)
    out = kb.zeros((M, N), np.float32)
    assert kb.lib.ea_gemm_fp8(ptr(aq), ptr(pack_scales(ae)), ptr(wq), ptr((we + 127).astype(np.uint8)), M, N, K,
                              ctypes.byref(epilogue(out)), kb.stream) == 0
    got = kb.down(out).astype(np.float64)
    assert np.isnan(got[3]).all()
    keep = np.arange(M) != 3
    ref, mag = (av @ wv.T)[keep], (np.abs(av) @ np.abs(wv).T)[keep]
    assert (np.abs(got[keep] - ref) <= (2 * (K + 2) * U32 + UNIT) * mag).all()


def test_gemm_fp8_residual_may_be_the_output(kb):
    M, N, K = 40, 16, 128
    aq, sa, wq, sw, ref, mag = gemm_case(M, N, K)
    r = np.random.default_rng(16).standard_normal((M, N)).astype(np.float16)
    out = kb.up(r.copy())
    e = epilogue(out)
    e.residual, e.ldr = ptr(out), N
    assert kb.lib.ea_gemm_fp8(ptr(aq), ptr(sa), ptr(wq), ptr(sw), M, N, K, ctypes.byref(e), kb.stream) == 0
    v = ref + r.astype(np.float64)
    assert (np.abs(kb.down(out) - v) <= (2 * (K + 2) * U32 + UNIT) * mag + U16 * np.abs(v) + TINY16 + 4 * U32 * np.abs(v)).all()


# ------------------------------------------------------------------------------------------------------------ weight gradient
@pytest.mark.parametrize("kernel", [0, 101, 102, 103])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (1, 8, 128), (64, 128, 128), (70, 104, 300), (130, 136, 77), (333, 24, 200), (600, 130, 129), (65, 7, 640),
                                   (2250, 264, 260)])
def test_gemm_fp8_wgrad(kb, M, N, K, kernel):
    force(kb, kernel)
    q, e = quantize(rows(17, M, K, np.float32))
    dy = rows(18, M, N, np.float16, 0.05)
    dw, db = kb.up(np.full((N + 1, K), 7, np.float32)), kb.up(np.full((N + 1,), 7, np.float32))
    nbytes = kb.lib.ea_gemm_fp8_wgrad_workspace_bytes(M, N, K)
    ws = kb.zeros((nbytes // 4,), np.float32) if nbytes else None
    assert kb.lib.ea_gemm_fp8_wgrad(ptr(dy), ptr(q), ptr(pack_scales(e)), ptr(dw), ptr(db), M, N, K, ptr(ws), nbytes, kb.stream) == 0
    x, d = values(q, e, K), dy.astype(np.float64)
    gw, gb = kb.down(dw), kb.down(db)
    # x / 2 in fp16 may lose its last bits below 2^-14: at most 2^-25 each, doubled
    assert (np.abs(gw[:N] - d.T @ x) <= 2 * (M + 2) * U32 * (np.abs(d).T @ np.abs(x)) + 2.0 ** -24 * np.abs(d).sum(0)[:, None] + 1e-30).all()
    assert (np.abs(gb[:N] - d.sum(0)) <= 2 * (M + 2) * U32 * np.abs(d).sum(0)).all()
    assert (gw[N] == 7).all() and gb[N] == 7


def test_gemm_fp8_wgrad_range(kb):
    """fp16's largest value (its code rounds up to 65536) and its smallest ones go through the 8-bit input."""
    x = np.zeros((4, 128), np.float16)
    x[0, 0], x[1, 1], x[2, 2], x[3, 3] = 65504, -65504, 2.0 ** -24, 1e-4
    q, e = quantize(x)
    dy = np.eye(4, 8).astype(np.float16)
    dw, db = kb.zeros((8, 128), np.float32), kb.zeros((8,), np.float32)
    assert kb.lib.ea_gemm_fp8_wgrad(ptr(dy), ptr(q), ptr(pack_scales(e)), ptr(dw), ptr(db), 4, 8, 128, None, 0, kb.stream) == 0
    assert np.abs(kb.down(dw)[:4] - values(q, e, 128)).max() <= 2.0 ** -24 and kb.down(dw)[0, 0] == 65536


@pytest.mark.parametrize("kernel", [0, 101, 102, 103])
def test_gemm_fp8_wgrad_keeps_nan_and_infinity_in_their_row_and_column(kb, kernel):
    """An infinity in dy column n and a NaN code in x column k: row n and column k of dw and db[n] alone show them."""
    M, N, K = 70, 264, 300
    force(kb, kernel)
    q, e = quantize(rows(19, M, K, np.float32))
    dy = rows(20, M, N, np.float16, 0.05)
    q[9, 140] = 0x7f
    cols = [21, 77, 200]
    dy[[3, 40, 69], cols] = np.inf, np.nan, -np.inf
    dw, db = kb.zeros((N, K), np.float32), kb.zeros((N,), np.float32)
    nbytes = kb.lib.ea_gemm_fp8_wgrad_workspace_bytes(M, N, K)
    ws = kb.zeros((nbytes // 4,), np.float32) if nbytes else None
    assert kb.lib.ea_gemm_fp8_wgrad(ptr(dy), ptr(q), ptr(pack_scales(e)), ptr(dw), ptr(db), M, N, K, ptr(ws), nbytes, kb.stream) == 0
    gw, gb = np.isfinite(kb.down(dw)), np.isfinite(kb.down(db))
    want = np.ones((N, K), bool)
    want[:, 140] = want[cols] = False
    assert np.array_equal(gw, want) and np.array_equal(gb, want[:, 0])


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_more_rows_than_an_index_holds_are_refused(emu_lib):
    """Rows counted in 32 bits end at 2^30; nothing is read before the refusal."""
    a = np.zeros((256, 256), np.float32)
    p, big = a.ctypes.data, (1 << 30) + 1
    e = epilogue(a)
    assert emu_lib.ea_layernorm_train(p, 0, p, p, 1e-5, p, None, None, p, big, 8, None) == -1
    assert emu_lib.ea_layernorm_bwd(p, p, 0, None, p, p, None, p, p, p, big, 8, p, 1 << 40, None) == -1
    assert emu_lib.ea_layernorm_bwd_workspace_bytes(big, 8) == 0
    assert emu_lib.ea_gemm_fp8(p, p, p, p, big, 16, 128, ctypes.byref(e), None) == -1
    assert emu_lib.ea_gemm_fp8(p, p, p, p, 16, (1 << 22) + 1, 128, ctypes.byref(e), None) == -1
    assert emu_lib.ea_gemm_fp8_wgrad(p, p, p, p, p, big, 16, 16, None, 0, None) == -1
    assert emu_lib.ea_gemm_fp8_wgrad_workspace_bytes(big, 16, 16) == 0
    one = torch.ones(8)
    for n in (big, (1 << 32) + 5):             # (the second is 5 in 32 bits)
        x = torch.zeros(1, 8, dtype=torch.float16).expand(n, 8)
        t = ops.Fp8Tensor.__new__(ops.Fp8Tensor)
        t.q, t.scale, t.cols, t.rows, t.shape, t.block_rows = torch.zeros(1, 128).to(torch.float8_e4m3fn), torch.zeros(1, 16), 8, n, (n, 8), 1
        w = ops.Fp8Tensor(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8), 8)
        for f in (lambda: ops.layernorm_train(x, one, one), lambda: ops.layernorm_backward(x, x, torch.zeros(1, 2).expand(n, 2), one),
                  lambda: ops.gemm_fp8(t, w), lambda: ops.gemm_fp8_wgrad(x, t)):
            with pytest.raises(ValueError, match="2\\^30"):
                f()


def test_the_c_entries_refuse(emu_lib):
    lib = emu_lib
    a = np.zeros((256, 256), np.float32)
    p, o = a.ctypes.data, a.ctypes.data + 1024
    assert lib.ea_quantize_fp8(None, 0, p, p, 1, 8, None) == -2
    assert lib.ea_quantize_fp8(p, 0, p, p, 0, 8, None) == -1
    assert lib.ea_quantize_fp8(p, 0, p, p, 1, 0, None) == -1
    assert lib.ea_quantize_fp8(p, 0, p + 1, p, 1, 8, None) == -2
    assert lib.ea_quantize_fp8(p, 0, p, p, 1 << 40, 8, None) == -1
    assert lib.ea_quantize_fp8_weight(p, 0, p, None, 8, 8, None) == -2
    assert lib.ea_quantize_fp8_weight(p, 0, p, p, 0, 8, None) == -1
    assert lib.ea_dequantize_fp8(p, p, 64, o, 0, 1, 8, None) == -2
    assert lib.ea_activation_fp8(p, 0, o, None, None, p, p, 1, 8, None) == -2                 # no activation
    assert lib.ea_activation_fp8(p, GELU, o, o, p, p, p, 1, 8, None) == -2                    # two outputs
    assert lib.ea_activation_fp8(p, GELU, None, None, None, p, p, 1, 8, None) == -2           # none
    assert lib.ea_activation_fp8(p, GELU, None, o, None, p, p, 1, 8, None) == -2              # codes without scales
    assert lib.ea_activation_fp8(p, GELU, o, None, None, p, p, 1, 0, None) == -1
    assert lib.ea_activation_fp8_bwd(p, p, None, GELU, o, 1, 8, None) == -2
    assert lib.ea_activation_fp8_bwd(p, p, p, 7, o, 1, 8, None) == -2
    assert lib.ea_layernorm_train(p, 0, p, p, 1e-5, None, None, None, p, 1, 8, None) == -2
    assert lib.ea_layernorm_train(p, 0, p, p, 1e-5, o, None, None, p, 1, 4097, None) == -1
    assert lib.ea_layernorm_train(p, 0, p, p, 1e-5, o, None, None, p + 4, 1, 8, None) == -2
    assert lib.ea_layernorm_bwd(p, p, 3, None, p, p, None, o, o, o, 1, 8, p, 1 << 20, None) == -2
    assert lib.ea_layernorm_bwd(p, p, 2, None, p, p, None, o, o, o, 1, 8, p, 1 << 20, None) == -2
    assert lib.ea_layernorm_bwd(p, p, 0, None, p, p, None, o, o, o, 1, 5000, p, 1 << 20, None) == -1
    assert lib.ea_layernorm_bwd(p, p, 0, None, p, p, None, o, o, o, 4096, 8, p, 0, None) == -4
    assert lib.ea_layernorm_bwd_workspace_bytes(0, 8) == 0 and lib.ea_layernorm_bwd_workspace_bytes(1, 4097) == 0
    e = epilogue(a)
    g = lambda **kw: lib.ea_gemm_fp8(kw.get("a", p), kw.get("sa", p), p, p, kw.get("M", 16), kw.get("N", 16), kw.get("K", 128),  # noqa: E731
                                     ctypes.byref(kw.get("e", e)), None)
    assert g(a=None) == -2 and g(a=p + 8) == -2 and g(sa=p + 1) == -2
    assert g(M=0) == -1 and g(N=-1) == -1 and g(K=0) == -1 and g(K=1 << 21) == -1
    assert g(N=512) == -2                                                                      # ldc < N
    for field, bad in (("act", GEGLU), ("bias_per_row", 1), ("rowvec", p), ("row_scale", p), ("ln_stats", p), ("row_stats_out", p),
                       ("gn_stats_out", p), ("gn_next_out", p), ("acc_scale_k", 64)):
        b = epilogue(a)
        setattr(b, field, bad)
        assert g(e=b) == -3, field
    b = epilogue(a)
    b.residual = b.residual32 = p
    assert g(e=b) == -2
    w = lambda **kw: lib.ea_gemm_fp8_wgrad(p, kw.get("x", p), p, kw.get("dw", o), o, kw.get("M", 4096), 16, kw.get("K", 16), None,  # noqa: E731
                                           kw.get("n", 0), None)
    assert w(x=None) == -2 and w(x=p + 4) == -2 and w(M=0) == -1 and w(K=1 << 21) == -1
    assert lib.ea_gemm_fp8_wgrad_workspace_bytes(4096, 16, 16) > 0 and w() == -4 and w(n=1 << 30) == -4
    assert lib.ea_gemm_fp8_wgrad_workspace_bytes(16, 16, 0) == 0


def test_the_public_functions_refuse():
    f16, f32 = torch.zeros(4, 8, dtype=torch.float16), torch.zeros(4, 8)
    q = torch.zeros(4, 128).to(torch.float8_e4m3fn)
    rows_s, weight_s = torch.zeros(1, 16, dtype=torch.uint8), torch.zeros(1, 1, dtype=torch.uint8)
    t, w = ops.Fp8Tensor(q, rows_s, 8), ops.Fp8Tensor(q, weight_s, 8)
    assert (t.block_rows, t.rows, tuple(t.shape), w.block_rows) == (1, 4, (4, 8), 128)
    bad = [lambda: ops.Fp8Tensor(q, rows_s, 129), lambda: ops.Fp8Tensor(q.view(torch.uint8), rows_s, 8), lambda: ops.Fp8Tensor(q, rows_s, 0),
           lambda: ops.Fp8Tensor(q, rows_s.int(), 8), lambda: ops.Fp8Tensor(q, torch.zeros(1, 4, dtype=torch.uint8), 8),
           lambda: ops.Fp8Tensor(q, rows_s, 8, (2, 8)),
           lambda: ops.quantize_fp8(f16.double()), lambda: ops.quantize_fp8(torch.zeros((), dtype=torch.float16)), lambda: ops.quantize_fp8("x"),
           lambda: ops.quantize_fp8(torch.zeros(4, 0)), lambda: ops.quantize_fp8_weight(torch.zeros(2, 2, 2)),
           lambda: ops.quantize_fp8_weight(torch.zeros(0, 8)), lambda: ops.dequantize_fp8(f16), lambda: ops.dequantize_fp8(t, torch.bfloat16),
           lambda: ops.layernorm_train(torch.zeros(1, 4097), torch.zeros(4097), torch.zeros(4097)),
           lambda: ops.layernorm_train(f16, torch.zeros(8).half(), torch.zeros(8)), lambda: ops.layernorm_train(f16, torch.zeros(7), torch.zeros(8)),
           lambda: ops.layernorm_backward(f32, f16, torch.zeros(4, 2), torch.zeros(8)),
           lambda: ops.layernorm_backward(f16, f16[:2], torch.zeros(4, 2), torch.zeros(8)),
           lambda: ops.layernorm_backward(f16, w, torch.zeros(4, 2), torch.zeros(8)),
           lambda: ops.layernorm_backward(f16, f16, torch.zeros(4, 1), torch.zeros(8)),
           lambda: ops.layernorm_backward(f16, f16, torch.zeros(4, 2), torch.zeros(8), residual=f32),
           lambda: ops.layernorm_backward(f16, f32, torch.zeros(4, 2), torch.zeros(8), residual=f16),
           lambda: ops.activation_fp8(f16, ops.ACT_NONE), lambda: ops.activation_fp8(f32, ops.ACT_GELU),
           lambda: ops.activation_fp8(torch.zeros(4, 7, dtype=torch.float16), ops.ACT_GEGLU),
           lambda: ops.activation_fp8_backward(f16, w, ops.ACT_GELU), lambda: ops.activation_fp8_backward(f16, t, ops.ACT_GEGLU),
           lambda: ops.activation_fp8_backward(f16, f16, ops.ACT_GELU), lambda: ops.activation_fp8_backward(f16[:3], t, ops.ACT_GELU),
           lambda: ops.gemm_fp8(w, w), lambda: ops.gemm_fp8(t, t), lambda: ops.gemm_fp8(f16, w),
           lambda: ops.gemm_fp8(t, ops.Fp8Tensor(q, weight_s, 9)), lambda: ops.gemm_fp8(t, w, act=ops.ACT_GEGLU),
           lambda: ops.gemm_fp8(t, w, bias=torch.zeros(5)), lambda: ops.gemm_fp8(t, w, bias=torch.zeros(4).half()),
           lambda: ops.gemm_fp8(t, w, residual=f16), lambda: ops.gemm_fp8(t, w, out=torch.zeros(4, 4, dtype=torch.bfloat16)),
           lambda: ops.gemm_fp8(t, w, out_dtype=torch.bfloat16),
           lambda: ops.gemm_fp8_wgrad(f32, t), lambda: ops.gemm_fp8_wgrad(f16[:3], t), lambda: ops.gemm_fp8_wgrad(f16, w)]
    for k, f in enumerate(bad):
        with pytest.raises(ValueError):
            f()
            pytest.fail(f"call {k} was not refused")
    one, zero = torch.ones(8), torch.zeros(4, 2)
    for f in (lambda: ops.quantize_fp8(f16), lambda: ops.quantize_fp8_weight(f16), lambda: ops.layernorm_train(f16, one, one),
              lambda: ops.layernorm_backward(f16, f16, zero, one), lambda: ops.activation_fp8(f16, ops.ACT_SILU),
              lambda: ops.activation_fp8_backward(f16, t, ops.ACT_SILU), lambda: ops.gemm_fp8(t, w), lambda: ops.gemm_fp8_wgrad(f16, t)):
        with pytest.raises(RuntimeError, match="MI355X"):      # no CPU path
            f()


def test_gemm_fp8_refuses_a_residual_that_overlaps_the_output():
    t = ops.Fp8Tensor(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 16, dtype=torch.uint8), 8)
    w = ops.Fp8Tensor(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8), 8)
    buf = torch.zeros(8, 4)
    for out, res in ((buf[:4], buf[1:5]), (buf[3:7], buf[:4]), (buf[:4], buf.view(torch.float16).view(16, 4)[:4])):
        with pytest.raises(ValueError, match="apart"):
            ops.gemm_fp8(t, w, out=out, residual=res)
    for out, res in ((buf[:4], buf[:4]), (buf[:4], buf[4:])):       # accepted: on the CPU only the missing device stops them
        with pytest.raises(RuntimeError, match="MI355X"):
            ops.gemm_fp8(t, w, out=out, residual=res)


# --------------------------------------------------------------------------------------------------------- capturing, on the CPU
def test_no_garbage_collection_inside_a_capture(monkeypatch):
    """A dead cycle is not collected while any thread captures, and collection is as it was afterwards, also behind errors."""
    import gc
    import threading

    class Fake:
        def __init__(self, graph, fail=False, **kw):
            self.fail = fail

        def __enter__(self):
            if self.fail:
                raise RuntimeError("no capture")

        def __exit__(self, *exc):
            return None
    monkeypatch.setattr(torch.cuda, "graph", Fake)
    assert gc.isenabled()
    with ops.graph_capture(None, capture_error_mode="thread_local"):
        assert not gc.isenabled()
        t = threading.Thread(target=lambda: ops.graph_capture(None).__enter__())      # a capture that is still open on another thread
        t.start()
        t.join()
    assert not gc.isenabled()
    ops.graph_capture(None).__exit__(None, None, None)
    assert gc.isenabled()
    with pytest.raises(RuntimeError):
        with ops.graph_capture(None, fail=True):
            pass
    with pytest.raises(KeyError):
        with ops.graph_capture(None):
            raise KeyError
    assert gc.isenabled()
    gc.disable()
    try:
        with ops.graph_capture(None):
            pass
        assert not gc.isenabled()                               # it was off before
    finally:
        gc.enable()


# ------------------------------------------------------------------------------------------- the public functions, on the GPU
def block_inputs(seed, shape, hidden, dtype=torch.float16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    C = shape[-1]
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    return dict(x=r(*shape).to(dtype), gamma=1 + 0.2 * r(C), beta=0.1 * r(C), w1=r(hidden, C) * C ** -0.5, b1=0.1 * r(hidden),
                w2=r(C, hidden) * hidden ** -0.5, b2=0.1 * r(C), dout=(0.02 * r(*shape)).half())


def block_weights(s):
    return dict(q1=ops.quantize_fp8_weight(s["w1"]), q2=ops.quantize_fp8_weight(s["w2"]), q1t=ops.quantize_fp8_weight(s["w1"].t().contiguous()),
                q2t=ops.quantize_fp8_weight(s["w2"].t().contiguous()))


def block(s, w):
    """x + Linear(GELU(Linear(LayerNorm(x)))), forward and backward, what is kept for the backward pass in 8 bits."""
    y8, stats = ops.layernorm_train(s["x"], s["gamma"], s["beta"], fp8=True)
    z = ops.gemm_fp8(y8, w["q1"], bias=s["b1"])
    h8, z8 = ops.activation_fp8(z, ops.ACT_GELU, fp8=True)
    out = ops.gemm_fp8(h8, w["q2"], bias=s["b2"], residual=s["x"])
    d8 = ops.quantize_fp8(s["dout"])
    dh = ops.gemm_fp8(d8, w["q2t"])
    dw2, db2 = ops.gemm_fp8_wgrad(s["dout"], h8)
    dz = ops.activation_fp8_backward(dh, z8, ops.ACT_GELU)
    dy = ops.gemm_fp8(ops.quantize_fp8(dz), w["q1t"])
    dw1, db1 = ops.gemm_fp8_wgrad(dz, y8)
    dx, dgamma, dbeta = ops.layernorm_backward(dy, s["x"], stats, s["gamma"], residual=s["dout"])
    return dict(y=y8.q, ys=y8.scale[:, :y8.rows], stats=stats, z=z, h=h8.q, hs=h8.scale[:, :h8.rows], zq=z8.q, out=out, dh=dh, dz=dz, dy=dy, dw1=dw1,
                db1=db1, dw2=dw2, db2=db2, dx=dx, dgamma=dgamma, dbeta=dbeta)


def same_bits(a, b):
    return all(torch.equal(a[k].view(torch.uint8) if a[k].dtype == torch.float8_e4m3fn else a[k],
                           b[k].view(torch.uint8) if b[k].dtype == torch.float8_e4m3fn else b[k]) for k in a)


@pytest.mark.gpu
@pytest.mark.parametrize("shape,hidden", [((2, 77, 320), 1280), ((3, 5, 136), 264), ((1, 1, 640), 640)])
def test_block_step_by_step(shape, hidden):
    """Every step of a whole block against the same step in 64 bits on the operands that it was really given."""
    s = block_inputs(1, shape, hidden)
    w = block_weights(s)
    M, C = shape[0] * shape[1], shape[2]
    d = lambda t: t.double().reshape(M, -1)  # noqa: E731
    v = lambda q, sc, c: ops.Fp8Tensor(q, torch.nn.functional.pad(sc, (0, -M % 16)).contiguous(), c).dequantize(torch.float32).double()  # noqa: E731
    r = block(s, w)
    assert tuple(r["out"].shape) == shape and tuple(r["z"].shape) == shape[:2] + (hidden,) and tuple(r["dx"].shape) == shape
    y, h = v(r["y"], r["ys"], C), v(r["h"], r["hs"], hidden)
    W1, W2 = (w[k].dequantize(torch.float32).double() for k in ("q1", "q2"))
    near = lambda got, ref, mag, n: ((d(got) - ref).abs() <= (2 * (n + 2) * U32 + UNIT) * mag + U16 * ref.abs() + TINY16 + 8 * U32 * ref.abs()).all()  # noqa: E731
    assert near(r["z"], y @ W1.t().contiguous() + s["b1"].double(), y.abs() @ W1.abs().t().contiguous(), C)
    res = d(s["x"])
    assert near(r["out"], h @ W2.t().contiguous() + s["b2"].double() + res, h.abs() @ W2.abs().t().contiguous() + res.abs(), hidden)
    dq = ops.quantize_fp8(s["dout"]).dequantize(torch.float32).double().reshape(M, C)
    assert near(r["dh"], dq @ W2, dq.abs() @ W2.abs(), C)
    zq = ops.quantize_fp8(r["z"]).dequantize(torch.float32).double().reshape(M, hidden)
    slope = 0.5 * torch.erfc(-zq / math.sqrt(2)) + zq * torch.exp(-zq * zq / 2) / math.sqrt(2 * math.pi)
    ref = d(r["dh"]) * slope
    assert ((d(r["dz"]) - ref).abs() <= U16 * ref.abs() + TINY16 + ACT_ABS * d(r["dh"]).abs() * zq.abs().clamp_min(1) + 8 * U32 * ref.abs()).all()
    eq = ops.quantize_fp8(r["dz"]).dequantize(torch.float32).double().reshape(M, hidden)
    assert near(r["dy"], eq @ W1, eq.abs() @ W1.abs(), hidden)
    for dw, db, dd, xx in ((r["dw1"], r["db1"], d(r["dz"]), y), (r["dw2"], r["db2"], d(s["dout"]), h)):
        tol = 2 * (M + 2) * U32 * (dd.abs().t().contiguous() @ xx.abs()) + 2.0 ** -24 * dd.abs().sum(0)[:, None] + 1e-30
        assert ((dw.double() - dd.t().contiguous() @ xx).abs() <= tol).all()
        assert ((db.double() - dd.sum(0)).abs() <= 2 * (M + 2) * U32 * dd.abs().sum(0)).all()
    mu, rs = r["stats"][:, :1].double(), r["stats"][:, 1:].double()
    n, g = (d(s["x"]) - mu) * rs, d(r["dy"]) * s["gamma"].double()
    s1, s2 = g.mean(1, keepdim=True), (g * n).mean(1, keepdim=True)
    ref = rs * (g - s1 - n * s2) + d(s["dout"])
    mag = rs * (g.abs() + g.abs().mean(1, keepdim=True) + n.abs() * (g * n).abs().mean(1, keepdim=True)) + d(s["dout"]).abs()
    assert ((d(r["dx"]) - ref).abs() <= U16 * ref.abs() + TINY16 + (2 * C + 16) * U32 * mag).all()
    for got, terms in ((r["dgamma"], d(r["dy"]) * n), (r["dbeta"], d(r["dy"]))):
        assert ((got.double() - terms.sum(0)).abs() <= (M + 16) * U32 * terms.abs().sum(0) + 1e-30).all()


@pytest.mark.gpu
def test_a_block_repeats_bit_for_bit_on_any_stream():
    s = block_inputs(2, (2, 333, 640), 2560)
    w = block_weights(s)
    ref = block(s, w)
    assert same_bits(ref, block(s, w))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        t = {k: v.clone() for k, v in s.items()}
        got = block(t, block_weights(t))
    # ... beside matrix products on the main stream
    a = torch.randn(4096, 4096, device="cuda", dtype=torch.float16)
    for _ in range(20):
        a = (a @ a).clamp_(-1, 1)
    for _ in range(4):
        with torch.cuda.stream(side):
            got2 = block(t, block_weights(t))
        a = (a @ a).clamp_(-1, 1)
    torch.cuda.synchronize()
    assert same_bits(ref, got) and same_bits(ref, got2)


@pytest.mark.gpu
def test_a_captured_block_replays_with_new_inputs():
    """Two graphs of two blocks, replayed on two streams at once, several times, with eager work in between: always the eager result."""
    cases = []
    for seed, shape, hidden in ((3, (2, 100, 320), 1280), (4, (1, 640, 648), 1296)):
        s = block_inputs(seed, shape, hidden)
        w = block_weights(s)
        block(s, w)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with ops.graph_capture(g):
            out = block(s, w)
        cases.append((s, w, g, out, torch.cuda.Stream()))
    for k in range(4):
        refs = []
        for s, w, g, out, st in cases:
            for name, t in block_inputs(10 + k, s["x"].shape, s["w1"].shape[0]).items():
                if name in ("x", "dout"):
                    s[name].copy_(t)
            refs.append({n: t.clone() for n, t in block(s, w).items()})
        torch.cuda.synchronize()
        for s, w, g, out, st in cases:
            with torch.cuda.stream(st):
                g.replay()
        torch.cuda.synchronize()
        for ref, (s, w, g, out, st) in zip(refs, cases):
            assert same_bits(ref, out), k


@pytest.mark.gpu
def test_empty_and_unaligned_inputs():
    e16, one = torch.empty(0, 5, 320, device="cuda", dtype=torch.float16), torch.ones(320, device="cuda")
    q = ops.quantize_fp8(e16)
    assert tuple(q.shape) == (0, 5, 320) and tuple(q.dequantize().shape) == (0, 5, 320)
    y, st = ops.layernorm_train(e16, one, one)
    dx, dg, db = ops.layernorm_backward(e16, e16, st, one)
    assert y.numel() == dx.numel() == st.numel() == 0 and not dg.any() and not db.any() and dg.shape == (320,)
    h, z = ops.activation_fp8(e16, ops.ACT_GEGLU)
    assert tuple(h.shape) == (0, 5, 160) and tuple(ops.activation_fp8_backward(h, z, ops.ACT_GEGLU).shape) == (0, 5, 320)
    w = ops.quantize_fp8_weight(torch.randn(24, 320, device="cuda"))
    assert tuple(ops.gemm_fp8(q, w).shape) == (0, 5, 24)
    dw, b = ops.gemm_fp8_wgrad(torch.empty(0, 5, 24, device="cuda", dtype=torch.float16), q)
    assert tuple(dw.shape) == (24, 320) and not dw.any() and not b.any()
    # contiguous, but one element off every alignment: the same rules of arithmetic, another code path
    g = torch.Generator(device="cuda").manual_seed(5)
    odd = lambda *s: torch.randn(math.prod(s) + 1, generator=g, device="cuda").half()[1:].view(*s)  # noqa: E731
    x, dy, res = odd(70, 320), odd(70, 320), odd(70, 320)
    qa, qb = ops.quantize_fp8(x), ops.quantize_fp8(x.clone())
    assert torch.equal(qa.q.view(torch.uint8), qb.q.view(torch.uint8)) and torch.equal(qa.scale[:, :70], qb.scale[:, :70])
    for act in (ops.ACT_SILU, ops.ACT_GEGLU):
        a, sa = ops.activation_fp8(x, act)
        b, sb = ops.activation_fp8(x.clone(), act)
        dh = odd(*a.shape)
        assert torch.equal(sa.q.view(torch.uint8), sb.q.view(torch.uint8))
        # two compilations of one formula: each within half a step of fp16 and ACT_ABS times its factors of the exact value
        for u, v in ((a, b), (ops.activation_fp8_backward(dh, sa, act), ops.activation_fp8_backward(dh.clone(), sb, act))):
            slack = 2 * TINY16 + 2 * ACT_ABS * float(x.abs().max().clamp_min(1) * dh.abs().max().clamp_min(1))
            assert ((u.double() - v.double()).abs() <= 2 * U16 * 1.001 * v.double().abs() + slack).all()
    close = lambda a, b, tol: (a.double() - b.double()).abs().max() <= tol * b.double().abs().max()  # noqa: E731
    ga = torch.randn(321, generator=g, device="cuda")[1:]
    (y1, s1), (y2, s2) = ops.layernorm_train(x, ga, ga), ops.layernorm_train(x.clone(), ga.clone(), ga.clone())
    assert close(y1, y2, 2 * U16) and close(s1, s2, 64 * U32)
    r1, r2 = ops.layernorm_backward(dy, x, s2, ga, res), ops.layernorm_backward(dy.clone(), x.clone(), s2, ga.clone(), res.clone())
    assert close(r1[0], r2[0], 2 * U16) and close(r1[1], r2[1], 1024 * U32) and close(r1[2], r2[2], 1024 * U32)
    w = ops.quantize_fp8_weight(torch.randn(24, 320, generator=g, device="cuda"))
    rs, o = odd(70, 24), odd(70, 24)
    assert torch.equal(ops.gemm_fp8(qa, w, residual=rs, out=o), ops.gemm_fp8(qa, w, residual=rs.clone()))
    (a1, b1), (a2, b2) = ops.gemm_fp8_wgrad(rs, qa), ops.gemm_fp8_wgrad(rs.clone(), qa)
    assert close(a1, a2, 1024 * U32) and close(b1, b2, 1024 * U32)


@pytest.mark.gpu
def test_offsets_behind_32_bits():
    """More than 2^31 bytes of codes and 2^32 bytes of fp16: the first and the last rows, and sums over all of them."""
    M, K, N = 1_100_001, 2048, 16
    g = torch.Generator(device="cuda").manual_seed(6)
    x = torch.randn(M, K, generator=g, device="cuda", dtype=torch.float16)
    q = ops.quantize_fp8(x)
    pick = torch.tensor([0, 1, 1_048_575, 1_048_576, M - 17, M - 1], device="cuda")
    few = ops.quantize_fp8(x[pick].contiguous())
    assert torch.equal(q.q.view(torch.uint8)[pick], few.q.view(torch.uint8)) and torch.equal(q.scale[:, pick], few.scale[:, :6])
    assert torch.equal(q.dequantize()[pick], few.dequantize())
    w = ops.quantize_fp8_weight(torch.randn(N, K, generator=g, device="cuda"))
    assert torch.equal(ops.gemm_fp8(q, w)[pick], ops.gemm_fp8(few, w))
    dy = (0.02 * torch.randn(M, N, generator=g, device="cuda")).half()
    dw, db = ops.gemm_fp8_wgrad(dy, q)
    ref, mag, step = torch.zeros(N, K, device="cuda", dtype=torch.float64), torch.zeros(N, K, device="cuda", dtype=torch.float64), 110_000
    for a in range(0, M, step):
        d, v = dy[a:a + step].double(), ops.Fp8Tensor(q.q[a:a + step], torch.nn.functional.pad(q.scale[:, a:min(a + step, M)],
                                                      (0, -min(step, M - a) % 16)).contiguous(), K).dequantize(torch.float32).double()
        ref += d.t().contiguous() @ v
        mag += d.abs().t().contiguous() @ v.abs()
    # n independent terms of size s: the partial sums grow like sqrt(k) s, each addition is off by at most 2 u32 of its partial sum, with
    # either sign: together 2 u32 s sqrt(1 + 2 + ... + n) = 1.4 u32 n s, under 2 u32 of the sum of magnitudes; 16 times that is allowed
    assert ((dw.double() - ref).abs() <= 32 * U32 * mag).all()
    assert ((db.double() - dy.double().sum(0)).abs() <= 32 * U32 * dy.double().abs().sum(0)).all()
    h, z = ops.activation_fp8(x, ops.ACT_GELU)
    h2, z2 = ops.activation_fp8(x[pick].contiguous(), ops.ACT_GELU)
    assert torch.equal(h[pick], h2) and torch.equal(z.q.view(torch.uint8)[pick], z2.q.view(torch.uint8))
    del h, z
    one = torch.ones(K, device="cuda")
    y, st = ops.layernorm_train(x, one, one)
    y2, st2 = ops.layernorm_train(x[pick].contiguous(), one, one)
    assert torch.equal(y[pick], y2) and torch.equal(st[pick], st2)
    dx, dg, db = ops.layernorm_backward(y, x, st, one)
    assert torch.equal(dx[pick], ops.layernorm_backward(y2, x[pick].contiguous(), st2, one)[0])
    assert ((db.double() - y.sum(0, dtype=torch.float64)).abs() <= 32 * U32 * y.abs().sum(0, dtype=torch.float64)).all()
