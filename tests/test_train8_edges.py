"""The 8-bit training operators at the edges of their ranges: exponents far from 0 in the weight gradient, and what the entries refuse.
Plain evaluations in 64 bits and tolerances as in test_train8.py."""
import ctypes

import numpy as np
import pytest
import torch

from editanything_amd import _lib as L
from editanything_amd import ops
from emu_util import epilogue, ptr
from test_train8 import (ACT_ABS, GEGLU, GELU, KERNELS, SILU, TINY16, U16, U32, UNIT, act64, encode, force, gemm_case, pack_scales, quantize, rows,
                         values)

FLUSH = 2.0 ** -126                        # fp32's smallest normal number: what lies below may be flushed


# ------------------------------------------------------------------------------------------- weight gradient: any exponent
def wgrad(kb, q, e, dy, kernel, K, splits=0):
    M, N = dy.shape
    if kernel or splits:
        assert L.set_tuning(kb.lib, variant=kernel, splits=splits) == 0
    dw, db = kb.up(np.full((N + 1, K), 7, np.float32)), kb.up(np.full((N + 1,), 7, np.float32))
    nbytes = kb.lib.ea_gemm_fp8_wgrad_workspace_bytes(M, N, K)
    ws = kb.zeros((nbytes // 4,), np.float32) if nbytes else None
    assert kb.lib.ea_gemm_fp8_wgrad(ptr(dy), ptr(q), ptr(pack_scales(e)), ptr(dw), ptr(db), M, N, K, ptr(ws), nbytes, kb.stream) == 0
    dw, db = kb.down(dw), kb.down(db)
    assert (dw[N] == 7).all() and db[N] == 7
    return dw[:N].astype(np.float64), db[:N].astype(np.float64)


def check_wgrad(q, e, dy, K, dw, db):
    """x in the matrix unit's type is exact, so only the sums round: a share of the magnitudes, and nothing absolute."""
    M, d, x = dy.shape[0], dy.astype(np.float64), values(q, e, K)
    assert (np.abs(dw - d.T @ x) <= 2 * (M + 2) * U32 * (np.abs(d).T @ np.abs(x)) + FLUSH).all()
    assert (np.abs(db - d.sum(0)) <= 2 * (M + 2) * U32 * np.abs(d).sum(0)).all()


WG = [0, 101, 102, 103]


@pytest.mark.parametrize("kernel", WG)
@pytest.mark.parametrize("octaves", [-90, -60, -40, -30, -20, 9, 12, 30, 110])
def test_wgrad_of_small_and_large_inputs(kb, octaves, kernel):
    q, e = quantize(rows(31, 150, 300, np.float32, 2.0 ** octaves))
    dy = rows(32, 150, 24, np.float16, 0.05)
    check_wgrad(q, e, dy, 300, *wgrad(kb, q, e, dy, kernel, 300))


@pytest.mark.parametrize("kernel", WG)
def test_wgrad_keeps_zeros_and_small_values_beside_a_large_one(kb, kernel):
    """One value above fp16's range in a block: the block's zeros stay zero and its other values what their codes say."""
    x = np.zeros((9, 300), np.float32)
    x[0, :4] = 0, 200000, 448, 0                  # E = 9
    x[1, 130:133] = 400000, -1024, 0              # E = 10
    x[2, 299] = 3
    q, e = quantize(x)
    dy = np.ones((9, 8), np.float16)
    dw, db = wgrad(kb, q, e, dy, kernel, 300)
    ref = dy.astype(np.float64).T @ values(q, e, 300)
    assert e[0, 0] == 9 and e[1, 1] == 10 and np.array_equal(dw, ref) and (ref[:, 1] >= 196608).all() and (db == 9).all()


@pytest.mark.parametrize("kernel", WG)
@pytest.mark.parametrize("kind", ["spread", "tiny beside zeros", "one block column", "few bits apart"])
def test_wgrad_of_rows_of_very_different_sizes(kb, kind, kernel):
    """Rows whose exponents lie further apart than fp16 reaches: the large rows' gradients are 0 in half of the columns, where the small rows'
    sums stand alone."""
    M, K, N = 150, 300, 24
    g = np.random.default_rng(33)
    x = rows(34, M, K, np.float32)
    if kind == "spread":
        x = x * 2.0 ** g.integers(-35, 36, (M, 1))
    elif kind == "tiny beside zeros":
        x = x * 2.0 ** -60
        x[20:70] = 0
    elif kind == "one block column":
        x[:, 128:256] *= 2.0 ** g.integers(-50, 20, (M, 1))
    else:
        x = x * 2.0 ** g.integers(-10, 11, (M, 1))
    x = x.astype(np.float32)
    q, e = quantize(x)
    dy = rows(35, M, N, np.float16, 0.05)
    big = e.max(0) > np.median(e.max(0))
    dy[np.ix_(big, np.arange(N) % 2 == 1)] = 0
    check_wgrad(q, e, dy, K, *wgrad(kb, q, e, dy, kernel, K))


@pytest.mark.parametrize("kernel", WG)
def test_wgrad_not_finite_in_rows_of_very_different_sizes(kb, kernel):
    M, K, N = 150, 300, 264
    q, e = quantize((rows(36, M, K, np.float32) * 2.0 ** np.random.default_rng(37).integers(-40, 40, (M, 1))).astype(np.float32))
    dy = rows(38, M, N, np.float16, 0.05)
    q[9, 140] = 0x7F
    cols = [21, 77, 200]
    dy[[3, 40, 69], cols] = np.inf, np.nan, -np.inf
    dw, db = wgrad(kb, q, e, dy, kernel, K)
    want = np.ones((N, K), bool)
    want[:, 140] = want[cols] = False
    assert np.array_equal(np.isfinite(dw), want) and np.array_equal(np.isfinite(db), want[:, 0])


@pytest.mark.parametrize("kernel", WG[1:])
def test_wgrad_units_change_along_a_slice(kb, kernel):
    """One slice longer than the 2048 rows under one unit, the rows' size changing along it, up and down, further than one unit reaches."""
    M, N, K = (2 if (kb.name, kernel) == ("emu", 101) else 4) * 2048 + 70, 8, 257 if kernel == 101 else 100      # (minutes on the emulation)
    g = np.random.default_rng(39)
    nb = -(-K // 128)
    q = np.zeros((M, nb * 128), np.uint8)
    q[:, :K] = g.integers(0, 0x60, (M, K)) | g.integers(0, 2, (M, K)) << 7
    size = np.array([0, 40, 45, -39, -45, 3, 4, -12, 70])                # by 1024 rows
    e = np.repeat(size, 1024)[None, :M] + g.integers(-3, 4, (nb, M))
    dy = (0.05 * g.standard_normal((M, N))).astype(np.float16)
    dy[(e.max(0) > 0)[:, None] & (np.arange(N) % 2 == 1)] = 0
    dw, db = wgrad(kb, q, e, dy, kernel, K, splits=1)
    d, x = dy.astype(np.float64), values(q, e, K)
    # terms with random signs: partial sums of n terms of size s stay within 16 sqrt(n) s, each addition is off by 2 u32 of its partial sum with
    # either sign -- together far below 32 u32 of the sum of magnitudes (n s)
    assert (np.abs(dw - d.T @ x) <= 32 * U32 * (np.abs(d).T @ np.abs(x)) + FLUSH).all()
    assert (np.abs(db - d.sum(0)) <= 32 * U32 * np.abs(d).sum(0)).all()


# ---------------------------------------------------------------------------------------------- products with fp32 accuracy
@pytest.mark.parametrize("kernel", [0, 102, 103, 104])
@pytest.mark.parametrize("form", ["plain", "bias gelu fp32", "bias silu residual", "residual32 scale"])
@pytest.mark.parametrize("M,N,K", [(1, 1, 1), (16, 8, 130), (70, 100, 300), (130, 136, 640), (33, 7, 77)])
def test_gemm_fp8_exact(kb, M, N, K, form, kernel):
    """The bound of test_gemm_fp8 without the matrix unit's share: only fp32 roundings are left."""
    force(kb, kernel)
    aq, sa, wq, sw, ref, mag = gemm_case(M, N, K, 41)
    g = np.random.default_rng(42)
    f32out = "fp32" in form
    out = kb.up(np.full((M + 1, N), 7, np.float32 if f32out else np.float16))
    bias = g.standard_normal(N).astype(np.float32) if "bias" in form else None
    res = g.standard_normal((M, N)).astype(np.float16) if "residual" in form and "32" not in form else None
    res32 = g.standard_normal((M, N)).astype(np.float32) if "residual32" in form else None
    act = GELU if "gelu" in form else SILU if "silu" in form else 0
    scale = 0.5 if "scale" in form else 1.0
    e = epilogue(out, bias=bias, act=act, scale=scale, residual=res, residual32=res32)
    assert kb.lib.ea_gemm_fp8_exact(ptr(aq), ptr(sa), ptr(wq), ptr(sw), M, N, K, ctypes.byref(e), kb.stream) == 0
    v = ref + (0 if bias is None else bias.astype(np.float64))
    err = 2 * (K + 2) * U32 * mag + U32 * np.abs(v)
    if act:
        err = 1.13 * err + ACT_ABS + 4 * U32 * np.abs(v)           # (neither slope exceeds 1.13)
        v = act64(v, act)[0]
    v = scale * v + (0 if res is None else res.astype(np.float64)) + (0 if res32 is None else res32.astype(np.float64))
    got = kb.down(out)
    assert (got[M] == 7).all()
    assert (np.abs(got[:M] - v) <= scale * err + (2 * U32 if f32out else U16) * np.abs(v) + TINY16 + 4 * U32 * np.abs(v)).all()


@pytest.mark.parametrize("signs", ["random", "alternating"])
@pytest.mark.parametrize("kernel", [0, 102, 103, 104])
def test_gemm_fp8_exact_small_products_beside_a_large_one(kb, kernel, signs):
    """One product of 2^16 and seven of 2^-2 in each eight neighbours: the 8-bit instruction cuts the seven away, this one may not.  K runs over
    two chunks of scale bytes; a NaN code reaches its row only; the exponents lie far apart."""
    M, N, K = 20, 24, 8450
    nb = -(-K // 128)
    a, w = np.zeros((M, nb * 128)), np.zeros((N, nb * 128))
    a[:, :K], w[:, :K] = 0.5, 0.5
    a[:, 3:K:8], w[:, 3:K:8] = 256, 256
    g = np.random.default_rng(43)
    if signs == "random":
        a[:, :K] *= np.where(g.random((M, K)) < 0.5, 1, -1)
    else:
        a[:, 3:K:16] = -256                                    # the large ones cancel, the small ones add up
    ea, ew = np.zeros((nb, M), np.int64), np.zeros((nb, 1), np.int64)
    ea[1::2], ew[1::2] = 100, -100                             # the product's exponent is 0, its factors' are not
    aq, wq = encode(a), encode(w)
    aq[4, 200] = 0x7F
    out = kb.up(np.full((M + 1, N), 7, np.float32))
    force(kb, kernel)
    assert kb.lib.ea_gemm_fp8_exact(ptr(aq), ptr(pack_scales(ea)), ptr(wq), ptr((ew + 127).astype(np.uint8)), M, N, K, ctypes.byref(epilogue(out)),
                                    kb.stream) == 0
    got = kb.down(out)
    assert (got[M] == 7).all() and np.isnan(got[4]).all()
    keep = np.arange(M) != 4
    # A block's sum is a multiple of 2^-2 below 2^21: exact.  Behind a block the accumulator is below `top`; below 2^22 it is exact too, below 2^23 the
    # addition of a block rounds to multiples of 2^-1, off by 2^-2 at most, once for each of the 67 blocks
    top = np.abs(np.cumsum([a[:, b * 128:b * 128 + 128] @ w[:, b * 128:b * 128 + 128].T for b in range(nb)], 0)).max()
    assert top < 2 ** 23
    assert (np.abs(got[:M] - a @ w.T)[keep] <= (0 if top < 2 ** 22 else nb * 0.25)).all()
    if signs == "alternating":
        assert top < 2 ** 22 and (np.abs(a @ w.T) > 1800).all()


def test_gemm_fp8_exact_refuses_as_gemm_fp8(emu_lib):
    a = np.zeros((256, 256), np.float32)
    p = a.ctypes.data
    e = epilogue(a)
    f = lambda M=16, N=16, K=128, q=p: emu_lib.ea_gemm_fp8_exact(q, p, p, p, M, N, K, ctypes.byref(e), None)  # noqa: E731
    assert f(q=None) == -2 and f(q=p + 8) == -2 and f(M=0) == f(N=-1) == f(K=1 << 21) == f(M=(1 << 30) + 1) == -1 and f(N=512) == -2
    e.act = GEGLU
    assert f() == -3


@pytest.mark.gpu
def test_an_fp32_product_is_exact_unless_told_otherwise():
    g = torch.Generator(device="cuda").manual_seed(44)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    for M, N, K in ((616, 2560, 1024), (8192, 640, 640), (33, 24, 320), (8192, 1280, 320)):
        a, w = ops.quantize_fp8(r(M, K)), ops.quantize_fp8_weight(r(N, K) * K ** -0.5)
        x, y = a.dequantize(torch.float32).double(), w.dequantize(torch.float32).double().t().contiguous()
        ref, mag = x @ y, x.abs() @ y.abs()
        got = {k: ops.gemm_fp8(a, w, out_dtype=torch.float32, exact=k).double() for k in (None, True, False)}
        assert torch.equal(got[None], got[True])
        assert ((got[True] - ref).abs() <= 2 * (K + 2) * U32 * mag + 4 * U32 * ref.abs()).all()
        assert ((got[False] - ref).abs() <= (2 * (K + 2) * U32 + UNIT) * mag + 4 * U32 * ref.abs()).all()
        half = {k: ops.gemm_fp8(a, w, exact=k) for k in (None, True, False)}
        assert torch.equal(half[None], half[False]) and torch.equal(half[True], got[True].to(torch.float32).half())


# -------------------------------------------------------------------------------------------------------- activations, backward
@pytest.mark.parametrize("H", [128, 77])
def test_geglu_value_gradient_of_strongly_negative_gates(kb, H):
    """dvalue = dh gelu(gate): it vanishes with the gate's GELU, however large the gate is."""
    gates = -np.array([0.5, 3, 5.5, 5.7, 8, 30, 100, 1000, 8192, 28672, 57344])
    z = np.zeros((2 * len(gates), H), np.float32)
    z[0::2], z[1::2] = 3.0, gates[:, None]
    z[1::2, 1::2] *= -1                                        # and positive ones, where it is the gate
    q, e = quantize(z)
    M, v = len(gates), values(q, e, H)
    dh = np.full((M, H), 100, np.float16)
    dh[:, 2] = -100
    dz = kb.zeros((M, 2 * H), np.float16)
    assert kb.lib.ea_activation_fp8_bwd(ptr(dh), ptr(q), ptr(pack_scales(e)), GEGLU, ptr(dz), M, H, kb.stream) == 0
    with np.errstate(over="ignore"):
        ref = dh.astype(np.float64) * act64(v[1::2], GELU)[0]
        want = np.where(np.abs(ref) >= 65520, np.copysign(np.inf, ref), ref)
    got = kb.down(dz)[:, :H].astype(np.float64)
    inf = np.isinf(want)
    assert (got[inf] == want[inf]).all()
    # the GELU is off by ACT_ABS at most, wherever the gate lies
    got, ref = np.where(inf, 0, got), np.where(inf, 0, ref)
    assert (np.abs(got - ref) <= U16 * np.abs(ref) + TINY16 + ACT_ABS * 100 + 8 * U32 * np.abs(ref)).all()


@pytest.mark.parametrize("act", [SILU, GELU, GEGLU])
def test_slopes_of_the_largest_inputs(kb, act):
    """Inputs that only an Fp8Tensor of an fp32 tensor holds, up to what decodes to infinity: the slope is 0 or 1, a GEGLU's value gradient the
    gate or 0."""
    g = 2 if act == GEGLU else 1
    x = np.zeros((16, 128), np.float32)
    x[:, 0::2] = np.array([20, 100, 1e3, 7e4, 1e6, 3e10, 1e18, 1e19, 3e20, 1e30, 3e36, 1e37, 1e38, 2e38, 3e38, np.finfo(np.float32).max])[:, None]
    x[:, 1::2] = -x[:, 0::2]
    z = np.ones((16 * g, 128), np.float32)
    z[g - 1::g] = x
    q, e = quantize(z)
    dh = np.full((16, 128), 2, np.float16)
    dz = kb.zeros((16, g * 128), np.float16)
    assert kb.lib.ea_activation_fp8_bwd(ptr(dh), ptr(q), ptr(pack_scales(e)), act, ptr(dz), 16, 128, kb.stream) == 0
    got = kb.down(dz).astype(np.float64)
    want = np.where(x > 0, 2.0, 0.0)
    assert (np.abs(got[:, -128:] - want) <= U16 * want + ACT_ABS * 2 + TINY16).all()
    if g == 2:                             # the value's gradient: 2 gate or 0, infinite from 65520 on
        v = 2 * np.where(x > 0, values(q, e, 128)[1::2], 0.0)
        big = v >= 65520
        assert np.isposinf(got[:, :128][big]).all() and (np.abs(got[:, :128] - v)[~big] <= U16 * v[~big] + 2 * ACT_ABS + TINY16).all()


# ------------------------------------------------------------------------------------------------------------------ refusals
def test_more_than_a_launch_holds_is_refused(emu_lib):
    """2^32 threads along x are one too many; nothing is read or written before the refusal."""
    lib = emu_lib
    a = np.zeros((256, 256), np.float32)
    p, o = a.ctypes.data, a.ctypes.data + 65536
    for C, rows in ((8, 1 << 28), (384, 1 << 28), (385, 1 << 27), (768, 1 << 27), (769, 1 << 26), (4096, 1 << 26)):
        assert lib.ea_layernorm_train(p, 0, p, p, 1e-5, o, None, None, p, rows, C, None) == -1
        assert lib.ea_layernorm_train(p, 1, p, p, 1e-5, None, o, o, p, rows - 1, C, None) == -1
    for C, rows in ((8, 1 << 28), (512, (1 << 28) - 15), (513, 1 << 27), (1 << 20, 1 << 17)):
        assert lib.ea_quantize_fp8(p, 0, o, o, rows, C, None) == -1
        assert lib.ea_dequantize_fp8(p, p, 1, o, 0, rows, C, None) == -1
        assert lib.ea_activation_fp8(p, GELU, o, None, None, o, o, rows, C, None) == -1
        assert lib.ea_activation_fp8_bwd(p, p, p, SILU, o, rows, C, None) == -1
    assert lib.ea_quantize_fp8(p, 0, o, o, (1 << 62) + 5, 1 << 24, None) == -1
    e = epilogue(a)
    e.ldc = 1 << 22
    for fn in (lib.ea_gemm_fp8, lib.ea_gemm_fp8_exact):
        for kernel in KERNELS:
            assert L.set_tuning(lib, variant=kernel) == 0
            assert fn(p, p, p, p, 1 << 30, 1 << 22, 128, ctypes.byref(e), None) == -1
    assert L.set_tuning(lib, variant=101) == 0
    assert lib.ea_layernorm_bwd(p, p, 0, None, p, p, None, o, o, o, 1 << 28, 8, None, 0, None) == -1
    lib.ea_set_tuning(None)
    big = lib.ea_gemm_fp8_wgrad_workspace_bytes(1 << 20, 1 << 20, 1 << 20)
    assert lib.ea_gemm_fp8_wgrad(p, p, p, o, o, 1 << 20, 1 << 20, 1 << 20, p if big else None, big, None) == -1


def test_outputs_that_share_memory_with_inputs_are_refused(emu_lib):
    """Which thread reads an element before which writes it is no caller's business: the C entries refuse what they cannot get right, and take
    the in-place calls that they can."""
    lib = emu_lib
    m = np.zeros(1 << 20, np.uint8)
    at = lambda kib: m.ctypes.data + 1024 * kib  # noqa: E731
    # LayerNorm backward: up to 1024 rows the column sums read all of x and dy beside the writers of dx
    bwd = lambda dy=0, x=100, dx=200, res=None, st=300, ga=310, dg=320, db=330, kind=0, M=64: lib.ea_layernorm_bwd(  # noqa: E731
        at(dy), at(x), kind, at(500) if kind == 2 else None, at(st), at(ga), None if res is None else at(res), at(dx), at(dg), at(db), M, 64, at(400), 1 << 20,
        None)
    assert bwd() == bwd(res=200) == bwd(kind=1) == bwd(kind=2) == bwd(dx=8) == bwd(dx=108) == 0          # (64 rows of 64: 8 KiB)
    assert bwd(dx=0) == bwd(dx=7) == bwd(dx=100) == bwd(dx=99) == bwd(dx=200, res=201) == bwd(dg=101) == bwd(dg=330) == bwd(db=200) == -2
    assert bwd(dx=100, kind=1) == bwd(dx=200, res=207) == bwd(ga=200) == bwd(st=201) == bwd(kind=2, dx=500) == -2
    fwd = lambda x=0, y=100, q=None, st=300, f32=0, ga=310: lib.ea_layernorm_train(  # noqa: E731
        at(x), f32, at(ga), at(320), 1e-5, at(y) if q is None else None, None if q is None else at(q), at(200), at(st), 64, 64, None)
    assert fwd() == fwd(y=0) == fwd(q=100) == fwd(f32=1) == 0
    assert fwd(y=0, f32=1) == fwd(y=7) == fwd(q=0) == fwd(q=200) == fwd(st=0) == fwd(st=100) == fwd(ga=100) == -2
    act = lambda fn, z=0, h=100, zq=200, zs=300: lib.ea_activation_fp8(at(z), fn, at(h), None, None, at(zq), at(zs), 64, 64, None)  # noqa: E731
    assert act(GELU) == act(GELU, h=0) == act(GEGLU) == 0
    assert act(GEGLU, h=0) == act(GELU, h=1) == act(GELU, zq=0) == act(GELU, zs=100) == act(SILU, zs=200) == -2
    assert lib.ea_activation_fp8(at(0), SILU, None, at(0), at(300), at(200), at(310), 64, 64, None) == -2
    use = lambda fn, dh=0, dz=100, zq=200, zs=300: lib.ea_activation_fp8_bwd(at(dh), at(zq), at(zs), fn, at(dz), 64, 64, None)  # noqa: E731
    assert use(GELU) == use(SILU, dz=0) == use(GEGLU) == 0
    assert use(GEGLU, dz=0) == use(GELU, dz=1) == use(GELU, dz=200) == use(GELU, dz=300) == -2
    assert lib.ea_quantize_fp8(at(0), 0, at(4), at(300), 64, 64, None) == lib.ea_quantize_fp8(at(0), 0, at(100), at(100), 64, 64, None) == -2
    assert lib.ea_quantize_fp8_weight(at(0), 1, at(15), at(300), 64, 64, None) == lib.ea_quantize_fp8_weight(at(0), 0, at(8), at(0), 64, 64, None) == -2
    assert lib.ea_dequantize_fp8(at(0), at(300), 1, at(7), 0, 64, 64, None) == lib.ea_dequantize_fp8(at(0), at(300), 128, at(300), 1, 64, 64, None) == -2

    # the product: 64 x 64 fp16 outputs (8 KiB), a at 0, its scales at 20, w at 40, its scales at 60, bias at 80
    def mm(fn, out=100, res=None, res32=None, ldc=64, ldr=64, f32=0, more=0):
        e = L.Epilogue()
        e.bias, e.scale, e.out, e.ldc, e.out_f32, e.ldr = at(80), 1.0, at(out), ldc, f32, ldr
        if res is not None:
            e.residual = at(res) + more
        if res32 is not None:
            e.residual32 = at(res32)
        return fn(at(0), at(20), at(40), at(60), 64, 64, 64, ctypes.byref(e), None)
    for fn in (lib.ea_gemm_fp8, lib.ea_gemm_fp8_exact):
        assert mm(fn) == mm(fn, res=100) == mm(fn, res=108) == mm(fn, res=92) == mm(fn, f32=1, res32=100) == 0
        assert mm(fn, ldc=128, ldr=128, res=100, more=128) == 0                 # two halves of one buffer's rows
        assert mm(fn, ldc=128, ldr=128, res=100, more=126) == mm(fn, ldc=128, ldr=128, res=100, more=130) == mm(fn, ldc=128, res=100) == -2
        assert mm(fn, res=101) == mm(fn, res=99) == mm(fn, res32=100) == mm(fn, f32=1, res=100) == mm(fn, res32=90) == -2
        assert mm(fn, out=4) == mm(fn, out=13) == mm(fn, out=40) == mm(fn, out=53) == mm(fn, out=60) == mm(fn, out=80) == -2
    wg = lambda dy=0, x=100, dw=200, db=300, ws=400, M=64: lib.ea_gemm_fp8_wgrad(at(dy), at(x), at(700), at(dw), at(db), M, 64, 64, at(ws), 1 << 20,  # noqa: E731
                                                                                None)
    assert wg() == 0
    assert wg(dw=0) == wg(dw=107) == wg(dw=700) == wg(db=200) == wg(db=100) == -2
    assert lib.ea_gemm_fp8_wgrad_workspace_bytes(700, 64, 64) > 0 and wg(M=700) == 0
    assert wg(M=700, ws=200) == wg(M=700, ws=80) == wg(M=700, ws=290) == -2


def test_gemm_fp8_refuses_an_output_that_is_an_operand():
    t = ops.Fp8Tensor(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 16, dtype=torch.uint8), 8)
    w = ops.Fp8Tensor(torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 1, dtype=torch.uint8), 8)
    b = torch.zeros(32)
    for out, bias in ((t.q.view(torch.float16)[0, :16].view(4, 4), None), (w.q.view(torch.float32)[3, 16:].view(4, 4), None), (b[:16].view(4, 4), b[12:16])):
        with pytest.raises(ValueError, match="apart"):
            ops.gemm_fp8(t, w, out=out, bias=bias)
    with pytest.raises(RuntimeError, match="MI355X"):               # accepted: on the CPU only the missing device stops it
        ops.gemm_fp8(t, w, out=b[:16].view(4, 4), bias=b[16:20])


def test_an_operand_that_requires_grad_is_refused_where_a_graph_is_recorded():
    x, one, zero = torch.zeros(4, 8, dtype=torch.float16), torch.ones(8), torch.zeros(4, 2)
    q, sc = torch.zeros(4, 128).to(torch.float8_e4m3fn), torch.zeros(1, 16, dtype=torch.uint8)
    t, w = ops.Fp8Tensor(q, sc, 8), ops.Fp8Tensor(q, torch.zeros(1, 1, dtype=torch.uint8), 8)
    gx, gone = x.clone().requires_grad_(), one.clone().requires_grad_()
    calls = [lambda: ops.quantize_fp8(gx), lambda: ops.quantize_fp8_weight(gx), lambda: ops.layernorm_train(gx, one, one),
             lambda: ops.layernorm_train(x, gone, one), lambda: ops.layernorm_train(x, one, gone), lambda: ops.layernorm_backward(gx, x, zero, one),
             lambda: ops.layernorm_backward(x, x, zero, gone), lambda: ops.layernorm_backward(x, x, zero, one, residual=gx),
             lambda: ops.activation_fp8(gx, ops.ACT_GELU), lambda: ops.activation_fp8_backward(gx, t, ops.ACT_GELU),
             lambda: ops.gemm_fp8(t, w, bias=torch.zeros(4, requires_grad=True)), lambda: ops.gemm_fp8(t, w, residual=gx[:, :4].contiguous()),
             lambda: ops.gemm_fp8(t, w, out=torch.zeros(4, 4, requires_grad=True)), lambda: ops.gemm_fp8_wgrad(gx, t)]
    for f in calls:
        with pytest.raises(RuntimeError, match="autograd"):
            f()
        with torch.no_grad(), pytest.raises(RuntimeError, match="MI355X"):      # accepted: on the CPU only the missing device stops it
            f()


@pytest.mark.gpu
def test_training_operators_inside_an_autograd_function():
    """A LayerNorm and a Linear in 8 bits as an autograd.Function's forward and backward pass; a written `out` is noticed by a graph that saved it."""
    g = torch.Generator(device="cuda").manual_seed(45)
    r = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731

    class Block(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, gamma, beta, w, b):
            n, stats = ops.layernorm_train(x, gamma, beta, fp8=True)
            ctx.save_for_backward(x, gamma, stats, w)
            ctx.n = n
            return ops.gemm_fp8(n, ops.quantize_fp8_weight(w), bias=b)

        @staticmethod
        def backward(ctx, dy):
            x, gamma, stats, w = ctx.saved_tensors
            dw, db = ops.gemm_fp8_wgrad(dy, ctx.n)
            dn = ops.gemm_fp8(ops.quantize_fp8(dy), ops.quantize_fp8_weight(w.t().contiguous()))
            return ops.layernorm_backward(dn, x, stats, gamma) + (dw, db)
    p = [r(77, 320).half(), 1 + 0.2 * r(320), 0.1 * r(320), r(640, 320) * 320 ** -0.5, 0.1 * r(640)]
    leaves = [t.clone().requires_grad_() for t in p]
    dy = (0.02 * r(77, 640)).half()
    got = torch.autograd.grad(Block.apply(*leaves), leaves, dy)

    class Ctx:
        def save_for_backward(self, *t):
            self.saved_tensors = t
    with torch.no_grad():
        ctx = Ctx()
        Block.forward(ctx, *p)
        ref = Block.backward(ctx, dy)
    assert all(torch.equal(a, b) for a, b in zip(got, ref))
    # ... and they are gradients: of the function in fp32, to what 8-bit operands give (each within 2^-4 of its value, signs random)
    m = [t.clone().float().requires_grad_() for t in p]
    out = torch.nn.functional.linear(torch.nn.functional.layer_norm(m[0], (320,), m[1], m[2]), m[3], m[4])
    for a, b in zip(got, torch.autograd.grad(out, m, dy.float())):
        assert (a.float() - b).norm() <= 2.0 ** -4 * b.norm()
    a, w = ops.quantize_fp8(p[0]), ops.quantize_fp8_weight(p[3])
    y = torch.zeros(77, 640, device="cuda", dtype=torch.float16)
    z = torch.ones(77, 640, device="cuda", dtype=torch.float16, requires_grad=True)
    prod = z * y
    ops.gemm_fp8(a, w, out=y)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        prod.sum().backward()
    with torch.inference_mode():
        ops.gemm_fp8(a, w, out=torch.zeros(77, 640, device="cuda", dtype=torch.float16))


# ------------------------------------------------------------------------------------------------------------- launch rules
def test_launch_rules_follow_the_measurements(emu_lib):
    """One launch or two of LayerNorm's backward pass, slices of the weight gradient: read off the workspaces."""
    ln = emu_lib.ea_layernorm_bwd_workspace_bytes
    for C in (8, 320, 1280, 4096):
        assert ln(1024, C) == 0 < ln(1025, C)
    for C in (77, 777, 3001):
        assert ln(768, C) == 0 < ln(769, C)                    # (1024 x 777: 13.6 us in one launch, 10.8 in two)
    slices = lambda M, N, K: max(1, emu_lib.ea_gemm_fp8_wgrad_workspace_bytes(M, N, K) // (4 * ((N * K + N + 3) // 4 * 4)))  # noqa: E731
    assert slices(616, 1280, 1024) == 1 and slices(16384, 1280, 5120) == 5       # the DMA kernels', as before
    assert slices(616, 1281, 1024) > 1 and slices(16384, 1281, 1280) > 6         # the any-N kernel's steps take three times as long


def test_pinned_slices_that_would_leave_one_empty_are_not_taken(emu_lib):
    M, N, K = 600, 24, 100                                     # ten steps: 6, 7, 8 and 9 slices would leave some empty
    q, e = quantize(rows(46, M, K, np.float32))
    dy = rows(47, M, N, np.float16, 0.05)
    d, x = dy.astype(np.float64), values(q, e, K)
    for splits in (1, 2, 3, 6, 9, 10, 11, 65, -1):
        assert L.set_tuning(emu_lib, splits=splits) == 0
        nbytes = emu_lib.ea_gemm_fp8_wgrad_workspace_bytes(M, N, K)
        if splits in (1, 2, 10):
            assert nbytes == (0 if splits == 1 else 4 * splits * (N * K + N))
        dw, db, ws = np.zeros((N, K), np.float32), np.zeros(N, np.float32), np.zeros(max(nbytes // 4, 4), np.float32)
        st = emu_lib.ea_gemm_fp8_wgrad(ptr(dy), ptr(q), ptr(pack_scales(e)), ptr(dw), ptr(db), M, N, K, ptr(ws) if nbytes else None, nbytes, None)
        emu_lib.ea_set_tuning(None)
        assert st == 0 and (np.abs(dw - d.T @ x) <= 2 * (M + 2) * U32 * (np.abs(d).T @ np.abs(x)) + FLUSH).all()
        assert (np.abs(db - d.sum(0)) <= 2 * (M + 2) * U32 * np.abs(d).sum(0)).all()
