"""The 8-bit training operators at the edges of their ranges: exponents far from 0 in the weight gradient, and what the entries refuse.
Plain evaluations in 64 bits and tolerances as in test_train8.py."""
import ctypes
import math

import numpy as np
import pytest
import torch

from editanything_amd import _lib as L
from editanything_amd import ops
from emu_util import epilogue, ptr
from test_train8 import (ACT_ABS, GEGLU, GELU, SILU, TINY16, U16, U32, UNIT, act64, decode, encode, force, gemm_case, pack_scales, quantize,
                         quantize_weight, rows, values)

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
    M, N, K = 4 * 2048 + 70, 8, 257 if kernel == 101 else 100
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
