"""Attention over the paged cache at its edges: infinities and NaN that tokens see, weights that are small beside the
largest, keys divided over CTAs under every mask, waits that give up."""
import ctypes as C

import numpy as np
import pytest
import torch

import ti_b200 as ti
from paged_ref import DT, Cache
from test_gpu_paged_ops import queries, run_attention, stream, within

pytestmark = pytest.mark.gpu
ODD = [float("nan"), float("inf"), -float("inf")]


def put(c, pool, s, j, h, dim, value):
    """value at position j of sequence s, kv head h (device pool)"""
    pool[int(c.table[c.rows[s], j // 16]), h, j % 16, dim] = value


def same_odd_values(got, want, ref, tol):
    """NaN and infinities exactly where `want` has them (0 elsewhere), the reference elsewhere"""
    got = got.cpu().double().numpy()
    fine = want == 0
    assert np.isfinite(got[fine]).all()
    assert (np.abs(got - ref)[fine] <= tol[fine]).all()
    np.testing.assert_array_equal(np.isnan(got[~fine]), np.isnan(want[~fine]))
    inf = np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])


# ------------------------------------------------------------------ infinities and NaN in V
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("heads, nkv", [(4, 2), (24, 2)])
@pytest.mark.parametrize("lens", [[61], [700, 40], [6000, 300]])  # the last: one sequence divided over CTAs
@pytest.mark.parametrize("many", [False, True])
def test_decode_keeps_the_infinities_it_sees(many, lens, heads, nkv, hd, dtype):
    c = Cache([(1, n) for n in lens], nkv, hd, dtype, seed=31)
    q = queries(c, heads)
    clean, ref, tol = run_attention(c, q, heads, "decode")
    within(clean, ref, tol)
    d = c.dev(decode=True)
    want = np.zeros((len(lens), heads, hd))
    for s, n in enumerate(lens):
        for i, j in enumerate(range(0, n, 7) if many else [n // 2, n // 2 + 1, n - 1]):
            h, dim, value = (i // 2) % nkv, (5 * j + i) % hd, ODD[i % 3]
            put(c, d["v"], s, j, h, dim, value)
            g = heads // nkv
            with np.errstate(invalid="ignore"):
                want[s, h * g:(h + 1) * g, dim] += value
    out, _, _ = run_attention(c, q, heads, "decode", d=d)
    same_odd_values(out, want, ref, tol)


@pytest.mark.parametrize("window", [0, 50])
def test_decode_ignores_the_infinities_it_does_not_see(window):
    # before the window, and behind the sequence's end (the pools' free slots hold NaN)
    c = Cache([(1, 333), (1, 60)], 2, 128, "f16", seed=32)
    q = queries(c, 8)
    clean, ref, tol = run_attention(c, q, 8, "decode", window=window)
    d = c.dev(decode=True)
    want = np.zeros((2, 8, 128))
    for s, n in enumerate([333, 60]):
        for i, j in enumerate([2, n - 55, n - 3]):
            put(c, d["v"], s, j, 0, 9 * i, float("inf"))
            if window == 0 or j >= n - window:
                want[s, :4, 9 * i] = float("inf")
    out, _, _ = run_attention(c, q, 8, "decode", window=window, d=d)
    same_odd_values(out, want, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("length", [90, 3000])  # 3000: divided over CTAs
def test_decode_infinity_counts_however_small_its_weight(length, dtype):
    # a key 400 below the others: its weight is e^-400, above zero, so its infinity is the result
    c = Cache([(1, length)], 1, 64, dtype, seed=33)
    c.K[0][:] = 0.0
    c.K[0][20:22] = -50.0
    d = c.dev(decode=True)
    for p in range(-(-length // 16)):
        m = min(16, length - p * 16)
        d["k"][int(c.table[c.rows[0], p]), :, :m] = c.K[0][p * 16:p * 16 + m].transpose(0, 1).cuda()
    q = torch.ones(1, 2, 64, dtype=DT[dtype])
    _, ref, tol = run_attention(c, q, 2, "decode", d=d)
    put(c, d["v"], 0, 20, 0, 3, float("inf"))
    put(c, d["v"], 0, 21, 0, 40, -float("inf"))
    put(c, d["v"], 0, 21, 0, 5, float("nan"))
    want = np.zeros((1, 2, 64))
    want[..., 3], want[..., 40], want[..., 5] = np.inf, -np.inf, np.nan
    out, _, _ = run_attention(c, q, 2, "decode", d=d)
    same_odd_values(out, want, ref, tol)
