"""Attention over the paged cache at its edges: infinities and NaN that tokens see, weights that are small beside the
largest, keys divided over CTAs under every mask, waits that give up."""
import ctypes as C
import os
import subprocess
import sys
import threading

import numpy as np
import pytest
import torch

import ti_b200 as ti
from paged_ref import DT, FLOOR, Cache, attend
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


def forms(c, heads, cap=0.0, bias=False, window=0, prefix=False, docs=0, scale=0.0):
    """arguments of `attend` for masks that differ from sequence to sequence and token to token"""
    slopes = (2.0 ** (-6.0 * (np.arange(heads) + 1) / heads)).astype(np.float32) if bias else None
    pre = np.array([(37 * (s + 3)) % (c.max_len + 9) for s in range(len(c.seqs))], np.int32) if prefix else None
    doc = None
    if docs:
        doc = np.zeros(c.tokens, np.int32)
        for s, (new, n) in enumerate(c.seqs):
            i = np.arange(n - new, n)
            doc[c.starts[s]:c.starts[s] + new] = i - i % docs
    return dict(cap=cap, slopes=slopes, window=window, prefix=pre, doc=doc, scale=scale)


def launch(c, d, q, heads, entry, form, out=None):
    dev = {k: torch.from_numpy(form[k]).cuda() for k in ("slopes", "prefix", "doc") if form[k] is not None}
    at = {k: v.data_ptr() for k, v in dev.items()}
    f = ti.AttnForm(scale=form["scale"], softcap=form["cap"], slopes=at.get("slopes"), sliding_window=form["window"],
                    prefix=at.get("prefix"), doc_start=at.get("doc"))
    dq = q.cuda()
    if out is None:
        out = torch.full((c.tokens, heads, c.hd), 3.0, dtype=DT[c.dtype], device="cuda")
    ti.check(getattr(ti.lib(), f"ti_op_paged_{entry}")(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(f), dq.data_ptr(),
                                                       heads * c.hd, heads, out.data_ptr(), heads * c.hd, stream()))
    torch.cuda.synchronize()
    return out


def sees(c, s, j, form):
    """which new tokens of sequence s see position j"""
    new, n = c.seqs[s]
    i = np.arange(n - new, n)
    ok = i >= j
    if form["prefix"] is not None:
        ok = ok | (j < form["prefix"][s])
    if form["window"]:
        ok = ok & (j > i - form["window"])
    if form["doc"] is not None:
        ok = ok & (j >= form["doc"][c.starts[s]:c.starts[s] + new])
    return ok


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


FORMS = {
    "plain": {},
    "cap": dict(cap=30.0),
    "bias": dict(bias=True),
    "window": dict(window=300),
    "prefix": dict(prefix=True),
    "docs": dict(docs=190),
    "all": dict(cap=8.0, bias=True, window=700, prefix=True, docs=411, scale=0.2),
}


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("hd, dtype", [(64, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("max_len", [0, 1 << 20])  # the second: keys divided over CTAs
def test_prefill_settles_the_odd_values_of_every_mask(max_len, hd, dtype, form):
    # rows that share tiles with an odd value and do not see it are computed again, the others take it, under every mask
    heads, nkv = 4, 1
    c = Cache([(500, 700), (3, 400), (130, 130)], nkv, hd, dtype, seed=34)
    c.max_len = max_len or c.max_len
    f = forms(c, heads, **FORMS[form])
    if f["prefix"] is not None:
        f["prefix"] = np.array([390, 399, 77], np.int32)
    q = queries(c, heads)
    ref, tol = attend(c, q, heads, **f)
    d = c.dev()
    clean = launch(c, d, q, heads, "prefill", f)
    within(clean, ref, tol)
    want = np.zeros((c.tokens, heads, hd))
    for s, n in enumerate([700, 400, 130]):
        for i, j in enumerate([0, 1, 2, 60, 61, 129, 128, 397, 398, 399, 400, 512, 600, 699]):
            if j < n and (s, i) != (0, 0):
                dim, value = (11 * j + 29 * i) % hd, ODD[i % 3]
                put(c, d["v"], s, j, 0, dim, value)
                with np.errstate(invalid="ignore"):
                    want[c.starts[s]:c.starts[s] + c.seqs[s][0], :, dim][sees(c, s, j, f)] += value
    same_odd_values(launch(c, d, q, heads, "prefill", f), want, ref, tol)


@pytest.mark.parametrize("dtype, hd", [("bf16", 64), ("f16", 128)])
def test_prefill_infinity_counts_however_small_its_weight(dtype, hd):
    c = Cache([(40, 200)], 1, hd, dtype, seed=35)
    c.K[0][:] = 0.0
    c.K[0][20:22] = -50.0
    d = c.dev()
    for p in range(13):
        m = min(16, 200 - p * 16)
        d["k"][int(c.table[c.rows[0], p]), :, :m] = c.K[0][p * 16:p * 16 + m].transpose(0, 1).cuda()
    q = torch.ones(40, 2, hd, dtype=DT[dtype])
    f = forms(c, 2)
    ref, tol = attend(c, q, 2, **f)
    put(c, d["v"], 0, 20, 0, 3, float("inf"))
    put(c, d["v"], 0, 21, 0, 40, -float("inf"))
    want = np.zeros((40, 2, hd))
    want[..., 3], want[..., 40] = np.inf, -np.inf
    same_odd_values(launch(c, d, q, 2, "prefill", f), want, ref, tol)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("where", ["first", "middle", "everywhere"])
def test_prefill_with_odd_values_takes_a_few_times_its_time(where, hd):
    # (what every row sees is settled by one reading of V; the rows of one tile before the middle are computed again)
    n, heads, nkv = 2048, 16, 4
    c = Cache([(n, n)], nkv, hd, "bf16", seed=36)
    d, f, q = c.dev(), forms(c, heads), queries(c, heads).cuda()
    out = torch.empty(n, heads, hd, dtype=torch.bfloat16, device="cuda")

    def fastest():
        fm, best = ti.AttnForm(), 1e9
        for _ in range(6):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            ti.check(ti.lib().ti_op_paged_prefill(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(fm), q.data_ptr(),
                                                  heads * hd, heads, out.data_ptr(), heads * hd, stream()))
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        return best

    clean = launch(c, d, q, heads, "prefill", f)
    base = fastest()
    for j in {"first": [0], "middle": [n // 2 + 13], "everywhere": range(n)}[where]:
        for h in range(nkv):
            put(c, d["v"], 0, j, h, 7, float("nan"))
    took = fastest()
    torch.cuda.synchronize()
    got, first = out.float(), {"first": 0, "middle": n // 2 + 13, "everywhere": 0}[where]
    assert got[first:, :, 7].isnan().all() and not got[:first, :, 7].isnan().any()
    got[:, :, 7], rest = 0, clean.float()
    rest[:, :, 7] = 0
    assert torch.equal(got, rest)
    assert took < 8 * base, f"{took:.3f} ms against {base:.3f}"


@pytest.mark.parametrize("hd, dtype", [(64, "bf16"), (128, "f16"), (256, "bf16")])
def test_prefill_join_keeps_the_odd_values_of_a_share_without_weight(hd, dtype):
    # keys divided over CTAs, and a distance bias that leaves the first share no weight in fp32: its NaN still counts
    heads = 2
    c = Cache([(20, 1500)], 1, hd, dtype, seed=37)
    f = forms(c, heads)
    f["slopes"] = np.array([0.5, 0.25], np.float32)
    q = queries(c, heads)
    ref, tol = attend(c, q, heads, **f)
    d = c.dev()
    within(launch(c, d, q, heads, "prefill", f), ref, tol)
    put(c, d["v"], 0, 3, 0, 17, float("nan"))
    want = np.zeros((20, heads, hd))
    want[..., 17] = np.nan
    same_odd_values(launch(c, d, q, heads, "prefill", f), want, ref, tol)


# ------------------------------------------------------------------ weights small beside the largest
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("gap", [10.0, 17.5, 19.0])  # weights of e^-10, 2^-25.2 and 2^-27.4 of the largest
@pytest.mark.parametrize("entry, new, hd, max_len", [("decode", 1, 64, 0), ("decode", 1, 128, 1), ("prefill", 3, 64, 0),
                                                     ("prefill", 3, 128, 1), ("prefill", 3, 256, 1)])
def test_many_small_weights_beside_a_large_one(entry, new, hd, max_len, gap, dtype):
    # one key takes nearly all the weight and its value is zero: the result is what the other 20,000 have together
    # (decode with max_len 1 runs in one CTA, so that warps meet many keys after the large one)
    n = 20000
    c = Cache([(new, n)], 1, hd, dtype, seed=38)
    c.max_len = max_len or c.max_len
    c.K[0][:] = 0.0
    c.K[0][40] = gap / hd ** 0.5  # q of ones: a score of hd k / sqrt(hd)
    c.V[0] = c.V[0].abs() + 0.5
    c.V[0][40] = 0.0
    at = c.table[c.rows[0]].long()
    pad = 16 * len(at) - n
    for pool, rows in ((c.k, c.K[0]), (c.v, c.V[0])):
        rows = torch.cat([rows, torch.zeros(pad, 1, hd, dtype=rows.dtype)])
        pool[at] = rows.view(-1, 16, 1, hd).transpose(1, 2)
    q = torch.ones(new, 2, hd, dtype=DT[dtype])
    f = forms(c, 2)
    ref, tol = attend(c, q, 2, **f)
    # attend allows each key half a smallest step of the type beside a largest p of 1; here it is of 2^15 p (decode: two
    # terms) or of 2^11 p at least (prefill)
    values = c.V[0][:, 0].double().abs().sum(0).numpy()
    tol = tol - FLOOR[dtype] * (1 + values) + FLOOR[dtype] * (1 + values * 2.0 ** (-15 if entry == "decode" else -11))
    assert (tol < 0.02 * ref).all() or dtype == "bf16"
    within(launch(c, c.dev(decode=entry == "decode"), q, 2, entry, f), ref, tol)


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("small", [1e-3, 1e-7, 1e-10])
@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_small_values_under_scores_at_the_low_end_of_a_cap(entry, small, hd):
    c = Cache([(1, 200)] if entry == "decode" else [(30, 200)], 1, hd, "bf16", seed=42)
    c.K[0] = torch.full_like(c.K[0], -12)
    c.V[0] = c.V[0] * small
    for p in range(13):
        m, page = min(16, 200 - p * 16), int(c.table[c.rows[0], p])
        c.k[page, :, :m] = c.K[0][p * 16:p * 16 + m].transpose(0, 1)
        c.v[page, :, :m] = c.V[0][p * 16:p * 16 + m].transpose(0, 1)
    q = torch.ones(c.tokens, 2, hd, dtype=torch.bfloat16)
    for cap in (20.0, 30.0, 41.0, 42.0, 46.0, 50.0, 51.0, 55.0):
        f = forms(c, 2, cap=cap)
        ref, tol = attend(c, q, 2, **f)
        within(launch(c, c.dev(decode=entry == "decode"), q, 2, entry, f), ref, tol, f"cap {cap}")


@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("cap", [65.0, 300.0, 2500.0, 10000.0])
@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_scores_far_below_a_wide_cap_keep_their_bits(entry, cap, bias, hd):
    # in tiles that rows see in part as in the others: tanh(u) is u to 2.9e-6 there, not cap - 2 cap / (e^2u + 1), which
    # is off by cap 2^-21 however small u is (a scale of 1 and a cap of 10,000: 0.005)
    heads = 2
    c = Cache([(1, 300)] if entry == "decode" else [(150, 300)], 1, hd, "f16", seed=43, std=3.0 / hd ** 0.5)
    q = queries(c, heads)
    f = forms(c, heads, cap=cap, bias=bias, scale=1.0)
    ref, _ = attend(c, q, heads, **f)
    out = launch(c, c.dev(decode=entry == "decode"), q, heads, entry, f).cpu().double().numpy()
    i = np.arange(300 - c.seqs[0][0], 300)[:, None]
    j = np.arange(300)[None]
    K, V, u = c.K[0][:, 0].double().numpy(), c.V[0][:, 0].double().numpy(), 2.0 ** -11
    for h in range(heads):
        qh = q[:, h].double().numpy()
        z = cap * np.tanh(qh @ K.T / cap)
        # fp32 products over hd terms; the polynomial, 2^-18 of the score, and its roundings; the exponential, 2^-16
        dz = (hd + 8) * 2.0 ** -24 * (np.abs(qh) @ np.abs(K).T) + np.abs(z) * (2.0 ** -18 + 2.0 ** -22) + 2.0 ** -16
        if bias:
            far = f["slopes"][h] * np.abs(i - j)
            z = z - far
            dz = dz + far * 2.0 ** -22
        z = np.where(j <= i, z, -np.inf)
        w = np.exp(z - z.max(-1, keepdims=True))
        w /= w.sum(-1, keepdims=True)
        # a score off by dz scales its p by 1 + dz; the p that a row has besides are off by their own
        off = w * np.where(j <= i, dz, 0)
        tol = u * np.abs(ref[:, h]) * 1.01 + (u * 1.01) * (w @ np.abs(V)) + 1.01 * (off @ np.abs(V) + off.sum(-1, keepdims=True) * np.abs(ref[:, h]))
        tol = tol + 2.0 ** -24
        assert (np.abs(out[:, h] - ref[:, h]) <= tol).all(), (np.abs(out[:, h] - ref[:, h]) / tol).max()


# ------------------------------------------------------------------ keys divided over CTAs
LONG = {
    "plain": {},
    "cap": dict(cap=25.0),
    "bias": dict(bias=True),
    "window": dict(window=1700),
    "prefix": dict(prefix=True),
    "docs": dict(docs=1300),
    "all": dict(cap=6.0, bias=True, window=2100, prefix=True, docs=2600, scale=0.2),
}


@pytest.mark.parametrize("form", LONG)
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("hd", [64, 128, 256])
def test_prefill_with_divided_keys_under_every_mask(hd, dtype, form):
    # up to a dozen shares; sequences with fewer key tiles than shares, one of none, rows whose range misses shares
    heads, nkv = 6, 2
    c = Cache([(37, 2900), (5, 1100), (0, 64), (3, 140), (1, 1)], nkv, hd, dtype, seed=45, pad_tokens=2, spare_rows=1)
    c.max_len = 1 << 20
    f, q = forms(c, heads, **LONG[form]), queries(c, heads)
    ref, tol = attend(c, q, heads, **f)
    out = launch(c, c.dev(), q, heads, "prefill", f)
    real = int(c.starts[-1])
    within(out[:real], ref[:real], tol[:real])
    assert (out[real:] == 3.0).all()


# ------------------------------------------------------------------ waits that give up
@pytest.mark.parametrize("hd, dtype", [(64, "bf16"), (128, "f16"), (256, "bf16")])
@pytest.mark.parametrize("max_len", [0, 1 << 20])
@pytest.mark.parametrize("step", [0, 2, 3])
def test_prefill_rows_are_nan_where_a_wait_gives_up(step, max_len, hd, dtype):
    # sequences of one key tile, of two and three, and of many
    heads, nkv = 4, 1
    seqs = [(30, 50), (20, 150), (700, 1500), (1, 1), (0, 9)]
    c = Cache(seqs, nkv, hd, dtype, seed=39, pad_tokens=2)
    c.max_len = max_len or c.max_len
    d, f, q = c.dev(), forms(c, heads), queries(c, heads)
    ref, tol = attend(c, q, heads, **f)
    clean = launch(c, d, q, heads, "prefill", f)
    real = int(c.starts[-1])
    within(clean[:real], ref[:real], tol[:real])
    try:
        ti.check(ti.lib().ti_selftest_paged_stop(step))
        out = launch(c, d, q, heads, "prefill", f)
    finally:
        ti.check(ti.lib().ti_selftest_paged_stop(-1))
    lost = out[:real].isnan().any(-1)
    assert torch.equal(out[:real].isnan().all(-1), lost)         # whole rows
    assert torch.equal(out[:real][~lost], clean[:real][~lost])    # and the others as ever
    s0, s1, s2 = (int(x) for x in c.starts[1:4])
    assert lost.all() if step == 0 else not lost[:s0].any()
    assert lost[s1:s2].any() or max_len  # (divided over CTAs, two key tiles may be all that a block has)
    assert (out[real:] == 3.0).all()
    assert torch.equal(launch(c, d, q, heads, "prefill", f), clean)


@pytest.mark.parametrize("hd, dtype", [(64, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("heads, lens, step", [(4, [900], 0), (4, [5000, 40, 700], 0), (12, [5000, 40, 700], 1), (4, [60000], 5)])
def test_decode_rows_are_nan_where_a_wait_gives_up(heads, lens, step, hd, dtype):
    c = Cache([(1, n) for n in lens], 1, hd, dtype, seed=40)
    d, f, q = c.dev(decode=True), forms(c, heads), queries(c, heads)
    ref, tol = attend(c, q, heads, **f)
    clean = launch(c, d, q, heads, "decode", f)
    within(clean, ref, tol)
    try:
        ti.check(ti.lib().ti_selftest_paged_stop(step))
        out = launch(c, d, q, heads, "decode", f)
    finally:
        ti.check(ti.lib().ti_selftest_paged_stop(-1))
    lost = out.isnan().any(-1)
    assert torch.equal(out.isnan().all(-1), lost) and torch.equal(out[~lost], clean[~lost])
    assert lost[0].all()
    assert torch.equal(launch(c, d, q, heads, "decode", f), clean)


@pytest.mark.parametrize("hd, dtype, tokens", [(256, "bf16", 128), (128, "f16", 256), (64, "bf16", 512)])
@pytest.mark.parametrize("step", [8, 9, 16])
def test_decode_blocks_of_many_sequences_give_up_for_good(step, hd, dtype, tokens):
    # sequences of eight steps each, several a block: later ones meet slots whose phase looks like one that has come
    heads, n = 2, 1200
    c = Cache([(1, tokens)] * n, 1, hd, dtype, seed=48)
    d, f, q = c.dev(decode=True), forms(c, heads), queries(c, heads)
    clean = launch(c, d, q, heads, "decode", f)
    assert clean.isfinite().all()
    try:
        ti.check(ti.lib().ti_selftest_paged_stop(step))
        out = launch(c, d, q, heads, "decode", f)
    finally:
        ti.check(ti.lib().ti_selftest_paged_stop(-1))
    lost = out.isnan().all(-1)
    assert lost.any() and not lost.all() and torch.equal(out[~lost], clean[~lost])
    assert torch.equal(launch(c, d, q, heads, "decode", f), clean)


# ------------------------------------------------------------------ pages that do not exist
@pytest.mark.parametrize("form", ["plain", "cap", "bias", "all"])
@pytest.mark.parametrize("hd, dtype", [(64, "f16"), (128, "bf16"), (256, "f16")])
@pytest.mark.parametrize("entry, max_len", [("decode", 0), ("prefill", 0), ("prefill", 1 << 20)])
def test_pages_that_do_not_exist_are_zeros_that_take_weight(entry, max_len, hd, dtype, form):
    # with every real score far below zero the zeros take most of the weight
    heads = 4
    seqs = [(1, 600), (1, 33)] if entry == "decode" else [(150, 600), (33, 33)]
    c = Cache(seqs, 1, hd, dtype, seed=41)
    c.max_len = max_len or c.max_len
    for s, (_, n) in enumerate(seqs):
        c.K[s] = -c.K[s].abs()
        for p in range(-(-n // 16)):
            m = min(16, n - p * 16)
            c.k[int(c.table[c.rows[s], p]), :, :m] = c.K[s][p * 16:p * 16 + m].transpose(0, 1)
    for s, p, bad in ((0, 0, -1), (0, 9, c.n_pages), (0, 37, 2**31 - 1), (1, 1, -2**31)):
        c.table[c.rows[s], p] = bad
        c.K[s][p * 16:p * 16 + 16] = 0
        c.V[s][p * 16:p * 16 + 16] = 0
    q, f = queries(c, heads).abs(), forms(c, heads, **FORMS[form])
    ref, tol = attend(c, q, heads, **f)
    within(launch(c, c.dev(decode=entry == "decode"), q, heads, entry, f), ref, tol)


# ------------------------------------------------------------------ calls at once
def test_two_host_threads_on_streams_of_their_own():
    # divided and joined calls, with scratch, one of them settling odd values: every result as when made alone
    heads = 4
    jobs = []
    for seed, (entry, seqs) in enumerate([("decode", [(1, 5000), (1, 70)]), ("prefill", [(40, 3000), (130, 130)])]):
        c = Cache(seqs, 1, 128, "bf16", seed=50 + seed)
        d, f, q = c.dev(decode=entry == "decode"), forms(c, heads, cap=20.0), queries(c, heads).cuda()
        put(c, d["v"], 0, 60, 0, 9, float("inf"))
        put(c, d["v"], 1, 65, 0, 11, float("nan"))
        fm = ti.AttnForm(softcap=20.0)
        jobs.append((c, d, f, q, entry, fm, launch(c, d, q, heads, entry, f).view(torch.int16).clone()))
    failed = []

    def work(c, d, f, q, entry, fm, want):
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            outs = [torch.zeros(c.tokens, heads, 128, dtype=torch.bfloat16, device="cuda") for _ in range(30)]
            for out in outs:
                st = getattr(ti.lib(), f"ti_op_paged_{entry}")(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(fm), q.data_ptr(),
                                                               heads * 128, heads, out.data_ptr(), heads * 128, s.cuda_stream)
                if st != 0:
                    failed.append((entry, st))
        s.synchronize()
        failed.extend(entry for out in outs if not torch.equal(out.view(torch.int16), want))

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=job) for job in jobs for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not failed


# ------------------------------------------------------------------ large pools
def test_pages_past_two_to_the_31_elements():
    # pools of 2.3e9 elements each, the sequences' pages at their end
    heads, nkv, hd, n_pages = 8, 8, 256, 70000
    dec, pre = Cache([(1, 500), (1, 20)], nkv, hd, "bf16", seed=47), Cache([(90, 500), (20, 20)], nkv, hd, "bf16", seed=47)
    pools = {w: torch.empty(n_pages, nkv, 16, hd, dtype=torch.bfloat16, device="cuda") for w in "kv"}
    shift = n_pages - dec.n_pages
    for entry, c in (("decode", dec), ("prefill", pre)):
        f, q = forms(c, heads), queries(c, heads)
        ref, tol = attend(c, q, heads, **f)
        c.table = torch.where(c.table >= 0, c.table + shift, c.table)
        d = c.dev(decode=entry == "decode")
        for w in "kv":
            pools[w][shift:] = d[w]
        d["k"], d["v"] = pools["k"], pools["v"]
        d["kv"].k_pages, d["kv"].v_pages, d["kv"].n_pages = pools["k"].data_ptr(), pools["v"].data_ptr(), n_pages
        out = launch(c, d, q, heads, entry, f)
        within(out, ref, tol)
        put(c, d["v"], 0, 450, 3, 200, float("inf"))
        want = np.zeros(ref.shape)
        want[:c.seqs[0][0], 3, 200][sees(c, 0, 450, f)] = np.inf
        same_odd_values(launch(c, d, q, heads, entry, f), want, ref, tol)
        # and the append: new rows into the same slots
        rows = torch.randn(c.tokens, 2, nkv, hd, device="cuda").bfloat16()
        ti.check(ti.lib().ti_op_kv_append(C.byref(d["kv"]), C.byref(d["batch"]), None, None, 0, rows.data_ptr(),
                                          2 * nkv * hd, rows.data_ptr() + 2 * nkv * hd, 2 * nkv * hd, 0, None, 0, stream()))
        for s, (new, n) in enumerate(c.seqs):
            at = torch.arange(n - new, n)
            page = c.table[c.rows[s]][at // 16].long().cuda()
            for i, w in enumerate("kv"):
                t0 = int(c.starts[s])
                assert torch.equal(d[w][page, :, (at % 16).cuda()], rows[t0:t0 + new, i])


# ------------------------------------------------------------------ errors
def test_an_earlier_calls_error_is_not_this_ones():
    c = Cache([(1, 20)], 1, 64, "bf16", seed=46)
    d, x = c.dev(decode=True), torch.ones(1, 2, 64, dtype=torch.bfloat16, device="cuda")
    fr, pos = torch.ones(32, device="cuda"), torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    r = ti.RopeAxes(rot_dim=64, inv_freq=fr.data_ptr(), n_axes=1, pos=pos.data_ptr(), pos_stride=1)
    at, calls = x.data_ptr(), {
        "rope": lambda: ti.lib().ti_op_rope_axes(ti.DTYPE_BF16, at, 128, at, 128, 1, 2, 64, C.byref(r), stream()),
        "append": lambda: ti.lib().ti_op_kv_append(C.byref(d["kv"]), C.byref(d["batch"]), None, None, 0, at, 64, at, 64, 0,
                                                   None, 0, stream()),
        "prefill": lambda: ti.lib().ti_op_paged_prefill(C.byref(d["kv"]), C.byref(d["batch"]), None, at, 128, 2, at, 128,
                                                        stream()),
        "decode": lambda: ti.lib().ti_op_paged_decode(C.byref(d["kv"]), C.byref(d["batch"]), None, at, 128, 2, at, 128,
                                                      stream()),
    }
    for name, call in calls.items():
        assert ti.lib().ti_set_device(99) != 0
        assert call() == 0, (name, ti.lib().ti_last_error().decode())
    torch.cuda.synchronize()


# ------------------------------------------------------------------ scratch
POOL = """
import ctypes as C, sys
sys.path[:0] = [%r, %r]
import torch
import ti_b200 as ti
from paged_ref import Cache
from test_gpu_paged_ops import queries, run_attention, within
rt = C.CDLL("libcudart.so.12")
def default_threshold():
    pool, value = C.c_void_p(), C.c_uint64()
    assert rt.cudaDeviceGetDefaultMemPool(C.byref(pool), 0) == 0
    assert rt.cudaMemPoolGetAttribute(pool, 4, C.byref(value)) == 0  # cudaMemPoolAttrReleaseThreshold
    return value.value
torch.zeros(1, device="cuda")
before = default_threshold()
c = Cache([(1, 3000), (1, 40)], 1, 64, "bf16", seed=5)
if sys.argv[1] == "captured":  # the process's first call, in a captured stream
    d = c.dev(decode=True)
    q = queries(c, 4).cuda()
    out = torch.zeros_like(q)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ti.check(ti.lib().ti_op_paged_decode(C.byref(d["kv"]), C.byref(d["batch"]), None, q.data_ptr(), 256, 4,
                                             out.data_ptr(), 256, torch.cuda.current_stream().cuda_stream))
    g.replay()
    want, ref, tol = run_attention(c, q.cpu(), 4, "decode")
    within(want, ref, tol)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
else:
    out, ref, tol = run_attention(c, queries(c, 4), 4, "decode")
    within(out, ref, tol)
    p = Cache([(3, 3000)], 1, 64, "bf16", seed=5)
    out, ref, tol = run_attention(p, queries(p, 4), 4, "prefill")  # keys divided: with scratch
    within(out, ref, tol)
assert default_threshold() == before, (before, default_threshold())
ti.check(ti.lib().ti_shutdown())
out, ref, tol = run_attention(c, queries(c, 4), 4, "decode")  # and the library stays usable
within(out, ref, tol)
"""


@pytest.mark.parametrize("first", ["plain", "captured"])
def test_scratch_leaves_the_default_pool_as_it_is(first):
    here = os.path.dirname(os.path.abspath(__file__))
    code = POOL % (os.path.join(os.path.dirname(here), "tensor-inference_b200"), here)
    r = subprocess.run([sys.executable, "-c", code, first], capture_output=True, text=True, timeout=240)
    assert r.returncode == 0, r.stdout + r.stderr
