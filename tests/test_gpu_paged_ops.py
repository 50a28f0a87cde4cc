"""The serving operators over the paged cache on the GPU: rotation on several axes,
append, ragged prefill attention and decode attention, each against its plain form
in float64 with tolerances counted in roundings, and a serving run of all of them."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

import ti_b200 as ti
from paged_ref import CODE, DT, FLOOR, HALF_STEP, Cache, attend, axis_of_pair, rotate

pytestmark = pytest.mark.gpu
THETA = 500000.0


def stream():
    return torch.cuda.current_stream().cuda_stream


def freqs(rot_dim):
    return torch.from_numpy(ti.rope_inv_freq(rot_dim, THETA))


def rope_struct(rot_dim, fr, pos, sections=(), interleaved=0):
    n_axes = max(1, len(sections))
    return ti.RopeAxes(rot_dim=rot_dim, inv_freq=fr.data_ptr(), n_axes=n_axes,
                       sections=(C.c_int * 4)(*list(sections) + [0] * (4 - len(sections))), interleaved=interleaved,
                       pos=None if pos is None else pos.data_ptr(), pos_stride=0 if pos is None else pos.stride(0))


def angles(rot_dim, pos, sections=(), interleaved=0):
    ax = axis_of_pair(rot_dim // 2, max(1, len(sections)), sections, interleaved)
    return pos.double().numpy()[ax].T * freqs(rot_dim).double().numpy()


def within(got, ref, tol, msg=""):
    got = got.detach().cpu().double().numpy().reshape(ref.shape)
    assert np.isfinite(got).all(), msg + " not finite"
    worst = (np.abs(got - ref) - tol).max() if ref.size else 0.0
    where = np.unravel_index(np.argmax(np.abs(got - ref) - tol), ref.shape) if ref.size else ()
    assert worst <= 0, f"{msg} off by {np.abs(got - ref)[where]:.3e} (allowed {tol[where]:.3e}) at {where}"


# ------------------------------------------------------------------ rotation
ROPE = [
    # tokens, heads, hd, rot_dim, sections, interleaved
    (1, 1, 64, 64, (), 0), (3, 5, 128, 128, (), 0), (37, 16, 64, 64, (16, 16), 0), (130, 28, 128, 128, (24, 20, 20), 1),
    (20, 3, 96, 64, (10, 12, 10), 1), (9, 2, 80, 80, (40, 0, 0, 0), 0), (9, 2, 80, 20, (4, 3, 2, 1), 0),
    (400, 2, 256, 256, (50, 60, 18), 0), (5, 3, 6, 2, (), 0), (7, 1, 1024, 512, (100, 156), 1),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16", "f32"])
@pytest.mark.parametrize("tokens, heads, hd, rot, sections, inter", ROPE)
def test_rope_axes(dtype, tokens, heads, hd, rot, sections, inter):
    g = torch.Generator().manual_seed(tokens)
    x = torch.randn(tokens, heads, hd, generator=g).to(DT[dtype])
    # positions up to the largest and below zero: an fp32 angle would be off by whole radians
    pos = torch.randint(-2**31, 2**31 - 1, (max(1, len(sections)), tokens + 3), generator=g).to(torch.int32)
    pos[:, : tokens // 2] = torch.randint(0, 5000, (pos.shape[0], tokens // 2), generator=g).to(torch.int32)
    dx, dp, fr = x.cuda(), pos.cuda(), freqs(rot).cuda()
    out = torch.full_like(dx, float("nan"))
    ti.check(ti.lib().ti_op_rope_axes(CODE[dtype], dx.data_ptr(), heads * hd, out.data_ptr(), heads * hd, tokens, heads,
                                      hd, C.byref(rope_struct(rot, fr, dp, sections, inter)), stream()))
    ref, off = rotate(x.double().numpy(), angles(rot, pos[:, :tokens], sections, inter), rot)
    within(out, ref, HALF_STEP[dtype] * np.abs(ref) * 1.01 + off + FLOOR[dtype])
    # in place, the same bits
    ti.check(ti.lib().ti_op_rope_axes(CODE[dtype], dx.data_ptr(), heads * hd, dx.data_ptr(), heads * hd, tokens, heads,
                                      hd, C.byref(rope_struct(rot, fr, dp, sections, inter)), stream()))
    assert torch.equal(dx, out)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("offset, gap", [(0, 8), (1, 0), (3, 5), (8, 24)])
def test_rope_axes_strides_and_alignment(dtype, offset, gap):
    tokens, heads, hd = 11, 3, 64
    width = heads * hd
    g = torch.Generator().manual_seed(gap)
    buf = torch.randn(offset + tokens * (width + gap), generator=g).to(DT[dtype]).cuda()
    out = torch.zeros(7 + tokens * (width + 2), dtype=DT[dtype], device="cuda")
    pos = torch.randint(0, 100000, (1, tokens), generator=g).to(torch.int32)
    fr, dp = freqs(hd).cuda(), pos.cuda()
    es = buf.element_size()
    ti.check(ti.lib().ti_op_rope_axes(CODE[dtype], buf.data_ptr() + offset * es, width + gap, out.data_ptr() + 7 * es,
                                      width + 2, tokens, heads, hd, C.byref(rope_struct(hd, fr, dp)), stream()))
    x = buf[offset:].view(tokens, width + gap)[:, :width].reshape(tokens, heads, hd)
    ref, off = rotate(x.cpu().double().numpy(), angles(hd, pos), hd)
    rows = out[7:].view(tokens, width + 2)
    within(rows[:, :width], ref.reshape(tokens, width), (HALF_STEP[dtype] * np.abs(ref) * 1.01 + off).reshape(tokens, width))
    assert not rows[:, width:].any() and not out[:7].any()  # the gaps are left as they were


# ------------------------------------------------------------------ append
APPEND = [
    # (new, length) per sequence, heads, nkv, hd, pad tokens
    ([(1, 1)], 4, 2, 64, 0), ([(1, 17), (1, 16), (1, 33)], 8, 8, 128, 0),
    ([(5, 5), (0, 12), (33, 50), (0, 0), (1, 32)], 6, 2, 64, 7), ([(70, 200), (129, 129)], 28, 4, 128, 3),
    ([(3, 20)], 3, 1, 256, 0), ([(17, 40), (2, 2)], 5, 5, 10, 1),
]


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("axes", [0, 1, 3])
@pytest.mark.parametrize("seqs, heads, nkv, hd, pad", APPEND)
def test_kv_append(dtype, axes, seqs, heads, nkv, hd, pad):
    c = Cache(seqs, nkv, hd, dtype, seed=hd, pad_tokens=pad, spare_rows=2)
    d = c.dev()
    before_k, before_v = d["k"].clone(), d["v"].clone()
    g = torch.Generator().manual_seed(axes)
    T = c.tokens
    qkv = torch.randn(T, (heads + 2 * nkv) * hd, generator=g).to(DT[dtype])
    dq, es = qkv.cuda(), 2
    q_out = torch.full((T, heads, hd), 7.0, dtype=DT[dtype], device="cuda")
    half = hd // 2
    sections = (half - 2 * (half // 3), half // 3, half // 3) if axes == 3 else ()
    pos = torch.randint(0, 3000, (max(1, axes), T), generator=g).to(torch.int32)
    dp, fr = pos.cuda(), freqs(hd).cuda()
    # one axis takes the position in the cache when it is given none
    r = rope_struct(hd, fr, dp if axes == 3 else None, sections, 1) if axes else None
    base, w = dq.data_ptr(), dq.shape[1]
    ti.check(ti.lib().ti_op_kv_append(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(r) if r else None, base, w,
                                      base + heads * hd * es, w, base + (heads + nkv) * hd * es, w, heads,
                                      q_out.data_ptr(), heads * hd, stream()))
    at = np.zeros(T, np.int64)
    for s, (new, n) in enumerate(seqs):
        at[c.starts[s]:c.starts[s] + new] = np.arange(n - new, n)
    x = qkv.double().numpy().reshape(T, heads + 2 * nkv, hd)
    ang = angles(hd, pos, sections, 1) if axes == 3 else angles(hd, torch.from_numpy(at)[None])
    if not axes:
        ang = np.zeros_like(ang)
    y, off = rotate(x, ang, hd)
    tol = HALF_STEP[dtype] * np.abs(y) * 1.01 + off + FLOOR[dtype] if axes else np.zeros_like(y)
    real = int(c.starts[-1])
    within(q_out[:real], y[:real, :heads], tol[:real, :heads], "q")
    assert (q_out[real:] == 7.0).all()  # padding rows belong to nobody
    for s, (new, n) in enumerate(seqs):
        t = slice(int(c.starts[s]), int(c.starts[s]) + new)
        within(c.read(d["k"], s)[n - new:], y[t, heads:heads + nkv], tol[t, heads:heads + nkv], "k")
        assert torch.equal(c.read(d["v"], s)[n - new:], qkv.view(T, -1, hd)[t, heads + nkv:])
        assert torch.equal(c.read(d["k"], s)[:n - new], c.K[s][:n - new])
        assert torch.equal(c.read(d["v"], s)[:n - new], c.V[s][:n - new])
    # slots of no sequence are untouched (NaN before and after): compare bits everywhere else
    new_slots = torch.zeros(c.n_pages, 16, dtype=torch.bool)
    for s, (new, n) in enumerate(seqs):
        for i in range(n - new, n):
            new_slots[c.table[c.rows[s], i // 16], i % 16] = True
    for a, b in ((d["k"], before_k), (d["v"], before_v)):
        a, b = a.cpu().view(torch.int16).transpose(1, 2), b.cpu().view(torch.int16).transpose(1, 2)
        assert torch.equal(a[~new_slots], b[~new_slots])


@pytest.mark.parametrize("tokens", [3, 700])
def test_kv_append_rotates_q_in_place(tokens):
    heads, nkv, hd = 4, 2, 64
    c = Cache([(tokens, tokens + 5)], nkv, hd, "bf16", seed=2)
    d = c.dev()
    g = torch.Generator().manual_seed(2)
    qkv = torch.randn(tokens, (heads + 2 * nkv) * hd, generator=g).to(torch.bfloat16)
    dq, w, es, fr = qkv.cuda(), qkv.shape[1], 2, freqs(hd).cuda()
    r = rope_struct(hd, fr, None)
    b = dq.data_ptr()
    ti.check(ti.lib().ti_op_kv_append(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(r), b, w, b + heads * hd * es, w,
                                      b + (heads + nkv) * hd * es, w, heads, b, w, stream()))
    x = qkv.double().numpy().reshape(tokens, -1, hd)
    y, off = rotate(x, angles(hd, torch.arange(5, tokens + 5)[None]), hd)
    tol = HALF_STEP["bf16"] * np.abs(y) * 1.01 + off + FLOOR["bf16"]
    got = dq.view(tokens, -1, hd)
    within(got[:, :heads], y[:, :heads], tol[:, :heads])
    assert torch.equal(got[:, heads:].cpu(), qkv.view(tokens, -1, hd)[:, heads:])  # k and v rows are inputs only
    within(c.read(d["k"], 0)[5:], y[:, heads:heads + nkv], tol[:, heads:heads + nkv])


def test_kv_append_without_q_and_with_bad_ids():
    c = Cache([(4, 20), (3, 3), (2, 40), (2, 18)], 2, 64, "bf16", seed=3)
    c.table[c.rows[0], 1] = c.n_pages  # the page of positions 16..19 of sequence 0 does not exist
    c.table[c.rows[1], 0] = -5
    d = c.dev()
    d["len"][2] = 16 * c.wide + 2  # its new positions lie past the page table
    d["rows"][3] = 99              # no such row
    before = d["k"].clone(), d["v"].clone()
    g = torch.Generator().manual_seed(1)
    kv = torch.randn(c.tokens, 2, 2, 64, generator=g).to(torch.bfloat16).cuda()
    ti.check(ti.lib().ti_op_kv_append(C.byref(d["kv"]), C.byref(d["batch"]), None, None, 0, kv.data_ptr(), 256,
                                      kv.data_ptr() + 256, 256, 0, None, 0, stream()))
    for a, b in zip((d["k"], d["v"]), before):
        assert torch.equal(a.view(torch.int16), b.view(torch.int16))  # nothing was written anywhere


# ------------------------------------------------------------------ attention
FORMS = {
    "plain": {},
    "cap": dict(cap=20.0),
    "bias": dict(alibi=True),
    "window": dict(window=19),
    "prefix": dict(prefix=True),
    "docs": dict(docs=True),
    "all": dict(cap=5.0, alibi=True, window=150, prefix=True, docs=True, scale=0.3),
}


def run_attention(c, q, heads, entry, cap=0.0, alibi=False, window=0, prefix=False, docs=False, scale=0.0, out=None,
                  d=None, indirect=True):
    """(out, reference rows, tolerance)"""
    d = d or c.dev(decode=entry == "decode", indirect=indirect)
    T, hd = c.tokens, c.hd
    g = np.random.default_rng(heads + window)
    slopes = np.float32(2.0) ** (-8.0 * (np.arange(heads) + 1) / heads) if alibi else None
    pre = g.integers(0, c.max_len + 20, len(c.seqs)).astype(np.int32) if prefix else None
    doc = None
    if docs:  # some documents start after their token: those rows see nothing
        doc = np.zeros(T, np.int32)
        for s, (new, n) in enumerate(c.seqs):
            i = np.arange(n - new, n)
            doc[c.starts[s]:c.starts[s] + new] = i - i % 23 + (i % 7 == 3) * 40
    keep = [torch.from_numpy(np.ascontiguousarray(x)).cuda() if x is not None else None
            for x in (None if slopes is None else slopes.astype(np.float32), pre, doc)]
    f = ti.AttnForm(scale=scale, softcap=cap, slopes=None if keep[0] is None else keep[0].data_ptr(),
                    sliding_window=window, prefix=None if keep[1] is None else keep[1].data_ptr(),
                    doc_start=None if keep[2] is None else keep[2].data_ptr())
    dq = q.cuda()
    out = torch.full((T, heads, hd), 3.0, dtype=DT[c.dtype], device="cuda") if out is None else out
    fn = getattr(ti.lib(), f"ti_op_paged_{entry}")
    ti.check(fn(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(f), dq.data_ptr(), dq.stride(0), heads, out.data_ptr(),
                out.stride(0), stream()))
    ref, tol = attend(c, q, heads, cap=cap, slopes=slopes, window=window, prefix=pre, doc=doc, scale=scale)
    return out, ref, tol


def queries(c, heads, seed=5, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(c.tokens, heads, c.hd, generator=g) * std).to(DT[c.dtype])


PREFILL = [
    # (new, length) per sequence, heads, nkv, pad tokens
    ([(1, 1)], 2, 1, 0),
    ([(7, 7), (1, 40), (0, 30), (0, 0), (16, 16)], 4, 2, 5),
    ([(129, 129), (60, 260)], 8, 2, 0),
    ([(300, 300)], 3, 3, 2),
    ([(33, 700), (2, 129)], 7, 1, 0),
    ([(20, 300)] * 3 + [(128, 128)], 40, 2, 0),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("seqs, heads, nkv, pad", PREFILL)
def test_paged_prefill(seqs, heads, nkv, pad, hd, form):
    dtype = "f16" if (len(seqs) + heads) % 2 else "bf16"
    c = Cache(seqs, nkv, hd, dtype, seed=hd + heads, pad_tokens=pad, spare_rows=1)
    out, ref, tol = run_attention(c, queries(c, heads), heads, "prefill", **FORMS[form])
    real = int(c.starts[-1])
    within(out[:real], ref[:real], tol[:real])
    assert (out[real:] == 3.0).all()


DECODE = [
    ([1], 2, 1), ([16], 4, 4), ([1, 17, 0, 64, 33], 8, 2), ([700, 2, 129], 28, 4), ([2000], 32, 4), ([300, 5], 16, 1),
    ([40, 41], 40, 2), ([5000, 1], 8, 1),
]


@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("lens, heads, nkv", DECODE)
def test_paged_decode(lens, heads, nkv, hd, form):
    dtype = "f16" if (len(lens) + hd // 64) % 2 else "bf16"
    c = Cache([(1, n) for n in lens], nkv, hd, dtype, seed=hd + heads, spare_rows=1)
    out, ref, tol = run_attention(c, queries(c, heads), heads, "decode", **FORMS[form])
    within(out, ref, tol)


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_both_types_at_one_shape(entry, dtype):
    c = Cache([(1, 90), (1, 300)] if entry == "decode" else [(50, 90), (200, 300)], 2, 128, dtype, seed=9)
    out, ref, tol = run_attention(c, queries(c, 8), 8, entry, cap=30.0)
    within(out, ref, tol)


@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_large_scores_reach_the_cap(entry):
    # scores far past the cap on both sides: tanh saturates, and one key takes most of the weight without it
    c = Cache([(1, 260), (1, 31)] if entry == "decode" else [(40, 260), (31, 31)], 1, 64, "bf16", seed=2, std=6.0)
    for cap in (0.0, 2.0, 50.0):
        out, ref, tol = run_attention(c, queries(c, 4, std=6.0), 4, entry, cap=cap)
        within(out, ref, tol, f"cap {cap}")


@pytest.mark.parametrize("dtype", ["bf16", "f16"])
@pytest.mark.parametrize("cap", [2e-4, 0.02, 1.0, 54.0, 56.0, 300.0, 1000.0])
@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_caps_of_any_size(entry, cap, dtype):
    # far below the scores (all of them at the cap), about them, and far above (no cap in effect)
    c = Cache([(1, 260), (1, 31)] if entry == "decode" else [(40, 260), (31, 31)], 1, 64, dtype, seed=2, std=2.0)
    out, ref, tol = run_attention(c, queries(c, 4, std=2.0), 4, entry, cap=cap)
    within(out, ref, tol)


@pytest.mark.parametrize("entry", ["prefill", "decode"])
@pytest.mark.parametrize("sign", [-1.0, 1.0])
def test_scores_all_at_one_end_of_the_cap(entry, sign):
    # every score at -cap or at +cap, values up to 1e20: weights far from 1 must not leave the range
    c = Cache([(1, 200)] if entry == "decode" else [(30, 200)], 1, 64, "bf16", seed=3)
    c.K[0] = torch.full_like(c.K[0], sign * 10)
    c.V[0] = c.V[0] * 1e20
    for p in range(-(-200 // 16)):
        m = min(16, 200 - p * 16)
        page = int(c.table[c.rows[0], p])
        c.k[page, :, :m] = c.K[0][p * 16:p * 16 + m].transpose(0, 1)
        c.v[page, :, :m] = c.V[0][p * 16:p * 16 + m].transpose(0, 1)
    q = torch.ones(c.tokens, 2, 64, dtype=torch.bfloat16)
    for cap in (30.0, 50.0, 55.0, 60.0):
        out, ref, tol = run_attention(c, q, 2, entry, cap=cap)
        within(out, ref, tol, f"cap {cap}")


@pytest.mark.parametrize("form", ["plain", "all"])
def test_many_sequences(form):
    # more sequences than one round of the look-ups takes, empty ones among them
    g = np.random.default_rng(1)
    lens = [int(n) for n in g.integers(0, 50, 700)]
    c = Cache([(1, n) for n in lens], 1, 64, "bf16", seed=1)
    out, ref, tol = run_attention(c, queries(c, 2), 2, "decode", **FORMS[form])
    within(out, ref, tol)
    c = Cache([(int(min(n, g.integers(0, 4))), n) for n in lens[:150]], 2, 64, "f16", seed=2, pad_tokens=3)
    out, ref, tol = run_attention(c, queries(c, 4), 4, "prefill", **FORMS[form])
    real = int(c.starts[-1])
    within(out[:real], ref[:real], tol[:real])
    assert (out[real:] == 3.0).all()


@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_slopes_of_any_sign(entry):
    heads = 6
    c = Cache([(1, 300), (1, 40)] if entry == "decode" else [(20, 300), (40, 40)], 2, 64, "bf16", seed=6)
    q = queries(c, heads)
    slopes = torch.tensor([0.0, -0.01, 1e-13, 3.0, 0.5, 1e-6])
    for cap in (0.0, 10.0):
        d = c.dev(decode=entry == "decode")
        ds, dq, out = slopes.cuda(), q.cuda(), torch.zeros(c.tokens, heads, 64, dtype=torch.bfloat16, device="cuda")
        pre = torch.tensor([200, 7], dtype=torch.int32)
        dp = pre.cuda()
        f = ti.AttnForm(softcap=cap, slopes=ds.data_ptr(), prefix=dp.data_ptr())
        ti.check(getattr(ti.lib(), f"ti_op_paged_{entry}")(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(f), dq.data_ptr(),
                                                           heads * 64, heads, out.data_ptr(), heads * 64, stream()))
        ref, tol = attend(c, q, heads, cap=cap, slopes=slopes.double().numpy(), prefix=pre.numpy())
        within(out, ref, tol, f"cap {cap}")


@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_without_row_indirection_and_with_strides(entry):
    heads, hd = 4, 64
    c = Cache([(1, 50), (1, 3)] if entry == "decode" else [(9, 50), (3, 3)], 2, hd, "bf16", seed=4)
    c.rows = torch.arange(2, dtype=torch.int32)
    c2 = Cache([(n, m) for n, m in c.seqs], 2, hd, "bf16", seed=4)
    order = c2.rows.long()
    c.table = c2.table[order].contiguous()  # the same sequences as rows 0, 1
    q = queries(c, heads)
    base, ref, tol = run_attention(c, q, heads, entry, indirect=False)
    within(base, ref, tol)
    # rows 5 elements apart and off the 16-byte grid give the same bits
    T, width = c.tokens, heads * hd
    d = c.dev(decode=entry == "decode", indirect=False)
    qb = torch.zeros(1 + T * (width + 5), dtype=torch.bfloat16, device="cuda")
    qb[1:].view(T, width + 5)[:, :width] = q.cuda().view(T, width)
    ob = torch.full((3 + T * (width + 7),), 9.0, dtype=torch.bfloat16, device="cuda")
    fn = getattr(ti.lib(), f"ti_op_paged_{entry}")
    ti.check(fn(C.byref(d["kv"]), C.byref(d["batch"]), None, qb.data_ptr() + 2, width + 5, heads, ob.data_ptr() + 6,
                width + 7, stream()))
    rows = ob[3:].view(T, width + 7)
    assert torch.equal(rows[:, :width].reshape(T, heads, hd), base)
    assert (rows[:, width:] == 9.0).all() and (ob[:3] == 9.0).all()


@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_bad_ids_read_as_zero_keys_and_nothing_else(entry):
    heads, hd = 4, 64
    c = Cache([(1, 40), (1, 60), (1, 20)] if entry == "decode" else [(9, 40), (10, 60), (4, 20)], 2, hd, "bf16", seed=8)
    q = queries(c, heads)
    good, ref, tol = run_attention(c, q, heads, entry)
    d = c.dev(decode=entry == "decode")
    d["table"][c.rows[0], 1] = 10**6   # a page that does not exist: its 16 keys and values read as zeros
    d["rows"][1] = -3                  # a row that does not exist: no keys, zero rows
    c.K[0][16:32] = 0
    c.V[0][16:32] = 0
    out, ref, tol = run_attention(c, q, heads, entry, d=d)
    t1, t2 = int(c.starts[1]), int(c.starts[2])
    within(out[:t1], ref[:t1], tol[:t1])
    assert not out[t1:t2].any()
    assert torch.equal(out[t2:], good[t2:])


def test_lengths_past_max_len_and_past_the_table():
    # max_len only divides the work; a length past the page table ends at the table's last slot
    heads, hd = 8, 128
    for entry, seqs in (("decode", [(1, 1500), (1, 64)]), ("prefill", [(30, 1500), (64, 64)])):
        c = Cache(seqs, 2, hd, "bf16", seed=6)
        q = queries(c, heads)
        c.max_len = 10
        out, ref, tol = run_attention(c, q, heads, entry)
        within(out, ref, tol)
        d = c.dev(decode=entry == "decode")
        d["len"][0] = 16 * c.wide + 40  # every new token now sees all slots of its row; the last page's tail is NaN
        d["kv"].pt_stride = c.wide
        n = 16 * c.wide
        pool_k, pool_v = d["k"], d["v"]
        last = int(c.table[c.rows[0], c.wide - 1])
        pool_k[last], pool_v[last] = pool_k[last].nan_to_num(0.0), pool_v[last].nan_to_num(0.0)
        out2 = torch.zeros_like(out)
        dq = q.cuda()
        fn = getattr(ti.lib(), f"ti_op_paged_{entry}")
        ti.check(fn(C.byref(d["kv"]), C.byref(d["batch"]), None, dq.data_ptr(), heads * hd, heads, out2.data_ptr(),
                    heads * hd, stream()))
        new = seqs[0][0]
        full = Cache([(new, n)], 2, hd, "bf16", seed=1)
        full.K[0] = torch.zeros(n, 2, hd, dtype=torch.bfloat16)
        full.V[0] = torch.zeros(n, 2, hd, dtype=torch.bfloat16)
        full.K[0][:1500], full.V[0][:1500] = c.K[0], c.V[0]
        # positions 16 wide + 40 - new ..: at least the last slot, so every token sees all n keys
        ref2, tol2 = attend(full, q[:new], heads, prefix=[n])
        if new <= 40:
            within(out2[:new], ref2, tol2)
        assert torch.equal(out2[new:], out[new:])


@pytest.mark.parametrize("entry", ["prefill", "decode"])
def test_nan_outside_the_mask_does_not_enter(entry):
    # keys and values that no token sees (before a window, before a document) hold NaN and infinities
    heads, hd = 4, 128
    seqs = [(1, 400), (1, 90)] if entry == "decode" else [(20, 400), (10, 90)]
    c = Cache(seqs, 2, hd, "bf16", seed=12)
    q = queries(c, heads)
    clean, ref, tol = run_attention(c, q, heads, entry, window=50)
    within(clean, ref, tol)
    d = c.dev(decode=entry == "decode")
    for s, (new, n) in enumerate(seqs):
        for i in range(0, n - new - 49):
            page = int(c.table[c.rows[s], i // 16])
            d["k"][page, :, i % 16] = float("nan") if i % 2 else float("inf")
            d["v"][page, :, i % 16] = float("inf") if i % 3 else float("nan")
    out, _, _ = run_attention(c, q, heads, entry, window=50, d=d)
    assert torch.equal(out, clean)


@pytest.mark.parametrize("dtype, cap", [("bf16", 0.0), ("bf16", 20.0), ("f16", 0.0), ("f16", 20.0)])
@pytest.mark.parametrize("hd", [64, 128, 256])
@pytest.mark.parametrize("window, max_len", [(90, 200), (0, 200), (0, 4096)])  # the last: keys divided over CTAs
@pytest.mark.parametrize("odd", [[61], [3, 61, 62, 130], list(range(20, 120))])
def test_nan_and_infinities_in_v_reach_the_rows_that_see_them(odd, window, max_len, hd, dtype, cap):
    # rows before the key, or whose window has passed it, share its tiles and stay finite; the others get a NaN
    # or an infinity of its sign in that dimension alone
    heads = 4
    c = Cache([(150, 200)], 2, hd, dtype, seed=13)
    c.max_len = max_len
    q = queries(c, heads)
    clean, ref, tol = run_attention(c, q, heads, "prefill", window=window, cap=cap)
    within(clean, ref, tol)
    d = c.dev()
    values = [float("nan"), float("inf"), -float("inf")]
    want = np.zeros((150, heads, hd))
    for n, j in enumerate(odd):
        page, dim, h = int(c.table[c.rows[0], j // 16]), (7 * j) % hd, j % 2
        d["v"][page, h, j % 16, dim] = values[n % 3]
        i = np.arange(50, 200)
        rows = (i >= j) & ((i - j < window) | (window == 0))
        with np.errstate(invalid="ignore"):
            want[rows, 2 * h:2 * h + 2, dim] += values[n % 3]
    out, _, _ = run_attention(c, q, heads, "prefill", window=window, cap=cap, d=d)
    got = out.cpu().double().numpy()
    fine = want == 0
    assert np.isfinite(got[fine]).all()
    # the odd values are single dimensions of V: every other output keeps its value
    assert (np.abs(got - ref)[fine] <= tol[fine]).all()
    np.testing.assert_array_equal(np.isnan(got[~fine]), np.isnan(want[~fine]))
    inf = ~fine & np.isinf(want)
    np.testing.assert_array_equal(got[inf], want[inf])


def test_lowest_values_in_keys_are_ordinary_scores():
    # keys at the type's lowest value give scores near its range's end, not masks
    c = Cache([(1, 20)], 1, 64, "bf16", seed=1)
    c.K[0][:10] = torch.finfo(torch.bfloat16).min / 2 ** 70
    page = c.table[c.rows[0], 0].item()
    c.k[page, :, :10] = c.K[0][:10].transpose(0, 1)
    q = torch.ones(1, 2, 64, dtype=torch.bfloat16)
    for entry in ("decode", "prefill"):
        out, ref, tol = run_attention(c, q, 2, entry)
        within(out, ref, tol)


# ------------------------------------------------------------------ the operators together
@pytest.mark.parametrize("dtype", ["bf16", "f16"])
def test_serving_run(dtype):
    """Prompts appended and attended in two chunks, then single tokens: the same rows as
    one prefill over everything (within two results' tolerances), from the projections on."""
    heads, nkv, hd, lens = 8, 2, 64, [70, 5, 131]
    c = Cache([(n, n) for n in lens], nkv, hd, dtype, seed=21)
    g = torch.Generator().manual_seed(3)
    qkv = torch.randn(sum(lens), (heads + 2 * nkv) * hd, generator=g).to(DT[dtype]).cuda()
    fr = freqs(hd).cuda()
    r = rope_struct(hd, fr, None)
    form = ti.AttnForm(softcap=25.0, sliding_window=60)
    w, es = qkv.shape[1], 2

    def step(d, rows, start, length, out, decode=False):
        n = rows.shape[0]
        batch = ti.Ragged(n_seqs=len(lens), n_tokens=n, start=None if decode else start.data_ptr(),
                          kv_len=length.data_ptr(), row=d["rows"].data_ptr(), max_len=max(lens))
        q = torch.empty(n, heads, hd, dtype=DT[dtype], device="cuda")
        b = rows.data_ptr()
        ti.check(ti.lib().ti_op_kv_append(C.byref(d["kv"]), C.byref(batch), C.byref(r), b, w, b + heads * hd * es, w,
                                          b + (heads + nkv) * hd * es, w, heads, q.data_ptr(), heads * hd, stream()))
        fn = ti.lib().ti_op_paged_decode if decode else ti.lib().ti_op_paged_prefill
        ti.check(fn(C.byref(d["kv"]), C.byref(batch), C.byref(form), q.data_ptr(), heads * hd, heads, out.data_ptr(),
                    heads * hd, stream()))
        return q

    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    at = [sum(lens[:s]) for s in range(3)]
    d = c.dev()
    whole = torch.empty(sum(lens), heads, hd, dtype=DT[dtype], device="cuda")
    q = step(d, qkv, i32(at + [sum(lens)]), i32(lens), whole)
    k_all, v_all = d["k"].clone(), d["v"].clone()
    # the reference, from the rotated rows in the cache
    for s in range(3):
        c.K[s], c.V[s] = c.read(d["k"], s), c.read(d["v"], s)
    ref, tol = attend(c, q.cpu(), heads, cap=25.0, window=60)
    within(whole, ref, tol, "whole")

    d = c.dev()
    d["k"].fill_(float("nan")), d["v"].fill_(float("nan"))
    got = torch.zeros_like(whole)
    done = [0, 0, 0]
    for chunk in ([30, 3, 100], [38, 0, 29]):
        idx = torch.cat([torch.arange(at[s] + done[s], at[s] + done[s] + chunk[s]) for s in range(3)]).cuda()
        start = [sum(chunk[:s]) for s in range(4)]
        done = [a + b for a, b in zip(done, chunk)]
        out = torch.zeros(len(idx), heads, hd, dtype=DT[dtype], device="cuda")
        step(d, qkv[idx], i32(start), i32(done), out)
        got[idx] = out
    for _ in range(2):
        idx = torch.tensor([at[s] + done[s] for s in range(3)]).cuda()
        done = [x + 1 for x in done]
        out = torch.zeros(3, heads, hd, dtype=DT[dtype], device="cuda")
        step(d, qkv[idx], None, i32(done), out, decode=True)
        got[idx] = out
    assert done == lens
    for s in range(3):
        assert torch.equal(c.read(d["k"], s), c.read(k_all, s)) and torch.equal(c.read(d["v"], s), c.read(v_all, s))
    within(got, ref, tol, "chunks")


def test_streams_graphs_and_repeats():
    """Two captured graphs that share the cache and replay in turn, a side stream, and the
    same call twice: all the same bits."""
    heads, nkv, hd = 8, 1, 128
    c = Cache([(1, 3000), (1, 40)], nkv, hd, "bf16", seed=5)
    p = Cache([(20, 900), (70, 70)], nkv, hd, "bf16", seed=6)
    qd, qp = queries(c, heads).cuda(), queries(p, heads).cuda()
    dd, dp = c.dev(decode=True), p.dev()
    f = ti.AttnForm(softcap=30.0)

    def call(entry, d, q, out):
        ti.check(getattr(ti.lib(), f"ti_op_paged_{entry}")(C.byref(d["kv"]), C.byref(d["batch"]), C.byref(f), q.data_ptr(),
                                                           heads * hd, heads, out.data_ptr(), heads * hd, stream()))

    outs = [torch.zeros_like(qd), torch.zeros_like(qp)]
    call("decode", dd, qd, outs[0])
    call("prefill", dp, qp, outs[1])
    want = [o.clone() for o in outs]
    assert want[0].isfinite().all() and want[1].isfinite().all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for o in outs:
            o.zero_()
        call("decode", dd, qd, outs[0])
        call("prefill", dp, qp, outs[1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(outs, want))
    graphs = []
    for entry, d, q, out in (("decode", dd, qd, outs[0]), ("prefill", dp, qp, outs[1])):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            call(entry, d, q, out)
            call(entry, d, q, out)
        graphs.append(gr)
    for _ in range(3):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
        graphs[1].replay()  # at the same time as the first
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_host_memory_is_refused():
    c = Cache([(1, 5)], 1, 64, "bf16")
    d = c.dev(decode=True)
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    st = ti.lib().ti_op_paged_decode(C.byref(d["kv"]), C.byref(d["batch"]), None, q.cuda().data_ptr(), 128, 2,
                                     q.data_ptr(), 128, stream())
    assert st == ti.TI_ERR_INVALID and "device memory" in ti.lib().ti_last_error().decode()


@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_another_device_than_the_current_one():
    with torch.cuda.device(1):
        c = Cache([(1, 300), (1, 20)], 2, 64, "bf16", seed=7)
        q = queries(c, 4)
        d = c.dev(decode=True)
        dq, out = q.cuda(), torch.zeros(2, 4, 64, dtype=torch.bfloat16, device="cuda")
        s = torch.cuda.Stream()
        torch.cuda.synchronize()
    with torch.cuda.device(0):
        ti.check(ti.lib().ti_op_paged_decode(C.byref(d["kv"]), C.byref(d["batch"]), None, dq.data_ptr(), 256, 4,
                                             out.data_ptr(), 256, s.cuda_stream))
        assert torch.cuda.current_device() == 0
    torch.cuda.synchronize(1)
    ref, tol = attend(c, q, 4)
    within(out, ref, tol)
