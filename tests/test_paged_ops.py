"""The serving operators over the paged cache without a GPU: what they refuse
before touching a device, and the host-side frequency table."""
import ctypes as C

import numpy as np
import pytest

import oracle
import ti_b200 as ti

P = 0x10000  # a 16-byte aligned address that is never read: every call here is refused first


def rope(**kw):
    d = dict(rot_dim=64, inv_freq=P, n_axes=1, sections=(C.c_int * 4)(), interleaved=0, pos=P, pos_stride=100)
    d.update(kw)
    d["sections"] = (C.c_int * 4)(*d["sections"])
    return ti.RopeAxes(**d)


def kv(**kw):
    d = dict(dtype=ti.DTYPE_BF16, n_kv=2, head_dim=64, k_pages=P, v_pages=P, n_pages=8, page_table=P, table_rows=4,
             pt_stride=2)
    d.update(kw)
    return ti.PagedKv(**d)


def ragged(**kw):
    d = dict(n_seqs=2, n_tokens=5, start=P, kv_len=P, row=None, max_len=32)
    d.update(kw)
    return ti.Ragged(**d)


def form(**kw):
    return ti.AttnForm(**kw)


def refused(status, code, word):
    assert status == code
    assert word in ti.lib().ti_last_error().decode()


@pytest.mark.parametrize("args, word", [
    (dict(x=None), "null"), (dict(out=None), "null"), (dict(n=-1), "shape"), (dict(heads=0), "shape"),
    (dict(hd=63), "shape"), (dict(hd=2048), "shape"), (dict(xs=127), "stride"), (dict(os=100), "stride"),
    (dict(x=P, out=P, os=256), "in place"),
])
def test_rope_axes_refuses_bad_arguments(args, word):
    a = dict(dtype=ti.DTYPE_BF16, x=P, xs=128, out=2 * P, os=128, n=5, heads=2, hd=64)
    a.update(args)
    refused(ti.lib().ti_op_rope_axes(a["dtype"], a["x"], a["xs"], a["out"], a["os"], a["n"], a["heads"], a["hd"],
                                     C.byref(rope()), None), ti.TI_ERR_INVALID, word)


def test_rope_axes_refuses_types_it_does_not_rotate():
    refused(ti.lib().ti_op_rope_axes(ti.DTYPE_I32, P, 128, 2 * P, 128, 5, 2, 64, C.byref(rope()), None),
            ti.TI_ERR_UNSUPPORTED, "dtype")


@pytest.mark.parametrize("kw, word", [
    (dict(rot_dim=0), "rot_dim"), (dict(rot_dim=33), "rot_dim"), (dict(rot_dim=66), "rot_dim"),
    (dict(inv_freq=None), "inv_freq"), (dict(n_axes=0), "axes"), (dict(n_axes=5), "axes"), (dict(pos=None), "positions"),
    (dict(n_axes=2, sections=(16, 15, 0, 0)), "sections"), (dict(n_axes=2, sections=(40, -8, 0, 0)), "negative"),
    (dict(n_axes=3, sections=(2**31 - 1, 2**31 - 1, 34, 0)), "sections"),
    (dict(n_axes=2, sections=(16, 16, 0, 0), pos_stride=4), "pos_stride"),
])
def test_rotation_refuses_bad_axes(kw, word):
    r = rope(**kw)
    refused(ti.lib().ti_op_rope_axes(ti.DTYPE_BF16, P, 128, 2 * P, 128, 5, 2, 64, C.byref(r), None),
            ti.TI_ERR_INVALID, word)
    if kw.get("pos", P) is not None:
        refused(ti.lib().ti_op_kv_append(C.byref(kv()), C.byref(ragged()), C.byref(r), None, 0, P, 128, P, 128, 0,
                                         None, 0, None), ti.TI_ERR_INVALID, word)


def test_append_needs_positions_for_several_axes_only():
    r = rope(n_axes=2, sections=(16, 16, 0, 0), pos=None)
    refused(ti.lib().ti_op_kv_append(C.byref(kv()), C.byref(ragged()), C.byref(r), None, 0, P, 128, P, 128, 0, None,
                                     0, None), ti.TI_ERR_INVALID, "positions")


BAD_CACHES = [
    (dict(dtype=ti.DTYPE_F32), {}, ti.TI_ERR_UNSUPPORTED, "dtype"),
    (dict(n_kv=0), {}, ti.TI_ERR_INVALID, "empty"),
    (dict(n_pages=0), {}, ti.TI_ERR_INVALID, "empty"),
    (dict(table_rows=0), {}, ti.TI_ERR_INVALID, "empty"),
    (dict(pt_stride=0), {}, ti.TI_ERR_INVALID, "empty"),
    (dict(k_pages=None), {}, ti.TI_ERR_INVALID, "null"),
    (dict(v_pages=None), {}, ti.TI_ERR_INVALID, "null"),
    (dict(page_table=None), {}, ti.TI_ERR_INVALID, "null"),
    (dict(k_pages=P + 2), {}, ti.TI_ERR_INVALID, "aligned"),
    (dict(n_pages=2**31 - 1), {}, ti.TI_ERR_UNSUPPORTED, "rows"),
    (dict(pt_stride=2**28), {}, ti.TI_ERR_UNSUPPORTED, "rows"),
    ({}, dict(n_seqs=-1), ti.TI_ERR_INVALID, "negative"),
    ({}, dict(n_tokens=-1), ti.TI_ERR_INVALID, "negative"),
    ({}, dict(start=None), ti.TI_ERR_INVALID, "start"),
    ({}, dict(kv_len=None), ti.TI_ERR_INVALID, "kv_len"),
    ({}, dict(n_seqs=5), ti.TI_ERR_INVALID, "page-table"),
]


@pytest.mark.parametrize("cache, batch, code, word", BAD_CACHES)
def test_every_entry_refuses_bad_caches_and_batches(cache, batch, code, word):
    c, b = kv(**cache), ragged(**batch)
    refused(ti.lib().ti_op_kv_append(C.byref(c), C.byref(b), C.byref(rope()), None, 0, P, 128, P, 128, 0, None, 0,
                                     None), code, word)
    refused(ti.lib().ti_op_paged_prefill(C.byref(c), C.byref(b), None, P, 256, 4, P, 256, None), code, word)
    b.start = None
    if "start" not in batch and batch.get("n_tokens", 0) >= 0 and batch.get("n_seqs", 0) >= 0:
        b.n_tokens = b.n_seqs
        refused(ti.lib().ti_op_paged_decode(C.byref(c), C.byref(b), None, P, 256, 4, P, 256, None), code, word)


@pytest.mark.parametrize("args, word", [
    (dict(k=None), "null"), (dict(v=None), "null"), (dict(ks=127), "stride"), (dict(vs=1), "stride"),
    (dict(q=P, q_out=None), "q_out"), (dict(q=P, q_out=P, heads=0), "q_out"), (dict(q=P, q_out=2 * P, qs=255), "stride"),
    (dict(q=P, q_out=P, qs=256, os=512), "in place"),
])
def test_append_refuses_bad_rows(args, word):
    a = dict(q=None, qs=256, k=P, ks=128, v=P, vs=128, heads=4, q_out=None, os=256)
    a.update(args)
    refused(ti.lib().ti_op_kv_append(C.byref(kv()), C.byref(ragged()), C.byref(rope()), a["q"], a["qs"], a["k"], a["ks"],
                                     a["v"], a["vs"], a["heads"], a["q_out"], a["os"], None), ti.TI_ERR_INVALID, word)


@pytest.mark.parametrize("entry", ["ti_op_paged_prefill", "ti_op_paged_decode"])
@pytest.mark.parametrize("args, code, word", [
    (dict(q=None), ti.TI_ERR_INVALID, "null"), (dict(out=None), ti.TI_ERR_INVALID, "null"),
    (dict(heads=3), ti.TI_ERR_INVALID, "heads"), (dict(heads=0), ti.TI_ERR_INVALID, "heads"),
    (dict(hd=96), ti.TI_ERR_UNSUPPORTED, "head_dim"), (dict(qs=255), ti.TI_ERR_INVALID, "stride"),
    (dict(os=0), ti.TI_ERR_INVALID, "stride"), (dict(form=dict(softcap=-1.0)), ti.TI_ERR_INVALID, "softcap"),
    (dict(form=dict(softcap=float("nan"))), ti.TI_ERR_INVALID, "softcap"),
    (dict(form=dict(scale=float("inf"))), ti.TI_ERR_INVALID, "scale"),
    (dict(form=dict(scale=-0.1)), ti.TI_ERR_INVALID, "scale"),
    (dict(form=dict(softcap=1e-6)), ti.TI_ERR_UNSUPPORTED, "softcap"),
    (dict(form=dict(softcap=1e4)), ti.TI_ERR_UNSUPPORTED, "softcap"),
])
def test_attention_refuses_bad_arguments(entry, args, code, word):
    a = dict(q=P, qs=256, heads=4, out=P, os=256, hd=64, form={})
    a.update(args)
    b = ragged(start=None, n_tokens=2) if entry.endswith("decode") else ragged()
    refused(getattr(ti.lib(), entry)(C.byref(kv(head_dim=a["hd"])), C.byref(b), C.byref(form(**a["form"])), a["q"],
                                     a["qs"], a["heads"], a["out"], a["os"], None), code, word)


def test_decode_refuses_a_ragged_batch():
    refused(ti.lib().ti_op_paged_decode(C.byref(kv()), C.byref(ragged()), None, P, 256, 4, P, 256, None),
            ti.TI_ERR_INVALID, "start")


def test_null_structs_are_refused():
    for entry in (ti.lib().ti_op_paged_prefill, ti.lib().ti_op_paged_decode):
        refused(entry(None, C.byref(ragged(start=None, n_tokens=2)), None, P, 256, 4, P, 256, None), ti.TI_ERR_INVALID,
                "null")
        refused(entry(C.byref(kv()), None, None, P, 256, 4, P, 256, None), ti.TI_ERR_INVALID, "null")
    refused(ti.lib().ti_op_kv_append(C.byref(kv()), None, None, None, 0, P, 128, P, 128, 0, None, 0, None),
            ti.TI_ERR_INVALID, "null")
    refused(ti.lib().ti_op_rope_axes(ti.DTYPE_BF16, P, 128, 2 * P, 128, 5, 2, 64, None, None), ti.TI_ERR_INVALID, "null")


def test_empty_calls_do_nothing():
    # no tokens: nothing to launch, so no device is needed
    assert ti.lib().ti_op_rope_axes(ti.DTYPE_BF16, P, 128, 2 * P, 128, 0, 2, 64, C.byref(rope()), None) == 0
    b = ragged(n_seqs=0, n_tokens=0, start=None, kv_len=None)
    assert ti.lib().ti_op_kv_append(C.byref(kv()), C.byref(b), C.byref(rope()), None, 0, P, 128, P, 128, 0, None, 0,
                                    None) == 0
    assert ti.lib().ti_op_paged_prefill(C.byref(kv()), C.byref(b), None, P, 256, 4, P, 256, None) == 0
    assert ti.lib().ti_op_paged_decode(C.byref(kv()), C.byref(b), None, P, 256, 4, P, 256, None) == 0


@pytest.mark.parametrize("scaling", [None, (1, 8.0, 1.0, 4.0, 8192)])
def test_frequency_table_is_the_engines(scaling):
    ref = np.empty(64, np.float32)
    osc = oracle.RopeScaling(*scaling) if scaling else None
    oracle.lib().orc_rope_freqs(128, 500000.0, C.byref(osc) if osc else None, oracle.ptr(ref))
    np.testing.assert_array_equal(ti.rope_inv_freq(128, 500000.0, ti.RopeScaling(*scaling) if scaling else None), ref)


def test_frequency_table_refuses_bad_arguments():
    out = np.empty(8, np.float32)
    for hd, theta in ((0, 1e4), (7, 1e4), (16, 0.0), (16, -1.0)):
        refused(ti.lib().ti_rope_inv_freq(hd, theta, None, out.ctypes.data_as(C.c_void_p)), ti.TI_ERR_INVALID, "head_dim")
    refused(ti.lib().ti_rope_inv_freq(16, 1e4, None, None), ti.TI_ERR_INVALID, "null")
