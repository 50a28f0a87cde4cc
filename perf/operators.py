"""Serving operators over the paged KV cache, as cases to time and compare.

Four operators make one attention step of a served model: rotating q and k by their positions on one
or several axes (`ti_op_rope_axes`, also used alone by encoders that keep no cache), the same rotation
with the append of k and v to the pages (`ti_op_kv_append`), attention of a ragged batch of new tokens
over the pages (`ti_op_paged_prefill`) and its form for one new token a sequence
(`ti_op_paged_decode`).  The attention takes scores capped by a tanh, a bias that falls with the
distance, a sliding window, a prefix that sees itself both ways, and documents packed in a sequence.

With `own` false, `run` computes them from elementary torch operations in 32 bits (angles in 64); with
`own` true it calls the library through its Python binding.
"""
import ctypes
import math
import os
import random
import sys

import torch

own = False

PAGE = 16  # tokens of a page
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
THETA = 500000.0


# ---------------------------------------------------------------- cases
def _rope(name, tokens, heads, head_dim, dtype, axes, interleaved, far):
    return {"name": name, "op": "rope", "tokens": tokens, "heads": heads, "head_dim": head_dim, "dtype": dtype,
            "axes": axes, "interleaved": interleaved, "far": far}


def _paged(name, op, heads, kv_heads, head_dim, dtype, seqs, new, length, mix, **more):
    """`seqs` sequences with up to `new` new tokens and `length` positions in all; `mix` 0: every
    sequence at the most, else the seed of the spread of their lengths."""
    c = {"name": name, "op": op, "heads": heads, "kv_heads": kv_heads, "head_dim": head_dim, "dtype": dtype,
         "seqs": seqs, "new": new, "len": length, "mix": mix}
    if op == "append":
        return {**c, "axes": 1, "interleaved": False, **more}
    return {**c, "cap": 0.0, "window": 0, "alibi": False, "prefix": 0, "docs": 0, **more}


def listed():
    return [
        # the patches of one picture (27 x 37) in a vision encoder, rotated by row and column
        _rope("rope_picture", 999, 16, 64, "f16", 2, False, 64),
        # the queries of a long video prompt: time, height, width in turn over the pairs
        _rope("rope_video", 16384, 32, 128, "bf16", 3, True, 100000),
        # one decode step of one sequence: the launch is all there is
        _paged("append_one", "append", 32, 4, 64, "bf16", 1, 1, 130, 0),
        # one decode step of a full batch, 70B head shape
        _paged("append_batch", "append", 64, 8, 128, "bf16", 64, 1, 640, 3),
        # prompts of ragged lengths with pictures in them, three axes
        _paged("append_prompts", "append", 28, 4, 128, "f16", 9, 2047, 2500, 5, axes=3),
        # short prompts of many users in one launch, wide heads, capped scores
        _paged("prefill_short", "prefill", 16, 16, 256, "bf16", 11, 300, 331, 7, cap=50.0),
        # one long prompt, capped, in a layer with a window
        _paged("prefill_long", "prefill", 32, 8, 128, "bf16", 1, 8192, 8192, 0, cap=30.0, window=4096),
        # distance bias, and prefixes (a picture, an instruction) that see themselves both ways
        _paged("prefill_prefix", "prefill", 32, 4, 64, "f16", 4, 1500, 1500, 9, alibi=True, prefix=700),
        # a few new tokens over a long cache with packed documents: little work in rows, much in length
        _paged("prefill_chunk", "prefill", 32, 8, 128, "bf16", 1, 33, 60001, 0, docs=50000),
        # the first tokens of one user
        _paged("decode_one", "decode", 32, 4, 64, "bf16", 1, 1, 513, 0, cap=50.0),
        # a served batch of ragged lengths, distance bias
        _paged("decode_batch", "decode", 32, 8, 128, "f16", 32, 1, 8191, 11, alibi=True),
        # two users far into a long context
        _paged("decode_long", "decode", 64, 8, 128, "bf16", 2, 1, 131071, 0, cap=30.0),
    ]


def _log(rng, lo, hi):
    """A whole number between lo and hi, even over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rope", "append", "prefill", "prefill", "decode", "decode"])
    if op == "rope":
        heads, head_dim = rng.choice([(16, 64), (16, 128), (32, 128), (28, 128), (16, 256)])
        c = _rope("", _log(rng, 1, 16384 * 4096 // max(4096, heads * head_dim)), heads, head_dim,
                  rng.choice(["bf16", "f16", "f32"] if heads * head_dim < 4096 else ["bf16", "f16"]),
                  rng.randint(1, 4), rng.random() < 0.5, _log(rng, 64, 200000))
        del c["name"]
        return c
    heads, kv_heads, head_dim = rng.choice([(32, 8, 128), (28, 4, 128), (32, 4, 64), (64, 8, 128), (16, 16, 256),
                                            (8, 1, 256), (12, 12, 64)])
    dtype = rng.choice(["bf16", "f16"])
    mix = rng.randint(1, 1 << 20)
    if op == "append":
        seqs = _log(rng, 1, 64)
        new = _log(rng, 1, max(1, 8192 // seqs))
        c = _paged("", op, heads, kv_heads, head_dim, dtype, seqs, new, new + _log(rng, 1, 2000), mix,
                   axes=rng.randint(1, 3), interleaved=rng.random() < 0.5)
    elif op == "prefill":
        seqs = _log(rng, 1, 16)
        new = _log(rng, 2, 4096 // seqs)
        room = 10 ** 11 // (seqs * heads * head_dim * new)  # no more work than the long prompt
        length = new + _log(rng, 1, max(1, min(32768, room) - new))
        c = _paged("", op, heads, kv_heads, head_dim, dtype, seqs, new, length, mix)
    else:
        seqs = _log(rng, 1, 64)
        c = _paged("", op, heads, kv_heads, head_dim, dtype, seqs, 1,
                   _log(rng, 1, 2 ** 28 // (seqs * kv_heads * head_dim)), mix)
    if op != "append":
        c["cap"] = rng.choice([0.0, 30.0, 50.0])
        c["window"] = rng.choice([0, 0, _log(rng, 1, c["len"])])
        c["alibi"] = rng.random() < 0.4
        c["prefix"] = rng.choice([0, 0, _log(rng, 1, c["len"])])
        c["docs"] = rng.choice([0, 0, _log(rng, 1, c["len"])])
    del c["name"]
    return c


def _lengths(case):
    """(new tokens, positions in all) of every sequence, from the case alone."""
    r = random.Random(case["mix"])
    new, total = [case["new"]], [case["len"]]
    for _ in range(case["seqs"] - 1):
        n = case["new"] if case["mix"] == 0 else _log(r, 1, case["new"])
        new.append(n)
        total.append(case["len"] if case["mix"] == 0 else r.randint(n, case["len"]))
    return new, total


def _prefixes(case):
    r = random.Random(case["mix"] + 1)
    return [r.randint(0, case["prefix"]) for _ in range(case["seqs"])]


def _sections(case):
    """Pairs of each axis: as even as they come, the first axis takes the rest."""
    half, n = case["head_dim"] // 2, case["axes"]
    return [half - (n - 1) * (half // n)] + [half // n] * (n - 1)


def _axis_of_pair(case):
    n, sections = case["axes"], _sections(case)
    if case["interleaved"]:
        return [i % n if i // n < sections[i % n] else 0 for i in range(case["head_dim"] // 2)]
    return [a for a in range(n) for _ in range(sections[a])]


# ---------------------------------------------------------------- inputs
def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt, hd = DTYPES[case["dtype"]], case["head_dim"]

    def normal(*shape, std=1.0):
        return torch.randn(*shape, generator=g, device="cuda", dtype=dt).mul_(std)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=g, device="cuda", dtype=torch.int32)

    s = {"case": case}
    if case["op"] in ("rope", "append"):
        s["inv_freq"] = torch.tensor([THETA ** (-2.0 * i / hd) for i in range(hd // 2)], device="cuda")
        s["axis"] = torch.tensor(_axis_of_pair(case), device="cuda")
    if case["op"] == "rope":
        s["x"] = normal(case["tokens"], case["heads"], hd)
        s["pos"] = whole(0, case["far"], case["axes"], case["tokens"])
        s["out"] = torch.empty_like(s["x"])
        return s

    heads, nkv, seqs = case["heads"], case["kv_heads"], case["seqs"]
    new, total = _lengths(case)
    tokens, starts = sum(new), [sum(new[:i]) for i in range(seqs + 1)]
    wide = -(-case["len"] // PAGE)
    need = [-(-t // PAGE) for t in total]
    n_pages = sum(need) + 3
    ids = torch.randperm(n_pages, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(seqs, wide, dtype=torch.int32, device="cuda")
    at = torch.arange(wide, device="cuda") < torch.tensor(need, device="cuda")[:, None]
    table[at] = ids[:sum(need)]  # scattered over the pool, as after a while of serving
    s.update(tokens=tokens, starts=starts, table=table, n_pages=n_pages,
             start=torch.tensor(starts, dtype=torch.int32, device="cuda"),
             kv_len=torch.tensor(total, dtype=torch.int32, device="cuda"),
             k_pages=normal(n_pages, nkv, PAGE, hd), v_pages=normal(n_pages, nkv, PAGE, hd))
    s["seq_of"] = torch.repeat_interleave(torch.arange(seqs, device="cuda"), torch.tensor(new, device="cuda"))
    s["at"] = (torch.arange(tokens, device="cuda") - s["start"][s["seq_of"]]
               + (s["kv_len"] - torch.tensor(new, device="cuda", dtype=torch.int32))[s["seq_of"]])
    if case["op"] == "append":
        s["qkv"] = normal(tokens, (heads + 2 * nkv) * hd)  # the projections' output, one row a token
        # with one axis the position in the cache; else a picture's row and column from its first token on
        s["pos"] = torch.stack([s["at"].to(torch.int32)] + [whole(0, 64, tokens) + s["at"].to(torch.int32)
                                                            for _ in range(case["axes"] - 1)])
        s["out"] = torch.empty(tokens, heads, hd, device="cuda", dtype=dt)
        return s
    s["q"] = normal(tokens, heads, hd, std=2.0)
    s["out"] = torch.empty_like(s["q"])
    s["slopes"] = torch.tensor([2.0 ** (-8.0 * (h + 1) / heads) for h in range(heads)], device="cuda")
    s["prefix"] = torch.tensor(_prefixes(case), dtype=torch.int32, device="cuda")
    s["doc"] = (s["at"] - s["at"] % max(1, case["docs"])).to(torch.int32)
    return s


# ---------------------------------------------------------------- plain forms
def _rotate(x, pos, s):
    """x [tokens, heads, hd] rotated in 32 bits by angles made in 64."""
    half = x.shape[-1] // 2
    angle = pos[s["axis"]].t().double() * s["inv_freq"].double()  # [tokens, half]
    c, n = angle.cos().float()[:, None], angle.sin().float()[:, None]
    x0, x1 = x[..., :half].float(), x[..., half:].float()
    return torch.cat([x0 * c - x1 * n, x0 * n + x1 * c], dim=-1).to(x.dtype)


def _append(s):
    case = s["case"]
    heads, nkv, hd = case["heads"], case["kv_heads"], case["head_dim"]
    rows = s["qkv"].view(s["tokens"], heads + 2 * nkv, hd)
    page = s["table"][s["seq_of"], s["at"] // PAGE].long()
    s["k_pages"][page, :, s["at"] % PAGE] = _rotate(rows[:, heads:heads + nkv], s["pos"], s)
    s["v_pages"][page, :, s["at"] % PAGE] = rows[:, heads + nkv:]
    return {"q": _rotate(rows[:, :heads], s["pos"], s), "k_pages": s["k_pages"], "v_pages": s["v_pages"]}


def _range(s):
    """The positions [lo, hi) that each new token attends to."""
    case, i = s["case"], s["at"]
    lo = torch.zeros_like(i)
    if case["window"]:
        lo = torch.maximum(lo, i - case["window"] + 1)
    if case["docs"]:
        lo = torch.maximum(lo, s["doc"])
    hi = i + 1
    if case["prefix"]:
        hi = torch.maximum(hi, s["prefix"][s["seq_of"]])
    return lo, torch.minimum(hi, s["kv_len"][s["seq_of"]])


def _attention(s):
    """All sequences padded to the longest: scores, mask, softmax and product in 32 bits."""
    case = s["case"]
    heads, nkv, hd, seqs, n, L = (case[k] for k in ("heads", "kv_heads", "head_dim", "seqs", "new", "len"))
    group, dev = heads // nkv, s["q"].device
    pages = s["table"].long()
    j = torch.arange(L, device=dev)

    def cached(pool):
        return pool[pages].transpose(1, 2).reshape(seqs, nkv, -1, hd)[:, :, :L].float()

    k, v = cached(s["k_pages"]), cached(s["v_pages"])
    v = torch.where((j < s["kv_len"][:, None])[:, None, :, None], v, 0.0)
    t = s["start"][:-1, None].long() + torch.arange(n, device=dev)  # [seqs, n] rows of q
    real = t < s["start"][1:, None]
    t = torch.where(real, t, 0)
    q = s["q"][t].view(seqs, n, nkv, group, hd).permute(0, 2, 3, 1, 4).reshape(seqs, nkv, group * n, hd).float()
    z = (q @ k.transpose(-1, -2)).view(seqs, nkv, group, n, L).mul_(1.0 / math.sqrt(hd))
    if case["cap"]:
        z = z.div_(case["cap"]).tanh_().mul_(case["cap"])
    if case["alibi"]:
        far = (s["at"][t][:, :, None] - j).abs().float()
        z -= s["slopes"].view(nkv, group, 1, 1) * far[:, None, None]
    lo, hi = _range(s)
    seen = (j >= lo[t][:, :, None]) & (j < hi[t][:, :, None]) & real[:, :, None]
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    p = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    o = p.view(seqs, nkv, group * n, L) @ v
    o = o / torch.where(total == 0, 1.0, total).view(seqs, nkv, group * n, 1)
    o = o.view(seqs, nkv, group, n, hd).permute(0, 3, 1, 2, 4).reshape(seqs, n, heads, hd)
    return o[real].to(s["q"].dtype)


# ---------------------------------------------------------------- the library's operators
def _binding():
    at = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "tensor-inference_b200")
    if at not in sys.path:
        sys.path.insert(0, at)
    import ti_b200

    return ti_b200


def _handles(s):
    """The descriptions of cache, batch, rotation and scores that a program makes once for its buffers."""
    ti, case = _binding(), s["case"]
    dtype = {"bf16": ti.DTYPE_BF16, "f16": ti.DTYPE_F16, "f32": ti.DTYPE_F32}[case["dtype"]]
    h = {"ti": ti, "lib": ti.lib(), "dtype": dtype}
    if case["op"] in ("rope", "append"):
        sections = _sections(case) + [0] * (4 - case["axes"])
        h["rope"] = ti.RopeAxes(rot_dim=case["head_dim"], inv_freq=s["inv_freq"].data_ptr(), n_axes=case["axes"],
                                sections=(ctypes.c_int * 4)(*sections), interleaved=int(case["interleaved"]),
                                pos=s["pos"].data_ptr(), pos_stride=s["pos"].stride(0))
    if case["op"] == "rope":
        return h
    h["kv"] = ti.PagedKv(dtype=dtype, n_kv=case["kv_heads"], head_dim=case["head_dim"],
                         k_pages=s["k_pages"].data_ptr(), v_pages=s["v_pages"].data_ptr(), n_pages=s["n_pages"],
                         page_table=s["table"].data_ptr(), table_rows=case["seqs"], pt_stride=s["table"].stride(0))
    h["batch"] = ti.Ragged(n_seqs=case["seqs"], n_tokens=s["tokens"],
                           start=None if case["op"] == "decode" else s["start"].data_ptr(),
                           kv_len=s["kv_len"].data_ptr(), row=None, max_len=case["len"])
    if case["op"] != "append":
        h["form"] = ti.AttnForm(scale=0.0, softcap=case["cap"],
                                slopes=s["slopes"].data_ptr() if case["alibi"] else None,
                                sliding_window=case["window"],
                                prefix=s["prefix"].data_ptr() if case["prefix"] else None,
                                doc_start=s["doc"].data_ptr() if case["docs"] else None)
    return h


def _library(s):
    if "handles" not in s:
        s["handles"] = _handles(s)
    h, case, ref = s["handles"], s["case"], ctypes.byref
    ti, lib, stream = h["ti"], h["lib"], torch.cuda.current_stream().cuda_stream
    heads, hd = case["heads"], case["head_dim"]
    if case["op"] == "rope":
        ti.check(lib.ti_op_rope_axes(h["dtype"], s["x"].data_ptr(), s["x"].stride(0), s["out"].data_ptr(),
                                     s["out"].stride(0), case["tokens"], heads, hd, ref(h["rope"]), stream))
        return s["out"]
    if case["op"] == "append":
        row, size, base = s["qkv"].stride(0), s["qkv"].element_size(), s["qkv"].data_ptr()
        k = base + heads * hd * size
        ti.check(lib.ti_op_kv_append(ref(h["kv"]), ref(h["batch"]), ref(h["rope"]), base, row, k, row,
                                     k + case["kv_heads"] * hd * size, row, heads, s["out"].data_ptr(),
                                     s["out"].stride(0), stream))
        return {"q": s["out"], "k_pages": s["k_pages"], "v_pages": s["v_pages"]}
    op = lib.ti_op_paged_decode if case["op"] == "decode" else lib.ti_op_paged_prefill
    ti.check(op(ref(h["kv"]), ref(h["batch"]), ref(h["form"]), s["q"].data_ptr(), s["q"].stride(0), heads,
                s["out"].data_ptr(), s["out"].stride(0), stream))
    return s["out"]


def run(state):
    if own:
        return _library(state)
    case = state["case"]
    if case["op"] == "rope":
        return _rotate(state["x"], state["pos"], state)
    if case["op"] == "append":
        return _append(state)
    return _attention(state)


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size, hd, heads = (4 if case["dtype"] == "f32" else 2), case["head_dim"], case["heads"]
    if case["op"] == "rope":
        n = case["tokens"] * heads * hd
        return {"bytes": 2 * n * size + 4 * case["tokens"] * case["axes"] + 2 * hd, "flops": 3 * n}
    nkv = case["kv_heads"]
    new, total = _lengths(case)
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": tokens * (2 * heads + 4 * nkv) * hd * size + 4 * tokens * case["axes"],
                "flops": 3 * tokens * (heads + nkv) * hd}
    pairs = read = 0
    for n, t, prefix in zip(new, total, _prefixes(case)):
        first = None
        for i in range(t - n, t):
            lo = max(0, i - case["window"] + 1 if case["window"] else 0, i - i % case["docs"] if case["docs"] else 0)
            hi = min(t, max(i + 1, prefix if case["prefix"] else 0))
            pairs += hi - lo
            first = lo if first is None else min(first, lo)
        read += t - first
    return {"bytes": 2 * tokens * heads * hd * size + 2 * read * nkv * hd * size, "flops": 4 * pairs * heads * hd}


# ---------------------------------------------------------------- from the definition, in 64 bits
def _turned(x, pos, case):
    """Every pair of x [tokens, heads, hd] as a complex number times e^(i angle)."""
    half, n = x.shape[-1] // 2, case["axes"]
    freq = torch.tensor([THETA ** (-2.0 * i / x.shape[-1]) for i in range(half)]).double().to(x.device)
    sections, axis = _sections(case), []
    for i in range(half):
        if case["interleaved"]:
            axis.append(i % n if i // n < sections[i % n] else 0)
        else:
            axis.append(next(a for a in range(n) if i < sum(sections[:a + 1])))
    angle = torch.stack([pos[a].double() * freq[i] for i, a in enumerate(axis)], dim=1)
    z = torch.complex(x[..., :half].double(), x[..., half:].double()) * torch.polar(torch.ones_like(angle), angle)[:, None]
    return torch.cat([z.real, z.imag], dim=-1)


def exact(case, seed):
    s = prepare(case, seed)
    heads, hd = case["heads"], case["head_dim"]
    if case["op"] == "rope":
        return _turned(s["x"], s["pos"], case)
    nkv = case["kv_heads"]
    new, total = _lengths(case)
    if case["op"] == "append":
        x = s["qkv"].view(-1, heads + 2 * nkv, hd)
        q, k, v = _turned(x[:, :heads], s["pos"], case), _turned(x[:, heads:heads + nkv], s["pos"], case), x[:, heads + nkv:]
        kp, vp = s["k_pages"].double(), s["v_pages"].double()
        t = 0
        for b in range(case["seqs"]):
            for i in range(total[b] - new[b], total[b]):
                page = s["table"][b, i // PAGE]
                kp[page, :, i % PAGE], vp[page, :, i % PAGE] = k[t], v[t].double()
                t += 1
        return {"q": q, "k_pages": kp, "v_pages": vp}
    out = torch.zeros(sum(new), heads, hd, dtype=torch.float64, device="cuda")
    prefixes, t0 = _prefixes(case), 0
    for b in range(case["seqs"]):
        j = torch.arange(total[b], device="cuda")
        page = s["table"][b, j // PAGE].long()
        for r in range(0, new[b], 1024):
            rows = torch.arange(r, min(new[b], r + 1024), device="cuda")
            i = (rows + total[b] - new[b])[:, None]
            seen = j <= i
            if case["prefix"]:
                seen = seen | (j < prefixes[b])
            if case["window"]:
                seen = seen & (j > i - case["window"])
            if case["docs"]:
                seen = seen & (j >= i // case["docs"] * case["docs"])
            for h in range(heads):
                k, v = (s[w][page, h * nkv // heads, j % PAGE].double() for w in ("k_pages", "v_pages"))
                z = s["q"][t0 + rows, h].double() @ k.T / math.sqrt(hd)
                if case["cap"]:
                    z = case["cap"] * torch.tanh(z / case["cap"])
                if case["alibi"]:
                    z = z - 2.0 ** (-8.0 * (h + 1) / heads) * (i - j).abs()
                out[t0 + rows, h] = torch.softmax(z.masked_fill(~seen, -math.inf), dim=-1) @ v
        t0 += new[b]
    return out
