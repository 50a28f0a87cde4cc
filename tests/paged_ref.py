"""Plain float64 forms of the serving operators over the paged cache, and how far a
correct kernel may be from them."""
import math

import numpy as np
import torch

import ti_b200 as ti

DT = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
CODE = {"bf16": ti.DTYPE_BF16, "f16": ti.DTYPE_F16, "f32": ti.DTYPE_F32}
HALF_STEP = {d: torch.finfo(t).eps / 2 for d, t in DT.items()}  # one rounding, relative to the value
# below its normal range a type rounds by half its smallest step whatever the value
FLOOR = {d: torch.finfo(t).smallest_normal * torch.finfo(t).eps / 2 for d, t in DT.items()}


def axis_of_pair(half, n_axes, sections, interleaved):
    if n_axes == 1:
        return [0] * half
    if interleaved:
        return [i % n_axes if i // n_axes < sections[i % n_axes] else 0 for i in range(half)]
    return [a for a in range(n_axes) for _ in range(sections[a])]


def rotate(x, angle, rot_dim):
    """x [tokens, heads, hd] float64 by angle [tokens, rot_dim / 2]; and the most an fp32
    evaluation may be off: the reduced angle (fp32, in half turns) is off by half a step of 2^-24
    times pi, cosine and sine by two steps of 2^-24, each product by half a step: under 2^-21
    of |x0| + |x1|."""
    half = rot_dim // 2
    c, s = np.cos(angle)[:, None], np.sin(angle)[:, None]
    x0, x1 = x[..., :half], x[..., half:rot_dim]
    y = np.concatenate([x0 * c - x1 * s, x0 * s + x1 * c, x[..., rot_dim:]], -1)
    off = (np.abs(x0) + np.abs(x1)) * 2.0 ** -21
    return y, np.concatenate([off, off, np.zeros_like(x[..., rot_dim:])], -1)


class Cache:
    """Sequences of (new, length) tokens over shuffled pages; every slot that no sequence
    holds is filled with NaN."""

    def __init__(self, seqs, nkv, hd, dtype, seed=0, std=1.0, pad_tokens=0, spare_rows=0):
        g = torch.Generator().manual_seed(seed)
        self.seqs, self.nkv, self.hd, self.dtype, self.pad = seqs, nkv, hd, dtype, pad_tokens
        self.wide = max(1, max([-(-n // 16) for _, n in seqs], default=1))
        need = sum(-(-n // 16) for _, n in seqs)
        self.n_pages = need + 2
        ids = torch.randperm(self.n_pages, generator=g)[:need].tolist()
        self.rows = torch.randperm(len(seqs) + spare_rows, generator=g)[:len(seqs)].to(torch.int32)
        self.table = torch.full((len(seqs) + spare_rows, self.wide), -1, dtype=torch.int32)
        nan = float("nan")
        self.k = torch.full((self.n_pages, nkv, 16, hd), nan, dtype=DT[dtype])
        self.v = torch.full((self.n_pages, nkv, 16, hd), nan, dtype=DT[dtype])
        self.K, self.V = [], []  # per sequence [length, nkv, hd]
        for s, (_, n) in enumerate(seqs):
            pages = [ids.pop() for _ in range(-(-n // 16))]
            self.table[self.rows[s], :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            kk = (torch.randn(n, nkv, hd, generator=g) * std).to(DT[dtype])
            vv = torch.randn(n, nkv, hd, generator=g).to(DT[dtype])
            self.K.append(kk)
            self.V.append(vv)
            for p, page in enumerate(pages):
                m = min(16, n - p * 16)
                self.k[page, :, :m] = kk[p * 16:p * 16 + m].transpose(0, 1)
                self.v[page, :, :m] = vv[p * 16:p * 16 + m].transpose(0, 1)
        self.starts = np.concatenate([[0], np.cumsum([n for n, _ in seqs])]).astype(np.int32)
        self.tokens = int(self.starts[-1]) + pad_tokens
        self.max_len = max([n for _, n in seqs], default=1)

    def dev(self, decode=False, indirect=True):
        """device tensors and the two structs over them"""
        d = {"k": self.k.cuda(), "v": self.v.cuda(), "table": self.table.cuda(), "rows": self.rows.cuda(),
             "start": torch.from_numpy(self.starts).cuda(),
             "len": torch.tensor([n for _, n in self.seqs], dtype=torch.int32).cuda()}
        d["kv"] = ti.PagedKv(dtype=CODE[self.dtype], n_kv=self.nkv, head_dim=self.hd, k_pages=d["k"].data_ptr(),
                             v_pages=d["v"].data_ptr(), n_pages=self.n_pages, page_table=d["table"].data_ptr(),
                             table_rows=self.table.shape[0], pt_stride=self.wide)
        d["batch"] = ti.Ragged(n_seqs=len(self.seqs), n_tokens=self.tokens,
                               start=None if decode else d["start"].data_ptr(), kv_len=d["len"].data_ptr(),
                               row=d["rows"].data_ptr() if indirect else None, max_len=self.max_len)
        return d

    def read(self, pool, s):
        """[length, nkv, hd] of sequence s out of a pool"""
        n = self.seqs[s][1]
        pages = self.table[self.rows[s]].long()[:-(-n // 16)]
        return pool.cpu()[pages].transpose(1, 2).reshape(-1, self.nkv, self.hd)[:n]


def attend(cache, q, heads, cap=0.0, slopes=None, window=0, prefix=None, doc=None, scale=0.0):
    """float64 rows [tokens, heads, hd] of cache's sequences for q, and the largest error of a
    kernel that rounds the probabilities and the result to the type and computes the rest in
    fp32.  With u = half a step of the type: u |o| for the result, u sum p |v| for the
    probabilities; scores off by dz scale each p by at most 1 + 2 dz.  dz counts fp32 products
    over hd terms, 2^-16 for the exponential and the cap's polynomial (2.1e-7 of the cap) and,
    above a cap of 32, cap 2^-21: tanh as cap - 2 cap / (e^(2u) + 1) with the exponential off by
    2^-22 and the reciprocal by 2^-23 of a term below 2 cap, and one rounding near cap (2^-24)."""
    group, hd = heads // cache.nkv, cache.hd
    u = HALF_STEP[cache.dtype]
    out = np.zeros((q.shape[0], heads, hd))
    tol = np.zeros_like(out)
    scale = scale or 1.0 / math.sqrt(hd)
    qd = q.double().numpy()
    for s, (new, n) in enumerate(cache.seqs):
        if n == 0:
            continue
        K, V = cache.K[s].double().numpy(), cache.V[s].double().numpy()
        t0 = int(cache.starts[s])
        i = np.arange(n - new, n)[:, None]
        j = np.arange(n)[None, :]
        seen = j <= i
        if prefix is not None:
            seen = seen | (j < int(prefix[s]))
        if window > 0:
            seen = seen & (j > i - window)
        if doc is not None:
            seen = seen & (j >= doc[t0:t0 + new, None])
        seen = seen & (i >= 0)
        for h in range(heads):
            k, v = K[:, h // group], V[:, h // group]
            qh = qd[t0:t0 + new, h]
            z = qh @ k.T * scale
            dz = (hd + 8) * 2.0 ** -24 * (np.abs(qh) @ np.abs(k).T * abs(scale))
            if cap:
                z = cap * np.tanh(z / cap)
            if slopes is not None:
                bias = float(slopes[h]) * np.abs(i - j)
                z = z - bias
                dz = dz + np.abs(bias) * 2.0 ** -22
            dz = dz + max(2.0 ** -16, cap * 2.0 ** -21) + np.abs(z) * 2.0 ** -22
            z = np.where(seen, z, -np.inf)
            dz = np.where(seen, dz, 0).max(-1, keepdims=True)
            top = z.max(-1, keepdims=True)
            p = np.where(seen, np.exp(z - np.where(np.isfinite(top), top, 0)), 0)
            tot = p.sum(-1, keepdims=True)
            w = p / np.where(tot == 0, 1, tot)
            o, a = w @ v, w @ np.abs(v)
            out[t0:t0 + new, h] = o
            tiny = FLOOR[cache.dtype] * (1 + seen @ np.abs(v))  # probabilities and results below the type's range
            tol[t0:t0 + new, h] = u * np.abs(o) * 1.01 + (u * 1.01 + 2 * dz) * a + tiny
    return out, tol
