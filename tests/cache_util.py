"""Caches, trees and 64-bit references of the operators on a cache whose rows are not its positions.

A cache is built from its logical rows (one [Hkv, rows, D] pair per sequence); every element that no operator may read holds
NaN, so that a row too many shows.  References are float64 on the CPU, written from the definitions."""
import math
import random

import numpy as np
import torch

HALF_STEP = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8}


class Cache:
    """rows[b]: number of rows that hold data; cap: rows that a block can hold."""

    def __init__(self, seed, rows, Hkv, D, dtype, paged=0, cap=None, spare=0, v_scale=1.0):
        g = torch.Generator().manual_seed(seed)
        self.B, self.Hkv, self.D, self.dtype, self.page = len(rows), Hkv, D, dtype, paged
        self.cap = cap or max(max(rows), 1)
        self.rows = rows
        # logical contents, already of the cache's type
        self.k = [torch.randn(Hkv, r, D, generator=g).to(dtype) for r in rows]
        self.v = [(torch.randn(Hkv, r, D, generator=g) * v_scale).to(dtype) for r in rows]
        rng = random.Random(seed)
        if paged:
            self.max_pages = -(-self.cap // paged) + spare
            used = sum(-(-max(r, 1) // paged) for r in rows)
            self.n_pages = used + 3
            order = list(range(self.n_pages))
            rng.shuffle(order)
            table = np.full((self.B, self.max_pages), -1, np.int32)
            kp = torch.full((self.n_pages, Hkv, paged, D), float("nan"), dtype=dtype)
            vp = kp.clone()
            for b, r in enumerate(rows):
                for i in range(-(-max(r, 1) // paged)):
                    table[b, i] = pg = order.pop()
                    m = min(paged, r - i * paged)
                    if m > 0:
                        kp[pg, :, :m] = self.k[b][:, i * paged:i * paged + m]
                        vp[pg, :, :m] = self.v[b][:, i * paged:i * paged + m]
            self.table_host = table
            self.kd, self.vd, self.table = kp.cuda(), vp.cuda(), torch.from_numpy(table).cuda()
        else:
            self.head_stride = self.cap * D + 8 * rng.randrange(3)
            off, at = [], 8 * rng.randrange(4)
            for _ in range(self.B):
                off.append(at)
                at += Hkv * self.head_stride + 8 * rng.randrange(5)
            kf = torch.full((at + 64,), float("nan"), dtype=dtype)
            vf = kf.clone()
            for b, r in enumerate(rows):
                for h in range(Hkv):
                    s = off[b] + h * self.head_stride
                    kf[s:s + r * D] = self.k[b][h].flatten()
                    vf[s:s + r * D] = self.v[b][h].flatten()
            self.off_host = off
            self.kd, self.vd, self.off = kf.cuda(), vf.cuda(), torch.tensor(off, dtype=torch.int64).cuda()

    def where(self):
        """Keyword arguments of the contiguous calls."""
        return dict(kv_off=self.off, head_stride=self.head_stride, max_seq=self.cap)

    def block(self, t, b, rows=None):
        """Rows 0 .. rows-1 of sequence b of a device array, [Hkv, rows, D] on the CPU."""
        rows = self.rows[b] if rows is None else rows
        t = t.cpu()
        if self.page:
            pages = [int(x) for x in self.table_host[b, : -(-rows // self.page)]] if rows else []
            return torch.cat([t[p] for p in pages], 1)[:, :rows] if pages else torch.zeros(self.Hkv, 0, self.D, dtype=t.dtype)
        return torch.stack([t[self.off_host[b] + h * self.head_stride:][: rows * self.D].view(rows, self.D) for h in range(self.Hkv)])


def random_tree(rng, n, window=4):
    """Ancestor sets (bit sets) and depths; a parent is among the `window` tokens before."""
    sets, depth = [1], [0]
    for i in range(1, n):
        p = rng.randint(max(0, i - window), i - 1)
        sets.append(sets[p] | 1 << i)
        depth.append(depth[p] + 1)
    return sets, depth


def mask_words(sets_per_seq, n):
    words = (n + 63) // 64
    a = np.zeros((len(sets_per_seq), n, words), np.uint64)
    for b, sets in enumerate(sets_per_seq):
        for i, x in enumerate(sets):
            for w in range(words):
                a[b, i, w] = (x >> (64 * w)) & (2**64 - 1)
    return torch.from_numpy(a.view(np.int64)).cuda()


def attend(q, k, v, see, scale):
    """q [n, Hq, D], k, v [Hkv, rows, D] (float64), see [n, rows] bool -> out [n, Hq, D], m, l [n, Hq], weights [n, Hq, rows]
    and the error scale of the scores: scale * max_r sum_d |q_d k_rd| over the rows that are seen."""
    n, Hq, D = q.shape
    Hkv, L = k.shape[0], k.shape[1]
    G = Hq // Hkv
    qq = q.view(n, Hkv, G, D)
    kk, vv = torch.nan_to_num(k), v
    s = torch.einsum("ihgd,hrd->ihgr", qq, kk) * scale
    mag = torch.einsum("ihgd,hrd->ihgr", qq.abs(), kk.abs()) * scale
    hide = ~see[:, None, None, :]
    s = s.masked_fill(hide, -math.inf)
    mag = mag.masked_fill(hide, 0.0)
    if L == 0:
        z = torch.zeros(n, Hq, dtype=torch.float64)
        return torch.zeros_like(q), z - math.inf, z, torch.zeros(n, Hq, 0, dtype=torch.float64), 0.0
    m = s.amax(-1)
    e = torch.exp(s - torch.where(m == -math.inf, torch.zeros_like(m), m)[..., None])
    l = e.sum(-1)
    w = e / torch.where(l == 0, torch.ones_like(l), l)[..., None]
    out = torch.einsum("ihgr,hrd->ihgd", w, vv)
    return out.reshape(n, Hq, D), m.view(n, Hq), l.view(n, Hq), w.view(n, Hq, L), float(mag.max())


def attention_tolerance(D, rows, mag, v_max, out_dtype, wide=False):
    """How far an output may be off.  u = 2^-24.  A score is a sum of D products in 32 bits, then scaled: off by at most
    (D + 3) u mag, which moves every weight by that factor (numerator and sum: twice), the exponential by 2^-22; the sums over
    the rows add rows * u.  A weight is split into three bf16 terms for 32-bit results (2^-26 left) and two for bf16 results
    (2^-17 left); bf16 results of more than 32 query rows per KV head (wide) round it once, numerator and sum by 2^-8 each.
    The result is a weighted mean of values of at most v_max."""
    u = 2.0 ** -24
    rel = 2 * ((D + 3) * u * mag + 2.0 ** -22) + (rows + 2) * u
    rel += 2.0 ** -26 if out_dtype == torch.float32 else (2.0 ** -7 if wide else 2.0 ** -17)
    return rel * v_max


def assert_within(got, want, absolute, out_dtype, what):
    got, want = got.double(), want.double()
    assert torch.isfinite(got).all(), f"{what}: non-finite values"
    off = (got - want).abs() - HALF_STEP[out_dtype] * want.abs() * (1 + 2.0 ** -7)
    assert float(off.max()) <= absolute, f"{what}: {float(off.max()):.3e} above the rounding, {absolute:.3e} allowed"
