"""Turns of a conversation batch as a server takes them, with every operator of the cache in its place: drafted trees are rotated at
their depths and appended, verified in one pass, their accepted paths kept, the next token attended with scores, and the cache cut to
its budget -- after which the rows are no longer the positions.  Each step is checked in 64 bits against the state before it."""
import math
import random

import pytest
import torch

import cache_util as U
from nimllm_b200 import attention as A
from test_gpu_kv_compact import evict_rows
from test_gpu_rope_at import turned

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16
B, N, HQ, HKV, D, KEEP, CAP, TABLE = 4, 7, 6, 2, 64, 40, 64, 200
LENS = [30, 0, 1, 39]
TREES = [U.random_tree(random.Random(s), N) for s in range(B)]
N_NEW = [7, 7, 3, 5]
PATHS = [[0, 2, 5], [1], [], [0, 1, 2, 3, 4]]         # the operator only asks that they rise


class Turn:
    def __init__(self, act, cache_dtype, pool):
        g = torch.Generator().manual_seed(11)
        self.act, self.pool = act, pool
        if pool:
            self.k, self.v, self.table = pool.k(1), pool.v(1), pool.table()
            self.k.zero_(), self.v.zero_()
            self.where, self.paged = (self.k, self.v, self.table), True
        else:
            self.k, self.v = (torch.zeros(B, HKV, CAP, D, dtype=cache_dtype, device="cuda") for _ in range(2))
            self.paged = False
            self.strides = dict(seq_stride=HKV * CAP * D, head_stride=CAP * D, max_seq=CAP)
        self.cos, self.sin = A.rope_tables_scaled(TABLE, D // 2, 10000.0, kind="none")
        depth = torch.tensor([[t[1][i] if i < n else -10**6 for i in range(N)] for t, n in zip(TREES, N_NEW)], dtype=torch.int32)
        self.depth = depth.cuda()
        self.mask = U.mask_words([t[0] for t in TREES], N)
        self.n_new = torch.tensor(N_NEW, dtype=torch.int32).cuda()
        m = max(map(len, PATHS))
        self.path = torch.tensor([p + [0] * (m - len(p)) for p in PATHS], dtype=torch.int32).cuda()
        self.n_path = torch.tensor([len(p) for p in PATHS], dtype=torch.int32).cuda()
        self.len = torch.tensor(LENS, dtype=torch.int32).cuda()
        self.at = self.len + 50                                          # positions run ahead of the rows
        self.score = torch.zeros(B, HKV, CAP, device="cuda")
        for b, L in enumerate(LENS):                                     # what the conversations hold already
            for t in (self.k, self.v):
                x = torch.randn(HKV, CAP, D, generator=g).to(cache_dtype).cuda()
                for r in range(L):
                    if pool:
                        t[int(pool.table_host()[b, r // 32]), :, r % 32] = x[:, r]
                    else:
                        t[b, :, r] = x[:, r]
            self.score[b, :, :L] = torch.rand(HKV, L, generator=g).cuda()
        new = lambda n, h: torch.randn(B, n, h * D, generator=g).to(act).cuda()
        self.q, self.kn, self.vn = new(N, HQ), new(N, HKV), new(N, HKV)
        self.q1, self.k1, self.v1 = new(1, HQ), new(1, HKV), new(1, HKV)
        self.out, self.out1 = torch.zeros(B, N, HQ * D, dtype=act, device="cuda"), torch.zeros(B, HQ * D, dtype=act, device="cuda")
        self.kept = torch.zeros(B, HKV, KEEP, dtype=torch.int32, device="cuda")

    def append(self, q, k, v, pos):
        kw = dict(n_head=HQ, n_kv_head=HKV, head_dim=D, pos=pos, row0=self.len)
        if self.paged:
            return A.rope_append_at_paged(q, k, v, self.cos, self.sin, *self.where, **kw)[0]
        return A.rope_append_at(q, k, v, self.cos, self.sin, k_cache=self.k, v_cache=self.v, **self.strides, **kw)[0]

    def run(self, look=lambda *a: None):
        """One turn, all of it on the device."""
        heads = dict(n_kv_head=HKV, head_dim=D)
        pos = self.at[:, None] + self.depth
        look("before")
        q = self.append(self.q, self.kn, self.vn, pos)
        look("append", self.q, self.kn, self.vn, q, pos, N_NEW)
        tree = dict(n_head=HQ, max_len=CAP, seq_len=self.len, n_new=self.n_new, tree_mask=self.mask, out=self.out, **heads)
        if self.paged:
            A.decode_tree_paged(q, *self.where, **tree)
        else:
            A.decode_tree(q, self.k, self.v, **self.strides, **tree)
        look("tree", q)
        accept = dict(path=self.path, n_path=self.n_path, seq_len=self.len, n_draft=N, new_len=self.len, **heads)
        if self.paged:
            A.kv_accept_paged(*self.where, **accept)
        else:
            A.kv_accept(self.k, self.v, **self.strides, **accept)
        look("accept")
        self.at += self.n_path
        one = self.append(self.q1, self.k1, self.v1, self.at[:, None].contiguous())
        look("append", self.q1, self.k1, self.v1, one, self.at[:, None], [1] * B)
        self.len += 1
        self.at += 1
        scored = dict(n_head=HQ, max_len=CAP, seq_len=self.len, decay=0.5, out=self.out1, **heads)
        if self.paged:
            A.decode_scored_paged(one.view(B, HQ * D), *self.where, self.score, **scored)
        else:
            A.decode_scored(one.view(B, HQ * D), self.k, self.v, self.score, **self.strides, **scored)
        look("scored", one)
        evict = dict(score=self.score, seq_len=self.len, keep=KEEP, max_len=CAP, n_sink=2, n_recent=8, kept=self.kept, new_len=self.len, **heads)
        if self.paged:
            A.kv_evict_paged(*self.where, **evict)
        else:
            A.kv_evict(self.k, self.v, **self.strides, **evict)
        look("evict")

    def rows(self, b, n):
        """K and V rows 0 .. n - 1 of sequence b, float64."""
        if self.paged:
            pages = self.table[b, : -(-n // 32)].long()
            return [t[pages].transpose(0, 1).reshape(HKV, -1, D)[:, :n].double().cpu() for t in (self.k, self.v)]
        return [t[b, :, :n].double().cpu() for t in (self.k, self.v)]

    def state(self):
        return [x.clone() for x in (self.len, self.at, self.score, self.k, self.v, self.out, self.out1, self.kept)]


class Look:
    """Checks a step against the rows, lengths and scores before it."""

    def __init__(self, t):
        self.t = t

    def __call__(self, step, *a):
        t = self.t
        torch.cuda.synchronize()
        L = t.len.tolist()
        rows = [t.rows(b, CAP if not t.paged else t.pool.seq_rows(b)) for b in range(B)]
        score = t.score.double().cpu()
        if step == "append":
            q, k, v, got, pos, count = a
            for b in range(B):
                n = count[b]
                for x, y, h in ((q, got[b, :n].view(n, HQ, D), HQ), (k, rows[b][0][:, L[b]:L[b] + n].transpose(0, 1), HKV)):
                    want, mag = turned(x[b, :n].double().cpu().view(n, h, D), t.cos.cpu(), t.sin.cpu(), pos[b, :n].long().cpu(), "half")
                    half = max(U.HALF_STEP[t.act], U.HALF_STEP[t.k.dtype])
                    off = (y.double().cpu() - want).abs() - half * want.abs() * (1 + 2.0 ** -7) - 3 * 2.0 ** -24 * mag
                    assert float(off.max()) <= 0
                assert torch.equal(rows[b][1][:, L[b]:L[b] + n], v[b, :n].to(t.k.dtype).double().cpu().view(n, HKV, D).transpose(0, 1))
                assert torch.equal(rows[b][0][:, :L[b]], self.old[b][0][:, :L[b]])
        elif step == "tree":
            for b in range(B):
                n, total = N_NEW[b], L[b] + N_NEW[b]
                see = torch.ones(n, total, dtype=torch.bool)
                for i in range(n):
                    see[i, L[b]:] = torch.tensor([TREES[b][0][i] >> j & 1 for j in range(n)], dtype=torch.bool)
                k, v = (x[:, :total] for x in rows[b])
                want, _, _, _, mag = U.attend(a[0][b, :n].double().cpu().view(n, HQ, D), k, v, see, 1 / math.sqrt(D))
                U.assert_within(t.out[b, :n].cpu().view(n, HQ, D), want, U.attention_tolerance(D, total, mag, float(v.abs().max()), t.act), t.act, f"tree {b}")
                assert (t.out[b, n:] == 0).all()
        elif step == "accept":
            for b in range(B):
                at = self.L[b]
                assert L[b] == at + len(PATHS[b])
                for now, old in zip(rows[b], self.old[b]):
                    assert torch.equal(now[:, :L[b]], old[:, list(range(at)) + [at + x for x in PATHS[b]]])
        elif step == "scored":
            for b in range(B):
                k, v = (x[:, :L[b]] for x in rows[b])
                want, _, _, w, mag = U.attend(a[0][b].double().cpu().view(1, HQ, D), k, v, torch.ones(1, L[b], dtype=torch.bool), 1 / math.sqrt(D))
                U.assert_within(t.out1[b].cpu().view(1, HQ, D), want, U.attention_tolerance(D, L[b], mag, float(v.abs().max()), t.act), t.act, f"scored {b}")
                add = w[0].view(HKV, HQ // HKV, -1).sum(1)
                full = add + 0.5 * self.score[b, :, :L[b]]
                tol = U.attention_tolerance(D, L[b], mag, 1.0, F) * float(add.max()) + (HQ // HKV + 3) * 2.0 ** -24 * float(full.max())
                assert float((score[b, :, :L[b]] - full).abs().max()) <= tol
        elif step == "evict":
            for b in range(B):
                n = self.L[b]
                assert L[b] == min(n, KEEP)
                for h in range(HKV):
                    keep = evict_rows(self.score[b, h, :n].float(), n, KEEP, 2, 8)
                    assert t.kept[b, h].tolist() == keep + [-1] * (KEEP - len(keep))
                    for now, old in zip(rows[b], self.old[b]):
                        assert torch.equal(now[h, :L[b]], old[h, keep])
        self.old, self.L, self.score = rows, L, score


def _make(act, cache_dtype, paged):
    pool = None
    if paged:
        pool = A.PagedKvPool(2, B * 2 + 1, 32, HKV, D, B, 2, dtype=cache_dtype)
        for b in range(B):
            pool.reserve(b, CAP)
        pool.sync()
    return Turn(act, cache_dtype, pool), pool


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("act,cache_dtype", [(F, F), (F, H), (H, H)])
def test_turns(act, cache_dtype, paged):
    t, pool = _make(act, cache_dtype, paged)
    look = Look(t)
    for _ in range(4):
        t.run(look)
    assert t.len.tolist() == [min(40, L + 4 * (len(p) + 1)) for L, p in zip(LENS, PATHS)]
    if pool:
        free = pool.free_pages
        for b, L in enumerate(t.len.tolist()):
            pool.shrink(b, L)
        assert pool.free_pages == free + sum(2 - -(-L // 32) for L in t.len.tolist())
    assert A.decode_tree_status() == 0


@pytest.mark.parametrize("paged", [False, True])
@pytest.mark.parametrize("act,cache_dtype", [(F, F), (H, H)])
def test_a_turn_as_a_graph(act, cache_dtype, paged):
    """The lengths live on the device, so one captured turn serves every turn: the same bits as eager calls."""
    eager, p0 = _make(act, cache_dtype, paged)
    graph, p1 = _make(act, cache_dtype, paged)
    eager.run()
    first = eager.state()
    g, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(g, stream=side):
        graph.run()
    g.replay()
    torch.cuda.synchronize()
    same = lambda a, b: all(torch.equal(x, y) for x, y in zip(a, b))
    assert same(graph.state(), first)
    for _ in range(3):
        eager.run()
        g.replay()
    torch.cuda.synchronize()
    assert same(graph.state(), eager.state())


def test_two_streams_at_once():
    """Turns on two streams share no workspace."""
    a, _ = _make(F, F, False)
    b, _ = _make(H, H, False)
    want = []
    for t in (a, b):
        for _ in range(4):
            t.run()
        torch.cuda.synchronize()
        want.append(t.state())
    a, _ = _make(F, F, False)
    b, _ = _make(H, H, False)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(4):
        for s, t in zip(streams, (a, b)):
            with torch.cuda.stream(s):
                t.run()
    torch.cuda.synchronize()
    for t, w in zip((a, b), want):
        assert all(torch.equal(x, y) for x, y in zip(t.state(), w))


@pytest.mark.parametrize("dtype", [F, H])
def test_offsets_past_32_bits(dtype):
    """The second sequence lies 2^31 elements behind the first; the results are those of a small cache with the same rows."""
    L, n, cap, hkv, hq, far = 200, 5, 256, 2, 4, 2 ** 31 + 64
    big = [torch.empty(far + hkv * cap * D, dtype=dtype, device="cuda") for _ in range(2)]
    small = [torch.empty(2, hkv, cap, D, dtype=dtype, device="cuda") for _ in range(2)]
    off = torch.tensor([0, far], dtype=torch.int64, device="cuda")
    there = [(0, hkv * cap * D), (far, far + hkv * cap * D)]
    for x, y in zip(big, small):
        y.normal_()
        for b, (i, j) in enumerate(there):
            x[i:j] = y[b].flatten()
    len0 = torch.full((2,), L, dtype=torch.int32, device="cuda")
    cos, sin = A.rope_tables_scaled(TABLE + 100, D, 10000.0)
    q, k, v = (torch.randn(2, n, h * D, device="cuda") for h in (hq, hkv, hkv))
    results = []
    for (kc, vc), where in ((big, dict(kv_off=off)), (small, dict(seq_stride=hkv * cap * D))):
        where = dict(head_stride=cap * D, max_seq=cap, **where)
        heads = dict(n_kv_head=hkv, head_dim=D)
        lens, score = len0.clone(), torch.rand(2, hkv, cap, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
        qr = A.rope_append_at(q, k, v, cos, sin, n_head=hq, row0=lens, k_cache=kc, v_cache=vc, **heads, **where)[0]
        o = A.decode_tree(qr, kc, vc, n_head=hq, max_len=L, seq_len=lens, **heads, **where)
        A.kv_accept(kc, vc, torch.tensor([[1, 3], [2, 4]], dtype=torch.int32, device="cuda"), torch.full((2,), 2, dtype=torch.int32, device="cuda"),
                    lens, n_draft=n, new_len=lens, **heads, **where)
        s = A.decode_scored(qr[:, 0].contiguous(), kc, vc, score, n_head=hq, max_len=L + n, seq_len=lens, **heads, **where)
        _, kept = A.kv_evict(kc, vc, score, lens, keep=90, max_len=L + n, n_sink=4, n_recent=9, new_len=lens, **heads, **where)
        rows = [kc[i:j].view(hkv, cap, D)[:, :90].clone() if kc.dim() == 1 else kc[b, :, :90].clone() for b, (i, j) in enumerate(there)]
        results.append([o, s, score, kept, lens] + rows)
    for a, b in zip(*results):
        assert torch.equal(a, b)
