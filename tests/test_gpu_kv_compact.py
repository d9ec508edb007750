"""The accepted path of a drafted tree and the rows that an eviction keeps: rows moved in place, against gathered copies."""
import random

import pytest
import torch

import cache_util as U
from nimllm_b200 import attention as A

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16


def same(a, b):
    return torch.equal(torch.nan_to_num(a, nan=9.0), torch.nan_to_num(b, nan=9.0))


@pytest.mark.parametrize("paged", [0, 32])
@pytest.mark.parametrize("dtype,D", [(F, 64), (H, 64), (H, 128), (F, 128), (H, 8), (F, 4), (H, 80)])
@pytest.mark.parametrize("n", [1, 8, 65, 256])
def test_accept(n, dtype, D, paged):
    rng = random.Random(n * D)
    Hkv, lens = 3, [0, 1, 29, 200]
    B = len(lens)
    c = U.Cache(3, [l + n for l in lens], Hkv, D, dtype, paged)
    paths = [sorted(rng.sample(range(n), rng.randint(0, n))) for _ in range(B)]
    paths[1], paths[2] = list(range(n)), list(range(n // 2, n))             # nothing moves; everything moves
    m = max(1, max(len(p) for p in paths))
    path = torch.tensor([p + [rng.randint(-5, 300)] * (m - len(p)) for p in paths], dtype=torch.int32).cuda()
    n_path = torch.tensor([len(p) for p in paths], dtype=torch.int32).cuda()
    seq_len = torch.tensor(lens, dtype=torch.int32).cuda()
    kw = dict(n_draft=n, n_kv_head=Hkv, head_dim=D)
    k0, v0 = c.kd.clone(), c.vd.clone()
    if paged:
        new = A.kv_accept_paged(c.kd, c.vd, c.table, path, n_path, seq_len, **kw)
    else:
        new = A.kv_accept(c.kd, c.vd, path, n_path, seq_len, **c.where(), **kw)
    assert new.tolist() == [l + len(p) for l, p in zip(lens, paths)]
    assert seq_len.tolist() == lens
    for now, before in ((c.kd, k0), (c.vd, v0)):
        for b in range(B):
            old, got = c.block(before, b), c.block(now, b)
            L, p = lens[b], paths[b]
            assert torch.equal(got[:, :L], old[:, :L])
            assert torch.equal(got[:, L:L + len(p)], old[:, [L + x for x in p]])
            assert torch.equal(got[:, L + len(p):], old[:, L + len(p):])
    # in place of seq_len: the lengths change after the rows
    kd, vd = k0.clone(), v0.clone()
    if paged:
        A.kv_accept_paged(kd, vd, c.table, path, n_path, seq_len, new_len=seq_len, **kw)
    else:
        A.kv_accept(kd, vd, path, n_path, seq_len, new_len=seq_len, **c.where(), **kw)
    assert torch.equal(seq_len, new) and same(kd, c.kd) and same(vd, c.vd)


def test_accept_layers_and_bad_paths():
    n, Hkv, D, L, cap, layers = 12, 2, 64, 20, 32, 5
    kc = torch.randn(layers, 7, Hkv, cap, D, device="cuda")
    vc = torch.randn_like(kc)
    k0, v0 = kc.clone(), vc.clone()
    #        fine       repeats     falls        past n     negative    too long    past the block
    paths = [[1, 4, 7], [2, 2, 3], [5, 3, 9], [0, 12, 13], [3, -1, 4], [0, 2, 5], [2, 10, 11]]
    n_path = [3, 3, 3, 3, 3, 99, 3]
    used = [[1, 4, 7], [2], [5], [0], [3], [0, 2, 5], [2, 10]]
    lens = [L] * 6 + [21]
    new = A.kv_accept(kc, vc, torch.tensor(paths, dtype=torch.int32).cuda(), torch.tensor(n_path, dtype=torch.int32).cuda(),
                      torch.tensor(lens, dtype=torch.int32).cuda(), n_draft=n, n_kv_head=Hkv, head_dim=D, n_layer=layers,
                      layer_stride=7 * Hkv * cap * D, seq_stride=Hkv * cap * D, head_stride=cap * D, max_seq=cap)
    assert new.tolist() == [l + len(u) for l, u in zip(lens, used)]
    for now, old in ((kc, k0), (vc, v0)):
        want = old.clone()
        for b, u in enumerate(used):
            want[:, b, :, lens[b]:lens[b] + len(u)] = old[:, b][:, :, [lens[b] + x for x in u]]
        assert torch.equal(now, want)


def evict_rows(score, L, keep, sink, recent):
    """The kept rows of one KV head, by a sort of (score, -row) with NaN below everything."""
    if L <= keep:
        return list(range(L))
    mid = list(range(sink, L - recent))
    s = [float(x) for x in score]
    order = sorted(mid, key=lambda r: (-1, 0, r) if s[r] == float("inf") else (1, 0, r) if s[r] != s[r] else (0, -s[r], r))
    return sorted(list(range(sink)) + order[: keep - sink - recent] + list(range(L - recent, L)))


def _evict(seed, lens, Hkv, D, dtype, paged, keep, sink, recent, make=None, alias=False):
    c = U.Cache(seed, lens, Hkv, D, dtype, paged, cap=max(lens) + 1)
    g = torch.Generator().manual_seed(seed)
    score = torch.rand(len(lens), Hkv, max(lens) + 5, generator=g)
    if make:
        score = make(score, g)
    k0, v0, dev = c.kd.clone(), c.vd.clone(), score.cuda()
    seq_len = torch.tensor(lens, dtype=torch.int32).cuda()
    kw = dict(keep=keep, n_sink=sink, n_recent=recent, n_kv_head=Hkv, head_dim=D, max_len=max(lens), new_len=seq_len if alias else None)
    if paged:
        new, kept = A.kv_evict_paged(c.kd, c.vd, c.table, dev, seq_len, **kw)
    else:
        new, kept = A.kv_evict(c.kd, c.vd, dev, seq_len, **c.where(), **kw)
    assert new.tolist() == [min(L, keep) for L in lens]
    kept, dev = kept.cpu(), dev.cpu()
    for b, L in enumerate(lens):
        m = min(L, keep)
        for h in range(Hkv):
            rows = evict_rows(score[b, h, :L], L, keep, sink, recent)
            assert kept[b, h].tolist() == rows + [-1] * (keep - m), f"sequence {b}, head {h}"
            assert same(dev[b, h, :m], score[b, h, rows])
            assert (dev[b, h, m:L] == 0).all() and same(dev[b, h, L:], score[b, h, L:])
            for now, old in ((c.kd, k0), (c.vd, v0)):
                assert torch.equal(c.block(now, b)[h, :m], c.block(old, b)[h, rows])
    return c


@pytest.mark.parametrize("paged", [0, 32, 128])
@pytest.mark.parametrize("dtype,D", [(F, 64), (H, 128), (H, 8), (F, 4), (H, 80)])
def test_evict(dtype, D, paged):
    _evict(1, [0, 1, 49, 50, 51, 64, 333, 1025], 2, D, dtype, paged, 50, 4, 10)


@pytest.mark.parametrize("keep,sink,recent", [(1, 0, 0), (1, 1, 0), (1, 0, 1), (20, 20, 0), (20, 0, 20), (20, 7, 13), (2999, 0, 0), (2999, 10, 100), (1500, 4, 0), (3000, 1, 1)])
def test_evict_budgets(keep, sink, recent):
    _evict(2, [3000, 700, 2999], 2, 64, H, 0, keep, sink, recent, alias=keep % 2 == 0)


def _ties(s, g):
    return (s * 4).floor()                    # four values only


def _odd(s, g):
    s = s - 0.5                               # negative ones, both zeros, infinities, NaN
    u = torch.rand(s.shape, generator=g)
    s[u < 0.2] = 0.0
    s[(u >= 0.2) & (u < 0.4)] = -0.0
    s[(u >= 0.4) & (u < 0.5)] = float("nan")
    s[(u >= 0.5) & (u < 0.55)] = float("inf")
    s[(u >= 0.55) & (u < 0.6)] = -float("inf")
    return s


@pytest.mark.parametrize("make", [_ties, _odd, lambda s, g: s * 0, lambda s, g: s * 1e-42, lambda s, g: s * float("nan")])
@pytest.mark.parametrize("keep", [3, 100, 511, 900])
def test_evict_equal_and_odd_scores(make, keep):
    _evict(3, [1000, 100, 512], 3, 64, F, 0, keep, 1, 2, make)


def test_evict_long():
    _evict(4, [40000, 12345], 1, 64, H, 0, 9999, 4, 100)
    _evict(5, [70001], 2, 8, H, 256, 35000, 0, 0, _ties)


def test_evict_skips_rows_without_a_page():
    c = U.Cache(6, [100], 1, 64, H, 32)
    table = c.table.clone()
    table[0, 1] = c.n_pages                   # rows 32 .. 63
    score = torch.rand(1, 1, 100, generator=torch.Generator().manual_seed(1)).cuda()
    k0 = c.kd.clone()
    new, kept = A.kv_evict_paged(c.kd, c.vd, table, score, torch.tensor([100], dtype=torch.int32).cuda(), keep=50, n_kv_head=1, head_dim=64, max_len=100)
    old, got = c.block(k0, 0)[0], c.block(c.kd, 0)[0]
    for j, r in enumerate(kept[0, 0].tolist()):
        moved = not (32 <= j < 64) and not (32 <= r < 64)
        assert torch.equal(got[j], old[r] if moved else old[j])
