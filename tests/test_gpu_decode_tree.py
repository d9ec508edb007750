"""Attention of drafted tokens over a cache (nimllm_attn_decode_tree and _paged) and scored decode, against float64."""
import math
import random

import pytest
import torch

import cache_util as U
from nimllm_b200 import attention as A

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16


def _tree_case(seed, lens, n, Hq, Hkv, D, q_dtype, cache_dtype, out_dtype, paged, mask, ragged=True, partials=False, scale=None):
    rng = random.Random(seed)
    B = len(lens)
    n_new = [n if b % 3 != 1 else rng.randint(0, n) for b in range(B)] if ragged else [n] * B
    cache = U.Cache(seed, [l + m for l, m in zip(lens, n_new)], Hkv, D, cache_dtype, paged, cap=max(lens) + n + 3)
    q = torch.randn(B, n, Hq * D, generator=torch.Generator().manual_seed(seed + 1)).to(q_dtype)
    sets = []
    for b in range(B):
        s, _ = U.random_tree(rng, n)
        if mask == "empty":
            s = [0 if i % 3 == 0 else x for i, x in enumerate(s)]          # tokens that attend no draft at all
        sets.append(s)
    words = U.mask_words(sets, n) if mask != "chain" else None
    if mask == "chain":
        sets = [[(1 << (i + 1)) - 1 for i in range(n)]] * B
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out = torch.full((B, n, Hq * D), 7.0, dtype=out_dtype, device="cuda")
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=max(lens), seq_len=torch.tensor(lens, dtype=torch.int32).cuda(),
              n_new=torch.tensor(n_new, dtype=torch.int32).cuda() if ragged else None, tree_mask=words, scale=scale, out=out, partials=partials)
    if paged:
        got = A.decode_tree_paged(q.cuda(), cache.kd, cache.vd, cache.table, **kw)
    else:
        got = A.decode_tree(q.cuda(), cache.kd, cache.vd, **cache.where(), **kw)
    torch.cuda.synchronize()
    rec = got[1].view(B, n, Hq, D + 4).cpu() if partials else None
    o = out.cpu().view(B, n, Hq, D)
    for b in range(B):
        m = n_new[b]
        assert (o[b, m:] == 7.0).all(), "rows of tokens that do not exist were written"
        if m == 0:
            continue
        see = torch.zeros(m, lens[b] + m, dtype=torch.bool)
        see[:, : lens[b]] = True
        for i in range(m):
            for j in range(m):
                see[i, lens[b] + j] = bool(sets[b][i] >> j & 1)
        want, wm, wl, _, mag = U.attend(q[b, :m].double().view(m, Hq, D), cache.k[b].double(), cache.v[b].double(), see, scale)
        v_max = float(cache.v[b].double().abs().max()) if lens[b] + m else 0.0
        tol = U.attention_tolerance(D, lens[b] + m, mag, v_max, out_dtype, wide=cache_dtype == H and not partials and n * Hq // Hkv > 32)
        U.assert_within(o[b, :m], want, tol, out_dtype, f"sequence {b} ({lens[b]} rows, {m} drafts)")
        empty = ~see.any(1)
        assert (o[b, :m][empty] == 0).all()
        if partials:
            tol32 = U.attention_tolerance(D, lens[b] + m, mag, v_max, torch.float32)
            U.assert_within(rec[b, :m, :, :D], want, tol32, torch.float32, f"records of sequence {b}")
            live = ~empty
            lse = rec[b, :m, :, D].double() + torch.log(rec[b, :m, :, D + 1].double())
            want_lse = wm + torch.log(wl)
            # a sum of weights that are each off by the tolerance's factor moves the logarithm by as much
            assert float((lse - want_lse)[live].abs().max() if live.any() else 0.0) <= tol32 / v_max + 2.0 ** -22 * (1 + float(wm[live].abs().max() if live.any() else 0))
            assert (rec[b, :m, :, D + 1][empty] == 0).all()


LENS = [0, 1, 31, 32, 33, 63, 64, 65, 127, 128, 129, 250]


@pytest.mark.parametrize("paged", [0, 32, 64])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("types", [(F, F, F), (F, H, F), (H, H, H), (H, F, F), (F, F, H), (H, H, F), (F, H, H)])
def test_lengths_around_the_tiles(types, D, paged):
    _tree_case(11, LENS, 5, 6, 2, D, *types, paged, "tree")


@pytest.mark.parametrize("G,Hkv", [(1, 3), (2, 1), (3, 3), (4, 2), (7, 1), (8, 2), (16, 1)])
@pytest.mark.parametrize("cache_dtype", [F, H])
def test_group_sizes(cache_dtype, G, Hkv):
    _tree_case(12, [70, 0, 190, 64], 6, G * Hkv, Hkv, 64, H, cache_dtype, F, 0, "tree")


@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 32, 33, 63, 64, 65, 128, 129, 255, 256])
@pytest.mark.parametrize("cache_dtype", [F, H])
def test_tree_sizes(cache_dtype, n):
    _tree_case(13, [100, 0, 37], n, 8, 2, 128, F, cache_dtype, F, 64 if n % 2 else 0, "tree")
    _tree_case(14, [300, 1], n, 3, 3, 64, H, cache_dtype, H, 0, "tree", ragged=False)


@pytest.mark.parametrize("n,G", [(48, 3), (33, 8), (7, 6)])
@pytest.mark.parametrize("D,types", [(64, (F, H, F)), (64, (F, H, H)), (64, (H, H, H)), (128, (F, H, F)), (128, (F, H, H)), (128, (H, H, F)), (128, (H, H, H)), (64, (F, F, F))])
def test_many_segments(D, types, n, G):
    """More pieces than SMs, so that a CTA has several sequences, some of one token or without rows, between its cuts."""
    _tree_case(31, [130, 0, 300, 1, 64, 257, 0, 128, 5, 190, 31, 222], n, 8 * G, 8, D, *types, 0, "tree")


@pytest.mark.parametrize("mask", ["chain", "empty"])
@pytest.mark.parametrize("cache_dtype", [F, H])
def test_chain_and_tokens_without_drafts(cache_dtype, mask):
    _tree_case(15, [0, 90, 0, 64, 5], 37, 6, 2, 64, H, cache_dtype, F, 0, mask, partials=True)
    _tree_case(16, [0, 90, 0, 64, 5], 70, 8, 1, 128, F, cache_dtype, H, 32, mask, partials=True)


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_long_rows_are_split_and_joined(cache_dtype):
    _tree_case(17, [5000, 17, 2600], 9, 9, 3, 64, F, cache_dtype, F, 0, "tree", partials=True)
    _tree_case(18, [4100, 3], 24, 8, 2, 128, H, cache_dtype, H, 256, "tree", partials=True)


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_large_and_small_scores(cache_dtype):
    """A softmax that is all but one row, and one that is flat."""
    _tree_case(19, [400, 60], 4, 6, 2, 64, F, cache_dtype, F, 0, "tree", scale=6.0)
    _tree_case(20, [400, 60], 4, 6, 2, 64, F, cache_dtype, F, 0, "tree", scale=0.0)


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_hidden_keys_may_hold_anything(cache_dtype):
    """K of a sibling draft is NaN, infinity or the type's lowest value: the other branch does not notice."""
    n, Hq, Hkv, D, L = 6, 4, 2, 64, 75
    cache = U.Cache(21, [L + n], Hkv, D, cache_dtype, 0, cap=L + n)
    q = torch.randn(1, n, Hq * D).cuda()
    sets = [[1, 3, 5, 11, 21, 35]]           # drafts 1 and 2 are two branches behind draft 0
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L, seq_len=torch.tensor([L], dtype=torch.int32).cuda(), tree_mask=U.mask_words(sets, n))
    want = A.decode_tree(q, cache.kd, cache.vd, **cache.where(), **kw)
    for bad in (float("nan"), float("inf"), -float("inf"), torch.finfo(cache_dtype).min):
        kd = cache.kd.clone()
        for h in range(Hkv):
            at = cache.off_host[0] + h * cache.head_stride + (L + 2) * D
            kd[at:at + D] = bad
        got = A.decode_tree(q, kd, cache.vd, **cache.where(), **kw)
        for i in (0, 1, 3, 5):
            assert torch.equal(got[0, i], want[0, i]), f"token {i} does not attend draft 2 ({bad})"


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_pages_outside_the_pool_are_not_attended(cache_dtype):
    n, Hq, Hkv, D, L = 3, 4, 2, 64, 200
    cache = U.Cache(22, [L + n], Hkv, D, cache_dtype, 32)
    for entry in (-1, cache.n_pages, 2**31 - 1, -(2**31)):
        table = cache.table.clone()
        table[0, 2] = entry                  # rows 64 .. 95
        q = torch.randn(1, n, Hq * D, generator=torch.Generator().manual_seed(5)).to(H)
        got = A.decode_tree_paged(q.cuda(), cache.kd, cache.vd, table, n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L,
                                  seq_len=torch.tensor([L], dtype=torch.int32).cuda()).cpu()
        see = torch.zeros(n, L + n, dtype=torch.bool)
        for i in range(n):
            see[i, : L + i + 1] = True
        see[:, 64:96] = False
        want, _, _, _, mag = U.attend(q[0].double().view(n, Hq, D), cache.k[0].double(), cache.v[0].double(), see, 1 / math.sqrt(D))
        U.assert_within(got[0].view(n, Hq, D), want, U.attention_tolerance(D, L + n, mag, float(cache.v[0].abs().max()), F), F, f"entry {entry}")


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_lengths_outside_the_arguments_are_clamped(cache_dtype):
    """seq_len and n_new outside their ranges, and drafts that do not fit the block."""
    Hq, Hkv, D, n = 4, 2, 64, 5
    cache = U.Cache(23, [40] * 4, Hkv, D, cache_dtype, 0, cap=40)
    q = torch.randn(4, n, Hq * D, generator=torch.Generator().manual_seed(3)).to(H)
    got = A.decode_tree(q.cuda(), cache.kd, cache.vd, **cache.where(), n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=38,
                        seq_len=torch.tensor([-5, 38, 2**31 - 1, 20], dtype=torch.int32).cuda(),
                        n_new=torch.tensor([99, 5, 5, -1], dtype=torch.int32).cuda(), out=torch.zeros(4, n, Hq * D, device="cuda")).cpu()
    for b, (length, tokens, drafts) in enumerate([(0, 5, 5), (38, 5, 2), (38, 5, 2), (20, 0, 0)]):
        assert (got[b, tokens:] == 0).all()
        if not tokens:
            continue
        rows = length + drafts
        see = torch.zeros(tokens, rows, dtype=torch.bool)
        for i in range(tokens):
            see[i, : min(rows, length + i + 1)] = True
        want, _, _, _, mag = U.attend(q[b].double().view(n, Hq, D), cache.k[b][:, :rows].double(), cache.v[b][:, :rows].double(), see, 1 / math.sqrt(D))
        U.assert_within(got[b].view(n, Hq, D), want, U.attention_tolerance(D, rows, mag, float(cache.v[b].abs().max()), F), F, f"sequence {b}")


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_captured_on_another_stream_and_replayed(cache_dtype):
    """Two graphs with workspaces of their own, replayed in turn with new inputs, agree with eager calls bit for bit."""
    n, Hq, Hkv, D = 7, 6, 2, 64
    cache = U.Cache(24, [900 + n, 30 + n], Hkv, D, cache_dtype, 0)
    lens = torch.tensor([900, 30], dtype=torch.int32).cuda()
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=900, seq_len=lens, **cache.where())
    qs = [torch.randn(2, n, Hq * D, device="cuda") for _ in range(2)]
    score = torch.zeros(2, Hkv, 907, device="cuda")
    side = torch.cuda.Stream()
    A.decode_tree(qs[0], cache.kd, cache.vd, **kw)
    torch.cuda.synchronize()
    graphs = []
    for q in qs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            o = A.decode_tree(q, cache.kd, cache.vd, **kw)
            s = A.decode_scored(q[:, 0].contiguous(), cache.kd, cache.vd, score, **kw)
        graphs.append((g, o, s))
    for round_ in range(3):
        for q in qs:
            q.normal_(generator=torch.Generator(device="cuda").manual_seed(round_))
        score.zero_()
        for g, _, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        kept = [(o.clone(), s.clone()) for _, o, s in graphs]
        twice = score.clone()
        score.zero_()
        for (o, s), q in zip(kept, qs):
            assert torch.equal(o, A.decode_tree(q, cache.kd, cache.vd, **kw))
            assert torch.equal(s, A.decode_scored(q[:, 0].contiguous(), cache.kd, cache.vd, score, **kw))
        assert torch.equal(score, twice)


# ------------------------------------------------------------------------------------------------ scored decode
def _scored_case(seed, lens, Hq, Hkv, D, q_dtype, cache_dtype, out_dtype, paged, decay, scale=None):
    B = len(lens)
    cache = U.Cache(seed, lens, Hkv, D, cache_dtype, paged, cap=max(lens) + 2)
    g = torch.Generator().manual_seed(seed + 1)
    q = torch.randn(B, Hq * D, generator=g).to(q_dtype)
    old = torch.rand(B, Hkv, max(lens) + 9, generator=g)
    if decay == 0:
        old[:, :, ::3] = float("nan")
    score = old.cuda()
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=max(lens), seq_len=torch.tensor(lens, dtype=torch.int32).cuda(), decay=decay,
              out_dtype=out_dtype, scale=scale)
    if paged:
        out = A.decode_scored_paged(q.cuda(), cache.kd, cache.vd, cache.table, score, **kw)
    else:
        out = A.decode_scored(q.cuda(), cache.kd, cache.vd, score, **cache.where(), **kw)
    torch.cuda.synchronize()
    out, score = out.cpu().view(B, Hq, D), score.cpu()
    G = Hq // Hkv
    for b, L in enumerate(lens):
        want, _, _, w, mag = U.attend(q[b].double().view(1, Hq, D), cache.k[b].double(), cache.v[b].double(), torch.ones(1, L, dtype=torch.bool), scale)
        v_max = float(cache.v[b].double().abs().max()) if L else 0.0
        U.assert_within(out[b], want[0], U.attention_tolerance(D, L, mag, v_max, out_dtype), out_dtype, f"out {b}")
        add = w[0].view(Hkv, G, L).sum(1)
        full = add + (decay * old[b, :, :L].double() if decay else 0.0)
        # a weight is off by the factor of the tolerance (for values of 1), G of them and the old score are added in 32 bits
        tol = U.attention_tolerance(D, L, mag, 1.0, F) * float(add.max() if L else 0) + (G + 3) * 2.0 ** -24 * float(full.abs().max() if L else 0)
        if L:
            assert float((score[b, :, :L].double() - full).abs().max()) <= tol
        assert torch.equal(torch.nan_to_num(score[b, :, L:]), torch.nan_to_num(old[b, :, L:])), "scores behind the sequence changed"


@pytest.mark.parametrize("paged", [0, 32, 128])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("types", [(F, F, F), (F, H, F), (H, H, H), (H, F, F)])
def test_scored_lengths(types, D, paged):
    _scored_case(31, LENS + [1000], 6, 2, D, *types, paged, 1.0)


@pytest.mark.parametrize("G,Hkv", [(1, 1), (3, 3), (4, 8), (8, 1), (12, 2), (40, 1)])
@pytest.mark.parametrize("cache_dtype", [F, H])
def test_scored_groups(cache_dtype, G, Hkv):
    _scored_case(32, [130, 5, 64], G * Hkv, Hkv, 128, H, cache_dtype, F, 0, 0.5)


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_scored_decay_zero_does_not_read_and_long_rows(cache_dtype):
    _scored_case(33, [300, 0, 7], 6, 2, 64, F, cache_dtype, F, 0, 0.0)
    _scored_case(34, [9000, 4, 5555], 8, 2, 128, F, cache_dtype, F, 0, 1.0)
    _scored_case(35, [3000], 4, 4, 64, F, cache_dtype, H, 64, 1.0, scale=4.0)


@pytest.mark.parametrize("cache_dtype", [F, H])
def test_scored_skips_rows_without_a_page(cache_dtype):
    Hq, Hkv, D, L = 4, 2, 64, 100
    cache = U.Cache(36, [L], Hkv, D, cache_dtype, 32)
    table = cache.table.clone()
    table[0, 1] = -1
    score = torch.full((1, Hkv, L), 2.0, device="cuda")
    q = torch.randn(1, Hq * D, generator=torch.Generator().manual_seed(5)).to(H)
    A.decode_scored_paged(q.cuda(), cache.kd, cache.vd, table, score, n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L)
    see = torch.ones(1, L, dtype=torch.bool)
    see[:, 32:64] = False
    _, _, _, w, mag = U.attend(q.double().view(1, Hq, D), cache.k[0].double(), cache.v[0].double(), see, 1 / math.sqrt(D))
    add = w[0].view(Hkv, 2, L).sum(1)
    got = score.cpu()[0].double()
    assert (got[:, 32:64] == 2.0).all()
    assert float((got - 2.0 - add).abs().max()) <= U.attention_tolerance(D, L, mag, 1.0, F) * float(add.max()) + 5 * 2.0 ** -24 * 3


def test_zz_no_launch_gave_up():
    assert A.decode_tree_status(reset=False) == 0
