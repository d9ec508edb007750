"""Tree and scored decode where two kernels, two tiles or two lengths meet, and with values that are no numbers."""
import random

import pytest
import torch

import cache_util as U
from nimllm_b200 import attention as A
from test_gpu_decode_tree import _scored_case, _tree_case

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16


@pytest.mark.parametrize("Hq,q_dtype,D", [(129, F, 128), (160, F, 64), (257, H, 128), (300, H, 64)])
def test_scores_of_more_heads_than_a_tile(Hq, q_dtype, D):
    """The query tiles of a KV head (128 rows, 256 of a bf16 q) are cut apart from one another."""
    rng = random.Random(Hq)
    _scored_case(41, [rng.randint(200, 4000) for _ in range(32)], Hq, 1, D, q_dtype, H, F, 0, 1.0)


# (query heads, drafts): 4, 20, 48 and 160 query rows per KV head
@pytest.mark.parametrize("Hq,n", [(4, 2), (8, 5), (12, 8), (20, 16)])
@pytest.mark.parametrize("types", [(F, F, F), (F, H, F), (F, H, H), (H, H, H), (H, H, F)])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("L", [40, 300, 9000])
def test_nan_that_a_token_attends_reaches_its_result(L, D, types, Hq, n):
    """A query row with NaN, and every query row of a KV head with NaN in a row of K, has NaN results; the others keep their bits."""
    q_dtype, cache_dtype, out_dtype = types
    Hkv = 2
    G = Hq // Hkv
    cache = U.Cache(51, [L + n], Hkv, D, cache_dtype, 0, cap=L + n)
    q = torch.randn(1, n, Hq * D, generator=torch.Generator().manual_seed(52)).to(q_dtype).cuda()
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L, out_dtype=out_dtype)
    want = A.decode_tree(q, cache.kd, cache.vd, **cache.where(), **kw).view(n, Hq, D)
    assert torch.isfinite(want).all()
    bad_q = q.clone()
    bad_q.view(n, Hq, D)[n - 1, 1, 3] = float("nan")
    got = A.decode_tree(bad_q, cache.kd, cache.vd, **cache.where(), **kw).view(n, Hq, D)
    assert torch.isnan(got[n - 1, 1]).all()
    got[n - 1, 1] = want[n - 1, 1]
    assert torch.equal(got, want)
    for row in (0, 39, 70, 140, 200, L // 2, L - 1):       # both halves of a tile, tiles of both groups
        if row >= L:
            continue
        kd = cache.kd.clone()
        kd[cache.off_host[0] + row * D + 5] = float("nan")                       # KV head 0
        got = A.decode_tree(q, kd, cache.vd, **cache.where(), **kw).view(n, Hq, D)
        assert torch.isnan(got[:, :G]).all(), f"NaN in row {row}"
        assert torch.equal(got[:, G:], want[:, G:])


@pytest.mark.parametrize("Hq", [4, 24, 80, 320])
@pytest.mark.parametrize("types", [(F, F, F), (F, H, F), (H, H, H)])
@pytest.mark.parametrize("L", [40, 300, 9000])
def test_nan_that_a_token_attends_reaches_the_scores(L, types, Hq):
    """One weight that is no number makes the sum of its softmax, and with it every score of the KV head, none."""
    q_dtype, cache_dtype, out_dtype = types
    Hkv, D = 2, 64
    cache = U.Cache(53, [L], Hkv, D, cache_dtype, 0, cap=L)
    q = torch.randn(1, Hq * D, generator=torch.Generator().manual_seed(54)).to(q_dtype).cuda()
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L, out_dtype=out_dtype)
    want = torch.ones(1, Hkv, L, device="cuda")
    A.decode_scored(q, cache.kd, cache.vd, want, **cache.where(), **kw)
    for row in (0, 39, 70, 140, 200, L // 2, L - 1):
        if row >= L:
            continue
        kd = cache.kd.clone()
        kd[cache.off_host[0] + row * D + 5] = float("nan")
        score = torch.ones(1, Hkv, L, device="cuda")
        out = A.decode_scored(q, kd, cache.vd, score, **cache.where(), **kw).view(Hq, D)
        assert torch.isnan(out[: Hq // Hkv]).all() and torch.isfinite(out[Hq // Hkv:]).all()
        assert torch.isnan(score[0, 0]).all(), f"NaN in row {row}"
        assert torch.equal(score[0, 1], want[0, 1])


@pytest.mark.parametrize("Hq", [4, 24, 80])
@pytest.mark.parametrize("cache_dtype", [F, H])
@pytest.mark.parametrize("row", [0, 150, 299])
def test_an_infinite_score_leaves_no_number(row, cache_dtype, Hq):
    Hkv, D, L = 2, 64, 300
    cache = U.Cache(56, [L], Hkv, D, cache_dtype, 0, cap=L)
    cache.kd[cache.off_host[0] + row * D + 5] = float("inf")
    score = torch.zeros(1, Hkv, L, device="cuda")
    out = A.decode_scored(torch.ones(1, Hq * D, device="cuda"), cache.kd, cache.vd, score, n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L, **cache.where()).view(Hq, D)
    G = Hq // Hkv
    assert torch.isnan(out[:G]).all() and torch.isnan(score[0, 0]).all()
    assert torch.isfinite(out[G:]).all() and torch.isfinite(score[0, 1]).all()


@pytest.mark.parametrize("n,Hq,Hkv", [(5, 8, 2), (8, 4, 1), (17, 2, 2), (32, 1, 1)])
def test_weights_of_17_to_32_query_rows_keep_32_bits(n, Hq, Hkv):
    for seed in range(55, 60):
        _tree_case(seed, [100, 0, 37, 500], n, Hq, Hkv, 128, F, H, H, 0, "tree")
        _tree_case(seed, [60, 3000], n, Hq, Hkv, 128, F, H, H, 64, "chain", ragged=False)


@pytest.mark.parametrize("Hq,Hkv,D,q_dtype", [(20, 1, 128, F), (40, 1, 128, H), (40, 1, 64, H), (40, 1, 64, F), (96, 2, 128, F), (160, 1, 128, F), (300, 1, 64, H)])
def test_scores_beside_bf16_results_keep_32_bits(Hq, Hkv, D, q_dtype):
    _scored_case(61, [130, 5, 64, 700, 0, 3000], Hq, Hkv, D, q_dtype, H, H, 0, 1.0)
    _scored_case(62, [100, 257], Hq, Hkv, D, q_dtype, H, H, 32, 0.5)


@pytest.mark.parametrize("Hq", [4, 24, 80])
@pytest.mark.parametrize("cache_dtype", [F, H])
def test_scores_of_rows_that_count_as_hidden(cache_dtype, Hq):
    """Scaled scores below -1e30 everywhere: no NaN comes out of a sum that has nothing in it."""
    Hkv, D, L = 2, 64, 300
    k = -torch.ones(1, Hkv, L, D, dtype=cache_dtype, device="cuda")
    v = torch.ones_like(k)
    score = torch.full((1, Hkv, L), 3.0, device="cuda")
    out = A.decode_scored(torch.ones(1, Hq * D, device="cuda"), k, v, score, n_head=Hq, n_kv_head=Hkv, head_dim=D, max_len=L, max_seq=L, scale=1e30,
                          seq_stride=Hkv * L * D, head_stride=L * D, decay=0.5)
    assert torch.isfinite(out).all() and torch.isfinite(score).all()
    added = (score - 1.5).sum(-1)                          # nothing, or the equal weights of a softmax
    assert ((added == 0) | ((added - Hq // Hkv).abs() < 1e-3)).all()


@pytest.mark.parametrize("cache_dtype", [F, H])
@pytest.mark.parametrize("n,Hq,Hkv", [(2, 4, 2), (24, 2, 1)])
def test_more_sequences_than_threads(cache_dtype, n, Hq, Hkv):
    rng = random.Random(7)
    _tree_case(71, [0 if b % 7 == 3 else rng.randint(0, 70) for b in range(700)], n, Hq, Hkv, 64, H, cache_dtype, F, 0, "tree")


def test_calls_repeat_themselves_bit_for_bit():
    for types in ((F, F, F), (F, H, F), (H, H, H)):
        for n, Hq in ((1, 8), (5, 8), (24, 8), (64, 8)):
            cache = U.Cache(81, [5000 + n, 17 + n, 2600 + n], 2, 128, types[1], 64, cap=5100)
            q = torch.randn(3, n, Hq * 128, device="cuda").to(types[0])
            kw = dict(n_head=Hq, n_kv_head=2, head_dim=128, max_len=5000, out_dtype=types[2], seq_len=torch.tensor([5000, 17, 2600], dtype=torch.int32).cuda())
            a = A.decode_tree_paged(q, cache.kd, cache.vd, cache.table, **kw)
            sa = torch.zeros(3, 2, 5000, device="cuda")
            oa = A.decode_scored_paged(q[:, 0].contiguous(), cache.kd, cache.vd, cache.table, sa, **kw)
            for _ in range(5):
                assert torch.equal(a, A.decode_tree_paged(q, cache.kd, cache.vd, cache.table, **kw))
                s = torch.zeros_like(sa)
                assert torch.equal(oa, A.decode_scored_paged(q[:, 0].contiguous(), cache.kd, cache.vd, cache.table, s, **kw)) and torch.equal(s, sa)
