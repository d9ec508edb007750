"""Rows moved in place where blocks of layers, sequences and KV heads lie in any order that keeps them apart."""
import random

import pytest
import torch

import cache_util as U
from nimllm_b200 import attention as A

pytestmark = pytest.mark.gpu

LAYERS, B, HKV, CAP, D, N = 3, 4, 2, 40, 64, 9
# block number of (layer, sequence, head) in units of a block: nested in every order, and lines that mesh without nesting
ORDERS = [(8, 2, 1), (2, 6, 1), (1, 3, 12), (8, 1, 4), (3, 9, 50), (1, 3, 13), (2, 6, 3), (7, 4, 9), (10, 11, 7)]


@pytest.mark.parametrize("layer,seq,head", ORDERS)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_layouts(dtype, layer, seq, head):
    at = [(l * layer + b * seq + h * head) for l in range(LAYERS) for b in range(B) for h in range(HKV)]
    block = CAP * D
    if len(set(at)) < len(at):
        pytest.fail("the list holds a layout that overlaps")
    kc, vc = (torch.randn((max(at) + 1) * block, device="cuda").to(dtype) for _ in range(2))
    k0, v0 = kc.clone(), vc.clone()
    rng = random.Random(layer)
    lens = [0, 5, CAP - N, 17]
    paths = [sorted(rng.sample(range(N), 4)) for _ in lens]
    dev = lambda x: torch.tensor(x, dtype=torch.int32).cuda()
    where = dict(seq_stride=seq * block, head_stride=head * block, max_seq=CAP)
    new = A.kv_accept(kc, vc, dev(paths), dev([4] * B), dev(lens), n_draft=N, n_kv_head=HKV, head_dim=D, n_layer=LAYERS, layer_stride=layer * block, **where)
    assert new.tolist() == [x + 4 for x in lens]
    for now, old in ((kc, k0), (vc, v0)):
        want = old.clone().view(-1, CAP, D)
        for i, x in enumerate(at):
            b = i // HKV % B
            want[x, lens[b]:lens[b] + 4] = old.view(-1, CAP, D)[x, [lens[b] + p for p in paths[b]]]
        assert torch.equal(now.view(-1, CAP, D), want)
    score = torch.rand(B, HKV, CAP, device="cuda")
    k1 = kc.clone()
    new, kept = A.kv_evict(kc, vc, score, None, keep=12, n_kv_head=HKV, head_dim=D, max_len=CAP, **where)
    want = k1.clone().view(-1, CAP, D)
    for i, x in enumerate(at[: B * HKV]):                  # layer 0
        want[x, :12] = k1.view(-1, CAP, D)[x, kept[i // HKV, i % HKV].long()]
    assert torch.equal(kc.view(-1, CAP, D), want)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_accept_in_pages_of_several_layers(dtype):
    rng = random.Random(3)
    layers, n, Hkv, D, lens = 4, 9, 2, 64, [30, 0, 61]
    c = U.Cache(90, [l + n for l in lens], Hkv, D, dtype, 32)
    g = torch.Generator().manual_seed(91)
    kp, vp = (torch.randn(layers, *c.kd.shape, generator=g).to(dtype).cuda() for _ in range(2))
    k0, v0 = kp.clone(), vp.clone()
    paths = [sorted(rng.sample(range(n), 5)) for _ in lens]
    new = A.kv_accept_paged(kp, vp, c.table, torch.tensor(paths, dtype=torch.int32).cuda(), torch.tensor([5, 3, 4], dtype=torch.int32).cuda(),
                            torch.tensor(lens, dtype=torch.int32).cuda(), n_draft=n, n_kv_head=Hkv, head_dim=D, n_layer=layers)
    assert new.tolist() == [35, 3, 65]
    for now, before in ((kp, k0), (vp, v0)):
        for layer in range(layers):
            want = before[layer].clone()
            for b, (L, m) in enumerate(zip(lens, (5, 3, 4))):
                for i in range(m):
                    to, fro = L + i, L + paths[b][i]
                    tp, fp = int(c.table_host[b, to // 32]), int(c.table_host[b, fro // 32])
                    want[tp, :, to % 32] = before[layer][fp, :, fro % 32]
            assert torch.equal(now[layer], want)
