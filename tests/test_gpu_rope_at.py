"""Rotation at a position per token, both layouts, part of the head, with the append; and its gradient."""
import random

import pytest
import torch

import cache_util as U
from nimllm_b200 import attention as A

pytestmark = pytest.mark.gpu

F, H = torch.float32, torch.bfloat16


def turned(x, cos, sin, pos, layout, sign=1.0):
    """float64 rotation of x [..., heads, D] at table rows pos [...], and its error scale |a c| + |b s|."""
    h = cos.shape[1]
    c, s = cos.double()[pos].unsqueeze(-2), sin.double()[pos].unsqueeze(-2) * sign
    y, mag = x.clone(), x.abs()
    i0, i1 = (slice(0, h), slice(h, 2 * h)) if layout == "half" else (slice(0, 2 * h, 2), slice(1, 2 * h, 2))
    a, b = x[..., i0], x[..., i1]
    y[..., i0], y[..., i1] = a * c - b * s, a * s + b * c
    mag[..., i0], mag[..., i1] = (a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs()
    return y, mag


def check(got, want, mag, dtype, what):
    """Two products and a sum in 32 bits (3 * 2^-24 of their magnitudes), then the rounding of the type."""
    off = (got.double() - want).abs() - U.HALF_STEP[dtype] * want.abs() * (1 + 2.0 ** -7) - 3 * 2.0 ** -24 * mag
    assert float(off.max()) <= 0, f"{what}: {float(off.max()):.3e} too far"


@pytest.mark.parametrize("paged", [0, 32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot", [(64, 64), (64, 32), (128, 128), (128, 64), (128, 24), (96, 72), (80, 8), (8, 8)])
@pytest.mark.parametrize("act,cache", [(F, F), (F, H), (H, F), (H, H)])
def test_append_at(act, cache, D, rot, layout, paged):
    rng = random.Random(D * rot)
    Hq, Hkv, n, lens = 6, 2, 5, [0, 30, 3, 62]
    B, table = len(lens), 90
    cos, sin = A.rope_tables_scaled(table, rot, 10000.0, kind="linear", factor=2.0)
    g = torch.Generator().manual_seed(rot)
    q, k, v = (torch.randn(B, n, h * D, generator=g).to(act) for h in (Hq, Hkv, Hkv))
    pos = torch.tensor([[rng.randrange(table) if (b + t) % 4 else rng.choice([-1, -7, table, 2**31 - 1]) for t in range(n)] for b in range(B)], dtype=torch.int32)
    c = U.Cache(5, lens, Hkv, D, cache, paged, cap=66, spare=0)      # draft rows 66.. of the last sequence do not exist
    rows = torch.tensor(lens, dtype=torch.int32).cuda()
    q_out = torch.full((B, n, Hq * D), 5.0, dtype=act, device="cuda")
    k_out = torch.full((B, n, Hkv * D), 5.0, dtype=act, device="cuda")
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, layout=layout, pos=pos.cuda(), row0=rows, q_out=q_out, k_out=k_out)
    k0, v0 = c.kd.clone(), c.vd.clone()
    qd, kd, vd = q.cuda(), k.cuda(), v.cuda()
    if paged:
        A.rope_append_at_paged(qd, kd, vd, cos, sin, c.kd, c.vd, c.table, **kw)
    else:
        A.rope_append_at(qd, kd, vd, cos, sin, k_cache=c.kd, v_cache=c.vd, **c.where(), **kw)
    torch.cuda.synchronize()
    assert torch.equal(qd.cpu(), q) and torch.equal(kd.cpu(), k)
    live = (pos >= 0) & (pos < table)
    safe = pos.clamp(0, table - 1).long()
    for got, x, h in ((q_out, q, Hq), (k_out, k, Hkv)):
        want, mag = turned(x.double().view(B, n, h, D), cos.cpu(), sin.cpu(), safe, layout)
        got = got.cpu().view(B, n, h, D)
        check(got[live], want[live], mag[live], act, "rotated")
        assert (got[~live] == 5.0).all()
    wk, mk = turned(k.double().view(B, n, Hkv, D), cos.cpu(), sin.cpu(), safe, layout)
    expect_k, expect_v = k0.clone().cpu(), v0.clone().cpu()
    gk, gv = c.kd.cpu(), c.vd.cpu()

    def at(t, b, h, r):
        if paged:
            pg = int(c.table_host[b, r // paged]) if r // paged < c.max_pages else -1
            return t[pg, h, r % paged] if pg >= 0 else None
        s = c.off_host[b] + h * c.head_stride + r * D
        return t[s:s + D] if r < 66 else None

    for b in range(B):
        for t in range(n):
            for h in range(Hkv):
                if live[b, t] and at(gk, b, h, lens[b] + t) is not None:
                    check(at(gk, b, h, lens[b] + t), wk[b, t, h], mk[b, t, h], cache, "cached k")
                    assert torch.equal(at(gv, b, h, lens[b] + t), v[b, t].view(Hkv, D)[h].to(cache))
                    at(expect_k, b, h, lens[b] + t).copy_(at(gk, b, h, lens[b] + t))
                    at(expect_v, b, h, lens[b] + t).copy_(at(gv, b, h, lens[b] + t))
    assert torch.equal(torch.nan_to_num(gk, nan=9.0), torch.nan_to_num(expect_k, nan=9.0)), "another row of K changed"
    assert torch.equal(torch.nan_to_num(gv, nan=9.0), torch.nan_to_num(expect_v, nan=9.0)), "another row of V changed"


@pytest.mark.parametrize("act", [F, H])
def test_in_place_default_positions_and_no_tables(act):
    B, n, Hq, Hkv, D = 2, 9, 4, 2, 64
    cos, sin = A.rope_tables_scaled(64, D, 10000.0)
    q, k, v = (torch.randn(B, n, h * D, device="cuda").to(act) for h in (Hq, Hkv, Hkv))
    kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D)
    q1, k1 = A.rope_append_at(q, k, v, cos, sin, first_row=3, **kw)
    q2, k2 = q.clone(), k.clone()
    A.rope_append_at(q2, k2, v, cos, sin, first_row=3, q_out=q2, k_out=k2, **kw)
    assert torch.equal(q1, q2) and torch.equal(k1, k2)
    # the rotation that rope_append does at consecutive positions
    q3, k3 = q.clone(), k.clone()
    A.rope_append(q3, k3, v, cos, sin, pos0=3, **kw)
    assert torch.equal(q1, q3) and torch.equal(k1, k3)
    cache = torch.zeros(2, B, Hkv, 16, D, device="cuda")
    qn, _ = A.rope_append_at(q, k, v, None, None, first_row=2, k_cache=cache[0], v_cache=cache[1], seq_stride=Hkv * 16 * D, head_stride=16 * D, max_seq=16, **kw)
    assert torch.equal(qn, q)
    assert torch.equal(cache[0][:, :, 2:11], k.float().view(B, n, Hkv, D).transpose(1, 2))
    assert (cache[:, :, :, :2] == 0).all() and (cache[:, :, :, 11:] == 0).all()


@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,rot,dtype", [(64, 64, F), (64, 16, H), (128, 128, H), (128, 96, F)])
def test_gradient(D, rot, dtype, layout):
    """Against the transposed rotation in float64, against differences of the forward, and zero for padding."""
    B, n, Hq, Hkv = 2, 11, 3, 1
    cos, sin = A.rope_tables_scaled(40, rot, 10000.0, gain=1.25)
    g = torch.Generator().manual_seed(rot)
    dq, dk = (torch.randn(B, n, h * D, generator=g).to(dtype) for h in (Hq, Hkv))
    pos = torch.randint(0, 40, (B, n), generator=g, dtype=torch.int32)
    pos[0, 3], pos[1, 0] = -1, 40
    gq, gk = A.rope_at_backward(dq.cuda(), dk.cuda(), cos, sin, n_head=Hq, n_kv_head=Hkv, head_dim=D, layout=layout, pos=pos.cuda())
    live = (pos >= 0) & (pos < 40)
    for got, x, h in ((gq, dq, Hq), (gk, dk, Hkv)):
        want, mag = turned(x.double().view(B, n, h, D), cos.cpu(), sin.cpu(), pos.clamp(0, 39).long(), layout, -1.0)
        got = got.cpu().view(B, n, h, D)
        check(got[live], want[live], mag[live], dtype, "gradient")
        assert (got[~live] == 0).all()
    one, none = A.rope_at_backward(dq.cuda(), None, cos, sin, n_head=Hq, n_kv_head=Hkv, head_dim=D, layout=layout, pos=pos.cuda(), in_place=True)
    assert none is None and torch.equal(one, gq)
    if dtype == F:
        # <dq, R x'> - <dq, R x> = <R^T dq, x' - x>: the rotation is linear, so a difference of any size is its derivative.
        x = torch.randn(B, n, Hq * D, generator=g)
        k = torch.zeros(B, n, Hkv * D).cuda()
        kw = dict(n_head=Hq, n_kv_head=Hkv, head_dim=D, layout=layout, pos=pos.cuda())
        y0, _ = A.rope_append_at(torch.zeros_like(x).cuda(), k, None, cos, sin, q_out=torch.zeros_like(x).cuda(), **kw)
        y1, _ = A.rope_append_at(x.cuda(), k, None, cos, sin, q_out=torch.zeros_like(x).cuda(), **kw)
        m = live[..., None]
        left = (dq.double() * (y1 - y0).cpu().double() * m).sum()
        right = (gq.cpu().double() * x.double()).sum()
        # each side is a sum of products whose factors are off by 3 roundings of magnitudes of at most 2 * 1.25
        assert abs(float(left - right)) <= 3 * 2.0 ** -24 * 2.5 * float((dq.double().abs() * x.double().abs().amax()).sum()) * 2
