"""CPU tests of the operators on a cache whose rows are not its positions: refusals, scaled tables, pages given back."""
import ctypes as C
import math

import numpy as np
import pytest
import torch

from nimllm_b200 import _lib
from nimllm_b200 import attention as A

L = _lib.lib()
P = C.c_void_p(256)


def refused(rc, code, word):
    assert rc == code and word.encode() in L.nimllm_attn_last_error(), (rc, L.nimllm_attn_last_error())


def _rope(**o):
    a = dict(q=P, q_out=P, Hq=4, k=P, k_out=P, v=P, act=0, cos=P, sin=P, rot=64, layout=0, rows=16, pos=None, row0=None, first=0,
             kc=P, vc=P, cache=0, off=None, ss=4096, hs=2048, cap=32, B=1, n=1, Hkv=2, D=64, st=None)
    a.update(o)
    return L.nimllm_rope_append_at(*a.values())


@pytest.mark.parametrize("change,code,word", [
    (dict(cos=None), 1, "both RoPE tables"), (dict(q_out=None), 1, "q and q_out"), (dict(vc=None), 1, "both cache pointers"),
    (dict(k=None), 1, "k_new"), (dict(v=None), 1, "v_new"), (dict(rot=60), 1, "rot_dim"), (dict(rot=72), 1, "rot_dim"), (dict(rot=0), 1, "rot_dim"),
    (dict(rows=0), 1, "table_rows"), (dict(layout=2), 1, "layout"), (dict(act=2), 1, "dtype"), (dict(cache=7), 1, "dtype"), (dict(D=60), 1, "bad shape"),
    (dict(hs=2050), 1, "multiples of 16"), (dict(cap=0), 1, "max_seq"), (dict(q=C.c_void_p(8)), 1, "aligned"), (dict(kc=C.c_void_p(24)), 1, "aligned"),
    (dict(cos=C.c_void_p(4)), 1, "aligned"), (dict(n=-1), 1, "bad shape")])
def test_rope_at_refusals(change, code, word):
    refused(_rope(**change), code, word)


def test_rope_at_of_nothing():
    assert _rope(n=0) == 0 and _rope(B=0) == 0


def test_rope_at_bwd_refusals():
    f = L.nimllm_rope_at_bwd
    refused(f(P, P, 4, P, P, 0, None, P, 64, 0, 16, None, 0, 1, 1, 2, 64, None), 1, "tables")
    refused(f(P, None, 4, P, P, 0, P, P, 64, 0, 16, None, 0, 1, 1, 2, 64, None), 1, "gradient")
    refused(f(None, None, 4, None, None, 0, P, P, 64, 0, 16, None, 0, 1, 1, 2, 64, None), 1, "gradient")
    refused(f(P, C.c_void_p(8), 4, P, P, 0, P, P, 64, 0, 16, None, 0, 1, 1, 2, 64, None), 1, "aligned")


def _tree(**o):
    a = dict(q=P, qt=0, k=P, v=P, ct=1, off=None, ss=65536, hs=16384, cap=128, len=None, max_len=100, n_new=None, mask=None, out=P, ot=0, rec=None,
             B=1, n=4, Hq=4, Hkv=2, D=64, scale=0.125, ws=None, bytes=0, st=None)
    a.update(o)
    return L.nimllm_attn_decode_tree(*a.values())


@pytest.mark.parametrize("change,code,word", [
    (dict(q=None), 1, "null"), (dict(out=None), 1, "null"), (dict(k=None), 1, "null cache"), (dict(Hq=5), 1, "bad shape"), (dict(n=0), 1, "bad shape"),
    (dict(max_len=-1), 1, "bad shape"), (dict(n=257), 2, "257"), (dict(D=96), 2, "head_dim"), (dict(qt=3), 1, "dtype"), (dict(ct=2), 1, "dtype"), (dict(cap=0), 1, "max_seq"),
    (dict(hs=16386), 1, "multiples of 16"), (dict(ss=3), 1, "multiples of 16"), (dict(mask=C.c_void_p(12)), 1, "8-byte"), (dict(B=70000), 2, "too large"),
    (dict(out=C.c_void_p(8)), 1, "aligned")])
def test_tree_refusals(change, code, word):
    refused(_tree(**change), code, word)


def test_workspaces_are_asked_for():
    need = L.nimllm_attn_decode_tree_workspace_bytes(4, 8, 32, 8, 128, 100000, 0)
    assert need > 0
    refused(_tree(ct=0, B=4, n=8, Hq=32, Hkv=8, D=128, max_len=100000), 3, "workspace")
    refused(_tree(ct=0, B=4, n=8, Hq=32, Hkv=8, D=128, max_len=100000, ws=P, bytes=need - 1), 3, "workspace")
    refused(_tree(ct=0, B=4, n=8, Hq=32, Hkv=8, D=128, max_len=100000, ws=C.c_void_p(264), bytes=need), 1, "256-byte")
    assert L.nimllm_attn_decode_scored_workspace_bytes(1, 4, 2, 64, 100, 1) >= 4 * 128 * 4
    assert L.nimllm_attn_decode_scored_workspace_bytes(0, 4, 2, 64, 100, 1) == 0
    assert L.nimllm_attn_decode_tree_workspace_bytes(1, 300, 4, 2, 64, 100, 1) == 0


@pytest.mark.parametrize("shape", [dict(max_len=2**31 - 1), dict(max_len=2**30 + 1), dict(batch=65536), dict(Hq=2**30, Hkv=2**30), dict(Hq=2**31 - 2, Hkv=1)])
@pytest.mark.parametrize("dtype", [0, 1])
def test_no_workspace_for_shapes_that_are_refused(dtype, shape):
    a = {**dict(batch=1, n=256, Hq=4, Hkv=2, D=64, max_len=100), **shape}
    assert L.nimllm_attn_decode_tree_workspace_bytes(*a.values(), dtype) == 0
    refused(_tree(B=a["batch"], n=256, Hq=a["Hq"], Hkv=a["Hkv"], max_len=a["max_len"], ct=dtype), 2, "too large")
    del a["n"]
    assert L.nimllm_attn_decode_scored_workspace_bytes(*a.values(), dtype) == 0


def test_paged_refusals():
    f = L.nimllm_attn_decode_tree_paged
    tail = (None, 100, None, None, P, 0, None, 1, 4, 4, 2, 64, 0.125, None, 0, None)
    refused(f(P, 0, P, P, 1, None, 4, 32, 9, *tail), 1, "null pages")
    refused(f(P, 0, P, P, 1, P, 4, 48, 9, *tail), 1, "page_rows")
    refused(f(P, 0, P, P, 1, P, 4, 16, 9, *tail), 1, "page_rows")
    refused(f(P, 0, P, P, 1, P, 0, 32, 9, *tail), 1, "max_pages")
    refused(f(P, 0, P, P, 1, P, 4, 32, 0, *tail), 1, "n_pages")
    refused(f(P, 0, C.c_void_p(8), P, 1, P, 4, 32, 9, *tail), 1, "aligned")
    refused(f(P, 0, P, P, 1, P, 2**30, 32, 9, *tail), 1, "max_pages")


def test_scored_refusals():
    f = L.nimllm_attn_decode_scored

    def go(**o):
        a = dict(q=P, qt=0, k=P, v=P, ct=1, off=None, ss=65536, hs=16384, cap=128, len=None, max_len=100, out=P, ot=0, score=P, rows=100, decay=1.0,
                 B=1, Hq=4, Hkv=2, D=64, scale=0.125, ws=None, bytes=0, st=None)
        a.update(o)
        return f(*a.values())
    refused(go(score=None), 1, "score")
    refused(go(rows=99), 1, "99 scores")
    refused(go(max_len=0), 1, "max_len")
    refused(go(D=32), 2, "head_dim")
    refused(go(), 3, "workspace")


@pytest.mark.parametrize("heads", [6145, 8192])
def test_scored_refuses_more_heads_than_a_block_holds(heads):
    """The update of the scores would not launch, behind an attention that has."""
    a = dict(q=P, qt=0, k=P, v=P, ct=1, off=None, ss=65536, hs=16384, cap=128, len=None, max_len=100, out=P, ot=0, score=P, rows=100, decay=1.0,
             B=1, Hq=heads, Hkv=1, D=64, scale=0.125, ws=None, bytes=0, st=None)
    refused(L.nimllm_attn_decode_scored(*a.values()), 2, "query heads per KV head")


def test_accept_refusals():
    f = L.nimllm_kv_accept

    def go(**o):
        a = dict(k=P, v=P, ct=1, L=2, ls=1 << 20, off=None, ss=65536, hs=16384, cap=128, path=P, mp=4, np=P, len=P, new=P, n=8, B=1, Hkv=2, D=64, st=None)
        a.update(o)
        return f(*a.values())
    refused(go(path=None), 1, "null path")
    refused(go(new=None), 1, "null path")
    refused(go(mp=9), 2, "max_path")
    refused(go(n=257, mp=4), 2, "n 257")
    refused(go(mp=0), 1, "bad shape")
    refused(go(L=0), 1, "bad shape")
    refused(go(ls=12), 1, "layer_stride")
    refused(go(D=60), 2, "16 bytes")


@pytest.mark.parametrize("change,word", [
    (dict(ls=0), "layer_stride 0"), (dict(ls=8192 - 8), "overlap"), (dict(ls=-(8192 - 8)), "overlap"), (dict(hs=0), "head_stride 0"), (dict(hs=8192 - 8), "overlap"),
    (dict(ss=0, B=2), "seq_stride 0"), (dict(ss=8192, B=2, hs=8192), "overlap"),             # sequence 1, head 0 is sequence 0, head 1
    (dict(ls=3 * 8192, hs=8192, Hkv=4), "overlap"), (dict(ls=5 * 8192, ss=2 * 8192, hs=8192, B=4), "overlap"), (dict(ls=8192, off=P), "overlap")])
def test_accept_refuses_blocks_that_overlap(change, word):
    a = dict(k=P, v=P, ct=1, L=2, ls=1 << 20, off=None, ss=65536, hs=16384, cap=128, path=P, mp=4, np=P, len=P, new=P, n=8, B=1, Hkv=2, D=64, st=None)
    a.update({**dict(hs=8192), **change})
    refused(L.nimllm_kv_accept(*a.values()), 1, word)


@pytest.mark.parametrize("ls", [0, 9 * 2 * 32 * 64 - 8])
def test_accept_refuses_pages_of_layers_that_overlap(ls):
    refused(L.nimllm_kv_accept_paged(P, P, 1, 2, ls, P, 4, 32, 9, P, 4, P, P, P, 8, 1, 2, 64, None), 1, "overlap")


@pytest.mark.parametrize("change", [dict(hs=0), dict(ss=0, B=2), dict(ss=8192, hs=8192, B=2), dict(hs=4096, off=P)])
def test_evict_refuses_blocks_that_overlap(change):
    a = dict(k=P, v=P, ct=1, off=None, ss=65536, hs=16384, cap=128, score=P, rows=128, len=P, max_len=128, keep=64, sink=4, recent=8, kept=P, new=P,
             B=1, Hkv=2, D=64, st=None)
    a.update(change)
    refused(L.nimllm_kv_evict(*a.values()), 1, "overlap")


def test_evict_refusals():
    f = L.nimllm_kv_evict

    def go(**o):
        a = dict(k=P, v=P, ct=1, off=None, ss=65536, hs=16384, cap=128, score=P, rows=128, len=P, max_len=128, keep=64, sink=4, recent=8, kept=P, new=P,
                 B=1, Hkv=2, D=64, st=None)
        a.update(o)
        return f(*a.values())
    refused(go(score=None), 1, "null score")
    refused(go(kept=None), 1, "null score")
    refused(go(keep=0), 1, "keep")
    refused(go(sink=60), 1, "keep")
    refused(go(sink=-1), 1, "keep")
    refused(go(recent=2**31 - 1), 1, "keep")
    refused(go(max_len=129), 1, "holds 128 rows")
    refused(go(rows=100), 1, "100 scores")


def test_python_checks_shapes_before_anything_runs():
    t = torch.zeros(1, 4, 256)
    with pytest.raises(_lib.NimllmAttnError, match="device tensor"):
        A.decode_tree(t, t, t, n_head=4, n_kv_head=2, head_dim=64, max_len=4, max_seq=8)
    with pytest.raises(_lib.NimllmAttnError, match="device tensor"):
        A.rope_append_at(t, t, t, None, None, n_head=4, n_kv_head=4, head_dim=64)


@pytest.fixture
def on_cpu(monkeypatch):
    """The wrappers' own checks, with tensors on the CPU and a library that must not be reached."""
    monkeypatch.setattr(A, "_on", lambda t: (-1, A._here))

    class NotReached:
        def __getattr__(self, name):
            raise AssertionError(f"{name} was called")
    monkeypatch.setattr(A, "lib", NotReached)


def test_pages_of_several_layers_are_refused_by_calls_for_one(on_cpu):
    pages, table = torch.zeros(3, 8, 2, 32, 64), torch.zeros(1, 4, dtype=torch.int32)
    q, kw = torch.zeros(1, 2, 256), dict(n_head=4, n_kv_head=2, head_dim=64)
    kv = torch.zeros(1, 2, 128)
    calls = [lambda p: A.decode_tree_paged(q, p, p, table, max_len=10, **kw),
             lambda p: A.decode_scored_paged(q[:, 0], p, p, table, torch.zeros(1, 2, 10), max_len=10, **kw),
             lambda p: A.rope_append_at_paged(q, kv, kv, None, None, p, p, table, **kw),
             lambda p: A.kv_evict_paged(p, p, table, torch.zeros(1, 2, 10), None, keep=4, n_kv_head=2, head_dim=64, max_len=10)]
    for call in calls:
        with pytest.raises(_lib.NimllmAttnError, match="one layer"):
            call(pages)
        for one in (pages[0], pages[:1]):                  # as before
            with pytest.raises(AssertionError, match="was called"):
                call(one)
        with pytest.raises(_lib.NimllmAttnError, match="expected"):
            call(pages[0, 0])
    ints = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(_lib.NimllmAttnError, match="4 layers expected"):
        A.kv_accept_paged(pages, pages, table, ints.view(1, 1), ints, ints, n_draft=1, n_kv_head=2, head_dim=64, n_layer=4)
    with pytest.raises(AssertionError, match="was called"):
        A.kv_accept_paged(pages, pages, table, ints.view(1, 1), ints, ints, n_draft=1, n_kv_head=2, head_dim=64, n_layer=2)


@pytest.mark.parametrize("strides", [dict(seq_stride=-8192, head_stride=4096), dict(seq_stride=8192, head_stride=-4096)])
def test_blocks_in_front_of_a_cache_are_refused(on_cpu, strides):
    c, q, kv = torch.zeros(3 * 8192), torch.zeros(3, 2, 256), torch.zeros(3, 2, 128)
    score, ints = torch.zeros(3, 2, 64), torch.zeros(3, dtype=torch.int32)
    heads, kv_heads, where = dict(n_head=4, n_kv_head=2, head_dim=64), dict(n_kv_head=2, head_dim=64), dict(max_seq=64)
    calls = [lambda **w: A.decode_tree(q, c, c, max_len=10, **heads, **w), lambda **w: A.decode_scored(q[:, 0].contiguous(), c, c, score, max_len=10, **heads, **w),
             lambda **w: A.rope_append_at(q, kv, kv, None, None, k_cache=c, v_cache=c, **heads, **w),
             lambda **w: A.kv_accept(c, c, ints.view(3, 1), ints, ints, n_draft=1, **kv_heads, **w),
             lambda **w: A.kv_evict(c, c, score, None, keep=4, max_len=64, **kv_heads, **w)]
    for call in calls:
        with pytest.raises(_lib.NimllmAttnError, match="first block"):
            call(**strides, **where)
        with pytest.raises(AssertionError, match="was called"):
            call(seq_stride=8192, head_stride=4096, **where)
    with pytest.raises(_lib.NimllmAttnError, match="first block"):
        A.kv_accept(c, c, ints.view(3, 1), ints, ints, n_draft=1, n_layer=2, layer_stride=-3 * 8192, seq_stride=8192, head_stride=4096, **kv_heads, **where)


def test_one_cache_of_two_is_refused(on_cpu):
    kv, c, kw = torch.zeros(1, 2, 128), torch.zeros(8192), dict(n_head=4, n_kv_head=2, head_dim=64, head_stride=4096, max_seq=64)
    for k_cache, v_cache in ((c, None), (None, c)):
        with pytest.raises(_lib.NimllmAttnError, match="both"):
            A.rope_append_at(None, kv, kv, None, None, k_cache=k_cache, v_cache=v_cache, **kw)


def _freqs(rot, base):
    return base ** (-2.0 * np.arange(rot // 2) / rot)


@pytest.mark.parametrize("kind,factor", [("none", 1.0), ("linear", 8.0), ("base", 4.0), ("ramp", 16.0)])
def test_scaled_tables(kind, factor):
    rot, base, rows, orig, low, high, gain = 64, 10000.0, 5000, 2048, 1.0, 32.0, 1.1
    cos, sin = A.rope_tables_scaled(rows, rot, base, kind=kind, factor=factor, low=low, high=high, orig_len=orig, gain=gain, device="cpu")
    w = _freqs(rot, base)
    if kind == "linear":
        w = w / factor
    elif kind == "base":
        w = _freqs(rot, base * factor ** (rot / (rot - 2)))
        assert abs(w[-1] * factor / _freqs(rot, base)[-1] - 1) < 1e-12
    elif kind == "ramp":
        t = orig * w / (2 * math.pi)
        keep = np.clip((t - low) / (high - low), 0, 1)
        assert keep.max() == 1 and keep.min() == 0
        w = w * keep + w / factor * (1 - keep)
    angle = np.arange(rows)[:, None] * w[None]
    # half a step of the table's type, and 2^-40 for angles computed in another order
    for got, want in ((cos, gain * np.cos(angle)), (sin, gain * np.sin(angle))):
        assert (np.abs(got.numpy().astype(np.float64) - want) <= 2.0 ** -24 * np.abs(want) + 2.0 ** -40 * gain).all()


def test_scaled_tables_refusals():
    c = np.zeros((4, 32), np.float32)
    f = lambda **o: L.nimllm_rope_tables_scaled_host(*{**dict(c=c.ctypes.data, s=c.ctypes.data, n=4, rot=64, base=1e4, kind=1, factor=2.0, low=1.0, high=4.0, orig=8, gain=1.0), **o}.values())
    assert f() == 0
    for bad in (dict(c=None), dict(rot=63), dict(base=-1.0), dict(kind=4), dict(factor=0.0), dict(kind=2, rot=2), dict(kind=3, low=4.0), dict(kind=3, orig=0), dict(factor=float("nan"))):
        assert f(**bad) == 1
    with pytest.raises(_lib.NimllmAttnError, match="unknown kind"):
        A.rope_tables_scaled(4, 64, 1e4, kind="twice", device="cpu")


def test_pool_shrink_gives_pages_back():
    pool = A.PagedKvPool(1, 10, 32, 1, 64, 2, 8, on_device=False)
    pool.reserve(0, 200)
    pool.reserve(1, 33)
    before = pool.table_host()
    pool.shrink(0, 65)
    t = pool.table_host()
    assert pool.free_pages == 10 - 3 - 2 and pool.seq_pages(0) == 3 and pool.seq_rows(0) == 65
    assert (t[0, :3] == before[0, :3]).all() and (t[0, 3:] == -1).all() and (t[1] == before[1]).all()
    pool.shrink(0, 400)                       # more than it holds: nothing changes
    assert pool.seq_rows(0) == 65
    pool.reserve(1, 7 * 32)
    assert pool.free_pages == 0
    assert len({x for x in pool.table_host().flatten().tolist() if x >= 0}) == 10
    pool.shrink(0, 0)
    assert pool.seq_pages(0) == 0 and pool.free_pages == 3
    for seq, rows in ((-1, 0), (2, 0), (0, -1)):
        with pytest.raises(_lib.NimllmAttnError):
            pool.shrink(seq, rows)
