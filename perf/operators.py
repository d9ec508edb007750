"""Operators of a KV cache whose rows are no longer its positions: a tree of drafted tokens, and an evicted cache.

  rope     rotation of q and k at a position of their own per token, in the half or the interleaved layout, of the whole
           head or its first part, with the append of the rows (and the gradient of the rotation)
  tree     attention of up to 256 drafted tokens a sequence over the cached rows and over each other by a tree mask
  accept   the rows of the accepted path moved down behind the committed ones, in every layer
  scored   decode attention that also adds every cached row's attention weight to a running score
  evict    the rows with the highest scores kept, beside the first and the last ones, in every KV head

`own` False: the operators in elementary torch operations, in 32 bits; True: the library's calls.
A case's lengths are spread over [lo, hi] by its seed.  Masks are 64-bit words, bit j: the token attends draft j."""
import math
import random
from types import SimpleNamespace

import torch

own = False

_T = {"f32": torch.float32, "bf16": torch.bfloat16}
_SIZE = {"f32": 4, "bf16": 2}


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    small = dict(Hq=9, Hkv=3, D=64)       # the heads of the 30-layer 135M-parameter model
    large = dict(Hq=32, Hkv=8, D=128)     # the heads of the long-context configuration
    return [
        # one conversation, its next token: only latency counts
        dict(name="rope one token", op="rope", B=1, n=1, **small, rot=64, layout="half", act="f32", cache="f32", page=0, lo=400, hi=512),
        # drafted trees of a batch go into a paged cache; half of every head rotates
        dict(name="rope drafted trees paged", op="rope", B=61, n=24, **large, rot=64, layout="interleaved", act="bf16", cache="bf16", page=64, lo=256, hi=2048),
        # the gradient of a training batch's rotation
        dict(name="rope gradient prompts", op="rope_bwd", B=4, n=8192, **large, rot=128, layout="half", act="bf16"),
        # one conversation with a few drafted tokens over the reference's own fp32 cache
        dict(name="tree one sequence f32", op="tree", B=1, n=7, **small, act="f32", cache="f32", out="f32", page=0, lo=300, hi=505),
        # a batch of conversations, small trees, the projection's fp32 q
        dict(name="tree ragged batch", op="tree", B=256, n=5, **small, act="f32", cache="bf16", out="f32", page=0, lo=512, hi=4096),
        # wide trees over long paged contexts
        dict(name="tree wide long paged", op="tree", B=8, n=64, **large, act="bf16", cache="bf16", out="bf16", page=256, lo=9000, hi=16384),
        # one conversation accepts a few of its drafts, all 30 layers
        dict(name="accept one sequence", op="accept", B=1, n=8, L=30, Hkv=3, D=64, cache="f32", page=0, lo=200, hi=500),
        # a batch accepts along wide trees
        dict(name="accept batch", op="accept", B=48, n=64, L=30, Hkv=8, D=128, cache="bf16", page=0, lo=64, hi=192),
        # decode steps that keep score: the fp32 path ...
        dict(name="scored one sequence f32", op="scored", B=1, **small, act="f32", cache="f32", out="f32", page=0, lo=700, hi=1000),
        # ... and a batch of long conversations in pages
        dict(name="scored batch paged", op="scored", B=32, **large, act="bf16", cache="bf16", out="bf16", page=128, lo=2048, hi=8192),
        # one conversation over its budget
        dict(name="evict one sequence", op="evict", B=1, Hkv=3, D=64, cache="f32", page=0, keep=384, sink=4, recent=64, lo=400, hi=512),
        # long conversations cut to a quarter
        dict(name="evict long batch", op="evict", B=8, Hkv=8, D=128, cache="bf16", page=0, keep=8192, sink=4, recent=512, lo=20000, hi=32768),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "rope_bwd", "tree", "tree", "accept", "scored", "evict"])
    G = rng.choice([1, 2, 3, 4, 5, 7, 8])
    Hkv = rng.choice([1, 2, 3, 4, 8])
    D = rng.choice([64, 128])
    act, cache, out = (rng.choice(["f32", "bf16"]) for _ in range(3))
    page = rng.choice([0, 0, 32, 64, 256])
    c = dict(op=op, B=_spread(rng, 1, 200))
    if op == "rope":
        c.update(n=_spread(rng, 1, 256), Hq=G * Hkv, Hkv=Hkv, D=D, rot=rng.choice([D, D // 2, D // 4]), layout=rng.choice(["half", "interleaved"]), act=act, cache=cache, page=page)
        span = 4000
    elif op == "rope_bwd":
        c.update(n=_spread(rng, 1, 9000), Hq=G * Hkv, Hkv=Hkv, D=D, rot=rng.choice([D, D // 2, D // 4]), layout=rng.choice(["half", "interleaved"]), act=act)
        c["B"] = max(1, min(c["B"], 20_000_000 // (c["n"] * (G + 1) * Hkv * D)))
        return c
    elif op == "tree":
        c.update(n=_spread(rng, 1, 256), Hq=G * Hkv, Hkv=Hkv, D=D, act=act, cache=cache, out=out, page=page)
        span = 16000
    elif op == "accept":
        c.update(n=_spread(rng, 1, 128), L=rng.choice([1, 12, 30]), Hkv=Hkv, D=D, cache=cache, page=page)
        span = 400
    elif op == "scored":
        c.update(Hq=G * Hkv, Hkv=Hkv, D=D, act=act, cache=cache, out=out, page=page)
        span = 32000
    else:
        c.update(Hkv=Hkv, D=D, cache=cache, page=page)
        span = 32000
    hi = _spread(rng, 16, span)
    lo = max(1, int(hi * rng.uniform(0.1, 1.0)))
    if op == "evict":
        c["keep"] = max(4, int(hi * rng.uniform(0.2, 0.9)))
        c["sink"] = rng.randrange(0, max(1, min(8, c["keep"] // 4)))
        c["recent"] = rng.randrange(0, max(1, c["keep"] // 4))
    # what the whole cache may hold: 300 MB, and the scores of a tree in 32 bits 600 MB
    cap = hi + c.get("n", 0)
    row = c.get("L", 1) * Hkv * D * 2 * _SIZE[cache]
    most = 300_000_000 // (row * cap)
    if op == "tree":
        most = min(most, 150_000_000 // (c["Hq"] * c["n"] * cap))
    if most < 1:
        hi = max(16, hi * max(most, 1) // 8)
        lo = min(lo, hi)
        if op == "evict":
            c["keep"] = min(c["keep"], hi)
            c["sink"], c["recent"] = min(c["sink"], c["keep"] // 4), min(c["recent"], c["keep"] // 4)
    c["B"] = max(1, min(c["B"], most))
    c.update(lo=lo, hi=hi)
    return c


def _lengths(case, seed):
    r = random.Random(seed * 7919 + 13)
    B = case["B"]
    lens = [r.randint(case["lo"], case["hi"]) for _ in range(B)]
    n = case.get("n", 0)
    # a fifth of a batch drafts fewer tokens than the others
    n_new = [n if b == 0 or r.random() < 0.8 else r.randint(1, n) for b in range(B)] if n else None
    return lens, n_new


def work(case):
    c = SimpleNamespace(**case)
    if c.op in ("rope", "rope_bwd"):
        act = _SIZE[c.act]
        cells = c.B * c.n * c.D
        tables = c.n * c.rot * 4 if c.op == "rope_bwd" else min(c.B * c.n, c.hi + c.n) * c.rot * 4
        if c.op == "rope_bwd":
            return {"bytes": 2 * cells * (c.Hq + c.Hkv) * act + tables, "flops": 3 * c.B * c.n * (c.Hq + c.Hkv) * c.rot}
        return {"bytes": cells * ((2 * c.Hq + 2 * c.Hkv) * act + 2 * c.Hkv * _SIZE[c.cache]) + tables + 4 * c.B * c.n,
                "flops": 3 * c.B * c.n * (c.Hq + c.Hkv) * c.rot}
    rows = c.B * (c.lo + c.hi) / 2
    if c.op == "tree":
        rows += c.B * c.n
        return {"bytes": rows * c.Hkv * c.D * 2 * _SIZE[c.cache] + c.B * c.n * c.Hq * c.D * (_SIZE[c.act] + _SIZE[c.out]),
                "flops": 4.0 * rows * c.n * c.Hq * c.D}
    if c.op == "scored":
        return {"bytes": rows * c.Hkv * (c.D * 2 * _SIZE[c.cache] + 8) + c.B * c.Hq * c.D * (_SIZE[c.act] + _SIZE[c.out]),
                "flops": 4.0 * rows * c.Hq * c.D}
    row = c.D * 2 * _SIZE[c.cache]
    if c.op == "accept":
        return {"bytes": 2.0 * c.B * _path_len(c.n) * c.L * c.Hkv * row, "flops": 0.0}
    kept = c.B * c.Hkv * min(c.keep, (c.lo + c.hi) / 2)
    return {"bytes": rows * c.Hkv * 4 + kept * (2 * row + 4 + 4), "flops": 0.0}


def _path_len(n):
    return max(1, (n + 3) // 4)


# ---------------------------------------------------------------------------------------------------- inputs
def _cache(shape, dtype, gen):
    return torch.randn(shape, device="cuda", dtype=dtype, generator=gen)


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def prepare(case, seed):
    c = SimpleNamespace(**case)
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = random.Random(seed * 104729 + 7)
    s = SimpleNamespace(c=c)

    if c.op in ("rope", "rope_bwd"):
        act = _T[c.act]
        rows = c.n if c.op == "rope_bwd" else c.hi + c.n
        # positions stretched by a factor of four, as for a context four times the trained one
        f = torch.arange(c.rot // 2, device="cuda", dtype=torch.float64)
        angle = (torch.arange(rows, device="cuda", dtype=torch.float64) / 4.0)[:, None] * (10000.0 ** (-2.0 * f / c.rot))[None]
        s.cos, s.sin = angle.cos().float(), angle.sin().float()
        s.q = torch.randn(c.B, c.n, c.Hq * c.D, device="cuda", dtype=act, generator=g)
        s.k = torch.randn(c.B, c.n, c.Hkv * c.D, device="cuda", dtype=act, generator=g)
        if c.op == "rope_bwd":
            return s
        s.v = torch.randn(c.B, c.n, c.Hkv * c.D, device="cuda", dtype=act, generator=g)
        s.q_out = torch.zeros_like(s.q)
    if c.op != "rope_bwd":
        lens, n_new = _lengths(case, seed)
        s.lens_host, s.max_len = lens, c.hi
        s.seq_len = _ints(lens)
        cap = c.hi + case.get("n", 0)
        dt, L = _T[c.cache], case.get("L", 0)
        if c.page:
            s.max_pages = -(-cap // c.page)
            s.cap = s.max_pages * c.page
            n_pages = c.B * s.max_pages
            s.table = torch.randperm(n_pages, device="cuda", generator=g).to(torch.int32).view(c.B, s.max_pages)
            shape = (n_pages, c.Hkv, c.page, c.D)
        else:
            s.cap, s.table = cap, None
            shape = (c.B, c.Hkv, cap, c.D)
        s.kc, s.vc = (_cache(((L,) if L else ()) + shape, dt, g) for _ in range(2))
    if c.op == "rope":
        s.n_new = n_new
        # the depth of every token in its tree; padding tokens have no position
        pos = []
        for b in range(c.B):
            depth = [0]
            for i in range(1, c.n):
                depth.append(depth[r.randint(max(0, i - 4), i - 1)] + 1)
            pos.append([lens[b] + depth[i] if i < n_new[b] else -1 for i in range(c.n)])
        s.pos = _ints(pos)
    elif c.op == "tree":
        s.q = torch.randn(c.B, c.n, c.Hq * c.D, device="cuda", dtype=_T[c.act], generator=g)
        words = (c.n + 63) // 64
        masks = []
        for b in range(c.B):
            m = [1]
            for i in range(1, c.n):
                m.append(m[r.randint(max(0, i - 4), i - 1)] | (1 << i))
            for x in m:
                for w in range(words):
                    v = (x >> (64 * w)) & (2**64 - 1)
                    masks.append(v - 2**64 if v >= 2**63 else v)
        s.mask = torch.tensor(masks, dtype=torch.int64, device="cuda").view(c.B, c.n, words)
        s.n_new = _ints(n_new)
        s.out = torch.zeros(c.B, c.n, c.Hq * c.D, device="cuda", dtype=_T[c.out])
        s.scale = 1.0 / math.sqrt(c.D)
    elif c.op == "accept":
        m = _path_len(c.n)
        s.path = _ints([sorted(r.sample(range(c.n), m)) for _ in range(c.B)])
        s.n_path = _ints([m if b == 0 else r.randint(0, m) for b in range(c.B)])
        s.new_len = torch.zeros_like(s.seq_len)
    elif c.op == "scored":
        s.q = torch.randn(c.B, c.Hq * c.D, device="cuda", dtype=_T[c.act], generator=g)
        s.score = torch.rand(c.B, c.Hkv, s.cap, device="cuda", generator=g)
        s.scale = 1.0 / math.sqrt(c.D)
    elif c.op == "evict":
        # sums of softmax weights: a few large, most small, some exactly nothing
        u = torch.rand(c.B, c.Hkv, s.cap, device="cuda", generator=g)
        s.score0 = torch.where(u < 0.05, torch.zeros_like(u), torch.exp(torch.randn(u.shape, device="cuda", generator=g) * 2 - 4))
    return s


# ---------------------------------------------------------------------------------------------------- plain forms
def _turn(x, cos, sin, layout, sign):
    """x [..., D] rotated by the angles of cos, sin [..., rot / 2], the rest of the head as it is."""
    h = cos.shape[-1]
    turned, rest = x[..., : 2 * h], x[..., 2 * h:]
    if layout == "half":
        a, b = turned[..., :h], turned[..., h:]
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
    y0, y1 = a * cos - sign * b * sin, sign * a * sin + b * cos
    y = torch.cat((y0, y1), -1) if layout == "half" else torch.stack((y0, y1), -1).flatten(-2)
    return torch.cat((y, rest), -1)


def _rows(s, t, layer=False):
    """The cache as [(layers,) B, Hkv, rows, D]."""
    if s.table is None:
        return t
    c, table = s.c, s.table.long()
    if layer:
        return t[:, table].transpose(2, 3).reshape(t.shape[0], c.B, c.Hkv, s.cap, c.D)
    return t[table].transpose(1, 2).reshape(c.B, c.Hkv, s.cap, c.D)


def _rope(s):
    c = s.c
    live = s.pos >= 0
    p = s.pos.clamp(min=0).long()
    cos, sin = s.cos[p][:, :, None], s.sin[p][:, :, None]
    q = _turn(s.q.float().view(c.B, c.n, c.Hq, c.D), cos, sin, c.layout, 1.0).flatten(2).to(s.q.dtype)
    s.q_out = torch.where(live[..., None], q, s.q_out)
    k = _turn(s.k.float().view(c.B, c.n, c.Hkv, c.D), cos, sin, c.layout, 1.0)
    v = s.v.view(c.B, c.n, c.Hkv, c.D)
    row = (s.seq_len[:, None] + torch.arange(c.n, device="cuda")).long()
    if s.table is None:
        at = (torch.arange(c.B, device="cuda")[:, None], slice(None), row)
    else:
        at = (s.table.long().gather(1, row // c.page), slice(None), row % c.page)
    for t, x in ((s.kc, k), (s.vc, v)):
        t[at] = torch.where(live[..., None, None], x.to(t.dtype), t[at])
    return {"q": s.q_out, "k": s.kc, "v": s.vc}


def _rope_bwd(s):
    c = s.c
    cos, sin = s.cos[: c.n, None], s.sin[: c.n, None]
    return tuple(_turn(x.float().view(c.B, c.n, -1, c.D), cos, sin, c.layout, -1.0).flatten(2).to(x.dtype) for x in (s.q, s.k))


def _softmax(x, allowed):
    x = x.masked_fill(~allowed, -math.inf)
    top = x.amax(-1, keepdim=True)
    e = torch.exp(x - torch.where(top == -math.inf, torch.zeros_like(top), top))
    total = e.sum(-1, keepdim=True)
    return e / torch.where(total == 0, torch.ones_like(total), total)


def _allowed(s):
    """[B, n, rows]: what every drafted token attends."""
    c = s.c
    j = torch.arange(c.n, device="cuda")
    bits = ((s.mask[:, :, j // 64] >> (j % 64)) & 1).bool()                     # [B, n, n]
    at = torch.arange(s.cap, device="cuda")[None] - s.seq_len[:, None]          # [B, rows]: draft number, < 0 committed
    of = bits.gather(2, at.clamp(0, c.n - 1).long()[:, None].expand(c.B, c.n, s.cap))
    return (at < 0)[:, None] | (of & ((at >= 0) & (at < s.n_new[:, None]))[:, None])


def _tree(s):
    c = s.c
    G = c.Hq // c.Hkv
    k, v = _rows(s, s.kc).float(), _rows(s, s.vc).float()
    q = s.q.float().view(c.B, c.n, c.Hkv, G, c.D).permute(0, 2, 3, 1, 4).reshape(c.B, c.Hkv, G * c.n, c.D)
    x = (q @ k.transpose(2, 3)) * s.scale
    w = _softmax(x.view(c.B, c.Hkv, G, c.n, s.cap), _allowed(s)[:, None, None])
    o = (w.view(c.B, c.Hkv, G * c.n, s.cap) @ v).view(c.B, c.Hkv, G, c.n, c.D).permute(0, 3, 1, 2, 4).reshape(c.B, c.n, c.Hq * c.D)
    live = torch.arange(c.n, device="cuda")[None] < s.n_new[:, None]
    s.out = torch.where(live[..., None], o.to(s.out.dtype), s.out)
    return s.out


def _accept(s):
    c = s.c
    m = s.path.shape[1]
    i = torch.arange(m, device="cuda")
    to = (s.seq_len[:, None] + i).long()                                        # [B, m]
    fro = torch.where(i[None] < s.n_path[:, None], s.seq_len[:, None] + s.path, to).long()
    for t in (s.kc, s.vc):
        if s.table is None:
            b = torch.arange(c.B, device="cuda")[:, None]
            t[:, b, :, to] = t[:, b, :, fro]
        else:
            page = s.table.long()
            t[:, page.gather(1, to // c.page), :, to % c.page] = t[:, page.gather(1, fro // c.page), :, fro % c.page]
    s.new_len = s.seq_len + s.n_path
    return {"k": s.kc, "v": s.vc, "len": s.new_len}


def _scored(s):
    c = s.c
    G = c.Hq // c.Hkv
    k, v = _rows(s, s.kc).float(), _rows(s, s.vc).float()
    x = (s.q.float().view(c.B, c.Hkv, G, c.D) @ k.transpose(2, 3)) * s.scale
    w = _softmax(x, (torch.arange(s.cap, device="cuda")[None] < s.seq_len[:, None])[:, None, None])
    s.score = s.score + w.sum(2)
    return (w @ v).view(c.B, c.Hq * c.D).to(_T[c.out]), s.score


def _evict(s):
    c = s.c
    at = torch.arange(s.cap, device="cuda")
    n = s.seq_len[:, None]
    surely = ((at < c.sink) | (at >= n - c.recent)) & (at < n)
    key = torch.where(surely[:, None], math.inf, torch.where((at < n)[:, None], s.score0, -math.inf))
    keep = torch.sort(key, dim=-1, descending=True, stable=True)[1][..., : c.keep].sort(-1)[0]     # [B, Hkv, keep]
    new_len = s.seq_len.clamp(max=c.keep)
    score = torch.where((at >= new_len[:, None])[:, None] & (at < n)[:, None], 0.0, s.score0)
    live = torch.arange(keep.shape[-1], device="cuda") < new_len[:, None, None]
    score[..., : keep.shape[-1]] = torch.where(live, s.score0.gather(2, keep), score[..., : keep.shape[-1]])
    if s.table is None:
        for t in (s.kc, s.vc):
            t[:, :, : keep.shape[-1]] = t.gather(2, keep[..., None].expand(-1, -1, -1, c.D))
    else:
        h = torch.arange(c.Hkv, device="cuda")[None, :, None]
        page = s.table.long()[:, None].expand(c.B, c.Hkv, s.max_pages)
        to = torch.arange(keep.shape[-1], device="cuda").expand_as(keep)
        for t in (s.kc, s.vc):
            t[page.gather(2, to // c.page), h, to % c.page] = t[page.gather(2, keep // c.page), h, keep % c.page]
    kept = torch.where(live, keep, -1).to(torch.int32)
    if kept.shape[-1] < c.keep:
        kept = torch.nn.functional.pad(kept, (0, c.keep - kept.shape[-1]), value=-1)
    return {"k": s.kc, "v": s.vc, "score": score, "kept": kept, "len": new_len}


# ---------------------------------------------------------------------------------------------------- the library's calls
def _own(s):
    from nimllm_b200 import attention as A

    c = s.c
    if c.op == "rope_bwd":
        return A.rope_at_backward(s.q, s.k, s.cos, s.sin, n_head=c.Hq, n_kv_head=c.Hkv, head_dim=c.D, layout=c.layout)
    heads = dict(n_kv_head=c.Hkv, head_dim=c.D)
    if s.table is None:
        where = dict(seq_stride=c.Hkv * s.cap * c.D, head_stride=s.cap * c.D, max_seq=s.cap)
    if c.op == "rope":
        more = dict(n_head=c.Hq, layout=c.layout, pos=s.pos, row0=s.seq_len, q_out=s.q_out, **heads)
        if s.table is None:
            A.rope_append_at(s.q, s.k, s.v, s.cos, s.sin, k_cache=s.kc, v_cache=s.vc, **where, **more)
        else:
            A.rope_append_at_paged(s.q, s.k, s.v, s.cos, s.sin, s.kc, s.vc, s.table, **more)
        return {"q": s.q_out, "k": s.kc, "v": s.vc}
    if c.op == "tree":
        more = dict(n_head=c.Hq, seq_len=s.seq_len, max_len=s.max_len, n_new=s.n_new, tree_mask=s.mask, scale=s.scale, out=s.out, **heads)
        if s.table is None:
            return A.decode_tree(s.q, s.kc, s.vc, **where, **more)
        return A.decode_tree_paged(s.q, s.kc, s.vc, s.table, **more)
    if c.op == "accept":
        more = dict(n_draft=c.n, n_layer=c.L, new_len=s.new_len, **heads)
        if s.table is None:
            A.kv_accept(s.kc, s.vc, s.path, s.n_path, s.seq_len, layer_stride=c.B * c.Hkv * s.cap * c.D, **where, **more)
        else:
            A.kv_accept_paged(s.kc, s.vc, s.table, s.path, s.n_path, s.seq_len, **more)
        return {"k": s.kc, "v": s.vc, "len": s.new_len}
    if c.op == "scored":
        more = dict(n_head=c.Hq, seq_len=s.seq_len, max_len=s.max_len, scale=s.scale, out_dtype=_T[c.out], **heads)
        if s.table is None:
            return A.decode_scored(s.q, s.kc, s.vc, s.score, **where, **more), s.score
        return A.decode_scored_paged(s.q, s.kc, s.vc, s.table, s.score, **more), s.score
    score = s.score0.clone()
    more = dict(keep=c.keep, n_sink=c.sink, n_recent=c.recent, max_len=s.max_len, **heads)
    if s.table is None:
        new_len, kept = A.kv_evict(s.kc, s.vc, score, s.seq_len, **where, **more)
    else:
        new_len, kept = A.kv_evict_paged(s.kc, s.vc, s.table, score, s.seq_len, **more)
    return {"k": s.kc, "v": s.vc, "score": score, "kept": kept, "len": new_len}


_PLAIN = {"rope": _rope, "rope_bwd": _rope_bwd, "tree": _tree, "accept": _accept, "scored": _scored, "evict": _evict}


def run(s):
    if own:
        return _own(s)
    return _PLAIN[s.c.op](s)


# ---------------------------------------------------------------------------------------------------- in 64 bits
def exact(case, seed):
    """From the definitions, sequence by sequence.  Moved rows are copies: accept and evict have no computed numbers."""
    s = prepare(case, seed)
    c = s.c
    if c.op in ("accept", "evict"):
        return None
    if c.op == "rope_bwd":
        return tuple(_turn64(x, s, torch.arange(c.n, device="cuda").expand(c.B, c.n), -1) for x in (s.q, s.k))

    def block(t, b):
        """The rows of sequence b, [Hkv, rows, D]."""
        if s.table is None:
            return t[b].double()
        return t[s.table[b].long()].double().permute(1, 0, 2, 3).reshape(c.Hkv, s.cap, c.D)

    G = c.Hq // c.Hkv
    if c.op == "rope":
        q = _turn64(s.q, s, s.pos.clamp(min=0).long(), 1) * (s.pos >= 0)[..., None]
        kk = _turn64(s.k, s, s.pos.clamp(min=0).long(), 1).view(c.B, c.n, c.Hkv, c.D)
        kc, vc = s.kc.double(), s.vc.double()
        for b in range(c.B):
            m = s.n_new[b]
            row = torch.arange(s.lens_host[b], s.lens_host[b] + m, device="cuda")
            if s.table is None:
                kc[b, :, row] = kk[b, :m].transpose(0, 1)
                vc[b, :, row] = s.v[b, :m].double().view(m, c.Hkv, c.D).transpose(0, 1)
            else:
                page = s.table[b].long()[row // c.page]
                kc[page, :, row % c.page] = kk[b, :m]
                vc[page, :, row % c.page] = s.v[b, :m].double().view(m, c.Hkv, c.D)
        return {"q": q, "k": kc, "v": vc}
    if c.op == "tree":
        out = torch.zeros(c.B, c.n, c.Hq, c.D, device="cuda", dtype=torch.float64)
        n_new, mask = s.n_new.tolist(), s.mask.tolist()
        for b in range(c.B):
            n, m = s.lens_host[b], n_new[b]
            see = torch.zeros(m, n + m, dtype=torch.bool)
            see[:, :n] = True
            for i in range(m):
                x = sum((w & (2**64 - 1)) << (64 * k) for k, w in enumerate(mask[b][i]))
                see[i, n:] = torch.tensor([bool(x >> j & 1) for j in range(m)])
            kb, vb = block(s.kc, b)[:, : n + m], block(s.vc, b)[:, : n + m]
            q = s.q[b, :m].double().view(m, c.Hkv, G, c.D)
            x = torch.einsum("ihgd,hrd->hgir", q, kb) * s.scale
            x = x.masked_fill(~see.cuda(), -math.inf)
            out[b, :m] = torch.einsum("hgir,hrd->ihgd", torch.softmax(x, -1), vb).reshape(m, c.Hq, c.D)
        return out.flatten(2)
    out = torch.zeros(c.B, c.Hq * c.D, device="cuda", dtype=torch.float64)
    score = s.score.double()
    for b in range(c.B):
        n = s.lens_host[b]
        kb, vb = block(s.kc, b)[:, :n], block(s.vc, b)[:, :n]
        w = torch.softmax(torch.einsum("hgd,hrd->hgr", s.q[b].double().view(c.Hkv, G, c.D), kb) * s.scale, -1)
        out[b] = torch.einsum("hgr,hrd->hgd", w, vb).reshape(-1)
        score[b, :, :n] += w.sum(1)
    return out, score


def _turn64(x, s, pos, sign):
    """The rotation as a complex product."""
    c = s.c
    h = s.cos.shape[1]
    x = x.double().view(x.shape[0], x.shape[1], -1, c.D)
    r, rest = x[..., : 2 * h], x[..., 2 * h:]
    z = torch.complex(r[..., :h], r[..., h:]) if c.layout == "half" else torch.view_as_complex(r.reshape(*r.shape[:-1], h, 2).contiguous())
    z = z * torch.complex(s.cos.double(), sign * s.sin.double())[pos][:, :, None]
    r = torch.cat((z.real, z.imag), -1) if c.layout == "half" else torch.view_as_real(z).flatten(-2)
    return torch.cat((r, rest), -1).flatten(2)
