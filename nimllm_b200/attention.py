"""Host layer over the C ABI, named after the reference's procedures.

  reference (src/model.nim, src/gpu.nim)          here
  ------------------------------------------     ---------------------------------
  initModel's RoPE table loop (:153-163)          rope_tables()
  KvCache / initKvCache / resetKvCache (:70-73,   KvCache (one device allocation per K and V,
    :729-746)                                       [layer][seq][kv head][row][D])
  forward()'s attention block (:494-508)          attn_forward()
  forwardCached()'s attention block (:788-840)    attn_forward_cached()
  (no counterpart: batch 1 only)                  decode_batch(), combine()
  chat loop's reset-when-full cache policy        PagedKvPool (pages shared by many sequences),
    (src/chat.nim:86-91)                            rope_append_paged(), decode_paged()
  (no counterpart: row == position there)         rope_append_at(), decode_tree(), kv_accept(),
                                                    decode_scored(), kv_evict(), their _paged forms,
                                                    rope_tables_scaled(), rope_at_backward()

torch is used for device memory and streams only; every computation goes through
libnimllm_attn.so and raises if that library is missing or reports an error."""
from __future__ import annotations

import math
from typing import Optional

import numpy as np
import torch

from . import _lib
from ._lib import BF16, F32, check, lib

_DT = {torch.float32: F32, torch.bfloat16: BF16}


def _code(t: torch.Tensor) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise _lib.NimllmAttnError(f"unsupported dtype {t.dtype}: float32 and bfloat16 are built") from None


def _ptr(t: Optional[torch.Tensor]):
    if t is None:
        return None
    if not t.is_cuda:
        raise _lib.NimllmAttnError("device tensor expected (there is no CPU path)")
    if not t.is_contiguous():
        raise _lib.NimllmAttnError("contiguous tensor expected")
    return t.data_ptr()


def _stream() -> int:
    return torch.cuda.current_stream().cuda_stream


class _Arena:
    """Caller-owned scratch, the role trackedCreate's arena plays in the reference
    (src/autograd.nim:37-51): grown outside the hot loop, reused by every call."""

    def __init__(self):
        self.buf = {}

    def get(self, nbytes: int, device) -> Optional[torch.Tensor]:
        if nbytes == 0:
            return None
        key = torch.device(device).index or 0
        cur = self.buf.get(key)
        if cur is None or cur.numel() < nbytes:
            cur = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
            self.buf[key] = cur
        return cur


_arena = _Arena()


def rope_tables(max_pos: int, head_dim: int, base: float, device="cuda"):
    """cos/sin tables [max_pos, D/2] fp32, computed on the host as initModel does."""
    cos = np.empty((max_pos, head_dim // 2), np.float32)
    sin = np.empty_like(cos)
    check(lib().nimllm_rope_tables_host(cos.ctypes.data, sin.ctypes.data, max_pos, head_dim, float(base)))
    return torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device)


class KvCache:
    """K and V as [n_layer, n_seq, Hkv, max_seq, D] device tensors plus the host `pos`."""

    def __init__(self, n_layer, n_seq, n_kv_head, max_seq, head_dim, dtype=torch.float32, device="cuda"):
        shape = (n_layer, n_seq, n_kv_head, max_seq, head_dim)
        self.k = torch.zeros(shape, dtype=dtype, device=device)
        self.v = torch.zeros(shape, dtype=dtype, device=device)
        self.pos = 0
        self.n_layer, self.n_seq, self.n_kv_head, self.max_seq, self.head_dim = shape
        self.seq_stride = n_kv_head * max_seq * head_dim
        self.head_stride = max_seq * head_dim

    def reset(self):
        self.k.zero_()
        self.v.zero_()
        self.pos = 0


class _DeviceView:
    """Device memory owned by the library, shown to torch through __cuda_array_interface__."""

    def __init__(self, ptr, shape, typestr, owner):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr, "data": (int(ptr), False), "version": 2}
        self._owner = owner


class PagedKvPool:
    """The library's block manager of the paged cache (nimllm_kvpool_*): pages shared by up to max_seqs
    sequences instead of the reference's one-conversation cache that is reset when full
    (src/chat.nim:86-91).  on_device=False keeps only the host table (no CUDA call)."""

    def __init__(self, n_layer, n_pages, page_rows, n_kv_head, head_dim, max_seqs, max_pages_per_seq,
                 dtype=torch.bfloat16, on_device=True):
        self.shape = (n_pages, n_kv_head, page_rows, head_dim)
        self.n_layer, self.max_seqs, self.max_pages, self.dtype, self.on_device = n_layer, max_seqs, max_pages_per_seq, dtype, on_device
        self._h = lib().nimllm_kvpool_create(n_layer, n_pages, page_rows, n_kv_head, head_dim, _DT[dtype], max_seqs,
                                             max_pages_per_seq, int(on_device))
        if not self._h:
            raise _lib.NimllmAttnError(lib().nimllm_attn_last_error().decode())

    def close(self):
        if self._h:
            lib().nimllm_kvpool_destroy(self._h)
            self._h = None

    __del__ = close

    def reserve(self, seq: int, rows_total: int):
        check(lib().nimllm_kvpool_reserve(self._h, seq, rows_total))

    def release(self, seq: int):
        check(lib().nimllm_kvpool_release(self._h, seq))

    def shrink(self, seq: int, rows_total: int):
        check(lib().nimllm_kvpool_shrink(self._h, seq, rows_total))

    def sync(self):
        check(lib().nimllm_kvpool_sync(self._h, _stream() if self.on_device else None))

    @property
    def free_pages(self) -> int:
        return lib().nimllm_kvpool_free_pages(self._h)

    def seq_pages(self, seq: int) -> int:
        return lib().nimllm_kvpool_seq_pages(self._h, seq)

    def seq_rows(self, seq: int) -> int:
        return lib().nimllm_kvpool_seq_rows(self._h, seq)

    def table_host(self) -> np.ndarray:
        import ctypes
        buf = (ctypes.c_int32 * (self.max_seqs * self.max_pages)).from_address(lib().nimllm_kvpool_table_host(self._h))
        return np.frombuffer(buf, dtype=np.int32).reshape(self.max_seqs, self.max_pages).copy()

    def table(self, first_seq: int = 0) -> torch.Tensor:
        ptr = lib().nimllm_kvpool_table(self._h, first_seq)
        if not ptr:
            raise _lib.NimllmAttnError("the pool has no device table (on_device=False or bad first_seq)")
        return torch.as_tensor(_DeviceView(ptr, (self.max_seqs - first_seq, self.max_pages), "<i4", self), device="cuda")

    def _pages(self, fn, layer):
        ptr = fn(self._h, layer)
        if not ptr:
            raise _lib.NimllmAttnError("the pool has no device pages (on_device=False or bad layer)")
        if self.dtype == torch.float32:
            return torch.as_tensor(_DeviceView(ptr, self.shape, "<f4", self), device="cuda")
        return torch.as_tensor(_DeviceView(ptr, self.shape, "<i2", self), device="cuda").view(torch.bfloat16)

    def k(self, layer: int) -> torch.Tensor:
        return self._pages(lib().nimllm_kvpool_k, layer)

    def v(self, layer: int) -> torch.Tensor:
        return self._pages(lib().nimllm_kvpool_v, layer)


def rope_append(q, k_new, v_new, cos, sin, *, n_head, n_kv_head, head_dim, pos0=0, seq_pos=None,
                k_cache=None, v_cache=None, kv_off=None, seq_stride=0, head_stride=0, cache_row0=0,
                max_seq=0, write_back_k=True):
    """Fused RoPE(q), RoPE(k_new) + cast + scatter of k_new / v_new into the cache."""
    B, n = k_new.shape[0], k_new.shape[1]
    check(lib().nimllm_rope_append(
        _ptr(q), n_head, _ptr(k_new), _ptr(v_new), _code(k_new), int(write_back_k), _ptr(cos), _ptr(sin),
        _ptr(seq_pos), pos0, _ptr(k_cache), _ptr(v_cache), _code(k_cache) if k_cache is not None else F32,
        _ptr(kv_off), seq_stride, head_stride, cache_row0, max_seq, B, n, n_kv_head, head_dim, _stream()))


def decode_batch(q, k_cache, v_cache, *, n_head, n_kv_head, head_dim, max_len, seq_len=None, kv_off=None,
                 seq_stride=0, head_stride=0, scale=None, chunk_rows=0, out=None, out_dtype=torch.float32,
                 partials=False):
    """GQA decode of a batch of independent sequences. Returns out [B, Hq*D] (and the
    (o, m, l) records [B*Hq, D+4] when partials=True)."""
    B = q.shape[0]
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    if out is None:
        out = torch.empty((B, n_head * head_dim), dtype=out_dtype, device=q.device)
    rec = torch.empty((B * n_head, head_dim + 4), dtype=torch.float32, device=q.device) if partials else None
    need = lib().nimllm_attn_decode_workspace_bytes(B, n_head, n_kv_head, head_dim, max_len, chunk_rows)
    ws = _arena.get(need, q.device)
    check(lib().nimllm_attn_decode(
        _ptr(q), _code(q), _ptr(k_cache), _ptr(v_cache), _code(k_cache), _ptr(kv_off), seq_stride, head_stride,
        _ptr(seq_len), max_len, _ptr(out), _code(out), _ptr(rec), B, n_head, n_kv_head, head_dim, scale,
        chunk_rows, _ptr(ws), need, _stream()))
    return (out, rec) if partials else out


def decode_paged(q, k_pages, v_pages, page_table, *, n_head, n_kv_head, head_dim, max_len, seq_len=None, scale=None,
                 out=None, out_dtype=torch.float32, partials=False):
    """GQA decode over a paged bf16 cache: k_pages / v_pages [n_pages, Hkv, page_rows, D], page_table
    int32 [B, max_pages].  Returns out [B, Hq*D] (and the (o, m, l) records when partials=True)."""
    B = q.shape[0]
    page_rows = k_pages.shape[2]
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    if out is None:
        out = torch.empty((B, n_head * head_dim), dtype=out_dtype, device=q.device)
    rec = torch.empty((B * n_head, head_dim + 4), dtype=torch.float32, device=q.device) if partials else None
    need = lib().nimllm_attn_decode_workspace_bytes(B, n_head, n_kv_head, head_dim, max_len, 0)
    ws = _arena.get(need, q.device)
    check(lib().nimllm_attn_decode_paged(
        _ptr(q), _code(q), _ptr(k_pages), _ptr(v_pages), _ptr(page_table), page_table.shape[1], page_rows,
        _ptr(seq_len), max_len, _ptr(out), _code(out), _ptr(rec), B, n_head, n_kv_head, head_dim, scale,
        _ptr(ws), need, _stream()))
    return (out, rec) if partials else out


def rope_append_paged(q, k_new, v_new, cos, sin, k_pages, v_pages, page_table, *, n_head, n_kv_head, head_dim,
                      pos0=0, seq_pos=None, write_back_k=True):
    """rope_append into a paged cache: k_pages / v_pages [n_pages, Hkv, page_rows, D], page_table int32
    [B, max_pages]; every new row finds its own page, so n > 1 may cross page boundaries."""
    B, n = k_new.shape[0], k_new.shape[1]
    check(lib().nimllm_rope_append_paged(
        _ptr(q), n_head, _ptr(k_new), _ptr(v_new), _code(k_new), int(write_back_k), _ptr(cos), _ptr(sin),
        _ptr(seq_pos), pos0, _ptr(k_pages), _ptr(v_pages), _code(k_pages), _ptr(page_table), page_table.shape[1],
        k_pages.shape[2], k_pages.shape[0], B, n, n_kv_head, head_dim, _stream()))


# ---- a cache whose rows are not its positions: drafted trees and evicted caches -------------------------------------
_LAYOUT = {"half": _lib.ROPE_HALF, "interleaved": _lib.ROPE_INTERLEAVED}
_SCALE_KIND = {"none": _lib.ROPE_SCALE_NONE, "linear": _lib.ROPE_SCALE_LINEAR, "base": _lib.ROPE_SCALE_BASE,
               "ramp": _lib.ROPE_SCALE_RAMP}


def _layout(name):
    try:
        return _LAYOUT[name]
    except KeyError:
        raise _lib.NimllmAttnError(f"unknown layout {name!r}: 'half' and 'interleaved' are built") from None


def _refuse(t, dtype, index):
    _ptr(t)
    if t.get_device() != index:
        raise _lib.NimllmAttnError(f"tensors on cuda:{t.get_device()} and on cuda:{index}")
    raise _lib.NimllmAttnError(f"{dtype} tensor expected, got {t.dtype}")


def _args(index, dtypes, tensors):
    """Data pointers of contiguous tensors on device `index`, each of its dtype (None: any).  None stays None."""
    ptrs = []
    for t, dt in zip(tensors, dtypes):
        if t is None:
            ptrs.append(None)
        else:
            if t.get_device() != index or (dt is not None and t.dtype is not dt) or not t.is_contiguous():
                _refuse(t, dt, index)
            ptrs.append(t.data_ptr())
    return ptrs


def _small(name, t, least):
    raise _lib.NimllmAttnError(f"{name} holds {t.numel()} elements, {least} are needed")


def _block_end(batch, n_kv_head, head_dim, seq_stride, head_stride, max_seq, layers=0, layer_stride=0):
    """Elements that the blocks of a contiguous cache without kv_off reach over, from its first element on."""
    if (seq_stride < 0 and batch > 1) or (head_stride < 0 and n_kv_head > 1) or (layer_stride < 0 and layers > 1):
        raise _lib.NimllmAttnError(f"seq_stride {seq_stride}, head_stride {head_stride}, layer_stride {layer_stride}: a cache starts with its first block")
    return (layers - 1 if layers > 1 else 0) * layer_stride + (batch - 1) * seq_stride + (n_kv_head - 1) * head_stride + max_seq * head_dim


def _check_blocks(k_cache, v_cache, end):
    if k_cache.numel() < end:
        _small("k_cache", k_cache, end)
    if v_cache.numel() < end:
        _small("v_cache", v_cache, end)


class _Here:
    """The context of a call whose tensors are on the current device."""

    def __enter__(self):
        pass

    def __exit__(self, *a):
        pass


_here = _Here()


def _on(t):
    """(device index, the context in which a call for tensors on it launches)"""
    index = t.get_device()
    if index < 0:
        raise _lib.NimllmAttnError("device tensor expected (there is no CPU path)")
    return index, _here if index == torch.cuda.current_device() else torch.cuda.device(index)


# the handle of the current stream, without building a Stream object (3 us) where torch has a way
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (lambda index: torch.cuda.current_stream(index).cuda_stream)


def _scratch(nbytes, device):
    # from the caching allocator of the current stream, so calls on two streams or in two graphs never share it
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def rope_tables_scaled(max_pos: int, rot_dim: int, base: float, *, kind="none", factor=1.0, low=1.0, high=32.0, orig_len=0,
                       gain=1.0, device="cuda"):
    """cos/sin tables [max_pos, rot_dim/2] for positions past the trained length: kind "linear" divides every frequency
    by factor, "base" stretches the base, "ramp" interpolates between both by the turns a frequency makes over orig_len
    positions (kept at `high` turns and more, divided at `low` and fewer)."""
    cos = np.empty((max_pos, rot_dim // 2), np.float32)
    sin = np.empty_like(cos)
    if kind not in _SCALE_KIND:
        raise _lib.NimllmAttnError(f"unknown kind {kind!r}: {sorted(_SCALE_KIND)} are built")
    check(lib().nimllm_rope_tables_scaled_host(cos.ctypes.data, sin.ctypes.data, max_pos, rot_dim, float(base), _SCALE_KIND[kind],
                                               float(factor), float(low), float(high), int(orig_len), float(gain)))
    return torch.from_numpy(cos).to(device), torch.from_numpy(sin).to(device)


_F32, _I32, _I64 = torch.float32, torch.int32, torch.int64


def _rope_at(index, q, k_new, v_new, cos, sin, n_head, n_kv_head, head_dim, layout, pos, row0, q_out, k_out, want_k, has_cache):
    B, n = k_new.shape[:2]
    if q is not None and q_out is None:
        q_out = torch.empty_like(q)
    if k_out is None and (want_k or not has_cache):
        k_out = torch.empty_like(k_new)
    act, tokens = k_new.dtype, B * n
    qs, kv = tokens * n_head * head_dim, tokens * n_kv_head * head_dim
    p = _args(index, (act, act, act, act, act, _F32, _F32, _I32, _I32), (q, q_out, k_new, k_out, v_new, cos, sin, pos, row0))
    if q is not None:
        if q.numel() < qs:
            _small("q", q, qs)
        if q_out.numel() < qs:
            _small("q_out", q_out, qs)
    if k_new.numel() < kv:
        _small("k_new", k_new, kv)
    if k_out is not None and k_out.numel() < kv:
        _small("k_out", k_out, kv)
    if v_new is not None and v_new.numel() < kv:
        _small("v_new", v_new, kv)
    if pos is not None and pos.numel() < tokens:
        _small("pos", pos, tokens)
    if row0 is not None and row0.numel() < B:
        _small("row0", row0, B)
    rows = rot = 0
    if cos is not None:
        rows, rot = cos.shape
        if sin is not None and sin.shape != cos.shape:
            raise _lib.NimllmAttnError("cos and sin differ in shape")
    return B, n, q_out if q is not None else None, k_out, (p[0], p[1], n_head, p[2], p[3], p[4], _code(k_new), p[5], p[6], 2 * rot,
                                                           _layout(layout), rows, p[7], p[8])


def rope_append_at(q, k_new, v_new, cos, sin, *, n_head, n_kv_head, head_dim, layout="half", pos=None, row0=None, first_row=0,
                   k_cache=None, v_cache=None, kv_off=None, seq_stride=0, head_stride=0, max_seq=0, q_out=None, k_out=None,
                   want_k=False):
    """Rotates q and k_new [B, n, heads*D] at pos [B, n] (int32; negative: padding, left alone) and appends k and v at the
    rows row0[b] + t.  cos/sin [rows, R/2] rotate the first R columns of every head.  Returns (q_out, k_out)."""
    index, here = _on(k_new)
    with here:
        B, n, q_out, k_out, head = _rope_at(index, q, k_new, v_new, cos, sin, n_head, n_kv_head, head_dim, layout, pos, row0, q_out,
                                            k_out, want_k, k_cache is not None)
        kc = vc = off = None
        code = F32
        if (k_cache is None) != (v_cache is None):
            raise _lib.NimllmAttnError("give both k_cache and v_cache or neither")
        if k_cache is not None:
            kc, vc, off = _args(index, (None, k_cache.dtype, _I64), (k_cache, v_cache, kv_off))
            code = _code(k_cache)
            if kv_off is None:
                _check_blocks(k_cache, v_cache, _block_end(B, n_kv_head, head_dim, seq_stride, head_stride, max_seq))
            elif kv_off.numel() < B:
                _small("kv_off", kv_off, B)
        check(lib().nimllm_rope_append_at(*head, first_row, kc, vc, code, off, seq_stride, head_stride, max_seq, B, n, n_kv_head, head_dim,
                                          _raw_stream(index)))
    return q_out, k_out


def _pages(index, k_pages, v_pages, page_table, batch, n_kv_head, head_dim, layers=None):
    """(pointers of K, V and the table, max_pages, page_rows, n_pages) of pages [n_pages, Hkv, page_rows, D], checked against the
    heads and the table; a layer axis in front only for a call that says how many layers it means (or where it has one entry)."""
    shape = k_pages.shape
    if layers is None and len(shape) == 5 and shape[0] != 1:
        raise _lib.NimllmAttnError(f"pages {tuple(shape)}: this call works on one layer, give pages[layer]")
    layers = layers or 1
    n_pages, heads, page_rows, width = shape[-4:] if len(shape) in (4, 5) else (0, 0, 0, 0)
    if heads != n_kv_head or width != head_dim or v_pages.shape != shape:
        raise _lib.NimllmAttnError(f"pages {tuple(shape)} / {tuple(v_pages.shape)}: [n_pages, {n_kv_head}, page_rows, {head_dim}] expected")
    if (shape[0] if len(shape) == 5 else 1) < layers:
        raise _lib.NimllmAttnError(f"pages {tuple(shape)}: {layers} layers expected")
    if page_table.dim() != 2 or page_table.shape[0] < batch:
        raise _lib.NimllmAttnError(f"page_table {tuple(page_table.shape)}: [{batch}, max_pages] expected")
    kp, vp, pt = _args(index, (None, k_pages.dtype, _I32), (k_pages, v_pages, page_table))
    return kp, vp, pt, page_table.shape[1], page_rows, n_pages


def rope_append_at_paged(q, k_new, v_new, cos, sin, k_pages, v_pages, page_table, *, n_head, n_kv_head, head_dim, layout="half",
                         pos=None, row0=None, first_row=0, q_out=None, k_out=None, want_k=False):
    """rope_append_at into pages [n_pages, Hkv, page_rows, D] with page_table int32 [B, max_pages]."""
    index, here = _on(k_new)
    with here:
        B, n, q_out, k_out, head = _rope_at(index, q, k_new, v_new, cos, sin, n_head, n_kv_head, head_dim, layout, pos, row0, q_out,
                                            k_out, want_k, True)
        kp, vp, pt, max_pages, page_rows, n_pages = _pages(index, k_pages, v_pages, page_table, B, n_kv_head, head_dim)
        check(lib().nimllm_rope_append_at_paged(*head, first_row, kp, vp, _code(k_pages), pt, max_pages, page_rows, n_pages, B, n, n_kv_head,
                                                head_dim, _raw_stream(index)))
    return q_out, k_out


def rope_at_backward(dq_rot, dk_rot, cos, sin, *, n_head, n_kv_head, head_dim, layout="half", pos=None, pos0=0, in_place=False):
    """Gradient of the rotation: (dq, dk) from the gradients of the rotated q and k [B, n, heads*D] (either may be None).
    Tokens without a position get zeros."""
    some = dq_rot if dq_rot is not None else dk_rot
    if some is None:
        raise _lib.NimllmAttnError("dq_rot or dk_rot is required")
    B, n = some.shape[:2]
    index, here = _on(some)
    with here:
        dq = dq_rot if in_place or dq_rot is None else torch.empty_like(dq_rot)
        dk = dk_rot if in_place or dk_rot is None else torch.empty_like(dk_rot)
        if dq_rot is not None and dq_rot.numel() < B * n * n_head * head_dim:
            _small("dq_rot", dq_rot, B * n * n_head * head_dim)
        if dk_rot is not None and dk_rot.numel() < B * n * n_kv_head * head_dim:
            _small("dk_rot", dk_rot, B * n * n_kv_head * head_dim)
        if pos is not None and pos.numel() < B * n:
            _small("pos", pos, B * n)
        if cos.shape != sin.shape:
            raise _lib.NimllmAttnError("cos and sin differ in shape")
        dt = some.dtype
        p = _args(index, (dt, dt, dt, dt, _F32, _F32, _I32), (dq_rot, dq, dk_rot, dk, cos, sin, pos))
        check(lib().nimllm_rope_at_bwd(p[0], p[1], n_head, p[2], p[3], _code(some), p[4], p[5], 2 * cos.shape[1], _layout(layout),
                                       cos.shape[0], p[6], pos0, B, n, n_kv_head, head_dim, _raw_stream(index)))
    return dq, dk


def _tree_io(index, q, n_new, tree_mask, seq_len, out, out_dtype, partials, n_head, head_dim):
    B, n = q.shape[:2]
    size = B * n * n_head * head_dim
    if out is None:
        # with n_new the rows of padding tokens are not written
        out = (torch.empty if n_new is None else torch.zeros)((B, n, n_head * head_dim), dtype=out_dtype, device=q.device)
    rec = (torch.empty if n_new is None else torch.zeros)((B * n * n_head, head_dim + 4), dtype=torch.float32, device=q.device) if partials else None
    p = _args(index, (None, _I32, _I32, _I64, None, _F32), (q, seq_len, n_new, tree_mask, out, rec))
    if q.numel() < size:
        _small("q", q, size)
    if out.numel() < size:
        _small("out", out, size)
    if seq_len is not None and seq_len.numel() < B:
        _small("seq_len", seq_len, B)
    if n_new is not None and n_new.numel() < B:
        _small("n_new", n_new, B)
    if tree_mask is not None and tree_mask.numel() < B * n * ((n + 63) // 64):
        _small("tree_mask", tree_mask, B * n * ((n + 63) // 64))
    return B, n, out, rec, p


def decode_tree(q, k_cache, v_cache, *, n_head, n_kv_head, head_dim, max_len, max_seq, seq_len=None, n_new=None, tree_mask=None,
                kv_off=None, seq_stride=0, head_stride=0, scale=None, out=None, out_dtype=torch.float32, partials=False):
    """Attention of the drafted tokens q [B, n, Hq*D]: token i of sequence b attends its seq_len[b] committed rows and the
    draft rows seq_len[b] + j with bit j set in tree_mask [B, n, ceil(n/64)] (int64; None: drafts 0 .. i).  Returns out
    [B, n, Hq*D] (and the (o, m, l) records [B*n*Hq, D+4] when partials=True)."""
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    index, here = _on(q)
    with here:
        B, n, out, rec, p = _tree_io(index, q, n_new, tree_mask, seq_len, out, out_dtype, partials, n_head, head_dim)
        kc, vc, off = _args(index, (None, k_cache.dtype, _I64), (k_cache, v_cache, kv_off))
        if kv_off is None:
            _check_blocks(k_cache, v_cache, _block_end(B, n_kv_head, head_dim, seq_stride, head_stride, max_seq))
        elif kv_off.numel() < B:
            _small("kv_off", kv_off, B)
        code, L = _code(k_cache), lib()
        need = L.nimllm_attn_decode_tree_workspace_bytes(B, n, n_head, n_kv_head, head_dim, max_len, code)
        ws = _scratch(need, q.device) if need else None
        check(L.nimllm_attn_decode_tree(
            p[0], _code(q), kc, vc, code, off, seq_stride, head_stride, max_seq, p[1], max_len, p[2], p[3], p[4], _code(out), p[5], B, n,
            n_head, n_kv_head, head_dim, scale, ws.data_ptr() if need else None, need, _raw_stream(index)))
    return (out, rec) if partials else out


def decode_tree_paged(q, k_pages, v_pages, page_table, *, n_head, n_kv_head, head_dim, max_len, seq_len=None, n_new=None,
                      tree_mask=None, scale=None, out=None, out_dtype=torch.float32, partials=False):
    """decode_tree over pages [n_pages, Hkv, page_rows, D] with page_table int32 [B, max_pages]."""
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    index, here = _on(q)
    with here:
        B, n, out, rec, p = _tree_io(index, q, n_new, tree_mask, seq_len, out, out_dtype, partials, n_head, head_dim)
        kp, vp, pt, max_pages, page_rows, n_pages = _pages(index, k_pages, v_pages, page_table, B, n_kv_head, head_dim)
        code, L = _code(k_pages), lib()
        need = L.nimllm_attn_decode_tree_workspace_bytes(B, n, n_head, n_kv_head, head_dim, max_len, code)
        ws = _scratch(need, q.device) if need else None
        check(L.nimllm_attn_decode_tree_paged(
            p[0], _code(q), kp, vp, code, pt, max_pages, page_rows, n_pages, p[1], max_len, p[2], p[3], p[4], _code(out), p[5], B, n, n_head,
            n_kv_head, head_dim, scale, ws.data_ptr() if need else None, need, _raw_stream(index)))
    return (out, rec) if partials else out


def decode_tree_status(reset: bool = True) -> int:
    """0 when every tree and scored decode over a bf16 cache on the current device since the last reset ran to completion,
    1 when a bounded wait inside one gave up (its outputs are incomplete).  Synchronises."""
    rc = lib().nimllm_attn_decode_tree_status(int(reset))
    if rc < 0:
        check(-rc)
    return rc


def _accept_io(index, path, n_path, seq_len, new_len):
    B, max_path = path.shape
    new_len = torch.empty_like(seq_len) if new_len is None else new_len
    p = _args(index, (_I32, _I32, _I32, _I32), (path, n_path, seq_len, new_len))
    if n_path.numel() < B or seq_len.numel() < B or new_len.numel() < B:
        raise _lib.NimllmAttnError(f"n_path, seq_len and new_len hold {B} elements each")
    return B, max_path, new_len, p


def kv_accept(k_cache, v_cache, path, n_path, seq_len, *, n_draft, n_kv_head, head_dim, max_seq, n_layer=1, layer_stride=0,
              kv_off=None, seq_stride=0, head_stride=0, new_len=None):
    """Moves the rows of the accepted drafts path[b][:n_path[b]] (int32 [B, max_path], increasing) down to the rows from
    seq_len[b] on, in n_layer layers, and returns new_len [B] (given: written there; it may be seq_len)."""
    index, here = _on(path)
    with here:
        B, max_path, new_len, p = _accept_io(index, path, n_path, seq_len, new_len)
        kc, vc, off = _args(index, (None, k_cache.dtype, _I64), (k_cache, v_cache, kv_off))
        if kv_off is None:
            _check_blocks(k_cache, v_cache, _block_end(B, n_kv_head, head_dim, seq_stride, head_stride, max_seq, n_layer, layer_stride))
        elif kv_off.numel() < B:
            _small("kv_off", kv_off, B)
        check(lib().nimllm_kv_accept(kc, vc, _code(k_cache), n_layer, layer_stride, off, seq_stride, head_stride, max_seq, p[0],
                                     max_path, p[1], p[2], p[3], n_draft, B, n_kv_head, head_dim, _raw_stream(index)))
    return new_len


def kv_accept_paged(k_pages, v_pages, page_table, path, n_path, seq_len, *, n_draft, n_kv_head, head_dim, n_layer=1, new_len=None):
    """kv_accept over pages [(n_layer,) n_pages, Hkv, page_rows, D]; all layers share the page table."""
    index, here = _on(path)
    with here:
        B, max_path, new_len, p = _accept_io(index, path, n_path, seq_len, new_len)
        kp, vp, pt, max_pages, page_rows, n_pages = _pages(index, k_pages, v_pages, page_table, B, n_kv_head, head_dim, n_layer)
        check(lib().nimllm_kv_accept_paged(kp, vp, _code(k_pages), n_layer, n_pages * n_kv_head * page_rows * head_dim, pt, max_pages,
                                           page_rows, n_pages, p[0], max_path, p[1], p[2], p[3], n_draft, B, n_kv_head, head_dim,
                                           _raw_stream(index)))
    return new_len


def _scored_io(index, q, score, seq_len, out, out_dtype, n_head, n_kv_head, head_dim):
    B, size = q.shape[0], q.shape[0] * n_head * head_dim
    shape = score.shape
    if len(shape) != 3 or shape[0] < B or shape[1] != n_kv_head:
        raise _lib.NimllmAttnError(f"score {tuple(shape)}: [{B}, {n_kv_head}, rows] expected")
    if out is None:
        out = torch.empty((B, n_head * head_dim), dtype=out_dtype, device=q.device)
    p = _args(index, (None, _I32, None, _F32), (q, seq_len, out, score))
    if q.numel() < size:
        _small("q", q, size)
    if out.numel() < size:
        _small("out", out, size)
    if seq_len is not None and seq_len.numel() < B:
        _small("seq_len", seq_len, B)
    return B, out, shape[2], p


def decode_scored(q, k_cache, v_cache, score, *, n_head, n_kv_head, head_dim, max_len, max_seq, seq_len=None, decay=1.0, kv_off=None,
                  seq_stride=0, head_stride=0, scale=None, out=None, out_dtype=torch.float32):
    """decode_batch that also updates score [B, Hkv, rows] (fp32): decay * score + the softmax weights of the query heads
    of each KV head, summed.  Returns out [B, Hq*D]."""
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    index, here = _on(q)
    with here:
        B, out, score_rows, p = _scored_io(index, q, score, seq_len, out, out_dtype, n_head, n_kv_head, head_dim)
        kc, vc, off = _args(index, (None, k_cache.dtype, _I64), (k_cache, v_cache, kv_off))
        if kv_off is None:
            _check_blocks(k_cache, v_cache, _block_end(B, n_kv_head, head_dim, seq_stride, head_stride, max_seq))
        elif kv_off.numel() < B:
            _small("kv_off", kv_off, B)
        code, L = _code(k_cache), lib()
        need = L.nimllm_attn_decode_scored_workspace_bytes(B, n_head, n_kv_head, head_dim, max_len, code)
        ws = _scratch(need, q.device)
        check(L.nimllm_attn_decode_scored(
            p[0], _code(q), kc, vc, code, off, seq_stride, head_stride, max_seq, p[1], max_len, p[2], _code(out), p[3], score_rows, decay,
            B, n_head, n_kv_head, head_dim, scale, ws.data_ptr(), need, _raw_stream(index)))
    return out


def decode_scored_paged(q, k_pages, v_pages, page_table, score, *, n_head, n_kv_head, head_dim, max_len, seq_len=None, decay=1.0,
                        scale=None, out=None, out_dtype=torch.float32):
    """decode_scored over pages [n_pages, Hkv, page_rows, D] with page_table int32 [B, max_pages]."""
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    index, here = _on(q)
    with here:
        B, out, score_rows, p = _scored_io(index, q, score, seq_len, out, out_dtype, n_head, n_kv_head, head_dim)
        kp, vp, pt, max_pages, page_rows, n_pages = _pages(index, k_pages, v_pages, page_table, B, n_kv_head, head_dim)
        code, L = _code(k_pages), lib()
        need = L.nimllm_attn_decode_scored_workspace_bytes(B, n_head, n_kv_head, head_dim, max_len, code)
        ws = _scratch(need, q.device)
        check(L.nimllm_attn_decode_scored_paged(
            p[0], _code(q), kp, vp, code, pt, max_pages, page_rows, n_pages, p[1], max_len, p[2], _code(out), p[3], score_rows, decay, B,
            n_head, n_kv_head, head_dim, scale, ws.data_ptr(), need, _raw_stream(index)))
    return out


def _evict_io(index, score, seq_len, keep, kept, new_len, n_kv_head, batch):
    shape = score.shape
    B = shape[0] if batch is None else batch
    if len(shape) != 3 or shape[0] < B or shape[1] != n_kv_head:
        raise _lib.NimllmAttnError(f"score {tuple(shape)}: [{B}, {n_kv_head}, rows] expected")
    if kept is None:
        kept = torch.empty((B, n_kv_head, max(keep, 0)), dtype=_I32, device=score.device)
    if new_len is None:
        new_len = torch.empty(B, dtype=_I32, device=score.device)
    p = _args(index, (_F32, _I32, _I32, _I32), (score, seq_len, kept, new_len))
    if kept.numel() < B * n_kv_head * keep:
        _small("kept", kept, B * n_kv_head * keep)
    if new_len.numel() < B or (seq_len is not None and seq_len.numel() < B):
        raise _lib.NimllmAttnError(f"seq_len and new_len hold {B} elements each")
    return B, shape[2], kept, new_len, p


def kv_evict(k_cache, v_cache, score, seq_len, *, keep, n_kv_head, head_dim, max_len, max_seq, n_sink=0, n_recent=0, kv_off=None,
             seq_stride=0, head_stride=0, kept=None, new_len=None, batch=None):
    """Cuts every sequence to `keep` rows: per KV head the first n_sink, the last n_recent and those with the largest
    score [B, Hkv, rows] in between, in order; K, V and score move.  Returns (new_len [B], kept [B, Hkv, keep])."""
    index, here = _on(score)
    with here:
        B, score_rows, kept, new_len, p = _evict_io(index, score, seq_len, keep, kept, new_len, n_kv_head, batch)
        kc, vc, off = _args(index, (None, k_cache.dtype, _I64), (k_cache, v_cache, kv_off))
        if kv_off is None:
            _check_blocks(k_cache, v_cache, _block_end(B, n_kv_head, head_dim, seq_stride, head_stride, max_seq))
        elif kv_off.numel() < B:
            _small("kv_off", kv_off, B)
        check(lib().nimllm_kv_evict(kc, vc, _code(k_cache), off, seq_stride, head_stride, max_seq, p[0], score_rows, p[1], max_len,
                                    keep, n_sink, n_recent, p[2], p[3], B, n_kv_head, head_dim, _raw_stream(index)))
    return new_len, kept


def kv_evict_paged(k_pages, v_pages, page_table, score, seq_len, *, keep, n_kv_head, head_dim, max_len, n_sink=0, n_recent=0, kept=None,
                   new_len=None, batch=None):
    """kv_evict over pages [n_pages, Hkv, page_rows, D]; give the empty pages back with PagedKvPool.shrink."""
    index, here = _on(score)
    with here:
        B, score_rows, kept, new_len, p = _evict_io(index, score, seq_len, keep, kept, new_len, n_kv_head, batch)
        kp, vp, pt, max_pages, page_rows, n_pages = _pages(index, k_pages, v_pages, page_table, B, n_kv_head, head_dim)
        check(lib().nimllm_kv_evict_paged(kp, vp, _code(k_pages), pt, max_pages, page_rows, n_pages, p[0], score_rows, p[1], max_len, keep,
                                          n_sink, n_recent, p[2], p[3], B, n_kv_head, head_dim, _raw_stream(index)))
    return new_len, kept


def _wtype(w, w_type):
    if w_type is not None:
        return w_type
    return {torch.float32: _lib.W_F32, torch.bfloat16: _lib.W_BF16}[w.dtype]


def qkv_rope_append(x_norm, wq, wk, wv, cos, sin, *, n_head, n_kv_head, head_dim, w_type=None, pos0=0, seq_pos=None,
                    k_cache=None, v_cache=None, kv_off=None, seq_stride=0, head_stride=0, cache_row0=0, max_seq=0,
                    want_kv=False):
    """The q / k / v projections, RoPE and the cache append of one decode step in one launch
    (forwardCached, src/model.nim:775-815).  x_norm [B, n_embd] fp32; weights [out, n_embd] as fp32 or
    bf16 tensors, or uint8 tensors of Q8_0 / Q4_0 blocks with w_type given.  Returns rotated q
    [B, Hq*D] (and rotated k, raw v [B, Hkv*D] with want_kv)."""
    B, n_embd = x_norm.shape
    q = torch.empty((B, n_head * head_dim), dtype=torch.float32, device=x_norm.device)
    k = torch.empty((B, n_kv_head * head_dim), dtype=torch.float32, device=x_norm.device) if want_kv or k_cache is None else None
    v = torch.empty_like(k) if k is not None else None
    check(lib().nimllm_qkv_rope_append(
        _ptr(x_norm), _ptr(wq), _ptr(wk), _ptr(wv), _wtype(wq, w_type), _ptr(q), _ptr(k), _ptr(v), _ptr(cos), _ptr(sin),
        _ptr(seq_pos), pos0, _ptr(k_cache), _ptr(v_cache), _code(k_cache) if k_cache is not None else F32, _ptr(kv_off),
        seq_stride, head_stride, cache_row0, max_seq, B, n_embd, n_head, n_kv_head, head_dim, _stream()))
    return (q, k, v) if k is not None else q


def wo_residual(attn_out, wo, x_resid, *, w_type=None):
    """x_resid + wo attn_out (src/model.nim:843-849) in one launch; attn_out [B, n_in], wo [n_embd, n_in]."""
    B, n_in = attn_out.shape
    n_embd = x_resid.shape[1]
    out = torch.empty_like(x_resid)
    check(lib().nimllm_wo_residual(_ptr(attn_out), _ptr(wo), _wtype(wo, w_type), _ptr(x_resid), _ptr(out), B, n_embd, n_in,
                                   _stream()))
    return out


def matvec(w, x, rows, *, w_type=None, residual=None):
    """y[b] = w x[b] (+ residual[b]); x [B, cols] fp32, w [rows, cols] in any of the weight types."""
    B, cols = x.shape
    y = torch.empty((B, rows), dtype=torch.float32, device=x.device)
    check(lib().nimllm_matvec(_ptr(w), _wtype(w, w_type), _ptr(x), _ptr(residual), _ptr(y), B, rows, cols, _stream()))
    return y


def matvec_status(reset: bool = True) -> int:
    """0 when every staged projection launch since the last reset ran to completion, 1 when a bounded wait
    for weight copies gave up (results of that launch are incomplete).  Synchronises the device."""
    rc = lib().nimllm_matvec_status(int(reset))
    if rc < 0:
        check(-rc)
    return rc


def combine(parts, head_dim, out_dtype=torch.float32, partials=False):
    """Merge (o, m, l) records [n_parts, rows, D+4] -> out [rows, D]."""
    n_parts, rows, W = parts.shape
    out = torch.empty((rows, head_dim), dtype=out_dtype, device=parts.device)
    rec = torch.empty((rows, W), dtype=torch.float32, device=parts.device) if partials else None
    check(lib().nimllm_attn_combine(_ptr(parts), n_parts, rows, head_dim, W, _ptr(out), _code(out), _ptr(rec),
                                    _stream()))
    return (out, rec) if partials else out


def attn_forward(q, k, v, cos, sin, *, n_head, n_kv_head, head_dim, pos0=0, save_cache=True, kv: KvCache = None,
                 layer=0, scale=None, lse=None):
    """forward()'s attention block: RoPE(q, k) then causal GQA attention.
    q [B,S,Hq*D] (or [S,Hq*D]), k, v [B,S,Hkv*D]. q and k are rotated in place like the
    reference's ropeFwd does; with kv given, rows pos0.. of the cache are filled."""
    squeeze = q.dim() == 2
    if squeeze:
        q, k, v = q.unsqueeze(0), k.unsqueeze(0), v.unsqueeze(0)
    B, S = q.shape[0], q.shape[1]
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    out = torch.empty_like(q)
    need = lib().nimllm_attn_prefill_workspace_bytes(B, S, n_head, n_kv_head, head_dim, _code(q))
    ws = _arena.get(need, q.device)
    kc = kv.k[layer] if kv is not None else None
    vc = kv.v[layer] if kv is not None else None
    check(lib().nimllm_attn_prefill(
        _ptr(q), _ptr(k), _ptr(v), _code(q), _ptr(cos), _ptr(sin), pos0, _ptr(out), B, S, n_head, n_kv_head,
        head_dim, scale, int(save_cache), _ptr(kc), _ptr(vc), _code(kc) if kc is not None else F32, None,
        kv.seq_stride if kv is not None else 0, kv.head_stride if kv is not None else 0,
        kv.max_seq if kv is not None else 0, _ptr(lse), _ptr(ws), need, _stream()))
    return out[0] if squeeze else out


def prefill_status(reset: bool = True) -> int:
    """0 when every bf16 prefill launch on the current device since the last reset ran to
    completion, 1 when a bounded wait inside one gave up (its outputs are incomplete).  Synchronises."""
    rc = lib().nimllm_attn_prefill_status(int(reset))
    if rc < 0:
        check(-rc)
    return rc


def attn_backward(q_rot, k_rot, v, out, dout, lse, cos, sin, *, n_head, n_kv_head, head_dim, pos0=0, scale=None):
    """Backward of the causal attention block (fp32): returns (dq, dk, dv) in the pre-RoPE space.
    q_rot / k_rot are the rotated activations attn_forward(save_cache=True) left, lse its row
    log-sum-exp [B, Hq, S]."""
    if q_rot.dim() == 2:
        q_rot, k_rot, v, out, dout = (t.unsqueeze(0) for t in (q_rot, k_rot, v, out, dout))
    B, S = q_rot.shape[0], q_rot.shape[1]
    scale = 1.0 / math.sqrt(head_dim) if scale is None else scale
    dq, dk, dv = torch.empty_like(q_rot), torch.empty_like(k_rot), torch.empty_like(v)
    need = lib().nimllm_attn_prefill_bwd_workspace_bytes(B, S, n_head, head_dim)
    ws = _arena.get(need, q_rot.device)
    check(lib().nimllm_attn_prefill_bwd(
        _ptr(q_rot), _ptr(k_rot), _ptr(v), _ptr(out), _ptr(dout), _ptr(lse), _ptr(cos), _ptr(sin), pos0,
        _ptr(dq), _ptr(dk), _ptr(dv), B, S, n_head, n_kv_head, head_dim, scale, _ptr(ws), need, _stream()))
    return dq, dk, dv


def attn_forward_cached(kv: KvCache, layer, q, k_new, v_new, cos, sin, *, n_head, scale=None, chunk_rows=0):
    """forwardCached()'s attention block for one new token per sequence (newTokens == 1):
    RoPE(q, k_new) at row kv.pos, append, attend rows 0..kv.pos.  q [n_seq, Hq*D],
    k_new / v_new [n_seq, Hkv*D].  The caller advances kv.pos after the last layer, as
    the reference does (src/model.nim:890)."""
    B = q.shape[0]
    D, Hkv = kv.head_dim, kv.n_kv_head
    kc, vc = kv.k[layer], kv.v[layer]
    rope_append(q.view(B, 1, -1), k_new.view(B, 1, -1), v_new.view(B, 1, -1), cos, sin, n_head=n_head,
                n_kv_head=Hkv, head_dim=D, pos0=kv.pos, k_cache=kc, v_cache=vc, seq_stride=kv.seq_stride,
                head_stride=kv.head_stride, max_seq=kv.max_seq)
    return decode_batch(q, kc, vc, n_head=n_head, n_kv_head=Hkv, head_dim=D, max_len=kv.pos + 1,
                        seq_stride=kv.seq_stride, head_stride=kv.head_stride, scale=scale,
                        chunk_rows=chunk_rows, out_dtype=torch.float32)
