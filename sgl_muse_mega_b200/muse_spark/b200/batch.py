"""The cache path of a batched step: several requests on one paged K/V pool, next to the one-request launches of
``headtail.py`` (window feeds) and ``head.py`` (rotation and append inside the qkv head).

A step runs ``BlockTables`` (pages, slots and positions of its new tokens), ``Rotary`` per layer (rotation of q and k by the
rows of a ``RopeTable``, append of k and v at the slots) and ``PrefixAttention`` per layer (the new rows over the pool, the
prefix that all requests share visited once). Each class owns its outputs and scratch, binds once, and ``launch(stream, pdl)``
enqueues it (graph-capturable: lengths are read on the device). A bound object may not overlap itself on two streams.

``status`` (i32 [16]; ``RopeTable`` has nothing to leave out) stays 0 until a launch leaves something out;
``include/mk_abi.h`` lists what.
"""

from __future__ import annotations

from typing import Optional

import torch

from ...common import host

ROPE_KINDS = {"none": 0, "linear": 1, "ntk": 2, "llama3": 3, "yarn": 4}
_ROPE_FIELDS = {
    "none": (), "linear": ("factor",), "ntk": ("factor",),
    "llama3": ("factor", "low_freq_factor", "high_freq_factor", "original_len"),
    "yarn": ("factor", "beta_fast", "beta_slow", "original_len"),
}  # fmt: skip


def _z(*shape, dtype, device):
    return torch.zeros(*shape, dtype=dtype, device=device)


def _check(name: str, t: torch.Tensor, dtype, shape=None, device=None, contiguous: bool = True):
    """The tensor is what the launch will read: type, shape (None: any extent), device, layout."""
    if not isinstance(t, torch.Tensor):
        raise ValueError(f"{name}: not a tensor")
    if t.dtype not in (dtype if isinstance(dtype, tuple) else (dtype,)):
        raise ValueError(f"{name}: dtype {t.dtype}, expected {dtype}")
    if shape is not None and (t.dim() != len(shape) or any(w is not None and s != w for s, w in zip(t.shape, shape))):
        raise ValueError(f"{name}: shape {tuple(t.shape)}, expected {tuple('any' if w is None else w for w in shape)}")
    if device is not None and t.device != device:
        raise ValueError(f"{name}: on {t.device}, expected {device}")
    if contiguous and not t.is_contiguous():
        raise ValueError(f"{name}: not contiguous")


def _heads(name: str, t: torch.Tensor, dtype, shape, device):
    """A [rows, heads, dim] tensor whose rows and heads may be strided (a slice of a fused projection row)."""
    _check(name, t, dtype, shape, device, contiguous=False)
    if t.numel() and t.stride(2) != 1:
        raise ValueError(f"{name}: the last dimension is strided")
    if t.shape[0] > 1 and t.stride(0) < (t.shape[1] - 1) * t.stride(1) + t.shape[2]:
        raise ValueError(f"{name}: rows overlap, or do not hold their heads (heads outermost)")
    if t.shape[1] > 1 and t.stride(1) < t.shape[2]:
        raise ValueError(f"{name}: heads overlap")


def _strides(t: Optional[torch.Tensor]):
    """(row, head) strides in elements; an extent of one has no stride that matters."""
    if t is None:
        return 0, 0
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * t.shape[2], t.stride(1) if t.shape[1] > 1 else t.shape[2]


class BlockTables:
    """Block table, slots and positions of a step from the requests' lengths; takes the new pages from the ring."""

    def __init__(self, lib: host.Library, module, *, seq_lens, new_lens, req_pool_indices, req_to_page, pages_owned, free_pages,
                 free_words, page_size: int, rows: int):  # fmt: skip
        """``seq_lens`` / ``new_lens`` / ``req_pool_indices``: i64 [batch], refreshed by the caller before each launch.
        ``req_to_page`` i32 [pool rows, width], ``pages_owned`` i32 [pool rows], ``free_pages`` i32 [ring] and
        ``free_words`` i64 [2] {head, tail} are the allocator's state, advanced by each launch. ``rows``: the most new
        tokens a step may bring."""
        i32, i64, dev = torch.int32, torch.int64, seq_lens.device
        _check("seq_lens", seq_lens, i64, (None,))
        batch = seq_lens.shape[0]
        _check("new_lens", new_lens, i64, (batch,), dev)
        _check("req_pool_indices", req_pool_indices, i64, (batch,), dev)
        _check("req_to_page", req_to_page, i32, (None, None), dev)
        pool, width = req_to_page.shape
        _check("pages_owned", pages_owned, i32, (pool,), dev)
        _check("free_pages", free_pages, i32, (None,), dev)
        _check("free_words", free_words, i64, (2,), dev)
        if batch < 1 or rows < 1:
            raise ValueError(f"batch {batch} / rows {rows}: at least one of each")
        self.block_table = torch.full((batch, width), -1, dtype=i32, device=dev)
        self.slots = _z(rows, dtype=i64, device=dev)
        self.positions = _z(rows, dtype=i64, device=dev)
        self.cu_rows = _z(batch + 1, dtype=i32, device=dev)
        self.kv_lens = _z(batch, dtype=i32, device=dev)
        self.ticket = _z(1, dtype=i32, device=dev)
        self.status = _z(16, dtype=i32, device=dev)
        self.keep = (seq_lens, new_lens, req_pool_indices, req_to_page, pages_owned, free_pages, free_words)
        self.bind = host.make(
            "MkBlockTablesBind", seq_lens=seq_lens, new_lens=new_lens, req_pool_indices=req_pool_indices, req_to_page=req_to_page,
            pool_rows=pool, width=width, pages_owned=pages_owned, free_pages=free_pages, ring=free_pages.numel(),
            free_words=free_words, page_size=page_size, batch=batch, rows=rows, block_table=self.block_table, slots=self.slots,
            positions=self.positions, cu_rows=self.cu_rows, kv_lens=self.kv_lens, ticket=self.ticket, status=self.status,
        )  # fmt: skip
        self.launch = lib.bind("mk_block_tables_bind", module, self.bind)


class RopeTable:
    """``cos_sin`` f32 [rows, rot]: cos | sin of positions ``first`` .., the layout of every ``cos_sin_cache`` of this package."""

    def __init__(self, lib: host.Library, module, *, rows: int, rot: int, theta: float, device, scaling: Optional[dict] = None,
                 first: int = 0):  # fmt: skip
        """``scaling``: None or ``dict(kind=..., ...)`` with kind ``linear`` / ``ntk`` (factor), ``llama3`` (factor,
        low_freq_factor, high_freq_factor, original_len) or ``yarn`` (factor, beta_fast, beta_slow, original_len)."""
        sc = dict(scaling or {})
        kind = sc.pop("kind", "none")
        if kind not in ROPE_KINDS:
            raise ValueError(f"scaling kind {kind!r} is not one of {sorted(ROPE_KINDS)}")
        if set(sc) != set(_ROPE_FIELDS[kind]):
            raise ValueError(f"scaling {kind!r} takes {_ROPE_FIELDS[kind]}, got {sorted(sc)}")
        if rows < 1 or rot < 8 or rot % 8:
            raise ValueError(f"rows {rows} / rot {rot}: at least one row, rot a multiple of 8")
        self.cos_sin = torch.empty(rows, rot, dtype=torch.float32, device=device)
        fields = dict.fromkeys(("factor", "low_freq_factor", "high_freq_factor", "beta_fast", "beta_slow", "original_len"), 0.0)
        fields.update({k: float(v) for k, v in sc.items()})
        self.bind = host.make("MkRopeTableBind", out=self.cos_sin, rows=rows, first=first, rot=rot, theta=float(theta),
                              kind=ROPE_KINDS[kind], **fields)  # fmt: skip
        self.launch = lib.bind("mk_rope_table_bind", module, self.bind)


class Rotary:
    """Rotates q (into ``q_out``) and k (into ``k_out`` and / or the cache) by their positions, appends k and v."""

    def __init__(self, lib: host.Library, module, *, q, positions, cos_sin_cache, k=None, v=None, slots=None, k_cache=None,
                 v_cache=None, q_out=None, k_out=None, n_rows=None, interleaved: bool = False, inverse: bool = False):  # fmt: skip
        """``q`` / ``k`` / ``v``: bf16 or f16 [rows, heads, dim], rows and heads may be strided (slices of a fused
        projection). ``cos_sin_cache`` f32 [positions, rot]: its width is the number of rotated dims. ``slots`` i64 [rows]:
        pool rows (negative: not appended). ``q_out``: a new tensor unless given; ``q_out=q`` / ``k_out=k`` rotate in
        place. ``n_rows`` i32 [1] on the device: live rows (the rest is left as it was). ``interleaved``: neighbouring pairs
        (the target's heads), else the two halves of the rotated dims (the draft's). ``inverse`` rotates back, which is also the
        rotation's gradient."""
        dev, dt = q.device, q.dtype
        _heads("q", q, (torch.bfloat16, torch.float16), (None, None, None), dev)
        rows, qh, dim = q.shape
        _check("positions", positions, torch.int64, (rows,), dev)
        _check("cos_sin_cache", cos_sin_cache, torch.float32, (None, None), dev)
        kvh, kv_rows = 0, 0
        if k is not None:
            _heads("k", k, dt, (rows, None, dim), dev)
            kvh = k.shape[1]
        if v is not None:
            _heads("v", v, dt, (rows, kvh, dim), dev)
        if k_cache is not None:
            _heads("k_cache", k_cache, dt, (None, kvh, dim), dev)
            kv_rows = k_cache.shape[0]
        if v_cache is not None:
            _heads("v_cache", v_cache, dt, (kv_rows, kvh, dim), dev)
        if slots is not None:
            _check("slots", slots, torch.int64, (rows,), dev)
        self.q_out = q_out if q_out is not None else _z(rows, qh, dim, dtype=dt, device=dev)
        _heads("q_out", self.q_out, dt, (rows, qh, dim), dev)
        self.k_out = k_out
        if k_out is not None:
            _heads("k_out", k_out, dt, (rows, kvh, dim), dev)
        if n_rows is not None:
            _check("n_rows", n_rows, torch.int32, (1,), dev)
        self.status = _z(16, dtype=torch.int32, device=dev)
        self.keep = (q, k, v, positions, cos_sin_cache, slots, k_cache, v_cache, n_rows)
        st = {}
        for name, t in (("q", q), ("k", k), ("v", v), ("qo", self.q_out), ("ko", k_out), ("kc", k_cache), ("vc", v_cache)):
            st[f"{name}_row"], st[f"{name}_head"] = _strides(t)
        self.bind = host.make(
            "MkRotaryBind", q=q, k=k, v=v, q_out=self.q_out, k_out=k_out, positions=positions, cos_sin_cache=cos_sin_cache,
            cos_sin_rows=cos_sin_cache.shape[0], slots=slots, k_cache=k_cache, v_cache=v_cache, kv_rows=kv_rows, n_rows=n_rows,
            rows=rows, q_heads=qh, kv_heads=kvh, head_dim=dim, rot=cos_sin_cache.shape[1], interleaved=int(interleaved),
            inverse=int(inverse), fp16=int(dt == torch.float16), status=self.status, **st,
        )  # fmt: skip
        self.launch = lib.bind("mk_rotary_bind", module, self.bind)


class PrefixAttention:
    """``out`` [rows, q heads, dim]: each request's new rows over its keys in the pool; the first ``prefix_len`` keys, the same
    cache rows for all requests, are visited once for the whole batch (0: plain batched attention)."""

    def __init__(self, lib: host.Library, module, *, q, k_cache, v_cache, block_table, kv_lens, cu_rows, prefix_len,
                 page_size: int, max_new: int, scale: float, window: int = 0, out=None, lse: bool = False):  # fmt: skip
        """``q`` bf16 or f16 [rows, q heads, 64 or 128]; ``k_cache`` / ``v_cache`` [slots, kv heads, dim]; ``block_table`` i32
        [batch, width], ``kv_lens`` i32 [batch] and ``cu_rows`` i32 [batch + 1] as ``BlockTables`` leaves them;
        ``prefix_len`` i32 [1]; ``max_new``: the most rows a request may have; ``window``: keys before its own that a row
        sees (0: all). ``lse``: also the softmax sums' natural logs, f32 [rows, q heads]."""
        dev, dt = q.device, q.dtype
        _heads("q", q, (torch.bfloat16, torch.float16), (None, None, None), dev)
        rows, qh, dim = q.shape
        _heads("k_cache", k_cache, dt, (None, None, dim), dev)
        slots, kvh, _ = k_cache.shape
        _heads("v_cache", v_cache, dt, (slots, kvh, dim), dev)
        i32 = torch.int32
        _check("kv_lens", kv_lens, i32, (None,), dev)
        batch = kv_lens.shape[0]
        _check("cu_rows", cu_rows, i32, (batch + 1,), dev)
        _check("prefix_len", prefix_len, i32, (1,), dev)
        _check("block_table", block_table, i32, (batch, None), dev, contiguous=False)
        if block_table.numel() and block_table.shape[1] > 1 and block_table.stride(1) != 1:
            raise ValueError("block_table: the last dimension is strided")
        self.out = out if out is not None else _z(rows, qh, dim, dtype=dt, device=dev)
        _heads("out", self.out, dt, (rows, qh, dim), dev)
        self.lse = _z(rows, qh, dtype=torch.float32, device=dev) if lse else None
        self.status = _z(16, dtype=i32, device=dev)
        self.keep = (q, k_cache, v_cache, block_table, kv_lens, cu_rows, prefix_len)
        st = {}
        for name, t in (("q", q), ("k", k_cache), ("v", v_cache), ("o", self.out)):
            st[f"{name}_row"], st[f"{name}_head"] = _strides(t)
        fields = dict(
            q=q, k_cache=k_cache, v_cache=v_cache, kv_rows=slots, block_table=block_table,
            table_row=block_table.stride(0) if batch > 1 else block_table.shape[1], width=block_table.shape[1], kv_lens=kv_lens,
            cu_rows=cu_rows, prefix_len=prefix_len, out=self.out, lse=self.lse, rows=rows, batch=batch, max_new=max_new,
            q_heads=qh, kv_heads=kvh, head_dim=dim, page_size=page_size, window=window, scale=float(scale),
            fp16=int(dt == torch.float16), ws=None, ws_bytes=0, status=self.status, **st,
        )  # fmt: skip
        self.consts = lib.prefix_attn_constants(host.make("MkPrefixAttnBind", **fields))
        self.ws = torch.empty(self.consts.ws_bytes, dtype=torch.uint8, device=dev)
        fields.update(ws=self.ws, ws_bytes=self.consts.ws_bytes)
        self.bind = host.make("MkPrefixAttnBind", **fields)
        self.launch = lib.bind("mk_prefix_attn_bind", module, self.bind)
