"""Quantised key/value cache: written, read back and attended over on the GPU.

A policy that keeps looking at what it saw (a stream of observation prefixes, an
instruction that stays) holds its keys and values here, in 4 or 8 bits instead
of 16: pages of 64 tokens from one pool, found through a table of page numbers
per sequence.  The format, the masks and the positions are those of
``vla_kv_cache`` and ``vla_kv_attention_args`` (include/vla_b200.h).

    cache = KVCache(batch=8, max_len=4096, layers=16, bits=4)
    lens = torch.zeros(8, dtype=torch.int32, device="cuda")
    for each step of n new tokens:
        for layer i:
            cache.append(k, v, lens, n, layer=i)                  # at lens[b] ..
            o = cache.attend(q, lens + n, window=2048, sinks=113, layer=i)
        lens += n

Lengths are the caller's int32 tensors on the GPU, so a step can be captured in a
CUDA graph and replayed as the sequences grow.  Every call runs on the current
stream of the cache's device; the memory that it allocates (outputs, workspace)
comes from torch's allocator on that stream.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Tuple

import torch

from . import _lib

BF16 = torch.bfloat16
PAGE = _lib.KV_PAGE
HEAD_DIM = 64


def block_bytes(bits: int) -> int:
    """Bytes of one page's block for one kv head."""
    n = _lib.load().vla_kv_block_bytes(bits)
    if n == 0:
        raise _lib.VlaError(_lib.VLA_E_INVALID, f"a cache holds 4 or 8 bits, not {bits}")
    return n


class KVCache:
    """Paged cache of ``layers`` layers.

    pool   uint8 [layers, pages, kv_heads, block_bytes(bits)]
    table  int32 [batch, max_pages]: page numbers, the same ones in every layer

    Without ``pages`` every sequence owns the ``ceil(max_len / 64)`` pages that
    it can need; with it, the caller fills ``table`` from a pool of that many."""

    def __init__(self, batch: int, max_len: int, kv_heads: int = 5, layers: int = 1, bits: int = 4,
                 pages: Optional[int] = None, device="cuda"):
        per_seq = -(-max_len // PAGE)
        own = pages is None
        pages = batch * per_seq if own else pages
        if own:
            table = torch.arange(pages, dtype=torch.int32, device=device).view(batch, per_seq)
        else:
            table = torch.full((batch, per_seq), -1, dtype=torch.int32, device=device)
        self._bind(torch.empty(layers, pages, kv_heads, block_bytes(bits), dtype=torch.uint8, device=device), table,
                   kv_heads, bits)

    @classmethod
    def wrap(cls, pool: torch.Tensor, table: torch.Tensor, kv_heads: int, bits: int) -> "KVCache":
        """The cache in memory that exists: pool [pages, kv_heads, bytes] (one
        layer) or [layers, pages, kv_heads, bytes], table [batch, max_pages]."""
        self = cls.__new__(cls)
        self._bind(pool if pool.dim() == 4 else pool[None], table, kv_heads, bits)
        return self

    def _bind(self, pool, table, kv_heads, bits):
        if pool.dtype != torch.uint8 or pool.dim() != 4 or not pool.is_contiguous() or pool.shape[2] != kv_heads or \
                pool.shape[3] != block_bytes(bits):
            raise ValueError(f"pool: need contiguous uint8 [layers, pages, {kv_heads}, {block_bytes(bits)}], got "
                             f"{pool.dtype} {tuple(pool.shape)}")
        if table.dtype != torch.int32 or table.dim() != 2 or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError("table: need int32 [batch, max_pages] with unit column stride")
        if table.shape[0] > 1 and table.stride(0) < table.shape[1]:
            raise ValueError(f"table: rows of {table.shape[1]} page numbers overlap at stride {table.stride(0)}: "
                             "need a table with rows of its own, .contiguous()")
        if table.device != pool.device or not pool.is_cuda:
            raise ValueError(f"table is on {table.device}, the pool on {pool.device}: need one CUDA device")
        self.pool, self.table = pool, table
        self.kv_heads, self.bits = kv_heads, bits
        self.batch, self.max_pages = table.shape
        self.layers = pool.shape[0]
        self.device = pool.device
        self._lib = _lib.load()
        self._desc = []
        for i in range(self.layers):
            d = _lib.KVCacheDesc()
            d.pool, d.table = pool[i].data_ptr(), table.data_ptr()
            d.table_ld = max(table.stride(0), self.max_pages)  # a single row may have any stride
            d.pages, d.max_pages, d.batch = pool.shape[1], self.max_pages, self.batch
            d.kv_heads, d.head_dim, d.bits = kv_heads, HEAD_DIM, bits
            self._desc.append((d, ctypes.byref(d)))
        self._append, self._read = self._lib.vla_kv_append_bf16, self._lib.vla_kv_read_bf16
        self._attend = self._lib.vla_kv_attention_bf16
        self._dev = pool.get_device()
        self._per_seq = torch.Size([self.batch])
        self._strides, self._plans = {}, {}  # of shapes and strides: _rows; of sizes: workspace bytes

    # -- arguments ---------------------------------------------------------
    # Calls of a few microseconds: what a shape, its strides and its type say is
    # worked out once per combination, and the device is switched only if it has to be.
    def _index(self, t: Optional[torch.Tensor], name: str) -> Optional[int]:
        if t is None:
            return None
        if t.dtype is not torch.int32 or t.shape != self._per_seq or t.get_device() != self._dev or \
                not t.is_contiguous():
            raise ValueError(f"{name}: need contiguous int32 [{self.batch}] on {self.device}, got {t.dtype} "
                             f"{tuple(t.shape)} on {t.device}")
        return t.data_ptr()

    def _rows(self, x: torch.Tensor, n: int, heads: int, name: str) -> Tuple[int, int]:
        """(row stride, sequence stride) of [batch * n, heads * 64],
        [batch, n, heads * 64] or [batch, n, heads, 64]."""
        key = (x.shape, x.stride(), x.dtype, x.get_device(), n, heads)
        got = self._strides.get(key)
        if got is None:
            if len(self._strides) >= 4096:  # callers with ever new lengths
                self._strides.clear()
            got = self._strides[key] = self._check_rows(x, n, heads, name)
        return got

    def _check_rows(self, x, n, heads, name):
        s, st = tuple(x.shape), x.stride()
        d, width = len(s), heads * HEAD_DIM
        if x.dtype != BF16 or x.device != self.device:
            raise ValueError(f"{name}: need bfloat16 on {self.device}, got {x.dtype} on {x.device}")
        if d == 2 and s == (self.batch * n, width) and st[1] == 1:
            row, batch = st[0], n * st[0]
        elif d == 3 and s == (self.batch, n, width) and st[2] == 1:
            row, batch = st[1], st[0]
        elif d == 4 and s == (self.batch, n, heads, HEAD_DIM) and st[3] == 1 and (heads == 1 or st[2] == HEAD_DIM):
            row, batch = st[1], st[0]
        else:
            raise ValueError(f"{name}: need [{self.batch * n}, {width}], [{self.batch}, {n}, {width}] or "
                             f"[{self.batch}, {n}, {heads}, {HEAD_DIM}] with packed heads, got {s} strides {st}")
        # a single row or sequence may have any stride
        return row if n > 1 or row >= width else width, batch if self.batch > 1 else 0

    def _call(self, fn, *args) -> None:
        if torch._C._cuda_getDevice() == self._dev:
            rc = fn(*args, torch._C._cuda_getCurrentRawStream(self._dev))
        else:
            with torch.cuda.device(self._dev):
                rc = fn(*args, torch._C._cuda_getCurrentRawStream(self._dev))
        if rc != _lib.VLA_OK:
            raise _lib.VlaError(rc, _lib.last_error())

    # -- operators ---------------------------------------------------------
    def append(self, k: torch.Tensor, v: torch.Tensor, start: torch.Tensor, n: int,
               count: Optional[torch.Tensor] = None, layer: int = 0) -> None:
        """Quantise ``n`` rows of K and V per sequence into tokens start[b] .. (the
        first count[b] of them, where given)."""
        h = self.kv_heads
        kr, kb = self._rows(k, n, h, "k")
        vr, vb = self._rows(v, n, h, "v")
        self._call(self._append, self._desc[layer][1], k.data_ptr(), kr, kb, v.data_ptr(), vr, vb, n,
                   self._index(start, "start"), self._index(count, "count"))

    def read(self, n: int, count: Optional[torch.Tensor] = None, start: Optional[torch.Tensor] = None, layer: int = 0,
             out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None) -> Tuple[torch.Tensor, torch.Tensor]:
        """K and V that tokens start[b] .. start[b] + n stand for, bfloat16
        [batch, n, kv_heads * 64]; rows from count[b] on are zeros."""
        h = self.kv_heads
        if out is None:
            w = h * HEAD_DIM
            shape, strides = (self.batch, n, w), (n * w, w, 1)
            out = (torch.empty_strided(shape, strides, dtype=BF16, device=self.device),
                   torch.empty_strided(shape, strides, dtype=BF16, device=self.device))
        k, v = out
        kr, kb = self._rows(k, n, h, "out k")
        vr, vb = self._rows(v, n, h, "out v")
        self._call(self._read, self._desc[layer][1], k.data_ptr(), kr, kb, v.data_ptr(), vr, vb, n,
                   self._index(start, "start"), self._index(count, "count"))
        return out

    def attend(self, q: torch.Tensor, lens: torch.Tensor, causal: bool = True, window: int = 0, sinks: int = 0,
               scale: float = 0.125, q_len: Optional[torch.Tensor] = None, max_len: int = 0, layer: int = 0,
               out: Optional[torch.Tensor] = None) -> torch.Tensor:
        """Attention of q [batch, Lq, heads, 64] (or [batch, Lq, heads * 64]) over
        the first lens[b] tokens; the query tokens are the newest of them (causal)
        or read all of them.  ``window`` keeps the last keys up to each query,
        ``sinks`` the first ones as well."""
        shape = q.shape
        d = len(shape)
        if d not in (3, 4) or shape[-1] % HEAD_DIM or d == 4 and shape[3] != HEAD_DIM:
            raise ValueError(f"q: need [batch, Lq, heads, 64] or [batch, Lq, heads * 64], got {tuple(shape)}")
        if not (0 <= window < 2 ** 31 and 0 <= sinks < 2 ** 31 and 0 <= max_len < 2 ** 31):
            raise ValueError(f"window={window}, sinks={sinks}, max_len={max_len}: need 0 .. 2^31 - 1")
        n, heads = shape[1], shape[2] if d == 4 else shape[2] // HEAD_DIM
        if out is None:
            out = torch.empty_like(q, memory_format=torch.contiguous_format)
        a = _lib.KVAttentionArgs()
        a.q, a.o = q.data_ptr(), out.data_ptr()
        a.q_row, a.q_batch = self._rows(q, n, heads, "q")
        a.o_row, a.o_batch = self._rows(out, n, heads, "out")
        a.lens, a.q_len = self._index(lens, "lens"), self._index(q_len, "q_len")
        a.Lq, a.Hq, a.causal, a.window, a.sinks, a.max_len, a.scale = n, heads, causal, window, sinks, max_len, scale
        desc, args = self._desc[layer][1], ctypes.byref(a)
        key = (n, heads, window, sinks, max_len)
        need = self._plans.get(key)
        new = need is None
        if new:
            with torch.cuda.device(self._dev):
                need = self._lib.vla_kv_attention_workspace(desc, args)
        if need:
            ws = torch.empty_strided((need,), (1,), dtype=torch.uint8, device=self.device)
            a.workspace, a.workspace_bytes = ws.data_ptr(), need
        self._call(self._attend, desc, args)
        if new:  # (0 bytes is also the answer to a call that is refused)
            if len(self._plans) >= 4096:
                self._plans.clear()
            self._plans[key] = need
        return out
